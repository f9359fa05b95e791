"""A paged key/value cache for decode steps and the attention over it.

One layer of a step, on fused QKV rows [T, (H + 2 Hkv) * head_dim] as
``kernels.linear_bf16`` writes them::

    ncm_model.rope_bf16(qkv, positions, cos, sin, H + Hkv, head_dim, out=qkv)
    kv_cache.append(cache, k_columns, v_columns, token_start, kv_lens, page_table)
    ctx = kv_cache.tree_attention(q_columns, cache, token_start, kv_lens, page_table, max_nodes=n)

``token_start`` [B + 1], ``kv_lens`` [B] and ``page_table`` [B, width] are int32
device tensors: sequence b's new tokens are rows token_start[b] ..
token_start[b + 1], and kv_lens[b] counts its keys with them. Position p lives
in slot p % page_size of page page_table[b, p // page_size].

After drafted tokens are verified, ``append`` the accepted ones' rows again, from the
step's own QKV rows and with ``kv_lens`` that count only them: they lie behind the context
then, quantised once.

ncmorph recomputes every position on each call (src/decoder.zig:50-58) and has no
counterpart. There is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .device import context_of, empty_rows, need_rows, need_vec, raw_stream

bf16, i32 = torch.bfloat16, torch.int32
FORMATS = {bf16: 0, torch.int8: 1, torch.float8_e4m3fn: 2}


class KVCache:
    """One layer's cache: pools k and v [pages, kv_heads, page_size, head_dim] in
    bf16, int8 or float8_e4m3fn, the quantised ones with one f32 scale per
    (page, head, slot). Holds the tensors it is given (`allocate` makes them) and
    nothing else, so several caches may share pools."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if not isinstance(k, torch.Tensor) or not isinstance(v, torch.Tensor) or not k.is_cuda:
            raise ValueError("k and v must be CUDA tensors")
        if k.dtype not in FORMATS or v.dtype != k.dtype:
            raise TypeError(f"k and v must both be bfloat16, int8 or float8_e4m3fn, got {k.dtype} and {v.dtype}")
        if k.dim() != 4 or v.shape != k.shape or v.device != k.device or not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("k and v must be contiguous [pages, kv_heads, page_size, head_dim] tensors of one device")
        if (k.dtype == bf16) != (k_scale is None) or (k.dtype == bf16) != (v_scale is None):
            raise ValueError("a quantised cache has k_scale and v_scale, a bfloat16 one has none")
        for s, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if s is not None and (s.dtype != torch.float32 or s.shape != k.shape[:3] or s.device != k.device or
                                  not s.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous float32 {tuple(k.shape[:3])} tensor on {k.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device = k.device
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.width = self.kv_heads * self.head_dim
        c = self._c = _lib.KvCache()
        c.k, c.v = k.data_ptr(), v.data_ptr()
        if k_scale is not None:
            c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        c.format = FORMATS[k.dtype]
        c.num_pages, c.kv_heads, c.page_size, c.head_dim = k.shape
        self._ref = ctypes.byref(c)
        self._workspaces = {}  # sizes by call shape

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = bf16,
                 device: int | torch.device | str = "cuda") -> "KVCache":
        """A cache with new pools (their contents are not initialised)."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype == bf16:
            return cls(k, v)
        return cls(k, v, *(torch.empty(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))


def _batch(cache: KVCache, token_start: torch.Tensor, kv_lens: torch.Tensor | None, page_table: torch.Tensor,
           rows: int) -> _lib.KvBatch:
    dev = cache.device
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2:
        raise ValueError("page_table must be a [batch, pages] tensor")
    B, width = page_table.shape
    b = _lib.KvBatch()
    b.table_stride = need_rows(page_table, i32, "page_table", dev, width)
    b.page_table = page_table.data_ptr()
    b.table_width, b.batch, b.rows = width, B, rows
    b.token_start = need_vec(token_start, i32, "token_start", dev, B + 1)
    b.kv_lens = need_vec(kv_lens, i32, "kv_lens", dev, B)
    return b


def append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, token_start: torch.Tensor, kv_lens: torch.Tensor,
           page_table: torch.Tensor) -> None:
    """Writes the new tokens' rows k and v [T, kv_heads * head_dim] bf16 (rows may
    be strided) behind what their sequences hold, quantised to the cache's
    format: code = round(127 x / A) with scale A / 127 (int8) or 448 for e4m3, A
    the largest magnitude of a token's head. A row with a NaN or an infinity
    reads back as NaN."""
    dev = cache.device
    ks, vs = need_rows(k, bf16, "k", dev, cache.width), need_rows(v, bf16, "v", dev, cache.width)
    if v.shape[0] != k.shape[0]:
        raise ValueError(f"k and v must have the same rows, got {k.shape[0]} and {v.shape[0]}")
    b = _batch(cache, token_start, kv_lens, page_table, k.shape[0])
    _lib.call("ncm_kv_cache_append", context_of(dev), cache._ref, ctypes.byref(b), k.data_ptr(), ks, v.data_ptr(), vs,
              raw_stream(dev))


def gather(cache: KVCache, row_start: torch.Tensor, page_table: torch.Tensor, rows: int | None = None,
           begin: torch.Tensor | None = None, out_k: torch.Tensor | None = None, out_v: torch.Tensor | None = None
           ) -> tuple[torch.Tensor, torch.Tensor]:
    """Reads positions back as bf16 rows [rows, kv_heads * head_dim]: row
    row_start[b] + i is position begin[b] + i of sequence b (begin None: 0).
    out_k / out_v may be column slices of wider rows (fused QKV rows for
    ncm_model.attention_bf16); without them `rows` says how many to make."""
    dev, width = cache.device, cache.width
    if rows is None:
        if out_k is None or out_v is None:
            raise ValueError("rows is needed without out_k and out_v")
        rows = out_k.shape[0] if isinstance(out_k, torch.Tensor) and out_k.dim() == 2 else 0
    ks = vs = width
    if out_k is None:
        out_k = empty_rows(rows, width, bf16, dev)
    else:
        ks = need_rows(out_k, bf16, "out_k", dev, width)
    if out_v is None:
        out_v = empty_rows(rows, width, bf16, dev)
    else:
        vs = need_rows(out_v, bf16, "out_v", dev, width)
    if out_k.shape[0] != rows or out_v.shape[0] != rows:
        raise ValueError("out_k and out_v must have the same rows")
    b = _batch(cache, row_start, None, page_table, rows)
    _lib.call("ncm_kv_cache_gather", context_of(dev), cache._ref, ctypes.byref(b),
              need_vec(begin, i32, "begin", dev, b.batch), out_k.data_ptr(), ks, out_v.data_ptr(), vs, raw_stream(dev))
    return out_k, out_v


def tree_attention(q: torch.Tensor, cache: KVCache, token_start: torch.Tensor, kv_lens: torch.Tensor,
                   page_table: torch.Tensor, max_nodes: int, tree_mask: torch.Tensor | None = None,
                   scale: float | None = None, heads: int | None = None, out: torch.Tensor | None = None,
                   return_lse: bool = False):
    """Attention of every sequence's new tokens (already appended) over its keys:
    q [T, heads * head_dim] bf16 (rows may be strided; heads defaults to what q's
    columns hold) -> [T, heads * head_dim] bf16, and with return_lse the log of
    the softmax sums [T, heads] f32. A new token sees every key in front of the new
    tokens, itself and the earlier new ones; with tree_mask [T, words] int32 those
    new tokens j whose bit j % 32 of word j / 32 is set. max_nodes bounds the new tokens of
    a sequence (at most 1024; a sequence with more is skipped and reported by
    device.sync) and picks the kernel, so give it what the step has at most. scale
    defaults to head_dim ** -0.5. A token that sees nothing gets zeros and -inf."""
    dev, hd = cache.device, cache.head_dim
    if heads is None:
        if not isinstance(q, torch.Tensor) or q.dim() != 2 or q.shape[1] % hd:
            raise ValueError(f"q must be a matrix of heads of {hd} columns")
        heads = q.shape[1] // hd
    width = heads * hd
    qs = need_rows(q, bf16, "q", dev, width)
    T = q.shape[0]
    b = _batch(cache, token_start, kv_lens, page_table, T)
    words = 0
    if tree_mask is not None:
        if not isinstance(tree_mask, torch.Tensor) or tree_mask.dim() != 2 or tree_mask.dtype != i32 or \
                tree_mask.device != dev or tree_mask.shape[0] != T or not tree_mask.is_contiguous() or \
                tree_mask.shape[1] < 1:  # (an empty mask has no address, and would be none)
            raise ValueError(f"tree_mask must be a contiguous int32 [{T}, words] tensor on {dev}")
        words = tree_mask.shape[1]
    if out is None:
        out, os_ = empty_rows(T, width, bf16, dev), width
    else:
        os_ = need_rows(out, bf16, "out", dev, width)
        if out.shape[0] != T:
            raise ValueError(f"out must have {T} rows, got {out.shape[0]}")
    lse = empty_rows(T, heads, torch.float32, dev) if return_lse else None
    ctx, bref = context_of(dev), ctypes.byref(b)
    # the size depends on nothing but these numbers
    size = cache._workspaces.get((heads, max_nodes, b.table_width, b.batch))
    if size is None:
        n = ctypes.c_uint64()
        _lib.call("ncm_tree_attention_workspace", ctx, cache._ref, bref, heads, max_nodes, ctypes.byref(n))
        if len(cache._workspaces) >= 256:
            cache._workspaces.clear()
        size = cache._workspaces[heads, max_nodes, b.table_width, b.batch] = n.value
    # (new memory for every call: calls on other streams and captured graphs share none)
    ws = empty_rows(1, size, torch.uint8, dev) if size else None
    _lib.call("ncm_tree_attention", ctx, cache._ref, bref, q.data_ptr(), qs,
              None if tree_mask is None else tree_mask.data_ptr(), words, heads, max_nodes,
              hd ** -0.5 if scale is None else scale, out.data_ptr(), os_, None if lse is None else lse.data_ptr(),
              None if ws is None else ws.data_ptr(), size, raw_stream(dev))
    return (out, lse) if return_lse else out
