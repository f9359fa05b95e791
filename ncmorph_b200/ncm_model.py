"""Device mirror of ncmorph's NCM body forward (src/ncm_model.zig:77-250) in
bf16 (the layer of src/decoder.zig:168-216), plus the per-op entry points it
is built from: RMSNorm, embedding gather, RoPE tables and masked attention.

Masks: "causal" (kernels.causal_mask), "block_diagonal" (ncm_mask.zig:10-42,
ncmorph's only NCM mask) and "block_causal" (each level also attends to
every earlier level; the BASELINE config-4 pattern).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field

import numpy as np
import torch

from . import _lib
from .device import context, context_of, empty_rows, need, need_rows, need_vec, ptr, raw_stream, stream_of

MASK_MODES = {"causal": 0, "block_diagonal": 1, "block_causal": 2}
bf16 = torch.bfloat16
LOGIT_TYPES = {torch.float32: 2, bf16: 0}  # NCM_DTYPE_F32, NCM_DTYPE_BF16


def make_mask(mode: str, prefix_length: int = 0, level_lengths=(), prefix_pad=(),
              sliding_window: int | None = None) -> _lib.Mask:
    m = _lib.Mask()
    m.mode = MASK_MODES[mode]
    m.sliding_window = int(sliding_window or 0)
    m.prefix_length = int(prefix_length)
    bits = 0
    for i, padded in enumerate(prefix_pad):
        if padded:
            bits |= 1 << i
    m.prefix_pad_mask = bits
    m.num_levels = len(level_lengths)
    for i, n in enumerate(level_lengths):
        m.level_lengths[i] = int(n)
    return m


def level_positions(prefix_length: int, level_lengths) -> np.ndarray:
    """ncm_position.fill_level_positions (src/ncm_position.zig:11-22)."""
    pos = list(range(prefix_length))
    for n in level_lengths:
        pos.extend(range(n))
    return np.asarray(pos, dtype=np.int32)


def rope_tables(head_dim: int, theta: float, positions, llama3: tuple | None = None
                ) -> tuple[np.ndarray, np.ndarray]:
    """Host RoPE tables [T, head_dim] with libm, as the reference builds them:
    rope_default's frequencies, or rope_llama3's when `llama3` = (factor,
    low_freq_factor, high_freq_factor, original_max_position_embeddings)."""
    pos = np.ascontiguousarray(positions, dtype=np.int32)
    T = pos.size
    c = np.empty((T, head_dim), np.float32)
    s = np.empty((T, head_dim), np.float32)
    vp = ctypes.c_void_p
    if llama3 is None:
        _lib.call("ncm_rope_tables_host", head_dim, float(theta), vp(pos.ctypes.data), T, vp(c.ctypes.data),
                  vp(s.ctypes.data))
    else:
        factor, low, high, orig = llama3
        _lib.call("ncm_rope_tables_llama3_host", head_dim, float(theta), float(factor), float(low), float(high),
                  int(orig), vp(pos.ctypes.data), T, vp(c.ctypes.data), vp(s.ctypes.data))
    return c, s


def rope_bf16(x: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, heads: int, head_dim: int,
              interleaved: bool = False, inverse: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions of the first `heads` heads of each row of x [T, >= heads *
    head_dim] bf16 (rows may be strided, e.g. fused QKV rows), row t at position
    positions[t] (int32) of the tables cos/sin [P, rotary_dim] f32 (rope_tables
    for positions 0..P-1). rotary_dim columns of every head are rotated, as
    halves (i, i + rotary_dim / 2) or, interleaved, as neighbours (2i, 2i + 1);
    the others are copied. Rounded once to bf16. `inverse` rotates back: the
    gradient. `out`: where to write (x itself: in place), default a new
    [T, heads * head_dim]."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    dev = x.device
    width = heads * head_dim
    stride = need_rows(x, bf16, "x", dev, width)
    T = x.shape[0]
    P, rotary = cos.shape
    if need_rows(cos, torch.float32, "cos", dev, rotary) != rotary and P > 1 or sin.shape != cos.shape or \
            need_rows(sin, torch.float32, "sin", dev, rotary) != rotary and P > 1:
        raise ValueError(f"cos and sin must be contiguous and of one shape, got {tuple(cos.shape)} and {tuple(sin.shape)}")
    pos = need_vec(positions, torch.int32, "positions", dev, T)
    if out is None:
        out, out_stride = empty_rows(T, width, bf16, dev), width
    else:
        out_stride = need_rows(out, bf16, "out", dev, width)
        if out.shape[0] != T:
            raise ValueError(f"out must have {T} rows, got {out.shape[0]}")
    _lib.call("ncm_rope_bf16", context_of(dev), x.data_ptr(), stride, out.data_ptr(), out_stride, pos, cos.data_ptr(),
              sin.data_ptr(), P, T, heads, head_dim, rotary, interleaved, inverse, raw_stream(dev))
    return out


def rms_norm_bf16(x: torch.Tensor, weight: torch.Tensor, eps: float, bias: torch.Tensor | None = None):
    rows, width = x.shape
    need(x, bf16, "x")
    need(weight, bf16, "weight", (width,))
    y = torch.empty_like(x)
    _lib.call("ncm_rms_norm_bf16", context(x.device), ptr(x), ptr(weight), ptr(bias), ptr(y), rows, width,
              float(eps), stream_of(x))
    return y


def embedding_gather(table: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
    vocab, width = table.shape
    need(table, bf16, "table")
    need(ids, torch.int32, "ids")
    out = torch.empty((ids.numel(), width), dtype=bf16, device=table.device)
    _lib.call("ncm_embedding_gather", context(table.device), ptr(table), vocab, width, ptr(ids), ids.numel(),
              ptr(out), stream_of(table))
    return out


def attention_bf16(qkv: torch.Tensor, heads: int, kv_heads: int, mask: _lib.Mask,
                   cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                   q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                   eps: float = 1e-6) -> torch.Tensor:
    """Context [T, heads*64] from fused QKV rows [T, (heads + 2*kv_heads)*64];
    QK-norm (if q_norm/k_norm [64] bf16 are given, with eps) and then RoPE (if
    cos/sin given) are applied to qkv in place."""
    T, stride = qkv.shape
    need(qkv, bf16, "qkv")
    out = torch.empty((T, heads * 64), dtype=bf16, device=qkv.device)
    if q_norm is None and k_norm is None:
        _lib.call("ncm_attention_bf16", context(qkv.device), ptr(qkv), stride, ptr(cos), ptr(sin), ptr(out), T, heads,
                  kv_heads, ctypes.byref(mask), stream_of(qkv))
    else:
        _lib.call("ncm_attention_qk_norm_bf16", context(qkv.device), ptr(qkv), stride, ptr(cos), ptr(sin),
                  ptr(q_norm), ptr(k_norm), eps, ptr(out), T, heads, kv_heads, ctypes.byref(mask), stream_of(qkv))
    return out


@dataclass
class LayerWeights:
    ln_1: torch.Tensor
    qkv: torch.Tensor
    o: torch.Tensor
    ln_2: torch.Tensor
    gate_up: torch.Tensor
    down: torch.Tensor
    qkv_bias: torch.Tensor | None = None
    o_bias: torch.Tensor | None = None
    # QK-norm scales [64] bf16 (ncm_model.zig:42-43): both or None
    q_norm: torch.Tensor | None = None
    k_norm: torch.Tensor | None = None


@dataclass
class Weights:
    input_projection: torch.Tensor
    input_projection_bias: torch.Tensor
    level_embedding: torch.Tensor
    final_norm: torch.Tensor
    layers: list = field(default_factory=list)
    final_norm_bias: torch.Tensor | None = None
    # post_upsample_convs (ncm_model.zig:71): [levels, vq, vq, 3] bf16 and [levels, vq] f32
    post_conv_weight: torch.Tensor | None = None
    post_conv_bias: torch.Tensor | None = None


@dataclass
class Config:
    hidden_size: int
    vq_width: int
    num_attention_heads: int
    num_key_value_heads: int
    intermediate_size: int
    level_lengths: tuple
    prefix_length: int = 0
    # "causal" is ncm_model's source_causal (src/ncm_model.zig:199-203), which
    # may carry a sliding window; the block masks take none
    mask: str = "block_causal"
    sliding_window: int | None = None
    rms_norm_epsilon: float = 1e-5
    rope_theta: float = 500000.0
    use_level_encoding: bool = True
    head_dim: int = 64
    # Llama 3 frequency scaling (rope_llama3, packages/kernels/root.zig:636-666):
    # (factor, low_freq_factor, high_freq_factor, original_max_position_embeddings),
    # or None for rope_default
    rope_llama3: tuple | None = None

    @property
    def seq_len(self) -> int:
        return self.prefix_length + sum(self.level_lengths)


def _vp(t):
    return None if t is None else t.data_ptr()


def forward(cfg: Config, w: Weights, inputs: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """ncm_model.forward on the GPU: inputs [T, vq_width] bf16 -> hidden [T, hidden] bf16."""
    T = cfg.seq_len
    need(inputs, bf16, "inputs", (T, cfg.vq_width))
    c = _lib.DecoderConfig()
    c.hidden_size, c.vq_width = cfg.hidden_size, cfg.vq_width
    c.num_attention_heads, c.num_key_value_heads = cfg.num_attention_heads, cfg.num_key_value_heads
    c.head_dim, c.intermediate_size = cfg.head_dim, cfg.intermediate_size
    c.rms_norm_epsilon, c.rope_theta = cfg.rms_norm_epsilon, cfg.rope_theta
    c.use_level_encoding = int(cfg.use_level_encoding)
    c.mask = make_mask(cfg.mask, cfg.prefix_length, cfg.level_lengths, sliding_window=cfg.sliding_window)
    if cfg.rope_llama3 is not None:
        c.rope_type = 1
        (c.rope_factor, c.rope_low_freq_factor, c.rope_high_freq_factor,
         c.rope_original_max_position_embeddings) = cfg.rope_llama3
    layers = (_lib.DecoderLayerWeights * len(w.layers))()
    for i, L in enumerate(w.layers):
        for name in ("ln_1", "qkv", "qkv_bias", "o", "o_bias", "ln_2", "gate_up", "down", "q_norm", "k_norm"):
            setattr(layers[i], name, _vp(getattr(L, name)))
    W = _lib.DecoderWeights()
    W.input_projection = _vp(w.input_projection)
    W.input_projection_bias = _vp(w.input_projection_bias)
    W.level_embedding = _vp(w.level_embedding)
    W.final_norm = _vp(w.final_norm)
    W.final_norm_bias = _vp(w.final_norm_bias)
    W.num_layers = len(w.layers)
    W.layers = layers
    if w.post_conv_weight is not None:
        L, V = len(cfg.level_lengths), cfg.vq_width
        need(w.post_conv_weight, bf16, "post_conv_weight", (L, V, V, 3))
        need(w.post_conv_bias, torch.float32, "post_conv_bias", (L, V))
    W.post_conv_weight = _vp(w.post_conv_weight)
    W.post_conv_bias = _vp(w.post_conv_bias)
    if out is None:
        out = torch.empty((T, cfg.hidden_size), dtype=bf16, device=inputs.device)
    _lib.call("ncm_ncm_forward", context(inputs.device), ctypes.byref(c), ctypes.byref(W), ptr(inputs), ptr(out),
              stream_of(inputs))
    return out


def apply_post_upsample_conv(input: np.ndarray, weight: np.ndarray, bias: np.ndarray, row_count: int, width: int,
                             device: int = 0) -> None:
    """ncm_model.apply_post_upsample_conv (src/ncm_model.zig:296-326) on the GPU:
    input [row_count, width] f32 (host) becomes input + bias + Conv1d_k3(input)
    in place; weight [width, width, 3] and bias [width] are f32 host arrays
    holding bf16 values. The convolution runs on tcgen05 with bf16 operands."""
    for a, n, name in ((input, row_count * width, "input"), (weight, width * width * 3, "weight"),
                       (bias, width, "bias")):
        if not isinstance(a, np.ndarray) or a.dtype != np.float32 or not a.flags.c_contiguous:
            raise TypeError(f"{name} must be a C-contiguous float32 numpy array")
        if a.size != n:
            raise ValueError(f"{name} has {a.size} elements, expected {n}")
    _lib.call("ncm_post_upsample_conv_host_f32", context(device), ctypes.c_void_p(input.ctypes.data),
              ctypes.c_void_p(weight.ctypes.data), ctypes.c_void_p(bias.ctypes.data), row_count, width)


def tied_head_logits(z: torch.Tensor, codebook: torch.Tensor, log_inv_T: float = 0.0,
                     bias: torch.Tensor | None = None, esq: torch.Tensor | None = None) -> torch.Tensor:
    """_TiedCodebookHead (PROJECT.md:222): logits [T, K] f32 =
    (2 z.E^T - E_sq) / mean(E_sq) * exp(log_inv_T) + bias, z [T, d] bf16, E [K, d] bf16."""
    T, d = z.shape
    K = codebook.shape[0]
    need(z, bf16, "z")
    need(codebook, bf16, "codebook", (K, d))
    for t, name in ((bias, "bias"), (esq, "esq")):
        if t is not None:
            need(t, torch.float32, name, (K,))
    out = torch.empty((T, K), dtype=torch.float32, device=z.device)
    _lib.call("ncm_tied_head_logits", context(z.device), ptr(z), ptr(codebook), ptr(esq), ptr(bias),
              float(log_inv_T), ptr(out), T, d, K, stream_of(z))
    return out


def tied_head_argmax(z: torch.Tensor, codebook: torch.Tensor, log_inv_T: float = 0.0,
                     bias: torch.Tensor | None = None, esq: torch.Tensor | None = None) -> torch.Tensor:
    """argmax_k of tied_head_logits (lowest k on ties) without materialising the logits -> int32 [T]."""
    T, d = z.shape
    K = codebook.shape[0]
    need(z, bf16, "z")
    need(codebook, bf16, "codebook", (K, d))
    for t, name in ((bias, "bias"), (esq, "esq")):
        if t is not None:
            need(t, torch.float32, name, (K,))
    codes = torch.empty(T, dtype=torch.int32, device=z.device)
    _lib.call("ncm_tied_head_argmax", context(z.device), ptr(z), ptr(codebook), ptr(esq), ptr(bias),
              float(log_inv_T), ptr(codes), T, d, K, stream_of(z))
    return codes


def process_logits(logits: torch.Tensor, tokens: torch.Tensor | None = None, token_start: torch.Tensor | None = None,
                   prompt_lens: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                   bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   bias_start: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                   allowed_rows: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Penalties, biases and grammar masks on next-token logits [R, V] (f32 or
    bf16, rows may be strided), as ncm_logits_process documents them; returns
    f32 [R, V], or writes to `out` (f32, or bf16 for bf16 logits; logits itself:
    in place). Row r's history is tokens[token_start[r] : token_start[r + 1]]
    (int32), the first prompt_lens[r] of it its prompt. repetition, frequency,
    presence [R] f32. Biases are bias[bias_start[r] : bias_start[r + 1]] of the
    tokens bias_ids. allowed [M, ceil(V / 32)] int32 holds bit masks (bit v % 32
    of word v / 32: token v may follow); row r uses mask allowed_rows[r] (int32,
    -1: none), or mask r."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor")
    if logits.dtype not in (torch.float32, bf16):
        raise TypeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [rows, vocab], got {tuple(logits.shape)}")
    dev = logits.device
    R, V = logits.shape
    stride = need_rows(logits, logits.dtype, "logits", dev, V)
    if out is None:
        out, out_stride = empty_rows(R, V, torch.float32, dev), V
    else:
        if not isinstance(out, torch.Tensor) or out.dtype not in (torch.float32, logits.dtype):
            raise TypeError(f"out must be a float32 or {logits.dtype} tensor")
        out_stride = need_rows(out, out.dtype, "out", dev, V)
        if tuple(out.shape) != (R, V):
            raise ValueError(f"out must have shape {(R, V)}, got {tuple(out.shape)}")
    i32, f32 = torch.int32, torch.float32
    r = _lib.LogitRules()
    if tokens is not None:
        r.tokens = need_vec(tokens, i32, "tokens", dev)
        r.num_tokens = tokens.shape[0]
        r.token_start = need_vec(token_start, i32, "token_start", dev, R + 1)
        r.prompt_lens = need_vec(prompt_lens, i32, "prompt_lens", dev, R)
        if r.num_tokens == 0:  # (an empty tensor has no address; no history yet is a history)
            r.tokens = r.token_start
    elif prompt_lens is not None or token_start is not None:
        raise ValueError("token_start and prompt_lens need tokens")
    r.repetition = need_vec(repetition, f32, "repetition", dev, R)
    r.frequency = need_vec(frequency, f32, "frequency", dev, R)
    r.presence = need_vec(presence, f32, "presence", dev, R)
    if bias is not None:
        r.bias = need_vec(bias, f32, "bias", dev)
        r.num_bias = bias.shape[0]
        r.bias_ids = need_vec(bias_ids, i32, "bias_ids", dev, bias.shape[0])
        r.bias_start = need_vec(bias_start, i32, "bias_start", dev, R + 1)
    elif bias_ids is not None or bias_start is not None:
        raise ValueError("bias_ids and bias_start need bias")
    if allowed is not None:
        r.allowed_stride = need_rows(allowed, i32, "allowed", dev, (V + 31) // 32)
        r.allowed = allowed.data_ptr()
        r.allowed_count = allowed.shape[0]
        if r.allowed_count == 0 and R > 0:
            raise ValueError("allowed must hold at least one mask")
        r.allowed_rows = need_vec(allowed_rows, i32, "allowed_rows", dev, R)
    elif allowed_rows is not None:
        raise ValueError("allowed_rows needs allowed")
    _lib.call("ncm_logits_process", context_of(dev), logits.data_ptr(), LOGIT_TYPES[logits.dtype], stride, out.data_ptr(),
              LOGIT_TYPES[out.dtype], out_stride, R, V, ctypes.byref(r), raw_stream(dev))
    return out
