"""The operators of a decode step through the public entry points, against their
definitions in 64 bits: rotary rows, the paged cache, attention of new tokens
over it, and the rules on logits.

Tolerances count roundings, each at most half a step relative to its value: 2^-8
for bf16, 2^-24 for f32.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = 2.0 ** -8, 2.0 ** -24
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FORMATS = [torch.bfloat16, torch.int8, torch.float8_e4m3fn]


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_dev):
    from ncmorph_b200 import device
    yield
    device.sync(cuda_dev)


def expect_range_error(dev):
    from ncmorph_b200 import _lib, device
    with pytest.raises(_lib.NcmError) as e:
        device.sync(dev)
    assert e.value.status == _lib.NCM_ERANGE


# ----------------------------------------------------------------- rotary rows

def tables(rows, rotary, dev):
    from ncmorph_b200 import ncm_model
    c, s = ncm_model.rope_tables(rotary, 10000.0, np.arange(rows))
    return torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev)


def rope_ref(x, pos, cos, sin, heads, hd, interleaved, inverse):
    T, r = x.shape[0], cos.shape[1]
    h = r // 2
    y = x[:, :heads * hd].double().reshape(T, heads, hd).clone()
    size = torch.zeros_like(y)
    c, s = cos[pos.long(), None, :h].double(), sin[pos.long(), None, :h].double()
    s = -s if inverse else s
    i = torch.arange(h)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    p, q = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = p * c - q * s, q * c + p * s
    size[..., a], size[..., b] = (p * c).abs() + (q * s).abs(), (q * c).abs() + (p * s).abs()
    return y.reshape(T, -1), size.reshape(T, -1)


@pytest.mark.parametrize("T,heads,hd,rotary", [(1, 1, 64, 64), (7, 5, 64, 32), (3, 40, 128, 64), (33, 3, 80, 20), (5, 2, 96, 96),
                                              (1000, 12, 64, 64), (2, 1, 6, 4), (9, 1, 2, 2), (4, 7, 16, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_rope_rows(cuda_dev, T, heads, hd, rotary, interleaved, inverse):
    from ncmorph_b200 import ncm_model
    g = torch.Generator().manual_seed(T * 31 + hd)
    x = torch.randn((T, heads * hd + 24), generator=g).to(torch.bfloat16)
    pos = torch.randint(0, 300, (T,), generator=g, dtype=torch.int32)
    cos, sin = tables(300, rotary, cuda_dev)
    xd = x.to(cuda_dev)
    y = ncm_model.rope_bf16(xd, pos.to(cuda_dev), cos, sin, heads, hd, interleaved=interleaved, inverse=inverse)
    ref, size = rope_ref(x, pos, cos.cpu(), sin.cpu(), heads, hd, interleaved, inverse)
    assert torch.all((y.cpu().double() - ref).abs() <= BF * ref.abs() + 3 * F32 * size)
    # in place on strided rows, columns behind the heads untouched; the same bits
    z = ncm_model.rope_bf16(xd, pos.to(cuda_dev), cos, sin, heads, hd, interleaved=interleaved, inverse=inverse, out=xd)
    assert z is xd and torch.equal(xd[:, :heads * hd], y) and torch.equal(xd[:, heads * hd:].cpu(), x[:, heads * hd:])


@pytest.mark.parametrize("shift", [1, 4])
def test_rope_unaligned_rows_have_the_same_bits(cuda_dev, shift):
    from ncmorph_b200 import ncm_model
    x = torch.randn((11, 3 * 64 + 40), device=cuda_dev).to(torch.bfloat16)
    pos = torch.arange(11, dtype=torch.int32, device=cuda_dev)
    cos, sin = tables(11, 48, cuda_dev)
    for inter in (False, True):
        want = ncm_model.rope_bf16(x[:, shift:].contiguous(), pos, cos, sin, 3, 64, interleaved=inter)
        assert torch.equal(ncm_model.rope_bf16(x[:, shift:], pos, cos, sin, 3, 64, interleaved=inter), want)


def test_rope_gradient(cuda_dev):
    """The inverse rotation is the gradient: against the formula's Jacobian in 64
    bits, and against differences of the 64-bit rotation."""
    from ncmorph_b200 import ncm_model
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 50, (4,), generator=g, dtype=torch.int32)
    cos, sin = tables(50, 32, cuda_dev)
    x, up = (torch.randn((4, 2 * 64), generator=g).to(torch.bfloat16) for _ in range(2))
    for inter in (False, True):
        dx = ncm_model.rope_bf16(up.to(cuda_dev), pos.to(cuda_dev), cos, sin, 2, 64, interleaved=inter, inverse=True).cpu().double()
        f = lambda v: rope_ref(v, pos, cos.cpu(), sin.cpu(), 2, 64, inter, False)[0]  # noqa: B023,E731
        v = x.double().requires_grad_()
        (f(v) * up.double()).sum().backward()
        bound = BF * v.grad.abs() + 4 * F32 * (1 + v.grad.abs()) * 8
        assert torch.all((dx - v.grad).abs() <= bound)
        for i, j in ((0, 0), (1, 33), (3, 70), (2, 127)):
            d = torch.zeros_like(x, dtype=torch.float64)
            d[i, j] = 1e-4
            slope = ((f(x.double() + d) - f(x.double() - d)) * up.double()).sum() / 2e-4
            assert abs(dx[i, j] - slope) <= bound[i, j] + 1e-9


def test_rope_position_out_of_the_table(cuda_dev):
    from ncmorph_b200 import ncm_model
    x = torch.randn((5, 64), device=cuda_dev).to(torch.bfloat16)
    cos, sin = tables(8, 64, cuda_dev)
    out = torch.full_like(x, 7.0)
    pos = torch.tensor([0, -1, 7, 8, 3], dtype=torch.int32, device=cuda_dev)
    ncm_model.rope_bf16(x, pos, cos, sin, 1, 64, out=out)
    expect_range_error(cuda_dev)
    assert torch.all(out[[1, 3]] == 7.0) and not torch.any(out[[0, 2, 4]] == 7.0)


# ------------------------------------------------------------------- the cache

def grid_e4m3(y):
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(y / step) * step


def quantise_ref(x, dtype):
    """Codes (as values) and scales of rows [..., head_dim], in 64 bits."""
    x = x.double()
    big = x.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(x).all(-1, keepdim=True)
    y = torch.where(fine & (big > 0), x * TOP[dtype] / torch.where(big > 0, big, 1.0), 0.0)
    codes = torch.round(y) if dtype == torch.int8 else grid_e4m3(y)
    scale = torch.where(fine, torch.where(big > 0, big / TOP[dtype], 1.0), math.nan)
    return codes, scale.squeeze(-1).float()


class World:
    """Sequences over a paged cache, and the same values in 64 bits."""

    def __init__(self, dev, dtype, lens, new, kvh=2, hd=64, page=16, seed=0, slack=3):
        from ncmorph_b200.kv_cache import KVCache
        g = self.g = torch.Generator().manual_seed(seed)
        self.dev, self.dtype, self.lens, self.new, self.kvh, self.hd, self.page = dev, dtype, lens, new, kvh, hd, page
        need = [-(-n // page) for n in lens]
        pages = sum(need) + slack
        order = torch.randperm(pages, generator=g).to(torch.int32)
        table = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        self.table_cpu, self.table = table, table.to(dev)
        self.cache = KVCache.allocate(pages, page, kvh, hd, dtype, dev)
        for t in (self.cache.k, self.cache.v):  # what was never written must not matter
            t.view(torch.uint8).fill_(0xFF)
        for t in (self.cache.k_scale, self.cache.v_scale):
            if t is not None:
                t.fill_(math.nan)
        total = sum(lens)
        self.k, self.v = (torch.randn((total, kvh * hd), generator=g).to(torch.bfloat16) for _ in range(2))
        self.at = np.concatenate([[0], np.cumsum(lens)]).astype(int)
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.start = self.starts(new)
        self.T = sum(new)

    def starts(self, counts):
        return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=self.dev)

    def fill(self):
        """Everything is appended as one chunk."""
        from ncmorph_b200 import kv_cache
        kv_cache.append(self.cache, self.k.to(self.dev), self.v.to(self.dev), self.starts(self.lens), self.kv_lens, self.table)
        return self

    def held(self, x):
        """What the cache holds for rows x, in 64 bits [rows, kvh, hd]."""
        x = x.view(-1, self.kvh, self.hd)
        if self.dtype == torch.bfloat16:
            return x.double()
        codes, scale = quantise_ref(x, self.dtype)
        return codes * scale.double()[..., None]


LENS = [[1], [15], [16], [17], [5, 0, 33, 1], [200, 64, 3]]


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("kvh,hd,page", [(2, 64, 16), (1, 128, 8), (3, 64, 64), (5, 128, 32)])
def test_append_and_gather(cuda_dev, dtype, lens, kvh, hd, page):
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, dtype, lens, lens, kvh, hd, page, seed=sum(lens)).fill()
    k, v = kv_cache.gather(w.cache, w.start, w.table, rows=w.T)
    for got, x, pool, scales in ((k, w.k, w.cache.k, w.cache.k_scale), (v, w.v, w.cache.v, w.cache.v_scale)):
        if dtype == torch.bfloat16:
            assert torch.equal(got.cpu(), x)
            continue
        codes, scale = quantise_ref(x.view(-1, kvh, hd), dtype)
        # the pools hold exactly these codes and scales, and only the slots written changed
        written = torch.zeros(w.cache.num_pages, page, dtype=torch.bool)
        row = 0
        for b, n in enumerate(lens):
            for p in range(n):
                at = (w.table_cpu[b, p // page].item(), slice(None), p % page)
                written[at[0], at[2]] = True
                assert torch.equal(pool[at].cpu().double(), codes[row])
                assert torch.equal(scales[at].cpu(), scale[row])
                row += 1
        rest = ~written[:, None, :].expand(-1, kvh, -1)
        assert torch.all(pool.cpu().view(torch.uint8)[rest] == 0xFF) and torch.all(torch.isnan(scales.cpu()[rest]))
        assert torch.equal(got.cpu(), (codes.float() * scale[..., None]).to(torch.bfloat16).flatten(1))


@pytest.mark.parametrize("dtype", FORMATS[1:])
def test_append_of_hard_rows(cuda_dev, dtype):
    """Halfway values, the largest and smallest magnitudes, zeros, NaN and infinities."""
    from ncmorph_b200 import kv_cache
    big = torch.finfo(torch.bfloat16).max
    tiny = 2.0 ** -133
    rows = torch.zeros((12, 64))
    rows[1, :3] = torch.tensor([1.0, 0.5, -0.5])  # 63.5 of 127 steps
    rows[2] = torch.arange(64) * 2.0 - 63
    rows[2, 0] = 254.0  # odd multiples of half a step
    rows[3] = big
    rows[3, 5], rows[3, 6] = -big, big / 256
    rows[4, 3] = tiny
    rows[5, :2] = torch.tensor([1.0, math.nan])
    rows[6, :2] = torch.tensor([math.inf, 1.0])
    rows[7, :2] = torch.tensor([-math.inf, math.nan])
    rows[8] = torch.logspace(-30, 2, 64)
    rows[9] = -torch.logspace(-3, 38, 64)
    rows[10, 63] = -1e-20
    rows[11] = torch.linspace(-1, 1, 64)
    x = rows.to(torch.bfloat16)
    w = World(cuda_dev, dtype, [12], [12], 1, 64, 16)
    w.k, w.v = x, x.flip(0)
    w.fill()
    k, v = kv_cache.gather(w.cache, w.start, w.table, rows=12)
    for got, src in ((k, x), (v, x.flip(0))):
        codes, scale = quantise_ref(src.view(12, 1, 64), dtype)
        want = (codes.float() * scale[..., None]).to(torch.bfloat16).flatten(1)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert torch.equal(got.cpu()[ok], want[ok])


@pytest.mark.parametrize("dtype", FORMATS[1:])
def test_codes_of_every_ratio(cuda_dev, dtype):
    """Every pair of bf16 mantissas, near and far exponents: the codes and scales of exact arithmetic."""
    A = torch.arange(128, 256).float()
    rows = []
    for shift in (0, 1, 2, 5, 7, 9):
        other = torch.arange(128, 256).float() * 2.0 ** -shift
        for i in range(128):
            x = torch.minimum(other, A[i]).view(2, 64).clone()
            x[:, 63] = A[i]
            rows.append(x * torch.tensor([[1.0], [-1.0]]))
    x = torch.cat(rows)
    x = (x * 2.0 ** torch.randint(-60, 60, (x.shape[0], 1)).float()).to(torch.bfloat16)
    w = World(cuda_dev, dtype, [x.shape[0]], [x.shape[0]], 1, 64, 128)
    w.k = w.v = x
    w.fill()
    codes, scale = quantise_ref(x.view(-1, 1, 64), dtype)
    table = w.table_cpu[0, : -(-x.shape[0] // 128)].long()
    got = w.cache.k.cpu()[table].reshape(-1, 64)[: x.shape[0]].double()
    assert torch.equal(got, codes[:, 0])
    assert torch.equal(w.cache.k_scale.cpu()[table].reshape(-1)[: x.shape[0]], scale[:, 0])


def test_gather_ranges_and_qkv_columns(cuda_dev):
    """A window of each sequence, into the K and V columns of fused QKV rows;
    rows behind the last sequence stay as they were."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, torch.int8, [40, 7, 90], [40, 7, 90], 2, 64, 16).fill()
    begin, count = [30, 0, 11], [10, 7, 64]
    qkv = torch.full((sum(count) + 4, (8 + 4) * 64), 9.0, device=cuda_dev).to(torch.bfloat16)
    kv_cache.gather(w.cache, w.starts(count), w.table, begin=torch.tensor(begin, dtype=torch.int32, device=cuda_dev),
                    out_k=qkv[:, 512:640], out_v=qkv[:, 640:768])
    row = 0
    for b in range(3):
        at = w.at[b] + begin[b]
        for x, cols in ((w.k, slice(512, 640)), (w.v, slice(640, 768))):
            want = w.held(x[at:at + count[b]]).float().to(torch.bfloat16).flatten(1)
            assert torch.equal(qkv[row:row + count[b], cols].cpu(), want)
        row += count[b]
    assert torch.all(qkv[:, :512] == 9.0) and torch.all(qkv[row:] == 9.0)


def test_cache_bounds_are_reported(cuda_dev):
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, torch.int8, [20, 20], [20, 20], 1, 64, 16).fill()
    before = w.cache.k.clone()
    for change in ("page", "lens", "start"):
        table, lens, start = w.table.clone(), w.kv_lens.clone(), w.start.clone()
        if change == "page":
            table[0, 0], table[1, 0], table[1, 1] = w.cache.num_pages, -5, 2 ** 30
        elif change == "lens":
            lens[0], lens[1] = 19, 1000  # fewer keys than new tokens; more than the table holds
        else:
            start[1], start[2] = -3, 100
        junk = torch.randn((40, 64), device=cuda_dev).to(torch.bfloat16)
        kv_cache.append(w.cache, junk, junk, start, lens, table)
        expect_range_error(cuda_dev)
        if change != "page":
            assert torch.equal(w.cache.k, before)
        else:
            w.fill()
    out = torch.full((40, 64), 3.0, device=cuda_dev).to(torch.bfloat16)
    kv_cache.gather(w.cache, w.start, w.table, begin=torch.tensor([30, -1], dtype=torch.int32, device=cuda_dev), out_k=out, out_v=out.clone())
    expect_range_error(cuda_dev)
    assert torch.all(out == 3.0)


# --------------------------------------------------------------- tree attention

def tree_masks(new, g, words=None):
    """Random trees: bool [T, n] per sequence and their packed bits."""
    words = words or max(1, -(-max(new) // 32))
    sees, bits = [], torch.zeros((sum(new), words), dtype=torch.int64)
    row = 0
    for n in new:
        m = torch.zeros((n, n), dtype=torch.bool)
        for i in range(n):
            if i:
                m[i] = m[int(torch.randint(0, i, (1,), generator=g))]
            m[i, i] = True
            for j in range(n):
                if m[i, j]:
                    bits[row + i, j // 32] |= 1 << (j % 32)
        row += n
        sees.append(m)
    return sees, torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)


def attend_ref(w, q, heads, sees, scale):
    """out, lse and their tolerances, in 64 bits, from what the cache holds."""
    outs, lses, tol_o, tol_l = [], [], [], []
    g, row = heads // w.kvh, 0
    K, V = w.held(w.k), w.held(w.v)
    for b, n in enumerate(w.new):
        if n == 0:
            continue
        L = w.lens[b]
        k, v = K[w.at[b]:w.at[b] + L], V[w.at[b]:w.at[b] + L]
        x = q[row:row + n].double().view(n, w.kvh, g, w.hd)
        seen = torch.ones((n, L), dtype=torch.bool)
        seen[:, L - n:] = torch.ones((n, n)).tril().bool() if sees is None else sees[b]
        k0 = torch.where(torch.isfinite(k), k, 0.0)
        t = torch.einsum("nhgd,lhd->nhgl", x, k) * scale
        t = torch.where(seen[:, None, None], t, -math.inf)
        size = (torch.einsum("nhgd,lhd->nhgl", x.abs(), k0.abs()) * abs(scale)).masked_fill(~seen[:, None, None], 0.0)
        top = t.amax(-1, keepdim=True).clamp(min=-1e300)
        p = torch.exp(t - top)
        total = p.sum(-1, keepdim=True)
        pn = torch.where(total > 0, p / torch.where(total > 0, total, 1.0), 0.0)
        vm = torch.where(torch.isfinite(v), v, 0.0)
        o = torch.einsum("nhgl,lhd->nhgd", pn, vm)
        odd = ~torch.isfinite(v)
        if odd.any():  # a visible value that is not finite takes its formula
            for i in range(n):
                for h in range(w.kvh):
                    cols = seen[i]
                    o[i, h] = (pn[i, h][:, cols][:, :, None] * v[cols, h][None]).sum(1)
        spread = torch.einsum("nhgl,lhd->nhgd", pn, vm.abs())
        # scores: a sum of head_dim products in f32, the scale's and the key scale's products; exp2
        # to 2^-22; the running sums and their merges, an f32 rounding a term
        ds = (w.hd + 6) * F32 * size.amax(-1, keepdim=True) + (L + 64) * F32 + 2 ** -21
        outs.append(o.reshape(n, -1))
        tol_o.append(((2 * ds + BF) * spread + BF * o.abs() + 1e-37).reshape(n, -1))
        lses.append((top + torch.log(total)).reshape(n, -1))
        tol_l.append((2 * ds + 4 * F32 * (top.abs().clamp(max=1e30) + 8)).reshape(n, -1))
        row += n
    return tuple(torch.cat(z) for z in (outs, lses, tol_o, tol_l))


def check_attention(out, lse, ref):
    o, l, to, tl = ref
    out, lse = out.cpu().double(), lse.cpu().double()
    assert torch.equal(torch.isnan(out), torch.isnan(o))
    fine = torch.isfinite(o)
    assert torch.equal(out[~fine & ~torch.isnan(o)], o[~fine & ~torch.isnan(o)])
    bad = (out - o).abs()[fine] > to[fine]
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} out of bounds, worst {((out - o).abs()[fine] / to[fine]).max():.3g}"
    empty = torch.isinf(l)
    assert torch.equal(torch.isinf(lse), empty) and torch.all(lse[empty] < 0)
    ok = torch.isfinite(l)
    assert torch.all((lse - l).abs()[ok] <= tl[ok])


SHAPES = [  # heads, kv_heads, head_dim, page: groups of 1, 3, 4, 5, 8
    (2, 2, 64, 16), (6, 2, 64, 8), (8, 2, 128, 16), (5, 1, 64, 64), (8, 1, 128, 32), (32, 8, 64, 32)]


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("lens", [[1], [2, 31, 32, 33], [127, 128, 129, 513], [700, 5, 2051]])
def test_single_tokens(cuda_dev, dtype, shape, lens):
    from ncmorph_b200 import kv_cache
    heads, kvh, hd, page = shape
    w = World(cuda_dev, dtype, lens, [1] * len(lens), kvh, hd, page, seed=len(lens)).fill()
    q = torch.randn((w.T, heads * hd), generator=w.g).to(torch.bfloat16)
    out, lse = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=1, return_lse=True)
    check_attention(out, lse, attend_ref(w, q, heads, None, hd ** -0.5))


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("lens,new", [([5], [5]), ([3, 40, 300, 64], [3, 1, 17, 0]), ([600, 70, 1111], [33, 64, 40]),
                                      ([1500, 90], [70, 90])])
@pytest.mark.parametrize("tree", [False, True])
def test_drafted_tokens(cuda_dev, dtype, shape, lens, new, tree):
    from ncmorph_b200 import kv_cache
    heads, kvh, hd, page = shape
    w = World(cuda_dev, dtype, lens, new, kvh, hd, page, seed=sum(lens)).fill()
    q = torch.randn((w.T, heads * hd), generator=w.g).to(torch.bfloat16)
    sees, bits = tree_masks(new, w.g)
    out, lse = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=max(new),
                                       tree_mask=bits.to(cuda_dev) if tree else None, scale=0.2, return_lse=True)
    check_attention(out, lse, attend_ref(w, q, heads, sees if tree else None, 0.2))


def test_chain_equals_its_tree_mask(cuda_dev):
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, torch.bfloat16, [900, 77], [45, 77], 2, 64, 16).fill()
    q = torch.randn((w.T, 8 * 64), generator=w.g).to(torch.bfloat16).to(cuda_dev)
    n = torch.cat([torch.arange(c) for c in w.new])
    bits = torch.stack([((1 << (n + 1 - 32 * i).clamp(0, 32)) - 1) for i in range(3)], 1)
    bits = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32).to(cuda_dev)
    a, la = kv_cache.tree_attention(q, w.cache, w.start, w.kv_lens, w.table, max_nodes=80, return_lse=True)
    b, lb = kv_cache.tree_attention(q, w.cache, w.start, w.kv_lens, w.table, max_nodes=80, tree_mask=bits, return_lse=True)
    assert torch.equal(a, b) and torch.equal(la, lb)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("rows", ["few", "many"])
def test_hidden_and_empty(cuda_dev, dtype, rows):
    """Rows whose mask leaves nothing, and keys and values that are not finite in
    hidden places (and in seen ones, where they show)."""
    from ncmorph_b200 import kv_cache
    n = 4 if rows == "few" else 40
    w = World(cuda_dev, dtype, [n, 100 + n], [n, n], 2, 64, 16)
    sees, bits = tree_masks([n, n], w.g)
    for s, r0 in ((sees[0], 0), (sees[1], n)):
        s[:, n - 2] = False  # nobody sees this node, but itself does not either
        s[n - 1, :] = False
        s[n - 1, n - 2] = r0 > 0  # in the second sequence one row sees it
    bits = torch.zeros_like(bits, dtype=torch.int64)
    for r0, s in ((0, sees[0]), (n, sees[1])):
        for i in range(n):
            for j in range(n):
                if s[i, j]:
                    bits[r0 + i, j // 32] |= 1 << (j % 32)
    bits = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)
    for at in (n - 2, 100 + 2 * n - 2):  # the hidden node's rows
        w.k[at] = math.nan
        w.v[at, ::3], w.v[at, 1::3] = math.nan, math.inf
    w.fill()
    q = torch.randn((2 * n, 8 * 64), generator=w.g).to(torch.bfloat16)
    out, lse = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=n,
                                       tree_mask=bits.to(cuda_dev), return_lse=True)
    ref = attend_ref(w, q, 8, sees, 0.125)
    shown = torch.zeros(2 * n, dtype=torch.bool)
    shown[2 * n - 1] = True  # sees a NaN key
    hidden = ~shown
    check_attention(out[hidden.to(cuda_dev)], lse[hidden.to(cuda_dev)], tuple(z[hidden] for z in ref))
    assert torch.all(torch.isnan(out[2 * n - 1].cpu()))
    assert torch.all(out[n - 1] == 0) and torch.all(lse[n - 1] == -math.inf)


@pytest.mark.parametrize("n,L,hd", [(6, 70, 64), (70, 150, 64), (140, 500, 64), (90, 800, 128)])
def test_seen_infinite_values(cuda_dev, n, L, hd):
    """A finite key whose value row holds an infinity reaches the rows that see it, and no others."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, torch.bfloat16, [L], [n], 1, hd, 16)
    c = L - n
    w.v[c + 2, 5], w.v[c + 3, 9], w.v[30, 40], w.v[c - 1, 50] = math.inf, -math.inf, math.inf, -math.inf
    w.fill()
    q = torch.randn((n, hd), generator=w.g).to(torch.bfloat16)
    out, lse = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=n, return_lse=True)
    out = out.cpu()
    want = torch.zeros((n, hd), dtype=torch.bool)
    want[2:, 5] = want[3:, 9] = want[:, 40] = want[:, 50] = True
    assert torch.equal(torch.isinf(out), want) and not torch.isnan(out).any()
    w.v[~torch.isfinite(w.v)] = 0.0
    o, l, to, tl = attend_ref(w, q, 1, None, hd ** -0.5)
    assert torch.all(((out.double() - o).abs() <= to) | want) and torch.all((lse.cpu().double() - l).abs() <= tl)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("new,hd", [((2, 1), 128), ((30, 1), 128), ((30, 17), 64), ((64, 40), 64)])
def test_sharp_and_wide_scores(cuda_dev, dtype, new, hd):
    """Scores far apart: the maximum moves often, and late."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, dtype, [1300, 400], list(new), 1, hd, 32, seed=5)
    ramp = torch.cat([torch.linspace(0.1, 4, n) for n in (1300, 400)])[:, None]
    w.k = (w.k.float() * ramp).to(torch.bfloat16)
    w.v = (w.v.float() * torch.exp(4 * torch.randn((1700, 1), generator=w.g))).to(torch.bfloat16)
    w.fill()
    for scale in (hd ** -0.5, -0.07, 0.0):
        q = (3 * torch.randn((w.T, 4 * hd), generator=w.g)).to(torch.bfloat16)
        out, lse = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=max(new), scale=scale,
                                           return_lse=True)
        check_attention(out, lse, attend_ref(w, q, 4, None, scale))


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("n,heads", [(1, 1), (4, 8), (20, 4)])
def test_many_small_terms_beside_a_large_one(cuda_dev, dtype, n, heads):
    """One key takes nearly all of the weight, with zeros in half of its value's columns;
    there 4000 keys of weight 2^-26 each are all there is, and not lost."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, dtype, [4000 + n], [n], 1, 64, 16)
    w.k.zero_()
    w.v.fill_(1.0)
    w.k[7, 0] = 1.0
    w.v[7, 32:] = 0.0
    w.fill()
    q = torch.zeros((n, heads * 64), dtype=torch.bfloat16)
    q[:, ::64] = 18.0  # 18 log2(e) = 25.97
    out = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=n, scale=1.0)
    o, _, to, _ = attend_ref(w, q, heads, None, 1.0)
    # f32 scores of 18 (2^-19), two roundings to 16 bits, and f16 half steps of 2^-32 of the largest term
    tol = 2.0 ** -18 * o.abs() + 2 * BF * o.abs() + (4000 * 2.0 ** -32 if dtype != torch.bfloat16 else 0)
    assert torch.all((out.cpu().double() - o).abs() <= tol)


def test_many_sequences_and_strided_rows(cuda_dev):
    """More sequences than a warp scans at once, empty ones among them, q and out
    as column slices of wider rows; rows behind the last sequence stay."""
    from ncmorph_b200 import kv_cache
    lens = [(17 * b) % 190 + 3 for b in range(75)]
    new = [b % 4 for b in range(75)]
    w = World(cuda_dev, torch.bfloat16, lens, new, 2, 64, 16).fill()
    wide = torch.randn((w.T + 5, 12 * 64), generator=w.g).to(torch.bfloat16).to(cuda_dev)
    out = torch.full((w.T + 5, 8 * 64 + 64), 5.0, device=cuda_dev).to(torch.bfloat16)
    table = torch.cat([w.table, w.table], 1)[:, :w.table.shape[1]]  # (strided rows)
    table = torch.empty((75, 90), dtype=torch.int32, device=cuda_dev).fill_(-7)[:, :40]
    table[:, :w.table.shape[1]] = w.table
    got = kv_cache.tree_attention(wide[:, 64:64 + 512], w.cache, w.start, w.kv_lens, table, max_nodes=3, heads=8, out=out[:, 64:])
    assert got.shape == (w.T + 5, 512)
    q = wide[:w.T, 64:576].cpu()
    o, l, to, tl = attend_ref(w, q, 8, None, 0.125)
    assert torch.all((out[:w.T, 64:].cpu().double() - o).abs() <= to)
    assert torch.all(out[w.T:] == 5.0) and torch.all(out[:, :64] == 5.0)


def test_attention_is_the_same_on_every_run_and_stream(cuda_dev):
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, torch.int8, [5000, 1200, 7], [9, 3, 1], 4, 64, 32).fill()
    q = torch.randn((13, 16 * 64), generator=w.g).to(torch.bfloat16).to(cuda_dev)
    call = lambda: kv_cache.tree_attention(q, w.cache, w.start, w.kv_lens, w.table, max_nodes=9, return_lse=True)  # noqa: E731
    first = call()
    for _ in range(5):
        again = call()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
        side.synchronize()
    assert torch.equal(first[0], other[0])


def test_attention_bounds_are_reported(cuda_dev):
    """A sequence whose numbers do not fit is skipped; the others are answered."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, torch.bfloat16, [50, 60, 70], [2, 2, 2], 1, 64, 16).fill()
    q = torch.randn((6, 64), generator=w.g).to(torch.bfloat16)
    good = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=2)
    for lens in ([50, 1, 70], [50, 10 ** 6, 70], [50, -4, 70]):
        out = torch.full((6, 64), 2.0, device=cuda_dev).to(torch.bfloat16)
        kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, torch.tensor(lens, dtype=torch.int32, device=cuda_dev), w.table,
                                max_nodes=2, out=out)
        expect_range_error(cuda_dev)
        assert torch.equal(out[[0, 1, 4, 5]], good[[0, 1, 4, 5]]) and torch.all(out[2:4] == 2.0)
    out = torch.full((6, 64), 2.0, device=cuda_dev).to(torch.bfloat16)
    kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=1, out=out)  # more nodes than said
    expect_range_error(cuda_dev)
    assert torch.all(out == 2.0)
    table = w.table.clone()
    table[1, 1] = w.cache.num_pages + 9
    out = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, table, max_nodes=2)
    expect_range_error(cuda_dev)
    assert torch.equal(out[[0, 1, 4, 5]], good[[0, 1, 4, 5]])


# ----------------------------------------------------------------------- logits

def logits_ref(x, hist, prompts, rep, freq, pres, biases, allowed):
    y, size = x.double().clone(), x.double().abs()
    size = torch.where(torch.isfinite(size), size, 0.0)
    for r in range(x.shape[0]):
        ids = hist[r]
        if len(ids):
            used = torch.unique(torch.tensor(ids))
            f = rep[r].double()
            y[r, used] = torch.where(y[r, used] > 0, y[r, used] / f, y[r, used] * f)
            size[r, used] *= max(float(f), 1 / float(f))
            for t in ids[max(0, prompts[r]):]:
                y[r, t] -= freq[r].double()
                size[r, t] += freq[r].abs().double()
            for t in set(ids[max(0, prompts[r]):]):
                y[r, t] -= pres[r].double()
                size[r, t] += pres[r].abs().double()
        for t, v in biases[r]:
            y[r, t] += v
            size[r, t] += abs(v)
        if allowed is not None and allowed[r] is not None:
            y[r, ~allowed[r]] = -math.inf
    return y, size


def pack_bits(allowed):
    M, V = allowed.shape
    bits = torch.zeros((M, -(-V // 32)), dtype=torch.int64)
    for v in range(V):
        bits[:, v // 32] |= allowed[:, v].long() << (v % 32)
    return torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)


@pytest.mark.parametrize("R,V", [(1, 1), (3, 31), (2, 33), (4, 8192), (2, 8193), (5, 1000), (3, 20001)])
@pytest.mark.parametrize("dtype,out_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                             (torch.bfloat16, torch.bfloat16)])
def test_logit_rules(cuda_dev, R, V, dtype, out_dtype):
    from ncmorph_b200 import ncm_model
    g = torch.Generator().manual_seed(V + R)
    rnd = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    x = (3 * torch.randn((R, V + 8), generator=g)).to(dtype)
    x[0, 0] = math.nan
    x[R - 1, V - 1] = -math.inf
    hist = [[rnd(min(V, 40)) for _ in range((0, 1, 50, 600)[r % 4])] for r in range(R)]
    hist[0] += [V - 1, V - 1]
    prompts = [rnd(len(h) + 1) for h in hist]
    rep, freq, pres = 1 + torch.rand(R, generator=g), torch.rand(R, generator=g) - 0.3, torch.rand(R, generator=g)
    biases = [[(rnd(min(V, 25)), float(torch.randn(1, generator=g))) for _ in range((30, 0, 1, 200)[r % 4])] for r in range(R)]
    allowed = torch.rand((R + 1, V), generator=g) < 0.4
    allowed[0] = False  # a state that allows nothing
    which = [r - 1 if r else R - 1 for r in range(R)]  # row 0: free (-1) when R == 1 ... else mask R - 1
    which[-1] = -1
    starts = lambda lists: torch.tensor(np.concatenate([[0], np.cumsum([len(z) for z in lists])]), dtype=torch.int32, device=cuda_dev)  # noqa: E731
    i32 = lambda z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    args = dict(tokens=i32([t for h in hist for t in h]), token_start=starts(hist), prompt_lens=i32(prompts),
                repetition=rep.to(cuda_dev), frequency=freq.to(cuda_dev), presence=pres.to(cuda_dev),
                bias_ids=i32([t for z in biases for t, _ in z]),
                bias=torch.tensor([v for z in biases for _, v in z], dtype=torch.float32, device=cuda_dev), bias_start=starts(biases),
                allowed=pack_bits(allowed).to(cuda_dev), allowed_rows=i32(which))
    xd = x.to(cuda_dev)
    out = torch.empty((R, V), dtype=out_dtype, device=cuda_dev)
    ncm_model.process_logits(xd[:, :V], out=out, **args)
    y, size = logits_ref(x[:, :V], hist, prompts, rep, freq, pres, biases, [allowed[m] if m >= 0 else None for m in which])
    got = out.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(y)) and torch.equal(torch.isinf(got), torch.isinf(y))
    fine = torch.isfinite(y)
    n = max([len(z) for z in biases] + [len(h) for h in hist]) + 4
    tol = n * F32 * size + (BF * y.abs() if out_dtype == torch.bfloat16 else 0)
    assert torch.all((got - y).abs()[fine] <= tol[fine])
    if dtype == out_dtype:  # in place, strided rows: the same bits, and nothing behind them
        ncm_model.process_logits(xd[:, :V], out=xd[:, :V], **args)
        assert torch.equal(xd[:, :V].nan_to_num(7.0), out.nan_to_num(7.0)) and torch.equal(xd[:, V:].cpu(), x[:, V:])


def test_logit_rules_alone(cuda_dev):
    """Each rule without the others; no rule at all is a copy."""
    from ncmorph_b200 import ncm_model
    x = torch.tensor([[1.0, -2.0, 3.0, 0.0, 5.0]], device=cuda_dev)
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    f32 = lambda *z: torch.tensor(z, dtype=torch.float32, device=cuda_dev)  # noqa: E731
    inf = math.inf
    hist = dict(tokens=i32(1, 2, 2), token_start=i32(0, 3))
    for args, want in (({}, [1, -2, 3, 0, 5]), (dict(hist, repetition=f32(2.0)), [1, -4, 1.5, 0, 5]),
                       (dict(hist, frequency=f32(0.5)), [1, -2.5, 2, 0, 5]), (dict(hist, presence=f32(0.25)), [1, -2.25, 2.75, 0, 5]),
                       (dict(hist, presence=f32(0.25), prompt_lens=i32(1)), [1, -2, 2.75, 0, 5]),
                       (dict(hist, frequency=f32(1.0), prompt_lens=i32(9)), [1, -2, 3, 0, 5]),
                       (dict(bias=f32(1.0, 2.0, 4.0), bias_ids=i32(4, 0, 4), bias_start=i32(0, 3)), [3, -2, 3, 0, 10]),
                       (dict(allowed=i32(0b01101).view(1, 1)), [1, -inf, 3, 0, -inf]),
                       (dict(allowed=i32(0).view(1, 1)), [-inf] * 5)):
        assert ncm_model.process_logits(x, **args).tolist() == [want]


def test_logit_bounds_are_reported(cuda_dev):
    from ncmorph_b200 import ncm_model
    x = torch.randn((2, 100), device=cuda_dev)
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    f32 = lambda *z: torch.tensor(z, dtype=torch.float32, device=cuda_dev)  # noqa: E731
    for args in (dict(tokens=i32(-1, 100, 2 ** 30), token_start=i32(0, 2, 3), frequency=f32(1, 1)),
                 dict(tokens=i32(5, 5), token_start=i32(0, -1, 9), frequency=f32(1, 1)),
                 dict(bias=f32(1, 1), bias_ids=i32(-7, 100), bias_start=i32(0, 1, 2)),
                 dict(bias=f32(1, 1), bias_ids=i32(3, 3), bias_start=i32(2, 1, 3)),
                 dict(allowed=i32(*[-1] * 8).view(2, 4), allowed_rows=i32(2, -2))):
        y = ncm_model.process_logits(x, **args)
        expect_range_error(cuda_dev)
        assert torch.equal(y, x)


# -------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", FORMATS)
def test_decode_steps_together(cuda_dev, dtype):
    """A prompt and two decode steps of one layer on fused QKV rows, then the head's
    rules: the last step captured into a graph and replayed on new inputs."""
    from ncmorph_b200 import kv_cache, ncm_model
    H, Hkv, hd, V = 8, 2, 64, 500
    g = torch.Generator().manual_seed(11)
    width = (H + 2 * Hkv) * hd
    cos, sin = tables(256, hd, cuda_dev)
    cache = kv_cache.KVCache.allocate(20, 16, Hkv, hd, dtype, cuda_dev)
    table = torch.randperm(20, generator=g)[:16].to(torch.int32).view(2, 8).to(cuda_dev)
    head = (torch.randn((V, H * hd), generator=g) * 0.05).to(torch.bfloat16).to(cuda_dev)
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    rules = dict(tokens=i32(1, 2, 3), token_start=i32(0, 1, 3), repetition=torch.full((2,), 1.3, device=cuda_dev))
    allowed = torch.ones((2, -(-V // 32)), dtype=torch.int32, device=cuda_dev) * -1

    def step(qkv, start, lens, pos, n, rows=None):
        ncm_model.rope_bf16(qkv, pos, cos, sin, H + Hkv, hd, out=qkv)
        kv_cache.append(cache, qkv[:, H * hd:(H + Hkv) * hd], qkv[:, (H + Hkv) * hd:], start, lens, table)
        return kv_cache.tree_attention(qkv, cache, start, lens, table, max_nodes=n, heads=H)

    def logits_of(ctx):
        from ncmorph_b200 import kernels
        return ncm_model.process_logits(kernels.linear_bf16(ctx, head), allowed=allowed, **rules)

    lens = [37, 64]
    chunks = [torch.randn((sum(lens), width), generator=g).to(torch.bfloat16)]
    chunks += [torch.randn((2, width), generator=g).to(torch.bfloat16) for _ in range(3)]
    prompt = chunks[0].to(cuda_dev)
    step(prompt, i32(0, 37, 101), i32(*lens), torch.cat([torch.arange(n) for n in lens]).to(torch.int32).to(cuda_dev), 64)
    qkv, start = chunks[1].to(cuda_dev), i32(0, 1, 2)
    kv_lens, pos = i32(38, 65), i32(37, 64)
    step(qkv, start, kv_lens, pos, 1)
    # the same call captured: lengths, positions and rows are read at replay
    static = chunks[2].to(cuda_dev)
    kv_lens.add_(1)
    pos.add_(1)
    warm = static.clone()
    logits_of(step(warm, start, kv_lens, pos, 1))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx = step(static, start, kv_lens, pos, 1)
        out = logits_of(ctx)
    static.copy_(chunks[2].to(cuda_dev))
    graph.replay()
    static.copy_(chunks[3].to(cuda_dev))
    kv_lens.add_(1)
    pos.add_(1)
    graph.replay()
    torch.cuda.synchronize()
    # in 64 bits, from the rows as they were rotated and held
    rot = lambda x, p: rope_ref(x, p, cos.cpu(), sin.cpu(), H + Hkv, hd, False, False)[0]  # noqa: E731
    for b in range(2):
        rows = [chunks[0][sum(lens[:b]):sum(lens[:b + 1])]] + [c[b:b + 1] for c in chunks[1:]]
        x = torch.cat(rows)
        n = x.shape[0]
        r = rot(x, torch.arange(n, dtype=torch.int32)).float().to(torch.bfloat16)
        k, v = r[:, H * hd:].view(n, Hkv, hd), x[:, (H + Hkv) * hd:].view(n, Hkv, hd)
        hold = (lambda z: z.double()) if dtype == torch.bfloat16 else (lambda z: quantise_ref(z, dtype)[0] * quantise_ref(z, dtype)[1].double()[..., None])
        q = r[-1, :H * hd].double().view(Hkv, H // Hkv, hd)
        p = torch.softmax(torch.einsum("hgd,lhd->hgl", q, hold(k)) * hd ** -0.5, -1)
        want = torch.einsum("hgl,lhd->hgd", p, hold(v)).reshape(-1)
        # a rotated bf16 value may round the other way here, and then move a code by one step
        step_k = {torch.bfloat16: BF, torch.int8: 1 / 127, torch.float8_e4m3fn: 2.0 ** -4}[dtype]
        slack = 4 * (BF + 0.02 * step_k * math.sqrt(n))
        got = ctx[b].cpu().double()
        assert torch.all((got - want).abs() <= slack * (want.abs() + 1)), (got - want).abs().max()
    y = (ctx.float() @ head.float().t()).cpu()
    for b, ids in ((0, [1]), (1, [2, 3])):
        y[b, ids] = torch.where(y[b, ids] > 0, y[b, ids] / 1.3, y[b, ids] * 1.3)
    assert torch.all((out.cpu() - y).abs() <= 2 * BF * y.abs() + 1e-4)


def test_prefill_over_gathered_rows(cuda_dev):
    """A cached context read back beside a chunk's rows feeds the prefill
    attention, which then agrees with attention over the cache."""
    from ncmorph_b200 import kv_cache, ncm_model
    H, Hkv, hd, n, L = 8, 2, 64, 24, 96
    w = World(cuda_dev, torch.bfloat16, [L], [n], Hkv, hd, 16).fill()
    q = torch.randn((n, H * hd), generator=w.g).to(torch.bfloat16).to(cuda_dev)
    out = kv_cache.tree_attention(q, w.cache, w.start, w.kv_lens, w.table, max_nodes=n)
    qkv = torch.zeros((L, (H + 2 * Hkv) * hd), dtype=torch.bfloat16, device=cuda_dev)
    qkv[L - n:, :H * hd] = q
    kv_cache.gather(w.cache, w.starts([L]), w.table, out_k=qkv[:, H * hd:(H + Hkv) * hd], out_v=qkv[:, (H + Hkv) * hd:])
    whole = ncm_model.attention_bf16(qkv, H, Hkv, ncm_model.make_mask("causal"))
    # both round their output and their probabilities to bf16 once, and |v| stays below 5
    assert torch.all((whole[L - n:].float() - out.float()).abs() <= 2 * BF * 5 + 2 * BF * out.float().abs())


def test_pools_beyond_32_bit_offsets(cuda_dev):
    """A pool of more than 2^32 bytes: slots behind the boundary are written and read."""
    from ncmorph_b200 import kv_cache
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    pages = (5 << 30) // (8 * 64 * 64 * 2)
    cache = kv_cache.KVCache.allocate(pages, 64, 8, 64, torch.bfloat16, cuda_dev)
    assert cache.k.numel() * 2 > 1 << 32
    table = torch.tensor([[pages - 1, 0, pages - 2, pages // 2]], dtype=torch.int32, device=cuda_dev)
    rows = torch.randn((250, 512), device=cuda_dev).to(torch.bfloat16)
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    kv_cache.append(cache, rows, rows.flip(0), i32(0, 250), i32(250), table)
    k, v = kv_cache.gather(cache, i32(0, 250), table, rows=250)
    assert torch.equal(k, rows) and torch.equal(v, rows.flip(0))
    assert torch.equal(cache.k[pages - 1].transpose(0, 1).reshape(64, 512), rows[:64])
    q = torch.randn((1, 8 * 64), device=cuda_dev).to(torch.bfloat16)
    out = kv_cache.tree_attention(q, cache, i32(0, 1), i32(250), table, max_nodes=1)
    p = torch.softmax(torch.einsum("hd,lhd->hl", q.view(8, 64).double(), rows.view(250, 8, 64).double()) / 8, -1)
    want = torch.einsum("hl,lhd->hd", p, rows.flip(0).view(250, 8, 64).double()).reshape(-1)
    assert torch.all((out[0].double() - want).abs() <= 2 * BF * 5)


def test_refusals(cuda_dev):
    """What the device forms refuse before any launch."""
    from ncmorph_b200 import _lib, kv_cache, ncm_model
    bf = lambda *s: torch.zeros(s, device=cuda_dev, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    cos, sin = tables(4, 64, cuda_dev)
    cache = kv_cache.KVCache.allocate(4, 16, 2, 64, torch.int8, cuda_dev)
    table, start, lens = i32(0, 1).view(1, 2), i32(0, 1), i32(1)
    x = bf(3, 256)
    with pytest.raises(_lib.NcmError):  # overlapping rows that are not the same
        ncm_model.rope_bf16(x[:2], i32(0, 1), cos, sin, 1, 64, out=x[1:])
    with pytest.raises(ValueError):
        ncm_model.rope_bf16(x, i32(0, 1), cos, sin, 1, 64)
    with pytest.raises(TypeError):
        ncm_model.rope_bf16(x.float(), i32(0, 1, 2), cos, sin, 1, 64)
    with pytest.raises(_lib.NcmError):  # wider than the head
        ncm_model.rope_bf16(x, i32(0, 1, 2), cos, sin, 1, 32)
    with pytest.raises(ValueError):
        kv_cache.append(cache, bf(1, 64), bf(1, 128), start, lens, table)
    with pytest.raises(ValueError):
        kv_cache.append(cache, bf(1, 128), bf(2, 128), start, lens, table)
    with pytest.raises(_lib.NcmError):  # rows that are not 16-byte aligned
        kv_cache.append(cache, bf(2, 130)[:, 1:129], bf(2, 128), start, lens, table)
    with pytest.raises(TypeError):
        kv_cache.append(cache, bf(1, 128), bf(1, 128), start.long(), lens, table)
    with pytest.raises(ValueError):
        kv_cache.append(cache, bf(1, 128), bf(1, 128), i32(0, 1, 1), lens, table)
    with pytest.raises(ValueError):
        kv_cache.KVCache(cache.k, cache.v)
    with pytest.raises(ValueError):
        kv_cache.gather(cache, start, table)
    for wrong in (dict(out_k=bf(1, 128), out_v=bf(2, 128)), dict(rows=2, out_k=bf(1, 128)), dict(rows=2, out_v=bf(1, 128)),
                  dict(out_k=bf(1, 128)), dict(out_k=bf(1, 64), out_v=bf(1, 128)), dict(rows=-1)):
        with pytest.raises((ValueError, RuntimeError)):
            kv_cache.gather(cache, start, table, **wrong)
    with pytest.raises(TypeError):
        kv_cache.gather(cache, start, table, out_k=[1], out_v=bf(1, 128))
    with pytest.raises(_lib.NcmError):  # three heads over two kv heads
        kv_cache.tree_attention(bf(1, 192), cache, start, lens, table, max_nodes=1)
    with pytest.raises(_lib.NcmError):
        kv_cache.tree_attention(bf(1, 256), cache, start, lens, table, max_nodes=0)
    with pytest.raises(ValueError):
        kv_cache.tree_attention(bf(1, 256), cache, start, lens, table, max_nodes=1, tree_mask=i32(1, 1).view(2, 1))
    q = bf(1, 256)
    with pytest.raises(_lib.NcmError):
        kv_cache.tree_attention(q, cache, start, lens, table, max_nodes=1, out=q)
    y = torch.zeros((2, 40), device=cuda_dev)
    with pytest.raises(_lib.NcmError):
        ncm_model.process_logits(y, repetition=torch.ones(2, device=cuda_dev))
    with pytest.raises(ValueError):
        ncm_model.process_logits(y, allowed=i32(1, 1).view(2, 1))
    with pytest.raises(TypeError):
        ncm_model.process_logits(y, out=bf(2, 40))
    with pytest.raises(TypeError):
        ncm_model.process_logits(y.double())


def test_empty_calls(cuda_dev):
    from ncmorph_b200 import kv_cache, ncm_model
    bf = lambda *s: torch.zeros(s, device=cuda_dev, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    cos, sin = tables(4, 64, cuda_dev)
    cache = kv_cache.KVCache.allocate(4, 16, 2, 64, torch.bfloat16, cuda_dev)
    assert ncm_model.rope_bf16(bf(0, 64), i32(), cos, sin, 1, 64).shape == (0, 64)
    table = i32(0, 1, 2, 3).view(2, 2)
    kv_cache.append(cache, bf(0, 128), bf(0, 128), i32(0, 0, 0), i32(0, 5), table)
    assert kv_cache.tree_attention(bf(0, 256), cache, i32(0, 0, 0), i32(0, 5), table, max_nodes=4).shape == (0, 256)
    out = kv_cache.tree_attention(bf(3, 256), cache, i32(0, 0, 0), i32(0, 5), table, max_nodes=4, out=torch.ones_like(bf(3, 256)))
    assert torch.all(out == 1)
    none = torch.zeros((0, 4), dtype=torch.int32, device=cuda_dev)
    kv_cache.append(cache, bf(2, 128), bf(2, 128), i32(0), i32(), none)
    assert ncm_model.process_logits(torch.zeros((0, 9), device=cuda_dev)).shape == (0, 9)


# ------------------------------------------------- limits, and calls at the same time

def test_positions_past_the_limit_are_reported(cuda_dev):
    """Positions that pass 2^30 or 32 bits although the page table would cover them."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, torch.bfloat16, [40], [2], 1, 64, 1024, slack=1).fill()
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    wide = torch.zeros((1, (1 << 21) + 8), dtype=torch.int32, device=cuda_dev)  # 2^31 + 8192 positions
    before = w.cache.k.clone()  # (holds NaN where nothing was written: compared as bits)
    rows = torch.ones((8, 64), device=cuda_dev).to(torch.bfloat16)
    for begin in (2 ** 31 - 4, 2 ** 30 - 4):
        out = torch.full((8, 64), 3.0, device=cuda_dev).to(torch.bfloat16)
        kv_cache.gather(w.cache, i32(0, 8), wide, begin=i32(begin), out_k=out, out_v=out.clone())
        expect_range_error(cuda_dev)
        assert torch.all(out == 3.0)
    for length in (2 ** 31 - 1, 2 ** 30 + 1):
        kv_cache.append(w.cache, rows, rows, i32(0, 8), i32(length), wide)
        expect_range_error(cuda_dev)
        assert torch.equal(w.cache.k.view(torch.int16), before.view(torch.int16))
        for n in (8, 512):  # (both attention kernels)
            out = torch.full((8, 64), 3.0, device=cuda_dev).to(torch.bfloat16)
            kv_cache.tree_attention(rows, w.cache, i32(0, 8), i32(length), wide, max_nodes=n, out=out)
            expect_range_error(cuda_dev)
            assert torch.all(out == 3.0)
    # the last position that the limit allows
    k, _ = kv_cache.gather(w.cache, i32(0, 8), wide, rows=8, begin=i32(2 ** 30 - 8))
    assert torch.equal(k.view(torch.int16), before[0, 0, 1016:].view(torch.int16))


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("page", [8, 1024])
@pytest.mark.parametrize("n,heads,hd", [(1, 64, 64), (1, 64, 128), (2, 4, 64), (100, 2, 128), (200, 2, 64)])
def test_smallest_and_largest_pages_and_groups(cuda_dev, dtype, page, n, heads, hd):
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, dtype, [1500, 200 + n], [n, n], 1, hd, page).fill()
    q = torch.randn((2 * n, heads * hd), generator=w.g).to(torch.bfloat16)
    out, lse = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=n, return_lse=True)
    check_attention(out, lse, attend_ref(w, q, heads, None, hd ** -0.5))


def test_most_nodes(cuda_dev):
    """1024 drafted tokens in one sequence beside one in another, with masks of 32 words."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, torch.bfloat16, [1300, 40], [1024, 1], 1, 64, 16).fill()
    sees, bits = tree_masks(w.new, w.g)
    assert bits.shape[1] == 32
    q = torch.randn((1025, 2 * 64), generator=w.g).to(torch.bfloat16)
    out, lse = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=1024,
                                       tree_mask=bits.to(cuda_dev), return_lse=True)
    check_attention(out, lse, attend_ref(w, q, 2, sees, 0.125))


def test_sequences_that_share_pages(cuda_dev):
    """Two sequences over the same prefix pages answer as each would alone."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, torch.int8, [200], [1], 2, 64, 16).fill()
    q = torch.randn((1, 8 * 64), generator=w.g).to(torch.bfloat16).to(cuda_dev)
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    call = lambda q, lens: kv_cache.tree_attention(q, w.cache, i32(*range(len(lens) + 1)), i32(*lens),  # noqa: E731
                                                   w.table.expand(len(lens), -1).contiguous(), max_nodes=1)
    both = call(torch.cat([q, q, q]), [200, 90, 200])
    assert torch.equal(both[0], both[2])
    for i, n in ((0, 200), (1, 90)):
        o = call(q, [n])[0].float()  # (another split of the keys)
        assert torch.all((both[i].float() - o).abs() <= 2 * BF * o.abs() + 2 * BF)


def test_two_streams_and_two_graphs_at_once(cuda_dev):
    """Calls that run at the same time share nothing; a graph may be captured
    without any call before it."""
    from ncmorph_b200 import kv_cache, ncm_model
    cos, sin = tables(4096, 128, cuda_dev)
    jobs = []
    for seed, dtype, n in ((1, torch.float8_e4m3fn, 3), (2, torch.float8_e4m3fn, 40), (3, torch.int8, 70)):
        w = World(cuda_dev, dtype, [3000, 900, 80], [n, n, n], 2, 128, 32, seed=seed).fill()
        x = torch.randn((3 * n, 8 * 128), generator=w.g).to(torch.bfloat16).to(cuda_dev)
        pos = torch.arange(3 * n, dtype=torch.int32, device=cuda_dev)
        hist = torch.randint(0, 1024, (500,), generator=w.g).to(torch.int32).to(cuda_dev)
        at = torch.linspace(0, 500, 3 * n + 1).int().to(cuda_dev)
        rep = torch.full((3 * n,), 1.5, device=cuda_dev)

        def run(w=w, x=x, pos=pos, hist=hist, at=at, rep=rep, n=n):
            q = ncm_model.rope_bf16(x, pos, cos, sin, 8, 128)
            out, lse = kv_cache.tree_attention(q, w.cache, w.start, w.kv_lens, w.table, max_nodes=n, return_lse=True)
            return out, lse, ncm_model.process_logits(out, tokens=hist, token_start=at, repetition=rep)
        jobs.append(run)
    graphs, outs = [], []
    for run in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
    want = [run() for run in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for turn in range(10):
        for out in outs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        eager = []
        for run, stream in zip(jobs, streams):
            with torch.cuda.stream(stream):
                eager.append(run())
        torch.cuda.synchronize()
        for a, b, c in zip(outs, want, eager):
            assert all(torch.equal(x, y) and torch.equal(z, y) for x, y, z in zip(a, b, c)), turn


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logit_rows_of_any_alignment(cuda_dev, dtype):
    """Rows that start on odd elements give the bits that aligned rows give."""
    from ncmorph_b200 import ncm_model
    g = torch.Generator().manual_seed(5)
    x = torch.randn((3, 3001), generator=g).to(dtype).to(cuda_dev)
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    args = dict(tokens=i32(*range(0, 3000, 7)), token_start=i32(0, 100, 100, 429), presence=torch.ones(3, device=cuda_dev),
                bias_ids=i32(2999, 3000, 0), bias=torch.ones(3, device=cuda_dev), bias_start=i32(0, 1, 1, 3))
    want = ncm_model.process_logits(torch.nn.functional.pad(x, (0, 7))[:, :3001], **args)
    odd = torch.zeros((3, 3013), dtype=dtype, device=cuda_dev)
    for shift in (1, 2, 3):
        odd[:, shift:shift + 3001] = x
        assert torch.equal(ncm_model.process_logits(odd[:, shift:shift + 3001], **args), want)


def test_refusals_of_sizes(cuda_dev):
    import ctypes
    from ncmorph_b200 import _lib, kv_cache, ncm_model
    from ncmorph_b200.device import context_of, raw_stream
    bf = lambda *s: torch.zeros(s, device=cuda_dev, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    cache = kv_cache.KVCache.allocate(64, 16, 1, 64, torch.bfloat16, cuda_dev)
    table, start, lens = torch.zeros((1, 64), dtype=torch.int32, device=cuda_dev), i32(0, 1), i32(1)
    for heads, nodes in ((1, 1025), (65, 1), (64, 513)):
        with pytest.raises(_lib.NcmError):
            kv_cache.tree_attention(bf(1, heads * 64), cache, start, lens, table, max_nodes=nodes)
    with pytest.raises(ValueError):  # a part of a head
        kv_cache.tree_attention(bf(1, 80), cache, start, lens, table, max_nodes=1)
    with pytest.raises(ValueError):
        kv_cache.tree_attention(bf(64), cache, start, lens, table, max_nodes=1)
    with pytest.raises(ValueError):
        kv_cache.tree_attention(bf(1, 64), cache, start, lens, table, max_nodes=1, tree_mask=[[1]])
    with pytest.raises(ValueError):  # a mask without words is not a chain
        kv_cache.tree_attention(bf(1, 64), cache, start, lens, table, max_nodes=1, tree_mask=torch.zeros((1, 0), dtype=torch.int32, device=cuda_dev))
    with pytest.raises(ValueError):
        ncm_model.process_logits(torch.zeros((1, 32), device=cuda_dev), allowed=torch.zeros((0, 1), dtype=torch.int32, device=cuda_dev),
                                 allowed_rows=i32(0))
    with pytest.raises(_lib.NcmError):
        kv_cache.tree_attention(bf(1, 64), cache, start, lens, table, max_nodes=1, tree_mask=torch.zeros((1, 33), dtype=torch.int32, device=cuda_dev))
    for shape in ((4, 1, 16, 96), (4, 1, 24, 64), (4, 1, 4, 64), (4, 1, 2048, 64)):
        odd = kv_cache.KVCache.allocate(*(shape[i] for i in (0, 2, 1, 3)), torch.bfloat16, cuda_dev)
        with pytest.raises(_lib.NcmError):
            kv_cache.append(odd, bf(1, shape[3]), bf(1, shape[3]), start, lens, table)
    # a workspace that is missing or too small
    q, out = bf(1, 64), bf(1, 64)
    b = kv_cache._batch(cache, start, lens, table, 1)
    n = ctypes.c_uint64()
    _lib.call("ncm_tree_attention_workspace", context_of(cache.device), cache._ref, ctypes.byref(b), 1, 1, ctypes.byref(n))
    ws = torch.empty(n.value, dtype=torch.uint8, device=cuda_dev)
    for p, size in ((None, n.value), (ws.data_ptr(), n.value - 1), (ws.data_ptr() + 4, n.value)):
        with pytest.raises(_lib.NcmError):
            _lib.call("ncm_tree_attention", context_of(cache.device), cache._ref, ctypes.byref(b), q.data_ptr(), 64, None, 0, 1, 1,
                      0.125, out.data_ptr(), 64, None, p, size, raw_stream(cache.device))
    # lists and rows past what the logit rules take
    x = torch.zeros((1, 32), device=cuda_dev)
    one = torch.ones(1, device=cuda_dev)
    for field, value in (("num_tokens", (1 << 30) + 1), ("num_bias", (1 << 30) + 1), ("num_tokens", -1), ("rows", 65536)):
        r = _lib.LogitRules()
        r.tokens, r.token_start, r.num_tokens = lens.data_ptr(), start.data_ptr(), 1
        r.bias_ids, r.bias, r.bias_start, r.num_bias = lens.data_ptr(), one.data_ptr(), start.data_ptr(), 1
        if field != "rows":
            setattr(r, field, value)
        with pytest.raises(_lib.NcmError):
            _lib.call("ncm_logits_process", context_of(cache.device), x.data_ptr(), ncm_model.LOGIT_TYPES[torch.float32], 32, x.data_ptr(),
                      ncm_model.LOGIT_TYPES[torch.float32], 32, value if field == "rows" else 1, 32, ctypes.byref(r), raw_stream(cache.device))


def test_no_history_yet(cuda_dev):
    """Empty lists are lists: the first step of a generation has no tokens."""
    from ncmorph_b200 import ncm_model
    x = torch.randn((2, 50), device=cuda_dev)
    i32 = lambda *z: torch.tensor(z, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    ones = torch.full((2,), 1.7, device=cuda_dev)
    args = dict(tokens=i32(), token_start=i32(0, 0, 0), repetition=ones, frequency=ones, presence=ones, prompt_lens=i32(0, 0),
                bias=torch.zeros(0, device=cuda_dev), bias_ids=i32(), bias_start=i32(0, 0, 0))
    assert torch.equal(ncm_model.process_logits(x, **args), x)
    args["tokens"], args["token_start"] = i32(), i32(0, 0, 1)  # a bound past the (empty) list
    assert torch.equal(ncm_model.process_logits(x, **args), x)
    expect_range_error(cuda_dev)


@pytest.mark.parametrize("n,L,hd,heads", [(40, 50, 64, 1), (40, 50, 128, 1), (40, 64, 64, 1), (20, 800, 128, 4), (40, 193, 64, 1),
                                          (33, 257, 128, 1), (40, 1100, 64, 1), (60, 449, 128, 2), (64, 600, 64, 4)])
def test_infinite_values_in_the_last_tile(cuda_dev, n, L, hd, heads):
    """Values that are not finite in the very last new tokens only, in every 16th column:
    a softmax group that never waited for that tile writes half of the columns."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, torch.bfloat16, [L, L - 1], [n, n], 1, hd, 16, seed=n + L)
    want = torch.zeros((n, hd), dtype=torch.bool)
    for end in (L, 2 * L - 1):
        w.v[end - 2, ::16], w.v[end - 1, 8::16] = math.inf, -math.inf
    want[n - 2:, ::16], want[n - 1:, 8::16] = True, True
    want = want.repeat(2, heads)
    w.fill()
    q = torch.randn((2 * n, heads * hd), generator=w.g).to(torch.bfloat16)
    args = (q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table)
    out, lse = kv_cache.tree_attention(*args, max_nodes=n, return_lse=True)
    for _ in range(20):
        again, lse2 = kv_cache.tree_attention(*args, max_nodes=n, return_lse=True)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
    out = out.cpu()
    assert torch.equal(torch.isinf(out), want) and not torch.isnan(out).any()
    up = torch.arange(hd).repeat(heads) % 16 == 0
    assert torch.all(out[:, up][want[:, up]] > 0) and torch.all(out[:, ~up][want[:, ~up]] < 0)
    w.v[~torch.isfinite(w.v)] = 0.0
    o, l, to, tl = attend_ref(w, q, heads, None, hd ** -0.5)
    assert torch.all(((out.double() - o).abs() <= to) | want) and torch.all((lse.cpu().double() - l).abs() <= tl)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("most,heads,hd", [(40, 4, 64), (12, 16, 128), (50, 16, 64), (60, 8, 128)])
@pytest.mark.parametrize("split", [False, True])
def test_many_items_of_many_rows(cuda_dev, dtype, most, heads, hd, split):
    """Several times as many items as the tcgen05 kernel has CTAs: runs of segments of one
    tile among longer ones, odd and even tile counts, sequences without new tokens and
    ones that leave warps, or one group of 128 rows, without any row."""
    from ncmorph_b200 import kv_cache
    g = torch.Generator().manual_seed(most * heads)
    lens = [int(x) for x in torch.randint(1, 201, (130,), generator=g)]
    lens[20:60] = [1 + (7 * b) % 64 for b in range(40)]
    if split:  # long ones are shared by several CTAs
        lens[70], lens[129] = 1537, 3000
    new = [min(n, int(x)) for n, x in zip(lens, torch.randint(0, most + 1, (130,), generator=g))]
    new[25:45] = [min(n, 1 + b % 3) for b, n in enumerate(lens[25:45])]
    w = World(cuda_dev, dtype, lens, new, 4, hd, 16, seed=most).fill()
    q = torch.randn((w.T, heads * hd), generator=w.g).to(torch.bfloat16)
    sees, bits = tree_masks(new, w.g)
    args = (q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table)
    out, lse = kv_cache.tree_attention(*args, max_nodes=most, tree_mask=bits.to(cuda_dev), return_lse=True)
    again, _ = kv_cache.tree_attention(*args, max_nodes=most, tree_mask=bits.to(cuda_dev), return_lse=True)
    assert torch.equal(out, again)
    check_attention(out, lse, attend_ref(w, q, heads, sees, hd ** -0.5))


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("n", [1, 5])
def test_split_changes_no_rounding_of_probabilities(cuda_dev, dtype, n):
    """A sequence alone and among others: its keys are dealt out differently, and maxima
    move by powers of two only, so the 16-bit probabilities stay.

    Scores have the same bits. A probability is 2^(t - m), whose difference of up to 2^4 is
    rounded by 2^-21: 2^-20 apart, relative to itself, in two splits, so it falls on two sides
    of a border of its rounding (steps of 2^-8 for one bf16 value or, over codes, 2^-11, relative to it) with a chance
    of 2^-12 or 2^-9, and is then a step off. For an output, a sum of many of random signs,
    that is sqrt(2^-12) 2^-8 or sqrt(2^-9) 2^-11 of itself, about 2^-14 or 2^-15.5; the f32 sums'
    order is below that. It takes another bf16 (steps of 2^-8 to 2^-7) with a chance of 1.6 % or 0.6 %.
    Probabilities rounded independently are 2^-9.3 (2^-12.3) apart: 40 % or 5 %."""
    from ncmorph_b200 import kv_cache
    lens = [1700, 2950, 300, 2100, 40, 900, 3500, 128, 1300, 2600, 777, 1500, 64]
    w = World(cuda_dev, dtype, lens, [n] * len(lens), 8, 64, 16, seed=n).fill()
    q = torch.randn((w.T, 32 * 64), generator=w.g).to(torch.bfloat16).to(cuda_dev)
    out, lse = kv_cache.tree_attention(q, w.cache, w.start, w.kv_lens, w.table, max_nodes=n, return_lse=True)
    alone, lse2 = kv_cache.tree_attention(q[:4 * n].contiguous(), w.cache, w.starts([n] * 4), w.kv_lens[:4].contiguous(),
                                          w.table[:4].contiguous(), max_nodes=n, return_lse=True)
    share = float((out[:4 * n] != alone).float().mean())
    assert share <= (0.08 if dtype == torch.bfloat16 else 0.025), share
    assert torch.all((lse[:4 * n] - lse2).abs() <= 2.0 ** -18 * (1 + lse2.abs()))


@pytest.mark.parametrize("start,n", [([0, 3, 5], 3), ([0, 2, 1], 2), ([0, 3, -2], 3), ([3, 3, 9], 0)])
def test_sequences_that_no_row_leads_to(cuda_dev, start, n):
    """The second sequence's rows are past the end, or fewer than none: reported, although
    the call has no row of it; the first one's n rows are written and read."""
    from ncmorph_b200 import device, kv_cache
    w = World(cuda_dev, torch.bfloat16, [20, 20], [1, 1], 1, 64, 16).fill()
    rows = torch.randn((3, 64), generator=w.g).to(torch.bfloat16).to(cuda_dev)
    starts = torch.tensor(start, dtype=torch.int32, device=cuda_dev)
    before = w.cache.k.clone()
    kv_cache.append(w.cache, rows, rows, starts, w.kv_lens, w.table)
    expect_range_error(cuda_dev)
    assert int((w.cache.k.view(torch.int16) != before.view(torch.int16)).any(-1).sum()) == n
    out = torch.full((3, 64), 3.0, device=cuda_dev).to(torch.bfloat16)
    kv_cache.gather(w.cache, starts, w.table, out_k=out, out_v=out.clone())
    expect_range_error(cuda_dev)
    assert torch.all(out[n:] == 3.0) and not torch.any((out[:n] == 3.0).all(-1))
    # one of many sequences, whose other numbers are those of empty ones
    at = torch.zeros(602, dtype=torch.int32, device=cuda_dev)
    lens, table = torch.zeros(601, dtype=torch.int32, device=cuda_dev), torch.zeros((601, 1), dtype=torch.int32, device=cuda_dev)
    kv_cache.append(w.cache, rows[:1], rows[:1], at, lens, table)
    device.sync(cuda_dev)
    at[451:] = -1
    kv_cache.append(w.cache, rows[:1], rows[:1], at, lens, table)
    expect_range_error(cuda_dev)


def test_single_rows_in_place_with_any_stride(cuda_dev):
    """One row's stride says nothing: two views of one row are the same row."""
    from ncmorph_b200 import ncm_model
    cos, sin = tables(9, 64, cuda_dev)
    pos = torch.tensor([7], dtype=torch.int32, device=cuda_dev)
    row = torch.randn(5 * 64, device=cuda_dev).to(torch.bfloat16)
    x, out = row.unsqueeze(0), row[:3 * 64].unsqueeze(0)
    assert x.stride(0) != out.stride(0)
    want = ncm_model.rope_bf16(x, pos, cos, sin, 3, 64)
    rest = row[3 * 64:].clone()
    ncm_model.rope_bf16(x, pos, cos, sin, 3, 64, out=out)
    assert torch.equal(out, want) and torch.equal(row[3 * 64:], rest)
    buf = torch.randn(40, device=cuda_dev)
    logits, out = torch.as_strided(buf, (1, 33), (40, 1)), torch.as_strided(buf, (1, 33), (48, 1))
    toks, at = torch.tensor([3, 3, 32], dtype=torch.int32, device=cuda_dev), torch.tensor([0, 3], dtype=torch.int32, device=cuda_dev)
    pen = torch.tensor([0.5], device=cuda_dev)
    want = ncm_model.process_logits(logits, toks, at, frequency=pen)
    tail = buf[33:].clone()
    ncm_model.process_logits(logits, toks, at, frequency=pen, out=out)
    assert torch.equal(out, want) and torch.equal(buf[33:], tail)


def test_rows_that_overlap_are_refused(cuda_dev):
    """Keys and values read back into each other, and rows that lie in a pool. Column
    slices of one buffer lie apart, whatever their order."""
    from ncmorph_b200 import _lib, kv_cache
    from ncmorph_b200.kv_cache import KVCache
    w = World(cuda_dev, torch.bfloat16, [9], [9], 1, 64, 16).fill()
    buf = torch.zeros((9, 192), dtype=torch.bfloat16, device=cuda_dev)
    at = w.starts([9])
    flat = buf.view(-1)
    shifted = torch.as_strided(flat, (4, 64), (128, 1), 8)
    whole = kv_cache.gather(w.cache, at, w.table, rows=9)
    for a, b in ((buf, buf), (buf[:, :64], buf[:, 32:96]), (buf[:, 120:184], buf[:, 64:192])):
        with pytest.raises(_lib.NcmError):
            kv_cache.gather(w.cache, at, w.table, out_k=a, out_v=b)
    with pytest.raises(_lib.NcmError):  # rows of other strides over one range
        kv_cache.gather(w.cache, w.starts([4]), w.table, out_k=buf[:4], out_v=shifted)
    for a, b in ((buf[:, :64], buf[:, 64:]), (buf[:, 128:], buf[:, :64]), (buf[:, 64:128], buf[:, 128:]),
                 (buf[:, 120:184], buf[:, 56:184])):  # (the first 64 columns of a slice are used)
        k, v = kv_cache.gather(w.cache, at, w.table, out_k=a, out_v=b)
        assert torch.equal(k[:, :64], whole[0]) and torch.equal(v[:, :64], whole[1])
    # one below the other, the last row of the first beside the first of the second
    k, v = torch.as_strided(flat, (5, 64), (128, 1), 0), torch.as_strided(flat, (5, 64), (128, 1), 4 * 128 + 64)
    kv_cache.gather(w.cache, w.starts([5]), w.table, out_k=k, out_v=v)
    assert torch.equal(k, whole[0][:5]) and torch.equal(v, whole[1][:5])
    arena = torch.zeros((4, 1, 16, 64), dtype=torch.bfloat16, device=cuda_dev)
    cache = KVCache(arena[:2], arena[2:])
    apart, inside, edge = buf[:, :64], arena[1, 0, 4:13], torch.zeros((9, 64), dtype=torch.bfloat16, device=cuda_dev)
    table = torch.zeros((1, 1), dtype=torch.int32, device=cuda_dev)
    for k, v in ((apart, inside), (inside, apart), (arena[3, 0, 7:], apart)):
        with pytest.raises(_lib.NcmError):
            kv_cache.append(cache, k, v, at, w.kv_lens, table)
        with pytest.raises(_lib.NcmError):
            kv_cache.gather(cache, at, table, out_k=k, out_v=v)
    kv_cache.append(cache, edge, edge, at, w.kv_lens, table)  # the same rows twice, only read


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("exponent", [-90, 80])
@pytest.mark.parametrize("n,heads", [(1, 4), (8, 4), (40, 4)])
def test_smallest_and_largest_values(cuda_dev, dtype, exponent, n, heads):
    """Values at both ends of the documented range: nothing is lost or overflows."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, dtype, [2000, 60 + n], [n, n], 2, 64, 16, seed=n)
    w.v = (w.v.double() * 2.0 ** exponent / w.v.double().abs().amax(1, keepdim=True)).to(torch.bfloat16)
    w.fill()
    q = torch.randn((w.T, heads * 64), generator=w.g).to(torch.bfloat16)
    out, lse = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=n, return_lse=True)
    o, l, to, tl = attend_ref(w, q, heads, None, 0.125)
    to = to - 1e-37  # (an allowance for results near the end of f32's range, where these are not)
    assert torch.all((out.cpu().double() - o).abs() <= to) and torch.all((lse.cpu().double() - l).abs() <= tl)


@pytest.mark.parametrize("dtype", FORMATS)
def test_accepted_tokens_are_appended_again(cuda_dev, dtype):
    """After drafted tokens are verified, the accepted ones lie apart in the cache. Their rows are
    still in the step's own arrays: appended again behind the context, they are the cache of
    a context that was written token by token, with the same codes."""
    from ncmorph_b200 import kv_cache
    w = World(cuda_dev, dtype, [50, 33], [9, 7], 2, 64, 16).fill()
    taken = [[0, 2, 5, 8], [1]]  # a path of each tree
    rows = torch.tensor([w.at[b] + w.lens[b] - w.new[b] + i for b in range(2) for i in taken[b]])
    lens = torch.tensor([w.lens[b] - w.new[b] + len(taken[b]) for b in range(2)], dtype=torch.int32, device=cuda_dev)
    kv_cache.append(w.cache, w.k[rows].to(cuda_dev), w.v[rows].to(cuda_dev), w.starts([4, 1]), lens, w.table)
    k, v = kv_cache.gather(w.cache, w.starts(lens.tolist()), w.table, rows=int(lens.sum()))
    order = torch.cat([torch.cat([torch.arange(w.at[b], w.at[b] + w.lens[b] - w.new[b]), rows[4 * b:4 + b]]) for b in range(2)])
    plain = World(cuda_dev, dtype, lens.tolist(), [1, 1], 2, 64, 16, seed=1)
    plain.k, plain.v = w.k[order], w.v[order]
    plain.fill()
    k2, v2 = kv_cache.gather(plain.cache, w.starts(lens.tolist()), plain.table, rows=int(lens.sum()))
    assert torch.equal(k, k2) and torch.equal(v, v2)


@pytest.mark.parametrize("lens", [[1, 2, 5], [12, 31, 79], [200, 1500, 3]])
@pytest.mark.parametrize("n,heads,hd", [(1, 1, 64), (1, 16, 64), (1, 16, 128), (3, 4, 64), (3, 4, 128), (4, 8, 64), (4, 8, 128)])
def test_probabilities_over_a_bf16_cache(cuda_dev, lens, n, heads, hd):
    """Up to 32 rows of a kv head: probabilities are two bf16 values. The first is cut off, up to
    2^-7 of a term below it, and half a step of the second, the rest, is 2^-8 of that; with
    the 2^-20 that are added, 2^-15 + 2^-20 of a term. So little but the output's own rounding is
    seen, and a row that sees one key returns its value: half of a bf16 step is 2^-9 of it or more."""
    from ncmorph_b200 import kv_cache
    new = [min(n, x) for x in lens]
    w = World(cuda_dev, torch.bfloat16, lens, new, 1, hd, 16, seed=n * hd).fill()
    q = torch.randn((w.T, heads * hd), generator=w.g).to(torch.bfloat16)
    out = kv_cache.tree_attention(q.to(cuda_dev), w.cache, w.start, w.kv_lens, w.table, max_nodes=n).cpu()
    o, _, to, _ = attend_ref(w, q, heads, None, hd ** -0.5)
    k0 = int(w.at[0])
    if lens[0] == new[0]:  # its first new token sees itself only
        assert torch.equal(out[0].view(heads, hd), w.v[k0].expand(heads, hd))
    # check_attention's tolerance holds 2^-8 of every term for P
    K, V = w.held(w.k), w.held(w.v)
    row = 0
    for b, m in enumerate(new):
        k, v = K[w.at[b]:w.at[b] + lens[b], 0], V[w.at[b]:w.at[b] + lens[b], 0]
        t = torch.einsum("nhd,ld->nhl", q[row:row + m].double().view(m, heads, hd), k) * hd ** -0.5
        seen = torch.arange(lens[b])[None] <= lens[b] - m + torch.arange(m)[:, None]
        p = torch.softmax(t.masked_fill(~seen[:, None], -math.inf), -1)
        spread = torch.einsum("nhl,ld->nhd", p, v.abs()).reshape(m, -1)
        tol = to[row:row + m] - (BF - 2.0 ** -15 - 2.0 ** -20) * spread
        assert torch.all((out[row:row + m].double() - o[row:row + m]).abs() <= tol)
        row += m
