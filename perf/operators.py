"""What the decode-step operators are measured on: rotary positions, the paged
key/value cache (written and read back), attention of drafted tokens over it,
and the penalties, biases and grammar masks on the head's logits.

``run`` computes a case in plain torch operations in 32 bits, or, with ``own``
set, by the framework's entry points; ``exact`` computes it from the
definitions in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
POOL_DTYPE = {"bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


# --------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of 48 sequences through the decoder's 32 query and 8 key heads of 64
        dict(name="rope step", op="rope", T=48, heads=40, head_dim=64, rotary=64, interleaved=False, inverse=False,
             positions=131072),
        # the gradient of a long prompt's rotation, half of a 128-wide head, neighbouring pairs
        dict(name="rope gradient", op="rope", T=16384, heads=40, head_dim=128, rotary=64, interleaved=True, inverse=True,
             positions=32768),
        # one new token for each of 64 sequences: the write of every decode step
        dict(name="cache write step", op="write", batch=64, nodes=1, longest=4099, kv_heads=8, head_dim=64, page=16,
             fmt="int8"),
        # prompt chunks of different lengths entering the cache
        dict(name="cache write chunks", op="write", batch=8, nodes=2048, longest=8192, kv_heads=8, head_dim=128, page=64,
             fmt="e4m3"),
        # a few short contexts read back, pages that end inside a row block
        dict(name="cache read short", op="read", batch=4, longest=701, kv_heads=8, head_dim=128, page=16, fmt="e4m3"),
        # whole contexts read back as rows for the prefill attention
        dict(name="cache read long", op="read", batch=16, longest=16384, kv_heads=8, head_dim=64, page=32, fmt="int8"),
        # the smallest decode step: single tokens over short contexts, latency only
        dict(name="attend short", op="attend", batch=4, nodes=1, longest=200, heads=32, kv_heads=8, head_dim=64, page=16,
             fmt="bf16", tree=False),
        # a serving batch, contexts from 2 thousand to 32 thousand tokens, single tokens
        dict(name="attend batch", op="attend", batch=32, nodes=1, longest=32768, heads=32, kv_heads=8, head_dim=64, page=32,
             fmt="int8", tree=False),
        # drafted trees of up to 26 tokens over medium contexts, 128-wide heads
        dict(name="attend trees", op="attend", batch=8, nodes=26, longest=8191, heads=32, kv_heads=8, head_dim=128, page=64,
             fmt="e4m3", tree=True),
        # two large trees over very long contexts
        dict(name="attend long trees", op="attend", batch=2, nodes=64, longest=131072, heads=32, kv_heads=8, head_dim=64,
             page=64, fmt="bf16", tree=True),
        # one step of a few requests on the language-model head
        dict(name="logits step", op="logits", rows=4, vocab=128256, history=900, biases=24, dtype="f32", grammar=True),
        # a codebook head's rows for a whole level, bf16 logits, long histories
        dict(name="logits level", op="logits", rows=512, vocab=16384, history=4000, biases=300, dtype="bf16", grammar=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attend", "attend", "logits"])
    if op == "rope":
        hd = rng.choice([64, 80, 96, 128])
        return dict(op=op, T=_log_int(rng, 1, 12000), heads=rng.choice([1, 3, 5, 12, 24, 40]), head_dim=hd,
                    rotary=rng.choice([hd, hd // 2, 32, 20]), interleaved=rng.random() < 0.5,
                    inverse=rng.random() < 0.5, positions=_log_int(rng, 64, 131072))
    fmt = rng.choice(["bf16", "int8", "e4m3"])
    cache = dict(kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), fmt=fmt)
    if op == "write":
        nodes = _log_int(rng, 1, 2000)
        return dict(op=op, batch=_log_int(rng, 1, max(1, min(64, 16000 // nodes))), nodes=nodes,
                    longest=_log_int(rng, nodes, 8000), **cache)
    if op == "read":
        return dict(op=op, batch=_log_int(rng, 1, 12), longest=_log_int(rng, 1, 10000), **cache)
    if op == "attend":
        nodes = rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 2, 64)])
        batch = _log_int(rng, 1, 32)
        longest = _log_int(rng, nodes, max(nodes + 1, min(65000, 400000 // (batch * max(1, nodes // 8)))))
        return dict(op=op, batch=batch, nodes=nodes, longest=longest, heads=cache["kv_heads"] * rng.choice([1, 2, 4, 5, 8] if cache["kv_heads"] < 8 else [1, 2, 4]),
                    tree=nodes > 1 and rng.random() < 0.7, **cache)
    vocab = rng.choice([_log_int(rng, 500, 150000), 4096, 8192, 16384, 128256])
    return dict(op=op, rows=_log_int(rng, 1, max(1, min(512, 8000000 // vocab))), vocab=vocab, history=_log_int(rng, 1, 4000),
                biases=rng.choice([0, 1, 17, 300]), dtype=rng.choice(["f32", "bf16"]), grammar=rng.random() < 0.6)


def _lengths(case):
    """Tokens in the cache and new tokens of each sequence: by the case alone, so that every seed has the same work."""
    B, longest, nodes = case["batch"], case["longest"], case.get("nodes", 0)
    new = [max(1, nodes - (b * 5) % (nodes // 2 + 1)) if nodes else 0 for b in range(B)]
    lens = [max(1, new[b], int(longest * 16.0 ** (-b / max(1, B - 1))) - (b * 7) % 5) for b in range(B)]
    return lens, new


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["T"] * case["heads"]
        return {"bytes": 4 * n * case["head_dim"] + case["T"] * (4 + 4 * case["rotary"]), "flops": 3 * n * case["rotary"]}
    if op == "logits":
        n, size = case["rows"] * case["vocab"], 4 if case["dtype"] == "f32" else 2
        lists = case["rows"] * (4 * case["history"] + 8 * case["biases"])
        return {"bytes": n * (size + 4) + (n // 8 if case["grammar"] else 0) + lists, "flops": 4 * n}
    lens, new = _lengths(case)
    row = case["kv_heads"] * case["head_dim"]  # one token's keys, or its values
    held = row * (2 if case["fmt"] == "bf16" else 1) + (0 if case["fmt"] == "bf16" else 4 * case["kv_heads"])
    if op == "write":  # rows in, codes out; codes in, rows out
        return {"bytes": sum(new) * 2 * (2 * row + held + held + 2 * row), "flops": sum(new) * 2 * 4 * row}
    if op == "read":
        return {"bytes": sum(lens) * 2 * (held + 2 * row), "flops": sum(lens) * 2 * row}
    width = case["heads"] * case["head_dim"]
    return {"bytes": sum(lens) * 2 * held + sum(new) * (4 * width + 4 * case["heads"]),
            "flops": 4 * width * sum(a * b for a, b in zip(lens, new))}


# -------------------------------------------------------------------- inputs

def _quantise(x, fmt):
    """Codes and scales of rows of the last dimension: code = round(M x / max|x|), scale = max|x| / M."""
    top = CODE_MAX[fmt]
    x = x.float()
    big = x.abs().amax(-1, keepdim=True)
    some = big > 0
    y = x * top / torch.where(some, big, 1.0)
    codes = torch.round(y).to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)
    scale = torch.where(some, big / top, 1.0)
    return codes, scale.squeeze(-1)


def _starts(counts):
    total = [0]
    for n in counts:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device=DEV)


def _tree_bits(rng, n, words):
    """Rows of bits: each node sees its ancestors and itself; parents are drawn among the earlier nodes."""
    rows, words_of = [], []
    for i in range(n):
        bits = 1 << i
        if i:
            bits |= rows[rng.randrange(max(0, i - 6), i)]
        rows.append(bits)
        words_of.append([((bits >> (32 * w)) & 0xFFFFFFFF) - ((bits >> (32 * w + 31) & 1) << 32) for w in range(words)])
    return words_of


def _cache_inputs(case, seed, g):
    lens, new = _lengths(case)
    B, page, kvh, hd, fmt = case["batch"], case["page"], case["kv_heads"], case["head_dim"], case["fmt"]
    need = [-(-n // page) for n in lens]
    width = max(need) + 1
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    at = torch.zeros((B, width), dtype=torch.int64)
    used = 0
    for b, n in enumerate(need):
        at[b, :n] = torch.arange(used, used + n)
        used += n
    table = order[at.to(DEV)].contiguous()
    s = dict(case=case, lens=lens, new=new, page_table=table, kv_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
             token_start=_starts(new if sum(new) else lens))
    shape = (pages, kvh, page, hd)
    channel = torch.exp(0.5 * torch.randn((kvh, 1, hd), generator=g, device=DEV))  # keys have strong and weak channels
    for name in ("k", "v"):
        pool = torch.empty(shape, dtype=POOL_DTYPE[fmt], device=DEV)
        scales = None if fmt == "bf16" else torch.empty(shape[:3], dtype=torch.float32, device=DEV)
        step = max(1, (1 << 26) // (kvh * page * hd))
        for p in range(0, pages, step):
            x = torch.randn((min(step, pages - p),) + shape[1:], generator=g, device=DEV)
            x = (x * channel if name == "k" else x).to(torch.bfloat16)
            if fmt == "bf16":
                pool[p:p + step] = x
            else:
                pool[p:p + step], scales[p:p + step] = _quantise(x, fmt)
        s[name], s[name + "_scale"] = pool, scales
    if own:  # the handle that a program keeps beside its pools: it holds these tensors and nothing computed from them
        from ncmorph_b200 import kv_cache
        s["cache"] = kv_cache.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    if op == "rope":
        half = case["rotary"] // 2
        freq = 500000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        angle = torch.arange(case["positions"], dtype=torch.float64, device=DEV)[:, None] * freq
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
        return dict(case=case, x=torch.randn((case["T"], case["heads"] * case["head_dim"]), generator=g, device=DEV).to(torch.bfloat16),
                    positions=torch.randint(0, case["positions"], (case["T"],), generator=g, device=DEV, dtype=torch.int32),
                    cos=torch.cat([cos, cos], 1), sin=torch.cat([sin, sin], 1))
    if op == "logits":
        R, V, rng = case["rows"], case["vocab"], random.Random(seed)
        logits = 3.0 * torch.randn((R, V), generator=g, device=DEV)
        u = torch.rand((R, case["history"]), generator=g, device=DEV, dtype=torch.float64)
        tokens = (V * u ** 3).long().clamp_(max=V - 1).to(torch.int32)  # few tokens are frequent
        s = dict(case=case, logits=logits if case["dtype"] == "f32" else logits.to(torch.bfloat16), tokens=tokens.reshape(-1),
                 token_start=_starts([case["history"]] * R),
                 prompt_lens=torch.tensor([rng.randrange(case["history"] + 1) for _ in range(R)], dtype=torch.int32, device=DEV),
                 repetition=1.0 + 0.5 * torch.rand(R, generator=g, device=DEV),
                 frequency=0.3 * torch.rand(R, generator=g, device=DEV), presence=0.6 * torch.rand(R, generator=g, device=DEV),
                 bias_ids=None, bias=None, bias_start=None, allowed=None, allowed_rows=None)
        if case["biases"]:
            n = min(case["biases"], V)
            ids = [torch.randperm(V, generator=g, device=DEV)[:n] for _ in range(R)]
            s["bias_ids"] = torch.cat(ids).to(torch.int32)
            s["bias"] = 4.0 * torch.randn(R * n, generator=g, device=DEV)
            s["bias_start"] = _starts([n] * R)
        if case["grammar"]:  # a quarter of the rows are free, the others share a few grammar states
            states, words = max(1, R // 2), -(-V // 32)
            bits = torch.randint(-2 ** 31, 2 ** 31, (3, states, words), generator=g, device=DEV, dtype=torch.int64)
            s["allowed"] = (bits[0] & bits[1] & bits[2]).to(torch.int32)
            s["allowed_rows"] = torch.tensor([-1 if r % 4 == 3 else rng.randrange(states) for r in range(R)], dtype=torch.int32, device=DEV)
        return s
    s = _cache_inputs(case, seed, g)
    T, row = sum(s["new"]), case["kv_heads"] * case["head_dim"]
    if op == "write":
        s["new_k"] = torch.randn((T, row), generator=g, device=DEV).to(torch.bfloat16)
        s["new_v"] = torch.randn((T, row), generator=g, device=DEV).to(torch.bfloat16)
        s["begin"] = torch.tensor([a - b for a, b in zip(s["lens"], s["new"])], dtype=torch.int32, device=DEV)
    if op == "attend":
        s["q"] = torch.randn((T, case["heads"] * case["head_dim"]), generator=g, device=DEV).to(torch.bfloat16)
        s["tree_mask"] = None
        if case["tree"]:
            rng, words = random.Random(seed), -(-case["nodes"] // 32)
            s["tree_mask"] = torch.tensor([r for n in s["new"] for r in _tree_bits(rng, n, words)], dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------- plain forms

def _rope(s):
    c = s["case"]
    T, H, hd, r = c["T"], c["heads"], c["head_dim"], c["rotary"]
    h = r // 2
    x = s["x"].view(T, H, hd).float()
    p = s["positions"].long()
    cos, sin = s["cos"][p, None, :h], s["sin"][p, None, :h]
    if c["inverse"]:
        sin = -sin
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :h], x[..., h:r])
    y = x.clone()
    ra, rb = a * cos - b * sin, b * cos + a * sin
    if c["interleaved"]:
        y[..., 0:r:2], y[..., 1:r:2] = ra, rb
    else:
        y[..., :h], y[..., h:r] = ra, rb
    return y.to(torch.bfloat16).view(T, H * hd)


def _row_places(s, begin, counts):
    """Page and offset in it of each packed row: row i of sequence b is its position begin[b] + i."""
    start = s["token_start"].long()
    T = sum(counts)
    seq = torch.searchsorted(start, torch.arange(T, device=DEV), right=True) - 1
    pos = torch.arange(T, device=DEV) - start[seq] + begin.long()[seq]
    page = s["case"]["page"]
    return s["page_table"][seq, pos // page].long(), pos % page


def _read_rows(s, name, page, off):
    x = s[name][page, :, off].float()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][page, :, off][..., None]
    return x.to(torch.bfloat16).flatten(1)


def _write(s):
    c = s["case"]
    page, off = _row_places(s, s["begin"], s["new"])
    for name in ("k", "v"):
        x = s["new_" + name].view(-1, c["kv_heads"], c["head_dim"])
        if c["fmt"] == "bf16":
            s[name][page, :, off] = x
        else:
            codes, scale = _quantise(x, c["fmt"])
            s[name].view(torch.uint8)[page, :, off] = codes.view(torch.uint8)
            s[name + "_scale"][page, :, off] = scale
    return {"k": _read_rows(s, "k", page, off), "v": _read_rows(s, "v", page, off)}


def _read(s):
    page, off = _row_places(s, torch.zeros_like(s["kv_lens"]), s["lens"])
    return {"k": _read_rows(s, "k", page, off), "v": _read_rows(s, "v", page, off)}


def _keys_padded(s, name):
    """[batch, kv_heads, keys, head_dim] in 32 bits, keys behind a sequence's last among them."""
    t = s["page_table"].long()
    x = s[name][t].float()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][t][..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s):
    c = s["case"]
    B, n, kvh, hd = c["batch"], max(s["new"]), c["kv_heads"], c["head_dim"]
    g = c["heads"] // kvh
    start, T = s["token_start"].long(), sum(s["new"])
    node = torch.arange(n, device=DEV)
    count = start[1:] - start[:-1]
    row = (start[:-1, None] + node).clamp(max=T - 1)  # [B, n]
    q = s["q"][row].float().view(B, n, kvh, g, hd).permute(0, 2, 1, 3, 4).reshape(B, kvh, n * g, hd)
    k = _keys_padded(s, "k")
    scores = torch.matmul(q, k.transpose(2, 3)) * hd ** -0.5
    del k
    key = torch.arange(scores.shape[-1], device=DEV)
    at = key - (s["kv_lens"].long() - count)[:, None]  # which new token a key is; negative: context
    if s["tree_mask"] is None:
        seen = at[:, None, :] <= node[:, None]
    else:
        bits = s["tree_mask"].long()[row]  # [B, n, words]
        word = (at.clamp(min=0) // 32).clamp(max=bits.shape[-1] - 1)
        bit = torch.gather(bits, 2, word[:, None, :].expand(B, n, -1)) >> (at.clamp(min=0) % 32)[:, None, :]
        seen = (at[:, None, :] < 0) | (bit & 1).bool()
    seen = seen & (at < count[:, None])[:, None, :]
    scores.masked_fill_(~seen[:, None].repeat_interleave(g, 2), -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, _keys_padded(s, "v")) / torch.where(total > 0, total, 1.0)
    lse = top + torch.log(total)
    live = node < count[:, None]
    out = out.view(B, kvh, n, g, hd).permute(0, 2, 1, 3, 4)[live].reshape(T, c["heads"] * hd).to(torch.bfloat16)
    return {"out": out, "lse": lse.view(B, kvh, n, g).permute(0, 2, 1, 3)[live].reshape(T, c["heads"])}


def _logits(s):
    c = s["case"]
    R, V = c["rows"], c["vocab"]
    x = s["logits"].float()
    start = s["token_start"].long()
    at = torch.arange(s["tokens"].numel(), device=DEV)
    row = torch.searchsorted(start, at, right=True) - 1
    place = row * V + s["tokens"].long()
    ones = torch.ones_like(place, dtype=torch.int32)
    produced = (at - start[row] >= s["prompt_lens"].long()[row]).to(torch.int32)
    seen = torch.zeros(R * V, dtype=torch.int32, device=DEV).index_add_(0, place, ones).view(R, V) > 0
    count = torch.zeros(R * V, dtype=torch.int32, device=DEV).index_add_(0, place, produced).view(R, V)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        n = torch.arange(s["bias"].numel(), device=DEV)
        owner = torch.searchsorted(s["bias_start"].long(), n, right=True) - 1
        x = x.reshape(-1).index_add(0, owner * V + s["bias_ids"].long(), s["bias"]).view(R, V)
    if s["allowed"] is not None:
        token = torch.arange(V, device=DEV)
        bits = s["allowed"][s["allowed_rows"].long().clamp(min=0)][:, token // 32] >> (token % 32).to(torch.int32)
        x = torch.where((bits & 1).bool() | (s["allowed_rows"] < 0)[:, None], x, -math.inf)
    return x


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"rope": _rope, "write": _write, "read": _read, "attend": _attend, "logits": _logits}[op](s)
    from ncmorph_b200 import kv_cache, ncm_model
    c = s["case"]
    if op == "rope":
        return ncm_model.rope_bf16(s["x"], s["positions"], s["cos"], s["sin"], c["heads"], c["head_dim"],
                                   interleaved=c["interleaved"], inverse=c["inverse"])
    if op == "logits":
        return ncm_model.process_logits(s["logits"], s["tokens"], s["token_start"], prompt_lens=s["prompt_lens"],
                                        repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                                        bias_ids=s["bias_ids"], bias=s["bias"], bias_start=s["bias_start"],
                                        allowed=s["allowed"], allowed_rows=s["allowed_rows"])
    if op == "write":
        kv_cache.append(s["cache"], s["new_k"], s["new_v"], s["token_start"], s["kv_lens"], s["page_table"])
        k, v = kv_cache.gather(s["cache"], s["token_start"], s["page_table"], rows=s["new_k"].shape[0], begin=s["begin"])
        return {"k": k, "v": v}
    if op == "read":
        k, v = kv_cache.gather(s["cache"], s["token_start"], s["page_table"], rows=sum(s["lens"]))
        return {"k": k, "v": v}
    out, lse = kv_cache.tree_attention(s["q"], s["cache"], s["token_start"], s["kv_lens"], s["page_table"],
                                       max_nodes=c["nodes"], tree_mask=s["tree_mask"], return_lse=True)
    return {"out": out, "lse": lse}


# ------------------------------------------------------------- in 64 bits

def _e4m3_grid(y):
    """The nearest e4m3 value (ties to the even one) of |y| <= 448, in 64 bits."""
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(y / step) * step


def _read_back(x, fmt):
    """What a cache of this format returns for rows of the last dimension."""
    x = x.double()
    if fmt == "bf16":
        return x
    top = CODE_MAX[fmt]
    big = x.abs().amax(-1, keepdim=True)
    y = (x * top) / torch.where(big > 0, big, 1.0)
    return (torch.round(y) if fmt == "int8" else _e4m3_grid(y)) * (big / top)


def _sequence_rows(s, name, b):
    """[length, kv_heads, head_dim] of one sequence, in 64 bits."""
    page, L = s["case"]["page"], s["lens"][b]
    ids = s["page_table"][b, : -(-L // page)].long()
    x = s[name][ids].double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][ids].double().unsqueeze(-1)
    return x.permute(0, 2, 1, 3).reshape(-1, *x.shape[1:2], x.shape[3])[:L]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        T, H, hd, r = case["T"], case["heads"], case["head_dim"], case["rotary"]
        h = r // 2
        i = torch.arange(h, device=DEV)
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + h)
        turn = torch.complex(s["cos"][:, :h].double(), s["sin"][:, :h].double())[s["positions"].long()][:, None]
        x = s["x"].view(T, H, hd).double()
        z = torch.complex(x[..., first], x[..., second]) * (turn.conj() if case["inverse"] else turn)
        x[..., first], x[..., second] = z.real, z.imag
        return x.view(T, H * hd)
    if op == "write":
        return {n: _read_back(s["new_" + n].view(-1, case["kv_heads"], case["head_dim"]), case["fmt"]).flatten(1) for n in ("k", "v")}
    if op == "read":
        return {n: torch.cat([_sequence_rows(s, n, b) for b in range(case["batch"])]).flatten(1) for n in ("k", "v")}
    if op == "attend":
        kvh, hd = case["kv_heads"], case["head_dim"]
        g, at, outs, lses = case["heads"] // kvh, 0, [], []
        for b, (L, n) in enumerate(zip(s["lens"], s["new"])):
            q = s["q"][at:at + n].double().view(n, kvh, g, hd)
            dots = torch.einsum("nhgd,lhd->hgnl", q, _sequence_rows(s, "k", b)) / math.sqrt(hd)
            blocked = torch.zeros((n, L), dtype=torch.bool, device=DEV)
            if s["tree_mask"] is None:
                blocked[:, L - n:] = torch.ones((n, n), dtype=torch.bool, device=DEV).triu(1)
            else:
                j = torch.arange(n, device=DEV)
                words = s["tree_mask"][at:at + n].long() & 0xFFFFFFFF
                blocked[:, L - n:] = ((words[:, j // 32] >> (j % 32)) & 1) == 0
            dots.masked_fill_(blocked, -math.inf)
            lse = torch.logsumexp(dots, -1)
            dots = dots.sub_(lse.unsqueeze(-1)).exp_()
            outs.append(torch.einsum("hgnl,lhd->nhgd", dots, _sequence_rows(s, "v", b)).reshape(n, -1))
            lses.append(lse.permute(2, 0, 1).reshape(n, -1))
            at += n
        return {"out": torch.cat(outs), "lse": torch.cat(lses)}
    x = s["logits"].double()
    start = s["token_start"].tolist()
    for r in range(case["rows"]):
        ids = s["tokens"][start[r]:start[r + 1]].long()
        used = torch.unique(ids)
        f = s["repetition"][r].double()
        x[r, used] = torch.where(x[r, used] > 0, x[r, used] / f, x[r, used] * f)
        made, times = torch.unique(ids[int(s["prompt_lens"][r]):], return_counts=True)
        x[r, made] -= s["frequency"][r].double() * times + s["presence"][r].double()
        if s["bias"] is not None:
            a, b = s["bias_start"][r].item(), s["bias_start"][r + 1].item()
            x[r, s["bias_ids"][a:b].long()] += s["bias"][a:b].double()
        if s["allowed"] is not None and s["allowed_rows"][r] >= 0:
            words = s["allowed"][s["allowed_rows"][r].long()].long()
            bits = (words[:, None] >> torch.arange(32, device=DEV)) & 1
            x[r, bits.reshape(-1)[: case["vocab"]] == 0] = -math.inf
    return x
