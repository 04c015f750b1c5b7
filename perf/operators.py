"""What is measured of the decoder operators around the FP8 GEMMs: the RMS norm that feeds them, rotary positions, the
8-bit paged key / value cache and the attention that reads it.

`run` computes them in plain torch operations (own = False) or through the package's entry points (own = True) on what
`prepare` makes.  Lengths follow from the case alone, values from the seed.
"""

import math
import random

import torch

own = False

PAGE = 128  # tokens of a cache page: one scale per page and key / value head
LO, HI = -60, 60  # exponents that a cache scale may have
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token of a decode step entering a layer: a single row, launch latency
        {"name": "norm_one_token", "op": "norm", "tokens": 1, "hidden": 4096, "dtype": "bf16", "residual": True},
        # a batch without a residual in the other 16-bit type, odd row count
        {"name": "norm_333_f16", "op": "norm", "tokens": 333, "hidden": 5120, "dtype": "f16", "residual": False},
        # a prefill's tokens at the largest hidden size of the GEMM benchmark
        {"name": "norm_prefill", "op": "norm", "tokens": 8192, "hidden": 8192, "dtype": "bf16", "residual": True},
        # a decode batch far into long contexts, half layout
        {"name": "rope_decode", "op": "rope", "tokens": 48, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "far": 900000, "magnitude": 1.0, "dtype": "bf16"},
        # a prefill with interleaved pairs over half of the head and a magnitude factor
        {"name": "rope_prefill_part", "op": "rope", "tokens": 8191, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 64,
         "interleaved": True, "far": 100000, "magnitude": 1.2079, "dtype": "bf16"},
        # every sequence of a decode batch appends its token: rotation, quantisation, pages that must be rescaled
        {"name": "write_decode", "op": "write", "seqs": 128, "new_lo": 1, "new_hi": 1, "past_lo": 0, "past_hi": 1000, "heads": 32,
         "kv_heads": 8, "dim": 128, "rope": True, "dtype": "bf16", "lens": 1},
        # ragged prompts, some continuing in the middle of a page
        {"name": "write_prefill", "op": "write", "seqs": 6, "new_lo": 1, "new_hi": 4000, "past_lo": 0, "past_hi": 700, "heads": 32,
         "kv_heads": 8, "dim": 128, "rope": True, "dtype": "bf16", "lens": 2},
        # a cache read back in 16 bits
        {"name": "read_back", "op": "read", "seqs": 12, "len_lo": 100, "len_hi": 8192, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "lens": 3},
        # one sequence answering: latency
        {"name": "attend_one", "op": "attend", "seqs": 1, "new_lo": 1, "new_hi": 1, "past_lo": 2000, "past_hi": 2000, "heads": 32,
         "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "dtype": "bf16", "lens": 4},
        # a decode batch of very different lengths: the cache's bytes
        {"name": "attend_batch", "op": "attend", "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 0, "past_hi": 16000, "heads": 32,
         "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "dtype": "bf16", "lens": 5},
        # short drafts on long contexts under a sliding window with first tokens kept, small heads, eight to a group
        {"name": "attend_window", "op": "attend", "seqs": 40, "new_lo": 1, "new_hi": 4, "past_lo": 500, "past_hi": 12000, "heads": 64,
         "kv_heads": 8, "dim": 64, "window": 4096, "sinks": 4, "dtype": "f16", "lens": 6},
        # prompts in chunks, the second chunk of some: matrix products
        {"name": "attend_prefill", "op": "attend", "seqs": 4, "new_lo": 300, "new_hi": 2500, "past_lo": 0, "past_hi": 5000, "heads": 32,
         "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0, "dtype": "bf16", "lens": 7},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rope", "write", "read", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "norm":
        hidden = 128 * _log(rng, 1, 64)
        return {"op": op, "tokens": _log(rng, 1, 8192), "hidden": hidden, "dtype": dtype, "residual": rng.random() < 0.6}
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 3, 4, 8])
    if op == "rope":
        return {"op": op, "tokens": _log(rng, 1, 8192), "heads": heads, "kv_heads": kv, "dim": dim,
                "rotary": rng.choice([dim, dim // 2, 32]), "interleaved": rng.random() < 0.5, "far": _log(rng, 1000, 1000000),
                "magnitude": rng.choice([1.0, 1.2079]), "dtype": dtype}
    lens = rng.randrange(1 << 30)
    if op == "write":
        hi = _log(rng, 1, 3000)
        return {"op": op, "seqs": _log(rng, 1, max(1, min(128, 12000 // hi))), "new_lo": rng.randint(1, hi), "new_hi": hi, "past_lo": 0,
                "past_hi": _log(rng, 1, 1000), "heads": heads, "kv_heads": kv, "dim": dim, "rope": rng.random() < 0.7,
                "dtype": dtype, "lens": lens}
    if op == "read":
        hi = _log(rng, 1, 8192)
        return {"op": op, "seqs": _log(rng, 1, max(1, min(64, 90000 // hi))), "len_lo": rng.randint(1, hi), "len_hi": hi, "kv_heads": kv, "dim": dim,
                "dtype": dtype, "lens": lens}
    window = rng.choice([0, 0, _log(rng, 1, 5000)])
    sinks = rng.choice([0, 4, rng.randint(1, 200)]) if window else 0
    case = {"op": op, "heads": heads, "kv_heads": kv, "dim": dim, "window": window, "sinks": sinks, "dtype": dtype, "lens": lens}
    if rng.random() < 0.6:  # decode, drafts among it
        hi = _log(rng, 1, 16000)
        return {**case, "seqs": _log(rng, 1, max(1, min(96, 500000 // hi))), "new_lo": 1, "new_hi": rng.choice([1, 1, rng.randint(2, 8)]),
                "past_lo": rng.choice([0, hi // 2, hi]), "past_hi": hi}
    hi = _log(rng, 16, 2000)  # prompts
    return {**case, "seqs": rng.randint(1, 3), "new_lo": rng.randint(1, hi), "new_hi": hi, "past_lo": 0, "past_hi": _log(rng, 1, 4000)}


# ------------------------------------------------------------------ what a user's program has in hand
def _lengths(case):
    """(new, past) of every sequence; `read` has none that are new."""
    r = random.Random(case["lens"])
    if case["op"] == "read":
        return [0] * case["seqs"], [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["seqs"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    return new, [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["seqs"])]


def _randn(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _pow2(amax):
    """Smallest power of two s with amax / s <= 448, its exponent in [LO, HI]."""
    m, e = torch.frexp(amax)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(LO, HI)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax == 0, torch.full_like(e, LO), e))


def _filled(shape, g):
    """A cache's values: (bytes, scales), every block's largest value near the top of its format."""
    x = _randn(shape, torch.float16, g)
    s = _pow2(x.abs().amax((2, 3)).float())
    x = (x.float() / s[..., None, None]).to(torch.float8_e4m3fn)
    # blocks of different magnitudes
    return x, s * torch.ldexp(torch.ones_like(s), torch.randint(-2, 2, s.shape, generator=g, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": dict(case)}
    if case["op"] == "norm":
        shape = (case["tokens"], case["hidden"])
        x = _randn(shape, dtype, g)
        x[:, torch.randperm(case["hidden"], generator=g, device="cuda")[: max(1, case["hidden"] // 1000)]] *= 20  # outlier channels
        state["x"], state["weight"] = x, _randn(shape[1:], dtype, g, 0.2) + 1
        state["residual"] = _randn(shape, dtype, g, 2.0) if case["residual"] else None
        return state
    H, D = case["kv_heads"], case["dim"]
    if case["op"] == "rope" or case.get("rope"):
        R = case.get("rotary", D)
        state["inv_freq"] = (500000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).cuda()
    if case["op"] == "rope":
        T, Hq = case["tokens"], case["heads"]
        qk = _randn((T, Hq + H, D), dtype, g)
        state["q"], state["k"] = qk[:, :Hq], qk[:, Hq:]  # the two parts of one projection's output
        state["positions"] = torch.randint(0, case["far"], (T,), generator=g, device="cuda")
        return state
    new, past = _lengths(case)
    total = [n + p for n, p in zip(new, past)]
    T, B, pages = sum(new), case["seqs"], max(1, max(-(-t // PAGE) for t in total))
    count = sum(-(-t // PAGE) for t in total) + 3
    state["k_cache"], state["k_scale"] = _filled((count, H, PAGE, D), g)
    state["v_cache"], state["v_scale"] = _filled((count, H, D, PAGE), g)
    order = (torch.randperm(count - 1, generator=g, device="cuda") + 1).tolist()  # page 0 belongs to nobody
    table, at = torch.zeros((B, pages), dtype=torch.int32), 0
    for b, t in enumerate(total):
        n = -(-t // PAGE)
        table[b, :n] = torch.tensor(order[at : at + n], dtype=torch.int32)
        at += n
    state["block_table"] = table.cuda()
    state["seq_lens"] = torch.tensor(total, dtype=torch.int32).cuda()
    state["max_len"] = max(total)
    if case["op"] == "read":
        return state
    state["max_new"] = max(new)
    state["cu_seqlens"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32).cuda()
    qkv = _randn((T, case["heads"] + 2 * H, D), dtype, g)
    state["q"] = qkv[:, : case["heads"]]
    if case["op"] == "write":
        state["k"], state["v"] = qkv[:, case["heads"] : -H], qkv[:, -H:]
    else:
        state["q"] = state["q"].contiguous()
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return _RUN[state["case"]["op"]](state)


def _norm(st):
    x, w, res = st["x"], st["weight"], st["residual"]
    if own:
        import tilegym_b200 as tg

        return tg.rms_norm_quant(x, w, 1e-5, residual=res)
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    f = h.float()
    y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-5) * w.float()
    g = y.unflatten(-1, (-1, 128))
    s = g.abs().amax(-1) / 448.0
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (g / s[..., None]).clamp(-448, 448).flatten(-2).to(torch.float8_e4m3fn)
    return (q, s) if res is None else (q, s, h)


def _rotate(x, positions, inv_freq, interleaved, magnitude):
    """x [tokens, heads, dim] with its first 2 * len(inv_freq) values of a head turned; 32 bits out."""
    R = 2 * inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin = (angle.cos() * magnitude).float()[:, None], (angle.sin() * magnitude).float()[:, None]
    f = x.float()
    if interleaved:
        a, b = f[..., 0:R:2], f[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = f[..., : R // 2], f[..., R // 2 : R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, f[..., R:]), -1)


def _rope(st):
    c = st["case"]
    if own:
        import tilegym_b200 as tg

        return tg.apply_rope(st["q"], st["k"], st["positions"], st["inv_freq"], interleaved=c["interleaved"],
                             magnitude=c["magnitude"])
    args = st["positions"], st["inv_freq"], c["interleaved"], c["magnitude"]
    return _rotate(st["q"], *args).to(st["q"].dtype), _rotate(st["k"], *args).to(st["k"].dtype)


def _write(st):
    if own:
        import tilegym_b200 as tg

        cache = tg.FP8KVCache(st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
        inv_freq = st.get("inv_freq")
        q = tg.kv_cache_write(cache, st["k"], st["v"], st["block_table"], st["seq_lens"], cu_seqlens=st["cu_seqlens"],
                              inv_freq=inv_freq, q=None if inv_freq is None else st["q"])
        out = {"k": cache.k, "v": cache.v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}
        return out if q is None else {**out, "q": q}
    cu, lens, T = st["cu_seqlens"].long(), st["seq_lens"].long(), st["k"].shape[0]
    n = cu[1:] - cu[:-1]
    start = lens - n
    out, k = {}, st["k"]
    if "inv_freq" in st:
        token = torch.arange(T, device="cuda")
        seq = torch.searchsorted(cu[1:], token, right=True)
        positions = start[seq] + token - cu[seq]
        k = _rotate(k, positions, st["inv_freq"], False, 1.0).to(k.dtype)
        out["q"] = _rotate(st["q"], positions, st["inv_freq"], False, 1.0).to(k.dtype)
    tiles = (st["max_new"] + PAGE - 2) // PAGE + 1
    page = start[:, None] // PAGE + torch.arange(tiles, device="cuda")  # [seqs, tiles]
    touched = page * PAGE < lens[:, None]
    pos = page[..., None] * PAGE + torch.arange(PAGE, device="cuda")  # [seqs, tiles, PAGE]
    fresh = (pos >= start[:, None, None]) & (pos < lens[:, None, None])
    kept = (pos < start[:, None, None])[:, :, None, :, None]
    index = (cu[:-1, None, None] + pos - start[:, None, None]).clamp(0, T - 1)
    phys = st["block_table"].long().gather(1, page.clamp(max=st["block_table"].shape[1] - 1))
    phys = torch.where(touched, phys, torch.zeros_like(phys))  # page 0 is nobody's: it gets its own bytes again
    for name, x in (("k", k), ("v", st["v"])):
        cache, scale = st[name + "_cache"], st[name + "_scale"]
        x = x[index].float().transpose(2, 3)  # [seqs, tiles, heads, PAGE, dim]
        new = fresh[:, :, None, :, None]
        s = _pow2(torch.where(new & x.isfinite(), x.abs(), torch.zeros_like(x)).amax((-1, -2)))
        old_s = scale[phys]
        s = torch.where((start[:, None] > page * PAGE)[..., None], torch.maximum(s, old_s), s)
        s = torch.where(touched[..., None], s, old_s)
        old = cache.view(torch.uint8)[phys]
        byte = old if name == "k" else old.transpose(-1, -2)
        moved = (byte.view(torch.float8_e4m3fn).float() * (old_s / s)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        fill = (x / s[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        byte = torch.where(touched[..., None, None, None], torch.where(new, fill, torch.where(kept, moved, byte)), byte)
        cache.view(torch.uint8)[phys] = byte if name == "k" else byte.transpose(-1, -2)
        scale[phys] = s
        out[name], out[name + "_scale"] = cache, scale
    return out


def _gathered(st):
    """k, v [seqs, heads, length, dim] in 32 bits as the pages hold them."""
    t = st["block_table"].long()
    k = st["k_cache"].view(torch.uint8)[t].view(torch.float8_e4m3fn).float() * st["k_scale"][t][..., None, None]
    v = st["v_cache"].view(torch.uint8)[t].view(torch.float8_e4m3fn).float() * st["v_scale"][t][..., None, None]
    return k.transpose(1, 2).flatten(2, 3), v.transpose(-1, -2).transpose(1, 2).flatten(2, 3)


def _read(st):
    dtype = DTYPES[st["case"]["dtype"]]
    if own:
        import tilegym_b200 as tg

        cache = tg.FP8KVCache(st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
        return tg.kv_cache_read(cache, st["block_table"], st["seq_lens"], st["max_len"], dtype)
    keep = torch.arange(st["max_len"], device="cuda")[:, None, None] < st["seq_lens"][:, None, None, None]
    k, v = (x[:, :, : st["max_len"]].transpose(1, 2) for x in _gathered(st))
    zero = torch.zeros((), device="cuda")
    return torch.where(keep, k, zero).to(dtype).contiguous(), torch.where(keep, v, zero).to(dtype).contiguous()


def _attend(st):
    c, q = st["case"], st["q"]
    if own:
        import tilegym_b200 as tg

        cache = tg.FP8KVCache(st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
        return tg.paged_attention(q, cache, st["block_table"], st["seq_lens"], cu_seqlens=st["cu_seqlens"],
                                  max_q_len=st["max_new"], window=c["window"], sinks=c["sinks"])
    B, H, D, N, T = c["seqs"], c["kv_heads"], c["dim"], st["max_new"], q.shape[0]
    cu, lens = st["cu_seqlens"].long(), st["seq_lens"].long()
    n = cu[1:] - cu[:-1]
    row = torch.arange(N, device="cuda")
    qs = q[(cu[:-1, None] + row).clamp(max=T - 1)].float().unflatten(2, (H, -1))  # [seqs, N, heads, group, dim]
    k, v = _gathered(st)
    p = torch.einsum("bnhgd,bhld->bhgnl", qs, k).mul_(D ** -0.5)
    pos = (lens - n)[:, None] + row
    j = torch.arange(k.shape[2], device="cuda")
    seen = j <= pos[..., None]
    if c["window"]:
        seen = seen & ((j > pos[..., None] - c["window"]) | (j < c["sinks"]))
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    o = torch.einsum("bhgnl,bhld->bnhgd", p, v) / p.sum(-1).permute(0, 3, 1, 2)[..., None]
    token = torch.arange(T, device="cuda")
    seq = torch.searchsorted(cu[1:], token, right=True)
    return o.flatten(2, 3)[seq, token - cu[seq]].to(q.dtype)


_RUN = {"norm": _norm, "rope": _rope, "write": _write, "read": _read, "attend": _attend}


# ------------------------------------------------------------------ what a pass cannot do without
def _seen(case):
    """(pairs of a new token and a token that it sees, cached tokens that some new token sees) summed over the batch."""
    w, sinks, pairs, touched = case["window"], case["sinks"], 0, 0
    for n, p in zip(*_lengths(case)):
        for i in range(n):
            pos = p + i
            lo = max(0, pos - w + 1) if w else 0
            pairs += pos + 1 - lo + min(sinks, lo)
        lo = max(0, p - w + 1) if w else 0
        touched += p + n - lo + min(sinks, lo)
    return pairs, touched


def work(case):
    op = case["op"]
    if op == "norm":
        n = case["tokens"] * case["hidden"]
        return {"bytes": n * (2 + 1 + 4 / 128 + (4 if case["residual"] else 0)) + 2 * case["hidden"], "flops": 8 * n}
    H, D = case["kv_heads"], case["dim"]
    if op == "rope":
        n = case["tokens"] * (case["heads"] + H) * D
        return {"bytes": 4 * n + 8 * case["tokens"], "flops": 3 * n * case["rotary"] / D}
    new, past = _lengths(case)
    if op == "read":
        # every row of the padded answer is written
        return {"bytes": sum(past) * 2 * H * D + 4 * case["seqs"] * max(past) * H * D, "flops": 2 * sum(past) * H * D}
    T = sum(new)
    if op == "write":
        q = 4 * T * case["heads"] * D if case["rope"] else 0
        return {"bytes": T * H * D * 2 * (2 + 1) + q, "flops": T * D * (4 * H + (3 * (case["heads"] + H) if case["rope"] else 0))}
    pairs, touched = _seen(case)
    return {"bytes": 2 * touched * H * (D + 4 / PAGE) + 4 * T * case["heads"] * D, "flops": 4 * pairs * case["heads"] * D}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return _EXACT[case["op"]](st)


def _exact_norm(st):
    x, w = st["x"].double(), st["weight"].double()
    h = None
    if st["residual"] is not None:
        h = x + st["residual"].double()
        x = h.to(st["x"].dtype).double()  # the sum is kept in the stream's type, and that is what is normed
    y = w * x / torch.sqrt(torch.square(x).sum(1, keepdim=True) / x.shape[1] + 1e-5)
    blocks = y.reshape(x.shape[0], -1, 128)
    s = blocks.abs().max(2).values / 448
    s[s == 0] = 1
    q = (blocks / s[:, :, None]).reshape(x.shape)
    return (q, s) if h is None else (q, s, h)


def _exact_turn(x, positions, inv_freq, interleaved, magnitude):
    """The rotation as a product of complex numbers."""
    R = 2 * inv_freq.shape[0]
    x = x.double()
    first, second = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., : R // 2], x[..., R // 2 : R])
    phase = positions.double()[:, None, None] * inv_freq
    z = torch.complex(first, second) * torch.polar(torch.full_like(phase, magnitude), phase)
    out = x.clone()
    if interleaved:
        out[..., 0:R:2], out[..., 1:R:2] = z.real, z.imag
    else:
        out[..., : R // 2], out[..., R // 2 : R] = z.real, z.imag
    return out


def _exact_rope(st):
    c = st["case"]
    return tuple(_exact_turn(st[n], st["positions"], st["inv_freq"], c["interleaved"], c["magnitude"]) for n in ("q", "k"))


def _exact_write(st):
    cu, lens, table = st["cu_seqlens"].tolist(), st["seq_lens"].tolist(), st["block_table"].tolist()
    positions = torch.cat([torch.arange(t - (hi - lo), t) for t, lo, hi in zip(lens, cu[:-1], cu[1:])]).cuda()
    out, source = {}, {"k": st["k"].double(), "v": st["v"].double()}
    if "inv_freq" in st:
        out["q"] = _exact_turn(st["q"], positions, st["inv_freq"], False, 1.0)
        source["k"] = _exact_turn(st["k"], positions, st["inv_freq"], False, 1.0)
    for name, x in source.items():
        cache = st[name + "_cache"].float().double()
        cache = cache.transpose(-1, -2) if name == "v" else cache  # [pages, heads, PAGE, dim]
        scale = st[name + "_scale"].double()
        rounded = x.to(st["k"].dtype).double()  # what the 16-bit key says is the block's largest value
        for b, total in enumerate(lens):
            begin = total - (cu[b + 1] - cu[b])
            for page in range(begin // PAGE, -(-total // PAGE)):
                lo, hi, at = max(begin, page * PAGE), min(total, (page + 1) * PAGE), table[b][page]
                rows = slice(cu[b] + lo - begin, cu[b] + hi - begin)
                lo, hi = lo - page * PAGE, hi - page * PAGE
                amax = rounded[rows].abs().amax((0, 2))
                s = torch.exp2(torch.ceil(torch.log2(amax / 448)).clamp(LO, HI))
                if lo > 0:
                    s = torch.maximum(s, scale[at])
                    cache[at, :, :lo] *= (scale[at] / s)[:, None, None]
                cache[at, :, lo:hi] = x[rows].transpose(0, 1) / s[:, None, None]
                scale[at] = s
        out[name], out[name + "_scale"] = cache.transpose(-1, -2).contiguous() if name == "v" else cache, scale
    return out


def _exact_values(st, b, length):
    """k, v [heads, length, dim] of sequence b in 64 bits."""
    at = st["block_table"][b, : -(-length // PAGE)].long()
    k = st["k_cache"].view(torch.uint8)[at].view(torch.float8_e4m3fn).double() * st["k_scale"][at].double()[:, :, None, None]
    v = st["v_cache"].view(torch.uint8)[at].view(torch.float8_e4m3fn).double() * st["v_scale"][at].double()[:, :, None, None]
    H, D = k.shape[1], k.shape[3]
    k = k.permute(1, 0, 2, 3).reshape(H, -1, D)[:, :length]
    return k, v.permute(1, 0, 3, 2).reshape(H, -1, D)[:, :length]


def _exact_read(st):
    c = st["case"]
    out = [torch.zeros((c["seqs"], st["max_len"], c["kv_heads"], c["dim"]), dtype=torch.float64, device="cuda") for _ in "kv"]
    for b, length in enumerate(st["seq_lens"].tolist()):
        for o, x in zip(out, _exact_values(st, b, length)):
            o[b, :length] = x.transpose(0, 1)
    return tuple(out)


def _exact_attend(st):
    c, q = st["case"], st["q"].double()
    cu, lens = st["cu_seqlens"].tolist(), st["seq_lens"].tolist()
    out = torch.empty_like(q)
    for b, length in enumerate(lens):
        k, v = _exact_values(st, b, length)
        rows = q[cu[b] : cu[b + 1]].reshape(cu[b + 1] - cu[b], c["kv_heads"], -1, c["dim"])
        pos = torch.arange(length - rows.shape[0], length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None]
        hidden = j > pos
        if c["window"]:
            hidden |= (j <= pos - c["window"]) & (j >= c["sinks"])
        for h in range(c["kv_heads"]):
            score = rows[:, h].transpose(0, 1) @ k[h].T / math.sqrt(c["dim"])  # [group, rows, length]
            score[:, hidden] = -math.inf
            o = torch.softmax(score, -1) @ v[h]
            out[cu[b] : cu[b + 1]].view(rows.shape)[:, h] = o.transpose(0, 1)
    return out


_EXACT = {"norm": _exact_norm, "rope": _exact_rope, "write": _exact_write, "read": _exact_read, "attend": _exact_attend}
