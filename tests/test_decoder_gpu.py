"""The decoder operators around the GEMMs (rms_norm_quant, apply_rope, the paged 8-bit cache, paged_attention) against
their definitions in 64 bits.

Tolerances.  A rounding is off by at most half a step, eps / 2 relative (e4m3: 2^-4, or 2^-10 absolute below its normal
range).  32-bit work in front of it adds: the norm's sum of up to 65536 squares in at most 64 + 10 sequential additions
2^-24 * 74 < 5e-6 (halved by the root) and four roundings; a rotation 2^-21 + 2^-23 of |a| + |b| (hardware sine and cosine
of an exactly reduced angle, two products, a sum); attention what its comment says."""

import math

import pytest
import torch

from oracle import decoder_ref as D

pytestmark = pytest.mark.gpu

import tilegym_b200 as tg  # noqa: E402
from tilegym_b200 import _lib  # noqa: E402

F8 = torch.float8_e4m3fn
BF, HF = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(t):
    return torch.finfo(t).eps / 2


# ------------------------------------------------------------------ rms_norm_quant
def check_norm(x, w, eps, residual, offset, out):
    y8, s = out[0].cpu(), out[1].cpu()
    y, h = D.ref_rms_norm(x, w, eps, residual, offset)
    if residual is not None:
        assert torch.equal(out[2].cpu(), h)
    assert y8.dtype == F8 and y8.shape == x.shape and s.shape == x.shape[:-1] + (x.shape[-1] // 128,)
    blocks = y.unflatten(-1, (-1, 128))
    ref_s = blocks.abs().amax(-1) / 448
    ref_s[ref_s == 0] = 1
    assert bool(((s.double() - ref_s).abs() <= 1e-5 * ref_s).all())
    q = (blocks / ref_s[..., None]).flatten(-2)
    bound = torch.clamp(q.abs() * 2.0**-4, min=2.0**-10) + 2e-5 * q.abs()
    assert bool(((y8.double() - q).abs() <= bound).all())


@pytest.mark.parametrize("T,H", [(1, 128), (1, 4096), (3, 384), (297, 640), (1000, 1152), (300, 8192), (2, 65536), (700, 16384)])
@pytest.mark.parametrize("dtype,res,wdtype,offset", [(BF, True, BF, 0.0), (HF, False, HF, 0.0), (BF, False, torch.float32, 1.0), (HF, True, torch.float32, 0.0)])
def test_norm(dev, T, H, dtype, res, wdtype, offset):
    g = gen(T * 7 + H)
    x = torch.randn(T, H, generator=g).to(dtype)
    x[:, ::97] *= 20
    r = (2 * torch.randn(T, H, generator=g)).to(dtype) if res else None
    w = (torch.randn(H, generator=g) * 0.2 + (0 if offset else 1)).to(wdtype)
    out = tg.rms_norm_quant(x.to(dev), w.to(dev), 1e-5, residual=None if r is None else r.to(dev), weight_offset=offset)
    check_norm(x, w, 1e-5, r, offset, out)


def test_norm_zero_rows_shapes_strides_and_inplace(dev):
    g = gen(1)
    big = torch.randn(2, 5, 1024, generator=g).to(BF)
    x, w = big[..., 256:768], torch.randn(512, generator=g).to(BF)
    x[0, 1] = 0
    w[:128] = 0
    big = big.to(dev)
    res = torch.randn(2, 5, 512, generator=g).to(BF)
    rd = res.to(dev)
    out = tg.rms_norm_quant(big[..., 256:768], w.to(dev), 1e-6, residual=rd, inplace=True)
    assert out[2] is rd
    check_norm(x, w, 1e-6, res, 0.0, out)
    zero = torch.zeros(4, 256, dtype=BF, device=dev)
    y, s = tg.rms_norm_quant(zero, torch.ones(256, dtype=BF, device=dev))
    assert bool((y.float() == 0).all()) and bool((s == 1).all())
    y, s = tg.rms_norm_quant(torch.zeros(0, 256, dtype=BF, device=dev), torch.ones(256, dtype=BF, device=dev))
    assert y.shape == (0, 256) and s.shape == (0, 2)
    # an odd pitch and start: the rows are copied into place
    odd = torch.randn(6, 261, generator=g).to(BF)
    out = tg.rms_norm_quant(odd.to(dev)[:, 3:259], torch.ones(256, dtype=BF, device=dev), 1e-6)
    check_norm(odd[:, 3:259], torch.ones(256, dtype=BF), 1e-6, None, 0.0, out)


def test_norm_feeds_the_block_scaled_gemm(dev):
    g = gen(2)
    x, w = torch.randn(40, 512, generator=g).to(BF), (torch.randn(512, generator=g) * 0.1 + 1).to(BF)
    wq, ws = tg.weight_quant_block((torch.randn(256, 512, generator=g) * 0.05).to(BF).to(dev))
    y, s = tg.rms_norm_quant(x.to(dev), w.to(dev))
    got = tg.fp8_block_scaled_mm(y, wq, s, ws).cpu().double()
    a = (y.cpu().double().unflatten(-1, (-1, 128)) * s.cpu().double()[..., None]).flatten(-2)
    b = tg.weight_dequant(wq, ws, 128, torch.float32).cpu().double()
    ref = a @ b.T
    assert float((got - ref).abs().max()) <= float(ref.abs().max()) * 2 * half_step(BF)


# ------------------------------------------------------------------ apply_rope
def check_rope(x, positions, f, inter, m, got, dtype):
    ref = D.ref_rope(x, positions, f, inter, m)
    R = 2 * f.numel()
    other = x.double().clone()
    if inter:
        other[..., 0:R:2], other[..., 1:R:2] = x[..., 1:R:2].double(), x[..., 0:R:2].double()
    else:
        other[..., : R // 2], other[..., R // 2 : R] = x[..., R // 2 : R].double(), x[..., : R // 2].double()
    noise = (x.double().abs() + other.abs()) * m * 2.0**-20
    noise[..., R:] = 0
    tiny = 2.0**-25 if dtype == HF else 0.0
    assert bool(((got.cpu().double() - ref).abs() <= half_step(dtype) * ref.abs() + noise + tiny).all())
    assert torch.equal(got.cpu()[..., R:], x[..., R:])


@pytest.mark.parametrize("T,Hq,Hk,dim,R", [(1, 4, 1, 64, 64), (7, 8, 2, 128, 128), (130, 3, 3, 128, 32), (33, 5, 1, 80, 16), (3, 2, 1, 512, 512), (5, 1, 1, 16, 16)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_rope(dev, T, Hq, Hk, dim, R, inter, dtype):
    g = gen(T + dim + R)
    q, k = torch.randn(T, Hq, dim, generator=g).to(dtype), torch.randn(T, Hk, dim, generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (T,), generator=g)
    f, _ = tg.rope_frequencies(dim, 500000.0, R, device="cpu")
    qo, ko = tg.apply_rope(q.to(dev), k.to(dev), pos.to(dev), f.to(dev), inter, 1.25)
    check_rope(q, pos, f, inter, 1.25, qo, dtype)
    check_rope(k, pos, f, inter, 1.25, ko, dtype)


def test_rope_far_negative_and_int32_positions(dev):
    g = gen(4)
    q = torch.randn(6, 2, 64, generator=g).to(HF)
    f, _ = tg.rope_frequencies(64, device="cpu")
    pos = torch.tensor([0, 1, 2**31 - 1, -5, 2**24 + 1, 10**7])
    # 64-bit reference: products below 2^31 * 1 rad are good to 2^-22 rad in double
    qo, ko = tg.apply_rope(q.to(dev), None, pos.to(dev), f.to(dev))
    assert ko is None
    check_rope(q, pos, f, False, 1.0, qo, HF)
    q32, _ = tg.apply_rope(q.to(dev), None, pos.int().to(dev), f.to(dev))
    assert torch.equal(q32, qo)


def test_rope_inplace_and_strided(dev):
    g = gen(5)
    qkv = torch.randn(9, 6, 128, generator=g).to(BF)
    pos = torch.arange(9) * 1000
    f, _ = tg.rope_frequencies(128, 10000.0, 64, device="cpu")
    d = qkv.to(dev)
    qo, ko = tg.apply_rope(d[:, :4], d[:, 4:5], pos.to(dev), f.to(dev), inplace=True)
    assert qo.data_ptr() == d.data_ptr()
    check_rope(qkv[:, :4], pos, f, False, 1.0, d[:, :4], BF)
    check_rope(qkv[:, 4:5], pos, f, False, 1.0, d[:, 4:5], BF)
    assert torch.equal(d[:, 5].cpu(), qkv[:, 5])
    # heads in front of tokens, and an odd start: pitches of their own, or a copy
    t = qkv.transpose(0, 1).contiguous().to(dev).transpose(0, 1)
    qo, _ = tg.apply_rope(t, None, pos.to(dev), f.to(dev))
    check_rope(qkv, pos, f, False, 1.0, qo, BF)
    odd = torch.randn(4, 2, 67, generator=g).to(BF)
    qo, _ = tg.apply_rope(odd.to(dev)[..., 3:], None, pos[:4].to(dev), f[:16].to(dev))
    check_rope(odd[..., 3:], pos[:4], f[:16], False, 1.0, qo, BF)
    with pytest.raises(AssertionError):
        tg.apply_rope(odd.to(dev)[..., 3:], None, pos[:4].to(dev), f[:16].to(dev), inplace=True)


# ------------------------------------------------------------------ cache
def make_cache(pages, heads, dim, g, nan=False):
    """A cache full of other sequences' bytes (NaN among them), on the CPU."""
    k = torch.randint(0, 256, (pages, heads, 128, dim), generator=g, dtype=torch.uint8)
    v = torch.randint(0, 256, (pages, heads, dim, 128), generator=g, dtype=torch.uint8)
    if not nan:
        k[(k & 127) == 127] = 0
        v[(v & 127) == 127] = 0
    s = [2.0 ** torch.randint(-12, -5, (pages, heads), generator=g).float() for _ in "kv"]
    return [k.view(F8), v.view(F8), *s]


def tables(lens, g, spare=2, pad=0):
    """(block_table, number of pages): pages in random order, the rest of a row -1."""
    need = [-(-n // 128) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    t = torch.full((len(lens), max(need + [1]) + pad), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = torch.tensor(order[at : at + n], dtype=torch.int32)
        at += n
    return t, pages


def on(dev, cache):
    return tg.FP8KVCache(*(c.to(dev) for c in cache))


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def cumulative(new):
    return i32([sum(new[:b]) for b in range(len(new) + 1)])


def same_cache(got, ref):
    for a, b, name in zip(got, ref, ("k", "v", "k_scale", "v_scale")):
        if a.dtype == F8:  # bytes, but for the sign of a NaN, which says nothing
            a, b = ((x.view(torch.uint8).to(torch.int16).cpu() for x in (a, b)))
            a, b = torch.where((a & 127) == 127, 127, a), torch.where((b & 127) == 127, 127, b)
        wrong = int((a.cpu() != b).sum())
        assert wrong == 0, f"{wrong} values of {name} differ"


LENS = [([1], [0]), ([1, 1, 1], [0, 127, 128]), ([5, 0, 200], [3, 40, 100]), ([300, 1, 128, 129], [0, 500, 128, 127]), ([2] * 40, list(range(100, 140)))]


@pytest.mark.parametrize("new,past", LENS)
@pytest.mark.parametrize("heads,dim,dtype", [(1, 64, BF), (3, 128, BF), (2, 128, HF)])
def test_write_bytes(dev, new, past, heads, dim, dtype):
    g = gen(sum(new) + dim)
    lens = [n + p for n, p in zip(new, past)]
    table, pages = tables(lens, g, pad=1)
    ref = make_cache(pages, heads, dim, g, nan=True)
    cache = on(dev, ref)
    T = sum(new)
    k, v = ((torch.randn(T, heads, dim, generator=g) * 4 ** torch.randn(T, heads, 1, generator=g)).to(dtype) for _ in "kv")
    cu = cumulative(new)
    assert tg.kv_cache_write(cache, k.to(dev), v.to(dev), table.to(dev), i32(lens).to(dev), cu.to(dev)) is None
    D.ref_kv_write(ref, k, v, table, i32(lens), cu)
    same_cache(cache, ref)


def test_write_token_by_token_grows_scales(dev):
    g = gen(11)
    table, pages = tables([140], g)
    ref = make_cache(pages, 2, 64, g)
    cache = on(dev, ref)
    for t in range(140):
        x = torch.randn(1, 2, 64, generator=g).to(BF) * 2.0 ** (t // 20)
        k, v = x.to(BF), (x * 0.37).to(BF)
        tg.kv_cache_write(cache, k.to(dev), v.to(dev), table.to(dev), i32([t + 1]).to(dev))
        D.ref_kv_write(ref, k, v, table, i32([t + 1]), i32([0, 1]))
    same_cache(cache, ref)


def test_write_special_values(dev):
    g = gen(12)
    table, pages = tables([6, 3], g)
    ref = make_cache(pages, 1, 64, g)
    cache = on(dev, ref)
    k = torch.randn(9, 1, 64, generator=g).to(BF)
    k[0] = 0
    k[1, 0, :3] = torch.tensor([math.nan, math.inf, -math.inf])
    k[2] *= 1e-30
    v = k.clone()
    k[6:] = 0  # a page of zeros
    v[6:] = 3e38  # beyond the largest scale
    tg.kv_cache_write(cache, k.to(dev), v.to(dev), table.to(dev), i32([6, 3]).to(dev), i32([0, 6, 9]).to(dev))
    D.ref_kv_write(ref, k, v, table, i32([6, 3]), i32([0, 6, 9]))
    same_cache(cache, ref)
    assert float(cache.k_scale[int(table[1, 0]), 0]) == 2.0**-60 and float(cache.v_scale[int(table[1, 0]), 0]) == 2.0**60


def test_write_leaves_alone_what_it_must(dev):
    """Padded sequences, rows behind the last sequence, pages outside the cache or the table, lengths below the new tokens."""
    g = gen(13)
    ref = make_cache(4, 2, 64, g)
    cache = on(dev, ref)
    table = i32([[0, 99], [-7, 1], [2, 3], [0, 0]])
    lens, new = i32([130, 140, 300, 0]), [30, 20, 60, 1]
    cu = cumulative(new)
    T = 120  # nine rows belong to nobody
    k, v = (torch.randn(T, 2, 64, generator=g).to(BF) for _ in "kv")
    tg.kv_cache_write(cache, k.to(dev), v.to(dev), table.to(dev), lens.to(dev), cu.to(dev))
    D.ref_kv_write(ref, k, v, table, lens, cu)
    same_cache(cache, ref)
    # three new tokens of a sequence that says it has two: the one in front has no position
    tg.kv_cache_write(cache, k[:3].to(dev), v[:3].to(dev), table[:1].to(dev), i32([2]).to(dev), i32([0, 3]).to(dev))
    D.ref_kv_write(ref, k[:3], v[:3], table[:1], i32([2]), i32([0, 3]))
    same_cache(cache, ref)
    # offsets that make no sense stay inside the batch: nothing to check but that the call returns
    tg.kv_cache_write(on(dev, ref), k.to(dev), v.to(dev), table.to(dev), lens.to(dev), i32([50, 10, 400, -3, 120]).to(dev))
    _lib.device_status(0)


@pytest.mark.parametrize("dim,R,inter,dtype", [(128, 128, False, BF), (128, 64, True, BF), (64, 64, False, HF), (64, 16, True, HF)])
def test_write_rotates_as_apply_rope_does(dev, dim, R, inter, dtype):
    g = gen(dim + R)
    new, past = [1, 150, 0, 20], [70000, 100, 5, 0]
    lens = [n + p for n, p in zip(new, past)]
    table, pages = tables(lens, g)
    ref = make_cache(pages, 2, dim, g)
    a, b = on(dev, ref), on(dev, ref)
    T = sum(new)
    qkv = torch.randn(T, 10, dim, generator=g).to(dtype).to(dev)
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
    f, _ = tg.rope_frequencies(dim, 10000.0, R, device=dev)
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)]).to(dev)
    args = table.to(dev), i32(lens).to(dev), cumulative(new).to(dev)
    q1, k1 = tg.apply_rope(q, k, pos, f, inter, 1.1)
    tg.kv_cache_write(a, k1, v, *args)
    q2 = tg.kv_cache_write(b, k, v, *args, inv_freq=f, q=q, interleaved=inter, magnitude=1.1)
    assert torch.equal(q1, q2)
    same_cache(a, [x.cpu() for x in b])


@pytest.mark.parametrize("heads,dim,dtype", [(1, 64, BF), (3, 128, BF), (2, 128, HF)])
def test_read(dev, heads, dim, dtype):
    g = gen(dim + heads)
    lens = [0, 1, 127, 128, 129, 400]
    table, pages = tables(lens, g)
    ref = make_cache(pages, heads, dim, g)
    table[5, 1] = 12345  # a page outside the cache reads as zeros
    k, v = tg.kv_cache_read(on(dev, ref), table.to(dev), i32(lens).to(dev), 390, dtype)
    assert k.shape == v.shape == (6, 390, heads, dim) and k.dtype == dtype
    for b, n in enumerate(lens):
        t = table[b].clone()
        t[t == 12345] = 0
        rk, rv = D.cache_values(ref, t, n)
        for got, r in ((k, rk), (v, rv)):
            want = torch.zeros(390, heads, dim, dtype=dtype)
            want[: min(n, 390)] = r.transpose(0, 1)[:390].to(dtype)
            if b == 5:
                want[128:256] = 0
            assert torch.equal(got[b].cpu(), want)
    k, v = tg.kv_cache_read(on(dev, ref), table.to(dev), i32(lens).to(dev), 0)
    assert k.numel() == 0


# ------------------------------------------------------------------ paged_attention
#: What the probabilities may be off by, relative, before they meet the values.  The kernel for few rows splits them into
#: e4m3 terms, each rounding half a step (2^-4) of what the one before left: two for bf16, three for f16.  The one for many
#: rows rounds them to f16, half a step 2^-11.
P_ERROR = {BF: 2.0**-8, HF: 2.0**-11}


def allowed(dtype, o, mag, size, coarse):
    """Half a step of o, and of sum p |v|: the probabilities' rounding, and 32-bit noise.  A logit is a sum of 128 products in
    32 bits, off by at most 128 * 2^-24 of the sum of their magnitudes (`size`), which moves a probability by as much,
    relative; numerator and denominator: 2^-16 * size.  exp, sums and the running maximum's rescaling: 2^-14.
    The terms end at half of e4m3's smallest step, 2^-10, where the row's largest p * v_scale is 2^7 or more: 2^-17 of that
    times the values' bytes (`coarse`).
    A probability under 2^-126 of the largest is 0 in 32 bits: 2^-126 * 448 * 2^12 (the largest scale here) * 1000 tokens."""
    tiny = 2.0**-25 if dtype == HF else 2.0**-95
    return half_step(dtype) * o.abs() + (P_ERROR[dtype] + 2.0**-16 * size + 2.0**-14) * mag + 2.0**-17 * coarse + tiny


def check_attention(dev, q, ref, table, lens, new, got=None, **kw):
    cu = cumulative(new)
    if got is None:
        got = tg.paged_attention(q.to(dev), on(dev, ref), table.to(dev), i32(lens).to(dev), cu.to(dev), max_q_len=max(new + [1]), **kw)
    o, mag, *rest = D.ref_attention(q, ref, table, i32(lens), cu, **{k: v for k, v in kw.items() if k in ("scale", "window", "sinks")})
    bound = allowed(q.dtype, o, mag, *rest)
    n = int(cu[-1])
    diff = (got.cpu().double() - o).abs()[:n]
    assert bool((diff <= bound[:n]).all()), float((diff / (mag[:n] + 1e-30)).max())
    return got


def make_kv(lens, heads, dim, g, **kw):
    """A cache whose live tokens have ordinary values and whose other bytes are anything, NaN among them."""
    table, pages = tables(lens, g, **kw)
    ref = make_cache(pages, heads, dim, g, nan=True)
    cu = cumulative(lens)
    T = sum(lens)
    k, v = ((torch.randn(T, heads, dim, generator=g) * 2 ** torch.randn(T, heads, 1, generator=g)).to(BF) for _ in "kv")
    D.ref_kv_write(ref, k, v, table, i32(lens), cu)
    return table, ref


@pytest.mark.parametrize("lens", [[1], [128], [129, 1, 0, 700], [5] * 30, [3000, 17, 1500]])
@pytest.mark.parametrize("heads,group,dim,dtype", [(1, 1, 64, BF), (2, 4, 128, BF), (2, 8, 64, HF), (1, 3, 128, HF), (1, 64, 64, BF)])
def test_attention_single_tokens(dev, lens, heads, group, dim, dtype):
    g = gen(sum(lens) + dim + group)
    table, ref = make_kv(lens, heads, dim, g)
    q = (torch.randn(len(lens), heads * group, dim, generator=g) * 1.5).to(dtype)
    cache = on(dev, ref)
    got = tg.paged_attention(q.to(dev), cache, table.to(dev), i32(lens).to(dev))
    check_attention(dev, q, ref, table, lens, [1] * len(lens), got=got)
    for b, n in enumerate(lens):
        if n == 0:
            assert bool((got[b] == 0).all())


@pytest.mark.parametrize("new,past", [([4, 1, 3, 2], [0, 500, 127, 300]), ([8] * 3, [120, 1000, 0]), ([50, 7], [100, 0]), ([200, 1, 130], [0, 900, 128]), ([300], [1100])])
@pytest.mark.parametrize("heads,group,dim,dtype", [(2, 4, 128, BF), (1, 8, 64, HF), (2, 1, 128, HF), (1, 6, 64, BF)])
def test_attention_several_tokens(dev, new, past, heads, group, dim, dtype):
    g = gen(sum(new) + sum(past) + dim)
    lens = [n + p for n, p in zip(new, past)]
    table, ref = make_kv(lens, heads, dim, g)
    q = torch.randn(sum(new), heads * group, dim, generator=g).to(dtype)
    check_attention(dev, q, ref, table, lens, new)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (100, 0), (128, 130), (500, 4), (129, 1), (5000, 7)])
@pytest.mark.parametrize("new,past", [([1, 1, 1], [0, 700, 1500]), ([5, 1], [300, 640]), ([260, 30], [0, 500])])
@pytest.mark.parametrize("dim,dtype", [(128, BF), (64, HF)])
def test_attention_window_and_sinks(dev, window, sinks, new, past, dim, dtype):
    g = gen(window + sinks + dim)
    lens = [n + p for n, p in zip(new, past)]
    table, ref = make_kv(lens, 2, dim, g)
    q = torch.randn(sum(new), 6, dim, generator=g).to(dtype)
    check_attention(dev, q, ref, table, lens, new, window=window, sinks=sinks)


def test_attention_scale_peaks_and_blocks_of_any_magnitude(dev):
    """Scores in the hundreds, pages whose scales differ by 2^40, values that are zero for whole pages."""
    g = gen(21)
    lens = [900, 400]
    table, ref = make_kv(lens, 1, 128, g)
    for i, e in enumerate([0, -30, 12, 4, -60, 2, 0]):
        ref[3][int(table[0, i]), 0] = 2.0**e
    ref[1].view(torch.uint8)[int(table[1, 1])] = 0
    q = (torch.randn(2, 4, 128, generator=g) * 6).to(BF)
    check_attention(dev, q, ref, table, lens, [1, 1])
    check_attention(dev, q, ref, table, lens, [1, 1], scale=1e-6)
    check_attention(dev, q * 0, ref, table, lens, [1, 1])


def test_attention_nan_stays_with_those_who_see_it(dev):
    g = gen(22)
    lens, new = [600, 400], [1, 140]
    table, ref = make_kv(lens, 1, 64, g)
    ref[0].view(torch.uint8)[int(table[0, 0]), 0, 5, 3] = 127  # key of token 5
    ref[1].view(torch.uint8)[int(table[1, 2]), 0, 7, 64] = 255  # element 7 of the value of token 320
    q = torch.randn(141, 4, 64, generator=g).to(BF)
    for kw in ({}, {"window": 300}):
        got = tg.paged_attention(q.to(dev), on(dev, ref), table.to(dev), i32(lens).to(dev), i32([0, 1, 141]).to(dev), max_q_len=140, **kw)
        bad = got.isnan().cpu()
        assert bool(bad[0].all()) == (not kw) and bool(bad[0].any()) == (not kw)
        small = tg.paged_attention(q[:5].to(dev), on(dev, ref), table[1:].to(dev), i32([323]).to(dev), i32([0, 5]).to(dev), max_q_len=5, **kw)
        assert bool(small[2:, :, 7].isnan().all()) and int(small.isnan().sum()) == 3 * 4  # positions 318 .. 322
        want = torch.zeros_like(bad[1:])
        want[60:, :, 7] = True  # positions 260 .. 399: rows from 320 on see it
        assert torch.equal(bad[1:], want)
        clean = [c.clone() for c in ref]
        clean[0].view(torch.uint8)[int(table[0, 0]), 0, 5, 3] = 0
        clean[1].view(torch.uint8)[int(table[1, 2]), 0, 7, 64] = 0
        o, *rest = D.ref_attention(q, clean, table, i32(lens), i32([0, 1, 141]), **kw)
        rows = slice(1, 61)  # those in front of it are as if it were not there
        assert bool(((got.cpu().double() - o).abs() <= allowed(BF, o, *rest))[rows].all())


@pytest.mark.parametrize("n", [1, 70])
def test_attention_nan_keys_at_every_place_of_a_page(dev, n):
    """One NaN in the key of one token: every row that sees the token has no answer, whichever path its exponential takes."""
    g = gen(25)
    table, ref = make_kv([256], 1, 64, g)
    q = torch.randn(n, 2, 64, generator=g).to(BF).to(dev)
    cache = on(dev, ref)
    for t in range(0, 128):
        k = cache.k.clone()
        k.view(torch.uint8)[int(table[0, 0]), 0, t, t % 64] = 127
        got = tg.paged_attention(q, cache._replace(k=k), table.to(dev), i32([256]).to(dev), i32([0, n]).to(dev), max_q_len=n)
        assert bool(got.isnan().all()), t


@pytest.mark.parametrize("heads,group,dim,dtype", [(1, 1, 64, BF), (2, 8, 128, BF), (3, 4, 128, HF), (1, 3, 64, HF)])
@pytest.mark.parametrize("new,past", [([150], [4000]), ([130, 1, 0, 90], [1500, 600, 0, 5]), ([300], [0]), ([129], [385])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (900, 5)])
def test_attention_chunks_on_a_long_cache(dev, heads, group, dim, dtype, new, past, window, sinks):
    """Few blocks for the device: several share the pages of their rows, and parts are joined."""
    g = gen(27)
    lens = [n + p for n, p in zip(new, past)]
    table, ref = make_kv(lens, heads, dim, g)
    q = torch.randn(sum(new), heads * group, dim, generator=g).to(dtype)
    got = check_attention(dev, q, ref, table, lens, new, window=window, sinks=sinks)
    # the same bits whenever it runs
    again = check_attention(dev, q, ref, table, lens, new, window=window, sinks=sinks)
    assert torch.equal(got, again)


def test_attention_parts_follow_the_lengths_of_a_replay(dev):
    """A captured chunk whose sequence grows and shrinks between replays, beside a second graph of the same call."""
    g = gen(29)
    n, lens = 100, [3000, 101, 1200, 100]
    table, ref = make_kv([3000], 2, 128, g)
    cache, t, cu = on(dev, ref), table.to(dev), i32([0, n]).to(dev)
    length = i32([3000]).to(dev)
    q = [torch.randn(n, 8, 128, generator=g).to(BF).to(dev) for _ in range(2)]
    graphs, out = [], []
    tg.paged_attention(q[0], cache, t, length, cu, max_q_len=n)
    torch.cuda.synchronize()
    for x in q:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            out.append(tg.paged_attention(x, cache, t, length, cu, max_q_len=n))
    side = torch.cuda.Stream()
    for now in lens:
        length.fill_(now)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for x, got in zip(q, out):
            check_attention(dev, x.cpu(), ref, table, [now], [n], got=got)
            assert torch.equal(got, tg.paged_attention(x, cache, t, length, cu, max_q_len=n))


def test_attention_nan_reaches_over_parts(dev):
    """A NaN in one part of the pages: of a key for the rows that see it, of a value for its element."""
    g = gen(28)
    n, length = 100, 2000
    table, ref = make_kv([length], 1, 64, g)
    q = torch.randn(n, 2, 64, generator=g).to(BF).to(dev)
    cache = on(dev, ref)

    def run(**change):
        return tg.paged_attention(q, cache._replace(**change), table.to(dev), i32([length]).to(dev), i32([0, n]).to(dev), max_q_len=n)

    good = run()
    for at in (0, 700, 1500, 1950):
        see = (torch.arange(length - n, length) >= at).to(dev)
        k, v = cache.k.clone(), cache.v.clone()
        k.view(torch.uint8)[int(table[0, at // 128]), 0, at % 128, 5] = 127
        v.view(torch.uint8)[int(table[0, at // 128]), 0, 9, at % 128] = 255
        bad = run(k=k)
        assert bool(bad[see].isnan().all()) and torch.equal(bad[~see], good[~see])
        bad = run(v=v)
        assert bool(bad[see][:, :, 9].isnan().all())
        bad[..., 9] = good[..., 9]
        assert torch.equal(bad, good)


@pytest.mark.parametrize("n", [6, 150])
def test_attention_factors_that_are_no_numbers(dev, n):
    """A row of q with a NaN, a page whose scale is one or infinite: only rows that see something of it lose their answer."""
    g = gen(26)
    table, ref = make_kv([200], 1, 64, g)
    q = torch.randn(n, 2, 64, generator=g).to(BF).to(dev)

    def run(q, k_scale=ref[2], length=200):
        cache = on(dev, [ref[0], ref[1], k_scale, ref[3]])
        return tg.paged_attention(q, cache, table.to(dev), i32([length]).to(dev), i32([0, n]).to(dev), max_q_len=n)

    good = run(q)
    row = n // 2
    for value in (math.nan, math.inf):
        bad_q = q.clone()
        bad_q[row, 1, 3] = value
        bad = run(bad_q)
        assert bool(bad[row, 1].isnan().all())
        bad[row, 1] = good[row, 1]
        assert torch.equal(bad, good)
        scale = ref[2].clone()
        scale[table[0, 1], 0] = value
        bad = run(q, scale)
        see = (torch.arange(200 - n, 200) >= 128).to(dev)  # positions that see the second page
        assert bool(bad[see].isnan().all()) and torch.equal(bad[~see], good[~see])
        # a length that leaves the row nothing to see
        assert bool((run(bad_q, length=n - row - 1)[: row + 1] == 0).all())


@pytest.mark.parametrize("heads,group,new,past", [(1, 64, [3, 1], [200, 0]), (3, 5, [40, 13], [128, 300]), (2, 33, [2, 2], [127, 5]), (1, 1, [513], [1])])
def test_attention_group_sizes(dev, heads, group, new, past):
    g = gen(group)
    lens = [n + p for n, p in zip(new, past)]
    table, ref = make_kv(lens, heads, 64, g)
    q = torch.randn(sum(new), heads * group, 64, generator=g).to(BF)
    check_attention(dev, q, ref, table, lens, new)


def test_attention_padding_bad_pages_strides_and_out(dev):
    g = gen(23)
    lens, new = [300, 0, 200], [2, 1, 3]
    table, ref = make_kv(lens, 2, 64, g, pad=3)
    big = torch.randn(9, 4, 4, 64, generator=g).to(BF)
    q = big[:, 1]  # strided tokens; rows 6 .. 8 belong to nobody
    out = torch.full((9, 4, 64), 7.0, dtype=BF, device=dev)
    cu = cumulative(new)
    got = tg.paged_attention(big.to(dev)[:, 1], on(dev, ref), table.to(dev), i32(lens).to(dev), cu.to(dev), max_q_len=3, out=out)
    assert got is out and bool((out[6:] == 7).all()) and bool((out[2] == 0).all())
    check_attention(dev, q[:6], ref, table, lens, new, got=got[:6])
    # tokens on a page outside the cache are not seen
    bad = table.clone()
    bad[0, 0] = 1 << 30
    got = tg.paged_attention(q.to(dev), on(dev, ref), bad.to(dev), i32(lens).to(dev), cu.to(dev), max_q_len=3)
    o, *rest = D.ref_attention(q[:2], ref, table[:1, 1:], i32([172]), i32([0, 2]))
    assert bool(((got[:2].cpu().double() - o).abs() <= allowed(BF, o, *rest)).all())
    # a length beyond the table: what the table has
    got = tg.paged_attention(q[:1].to(dev), on(dev, ref), table[2:, :2].to(dev), i32([5000]).to(dev), i32([0, 1]).to(dev), max_q_len=1)
    assert got.shape == (1, 4, 64)
    got = tg.paged_attention(q[:0].to(dev), on(dev, ref), table.to(dev), i32(lens).to(dev), i32([0, 0, 0, 0]).to(dev))
    assert got.numel() == 0
    _lib.device_status(0)


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [150, 1]])
def test_attention_is_deterministic_on_any_stream_and_in_graphs(dev, new):
    g = gen(24)
    lens = [2500, 700]
    table, ref = make_kv(lens, 2, 128, g)
    q = torch.randn(sum(new), 8, 128, generator=g).to(BF)
    cache, qd, td, ld, cu = on(dev, ref), q.to(dev), table.to(dev), i32(lens).to(dev), cumulative(new).to(dev)

    def call():
        return tg.paged_attention(qd, cache, td, ld, cu, max_q_len=max(new))

    want = call()
    check_attention(dev, q, ref, table, lens, new, got=want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            outs.append(call())
    graphs, results = [], []
    torch.cuda.synchronize()
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            results.append(call())
        graphs.append(gr)
    for _ in range(3):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for o in outs + results:
        assert torch.equal(o, want)
    # lengths that change between replays
    shorter = [1000, 300]
    ld.copy_(i32(shorter))
    graphs[0].replay()
    torch.cuda.synchronize()
    check_attention(dev, q, ref, table, shorter, new, got=results[0])


def test_caches_beyond_four_gigabytes(dev):
    """Offsets that pass 32 bits: the same tokens in the last pages of a 4.9 GB cache (each of keys and values) and in a small one."""
    pages, heads, dim = 37500, 8, 128
    big = tg.FP8KVCache(torch.empty(pages, heads, 128, dim, dtype=torch.uint8, device=dev).view(F8),
                        torch.empty(pages, heads, dim, 128, dtype=torch.uint8, device=dev).view(F8),
                        torch.empty(pages, heads, device=dev), torch.empty(pages, heads, device=dev))
    small = tg.FP8KVCache.empty(6, heads, dim, dev)
    assert big.k.numel() > 2**32
    t1 = i32([[0, 3, 1], [2, 4, 5]])
    t2 = torch.where(t1 % 2 == 0, t1, pages - 6 + t1).to(torch.int32)  # page 0, 2, 4 and the last ones
    lens, new = i32([300, 200]), [300, 200]
    g = gen(31)
    k, v = (torch.randn(500, heads, dim, generator=g).to(BF).to(dev) for _ in "kv")
    q = torch.randn(500, 16, dim, generator=g).to(BF).to(dev)
    got = []
    for cache, t in ((small, t1), (big, t2)):
        args = t.to(dev), lens.to(dev)
        tg.kv_cache_write(cache, k, v, *args, cumulative(new).to(dev))
        one = tg.paged_attention(q[:2], cache, *args)
        many = tg.paged_attention(q, cache, *args, cumulative(new).to(dev), max_q_len=300)
        got.append((one, many, *tg.kv_cache_read(cache, *args, 300)))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert torch.equal(big.k_scale[t2[0, 1]], small.k_scale[t1[0, 1]])


def test_the_extension_and_ctypes_make_the_same_calls(dev, monkeypatch):
    """The ordinary calls go through the C++ extension, the others and those without it through ctypes: same bits, same errors."""
    assert _lib.fast is not None, "tilegym_b200/_bind.so is missing: run `python -m tilegym_b200.build`"
    g = gen(41)
    x, w, r = (torch.randn(*s, generator=g).to(BF).to(dev) for s in ((6, 256), (256,), (6, 256)))
    table, ref = make_kv([300, 100], 2, 64, g)
    qkv = torch.randn(4, 8, 64, generator=g).to(BF).to(dev)
    f, _ = tg.rope_frequencies(64, device=dev)
    td, ld, cu = table.to(dev), i32([300, 100]).to(dev), i32([0, 3, 4]).to(dev)
    out = torch.empty(4, 4, 64, dtype=BF, device=dev)

    def calls():
        cache = on(dev, ref)
        q = tg.kv_cache_write(cache, qkv[:, 4:6], qkv[:, 6:], td, ld, cu, inv_freq=f, q=qkv[:, :4])
        res = [*tg.rms_norm_quant(x, w, 1e-5), *tg.rms_norm_quant(x, w, 1e-5, residual=r, weight_offset=0.5),
               *tg.apply_rope(qkv[:, :4], qkv[:, 4:6], torch.arange(4, device=dev), f, True, 1.1), tg.apply_rope(qkv[:, :4], None, torch.arange(4, device=dev), f)[0],
               q, *cache, tg.paged_attention(q, cache, td, ld, cu, max_q_len=3), tg.paged_attention(q, cache, td, ld, cu, window=50, sinks=2, scale=0.2)]
        assert tg.paged_attention(q, cache, td, ld, cu, max_q_len=3, out=out) is out
        assert tg.kv_cache_write(cache, qkv[:, 4:6], qkv[:, 6:], td, ld, cu) is None
        rr = r.clone()
        assert tg.rms_norm_quant(x, w, 1e-5, residual=rr, inplace=True)[2] is rr
        with pytest.raises(_lib.TileGymB200Error):
            tg.paged_attention(q, cache, td, ld, cu, sinks=2)
        with pytest.raises(_lib.TileGymB200Error):
            tg.paged_attention(q.float(), cache, td, ld, cu)
        with pytest.raises(_lib.TileGymB200Error):
            tg.kv_cache_write(cache, qkv[:, 4:6], qkv[:, 6:], td.long(), ld, cu)
        with pytest.raises(AssertionError):
            tg.paged_attention(q, cache, td, ld, cu, out=out[:3])
        with pytest.raises(RuntimeError, match="no backward"):
            tg.apply_rope(qkv.clone().requires_grad_(), None, torch.arange(4, device=dev), f)
        return [*res, out.clone(), rr]

    fast = calls()
    monkeypatch.setattr(_lib, "fast", None)
    for a, b in zip(fast, calls()):
        assert torch.equal(a.view(torch.uint8) if a.dtype == F8 else a, b.view(torch.uint8) if b.dtype == F8 else b)


# ------------------------------------------------------------------ refusals on the device
def test_refuses_gradients(dev):
    x = torch.randn(2, 128, dtype=BF, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        tg.rms_norm_quant(x, torch.ones(128, dtype=BF, device=dev))
    with torch.no_grad():
        tg.rms_norm_quant(x, torch.ones(128, dtype=BF, device=dev))
