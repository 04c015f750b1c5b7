"""paged_attention where one token holds most of a row's weight and a long cache shares the rest: the weights of the many
are far below the largest one and still make the answer.

Tolerance: half a step of the output, and of sum p |v| the probabilities' own rounding and 32-bit noise, whatever the length
of the cache.
A probability is rounded to f16, half a step 2^-11, and in the kernel for few rows of bf16 to nine bits, 2^-9.  Below f16's
normal range that is 2^-25, and 2^-23 for the nine bits, where the row's largest is at least 2^8 (many rows) or 2^9 (few).
The many have 2^-21.3 of the largest each, on the mean, in the longest case here: 2^-13.3 and 2^-12.3, so that what ends is at
most 2^-11.7 (f16) and 2^-10.7 + 2^-12.7 (nine bits) of their sum.  Together: f16 2^-11 + 2^-11.7, bf16
2^-9 + 2^-11 + 2^-10.7 + 2^-12.7 < 2^-8.
A logit is a sum of 128 products in 32 bits, off by at most 128 * 2^-24 of the sum of their magnitudes (`size`), which
moves a probability by as much, relative; numerator and denominator: 2^-16 * size.  exp, sums and rescaling: 2^-14."""

import math

import pytest
import torch

from oracle import decoder_ref as D

pytestmark = pytest.mark.gpu

import tilegym_b200 as tg  # noqa: E402
from test_decoder_gpu import cumulative, gen, make_kv, on  # noqa: E402

F8 = torch.float8_e4m3fn
BF, HF = torch.bfloat16, torch.float16
PROBABILITY = {BF: 2.0**-8, HF: 2.0**-11 + 2.0**-11.7}


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def dominated(length, group, dim, n, share, spread, dtype):
    """(q [n, group, dim], cache on the CPU, table): the first token of a sequence takes `share` of each row and its value is
    near zero; the others' scores spread by `spread` and their values by 0.25 around 0.5."""
    g = torch.Generator().manual_seed(length + dim + group)
    pages = -(-length // 128)
    base = torch.randn(dim, generator=g)
    base = base * (math.sqrt(dim) / base.norm())
    k = torch.randn(pages, 1, 128, dim, generator=g) * spread
    v = torch.randn(pages, 1, dim, 128, generator=g) * 0.25 + 0.5
    table = torch.randperm(pages, generator=g).to(torch.int32)[None]
    # exp(top) = share / (1 - share) * (length - 1) * mean exp(score) of the others
    top = math.log(share / (1 - share) * (length - 1)) + spread * spread / 2
    first = int(table[0, 0])
    k[first, 0, 0] = base * (top / math.sqrt(dim))
    v[first, 0, :, 0] = torch.randn(dim, generator=g) * 2.0**-9
    cache = [D.to_e4m3(k * 2.0**6), D.to_e4m3(v * 2.0**7), torch.full((pages, 1), 2.0**-6), torch.full((pages, 1), 2.0**-7)]
    q = base + 0.02 * torch.randn(n, group, dim, generator=g)
    return q.to(dtype), cache, table


def check(dev, q, cache, table, length, n):
    got = tg.paged_attention(q.to(dev), tg.FP8KVCache(*(c.to(dev) for c in cache)), table.to(dev), i32([length]).to(dev), i32([0, n]).to(dev), max_q_len=n)
    compare(got.cpu()[None], q, cache, table, length)


def compare(got, q, cache, table, length):
    """got [.., tokens, heads, dim]"""
    o, mag, size, _ = D.ref_attention(q, cache, table, i32([length]), i32([0, q.shape[0]]))
    tiny = 2.0**-25 if q.dtype == HF else 0.0
    bound = torch.finfo(q.dtype).eps / 2 * o.abs() + (PROBABILITY[q.dtype] + 2.0**-16 * size + 2.0**-14) * mag + tiny
    off = (got.double() - o).abs()
    assert bool((off <= bound).all()), f"{float((off / o.abs()).max()):.2g} of the output, {float((off / bound).max()):.2g} of the bound"


# one sequence whose pages many blocks share; new tokens: rows of the kernel for few rows (4, 32) and for many (36)
@pytest.mark.parametrize("n", [1, 8, 9])
@pytest.mark.parametrize("length,share", [(4096, 0.95), (16000, 0.8), (32000, 0.9), (131072, 0.95)])
@pytest.mark.parametrize("dim,dtype", [(64, BF), (128, BF), (64, HF), (128, HF)])
def test_the_many_count_beside_one(dev, n, length, share, dim, dtype):
    q, cache, table = dominated(length, 4, dim, n, share, 0.5, dtype)
    check(dev, q, cache, table, length, n)


# every score of the many alike: roundings that do not average out (2^-21.3 of the whole each at the longest)
@pytest.mark.parametrize("n", [1, 8, 9])
@pytest.mark.parametrize("length,share", [(16000, 0.9), (131072, 0.95)])
@pytest.mark.parametrize("dim,dtype", [(128, BF), (64, HF)])
def test_the_many_count_where_they_are_alike(dev, n, length, share, dim, dtype):
    q, cache, table = dominated(length, 4, dim, n, share, 0.0, dtype)
    check(dev, q, cache, table, length, n)


# a batch of sequences that share their pages, more of them than blocks: a block goes through whole ones by itself
@pytest.mark.parametrize("n,group,dtype", [(1, 4, BF), (4, 8, BF), (1, 8, HF), (4, 8, HF), (20, 2, BF), (20, 2, HF)])
@pytest.mark.parametrize("length,share,dim", [(4096, 0.95, 64), (16000, 0.9, 128), (32000, 0.8, 64), (131072, 0.95, 128)])
def test_the_many_count_in_a_large_batch(dev, length, share, dim, n, group, dtype):
    copies = 320
    q, cache, table = dominated(length, group, dim, n, share, 0.5, dtype)
    cu = i32([b * n for b in range(copies + 1)])
    got = tg.paged_attention(q.repeat(copies, 1, 1).to(dev), tg.FP8KVCache(*(c.to(dev) for c in cache)), table.repeat(copies, 1).to(dev),
                             i32([length] * copies).to(dev), cu.to(dev), max_q_len=n)
    compare(got.cpu().unflatten(0, (copies, n)), q, cache, table, length)


@pytest.mark.parametrize("new,past,window,sinks", [([1] * 5, [0, 130, 900, 3000, 5000], 0, 0), ([4, 1, 3], [0, 2500, 127], 0, 0), ([4, 2, 4], [3000, 700, 5], 600, 4),
                                                   ([60, 1, 130], [3000, 200, 0], 0, 0), ([300, 7], [1000, 2000], 700, 130)])
@pytest.mark.parametrize("heads,group,dim,dtype", [(2, 4, 128, BF), (1, 8, 64, HF), (2, 1, 64, BF), (1, 5, 128, HF)])
def test_ordinary_batches_keep_the_same_bound(dev, new, past, window, sinks, heads, group, dim, dtype):
    """Pages of different scales, foreign bytes behind the ends.  v_scale rides in the exponent, so p * v_scale is what ends, at
    2^-31 of a row's largest, and it meets the values' bytes."""
    g = gen(sum(new) + sum(past) + dim)
    lens = [a + b for a, b in zip(new, past)]
    table, ref = make_kv(lens, heads, dim, g)
    q = torch.randn(sum(new), heads * group, dim, generator=g).to(dtype)
    cu = cumulative(new)
    got = tg.paged_attention(q.to(dev), on(dev, ref), table.to(dev), i32(lens).to(dev), cu.to(dev), max_q_len=max(new), window=window, sinks=sinks)
    o, mag, size, coarse = D.ref_attention(q, ref, table, i32(lens), cu, window=window, sinks=sinks)
    tiny = 2.0**-25 if dtype == HF else 0.0
    bound = torch.finfo(dtype).eps / 2 * o.abs() + (PROBABILITY[dtype] + 2.0**-16 * size + 2.0**-14) * mag + 2.0**-31 * coarse + tiny
    assert bool(((got.cpu().double() - o).abs() <= bound).all())
