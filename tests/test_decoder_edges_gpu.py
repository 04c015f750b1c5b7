"""Calls of the decoder operators at the edges of what their documentation allows."""

import math

import pytest
import torch

from oracle import decoder_ref as D

pytestmark = pytest.mark.gpu

import tilegym_b200 as tg  # noqa: E402

F8 = torch.float8_e4m3fn
BF, HF = torch.bfloat16, torch.float16


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def make_cache(pages, heads, dim, seed):
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(pages, heads, 128, dim, generator=g), torch.randn(pages, heads, dim, 128, generator=g)
    return [D.to_e4m3(k * 64), D.to_e4m3(v * 64), torch.full((pages, heads), 2.0**-6), torch.full((pages, heads), 2.0**-6)]


def on(dev, cache):
    return tg.FP8KVCache(*(c.to(dev) for c in cache))


# ------------------------------------------------------------------ paged_attention
@pytest.mark.parametrize("exponent", [-20, 0, 7, 10, 25, 60])
@pytest.mark.parametrize("n,length,pages", [(6, 4, 1), (100, 60, 1), (300, 200, 2), (100, 1200, 10)])
@pytest.mark.parametrize("dim,dtype", [(64, BF), (128, HF)])
def test_rows_that_see_nothing_are_zero_whatever_the_scales(dev, exponent, n, length, pages, dim, dtype):
    """A length below the new tokens, or pages that are not there in front of one that later rows see, of values of any size:
    zeros, and not what a sum that is nearly zero makes of them.  The rows beside them have their answer."""
    cache = make_cache(pages, 1, dim, n + dim)
    cache[3].fill_(2.0**exponent)
    table = torch.arange(pages, dtype=torch.int32)[None]
    if pages == 10:
        table[0, :9] = -1
    empty = n - length if pages < 10 else 9 * 128 - (length - n)
    q = torch.randn(n, 2, dim, generator=torch.Generator().manual_seed(n)).to(dtype)
    got = tg.paged_attention(q.to(dev), on(dev, cache), table.to(dev), i32([length]).to(dev), i32([0, n]).to(dev), max_q_len=n).cpu()
    assert bool((got[:empty] == 0).all())
    if exponent < 7 or dtype == BF:  # f16 ends at 2^16
        assert bool(got[empty:].isfinite().all()) and bool((got[empty:] != 0).any(-1).all())
