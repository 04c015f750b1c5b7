"""Calls of the decoder operators at the edges of what their documentation allows."""

import threading
import time

import pytest
import torch
from torch.autograd import forward_ad

from oracle import decoder_ref as D

pytestmark = pytest.mark.gpu

import tilegym_b200 as tg  # noqa: E402
from tilegym_b200 import _lib  # noqa: E402

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


@pytest.mark.parametrize("new,past,heads,group", [([1], [3000], 2, 4), ([1] * 400, [200] * 400, 2, 4), ([4, 8], [2000, 100], 1, 4), ([100], [4000], 1, 4), ([300, 70], [0, 500], 4, 2)])
def test_out_may_be_the_queries(dev, new, past, heads, group):
    lens = [a + b for a, b in zip(new, past)]
    pages = [-(-n // 128) for n in lens]
    cache = on(dev, make_cache(max(pages), heads, 64, len(new)))
    table = torch.arange(max(pages), dtype=torch.int32).repeat(len(new), 1)  # read only: pages are shared
    big = torch.randn(sum(new), 3, heads * group, 64, generator=torch.Generator().manual_seed(7)).to(BF).to(dev)
    q = big[:, 1]
    args = cache, table.to(dev), i32(lens).to(dev), i32([sum(new[:b]) for b in range(len(new) + 1)]).to(dev)
    want = tg.paged_attention(q, *args, max_q_len=max(new))
    around = big[:, ::2].clone()
    assert tg.paged_attention(q, *args, max_q_len=max(new), out=q) is q
    assert torch.equal(q, want) and torch.equal(big[:, ::2], around)


# ------------------------------------------------------------------ kv_cache_write
@pytest.mark.parametrize("scale", [1.5 * 2.0**-5, 1.0000001 * 2.0**-4, 1.75, 3e-9, 1.9 * 2.0**-30, 2.0**127, 1.5 * 2.0**100])
@pytest.mark.parametrize("new", [1, 3, 60])
@pytest.mark.parametrize("dim,dtype", [(64, BF), (128, HF)])
def test_append_to_a_page_whose_scale_is_no_power_of_two(dev, scale, new, dim, dtype):
    """Scales are fp32, positive: a page that came from elsewhere may have any.  New tokens are right under the scale that the
    page keeps, earlier ones under the one that it moves to.

    A byte is off by half a step, 2^-4 of the value or 2^-10 of the scale, and the quotient in front of it by 2^-23."""
    g = torch.Generator().manual_seed(new + dim)
    past = 50
    cache = make_cache(2, 2, dim, new)
    cache[2].fill_(scale)
    cache[3].fill_(scale)
    before = [x[:, :past].clone() for x in D.cache_values(cache, i32([1]), past + new)]
    k, v = (torch.randn(new, 2, dim, generator=g).to(dtype) for _ in "kv")
    table, lens = i32([[1]]), i32([past + new])
    got = on(dev, cache)
    tg.kv_cache_write(got, k.to(dev), v.to(dev), table.to(dev), lens.to(dev), i32([0, new]).to(dev))
    back = [c.cpu() for c in got]
    for x, old, after, s in zip((k, v), before, D.cache_values(back, i32([1]), past + new), (back[2], back[3])):
        want = torch.cat((old, x.double().transpose(0, 1)), 1)
        s = s[1, :, None, None].double()
        bound = torch.clamp(want.abs() * 2.0**-4, min=2.0**-10 * s) * (1 + 2.0**-20)
        assert bool(((after - want).abs() <= bound).all()), float(((after - want).abs() / bound).max())
        # a scale that is large enough is kept, and with it the earlier bytes
        if scale > 2.0**-6:
            assert bool((s == torch.tensor(scale, dtype=torch.float32).double()).all()) and torch.equal(after[:, :past], old)


# ------------------------------------------------------------------ host side
@pytest.mark.parametrize("call", ["norm", "rope", "write", "attention"])
def test_a_full_launch_queue_holds_up_its_own_thread_only(dev, call):
    """A thread whose launches wait for room behind a long kernel (half a second or so) leaves the interpreter to the others."""
    x, w = torch.ones(1, 128, dtype=BF, device=dev), torch.ones(128, dtype=BF, device=dev)
    q, kv, at = torch.ones(1, 2, 64, dtype=BF, device=dev), torch.ones(1, 1, 64, dtype=BF, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    f, _ = tg.rope_frequencies(64, device=dev)
    cache, table, lens = tg.FP8KVCache.empty(1, 1, 64, dev), i32([[0]]).to(dev), i32([1]).to(dev)
    calls = {"norm": lambda: tg.rms_norm_quant(x, w), "rope": lambda: tg.apply_rope(q, kv, at, f),
             "write": lambda: tg.kv_cache_write(cache, kv, kv, table, lens), "attention": lambda: tg.paged_attention(q, cache, table, lens)}
    calls[call]()
    torch.cuda.synchronize()

    def launch():
        torch.cuda.set_device(dev)
        torch.cuda._sleep(1_000_000_000)
        for _ in range(3000):  # more than the queue holds
            calls[call]()

    thread = threading.Thread(target=launch)
    longest, last = 0.0, time.perf_counter()
    start = last
    thread.start()
    while thread.is_alive():
        time.sleep(0.001)
        now = time.perf_counter()
        longest, last = max(longest, now - last), now
    thread.join()
    torch.cuda.synchronize()
    assert last - start > 0.2, "the queue was never full"
    assert longest < 0.1, f"this thread stood still for {longest:.2f} s"


# ------------------------------------------------------------------ derivatives
@pytest.mark.parametrize("extension", [True, False])
def test_tangents_are_refused(dev, extension, monkeypatch):
    """A result that silently loses a derivative is refused, in forward mode too."""
    if not extension:
        monkeypatch.setattr(_lib, "fast", None)
    x, w = torch.ones(1, 128, dtype=BF, device=dev), torch.ones(128, dtype=BF, device=dev)
    q, kv, at = torch.ones(1, 2, 64, dtype=BF, device=dev), torch.ones(1, 1, 64, dtype=BF, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    f, _ = tg.rope_frequencies(64, device=dev)
    cache, table, lens = tg.FP8KVCache.empty(1, 1, 64, dev), i32([[0]]).to(dev), i32([1]).to(dev)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: tg.rms_norm_quant(dual(x), w), lambda: tg.rms_norm_quant(x, w, residual=dual(x)), lambda: tg.apply_rope(dual(q), kv, at, f),
                     lambda: tg.apply_rope(q, dual(kv), at, f), lambda: tg.kv_cache_write(cache, dual(kv), kv, table, lens),
                     lambda: tg.kv_cache_write(cache, kv, dual(kv), table, lens), lambda: tg.kv_cache_write(cache, kv, kv, table, lens, inv_freq=f, q=dual(q)),
                     lambda: tg.paged_attention(dual(q), cache, table, lens)):
            with pytest.raises(RuntimeError, match="no backward"):
                call()
        tg.paged_attention(q, cache, table, lens)  # the others are served
