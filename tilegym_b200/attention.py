"""Rotary positions, the paged 8-bit key / value cache and the attention that reads it: the operators of a decoder layer
between its FP8 GEMMs.

The cache (`FP8KVCache`) keeps pages of 128 tokens per key / value head in e4m3 with ONE power-of-two scale per page and
head, for keys and for values.  `kv_cache_write` quantises new tokens as it writes them (rotating keys and queries on the
way), `paged_attention` attends over the cache for single tokens, drafts and prompts alike, `kv_cache_read` brings pages
back to 16 bits.  A batch is ragged: sequence b's new tokens are rows [cu_seqlens[b], cu_seqlens[b + 1]) of the token
dimension and its last positions, seq_lens[b] counts them in.  Everything is enqueued on the current stream and nothing
is read back, so the calls can be captured into a CUDA graph whose tables change between replays.
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib, ops

PAGE_TOKENS = 128  # tokens of a cache page, and of a scale

_INT_MAX = 2**31 - 1
_FEW_ROWS = 32  # (new tokens, heads of a group) that the kernel for few rows takes
_FP8 = torch.float8_e4m3fn
_16BIT = (torch.bfloat16, torch.float16)


class FP8KVCache(NamedTuple):
    """k [pages, kv_heads, 128, head_dim] and v [pages, kv_heads, head_dim, 128] (values lie [dim][token]) in
    float8_e4m3fn, k_scale / v_scale [pages, kv_heads] fp32, positive (what `kv_cache_write` sets is a power of two).  A value
    is its byte times its block's scale."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, head_dim: int, device="cuda") -> "FP8KVCache":
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        return cls(
            torch.zeros((num_pages, num_kv_heads, PAGE_TOKENS, head_dim), dtype=torch.uint8, device=device).view(_FP8),
            torch.zeros((num_pages, num_kv_heads, head_dim, PAGE_TOKENS), dtype=torch.uint8, device=device).view(_FP8),
            torch.ones((num_pages, num_kv_heads), dtype=torch.float32, device=device),
            torch.ones((num_pages, num_kv_heads), dtype=torch.float32, device=device),
        )


def rope_frequencies(
    head_dim: int, base: float = 10000.0, rotary_dim: Optional[int] = None, scaling: Optional[dict] = None, device="cuda"
) -> Tuple[torch.Tensor, float]:
    """(inv_freq, magnitude): what `apply_rope` and `kv_cache_write` take, computed in 64 bits.

    inv_freq[i] = base^(-2 i / rotary_dim) radians per position (float64, rotary_dim / 2 values), changed by `scaling`
    as model configurations write it (`rope_type` or `type`):
      "default"  nothing
      "linear"   divided by `factor`
      "llama3"   divided by `factor` where the wavelength is over original_max_position_embeddings / low_freq_factor,
                 untouched below / high_freq_factor, blended in between
      "yarn"     divided by `factor` where a pair turns less than beta_slow times over the original length, untouched
                 over beta_fast times, a ramp over the pairs in between; magnitude 0.1 ln(factor) + 1 (attention_factor,
                 or the quotient of the mscale / mscale_all_dim forms, where given)
    """
    R = head_dim if rotary_dim is None else rotary_dim
    if R % 16 != 0 or not 0 < R <= head_dim:
        raise ValueError(f"rotary_dim must be a multiple of 16 up to head_dim, got {R}")
    f = base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    magnitude = 1.0
    kind = "default" if not scaling else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "linear":
        f = f / float(scaling["factor"])
    elif kind == "llama3":
        factor, low, high = (float(scaling[k]) for k in ("factor", "low_freq_factor", "high_freq_factor"))
        turns = scaling["original_max_position_embeddings"] * f / (2 * math.pi)  # over the original length
        blend = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        f = f * (blend + (1.0 - blend) / factor)
    elif kind == "yarn":
        factor, length = float(scaling["factor"]), scaling["original_max_position_embeddings"]

        def pair_that_turns(times: float) -> float:  # index of the pair that turns so many times over the length
            return R * math.log(length / (times * 2 * math.pi)) / (2 * math.log(base))

        low, high = pair_that_turns(scaling.get("beta_fast") or 32.0), pair_that_turns(scaling.get("beta_slow") or 1.0)
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, R - 1)
        if low == high:
            high += 0.001
        ramp = ((torch.arange(R // 2, dtype=torch.float64) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * ((1.0 - ramp) + ramp / factor)

        def grown(m: float) -> float:
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

        if scaling.get("attention_factor") is not None:
            magnitude = float(scaling["attention_factor"])
        elif scaling.get("mscale") and scaling.get("mscale_all_dim"):
            magnitude = grown(scaling["mscale"]) / grown(scaling["mscale_all_dim"])
        else:
            magnitude = grown(1.0)
    elif kind != "default":
        raise NotImplementedError(f"rope scaling {kind!r} is not implemented (default, linear, llama3, yarn)")
    return f.to(device), magnitude


def _heads(x: torch.Tensor, name: str) -> Tuple[torch.Tensor, bytes]:
    """[tokens, heads, dim] as the kernels read it (itself, or a copy where a pitch breaks the 16-byte alignment), and its
    descriptor.  The tensor has to be held until the launch: the allocator would hand a copy's memory to the next one."""
    if x.dim() != 3:
        raise _lib.TileGymB200Error(-6, f"{name} must be [tokens, heads, head_dim]")
    if x.dtype not in _16BIT:
        raise _lib.TileGymB200Error(-2, f"{name} must be bf16 or f16, got {x.dtype}")
    n0, n1, n2 = x.shape
    s0, s1, s2 = x.stride()
    if s2 != 1 or s0 % 8 or s1 % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        s0, s1 = n1 * n2, n2
    return x, _lib.desc3d(x.data_ptr(), n0, n1, n2, s0, s1, x.dtype)


def _new_heads(x: torch.Tensor) -> Tuple[torch.Tensor, bytes]:
    """A dense new tensor of x's shape and type, and its descriptor."""
    n0, n1, n2 = x.shape
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    return out, _lib.desc3d(out.data_ptr(), n0, n1, n2, n1 * n2, n2, x.dtype)


def _frequencies(inv_freq: torch.Tensor) -> torch.Tensor:
    if inv_freq.dtype != torch.float64:
        inv_freq = inv_freq.to(torch.float64)
    return inv_freq if inv_freq.is_contiguous() else inv_freq.contiguous()


def _table(t: Optional[torch.Tensor], name: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != torch.int32:
        raise _lib.TileGymB200Error(-2, f"{name} must be int32, got {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def _tables(block_table, seq_lens, cu_seqlens):
    return _table(block_table, "block_table"), _table(seq_lens, "seq_lens"), _table(cu_seqlens, "cu_seqlens")


def apply_rope(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    interleaved: bool = False,
    magnitude: float = 1.0,
    inplace: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotates q (tokens, heads, head_dim) and k (tokens, kv_heads, head_dim; may be None) by their positions: (q, k).

    Pair i of a head turns by positions[t] * inv_freq[i] (see `rope_frequencies`; the angle is reduced exactly, at any
    position); 2 * len(inv_freq) elements of a head are rotated and the others copied.  Pairs are (i, i + R / 2), or
    (2 i, 2 i + 1) with interleaved=True.  cos and sin are scaled by `magnitude`.  positions (tokens,) int32 or int64.
    With inplace=True q and k are overwritten (their pitches must keep 16-byte alignment) and only the rotated elements
    are touched.
    """
    if _lib.fast is not None:
        result = _lib.fast.apply_rope(q, k, positions, inv_freq, interleaved, magnitude, inplace)
        if result is not None:
            return result
    dev = ops._cuda_index(q, k, positions, inv_freq)
    ops._no_grad_inputs(q, k)
    q1, q_desc = _heads(q, "q")
    k1, k_desc = (None, None) if k is None else _heads(k, "k")
    if inplace:
        assert q1 is q and k1 is k, "in-place rotation needs dense heads on 16-byte boundaries"
        qo, qo_desc, ko, ko_desc = q, q_desc, k, k_desc
    else:
        qo, qo_desc = _new_heads(q)
        ko, ko_desc = (None, None) if k is None else _new_heads(k)
    if positions.dtype not in (torch.int32, torch.int64):
        raise _lib.TileGymB200Error(-2, f"positions must be int32 or int64, got {positions.dtype}")
    if not positions.is_contiguous():
        positions = positions.contiguous()
    inv_freq = _frequencies(inv_freq)
    rc = _lib.lib().tg_apply_rope(
        qo_desc, ko_desc, q_desc, k_desc, _lib.desc(positions), _lib.desc(inv_freq), 1 if interleaved else 0, float(magnitude), dev,
        torch._C._cuda_getCurrentRawStream(dev),
    )
    _lib.check_rc(rc)
    return qo, ko


def kv_cache_write(
    cache: FP8KVCache,
    k: torch.Tensor,
    v: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    inv_freq: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    magnitude: float = 1.0,
) -> Optional[torch.Tensor]:
    """Quantises new keys and values into the cache's pages, in one launch; returns the rotated q, or None without q.

    k, v (tokens, kv_heads, head_dim) bf16 or f16; block_table (seqs, pages per sequence) int32, seq_lens (seqs,) int32
    lengths including the new tokens, cu_seqlens (seqs + 1,) int32 (None: one new token per sequence).  With inv_freq
    the keys are rotated at their positions first (rounded to 16 bits, as `apply_rope` would leave them), and q
    (tokens, heads, head_dim) is rotated into a new tensor.

    The scale of a (page, head) is the smallest power of two that takes its largest finite new value to at most 448
    (exponent within +-60).  A page with earlier tokens keeps the larger of its own scale and that one; where it grew,
    the earlier bytes are moved to it.  NaN stays NaN, infinities saturate, and neither counts for the scale.  Only the
    new tokens' bytes (and the earlier ones of a page whose scale grew) are written.  Rows of the batch outside
    cu_seqlens, positions outside the table and pages outside the cache are left alone (their rows of q are unspecified).
    A page that is written must belong to one sequence and stand once in its row of the table.
    """
    if _lib.fast is not None:
        result = _lib.fast.kv_cache_write(*cache, k, v, block_table, seq_lens, cu_seqlens, inv_freq, q, interleaved, magnitude)
        if result is not None:
            return result[0]
    dev = ops._cuda_index(*cache, k, v, block_table, seq_lens, cu_seqlens, inv_freq, q)
    ops._no_grad_inputs(k, v, q)
    qo = qo_desc = q_desc = None
    if q is not None:
        if inv_freq is None:
            raise _lib.TileGymB200Error(-6, "q is passed to be rotated: inv_freq is missing")
        q, q_desc = _heads(q, "q")
        qo, qo_desc = _new_heads(q)
    k, k_desc = _heads(k, "k")
    v, v_desc = _heads(v, "v")
    block_table, seq_lens, cu_seqlens = _tables(block_table, seq_lens, cu_seqlens)
    if inv_freq is not None:
        inv_freq = _frequencies(inv_freq)
    desc = _lib.desc
    rc = _lib.lib().tg_kv_cache_write(
        desc(cache.k), desc(cache.v), desc(cache.k_scale), desc(cache.v_scale), k_desc, v_desc, desc(block_table), desc(seq_lens),
        desc(cu_seqlens), qo_desc, q_desc, desc(inv_freq), 1 if interleaved else 0, float(magnitude), dev,
        torch._C._cuda_getCurrentRawStream(dev),
    )
    _lib.check_rc(rc)
    return qo


def kv_cache_read(
    cache: FP8KVCache,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    max_len: int,
    dtype: torch.dtype = torch.bfloat16,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v), each (seqs, max_len, kv_heads, head_dim) in `dtype` (bf16: exact under power-of-two scales), with zeros behind a sequence's length
    (and where the table has no page of the cache)."""
    dev = ops._need_cuda(*cache, block_table, seq_lens)
    if dtype not in _16BIT:
        raise _lib.TileGymB200Error(-2, f"kv_cache_read returns bf16 or f16, not {dtype}")
    if max_len < 0:
        raise _lib.TileGymB200Error(-6, "max_len must not be negative")
    shape = (seq_lens.shape[0], int(max_len), cache.k.shape[1], cache.k.shape[3])
    k = torch.empty(shape, dtype=dtype, device=dev)
    v = torch.empty(shape, dtype=dtype, device=dev)
    block_table, seq_lens, _ = _tables(block_table, seq_lens, None)
    rc = _lib.lib().tg_kv_cache_read(
        _lib.desc(k), _lib.desc(v), _lib.desc(cache.k), _lib.desc(cache.v), _lib.desc(cache.k_scale), _lib.desc(cache.v_scale),
        _lib.desc(block_table), _lib.desc(seq_lens), dev.index, ops._stream(dev),
    )
    _lib.check_rc(rc)
    return k, v


def paged_attention(
    q: torch.Tensor,
    cache: FP8KVCache,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    max_q_len: Optional[int] = None,
    scale: Optional[float] = None,
    window: int = 0,
    sinks: int = 0,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Causal attention of new tokens over the cache, which already holds them: (tokens, heads, head_dim) in q's type.

    q (tokens, heads, head_dim) bf16 or f16, heads a multiple of the cache's heads (at most 64 times): heads
    h * group .. (h + 1) * group - 1 read cache head h.  Tables as in `kv_cache_write`.  A token at position i sees
    positions j <= i; with window > 0 of those only j > i - window or j < sinks.  scale: of the products, positive
    (1 / sqrt(head_dim) by default).  max_q_len bounds the new tokens of any sequence (1 without cu_seqlens, else the
    batch's token count by default); saying that it is small selects the kernel for few rows, and rows beyond it are not
    computed.  One kernel serves the whole batch: single tokens beside a chunk of a prompt are faster as two calls.  A token that
    sees nothing (a sequence of length 0 in a padded batch) gets zeros; rows outside cu_seqlens are not written.  out may be q.
    """
    dev = ops._cuda_index(q, *cache, block_table, seq_lens, cu_seqlens, out)
    if q.dim() != 3:
        raise _lib.TileGymB200Error(-6, "q must be [tokens, heads, head_dim]")
    tokens, heads, dim = q.shape
    bound = 1 if cu_seqlens is None else max(tokens, 1)
    max_q_len = bound if max_q_len is None else min(int(max_q_len), bound)
    window, sinks = min(int(window), _INT_MAX), min(int(sinks), _INT_MAX)  # beyond any position they mean the same
    kv_heads = cache.k.shape[1]
    if max_q_len * heads <= _FEW_ROWS * kv_heads:  # nothing more counts
        need = _workspace_bytes(heads, kv_heads, dim, max_q_len, 0, 0, 0, dev)
    else:
        seqs = seq_lens.numel()
        need = _workspace_bytes(heads, kv_heads, dim, max_q_len, tokens, seqs, block_table.numel() // max(seqs, 1), dev)
    scale = dim ** -0.5 if scale is None else float(scale)
    if _lib.fast is not None:
        result = _lib.fast.paged_attention(q, *cache, block_table, seq_lens, cu_seqlens, max_q_len, scale, window, sinks, out, need)
        if result is not None:
            return result if out is None else out
    ops._no_grad_inputs(q)
    q, q_desc = _heads(q, "q")
    if out is None:
        out, out_desc = _new_heads(q)
    else:
        assert out.shape == q.shape and out.dtype == q.dtype, "out must have q's shape and type"
        out_desc = _lib.desc(out)
    block_table, seq_lens, cu_seqlens = _tables(block_table, seq_lens, cu_seqlens)
    # allocated per call: calls on other streams, and graphs that are replayed side by side, never share it
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    desc = _lib.desc
    rc = _lib.lib().tg_paged_attention(
        out_desc, q_desc, desc(cache.k), desc(cache.v), desc(cache.k_scale), desc(cache.v_scale), desc(block_table), desc(seq_lens),
        desc(cu_seqlens), max_q_len, scale, window, sinks,
        0 if ws is None else ws.data_ptr(), need, dev, torch._C._cuda_getCurrentRawStream(dev),
    )
    _lib.check_rc(rc)
    return out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(heads: int, kv_heads: int, dim: int, max_q_len: int, tokens: int, seqs: int, pages_per_seq: int, dev: int) -> int:
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    return _lib.lib().tg_paged_attention_workspace_bytes(heads, kv_heads, dim, max_q_len, tokens, seqs, pages_per_seq, sms)
