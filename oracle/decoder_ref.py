"""Plain CPU definitions of the decoder operators, in 64 bits where they compute and bit by bit where they quantise.
Test infrastructure: written from the formulas, one sequence, page and head at a time."""

from __future__ import annotations

import math

import torch

PAGE = 128
FP8 = torch.float8_e4m3fn


def ref_rms_norm(x, weight, eps, residual=None, offset=0.0):
    """(y f64, h): y unrounded, h the sum in x's type."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    f = h.double()
    return f / torch.sqrt((f * f).mean(-1, keepdim=True) + eps) * (weight.double() + offset), h


def ref_rope(x, positions, inv_freq, interleaved=False, magnitude=1.0):
    """f64 rotation of x [tokens, heads, dim]."""
    R = 2 * inv_freq.numel()
    a = positions.double()[:, None] * inv_freq.double()
    c, s = (torch.cos(a) * magnitude)[:, None], (torch.sin(a) * magnitude)[:, None]
    o = x.double().clone()
    i, j = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    u, v = x.double()[..., i], x.double()[..., j]
    o[..., i], o[..., j] = u * c - v * s, v * c + u * s
    return o


def cache_scale(amax: float) -> float:
    if amax == 0:
        return 2.0**-60
    return 2.0 ** min(max(math.ceil(math.log2(amax / 448.0)), -60), 60)


def to_e4m3(x):
    """f32 / f64 -> e4m3 bytes, saturating."""
    return x.float().clamp(-448, 448).to(FP8)


def ref_kv_write(cache, k, v, block_table, seq_lens, cu):
    """Writes (already rotated) k, v [tokens, heads, dim] into cache = [k, v, k_scale, v_scale] (CPU tensors), in place."""
    pages = cache[0].shape[0]
    for b, length in enumerate(seq_lens.tolist()):
        lo, hi = int(cu[b]), int(cu[b + 1])
        start = length - (hi - lo)
        for page in range(max(start, 0) // PAGE, -(-length // PAGE)):
            if page >= block_table.shape[1] or not 0 <= int(block_table[b, page]) < pages:
                continue
            phys = int(block_table[b, page])
            t0, t1 = max(start - page * PAGE, 0), min(length - page * PAGE, PAGE)
            rows = slice(lo + page * PAGE + t0 - start, lo + page * PAGE + t1 - start)
            for x, store, scale, is_v in ((k, cache[0], cache[2], False), (v, cache[1], cache[3], True)):
                for h in range(store.shape[1]):
                    new = x[rows, h].float()
                    finite = new[new.isfinite()]
                    s = cache_scale(float(finite.abs().max()) if finite.numel() else 0.0)
                    block = store[phys, h].view(torch.uint8)
                    block = block.T if is_v else block  # [token, dim], a view
                    if t0 > 0:
                        old = float(scale[phys, h])
                        if old >= s:
                            s = old
                        else:
                            block[:t0] = to_e4m3(block[:t0].contiguous().view(FP8).float() * (old / s)).view(torch.uint8)
                    block[t0:t1] = to_e4m3(new / s).view(torch.uint8)
                    scale[phys, h] = s


def cache_values(cache, block_table_row, length):
    """k, v [heads, length, dim] f64 of a sequence."""
    n = -(-length // PAGE)
    at = block_table_row[:n].long()
    k = cache[0].view(torch.uint8)[at].view(FP8).double() * cache[2][at].double()[..., None, None]
    v = cache[1].view(torch.uint8)[at].view(FP8).double() * cache[3][at].double()[..., None, None]
    H, D = k.shape[1], k.shape[3]
    return k.transpose(0, 1).reshape(H, -1, D)[:, :length], v.permute(1, 0, 3, 2).reshape(H, -1, D)[:, :length]


def ref_attention(q, cache, block_table, seq_lens, cu, scale=None, window=0, sinks=0):
    """(o, sum of p |v|, largest scale * sum |q k| of what a row sees [.., 1], largest p * v_scale times the sum of the
    bytes' |v|) [tokens, heads, dim] in f64; rows outside cu are zero."""
    T, Hq, D = q.shape
    o, mag, size, coarse = (torch.zeros(T, Hq, n, dtype=torch.float64) for n in (D, D, 1, D))
    scale = D**-0.5 if scale is None else scale
    for b, length in enumerate(seq_lens.tolist()):
        lo, hi = int(cu[b]), int(cu[b + 1])
        if hi == lo or length <= 0:
            continue
        k, v = cache_values(cache, block_table[b], length)
        H = k.shape[0]
        pos = torch.arange(length - (hi - lo), length)[:, None]
        j = torch.arange(length)[None]
        seen = j <= pos
        if window:
            seen &= (j > pos - window) | (j < sinks)
        for h in range(H):
            rows = q[lo:hi].double().unflatten(1, (H, -1))[:, h].transpose(0, 1)  # [group, n, D]
            s = (rows @ k[h].T * scale).masked_fill(~seen, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(m.isinf(), torch.zeros_like(m), m))
            p = torch.where(seen, p, torch.zeros_like(p))
            l = p.sum(-1, keepdim=True)
            p = p / torch.where(l == 0, torch.ones_like(l), l)
            # hidden values are not read, whatever they are
            vv = torch.where(seen.any(0)[:, None], v[h], torch.zeros_like(v[h]))
            g = rows.shape[0]
            o[lo:hi].view(hi - lo, H, g, D)[:, h] = (p @ vv).transpose(0, 1)
            mag[lo:hi].view(hi - lo, H, g, D)[:, h] = (p @ vv.abs()).transpose(0, 1)
            a = (rows.abs() @ k[h].abs().T * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            size[lo:hi].view(hi - lo, H, g, 1)[:, h] = a.transpose(0, 1)
            vs = cache[3][block_table[b, : -(-length // PAGE)].long(), h].double().repeat_interleave(PAGE)[:length]
            top = (p * vs).amax(-1, keepdim=True) * (seen.double() @ (vv.abs() / vs[:, None]))
            coarse[lo:hi].view(hi - lo, H, g, D)[:, h] = top.transpose(0, 1)
    return o, mag, size, coarse
