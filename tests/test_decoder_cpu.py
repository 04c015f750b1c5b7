"""Decoder operators without a GPU: frequencies against their formulas, refusals of the C entry points and of the Python
ones, and the CPU definitions against each other."""

import math

import pytest
import torch

import tilegym_b200 as tg
from oracle import decoder_ref as D
from tilegym_b200 import _lib, ops

F8 = torch.float8_e4m3fn
BF = torch.bfloat16


def _d(t):
    return _lib.desc(t)


# ------------------------------------------------------------------ frequencies
def test_frequencies_plain_and_linear():
    f, m = tg.rope_frequencies(128, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (64,) and m == 1.0 and float(f[0]) == 1.0
    assert abs(float(f[63]) - 10000.0 ** (-126 / 128)) < 1e-18
    half, _ = tg.rope_frequencies(128, 10000.0, rotary_dim=32, device="cpu")
    assert half.shape == (16,) and abs(float(half[1]) - 10000.0 ** (-2 / 32)) < 1e-16
    lin, m = tg.rope_frequencies(128, 10000.0, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert torch.allclose(lin * 4, f, rtol=1e-15) and m == 1.0


def test_frequencies_scaled_for_long_contexts():
    f, _ = tg.rope_frequencies(128, 500000.0, device="cpu")
    cfg = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}
    s, m = tg.rope_frequencies(128, 500000.0, scaling=cfg, device="cpu")
    for i in range(64):
        wave = 2 * math.pi / float(f[i])
        if wave < 8192 / 4:
            want = float(f[i])
        elif wave > 8192:
            want = float(f[i]) / 8
        else:
            t = (8192 / wave - 1) / (4 - 1)
            want = (1 - t) * float(f[i]) / 8 + t * float(f[i])
        assert abs(float(s[i]) - want) <= 1e-14 * want
    assert m == 1.0
    f, _ = tg.rope_frequencies(64, 10000.0, device="cpu")
    cfg = {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    s, m = tg.rope_frequencies(64, 10000.0, scaling=cfg, device="cpu")
    assert abs(m - (0.1 * math.log(16) + 1)) < 1e-15
    turns = 4096 * f / (2 * math.pi)
    # pairs that turn often keep their frequency, pairs that turn less than once are divided, in between monotonously
    assert torch.equal(s[turns > 64], f[turns > 64]) and torch.allclose(s[turns < 0.5] * 16, f[turns < 0.5], rtol=1e-15)
    ratio = s / f
    assert bool((ratio[1:] <= ratio[:-1] + 1e-15).all())
    _, m = tg.rope_frequencies(64, scaling={**cfg, "mscale": 0.7, "mscale_all_dim": 0.7}, device="cpu")
    assert m == 1.0
    _, m = tg.rope_frequencies(64, scaling={**cfg, "attention_factor": 1.5}, device="cpu")
    assert m == 1.5


def test_frequencies_refuse():
    for bad in (0, 8, 40, 144):
        with pytest.raises(ValueError):
            tg.rope_frequencies(128, rotary_dim=bad, device="cpu")
    with pytest.raises(NotImplementedError):
        tg.rope_frequencies(128, scaling={"rope_type": "longrope"}, device="cpu")


# ------------------------------------------------------------------ definitions
def test_cache_scale_is_the_smallest_power_of_two():
    for a in (1e-30, 0.01, 1.0, 447.9, 448.0, 448.1, 896.0, 1e5, 3e38):
        s = D.cache_scale(a)
        assert math.log2(s) == int(math.log2(s)) and -60 <= math.log2(s) <= 60
        if 2.0**-60 < s < 2.0**60:
            assert a / s <= 448 < a / (s / 2)


def test_a_value_survives_the_cache_within_half_a_step():
    g = torch.Generator().manual_seed(0)
    cache = [torch.zeros(2, 1, 128, 64, dtype=torch.uint8).view(F8), torch.zeros(2, 1, 64, 128, dtype=torch.uint8).view(F8), torch.ones(2, 1), torch.ones(2, 1)]
    k, v = torch.randn(150, 1, 64, generator=g), torch.randn(150, 1, 64, generator=g)
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    D.ref_kv_write(cache, k, v, table, torch.tensor([150]), [0, 150])
    for got, want in zip(D.cache_values(cache, table[0], 150), (k, v)):
        want = want.transpose(0, 1).double()
        # steps below the normal range: 2^-9 of a scale of at most max / 224
        assert bool(((got - want).abs() <= torch.clamp(want.abs() * 2.0**-4, min=float(want.abs().max()) / 224 * 2.0**-10)).all())


# ------------------------------------------------------------------ refusals
def test_norm_refusals():
    L = _lib.lib()
    x, w = torch.zeros(4, 256, dtype=BF), torch.zeros(256, dtype=BF)
    y, s, h = torch.zeros(4, 256, dtype=F8), torch.zeros(4, 2), torch.zeros(4, 256, dtype=BF)

    def call(Y=y, S=s, H=None, X=x, R=None, W=w, eps=1e-6):
        return L.tg_rms_norm_quant(_d(Y), _d(S), _d(H), _d(X), _d(R), _d(W), eps, 0.0, 0, 0)

    assert call(X=x.float()) == -2 and call(W=w.half()) == -2 and call(Y=y.view(torch.uint8)) == -2 and call(S=s.double()) == -2
    assert call(X=torch.zeros(4, 200, dtype=BF)) == -6
    assert call(W=torch.zeros(128, dtype=BF)) == -6 and call(S=torch.zeros(4, 3)) == -6 and call(Y=y[:3]) == -6
    assert call(R=x) == -5 and call(H=h) == -5  # one without the other
    assert call(R=x.half(), H=h) == -2 and call(R=x[:3], H=h) == -6
    assert call(eps=-1.0) == -6 and call(eps=float("nan")) == -6
    assert call(X=torch.zeros(4, 260, dtype=BF)[:, :256]) == -8  # rows off the 16-byte grid
    assert call(X=None) == -5
    e = torch.zeros(0, 256, dtype=BF)
    assert call(Y=y[:0], S=s[:0], X=e) == 0
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tg.rms_norm_quant(x, w)


def test_rope_refusals():
    L = _lib.lib()
    q, pos = torch.zeros(4, 2, 64, dtype=BF), torch.zeros(4, dtype=torch.int64)
    f = torch.ones(32, dtype=torch.float64)

    def call(Qo=q, Ko=None, Q=q, K=None, P=pos, F=f):
        return L.tg_apply_rope(_d(Qo), _d(Ko), _d(Q), _d(K), _d(P), _d(F), 0, 1.0, 0, 0)

    assert call(Q=q.float()) == -2 and call(P=pos.float()) == -2 and call(F=f.float()) == -2
    assert call(P=pos[:3]) == -6 and call(F=torch.ones(12, dtype=torch.float64)) == -6 and call(F=torch.ones(40, dtype=torch.float64)) == -6
    assert call(Q=torch.zeros(4, 2, 72, dtype=BF), Qo=torch.zeros(4, 2, 72, dtype=BF)) == -6
    assert call(K=q) == -5 and call(K=q[:3], Ko=q[:3]) == -6 and call(K=q.half(), Ko=q.half()) == -2
    assert call(Qo=q[:, :1]) == -6
    bad = torch.zeros(4, 2, 68, dtype=BF)[..., :64]
    assert call(Q=bad) == -8
    assert call(Q=q[:0], Qo=q[:0], P=pos[:0]) == 0
    assert call(K=q, Ko=q) == -6  # one tensor as q and k, in place
    assert call(Qo=torch.zeros(1, 2, 64, dtype=BF).expand(4, 2, 64)) == -6 and call(Qo=torch.zeros(4, 1, 64, dtype=BF).expand(4, 2, 64)) == -6
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tg.apply_rope(q, None, pos, f)


def cache(pages=3, heads=2, dim=64):
    c = tg.FP8KVCache.empty(pages, heads, dim, device="cpu")
    return list(c)


def test_cache_and_attention_refusals():
    L = _lib.lib()
    c = cache()
    t, lens, cu = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    x, q = torch.zeros(2, 2, 64, dtype=BF), torch.zeros(2, 8, 64, dtype=BF)
    f = torch.ones(32, dtype=torch.float64)

    def write(c=c, K=x, V=x, T=t, S=lens, C=None, Qo=None, Q=None, F=None):
        return L.tg_kv_cache_write(*map(_d, c), _d(K), _d(V), _d(T), _d(S), _d(C), _d(Qo), _d(Q), _d(F), 0, 1.0, 0, 0)

    def attend(c=c, O=q, Q=q, T=t, S=lens, C=None, n=1, scale=0.125, window=0, sinks=0, ws=0, size=0):
        return L.tg_paged_attention(_d(O), _d(Q), *map(_d, c), _d(T), _d(S), _d(C), n, scale, window, sinks, ws, size, 0, 0)

    def read(c=c, K=torch.zeros(2, 5, 2, 64, dtype=BF), V=torch.zeros(2, 5, 2, 64, dtype=BF), T=t, S=lens):
        return L.tg_kv_cache_read(_d(K), _d(V), *map(_d, c), _d(T), _d(S), 0, 0)

    def swap(i, new):
        return [new if i == j else y for j, y in enumerate(c)]

    for call in (write, attend, read):
        assert call(c=swap(0, c[0].view(torch.uint8))) == -2 and call(c=swap(2, c[2].double())) == -2
        assert call(c=swap(0, torch.zeros(3, 2, 64, 64, dtype=F8))) == -6  # pages of 64
        assert call(c=swap(1, torch.zeros(3, 2, 128, 64, dtype=F8))) == -6  # values lie [dim][token]
        assert call(c=swap(3, torch.ones(3, 3))) == -6 and call(c=swap(0, torch.zeros(3, 2, 128, 32, dtype=F8))) == -6
        assert call(c=swap(0, torch.zeros(3, 128, 2, 64, dtype=F8).transpose(1, 2))) == -6
        assert call(T=t.long()) == -2 and call(T=t[:1]) == -6 and call(S=lens.long()) == -2
    assert write(K=x.float()) == -2 and write(V=x.half()) == -2 and write(K=x[:1], V=x[:1]) == -6 and write(K=x[:, :1], V=x[:, :1]) == -6
    assert write(C=cu[:2]) == -6 and write(C=cu.long()) == -2
    assert write(Q=q, Qo=q) == -5 and write(Q=q, F=f) == -5 and write(F=f.float()) == -2
    assert write(K=torch.zeros(2, 2, 68, dtype=BF)[..., :64]) == -8
    assert write(K=x[:0], V=x[:0], C=cu) == 0
    assert attend(Q=q.float()) == -2 and attend(Q=q[:, :3], O=q[:, :3]) == -6 and attend(O=q[:1]) == -6
    wide = torch.zeros(2, 130, 64, dtype=BF)
    assert attend(Q=wide, O=wide) == -6  # 65 query heads on a cache head
    assert attend(n=0) == -6 and attend(window=-1) == -6 and attend(sinks=-1, window=4) == -6 and attend(sinks=2) == -6
    assert attend(scale=0.0) == -6 and attend(scale=float("nan")) == -6 and attend(scale=float("inf")) == -6
    assert attend(O=q[:1].expand(2, 8, 64)) == -6 and attend(O=q[:, :1].expand(2, 8, 64)) == -6
    assert attend(O=torch.zeros(5, 8, 64, dtype=BF).as_strided((2, 8, 64), (256, 64, 1))) == -6  # rows that reach into the next
    assert attend(Q=q[:1], O=q[:1]) == -6 and attend(Q=q[:0], O=q[:0], C=cu) == 0
    assert read(K=torch.zeros(2, 5, 2, 64)) == -2 and read(V=torch.zeros(2, 4, 2, 64, dtype=BF)) == -6
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        tg.paged_attention(q, tg.FP8KVCache(*c), t, lens)
    with pytest.raises(ValueError):
        tg.FP8KVCache.empty(3, 2, 96, device="cpu")


def test_operators_have_no_backward():
    x = torch.zeros(2, 128, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        ops._no_grad_inputs(x)
    with torch.no_grad():
        ops._no_grad_inputs(x)
    ops._no_grad_inputs(x.detach(), None)


def test_attention_workspace():
    def size(heads, kv, dim, n, tokens, seqs, pages, sms=148):
        return _lib.lib().tg_paged_attention_workspace_bytes(heads, kv, dim, n, tokens, seqs, pages, sms)

    assert size(32, 8, 128, 1, 0, 0, 0) > 0 and size(32, 8, 128, 1, 5, 5, 9) == size(32, 8, 128, 1, 0, 0, 0)
    assert size(32, 8, 128, 4096, 4096, 1, 4096) == 0  # blocks enough
    # 100 tokens: two pairs of tiles and heads of 8, 16 blocks, nine to a block's pages; no more parts than pages in fours
    assert size(32, 8, 128, 100, 100, 1, 400) == 16 * 9 * 256 * (128 * 4 + 8)
    assert size(32, 8, 128, 100, 100, 1, 11) == 16 * 2 * 256 * (128 * 4 + 8)
    assert size(32, 8, 128, 100, 100, 1, 7) == 0
    assert size(1, 1, 64, 65, 65, 1, 1 << 20) == 32 * 256 * (64 * 4 + 8)
    assert size(33, 8, 128, 1, 1, 1, 1) == 0 and size(0, 8, 128, 1, 1, 1, 1) == 0 and size(8, 0, 128, 1, 1, 1, 1) == 0


def test_layer_refusals():
    """What a layer has beside the projections that FP8DecoderLayer knows is refused before anything is quantised."""
    nn = torch.nn

    def layer(**change):
        m = nn.Module()
        m.self_attn, m.mlp = nn.Module(), nn.Module()
        m.mlp.act_fn = nn.SiLU()
        m.self_attn.scaling = 64**-0.5
        for name, value in change.items():
            owner, name = (m.self_attn, name[4:]) if name.startswith("att_") else (m.mlp, name[4:]) if name.startswith("mlp_") else (m, name)
            setattr(owner, name, value)
        return m

    f = torch.ones(32, dtype=torch.float64)
    for change in ({"att_q_norm": nn.LayerNorm(64)}, {"att_scaling": 0.2}, {"att_sinks": nn.Parameter(torch.zeros(8))}, {"mlp_act_fn": nn.GELU()},
                   {"pre_feedforward_layernorm": nn.LayerNorm(64)}, {"att_attn_logit_softcapping": 50.0}):
        with pytest.raises(NotImplementedError):
            tg.FP8DecoderLayer.from_layer(layer(**change), 64, f)
    with pytest.raises(AttributeError):  # an ordinary one gets as far as its projections
        tg.FP8DecoderLayer.from_layer(layer(), 64, f)
