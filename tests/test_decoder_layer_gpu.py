"""FP8DecoderLayer: the decoder operators and the FP8 GEMMs run together, as a serving loop would run them, against a plain
layer in fp32 on the dequantised weights and unquantised activations.

Tolerance: the layer rounds to e4m3 on its way from input to output in six places (norm, keys, values, attention's output,
norm, silu * mul), each at most half a step, 2^-4, relative to its values.  For independent errors spread evenly over a step
that is 2^-4 / sqrt(3) in the 2-norm, sqrt(6) of it for all six, 0.09 of what the layer adds to the residual stream.  A
second layer sees the first one's error too: sqrt(2) as much."""

import math

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

import tilegym_b200 as tg  # noqa: E402

BF = torch.bfloat16
STEP = math.sqrt(6) * 2.0**-4 / math.sqrt(3)


class Plain(nn.Module):
    """The weights of a small pre-norm decoder layer under the names that models use."""

    def __init__(self, hidden, heads, kv, dim, inter, bias, seed):
        super().__init__()
        g = torch.Generator().manual_seed(seed)

        def lin(i, o, b):
            m = nn.Linear(i, o, bias=b)
            m.weight.data = (torch.randn(o, i, generator=g) * 0.6 / math.sqrt(i)).to(BF)
            if b:
                m.bias.data = (torch.randn(o, generator=g) * 0.1).to(BF)
            return m

        self.input_layernorm, self.post_attention_layernorm = nn.RMSNorm(hidden, eps=1e-5), nn.RMSNorm(hidden, eps=1e-5)
        for n in (self.input_layernorm, self.post_attention_layernorm):
            n.weight.data = (1 + 0.1 * torch.randn(hidden, generator=g)).to(BF)
        self.self_attn, self.mlp = nn.Module(), nn.Module()
        a, m = self.self_attn, self.mlp
        a.q_proj, a.k_proj, a.v_proj = lin(hidden, heads * dim, bias), lin(hidden, kv * dim, bias), lin(hidden, kv * dim, bias)
        a.o_proj = lin(heads * dim, hidden, False)
        m.gate_proj, m.up_proj, m.down_proj = lin(hidden, inter, False), lin(hidden, inter, False), lin(inter, hidden, False)


def plain_forward(fp8, x, dim, window, sinks):
    """fp32 on the GPU, one whole sequence x [n, hidden]; returns what the layer adds to x."""
    w = {n: tg.weight_dequant(getattr(fp8, n), getattr(fp8, n + "_scale"), 128, torch.float32) for n in ("qkv", "o", "gate_up", "down")}

    def norm(v, g):
        return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + fp8.eps) * g.float()

    n = x.shape[0]
    qkv = norm(x, fp8.norm1) @ w["qkv"].T + (0 if fp8.qkv_bias is None else fp8.qkv_bias.float())
    q, k, v = qkv.view(n, -1, dim).split((fp8.num_heads, fp8.num_kv_heads, fp8.num_kv_heads), 1)
    a = torch.arange(n, device=x.device).double()[:, None] * fp8.inv_freq
    c, s = a.cos().float()[:, None], a.sin().float()[:, None]

    def turn(t):
        u, z = t[..., : dim // 2], t[..., dim // 2 :]
        return torch.cat((u * c - z * s, z * c + u * s), -1)

    q, k = turn(q), turn(k)
    g = fp8.num_heads // fp8.num_kv_heads
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    p = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(dim)
    i, j = torch.arange(n, device=x.device)[:, None], torch.arange(n, device=x.device)[None]
    seen = (j <= i) & ((j > i - window) | (j < sinks) if window else torch.ones_like(j <= i))
    o = torch.einsum("hij,jhd->ihd", p.masked_fill(~seen, -math.inf).softmax(-1), v).flatten(1)
    h = x + o @ w["o"].T
    gate, up = (norm(h, fp8.norm2) @ w["gate_up"].T).chunk(2, -1)
    return h + (nn.functional.silu(gate) * up) @ w["down"].T - x


def far(got, want):
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("hidden,heads,kv,dim,inter,bias,window,sinks", [(512, 8, 2, 64, 1024, True, 0, 0), (768, 6, 6, 128, 640, False, 150, 4)])
def test_prompts_then_single_tokens(dev, hidden, heads, kv, dim, inter, bias, window, sinks):
    layers = []
    f, _ = tg.rope_frequencies(dim, 10000.0, device=dev)
    for n in range(2):
        layers.append(tg.FP8DecoderLayer.from_layer(Plain(hidden, heads, kv, dim, inter, bias, n).to(dev), dim, f, window=window, sinks=sinks))
    assert layers[0].eps == 1e-5
    g = torch.Generator().manual_seed(5)
    full = [260, 131, 40]  # tokens of three sequences in the end
    x = [torch.randn(n, hidden, generator=g).to(BF).to(dev) for n in full]
    caches = [tg.FP8KVCache.empty(8, kv, dim, dev) for _ in layers]
    table = torch.tensor([[5, 0, 2], [7, 3, -1], [1, -1, -1]], dtype=torch.int32, device=dev)
    want = []
    for s in x:
        h = s.float()
        d0 = plain_forward(layers[0], h, dim, window, sinks)
        want.append((d0, plain_forward(layers[1], h + d0, dim, window, sinks)))

    def step(new, done):
        """Runs both layers over the next `new` tokens of every sequence; returns what they add, by sequence."""
        rows = torch.cat([s[d : d + n] for s, n, d in zip(x, new, done)])
        lens = torch.tensor([d + n for d, n in zip(done, new)], dtype=torch.int32, device=dev)
        cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=dev)
        h, res, out = rows, None, []
        for layer, cache in zip(layers, caches):
            h, res = layer(h, res, cache, table, lens, cu, max_q_len=max(new))
            out.append(h.float() + res.float())
        return [[o.split(new)[b] for o in out] for b in range(len(new))]

    done, got = [0, 0, 0], [[], [], []]
    for new in ([200, 100, 37], [50, 28, 0], [7, 2, 2], [1, 1, 0], [1, 0, 1], [1, 0, 0]):  # prompts, a second chunk, drafts, tokens
        for b, o in enumerate(step(new, done)):
            got[b].append(o)
            done[b] += new[b]
    assert done == full
    for b in range(3):
        after = [torch.cat([o[n] for o in got[b]]) for n in range(2)]
        assert far(after[0] - x[b].float(), want[b][0]) <= STEP
        assert far(after[1] - x[b].float() - want[b][0], want[b][1]) <= math.sqrt(2) * STEP
    # the second layer's stream is residual + hidden, kept in 16 bits in between


def test_decode_step_in_a_graph(dev):
    """A captured decode step whose tables move on between replays gives what eager calls give, bit for bit; a padded slot
    (length 0) stays out of the cache."""
    dim, kv = 64, 2
    f, _ = tg.rope_frequencies(dim, 10000.0, device=dev)
    layer = tg.FP8DecoderLayer.from_layer(Plain(256, 4, kv, dim, 512, False, 3).to(dev), dim, f)
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device=dev)
    g = torch.Generator().manual_seed(6)
    xs = [torch.randn(3, 256, generator=g).to(BF).to(dev) for _ in range(5)]
    lens = [[126 + i, i + 1, 0] for i in range(5)]

    def run(call):
        cache = tg.FP8KVCache.empty(6, kv, dim, dev)
        return cache, [call(cache, i) for i in range(5)]

    def eager(cache, i):
        h, r = layer(xs[i], None, cache, table, torch.tensor(lens[i], dtype=torch.int32, device=dev))
        return h.clone()

    c1, want = run(eager)
    x, n = xs[0].clone(), torch.tensor(lens[0], dtype=torch.int32, device=dev)
    c2 = tg.FP8KVCache.empty(6, kv, dim, dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = layer(x, None, c2, table, n)
    for i in range(5):
        x.copy_(xs[i])
        n.copy_(torch.tensor(lens[i], dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, want[i])
    for a, b in zip(c1, c2):
        assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
    assert bool((c1.k[4:].view(torch.uint8) == 0).all()) and bool((c1.k_scale[4:] == 1).all())


def test_layer_refusals(dev):
    f, _ = tg.rope_frequencies(64, device=dev)
    with pytest.raises(ValueError, match="head_dim"):
        tg.FP8DecoderLayer.from_layer(Plain(256, 4, 2, 32, 512, False, 1).to(dev), 32, f)
    with pytest.raises(ValueError, match="multiples of 128"):
        tg.FP8DecoderLayer.from_layer(Plain(256, 4, 2, 64, 200, False, 1).to(dev), 64, f)
    with pytest.raises(ValueError, match="multiple of num_kv_heads"):
        tg.FP8DecoderLayer.from_layer(Plain(256, 4, 3, 64, 256, False, 1).to(dev), 64, f)
