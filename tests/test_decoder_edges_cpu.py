"""Refusals of the decoder operators that need no GPU, at the edges of what their documentation allows."""

import pytest
import torch

import tilegym_b200 as tg
from tilegym_b200 import _lib

F8 = torch.float8_e4m3fn
BF = torch.bfloat16


def _d(t):
    return _lib.desc(t)


def test_norm_refuses_a_sum_over_rows_that_are_still_read():
    """H may take the place of X or of the residual where their rows are dense: row t of H then lies on row t.  With a pitch,
    or shifted, it would lie on rows that other blocks have still to read."""
    L = _lib.lib()
    w, y, s = torch.zeros(256, dtype=BF), torch.zeros(4, 256, dtype=F8), torch.zeros(4, 2)
    memory = torch.zeros(4096, dtype=BF)
    dense, pitched, shifted = memory[:1024].view(4, 256), memory.view(8, 512)[:4, :256], memory[256:1280].view(4, 256)
    other = torch.zeros(4, 256, dtype=BF)

    def call(H, X, R, T=4):
        return L.tg_rms_norm_quant(_d(y[:T]), _d(s[:T]), _d(H), _d(X), _d(R), _d(w), 1e-6, 0.0, 0, 0)

    for X, R in ((pitched, other), (other, pitched), (shifted, other), (other, shifted), (dense, pitched)):
        assert call(dense, X, R) == -6, (X.stride(), R.stride())
    if not torch.cuda.is_available():  # these get as far as the device, which must not be given host memory
        for H, X, R, T in ((dense, dense, other, 4), (dense, other, dense, 4), (dense, dense, dense, 4), (other, pitched, shifted, 4),
                           (dense[:1], pitched[:1], other[:1], 1)):
            assert call(H, X, R, T) != -6


# ------------------------------------------------------------------ FP8DecoderLayer.from_layer
class Built(tg.FP8DecoderLayer):
    """What from_layer found in a layer, without quantising it (which needs a GPU)."""

    def __init__(self, weights, num_heads, num_kv_heads, head_dim, inv_freq, magnitude=1.0, **kwargs):
        torch.nn.Module.__init__(self)
        self.found = dict(kwargs, num_heads=num_heads, num_kv_heads=num_kv_heads)


def plain_layer(norm=torch.nn.RMSNorm, **attention):
    nn = torch.nn
    m = nn.Module()
    m.self_attn, m.mlp = nn.Module(), nn.Module()
    a, p = m.self_attn, m.mlp
    a.q_proj, a.k_proj, a.v_proj, a.o_proj = (nn.Linear(256, n, bias=False) for n in (256, 128, 128, 256))
    p.gate_proj, p.up_proj, p.down_proj, p.act_fn = nn.Linear(256, 512, bias=False), nn.Linear(256, 512, bias=False), nn.Linear(512, 256, bias=False), nn.SiLU()
    m.input_layernorm, m.post_attention_layernorm = norm(256, eps=1e-6), norm(256, eps=1e-6)
    for name, value in attention.items():
        setattr(a, name, value)
    return m


def built(layer, **kwargs):
    return Built.from_layer(layer, 64, torch.ones(32, dtype=torch.float64), **kwargs).found


class Config:
    def __init__(self, **values):
        self.__dict__.update(values)


def test_layer_takes_over_the_sliding_window():
    """Where a layer keeps its window: on the attention, or in the model's configuration, for every layer or for some."""
    assert built(plain_layer()).get("window", 0) == 0
    assert built(plain_layer(sliding_window=None, config=Config(sliding_window=512))).get("window", 0) == 0
    assert built(plain_layer(sliding_window=512))["window"] == 512
    assert built(plain_layer(config=Config(sliding_window=4096)))["window"] == 4096
    assert built(plain_layer(config=Config(sliding_window=None))).get("window", 0) == 0
    assert built(plain_layer(config=Config(sliding_window=64, use_sliding_window=False))).get("window", 0) == 0
    kinds = Config(sliding_window=64, layer_types=["full_attention", "sliding_attention"])
    assert built(plain_layer(config=kinds, layer_idx=0)).get("window", 0) == 0
    assert built(plain_layer(config=kinds, layer_idx=1))["window"] == 64
    # what the caller says holds
    assert built(plain_layer(sliding_window=512), window=128, sinks=4)["window"] == 128
    assert built(plain_layer(sliding_window=512), window=0)["window"] == 0
    with pytest.raises(NotImplementedError, match="chunked_attention"):
        built(plain_layer(config=Config(layer_types=["chunked_attention"]), layer_idx=0))


def test_layer_takes_over_the_window_of_real_layers():
    transformers = pytest.importorskip("transformers")
    size = dict(hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, vocab_size=16)
    mistral = transformers.MistralModel(transformers.MistralConfig(sliding_window=48, **size))
    qwen = transformers.Qwen2Model(transformers.Qwen2Config(use_sliding_window=True, sliding_window=32, max_window_layers=1, **size))
    llama = transformers.LlamaModel(transformers.LlamaConfig(**size))
    assert [built(m).get("window", 0) for m in mistral.layers] == [48, 48]
    assert [built(m).get("window", 0) for m in qwen.layers] == [0, 32]
    assert [built(m).get("window", 0) for m in llama.layers] == [0, 0]


class Shifted(torch.nn.RMSNorm):
    """A norm whose weight counts from one."""

    def forward(self, x):
        return torch.nn.functional.rms_norm(x, (x.shape[-1],), self.weight + 1, self.eps)


def test_layer_refuses_what_it_would_compute_otherwise():
    nn = torch.nn

    def with_(owner, **values):
        layer = plain_layer()
        for name, value in values.items():
            setattr({"layer": layer, "attention": layer.self_attn, "mlp": layer.mlp}[owner], name, value)
        return layer

    built(plain_layer())
    for name in ("query_layernorm", "key_layernorm", "q_layernorm", "k_layernorm"):
        with pytest.raises(NotImplementedError, match=name):
            built(with_("attention", **{name: nn.RMSNorm(64)}))
    for owner, name, value, harmless in (("layer", "residual_multiplier", 0.22, 1.0), ("layer", "use_parallel_residual", True, False),
                                         ("attention", "use_rope", 0, 1), ("attention", "clip_qkv", 8.0, None)):
        with pytest.raises(NotImplementedError, match=name):
            built(with_(owner, **{name: value}))
        built(with_(owner, **{name: harmless}))
    with pytest.raises(NotImplementedError, match="clip_qkv"):
        built(plain_layer(config=Config(clip_qkv=8.0)))


def test_layer_refuses_norms_of_another_kind():
    nn = torch.nn
    with pytest.raises(NotImplementedError, match="input_layernorm"):
        built(plain_layer(nn.LayerNorm))
    with pytest.raises(NotImplementedError, match="input_layernorm"):
        built(plain_layer(Shifted))
    assert built(plain_layer(Shifted), weight_offset=1.0)["weight_offset"] == 1.0
    # an epsilon that is not the first norm's; one that the caller passes holds
    layer = plain_layer()
    layer.post_attention_layernorm.eps = 1e-3
    with pytest.raises(NotImplementedError, match="post_attention_layernorm"):
        built(layer)
    assert built(layer, eps=1e-4)["eps"] == 1e-4
    for dtype in (torch.bfloat16, torch.float16):
        assert built(plain_layer().to(dtype))["eps"] == 1e-6
    # a holder of weights that cannot be called is taken as an RMS norm
    layer = plain_layer()
    layer.input_layernorm = nn.Module()
    layer.input_layernorm.weight, layer.input_layernorm.eps = nn.Parameter(torch.ones(256)), 1e-5
    layer.post_attention_layernorm.eps = 1e-5
    assert built(layer)["eps"] == 1e-5


# ------------------------------------------------------------------ the extension is optional
@pytest.fixture
def bind_build(tmp_path, monkeypatch):
    """The build module with nothing to compile but the extension, into a folder of its own, by a compiler that the test plays."""
    import types

    from tilegym_b200 import build

    for name, path in (("LIB_PATH", "lib.so"), ("BIND_PATH", "_bind.so")):
        monkeypatch.setattr(build, name, str(tmp_path / path))
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path / "build"))
    monkeypatch.setattr(build, "SOURCES", [])
    (tmp_path / "lib.so").write_bytes(b"")
    calls, result = [], types.SimpleNamespace(returncode=0, stdout="", stderr="no such header")

    def run(cmd, **_):
        calls.append(cmd)
        if result.returncode == 0:
            (tmp_path / "_bind.so").write_bytes(b"built")
        return result

    monkeypatch.setattr(build.subprocess, "run", run)
    return build, calls, result, tmp_path / "_bind.so"


def test_build_goes_on_without_the_extension(bind_build, capsys):
    """Where torch's headers or g++ are missing the library is built all the same, and an extension of an older build, which may
    call it otherwise, is not left beside it."""
    build, calls, result, bind = bind_build
    bind.write_bytes(b"old")
    result.returncode = 1
    assert build.build(force=False) == build.LIB_PATH
    assert len(calls) == 1 and not bind.exists()
    assert "without" in capsys.readouterr().err


def test_extension_is_rebuilt_for_another_torch(bind_build, monkeypatch):
    build, calls, _, bind = bind_build
    build.build()
    assert len(calls) == 1 and bind.exists()
    build.build()
    assert len(calls) == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.build()
    assert len(calls) == 2


def test_extension_of_another_torch_is_not_called(monkeypatch):
    import types

    fake = types.SimpleNamespace(torch_version="9.9.9")
    assert _lib.usable_extension(fake) is None and _lib.usable_extension(None) is None
    fake.torch_version = torch.__version__
    assert _lib.usable_extension(fake) is fake
    assert _lib.fast is None or _lib.fast.torch_version == torch.__version__


# ------------------------------------------------------------------ derivatives
def test_operators_have_no_forward_derivative_either():
    from torch.autograd import forward_ad

    from tilegym_b200 import ops

    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(2, 128), torch.ones(2, 128))
        with pytest.raises(RuntimeError, match="no backward"):
            ops._no_grad_inputs(None, x)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no backward"):  # which has no say in tangents
            ops._no_grad_inputs(x)
        ops._no_grad_inputs(torch.zeros(2, 128), forward_ad.unpack_dual(x).primal)
    ops._no_grad_inputs(torch.zeros(2, 128))


# ------------------------------------------------------------------ outputs in the place of inputs
def test_outputs_in_the_place_of_inputs_lie_as_they_do():
    """apply_rope and paged_attention may write over what they read where every head lies on itself; the same memory under other
    pitches would be read by one warp or block after another has written it."""
    L = _lib.lib()
    memory = torch.zeros(4 * 4 * 64, dtype=BF)
    q = memory.view(4, 4, 64)
    other = memory.as_strided((4, 4, 64), (64, 256, 1))  # heads in front of tokens
    pos, f = torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    spare = torch.zeros(4, 4, 64, dtype=BF)

    def rope(Qo, Q, Ko=None, K=None):
        return L.tg_apply_rope(_d(Qo), _d(Ko), _d(Q), _d(K), _d(pos), _d(f), 0, 1.0, 0, 0)

    c = tg.FP8KVCache.empty(4, 4, 64, device="cpu")
    table, lens = torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, dtype=torch.int32)

    def attend(O, Q):
        return L.tg_paged_attention(_d(O), _d(Q), *map(_d, c), _d(table), _d(lens), None, 1, 0.125, 0, 0, 0, 0, 0, 0)

    assert rope(other, q) == -6 and rope(spare, spare, other, q) == -6
    assert attend(other, q) == -6
    if not torch.cuda.is_available():  # these get as far as the device
        assert rope(q, q) != -6 and rope(spare, q, q, q) != -6 and attend(q, q) != -6 and attend(other, other) != -6
