"""FP8DecoderLayer: a pre-norm decoder layer that runs on the FP8 GEMMs from its input to its output.

    norm 1     rms_norm_quant             residual added, normed, quantised 1 x 128 in one pass
    qkv        block-scaled GEMM          one fused weight
    cache      kv_cache_write             keys and queries rotated, keys and values quantised into their pages
    attention  paged_attention            over the 8-bit cache, new tokens included
    o_proj     act_quant + block-scaled GEMM
    norm 2     rms_norm_quant
    gate / up  block-scaled GEMM          one fused weight
    silu * mul with the 1 x 128 quantiser (the pass of the mixture-of-experts layer, with one group)
    down       block-scaled GEMM

Weights are quantised once in 128 x 128 blocks.  The layer is called with the pair (hidden, residual) that the norm's
fused addition makes natural: what a layer returns is the input of the next one, and hidden + residual after the last is
the residual stream.  Prompts, drafts and single tokens take the same call; nothing is read back to the host, so a decode
step can be captured into a CUDA graph (after a first GEMM call outside of it, like every GEMM here).
"""

from __future__ import annotations

from typing import Dict, Optional, Tuple

import torch
from torch import nn

from . import _lib, ops
from .attention import FP8KVCache, kv_cache_write, paged_attention

_FP8 = torch.float8_e4m3fn


def _refuse_other_layers(layer: nn.Module, head_dim: int) -> None:
    """Layers that compute something else with the same projections would come out wrong without a word."""
    att, mlp = layer.self_attn, layer.mlp
    for owner, names in ((att, ("q_norm", "k_norm", "query_layernorm", "key_layernorm", "q_layernorm", "k_layernorm", "sinks",
                                "attn_logit_softcapping", "clip_qkv")),
                         (getattr(att, "config", None), ("clip_qkv",)),
                         (layer, ("pre_feedforward_layernorm", "post_feedforward_layernorm"))):
        for name in names:
            if getattr(owner, name, None) is not None:
                raise NotImplementedError(f"FP8DecoderLayer does not implement {name}")
    if getattr(layer, "residual_multiplier", 1.0) != 1.0:
        raise NotImplementedError("FP8DecoderLayer does not implement a residual_multiplier")
    if getattr(layer, "use_parallel_residual", False):
        raise NotImplementedError("FP8DecoderLayer does not implement use_parallel_residual")
    if not getattr(att, "use_rope", True):
        raise NotImplementedError("FP8DecoderLayer rotates queries and keys: the layer's use_rope is off")
    scaling = getattr(att, "scaling", None)
    if scaling is not None and abs(scaling * head_dim**0.5 - 1.0) > 1e-6:
        raise NotImplementedError(f"FP8DecoderLayer scales scores by head_dim^-0.5, not by {scaling}")
    act = getattr(mlp, "act_fn", None)
    probe = torch.linspace(-4.0, 4.0, 9)
    if act is not None and not torch.allclose(act(probe), nn.functional.silu(probe), atol=1e-6):
        raise NotImplementedError("FP8DecoderLayer takes an MLP with silu")


def _refuse_other_norms(layer: nn.Module, eps: float, eps_given: bool, weight_offset: float) -> None:
    """The layer's norms are tried on two rows, ordinary values and ones whose squares are as small as eps."""
    for name in ("input_layernorm", "post_attention_layernorm"):
        norm = getattr(layer, name)
        if not callable(norm) or getattr(type(norm), "forward", None) is nn.Module.forward:
            continue  # holds a weight and nothing else
        w = norm.weight.detach()
        x = torch.linspace(0.5, 2.0, w.numel(), device=w.device)  # a mean that is not zero
        rows = torch.stack((x, x * (eps**0.5 if eps > 0 and not eps_given else 1.0))).to(w.dtype)
        f = rows.float()
        want = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + eps) * (w.float() + weight_offset)
        with torch.no_grad():
            got = norm(rows).float()
        # two roundings to 16 bits
        if got.shape != want.shape or not torch.allclose(got, want, rtol=2.0**-6, atol=1e-6):
            raise NotImplementedError(f"{name} is not an RMS norm of weight + {weight_offset} and eps {eps}")


def _window_of(layer: nn.Module) -> int:
    """The layer's sliding window (0: none): on its attention, or in the model's configuration for the layers that use it."""
    att = layer.self_attn
    config = getattr(att, "config", None)
    kinds, index = getattr(config, "layer_types", None), getattr(att, "layer_idx", None)
    kind = kinds[index] if kinds and index is not None else None
    if kind not in (None, "full_attention", "sliding_attention"):
        raise NotImplementedError(f"FP8DecoderLayer does not implement {kind}")
    if hasattr(att, "sliding_window"):
        window = att.sliding_window
    elif kind == "full_attention" or not getattr(config, "use_sliding_window", True):
        window = None
    else:
        window = getattr(config, "sliding_window", None)
    return 0 if window is None else int(window)


class FP8DecoderLayer(nn.Module):
    """Built by `from_layer` from a layer with `input_layernorm`, `self_attn.{q,k,v,o}_proj`, `post_attention_layernorm` and
    `mlp.{gate,up,down}_proj` (Llama, Mistral, Qwen2, ...).  Hidden and intermediate sizes must be multiples of 128,
    head_dim 64 or 128."""

    def __init__(self, weights: Dict[str, torch.Tensor], num_heads: int, num_kv_heads: int, head_dim: int, inv_freq: torch.Tensor,
                 magnitude: float = 1.0, interleaved: bool = False, eps: float = 1e-6, weight_offset: float = 0.0,
                 window: int = 0, sinks: int = 0, qkv_bias: Optional[torch.Tensor] = None, o_bias: Optional[torch.Tensor] = None):
        """weights: norm1, norm2 (hidden,), qkv ((num_heads + 2 num_kv_heads) * head_dim, hidden), o, gate_up (2 I, hidden:
        gate rows, then up rows), down, on a CUDA device.  inv_freq, magnitude: see `rope_frequencies`."""
        super().__init__()
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if num_heads % num_kv_heads != 0 or num_heads // num_kv_heads > 64:
            raise ValueError("num_heads must be a multiple of num_kv_heads, at most 64 times")
        hidden, inter = weights["norm1"].shape[0], weights["down"].shape[1]
        if hidden % 128 or inter % 128 or (num_heads * head_dim) % 128:
            raise ValueError("the hidden, intermediate and attention sizes must be multiples of 128 (the quantisation block)")
        want = {"norm1": (hidden,), "norm2": (hidden,), "qkv": ((num_heads + 2 * num_kv_heads) * head_dim, hidden),
                "o": (hidden, num_heads * head_dim), "gate_up": (2 * inter, hidden), "down": (hidden, inter)}
        for name, shape in want.items():
            if tuple(weights[name].shape) != shape:
                raise ValueError(f"{name} must be {shape}, got {tuple(weights[name].shape)}")
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.magnitude, self.interleaved, self.eps, self.weight_offset = magnitude, interleaved, eps, weight_offset
        self.window, self.sinks = window, sinks
        self.register_buffer("inv_freq", inv_freq.detach())
        with torch.no_grad():
            for name in ("norm1", "norm2"):
                self.register_buffer(name, weights[name].detach())
            for name in ("qkv", "o", "gate_up", "down"):
                q, s = ops.weight_quant_block(weights[name].detach())
                self.register_buffer(name, q)
                self.register_buffer(name + "_scale", s)
        self.register_buffer("qkv_bias", None if qkv_bias is None else qkv_bias.detach())
        self.register_buffer("o_bias", None if o_bias is None else o_bias.detach())

    @classmethod
    def from_layer(cls, layer: nn.Module, head_dim: int, inv_freq: torch.Tensor, magnitude: float = 1.0, eps: Optional[float] = None,
                   **kwargs) -> "FP8DecoderLayer":
        """Quantises a layer whose weights are on a CUDA device.  kwargs go to the constructor (window, sinks, ...); without
        `window` the layer's own is taken over."""
        att, mlp = layer.self_attn, layer.mlp
        _refuse_other_layers(layer, head_dim)
        kwargs.setdefault("window", _window_of(layer))
        parts = [att.q_proj, att.k_proj, att.v_proj]
        weights = {
            "norm1": layer.input_layernorm.weight, "norm2": layer.post_attention_layernorm.weight,
            "qkv": torch.cat([p.weight for p in parts]), "o": att.o_proj.weight,
            "gate_up": torch.cat([mlp.gate_proj.weight, mlp.up_proj.weight]), "down": mlp.down_proj.weight,
        }
        if any(p.bias is not None for p in (mlp.gate_proj, mlp.up_proj, mlp.down_proj)):
            raise NotImplementedError("FP8DecoderLayer takes an MLP without biases")
        if any((p.bias is None) != (parts[0].bias is None) for p in parts):
            raise NotImplementedError("q_proj, k_proj and v_proj must all have a bias or none")
        bias = None if parts[0].bias is None else torch.cat([p.bias for p in parts])
        eps_given = eps is not None
        if not eps_given:
            eps = getattr(layer.input_layernorm, "variance_epsilon", None) or getattr(layer.input_layernorm, "eps", None) or 1e-6
        _refuse_other_norms(layer, eps, eps_given, kwargs.get("weight_offset", 0.0))
        return cls(weights, att.q_proj.out_features // head_dim, att.k_proj.out_features // head_dim, head_dim, inv_freq, magnitude,
                   eps=eps, qkv_bias=bias, o_bias=att.o_proj.bias, **kwargs)

    def forward(
        self,
        hidden: torch.Tensor,
        residual: Optional[torch.Tensor],
        cache: FP8KVCache,
        block_table: torch.Tensor,
        seq_lens: torch.Tensor,
        cu_seqlens: Optional[torch.Tensor] = None,
        max_q_len: Optional[int] = None,
    ) -> Tuple[torch.Tensor, torch.Tensor]:
        """hidden, residual (tokens, hidden) bf16 or f16 (residual None: hidden starts the residual stream); tables as in
        `kv_cache_write`.  Writes this layer's `cache` and returns the next (hidden, residual)."""
        tokens = hidden.shape[0]
        if tokens == 0:
            return hidden, hidden if residual is None else residual
        dtype = hidden.dtype
        if residual is None:
            y, s = ops.rms_norm_quant(hidden, self.norm1, self.eps, weight_offset=self.weight_offset)
            residual = hidden
        else:
            y, s, residual = ops.rms_norm_quant(hidden, self.norm1, self.eps, residual=residual, weight_offset=self.weight_offset)
        qkv = ops.fp8_block_scaled_mm(y, self.qkv, s, self.qkv_scale, self.qkv_bias, dtype)
        qkv = qkv.view(tokens, self.num_heads + 2 * self.num_kv_heads, self.head_dim)
        q, k, v = qkv.split((self.num_heads, self.num_kv_heads, self.num_kv_heads), dim=1)
        q = kv_cache_write(cache, k, v, block_table, seq_lens, cu_seqlens, inv_freq=self.inv_freq, q=q, interleaved=self.interleaved,
                           magnitude=self.magnitude)
        o = paged_attention(q, cache, block_table, seq_lens, cu_seqlens, max_q_len=max_q_len, window=self.window, sinks=self.sinks)
        a8, a_s = ops.act_quant(o.view(tokens, -1), 128)
        attended = ops.fp8_block_scaled_mm(a8, self.o, a_s, self.o_scale, self.o_bias, dtype)
        y, s, residual = ops.rms_norm_quant(attended, self.norm2, self.eps, residual=residual, weight_offset=self.weight_offset)
        c = ops.fp8_block_scaled_mm(y, self.gate_up, s, self.gate_up_scale, None, dtype)
        inter = c.shape[1] // 2
        y8 = torch.empty((tokens, inter), dtype=_FP8, device=c.device)
        y_s = torch.empty((tokens, inter // 128), dtype=torch.float32, device=c.device)
        rows = torch.arange(0, tokens + 1, tokens, dtype=torch.int32, device=c.device)  # [0, tokens]: one range of rows
        _lib.check_rc(_lib.lib().tg_moe_silu_mul_quant(_lib.desc(y8), _lib.desc(y_s), _lib.desc(c), rows.data_ptr(), 1, 1, c.device.index,
                                                       ops._stream(c.device)))
        return ops.fp8_block_scaled_mm(y8, self.down, y_s, self.down_scale, None, dtype), residual

    def extra_repr(self) -> str:
        return f"heads={self.num_heads}, kv_heads={self.num_kv_heads}, head_dim={self.head_dim}, window={self.window}, sinks={self.sinks}"
