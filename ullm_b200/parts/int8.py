"""Parts whose matrices are held in 8 bits: a pre-norm decoder layer of grouped-query attention and a gated feed-forward, as
`prenorm_residual`, `paged_attention` and `gated_mlp` are, with every product's operands in 8 bits (csrc/rows_int8.cu,
csrc/linear_int8.cu).

A matrix [N, K] of the checkpoint becomes whole numbers with a scale per output channel when the weights are there; the rows in front of
a product get a scale per token in the kernel that makes them (the norm, the gated activation, or a kernel of its own behind the
attention).  Products are exact in 32 bits; what they leave, the residual stream, the attention and its cache keep the engine's dtype.
A row that is not finite makes its own token's results NaN and no other's.

`EngineConfig(quantization="int8")` builds a model of these (config/int8.py).  The reference has no quantized weights.
"""

from __future__ import annotations

import torch

from ..csrc import kernels
from .attention import PagedAttention
from .base import Block
from .block import PreNormResidualBlock
from .mlp import GatedMLP
from .norm import RMSNorm
from .registry import register_block, register_feed_forward, register_mixer


class Int8Rows:
    """Rows in 8 bits with a scale each, in the step's workspace.  `dtype`: the type of the rows that they stand for."""

    def __init__(self, ctx, name: str, rows: int, cols: int, dtype: torch.dtype):
        ws, wide = ctx.workspace, -(-cols // 16) * 16  # (rows on borders of 16 bytes)
        q = ws.tokens(name, rows, wide, torch.int8)
        self.q = q if wide == cols else q[:, :cols]
        self.scales = ws.tokens(name + ".scales", rows, 1, torch.float32).view(rows)
        self.shape, self.dtype = (rows, cols), dtype

    def times(self, weight: "Int8Matrix", out, bias=None):
        """out = these rows . weight^T (+ bias)"""
        kernels().linear_int8(self.q, self.scales, weight.q, weight.scales, out, bias)
        return out


class Int8Matrix:
    """A matrix [N, K] in 8 bits with a scale per row."""

    def __init__(self, weight: torch.Tensor):
        K = kernels()
        self.shape, self.dtype, self.device = tuple(weight.shape), weight.dtype, weight.device
        self.q = K.int8_rows(*weight.shape, device=weight.device)
        self.scales = torch.empty(weight.shape[0], dtype=torch.float32, device=weight.device)
        K.quantize_rows_int8(weight, self.q, self.scales)


@register_feed_forward("gated_mlp_int8")
class Int8GatedMLP(GatedMLP):
    """down(act(gate(x)) * up(x)) with both matrices, x (`Int8Rows`) and the activated rows in 8 bits."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        if self.activation not in ("silu", "gelu_tanh"):
            raise ValueError(f"activation {self.activation!r}: the 8-bit feed-forward has silu and gelu_tanh")

    def weights_loaded(self):
        n = self.names
        self.w_gate_up = Int8Matrix(self.w_gate_up)
        self.w_down = Int8Matrix(self.tensors[n["down"]])
        for name in (n["gate"], n["up"], n["down"]):
            del self.tensors[name]  # (the matrices as they came are let go of here)

    def gated_weights(self):
        return None

    def forward(self, x, ctx):
        T, I = x.shape[0], self.intermediate_size
        gu = x.times(self.w_gate_up, ctx.workspace.tokens("mlp.gate_up", T, 2 * I, x.dtype))
        rows = Int8Rows(ctx, "mlp.act8", T, I, x.dtype)
        kernels().act_mul_int8(gu, rows.q, rows.scales, 0 if self.activation == "silu" else 1)
        return rows.times(self.w_down, ctx.workspace.tokens("ffn.out", T, self.hidden_size, x.dtype))


@register_mixer("paged_attention_int8")
class Int8PagedAttention(PagedAttention):
    """Paged attention whose projections are products of 8-bit operands; x is `Int8Rows`.  Only the plain form (no option of the
    general path, keys and values of its own)."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        if self.general or not self.own_kv:
            raise ValueError("8-bit projections go with plain attention only (no convolution, cap, mixing, gate, bias by distance, "
                             "norm of whole rows or borrowed keys)")

    def weights_loaded(self):
        super().weights_loaded()
        n = self.names
        self.w_qkv = Int8Matrix(self.w_qkv)
        self.w_o = Int8Matrix(self.tensors[n["o"]])
        for name in (n["q"], n["k"], n["v"], n["o"]):
            del self.tensors[name]

    def takes_input_norm(self):
        return False

    def output_projection(self):
        return None

    def activation_elems(self):
        return super().activation_elems() + self.o_size

    def _project(self, attn, ctx, project_output: bool, out=None):
        if not project_output:
            raise NotImplementedError("an output projection of 8-bit operands that the caller makes")
        rows = Int8Rows(ctx, "attn.out8", *attn.shape, attn.dtype)
        kernels().quantize_rows_int8(attn, rows.q, rows.scales)
        if out is None:
            out = ctx.workspace.tokens("mixer.out", attn.shape[0], self.hidden_size, attn.dtype)
        return rows.times(self.w_o, out, self.w_o_bias)


@register_block("prenorm_residual_int8")
class PreNormResidualInt8Block(Block):
    """`prenorm_residual` for an 8-bit mixer and feed-forward: its two RMSNorms leave their rows in 8 bits."""

    def __init__(self, mixer, feed_forward, mixer_norm, feed_forward_norm, names=None):
        super().__init__()
        if not isinstance(mixer_norm, RMSNorm) or not isinstance(feed_forward_norm, RMSNorm):
            raise ValueError("a block of 8-bit products takes RMSNorms")
        self.mixer, self.feed_forward = mixer, feed_forward
        self.mixer_norm, self.feed_forward_norm = mixer_norm, feed_forward_norm
        self.names = PreNormResidualBlock(mixer, feed_forward, mixer_norm, feed_forward_norm, names).names

    subparts = PreNormResidualBlock.subparts
    activation_elems = PreNormResidualBlock.activation_elems

    def forward(self, x, residual, ctx, cache):
        """As `PreNormResidualBlock.forward`: x is what is still to be added to the stream (the embedding, with residual None, for
        the first block); returns (feed-forward output, residual)."""
        first = residual is None
        T, H = x.shape
        h = Int8Rows(ctx, "block.normed8", T, H, x.dtype)
        K = kernels()
        weight, eps = self.mixer_norm.rms_params()
        K.add_rmsnorm_int8(x, None if first else residual, weight, eps, h.q, h.scales)
        if first:
            residual = x
        a = self.mixer.forward(h, ctx, cache)
        weight, eps = self.feed_forward_norm.rms_params()
        K.add_rmsnorm_int8(a, residual, weight, eps, h.q, h.scales)
        return self.feed_forward.forward(h, ctx), residual
