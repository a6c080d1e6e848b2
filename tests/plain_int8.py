"""8-bit rows and their products in 64 bits, for the tests of csrc/rows_int8.cu and csrc/linear_int8.cu."""

import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, of the value
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # a step next to zero


def normed(x, residual, weight, eps):
    s = x.double() + (residual.double() if residual is not None else 0.0)
    return s / (s.pow(2).mean(1, keepdim=True) + eps).sqrt() * weight.double()


def gated(gate_up, act):
    """(act(gate) * up, the activation's exponent) of rows [gate | up]."""
    g, u = gate_up.double().chunk(2, dim=1)
    z = g if act == 0 else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g.pow(3))
    return g * torch.sigmoid(z) * u, z


def check_rows(q, scales, y, rel, scale_rel):
    """8-bit rows against the 64-bit rows y that they hold.  `rel`: how far a 32-bit element may be off before it is rounded, of its
    value; `scale_rel`: the same of a scale.  An element is the nearest whole multiple of y's own scale, or the other neighbour where
    32 bits cannot tell."""
    most = y.abs().amax(1)
    step = most / 127
    assert ((scales.double() - step).abs() <= scale_rel * step + 2.0 ** -149).all(), ((scales.double() - step).abs() / step).max()
    held = torch.where(step[:, None] > 0, y / step[:, None], 0.0)
    top = torch.where(step[:, None] > 0, rel.amax(1, keepdim=True) if torch.is_tensor(rel) else rel, 0.0)
    # its own error, the largest element's (the step goes by it), the quotient 127 / max and its product
    off = (q.double() - held).abs() - (0.5 + held.abs() * (rel + top + 2.0 ** -23))
    assert (off <= 0).all(), (off.max(), (off > 0).sum())
    assert int(q.int().abs().max()) <= 127


def product(x, x_scales, w, w_scales, bias=None):
    """(result, size of its product term) in 64 bits: sums of whole numbers below 2^53 are exact."""
    p = (x.double() @ w.double().t()) * x_scales.double()[:, None] * w_scales.double()
    return (p if bias is None else p + bias.double()), p.abs()


def check_product(got, ref, size):
    """The sum becomes a float32 and meets a scale (two roundings of the product), the other scale and the bias in one rounding, then
    the type's."""
    dt = got.dtype
    limit = size * 2 * 2.0 ** -24 * 1.01 + ref.abs() * (2.0 ** -24 + (HALF[dt] if dt != torch.float32 else 0.0)) * 1.01 + TINY[dt]
    err = (got.double() - ref).abs()
    assert (err <= limit).all(), f"{int((err > limit).sum())} of {err.numel()} results off, up to {float((err / limit).max()):.2f} of the limit"


class HeldMatrix:
    """A weight in 8 bits as the plain model's products meet it: h @ W.T with W's rows and h's as the values that they are held as."""

    def __init__(self, w):
        self.held = held(w)

    @property
    def T(self):
        return self

    def __rmatmul__(self, h):
        return held(h) @ self.held.T


def held(y):
    step = y.abs().amax(-1, keepdim=True) / 127
    return torch.where(step > 0, torch.round(y / step) * step, 0.0)


def held_weights(w):
    """The plain model's weights with the layers' matrices in 8 bits."""
    return {n: HeldMatrix(t.double()) if n.endswith("_proj.weight") else t.double() for n, t in w.items()}
