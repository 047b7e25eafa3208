"""CPU oracle of the 8-bit dense layer, in 64 bits - TEST INFRASTRUCTURE, not product
code. The reference has no counterpart of these steps in torch (vLLM's norm and
silu_and_mul run there in 16 bits, and its GEMMs quantise their own activations), so
the formulas are restated here: parity unpinned."""

from __future__ import annotations

import math

import torch

TINY = 2.0 ** -126        # the smallest normal fp32: a scale below it is 1


def group_scales(y: torch.Tensor, top: float, group: int) -> torch.Tensor:
    """[M, ceil(K / group)] of amax / top; NaN and infinities show in the scale."""
    m, k = y.shape
    pad = -k % group
    b = torch.cat([y, y.new_zeros(m, pad)], 1).view(m, -1, group).abs()
    amax = b.amax(-1)                      # torch's amax hands a NaN on
    s = amax / top
    return torch.where(s < TINY, torch.ones_like(s), s)


def spread(s: torch.Tensor, k: int, group: int) -> torch.Tensor:
    return s.repeat_interleave(group, 1)[:, :k]


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value (ties to even, saturating), in 64 bits; NaN stays."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), e.clamp_min(-5) - 4)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def rms_norm(x, weight, eps, residual=None):
    """(sum, y) in 64 bits."""
    s = x.double() if residual is None else x.double() + residual.double()
    return s, s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * weight.double()


def act_mul(x, activation):
    k = x.size(1) // 2
    g, u = x[:, :k].double(), x[:, k:].double()
    if activation == "silu":
        return g * torch.sigmoid(g) * u
    t = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    return 0.5 * g * (1 + torch.tanh(t)) * u


def quantise(y, fp8: bool):
    """(quotients y / scale, scales): [M, ceil(K / 128)] for e4m3, [M] for int8."""
    if fp8:
        s = group_scales(y, 448.0, 128)
        return y / spread(s, y.size(1), 128), s
    s = group_scales(y, 127.0, y.size(1))
    return y / s, s[:, 0]


def fp8_gemm(a_q, a_scale, w, w_scale, bias=None):
    """64-bit product of the dequantised operands."""
    n, k = w.shape
    a = a_q.double() * spread(a_scale.double(), k, 128)
    b = w.double() * spread(w_scale.double(), k, 128).repeat_interleave(128, 0)[:n]
    out = a @ b.t()
    return out if bias is None else out + bias.double()
