"""The 8-bit dense layer built from the strix ops: norm (with the residual's addition)
into 8 bits, the W8A8 products, the gated activation into 8 bits, and the MLP that runs
them one after the other.

Two forms, by what the weights are: FP8 (e4m3, one fp32 scale per 128 x 128 block;
activations e4m3 with one per (row, 128 columns)) and int8 (one scale per output
channel; activations int8 with one per row). In the reference the linear layers take
16-bit activations and quantise inside (csrc/gemm/w8a8_wmma_gemm.hip:508-529,
python/strix_vllm/fp8.py:121-262), with vLLM's 16-bit norm and silu_and_mul between.
"""

from __future__ import annotations

import torch
from torch import Tensor, is_grad_enabled
from torch.autograd import forward_ad
from torch.compiler import is_compiling
from torch.nn import Parameter

from . import torch_ops

try:   # not part of torch's public interface: without them every call takes the dispatcher
    from torch._C import _are_functorch_transforms_active, _is_tracing, _len_torch_dispatch_stack
except ImportError:
    _are_functorch_transforms_active = None

FP8 = torch.float8_e4m3fn


def _plain(*tensors) -> bool:
    """Whether a call on these operands (None: absent) is an ordinary one: no tracer's or
    other dispatch mode, no torch.func transform, no subclass among them (fake tensors,
    wrappers) and no derivative asked for. The operators have none: with requires_grad the
    dispatcher attaches a node that warns in the backward pass, and a forward-mode tangent
    would be lost without a word there too, so it is refused here."""
    if (_are_functorch_transforms_active is None or _are_functorch_transforms_active()
            or _len_torch_dispatch_stack() or _is_tracing()):
        return False
    for t in tensors:
        if t is not None and (type(t) is not Tensor and type(t) is not Parameter
                              or t.requires_grad and is_grad_enabled()):
            return False
    return True


def _refuse_tangents(*tensors) -> None:
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the 8-bit dense layer has no forward-mode derivative")


def _eager(first, *others) -> bool:
    """Whether a call may go to the op's implementation without the dispatcher (4 us of
    a call's 26, more than the smallest kernels run): plain CUDA tensors only, and CUDA
    as the first operand says (the implementation checks that the others are with it).
    Anything else takes torch.ops.strix, with its shape inference and errors."""
    if is_compiling():
        return False
    if getattr(forward_ad, "_current_level", 0) >= 0:   # a dual level is open
        _refuse_tangents(first, *others)
    return first.is_cuda and _plain(first, *others)


def _is_fp8(q_dtype: torch.dtype) -> bool:
    if q_dtype not in (FP8, torch.int8):
        raise RuntimeError(f"q_dtype must be float8_e4m3fn or int8, got {q_dtype}")
    return q_dtype == FP8


def rms_norm_quant(x, weight, eps: float = 1e-6, residual=None, residual_out=None, q_dtype=FP8):
    """(q, scales) of rms_norm(x + residual) * weight.

    x, residual: [M, K] bf16 / fp16; weight [K] of the same dtype or fp32. residual_out
    receives x + residual rounded to x's dtype: a tensor of its own, or x or residual
    itself for an update in place. The norm is taken of the fp32 sum, before that
    rounding. q_dtype float8_e4m3fn: scales fp32 [M, ceil(K / 128)], K a multiple of 16;
    int8: scales fp32 [M], K a multiple of 8. Scales and quotients are within a few fp32
    steps of amax / 448 (127) and y / scale."""
    fp8 = _is_fp8(q_dtype)
    if _eager(x, weight, residual, residual_out):
        return torch_ops._rms_norm_quant(x, weight, eps, residual, residual_out, fp8)
    ops = torch.ops.strix
    return (ops.rms_norm_quant_fp8 if fp8 else ops.rms_norm_quant_token_i8)(x, weight, eps, residual, residual_out)


def act_mul_quant(x, activation: str = "silu", q_dtype=FP8):
    """(q, scales) of act(x[:, :K]) * x[:, K:] for x [M, 2 K] (bf16, fp16 or fp32),
    activation silu or gelu_tanh; q and scales as rms_norm_quant returns them."""
    fp8 = _is_fp8(q_dtype)
    if _eager(x):
        return torch_ops._act_mul_quant(x, activation, fp8)
    ops = torch.ops.strix
    return (ops.act_mul_quant_fp8 if fp8 else ops.act_mul_quant_token_i8)(x, activation)


def fp8_gemm(a_q, a_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16):
    """[M, N] of a_q e4m3 [M, K] (a_scale fp32 [M, ceil(K / 128)]) and w e4m3 [N, K]
    (w_scale fp32 [ceil(N / 128), ceil(K / 128)]), K a multiple of 16. The two scales of a
    block are multiplied first, in fp32: their product has to be a normal number."""
    ns = torch_ops if _eager(a_q, a_scale, w, w_scale, bias) else torch.ops.strix
    return ns.w8a8_fp8_gemm(a_q, a_scale, w, w_scale, bias, out_dtype)


def fp8_gemm_act_mul_quant(a_q, a_scale, w, w_scale, activation: str = "silu"):
    """(q e4m3 [M, N], scales) of act(gate) * up, where w e4m3 [2 N, K] holds the gate
    rows and then the up rows: fp8_gemm and act_mul_quant without the 16-bit rows
    between them."""
    ns = torch_ops if _eager(a_q, a_scale, w, w_scale) else torch.ops.strix
    return ns.w8a8_fp8_gemm_act_mul_quant(a_q, a_scale, w, w_scale, activation)


def fused_mlp_fp8_w8a8(x, norm_weight, w13, w13_scale, w2, w2_scale, eps: float = 1e-6, residual=None,
                       residual_out=None, activation: str = "silu"):
    """One MLP block in FP8 W8A8: norm (x + residual) -> gate-up product with the gate
    -> down product. x [T, H] bf16 / fp16; w13 e4m3 [2 I, H], w2 e4m3 [H, I] with fp32
    128 x 128 block scales. Returns [T, H] of x's dtype (the residual stream's increment;
    the stream itself is residual_out)."""
    q, s = rms_norm_quant(x, norm_weight, eps, residual, residual_out)
    q, s = fp8_gemm_act_mul_quant(q, s, w13, w13_scale, activation)
    return fp8_gemm(q, s, w2, w2_scale, None, x.dtype)


def fused_mlp_int8_w8a8(x, norm_weight, w13, w13_scale, w2, w2_scale, eps: float = 1e-6, residual=None,
                        residual_out=None, activation: str = "silu"):
    """The same block over int8 weights [2 I, H] and [H, I] with one fp32 scale per output
    channel (H and I multiples of 128). Returns [T, H] of x's dtype. w8a8_int8_gemm rounds
    to bf16, so under fp16 the increment has bf16's eight significant bits."""
    q, s = rms_norm_quant(x, norm_weight, eps, residual, residual_out, torch.int8)
    h = torch.ops.strix.w8a8_int8_gemm(q, s, w13, w13_scale)
    q, s = act_mul_quant(h, activation, torch.int8)
    out = torch.ops.strix.w8a8_int8_gemm(q, s, w2, w2_scale)
    return out if x.dtype == torch.bfloat16 else out.to(x.dtype)
