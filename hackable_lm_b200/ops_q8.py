"""PyTorch operators of the 8-bit path over the libhlm_b200 C ABI.

The 8-bit format (``include/hlm_b200.h``): a group of values v is int8 codes and
one fp32 scale, ``a = max(max|v|, 2^-110)``, ``q = rint(v * (127 / a))``,
``scale = a / 127``, ``v ~ q * scale``.  A group is a whole row, except in
``swiglu_ckpt8``.  A group with an infinity or a NaN has scale NaN and codes 0.

Every operator is a ``torch.library.custom_op`` with a fake implementation, as
in :mod:`hackable_lm_b200.ops`; its body is one call of the compiled binding
(``csrc/binding.cpp``: checks, output allocation, the library call).  The
functions of this module try that call first: on plain CUDA tensors outside
``torch.compile``, with no gradient asked for, nothing goes through the
dispatcher, which costs more than the kernels of a single token.  The binding
returns None for any other tensors, which then take the registered operator.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .ops import _code, _require_cuda

CKPT_GROUP = 128
_compiling = torch.compiler.is_compiling


def _run(what: str, *args):
    """The binding's function, for the registered operators: tensors it does not take are refused."""
    out = getattr(_lib.binding(), what)(*args)
    if out is None:
        _require_cuda(*(t for t in args if isinstance(t, torch.Tensor)))
        raise RuntimeError(f"{what}: needs plain strided CUDA tensors")
    return out


# The binding's argument checks, for the fake implementations (torch.compile, meta tensors).
def _check(ok: bool, message: str) -> None:
    if not ok:
        raise RuntimeError(message)


def _check_rows(what: str, q: torch.Tensor, scale: torch.Tensor) -> None:
    _check(q.dtype == torch.int8 and scale.dtype == torch.float32 and q.dim() >= 1 and scale.shape == q.shape[:-1],
           f"{what}: needs int8 codes [..., C] and their fp32 scales [...], got {q.dtype} {tuple(q.shape)} and "
           f"{scale.dtype} {tuple(scale.shape)}")


def _check_cols(what: str, x: torch.Tensor) -> None:
    _code(x.dtype)
    _check(x.dim() >= 1 and x.shape[-1] >= 1, f"{what}: needs at least one column, got shape {tuple(x.shape)}")


def _check_norm(what: str, x: torch.Tensor, weight: Optional[torch.Tensor]) -> None:
    _check_cols(what, x)
    _check(weight is None or weight.shape == x.shape[-1:], f"{what}: weight must be [{x.shape[-1]}]")


def _check_gate_up(what: str, t: torch.Tensor) -> int:
    _check(t.dim() >= 1 and t.shape[-1] % 2 == 0,
           f"{what}: the last dimension must be even (gate | up), got shape {tuple(t.shape)}")
    return t.shape[-1] // 2


# ---------------------------------------------------------------------------
# Rows to 8 bits and back
# ---------------------------------------------------------------------------
@torch.library.custom_op("hackable_lm_b200::quantize_rows", mutates_args=())
def _quantize_rows_op(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return _run("quantize_rows", x)


@_quantize_rows_op.register_fake
def _quantize_rows_fake(x):
    _check_cols("quantize_rows", x)
    return (torch.empty(x.shape, dtype=torch.int8, device=x.device),
            torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device))


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q int8 [..., C], scale fp32 [...]) of x [..., C]."""
    out = None if _compiling() else _lib.binding().quantize_rows(x)
    return _quantize_rows_op(x) if out is None else out


@torch.library.custom_op("hackable_lm_b200::dequantize_rows", mutates_args=())
def _dequantize_rows_op(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return _run("dequantize_rows", q, scale, _code(dtype))


@_dequantize_rows_op.register_fake
def _dequantize_rows_fake(q, scale, dtype):
    _check_rows("dequantize_rows", q, scale)
    _code(dtype)
    return torch.empty(q.shape, dtype=dtype, device=q.device)


def dequantize_rows(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """q * scale of each row, rounded to ``dtype``."""
    out = None if _compiling() else _lib.binding().dequantize_rows(q, scale, _code(dtype))
    return _dequantize_rows_op(q, scale, dtype) if out is None else out


# ---------------------------------------------------------------------------
# RMSNorm with an 8-bit output
# ---------------------------------------------------------------------------
@torch.library.custom_op("hackable_lm_b200::rms_norm_q8", mutates_args=())
def _rms_norm_q8_op(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    return _run("residual_rms_norm_q8", None, x, weight, eps)


@_rms_norm_q8_op.register_fake
def _rms_norm_q8_fake(x, weight, eps):
    _check_norm("rms_norm_q8", x, weight)
    return _quantize_rows_fake(x)


def rms_norm_q8(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of rms_norm(x) [* weight], by rows."""
    out = None if _compiling() else _lib.binding().residual_rms_norm_q8(None, x, weight, eps)
    return _rms_norm_q8_op(x, weight, eps) if out is None else out


@torch.library.custom_op("hackable_lm_b200::residual_rms_norm_q8", mutates_args=())
def _residual_rms_norm_q8_op(residual: torch.Tensor, branch: torch.Tensor, weight: Optional[torch.Tensor],
                             eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _run("residual_rms_norm_q8", residual, branch, weight, eps)


@_residual_rms_norm_q8_op.register_fake
def _residual_rms_norm_q8_fake(residual, branch, weight, eps):
    _check_norm("residual_rms_norm_q8", branch, weight)
    _check(residual.shape == branch.shape and residual.dtype == branch.dtype,
           "residual_rms_norm_q8: residual and branch must match in shape and dtype")
    return (torch.empty(branch.shape, dtype=branch.dtype, device=branch.device), *_quantize_rows_fake(branch))


def residual_rms_norm_q8(residual: torch.Tensor, branch: torch.Tensor, weight: Optional[torch.Tensor],
                         eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(out, q, scale): out = residual + branch, and rms_norm(out) [* weight] in 8 bits by rows."""
    out = None if _compiling() else _lib.binding().residual_rms_norm_q8(residual, branch, weight, eps)
    return _residual_rms_norm_q8_op(residual, branch, weight, eps) if out is None else out


# ---------------------------------------------------------------------------
# 8-bit integer projection
# ---------------------------------------------------------------------------
@torch.library.custom_op("hackable_lm_b200::linear_q8", mutates_args=())
def _linear_q8_op(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                  out_dtype: torch.dtype) -> torch.Tensor:
    return _run("linear_q8", q, scale, weight, weight_scale, _code(out_dtype))


@_linear_q8_op.register_fake
def _linear_q8_fake(q, scale, weight, weight_scale, out_dtype):
    _check_rows("linear_q8", q, scale)
    _check_rows("linear_q8 (weight)", weight, weight_scale)
    _code(out_dtype)
    _check(weight.dim() == 2 and weight.shape[1] == q.shape[-1],
           f"linear_q8: weight must be [N, {q.shape[-1]}], got {tuple(weight.shape)}")
    return torch.empty((*q.shape[:-1], weight.shape[0]), dtype=out_dtype, device=q.device)


def linear_q8(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """(q * scale) @ (weight * weight_scale)^T with exact integer sums: q int8 [..., K] with a
    scale for each token, weight int8 [N, K] with a scale for each output channel; K a
    multiple of 16."""
    out = None if _compiling() else _lib.binding().linear_q8(q, scale, weight, weight_scale, _code(out_dtype))
    return _linear_q8_op(q, scale, weight, weight_scale, out_dtype) if out is None else out


# ---------------------------------------------------------------------------
# SwiGLU that keeps its input in 8 bits
# ---------------------------------------------------------------------------
def _ckpt_scale_cols(hidden: int) -> int:
    return 2 * (-(-hidden // CKPT_GROUP))


@torch.library.custom_op("hackable_lm_b200::swiglu_ckpt8", mutates_args=())
def _swiglu_ckpt8_op(gate_up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _run("swiglu_ckpt8", gate_up)


@_swiglu_ckpt8_op.register_fake
def _swiglu_ckpt8_fake(gate_up):
    _code(gate_up.dtype)
    hidden = _check_gate_up("swiglu_ckpt8", gate_up)
    lead = gate_up.shape[:-1]
    return (gate_up.new_empty((*lead, hidden)), gate_up.new_empty(gate_up.shape, dtype=torch.int8),
            gate_up.new_empty((*lead, _ckpt_scale_cols(hidden)), dtype=torch.float32))


@torch.library.custom_op("hackable_lm_b200::swiglu_ckpt8_backward", mutates_args=())
def _swiglu_ckpt8_backward_op(q: torch.Tensor, scale: torch.Tensor, grad_h: torch.Tensor) -> torch.Tensor:
    return _run("swiglu_ckpt8_backward", q, scale, grad_h)


@_swiglu_ckpt8_backward_op.register_fake
def _swiglu_ckpt8_backward_fake(q, scale, grad_h):
    _code(grad_h.dtype)
    hidden = _check_gate_up("swiglu_ckpt8_backward", q)
    lead = q.shape[:-1]
    _check(q.dtype == torch.int8 and scale.dtype == torch.float32 and grad_h.shape == (*lead, hidden)
           and scale.shape == (*lead, _ckpt_scale_cols(hidden)),
           "swiglu_ckpt8_backward: needs the codes and scales of swiglu_ckpt8 and a gradient "
           f"[..., {hidden}], got {tuple(q.shape)}, {tuple(scale.shape)}, {tuple(grad_h.shape)}")
    return grad_h.new_empty(q.shape)


def _swiglu_ckpt8_setup(ctx, inputs, output):
    _, q, scale = output
    ctx.save_for_backward(q, scale)
    ctx.mark_non_differentiable(q, scale)
    ctx.set_materialize_grads(False)


def _swiglu_ckpt8_bwd(ctx, grad_h, grad_q, grad_scale):
    if grad_h is None:
        return None
    q, scale = ctx.saved_tensors
    return swiglu_ckpt8_backward(q, scale, grad_h)


_swiglu_ckpt8_op.register_autograd(_swiglu_ckpt8_bwd, setup_context=_swiglu_ckpt8_setup)


def swiglu_ckpt8(gate_up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(h, q, scale): h = silu(gate) * up of gate_up [..., 2H], and gate_up in 8 bits with one
    scale for each 128 hidden units of the gate half and of the up half (scale [..., 2 * ceil(H / 128)],
    gate groups first).  Its gradient is that of SwiGLU at the values the codes stand for; gate_up
    itself is not kept."""
    out = None if _compiling() else _lib.binding().swiglu_ckpt8(gate_up)
    return _swiglu_ckpt8_op(gate_up) if out is None else out


def swiglu_ckpt8_backward(q: torch.Tensor, scale: torch.Tensor, grad_h: torch.Tensor) -> torch.Tensor:
    """grad_gate_up [..., 2H] from the codes and scales of swiglu_ckpt8 and grad_h [..., H]."""
    out = None if _compiling() else _lib.binding().swiglu_ckpt8_backward(q, scale, grad_h)
    return _swiglu_ckpt8_backward_op(q, scale, grad_h) if out is None else out


# ---------------------------------------------------------------------------
# Projection that keeps its input in 8 bits
# ---------------------------------------------------------------------------
@torch.library.custom_op("hackable_lm_b200::weight_grad_q8", mutates_args=())
def _weight_grad_q8_op(grad: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return _run("weight_grad_q8", grad, q, scale)


@_weight_grad_q8_op.register_fake
def _weight_grad_q8_fake(grad, q, scale):
    _check_rows("weight_grad_q8", q, scale)
    _check(grad.dtype in (torch.bfloat16, torch.float16), f"weight_grad_q8: grad must be bf16 or fp16, got {grad.dtype}")
    _check(grad.dim() >= 1 and grad.shape[:-1] == q.shape[:-1],
           "weight_grad_q8: grad [..., N] and the codes [..., K] must have the same rows, got "
           f"{tuple(grad.shape)} and {tuple(q.shape)}")
    return grad.new_empty((grad.shape[-1], q.shape[-1]))


def weight_grad_q8(grad: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """grad^T @ (q * scale) [N, K]: the weight gradient of a projection from its input in 8 bits
    (grad [..., N] bf16 or fp16, q int8 [..., K] with a scale for each row; N a multiple of 8, K of 16).
    The values read back are held in two values of grad's type (to 2^-15 of each in bf16, 2^-21 in
    fp16, whatever the scales' size, or 2^-39 of the largest value), the sums in fp32; the result is rounded once.  Takes 4 bytes of workspace for each code."""
    out = None if _compiling() else _lib.binding().weight_grad_q8(grad, q, scale)
    return _weight_grad_q8_op(grad, q, scale) if out is None else out


def linear_ckpt8_supported(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """Shapes and dtypes whose weight gradient ``weight_grad_q8`` takes."""
    return ((x.is_cuda or x.is_meta) and x.dtype in (torch.bfloat16, torch.float16) and weight.dtype == x.dtype
            and weight.dim() == 2 and x.shape[-1] == weight.shape[1] and weight.shape[0] % 8 == 0
            and weight.shape[1] % 16 == 0 and weight.numel() > 0)


def linear_in_own_type(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """F.linear whose result has x's type, as the gradients do, whatever autocast's type is."""
    if torch.is_autocast_enabled("cuda"):
        with torch.autocast("cuda", enabled=False):
            return torch.nn.functional.linear(x, weight)
    return torch.nn.functional.linear(x, weight)


@torch.library.custom_op("hackable_lm_b200::linear_ckpt8", mutates_args=())
def linear_ckpt8(x: torch.Tensor, weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, q, scale): y = x @ weight^T, and x in 8 bits by rows, kept for the weight gradient
    in place of x."""
    _require_cuda(x, weight)
    if not linear_ckpt8_supported(x, weight):
        raise RuntimeError("linear_ckpt8: needs bf16 or fp16 x [..., K] and weight [N, K] of one dtype with N a "
                           f"multiple of 8 and K of 16, got {x.dtype} {tuple(x.shape)}, {weight.dtype} "
                           f"{tuple(weight.shape)}")
    q, scale = _run("quantize_rows", x)
    return linear_in_own_type(x, weight), q, scale


@linear_ckpt8.register_fake
def _linear_ckpt8_fake(x, weight):
    return (x.new_empty((*x.shape[:-1], weight.shape[0])), *_quantize_rows_fake(x))


def _linear_ckpt8_setup(ctx, inputs, output):
    _, weight = inputs
    _, q, scale = output
    ctx.save_for_backward(weight, q, scale)
    ctx.mark_non_differentiable(q, scale)
    ctx.set_materialize_grads(False)


def _linear_ckpt8_bwd(ctx, grad_y, grad_q, grad_scale):
    if grad_y is None:
        return None, None
    weight, q, scale = ctx.saved_tensors
    g = grad_y.contiguous()
    grad_x = (g.reshape(-1, g.shape[-1]) @ weight).reshape(q.shape) if ctx.needs_input_grad[0] else None
    grad_w = weight_grad_q8(g, q, scale) if ctx.needs_input_grad[1] else None
    return grad_x, grad_w


linear_ckpt8.register_autograd(_linear_ckpt8_bwd, setup_context=_linear_ckpt8_setup)
