"""PyTorch operators of the 8-bit path over the libhlm_b200 C ABI.

The 8-bit format (``include/hlm_b200.h``): a group of values v is int8 codes and
one fp32 scale, ``a = max(max|v|, 2^-110)``, ``q = rint(v * (127 / a))``,
``scale = a / 127``, ``v ~ q * scale``.  A group is a whole row, except in
``swiglu_ckpt8``.  A group with an infinity or a NaN has scale NaN and codes 0.

Every operator is a ``torch.library.custom_op`` with a fake implementation, as
in :mod:`hackable_lm_b200.ops`.  Called on plain CUDA tensors outside
``torch.compile``, with no gradient asked for, the functions of this module go
straight to the library: the dispatcher costs more than the kernels of a
single token.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import check
from .ops import _DTYPE_CODE, _code, _require_cuda

CKPT_GROUP = 128


def _direct(*tensors: Optional[torch.Tensor]) -> bool:
    """Plain CUDA tensors, eager mode and no gradient asked for: no dispatcher needed."""
    if torch.compiler.is_compiling():
        return False
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and (type(t) not in _PLAIN or not t.is_cuda or (grad and t.requires_grad)):
            return False
    return True


_PLAIN = (torch.Tensor, torch.nn.Parameter)


_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream() builds an object around it (1.2 us)


def _device_of(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """Index of the CUDA device that all the tensors are on (raises where there is none)."""
    idx = first.get_device()
    for t in others:
        if t is not None and t.get_device() != idx:
            idx = -1
    if idx < 0 or not first.is_cuda:
        _require_cuda(first, *(t for t in others if t is not None))
        raise RuntimeError("hackable_lm_b200: all tensors must be on the same device")
    return idx


def _call(idx: int, name: str, *args) -> None:
    """Library call on the current stream of device ``idx``, with it current for the call's duration."""
    fn = _FNS.get(name)
    if fn is None:
        fn = _FNS[name] = getattr(_lib.load(), name)
    if torch.cuda.current_device() == idx:
        rc = fn(*args, _raw_stream(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(*args, _raw_stream(idx))
    if rc:
        check(rc, name)


_FNS: dict = {}


def _packed(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned, as the tensor-core kernels read it (a copy where it is not)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_rows(what: str, q: torch.Tensor, scale: torch.Tensor) -> None:
    if q.dtype != torch.int8 or scale.dtype != torch.float32 or q.dim() < 1 or scale.shape != q.shape[:-1]:
        raise RuntimeError(f"{what}: needs int8 codes [..., C] and their fp32 scales [...], got {q.dtype} "
                           f"{tuple(q.shape)} and {scale.dtype} {tuple(scale.shape)}")


def _check_cols(what: str, x: torch.Tensor) -> None:
    _code(x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"{what}: needs at least one column, got shape {tuple(x.shape)}")


# ---------------------------------------------------------------------------
# Rows to 8 bits and back
# ---------------------------------------------------------------------------
def _quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    _check_cols("quantize_rows", x)
    dev = _device_of(x)
    x = x.contiguous()
    cols = x.shape[-1]
    q = x.new_empty(x.shape, dtype=torch.int8)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    _call(dev, "hlm_quantize_rows", x.data_ptr(), q.data_ptr(), scale.data_ptr(), scale.numel(), cols,
          _DTYPE_CODE[x.dtype])
    return q, scale


_quantize_rows_op = torch.library.custom_op("hackable_lm_b200::quantize_rows", _quantize_rows, mutates_args=())


@_quantize_rows_op.register_fake
def _quantize_rows_fake(x):
    return (torch.empty(x.shape, dtype=torch.int8, device=x.device),
            torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device))


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q int8 [..., C], scale fp32 [...]) of x [..., C]."""
    return _quantize_rows(x) if _direct(x) else _quantize_rows_op(x)


def _dequantize_rows(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    _check_rows("dequantize_rows", q, scale)
    dev = _device_of(q, scale)
    code = _code(dtype)
    q, scale = q.contiguous(), scale.contiguous()
    out = q.new_empty(q.shape, dtype=dtype)
    if q.numel():
        _call(dev, "hlm_dequantize_rows", q.data_ptr(), scale.data_ptr(), out.data_ptr(), scale.numel(),
              q.shape[-1], code)
    return out


_dequantize_rows_op = torch.library.custom_op("hackable_lm_b200::dequantize_rows", _dequantize_rows,
                                              mutates_args=())


@_dequantize_rows_op.register_fake
def _dequantize_rows_fake(q, scale, dtype):
    return torch.empty(q.shape, dtype=dtype, device=q.device)


def dequantize_rows(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """q * scale of each row, rounded to ``dtype``."""
    return (_dequantize_rows if _direct(q, scale) else _dequantize_rows_op)(q, scale, dtype)


# ---------------------------------------------------------------------------
# RMSNorm with an 8-bit output
# ---------------------------------------------------------------------------
def _norm_weight(what: str, x: torch.Tensor, weight: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if weight is None:
        return None
    if weight.shape != x.shape[-1:]:
        raise RuntimeError(f"{what}: weight must be [{x.shape[-1]}], got {tuple(weight.shape)}")
    _device_of(x, weight)
    return weight.to(x.dtype).contiguous()


def _rms_norm_q8(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    _check_cols("rms_norm_q8", x)
    dev = _device_of(x)
    w = _norm_weight("rms_norm_q8", x, weight)
    x = x.contiguous()
    q = x.new_empty(x.shape, dtype=torch.int8)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    _call(dev, "hlm_residual_rms_norm_q8", None, x.data_ptr(), None if w is None else w.data_ptr(), None,
          q.data_ptr(), scale.data_ptr(), scale.numel(), x.shape[-1], float(eps), _DTYPE_CODE[x.dtype])
    return q, scale


_rms_norm_q8_op = torch.library.custom_op("hackable_lm_b200::rms_norm_q8", _rms_norm_q8, mutates_args=())


@_rms_norm_q8_op.register_fake
def _rms_norm_q8_fake(x, weight, eps):
    return _quantize_rows_fake(x)


def rms_norm_q8(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of rms_norm(x) [* weight], by rows."""
    return (_rms_norm_q8 if _direct(x, weight) else _rms_norm_q8_op)(x, weight, eps)


def _residual_rms_norm_q8(residual: torch.Tensor, branch: torch.Tensor, weight: Optional[torch.Tensor],
                          eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_cols("residual_rms_norm_q8", branch)
    dev = _device_of(residual, branch)
    if residual.shape != branch.shape or residual.dtype != branch.dtype:
        raise RuntimeError("residual_rms_norm_q8: residual and branch must match in shape and dtype")
    w = _norm_weight("residual_rms_norm_q8", branch, weight)
    residual, branch = residual.contiguous(), branch.contiguous()
    out = branch.new_empty(branch.shape)
    q = branch.new_empty(branch.shape, dtype=torch.int8)
    scale = branch.new_empty(branch.shape[:-1], dtype=torch.float32)
    _call(dev, "hlm_residual_rms_norm_q8", residual.data_ptr(), branch.data_ptr(),
          None if w is None else w.data_ptr(), out.data_ptr(), q.data_ptr(), scale.data_ptr(), scale.numel(),
          branch.shape[-1], float(eps), _DTYPE_CODE[branch.dtype])
    return out, q, scale


_residual_rms_norm_q8_op = torch.library.custom_op("hackable_lm_b200::residual_rms_norm_q8",
                                                   _residual_rms_norm_q8, mutates_args=())


@_residual_rms_norm_q8_op.register_fake
def _residual_rms_norm_q8_fake(residual, branch, weight, eps):
    return (torch.empty(branch.shape, dtype=branch.dtype, device=branch.device), *_quantize_rows_fake(branch))


def residual_rms_norm_q8(residual: torch.Tensor, branch: torch.Tensor, weight: Optional[torch.Tensor],
                         eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(out, q, scale): out = residual + branch, and rms_norm(out) [* weight] in 8 bits by rows."""
    fn = _residual_rms_norm_q8 if _direct(residual, branch, weight) else _residual_rms_norm_q8_op
    return fn(residual, branch, weight, eps)


# ---------------------------------------------------------------------------
# 8-bit integer projection
# ---------------------------------------------------------------------------
def _linear_q8(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
               out_dtype: torch.dtype) -> torch.Tensor:
    _check_rows("linear_q8", q, scale)
    _check_rows("linear_q8 (weight)", weight, weight_scale)
    code = _code(out_dtype)
    if weight.dim() != 2 or weight.shape[1] != q.shape[-1]:
        raise RuntimeError(f"linear_q8: weight must be [N, {q.shape[-1]}], got {tuple(weight.shape)}")
    dev = _device_of(q, scale, weight, weight_scale)
    N, K = weight.shape
    q, weight, scale, weight_scale = _packed(q), _packed(weight), scale.contiguous(), weight_scale.contiguous()
    out = q.new_empty((*q.shape[:-1], N), dtype=out_dtype)
    _call(dev, "hlm_linear_q8", q.data_ptr(), scale.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(),
          out.data_ptr(), scale.numel(), N, K, code)
    return out


_linear_q8_op = torch.library.custom_op("hackable_lm_b200::linear_q8", _linear_q8, mutates_args=())


@_linear_q8_op.register_fake
def _linear_q8_fake(q, scale, weight, weight_scale, out_dtype):
    return torch.empty((*q.shape[:-1], weight.shape[0]), dtype=out_dtype, device=q.device)


def linear_q8(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """(q * scale) @ (weight * weight_scale)^T with exact integer sums: q int8 [..., K] with a
    scale for each token, weight int8 [N, K] with a scale for each output channel; K a
    multiple of 16."""
    fn = _linear_q8 if _direct(q, scale, weight, weight_scale) else _linear_q8_op
    return fn(q, scale, weight, weight_scale, out_dtype)


# ---------------------------------------------------------------------------
# SwiGLU that keeps its input in 8 bits
# ---------------------------------------------------------------------------
def _ckpt_scale_cols(hidden: int) -> int:
    return 2 * (-(-hidden // CKPT_GROUP))


def _check_gate_up(what: str, width: int) -> int:
    if width % 2:
        raise RuntimeError(f"{what}: the last dimension must be even (gate | up), got {width}")
    return width // 2


def _swiglu_ckpt8(gate_up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    dev = _device_of(gate_up)
    code = _code(gate_up.dtype)
    hidden = _check_gate_up("swiglu_ckpt8", gate_up.shape[-1])
    gate_up = gate_up.contiguous()
    lead = gate_up.shape[:-1]
    h = gate_up.new_empty((*lead, hidden))
    q = gate_up.new_empty(gate_up.shape, dtype=torch.int8)
    scale = gate_up.new_empty((*lead, _ckpt_scale_cols(hidden)), dtype=torch.float32)
    if hidden:
        _call(dev, "hlm_swiglu_ckpt8_fwd", gate_up.data_ptr(), h.data_ptr(), q.data_ptr(), scale.data_ptr(),
              h.numel() // hidden, hidden, code)
    return h, q, scale


_swiglu_ckpt8_op = torch.library.custom_op("hackable_lm_b200::swiglu_ckpt8", _swiglu_ckpt8, mutates_args=())


@_swiglu_ckpt8_op.register_fake
def _swiglu_ckpt8_fake(gate_up):
    hidden = gate_up.shape[-1] // 2
    lead = gate_up.shape[:-1]
    return (gate_up.new_empty((*lead, hidden)), gate_up.new_empty(gate_up.shape, dtype=torch.int8),
            gate_up.new_empty((*lead, _ckpt_scale_cols(hidden)), dtype=torch.float32))


def _swiglu_ckpt8_backward(q: torch.Tensor, scale: torch.Tensor, grad_h: torch.Tensor) -> torch.Tensor:
    code = _code(grad_h.dtype)
    hidden = _check_gate_up("swiglu_ckpt8_backward", q.shape[-1])
    lead = q.shape[:-1]
    if (q.dtype != torch.int8 or scale.dtype != torch.float32 or grad_h.shape != (*lead, hidden)
            or scale.shape != (*lead, _ckpt_scale_cols(hidden))):
        raise RuntimeError("swiglu_ckpt8_backward: needs the codes and scales of swiglu_ckpt8 and a gradient "
                           f"[..., {hidden}], got {tuple(q.shape)}, {tuple(scale.shape)}, {tuple(grad_h.shape)}")
    dev = _device_of(q, scale, grad_h)
    q, scale, grad_h = q.contiguous(), scale.contiguous(), grad_h.contiguous()
    grad = grad_h.new_empty(q.shape)
    if hidden:
        _call(dev, "hlm_swiglu_ckpt8_bwd", q.data_ptr(), scale.data_ptr(), grad_h.data_ptr(), grad.data_ptr(),
              grad_h.numel() // hidden, hidden, code)
    return grad


_swiglu_ckpt8_backward_op = torch.library.custom_op("hackable_lm_b200::swiglu_ckpt8_backward",
                                                    _swiglu_ckpt8_backward, mutates_args=())


@_swiglu_ckpt8_backward_op.register_fake
def _swiglu_ckpt8_backward_fake(q, scale, grad_h):
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
    return (_swiglu_ckpt8 if _direct(gate_up) else _swiglu_ckpt8_op)(gate_up)


def swiglu_ckpt8_backward(q: torch.Tensor, scale: torch.Tensor, grad_h: torch.Tensor) -> torch.Tensor:
    """grad_gate_up [..., 2H] from the codes and scales of swiglu_ckpt8 and grad_h [..., H]."""
    return (_swiglu_ckpt8_backward if _direct(q, scale, grad_h) else _swiglu_ckpt8_backward_op)(q, scale, grad_h)


# ---------------------------------------------------------------------------
# Projection that keeps its input in 8 bits
# ---------------------------------------------------------------------------
def _weight_grad_q8(grad: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    _check_rows("weight_grad_q8", q, scale)
    if grad.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"weight_grad_q8: grad must be bf16 or fp16, got {grad.dtype}")
    if grad.dim() < 1 or grad.shape[:-1] != q.shape[:-1]:
        raise RuntimeError("weight_grad_q8: grad [..., N] and the codes [..., K] must have the same rows, got "
                           f"{tuple(grad.shape)} and {tuple(q.shape)}")
    dev = _device_of(grad, q, scale)
    grad, q, scale = _packed(grad), _packed(q), scale.contiguous()
    tokens, N, K = scale.numel(), grad.shape[-1], q.shape[-1]
    out = grad.new_empty((N, K))
    nbytes = _lib.load().hlm_weight_grad_q8_workspace_bytes(tokens, N, K)
    ws = grad.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call(dev, "hlm_weight_grad_q8", grad.data_ptr(), q.data_ptr(), scale.data_ptr(), out.data_ptr(),
          None if ws is None else ws.data_ptr(), nbytes, tokens, N, K, _DTYPE_CODE[grad.dtype])
    return out


_weight_grad_q8_op = torch.library.custom_op("hackable_lm_b200::weight_grad_q8", _weight_grad_q8, mutates_args=())


@_weight_grad_q8_op.register_fake
def _weight_grad_q8_fake(grad, q, scale):
    return grad.new_empty((grad.shape[-1], q.shape[-1]))


def weight_grad_q8(grad: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """grad^T @ (q * scale) [N, K]: the weight gradient of a projection from its input in 8 bits
    (grad [..., N] bf16 or fp16, q int8 [..., K] with a scale for each row; N a multiple of 8, K of 16)."""
    return (_weight_grad_q8 if _direct(grad, q, scale) else _weight_grad_q8_op)(grad, q, scale)


def linear_ckpt8_supported(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """Shapes and dtypes whose weight gradient ``weight_grad_q8`` takes."""
    return ((x.is_cuda or x.is_meta) and x.dtype in (torch.bfloat16, torch.float16) and weight.dtype == x.dtype
            and weight.dim() == 2 and x.shape[-1] == weight.shape[1] and weight.shape[0] % 8 == 0
            and weight.shape[1] % 16 == 0 and weight.numel() > 0)


@torch.library.custom_op("hackable_lm_b200::linear_ckpt8", mutates_args=())
def linear_ckpt8(x: torch.Tensor, weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, q, scale): y = x @ weight^T, and x in 8 bits by rows, kept for the weight gradient
    in place of x."""
    _device_of(x, weight)
    if not linear_ckpt8_supported(x, weight):
        raise RuntimeError("linear_ckpt8: needs bf16 or fp16 x [..., K] and weight [N, K] of one dtype with N a "
                           f"multiple of 8 and K of 16, got {x.dtype} {tuple(x.shape)}, {weight.dtype} "
                           f"{tuple(weight.shape)}")
    q, scale = _quantize_rows(x)
    return torch.nn.functional.linear(x, weight), q, scale


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
