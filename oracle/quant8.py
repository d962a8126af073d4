"""The 8-bit operators restated on the CPU, with sums and functions in 64 bits.

The codes are defined by 32-bit IEEE arithmetic (``a = max(max|v|, 2^-110)``,
``q = rint(v * (127 / a))``, ``scale = a / 127``), so those steps run in float32
and give the codes exactly; everything after them is float64.
"""
from __future__ import annotations

import torch

FLOOR = 2.0 ** -110
GROUP = 128


def quantize(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes int8, scale fp32) of the groups in the last dimension of float32 v."""
    assert v.dtype == torch.float32
    a = v.abs().amax(dim=-1, keepdim=True)  # propagates NaN
    finite = torch.isfinite(a)
    a = torch.where(finite, a, torch.ones_like(a)).clamp(min=FLOOR)
    most = torch.full_like(a, 127.0)  # a tensor: with a number, torch multiplies by a rounded reciprocal
    q = torch.where(finite, torch.round(v * (most / a)), torch.zeros_like(v))
    scale = torch.where(finite, a / most, torch.full_like(a, float("nan")))
    return q.to(torch.int8), scale.squeeze(-1)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return quantize(x.float())


def read_back(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return q.double() * scale.double().unsqueeze(-1)


def rms_norm_q8(residual, branch, weight, eps):
    """(out, codes, scale in float64); residual may be None (then out is branch)."""
    out = branch if residual is None else (residual.float() + branch.float()).to(branch.dtype)
    v = out.float() if weight is None else out.float() * weight.float()
    q, scale = quantize(v)
    rms = (out.double().pow(2).mean(dim=-1) + eps).sqrt()
    return out, q, scale.double() / rms


def linear_q8(q, scale, w, w_scale):
    acc = q.double() @ w.double().t()  # exact: below 2^53
    return acc * scale.double().unsqueeze(-1) * w_scale.double()


def group_codes(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes [..., H] and scales [..., ceil(H / 128)] of groups of 128 columns."""
    q, s = zip(*(quantize(p.float()) for p in x.split(GROUP, dim=-1)))
    return torch.cat(q, dim=-1), torch.stack(s, dim=-1)


def group_read_back(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    wide = scale.double().repeat_interleave(GROUP, dim=-1)[..., : q.shape[-1]]
    return q.double() * wide


def swiglu_ckpt8(gate_up):
    """(h float64, codes, scales) of gate_up [..., 2H]."""
    gate, up = gate_up.chunk(2, dim=-1)
    h = gate.double() * torch.sigmoid(gate.double()) * up.double()
    qg, sg = group_codes(gate)
    qu, su = group_codes(up)
    return h, torch.cat((qg, qu), dim=-1), torch.cat((sg, su), dim=-1)


def swiglu_ckpt8_backward(q, scale, grad_h):
    qg, qu = q.chunk(2, dim=-1)
    sg, su = scale.chunk(2, dim=-1)
    gate, up, d = group_read_back(qg, sg), group_read_back(qu, su), grad_h.double()
    s = torch.sigmoid(gate)
    return torch.cat((d * up * s * (1 + gate * (1 - s)), d * gate * s), dim=-1)


def weight_grad_q8(grad, q, scale):
    return grad.double().t() @ read_back(q, scale)
