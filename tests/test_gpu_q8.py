"""The 8-bit operators on the GPU against plain implementations in 64 bits (oracle.quant8).

Tolerances count roundings.  u = 2^-24 is half a step of fp32, E(t) half a step of the
output type (finfo.eps / 2), and T(t) half a step of its subnormals.

* codes: equal (the format defines them by IEEE fp32 steps); scales of quantize_rows too.
* read back: one fp32 product and the output rounding: (u + E) |y|.
* norm scale: a sum of n squares (every term positive, so at most n u relative whatever
  the order), mean, square root (2 ulp), two products: (n + 8) u; half of the sum's.
* linear_q8: the sum is exact; its conversion and two products are 3 u, then E.
* SwiGLU: sigmoid(x) from 2^(x log2 e) carries the argument's rounding, |x| u from the
  product and as much from the constant, and a few ulp for ex2, the sum and the
  divide: (2 |x| + 16) u.  A gradient is bounded with the magnitudes of its terms
  (1 + g (1 - s) can cancel).
* weight_grad_q8: each read-back value is rounded once to the operand type (E), the fp32
  sum of m terms adds m u of the sum of magnitudes, the result is rounded (E).
"""
from __future__ import annotations

import pytest
import torch

from oracle import quant8
from test_q8_host import bad_calls

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def half_subnormal(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def assert_within(actual, expected, bound, what):
    a, e = actual.detach().double().cpu(), expected.double()
    assert a.shape == e.shape, f"{what}: {tuple(a.shape)} vs {tuple(e.shape)}"
    assert torch.equal(torch.isnan(a), torch.isnan(e)), f"{what}: NaN in different places"
    err = torch.where(torch.isnan(e), torch.zeros_like(e), (a - e).abs())
    over = torch.where(torch.isnan(e), torch.zeros_like(e), err - bound)
    assert bool((over <= 0).all()), f"{what}: off by {err.max():.3e}, {over.max():.3e} over the bound"


def values(shape, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    cols = torch.exp(0.5 * torch.randn(shape[-1], generator=g))
    return (torch.randn(shape, generator=g) * cols * scale).to(dtype)


@pytest.fixture(autouse=True)
def device_error_stays_clear(cuda_device):
    from hackable_lm_b200 import _lib

    _lib.clear_device_error()
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------
ROW_SHAPES = [(1, 1), (3, 7), (1, 16), (5, 128), (67, 768), (9, 130), (33, 1000), (2, 4104), (3, 8192), (2, 20000),
              (4, 40001), (2, 3, 264), (300, 48)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROW_SHAPES)
def test_quantize_rows_and_back(shape, dtype, cuda_device):
    from hackable_lm_b200 import kernels

    x = values(shape, dtype, seed=sum(shape))
    q, scale = kernels.quantize_rows(x.to(cuda_device))
    eq, es = quant8.quantize_rows(x)
    assert torch.equal(q.cpu(), eq) and torch.equal(scale.cpu(), es)
    for out in DTYPES:
        y = kernels.dequantize_rows(q, scale, out)
        e = quant8.read_back(eq, es)
        assert y.dtype == out
        assert_within(y, e, e.abs() * (U + half_step(out)) + half_subnormal(out), f"read back {out}")


def _special_rows(dtype):
    """Rows where a code can go wrong: zeros, subnormals, one value, borders, the type's extremes,
    infinities and NaNs."""
    fi = torch.finfo(dtype)
    base = values((12, 256), torch.float32, seed=4)
    base[0] = 0.0
    base[1] = fi.smallest_normal * fi.eps * torch.randint(-3, 4, (256,), generator=torch.Generator().manual_seed(1))
    base[2] = 0.0
    base[2, 17] = -3.0
    base[3] = torch.arange(256).float() - 127.5      # half-way values between codes
    base[3, 0] = 127.0
    base[4] = torch.where(torch.arange(256) % 2 == 0, fi.max, -fi.max)
    base[5, 3] = float("inf")
    base[6, 250] = float("-inf")
    base[7, 100] = float("nan")
    base[8, 0] = float("nan")
    base[8, 1] = float("inf")
    base[9] = -0.0
    return base.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [256, 255, 13])
def test_quantize_special_rows(dtype, cols, cuda_device):
    from hackable_lm_b200 import kernels

    x = _special_rows(dtype)[:, :cols].contiguous()
    q, scale = kernels.quantize_rows(x.to(cuda_device))
    eq, es = quant8.quantize_rows(x)
    assert torch.equal(q.cpu(), eq)
    assert torch.equal(torch.nan_to_num(scale.cpu(), nan=-1.0), torch.nan_to_num(es, nan=-1.0))
    y = kernels.dequantize_rows(q, scale, torch.float32)
    assert torch.equal(torch.isnan(y.cpu()).all(dim=-1), torch.isnan(es))
    assert int(q.min()) >= -127


def test_quantize_strided_and_misaligned_inputs(cuda_device):
    from hackable_lm_b200 import kernels

    x = values((64, 96), torch.bfloat16, seed=7)
    for view in (x.t(), x[::2], x[:, 3:91], x.flatten()[1:1 + 63 * 96].view(63, 96)):
        dev = x.to(cuda_device).as_strided(view.shape, view.stride(), view.storage_offset())
        q, scale = kernels.quantize_rows(dev)
        eq, es = quant8.quantize_rows(view.contiguous())
        assert torch.equal(q.cpu(), eq) and torch.equal(scale.cpu(), es)
        flat = torch.empty(q.numel() + 1, dtype=torch.int8, device=cuda_device)
        flat[1:] = q.flatten()
        y = kernels.dequantize_rows(flat[1:].view(q.shape), scale, torch.float32)
        assert torch.equal(y, kernels.dequantize_rows(q, scale, torch.float32))


def test_quantize_offsets_past_32_bits(cuda_device):
    """70,000 rows of 32,768: the last rows start past 2^31 elements."""
    from hackable_lm_b200 import kernels

    x = torch.zeros(70000, 32768, dtype=torch.bfloat16, device=cuda_device)
    tail = values((3, 32768), torch.bfloat16, seed=9)
    x[-3:] = tail.to(cuda_device)
    q, scale = kernels.quantize_rows(x)
    eq, es = quant8.quantize_rows(tail)
    assert torch.equal(q[-3:].cpu(), eq) and torch.equal(scale[-3:].cpu(), es)
    assert int(q[:-3].abs().amax()) == 0
    y = kernels.dequantize_rows(q, scale, torch.bfloat16)
    assert torch.equal(y[-3:].float().cpu(), (eq.float() * es[:, None]).to(torch.bfloat16).float())
    assert not y[:-3].any()


# ---------------------------------------------------------------------------
# RMSNorm with an 8-bit output
# ---------------------------------------------------------------------------
def _check_norm(residual, branch, weight, eps, device):
    from hackable_lm_b200 import kernels

    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    n = branch.shape[-1]
    if residual is None:
        q, scale = kernels.rms_norm_q8(to(branch), to(weight), eps)
    else:
        out, q, scale = kernels.residual_rms_norm_q8(to(residual), to(branch), eps, to(weight))
    w = None if weight is None else weight.to(branch.dtype)
    eo, eq, es = quant8.rms_norm_q8(residual, branch, w, eps)
    if residual is not None:
        assert torch.equal(torch.nan_to_num(out.cpu().float(), nan=7e7), torch.nan_to_num(eo.float(), nan=7e7))
    assert torch.equal(q.cpu(), eq)
    assert_within(scale, es, es.abs() * (n / 2 + 8) * U + 2.0 ** -149, "scale")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROW_SHAPES)
@pytest.mark.parametrize("has_residual,has_weight", [(True, False), (True, True), (False, False), (False, True)])
def test_rms_norm_q8(shape, dtype, has_residual, has_weight, cuda_device):
    branch = values(shape, dtype, seed=1)
    residual = values(shape, dtype, seed=2, scale=3.0) if has_residual else None
    weight = values((shape[-1],), torch.float32, seed=3) if has_weight else None
    _check_norm(residual, branch, weight, 1e-6, cuda_device)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rms_norm_q8_special_rows(dtype, cuda_device):
    x = _special_rows(dtype)
    x[4] = 0.5  # the type's extremes overflow the sum of squares in bf16 and fp32: tested below
    _check_norm(torch.zeros_like(x), x, None, 1e-6, cuda_device)
    _check_norm(None, x, torch.full((256,), 2.0), 1e-5, cuda_device)


def test_rms_norm_q8_square_overflow_reads_back_as_the_norm(cuda_device):
    """Where the sum of squares overflows, 1/rms is zero and so is everything read back, as the
    bf16 norm itself is."""
    from hackable_lm_b200 import kernels

    x = torch.full((2, 64), 1e30, device=cuda_device)
    q, scale = kernels.rms_norm_q8(x, None, 1e-6)
    assert torch.equal(kernels.dequantize_rows(q, scale, torch.float32), kernels.rms_norm(x, None, 1e-6))


# ---------------------------------------------------------------------------
# 8-bit integer projection
# ---------------------------------------------------------------------------
def codes(shape, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, shape, generator=g, dtype=torch.int16).to(torch.int8)
    return q, torch.exp(torch.randn(shape[:-1], generator=g)) * 1e-2


def _check_linear(q, scale, w, w_scale, out_dtype, device):
    from hackable_lm_b200 import kernels

    y = kernels.linear_q8(q.to(device), scale.to(device), w.to(device), w_scale.to(device), out_dtype)
    e = quant8.linear_q8(q, scale, w, w_scale)
    assert y.dtype == out_dtype
    fits = e.abs() <= torch.finfo(out_dtype).max
    assert bool(fits[~torch.isnan(e)].all())
    assert_within(y, e, e.abs() * (3 * U + half_step(out_dtype)) + half_subnormal(out_dtype), "linear_q8")


LINEAR_SHAPES = [  # M, N, K
    (1, 1, 16), (1, 4096, 768), (2, 33, 48), (3, 1000, 2048), (4, 768, 16), (5, 129, 8192), (7, 2304, 768), (8, 16, 112),
    (9, 31, 1360), (16, 130, 768), (17, 128, 128), (31, 257, 400), (33, 768, 2048), (64, 512, 64), (65, 100, 4096),
    (127, 96, 144), (128, 128, 128), (129, 1111, 272), (200, 4096, 768), (255, 40, 16), (256, 256, 256), (257, 513, 1040),
    (777, 1111, 1360), (1000, 24, 528), (1500, 2304, 768), (1, 33, 2064), (1, 5000, 4112), (2, 2049, 4112), (4, 77, 2048),
    (6, 4096, 4096), (3, 8200, 1040), (1, 2, 131056)]


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", LINEAR_SHAPES)
def test_linear_q8(M, N, K, out_dtype, cuda_device):
    q, scale = codes((M, K), seed=M + N)
    w, w_scale = codes((N, K), seed=K)
    _check_linear(q, scale * (1e-2 if out_dtype == torch.float16 else 1.0), w, w_scale, out_dtype, cuda_device)


def _linear_tile(M, N, K, out_dtype):
    import ctypes

    from hackable_lm_b200 import _lib, ops

    tile = ctypes.c_int()
    _lib.check(_lib.load().hlm_linear_q8_plan(M, N, K, ops._code(out_dtype), ctypes.byref(tile)), "hlm_linear_q8_plan")
    return tile.value


# M, N, K, the kernel they run: the CTA-pair GEMM with several tiles a pair (a second round of its
# accumulators, rows and columns that end inside a tile, rows of the output that are no 16-byte
# multiples), and the cluster kernel's largest tile
DENSE_LINEAR_SHAPES = [(8192, 4096, 768, -256), (8190, 4096, 784, -256), (4100, 4095, 768, -256), (6400, 640, 768, -128),
                       (6401, 635, 400, -128), (128, 8192, 8192, 128), (100, 4099, 8192, 128)]


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,tile", DENSE_LINEAR_SHAPES)
def test_linear_q8_many_tiles(M, N, K, tile, out_dtype, cuda_device):
    """Against the exact sums, made in float64 on the GPU."""
    from hackable_lm_b200 import kernels

    assert _linear_tile(M, N, K, out_dtype) == tile
    q, scale = (t.to(cuda_device) for t in codes((M, K), seed=M))
    w, w_scale = (t.to(cuda_device) for t in codes((N, K), seed=N))
    if out_dtype == torch.float16:
        scale = scale * 1e-2
    y = kernels.linear_q8(q, scale, w, w_scale, out_dtype).double()
    e = quant8.linear_q8(q, scale, w, w_scale)
    over = (y - e).abs() - e.abs() * (3 * U + half_step(out_dtype)) - half_subnormal(out_dtype)
    assert float(over.max()) <= 0, f"over the bound by {float(over.max()):.3e}"


def test_linear_q8_shapes_reach_every_kernel(cuda_device):
    for out_dtype in DTYPES:
        reached = {_linear_tile(*shape[:3], out_dtype) for shape in LINEAR_SHAPES + DENSE_LINEAR_SHAPES}
        assert reached == {0, 16, 32, 64, 128, -128, -256}


@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_q8_largest_sums(M, cuda_device):
    """Codes of the largest magnitude: -128 (which the quantiser never writes) times itself over
    K = 131,056 sums to 2,147,221,504, just within 32 bits; and both signs of 127."""
    K = 131056
    w = torch.full((40, K), -128, dtype=torch.int8)
    q = torch.full((M, K), -128, dtype=torch.int8)
    q[0] = 127
    ones = torch.ones
    _check_linear(q, ones(M), w, ones(40), torch.float32, cuda_device)


def test_linear_q8_shapes_scales_and_strides(cuda_device):
    from hackable_lm_b200 import kernels

    q, scale = codes((2, 3, 96), seed=1)
    w, w_scale = codes((50, 96), seed=2)
    scale[1, 2] = float("nan")
    w_scale[7] = float("inf")
    q[0, 0] = 0  # 0 * inf
    y = kernels.linear_q8(q.to(cuda_device), scale.to(cuda_device), w.to(cuda_device), w_scale.to(cuda_device))
    assert y.shape == (2, 3, 50) and y.dtype == torch.bfloat16
    assert bool(torch.isnan(y[1, 2]).all()) and bool(torch.isnan(y[0, 0, 7]))
    assert bool(torch.isfinite(y[0, 1, :7]).all())
    # transposed and offset storages are laid out anew
    big = torch.zeros(97, 51, dtype=torch.int8, device=cuda_device)
    big[:96, 1:] = w.t().to(cuda_device)
    wt = big[:96, 1:].t()
    flat = torch.zeros(6 * 96 + 5, dtype=torch.int8, device=cuda_device)
    flat[5:] = q.flatten().to(cuda_device)
    y2 = kernels.linear_q8(flat[5:].view(2, 3, 96), scale.to(cuda_device), wt, w_scale.to(cuda_device))
    assert torch.equal(torch.nan_to_num(y2), torch.nan_to_num(y))


@pytest.mark.parametrize("M", [0, 1, 5])
def test_linear_q8_empty(M, cuda_device):
    from hackable_lm_b200 import kernels

    q = torch.zeros(M, 32, dtype=torch.int8, device=cuda_device)
    w = torch.zeros(0, 32, dtype=torch.int8, device=cuda_device)
    y = kernels.linear_q8(q, torch.ones(M, device=cuda_device), w, torch.ones(0, device=cuda_device))
    assert y.shape == (M, 0)


def test_linear_q8_offsets_past_32_bits(cuda_device):
    """An output of 70,000 x 32,768: the last rows start past 2^31 elements."""
    from hackable_lm_b200 import kernels

    q = torch.zeros(70000, 16, dtype=torch.int8, device=cuda_device)
    tail, scale = codes((3, 16), seed=5)
    q[-3:] = tail.to(cuda_device)
    s = torch.ones(70000, device=cuda_device)
    s[-3:] = scale.to(cuda_device)
    w, w_scale = codes((32768, 16), seed=6)
    y = kernels.linear_q8(q, s, w.to(cuda_device), w_scale.to(cuda_device))
    e = quant8.linear_q8(tail, scale, w, w_scale)
    assert_within(y[-3:], e, e.abs() * (3 * U + half_step(torch.bfloat16)), "last rows")
    assert not y[:-3].any()


# ---------------------------------------------------------------------------
# SwiGLU checkpoint
# ---------------------------------------------------------------------------
SWIGLU_SHAPES = [(1, 1), (3, 5), (2, 64), (4, 127), (5, 128), (7, 129), (33, 1000), (17, 2048), (2, 3, 272), (9, 2052), (300, 16)]


def _check_swiglu(gate_up, grad_h, device):
    from hackable_lm_b200 import ops

    dtype = gate_up.dtype
    h, q, scale = ops.swiglu_ckpt8(gate_up.to(device))
    eh, eq, es = quant8.swiglu_ckpt8(gate_up)
    gate = gate_up.chunk(2, dim=-1)[0].double()
    assert h.dtype == dtype
    tiny = half_subnormal(dtype) + 2.0 ** -126
    assert_within(h, eh, eh.abs() * ((2 * gate.abs() + 16) * U + half_step(dtype)) + tiny, "h")
    assert torch.equal(q.cpu(), eq)
    assert torch.equal(torch.nan_to_num(scale.cpu(), nan=-1.0), torch.nan_to_num(es, nan=-1.0))
    grad = ops.swiglu_ckpt8_backward(q, scale, grad_h.to(device))
    e = quant8.swiglu_ckpt8_backward(eq, es, grad_h)
    (qg, qu), (sg, su) = eq.chunk(2, dim=-1), es.chunk(2, dim=-1)
    g, u, d = quant8.group_read_back(qg, sg), quant8.group_read_back(qu, su), grad_h.double()
    s = torch.sigmoid(g)
    size = torch.cat(((d * u * s).abs() * (1 + g.abs() * (1 - s + 2 * U)), (d * g * s).abs()), dim=-1)
    reach = torch.cat((g, g), dim=-1).abs()
    assert_within(grad, e, size * (2 * reach + 20) * U + e.abs() * half_step(dtype) + tiny, "grad_gate_up")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SWIGLU_SHAPES)
def test_swiglu_ckpt8(shape, dtype, cuda_device):
    gate_up = values((*shape[:-1], 2 * shape[-1]), dtype, seed=sum(shape))
    grad_h = values(shape, dtype, seed=5, scale=0.1)
    _check_swiglu(gate_up, grad_h, cuda_device)


@pytest.mark.parametrize("dtype", DTYPES)
def test_swiglu_ckpt8_far_and_zero_values(dtype, cuda_device):
    """Gates far on both sides (the sigmoid saturates), zero groups, and one large value in a group."""
    gate_up = values((4, 2 * 300), dtype, seed=3)
    gate_up[0, :300] = torch.linspace(-60, 60, 300).to(dtype)
    gate_up[1] = 0
    gate_up[2, 130] = 300.0
    _check_swiglu(gate_up, values((4, 300), dtype, seed=6), cuda_device)


@pytest.mark.parametrize("hidden", [128, 129, 1000])
def test_swiglu_ckpt8_fp32_gradient_of_far_gates(hidden, cuda_device):
    """fp32 gradients keep their bits however far the gate is.  The scales are powers of two, so the
    values read back are exact.  e^-g is off by an ulp (2 U), s = 1 / (1 + e) by 7 U (the divide
    by 2 ulp), its complement by 10 U (e s, or 1 - s where s is at most a half), so d g s by 9 U and
    d u s (1 + g (1 - s)) by 22 U of the magnitudes."""
    from hackable_lm_b200 import ops

    g = torch.Generator().manual_seed(hidden)
    rows, groups = 12, -(-hidden // 128)
    q = torch.randint(-127, 128, (rows, 2 * hidden), generator=g, dtype=torch.int16).to(torch.int8)
    scale = 2.0 ** torch.randint(-6, 0, (rows, 2 * groups), generator=g).float()
    d = values((rows, hidden), torch.float32, seed=2, scale=0.1)
    grad = ops.swiglu_ckpt8_backward(q.to(cuda_device), scale.to(cuda_device), d.to(cuda_device))
    e = quant8.swiglu_ckpt8_backward(q, scale, d)
    (qg, qu), (sg, su) = q.chunk(2, dim=-1), scale.chunk(2, dim=-1)
    gate, up, dd = quant8.group_read_back(qg, sg), quant8.group_read_back(qu, su), d.double()
    s, rest = torch.sigmoid(gate), torch.sigmoid(-gate)
    bound = torch.cat(((dd * up * s).abs() * (1 + gate.abs() * rest) * 22 * U, (dd * gate * s).abs() * 9 * U), dim=-1)
    assert_within(grad, e, bound + 2.0 ** -126, "grad_gate_up")


@pytest.mark.parametrize("hidden", [64, 100, 129, 2048])
@pytest.mark.parametrize("dtype", DTYPES)
def test_swiglu_ckpt8_output_is_swiglu(hidden, dtype, cuda_device):
    """The forward's output has the bits of kernels.swiglu_triton, with and without a gradient."""
    from hackable_lm_b200 import kernels

    gate_up = values((37, 2 * hidden), dtype, seed=hidden).to(cuda_device)
    plain = kernels.swiglu_triton(gate_up)
    assert torch.equal(kernels.swiglu_ckpt8(gate_up), plain)
    assert torch.equal(kernels.swiglu_ckpt8(gate_up.requires_grad_(True)), plain)


@pytest.mark.parametrize("dtype", DTYPES)
def test_swiglu_ckpt8_output_is_swiglu_for_every_16_bit_gate(dtype, cuda_device):
    """Every 16-bit gate (and 2^20 fp32 ones over the whole range), NaNs and infinities among them."""
    from hackable_lm_b200 import kernels, ops

    if dtype == torch.float32:
        g = torch.Generator().manual_seed(3)
        gate = torch.cat((torch.randn(1 << 19, generator=g) * 30, torch.randint(-2 ** 31, 2 ** 31 - 1, (1 << 19,), generator=g,
                                                                              dtype=torch.int32).view(torch.float32)))
    else:
        gate = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    gate = gate.reshape(-1, 256)
    gate_up = torch.cat((gate, torch.ones_like(gate)), dim=1).to(cuda_device)
    plain, h = kernels.swiglu_triton(gate_up), ops.swiglu_ckpt8(gate_up)[0]
    assert torch.equal(torch.isnan(plain), torch.isnan(h))
    assert torch.equal(torch.nan_to_num(plain, nan=0.0, posinf=1.0, neginf=-1.0), torch.nan_to_num(h, nan=0.0, posinf=1.0, neginf=-1.0))


def test_swiglu_ckpt8_nonfinite_groups_poison_only_themselves(cuda_device):
    from hackable_lm_b200 import ops

    gate_up = values((2, 2 * 512), torch.bfloat16, seed=3)
    gate_up[0, 200] = float("nan")          # gate group 1
    gate_up[1, 512 + 511] = float("inf")    # up group 3
    _, q, scale = ops.swiglu_ckpt8(gate_up.to(cuda_device))
    bad = torch.isnan(scale.cpu())
    assert bad.nonzero().tolist() == [[0, 1], [1, 4 + 3]]
    grad = ops.swiglu_ckpt8_backward(q, scale, torch.ones(2, 512, dtype=torch.bfloat16, device=cuda_device)).cpu()
    assert bool(torch.isnan(grad[0, 128:256]).all()) and bool(torch.isnan(grad[0, 512 + 128:512 + 256]).all())
    assert bool(torch.isfinite(grad[0, :128]).all()) and bool(torch.isfinite(grad[0, 256:512]).all())
    assert bool(torch.isnan(grad[1, 384:512]).all()) and bool(torch.isfinite(grad[1, 512:]).all())


def test_swiglu_ckpt8_autograd_strides_and_second_backward(cuda_device):
    from hackable_lm_b200 import kernels, ops

    gate_up = values((6, 8, 2 * 96), torch.bfloat16, seed=8).to(cuda_device)
    x = gate_up.transpose(0, 1).requires_grad_(True)
    h = kernels.swiglu_ckpt8(x)
    d = values((8, 6, 96), torch.bfloat16, seed=9).to(cuda_device)
    (g1,) = torch.autograd.grad(h, x, d.expand(8, 6, 96), retain_graph=True)
    (g2,) = torch.autograd.grad(h, x, d)
    hh, q, scale = ops.swiglu_ckpt8(gate_up.transpose(0, 1))
    assert torch.equal(h, hh) and torch.equal(g1, g2)
    assert torch.equal(g1, ops.swiglu_ckpt8_backward(q, scale, d))
    (g3,) = torch.autograd.grad(kernels.swiglu_ckpt8(x).sum(), x)  # an expanded gradient of ones
    assert torch.equal(g3, ops.swiglu_ckpt8_backward(q, scale, torch.ones_like(d)))


def test_swiglu_ckpt8_offsets_past_32_bits(cuda_device):
    from hackable_lm_b200 import ops

    gate_up = torch.zeros(70000, 32768, dtype=torch.bfloat16, device=cuda_device)
    tail = values((2, 32768), torch.bfloat16, seed=9)
    gate_up[-2:] = tail.to(cuda_device)
    h, q, scale = ops.swiglu_ckpt8(gate_up)
    del gate_up
    eh, eq, es = quant8.swiglu_ckpt8(tail)
    assert torch.equal(q[-2:].cpu(), eq) and torch.equal(scale[-2:].cpu(), es)
    assert not h[:-2].any() and not q[:-2].any()
    grad = ops.swiglu_ckpt8_backward(q, scale, h)
    small = ops.swiglu_ckpt8_backward(q[-2:], scale[-2:], h[-2:])
    assert torch.equal(grad[-2:], small) and not grad[:-2].any()


# ---------------------------------------------------------------------------
# weight gradient from 8 bits
# ---------------------------------------------------------------------------
def _check_wgrad(grad, q, scale, device):
    from hackable_lm_b200 import ops

    y = ops.weight_grad_q8(grad.to(device), q.to(device), scale.to(device))
    e = quant8.weight_grad_q8(grad, q, scale)
    size = grad.double().abs().t() @ quant8.read_back(q, scale).abs()
    E = half_step(grad.dtype)
    m = q.shape[0]
    assert y.dtype == grad.dtype
    # the values read back are rounded to the operand type too: half a subnormal step each
    sub = grad.double().abs().sum(dim=0).unsqueeze(1) * half_subnormal(grad.dtype)
    bound = size * (E + (m + 4) * U) * (1 + 2 * E) + sub + e.abs() * E + half_subnormal(grad.dtype)
    assert_within(y, e, bound, "grad_w")


WGRAD_SHAPES = [  # tokens, N, K
    (1, 8, 16), (2, 16, 32), (63, 24, 16), (64, 128, 128), (65, 136, 144), (127, 256, 256), (200, 520, 272), (333, 8, 2064),
    (1003, 520, 272), (1024, 768, 768), (2500, 264, 528), (4096, 256, 128), (777, 2304, 768)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,N,K", WGRAD_SHAPES)
def test_weight_grad_q8(tokens, N, K, dtype, cuda_device):
    q, scale = codes((tokens, K), seed=tokens)
    _check_wgrad(values((tokens, N), dtype, seed=N, scale=0.1), q, scale, cuda_device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,N,K", [(1000, 2048, 2064), (4090, 2304, 768), (130, 8, 4096)])
def test_weight_grad_q8_wide_tiles_and_splits(tokens, N, K, dtype, cuda_device):
    """Sizes of the 256 x 256 tiles, whole and with the tokens split, and of a row of narrow ones."""
    q, scale = codes((tokens, K), seed=tokens)
    _check_wgrad(values((tokens, N), dtype, seed=N, scale=0.1), q, scale, cuda_device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,N,K", [(1, 24, 48), (2, 264, 272), (63, 24, 16), (65, 520, 2064), (130, 2048, 2304)])
def test_weight_grad_q8_keeps_the_bits_of_what_it_reads_back(tokens, N, K, dtype, cuda_device):
    """The values read back are not rounded to the gradient's type: they are held in two of its
    values, the first cut (within eps of it), the rest rounded, which leaves eps * E of it, and
    in fp16 at most its smallest value.  Their product with fp32 (U), the sum of 2 m terms, the
    result's rounding."""
    from hackable_lm_b200 import ops

    q, scale = codes((tokens, K), seed=tokens)
    grad = values((tokens, N), dtype, seed=N, scale=0.1)
    y = ops.weight_grad_q8(grad.to(cuda_device), q.to(cuda_device), scale.to(cuda_device))
    e = quant8.weight_grad_q8(grad, q, scale)
    size = grad.double().abs().t() @ quant8.read_back(q, scale).abs()
    E = half_step(dtype)
    sub = grad.double().abs().sum(dim=0).unsqueeze(1) * 2 * half_subnormal(dtype)
    bound = size * (2 * E * E + (2 * tokens + 4) * U) + sub
    assert_within(y, e, bound + (e.abs() + bound) * E + half_subnormal(dtype), "grad_w")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,N,K", [(1003, 520, 272), (4096, 256, 128), (4090, 768, 2048)])
def test_weight_grad_q8_is_as_exact_as_its_result_can_be(tokens, N, K, dtype, cuda_device):
    """Over all elements, the error against 64 bits is that of the exact result rounded once: what the
    operands and the sum add is 2^-7 of a half step of the result and less (5% is allowed for)."""
    from hackable_lm_b200 import ops

    q, scale = codes((tokens, K), seed=tokens)
    grad = values((tokens, N), dtype, seed=N, scale=0.1)
    e = quant8.weight_grad_q8(grad, q, scale)
    y = ops.weight_grad_q8(grad.to(cuda_device), q.to(cuda_device), scale.to(cuda_device)).cpu().double()
    assert float((y - e).norm()) <= 1.05 * float((e.to(dtype).double() - e).norm())


# tokens, N, K, columns of a tile, whether the tokens are split (whole: with one and with several tiles a pair)
PLANNED_WGRAD_SHAPES = [(200, 520, 272, 128, False), (500, 6400, 640, 128, False), (1003, 520, 272, 128, True),
                        (20000, 264, 272, 128, True), (1000, 2048, 2064, 256, False), (300, 8192, 4096, 256, False),
                        (4090, 2304, 768, 256, True), (8192, 2304, 768, 256, True), (32768, 768, 2048, 256, True)]


def _wgrad_plan(tokens, N, K):
    import ctypes

    from hackable_lm_b200 import _lib

    columns, splits = ctypes.c_int(), ctypes.c_int()
    _lib.check(_lib.load().hlm_weight_grad_q8_plan(tokens, N, K, ctypes.byref(columns), ctypes.byref(splits)), "plan")
    return columns.value, splits.value


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,N,K,columns,split", PLANNED_WGRAD_SHAPES)
def test_weight_grad_q8_planned_tiles_and_splits(tokens, N, K, columns, split, dtype, cuda_device):
    """Each tile width with the tokens whole and split, against the product in float64 (made on the
    GPU): every element within its own bound, and all together as exact as the exact result rounded
    once (within 5%), so that no part of the tokens is missing or counted twice."""
    from hackable_lm_b200 import ops

    got_columns, splits = _wgrad_plan(tokens, N, K)
    assert (got_columns, splits > 1) == (columns, split)
    q, scale = (t.to(cuda_device) for t in codes((tokens, K), seed=tokens))
    grad = values((tokens, N), dtype, seed=N, scale=0.1).to(cuda_device)
    y = ops.weight_grad_q8(grad, q, scale).double()
    e = quant8.weight_grad_q8(grad, q, scale)
    size = grad.double().abs().t() @ quant8.read_back(q, scale).abs()
    E = half_step(dtype)
    sub = grad.double().abs().sum(dim=0).unsqueeze(1) * 2 * half_subnormal(dtype)
    bound = size * (2 * E * E + (2 * tokens + 4) * U) + sub
    over = (y - e).abs() - bound - (e.abs() + bound) * E - half_subnormal(dtype)
    assert float(over.max()) <= 0, f"over the bound by {float(over.max()):.3e}"
    assert float((y - e).norm()) <= 1.05 * float((e.to(dtype).double() - e).norm())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [50, 3000, 200000])
@pytest.mark.parametrize("least,most,reach", [(2.0 ** 4, 2.0 ** 11, 2.0 ** -12), (2.0 ** -40, 2.0 ** -30, 2.0 ** 13),
                                              (2.0 ** -20, 2.0 ** 5, 2.0 ** -4), (2.0 ** -117, 2.0 ** -110, 2.0 ** 15),
                                              (2.0 ** 105, 2.0 ** 120, 2.0 ** -14)])
def test_weight_grad_q8_scales_outside_the_gradients_type(least, most, reach, tokens, dtype, cuda_device):
    """Codes may stand for values that the gradient's type cannot hold (fp16: over 65504, or below
    2^-24).  Their product with the gradient counts all the same: each value is off as it is
    elsewhere, and in fp16 by at most 2^-24 of a unit that is 2^-7 of the largest scale's power
    of two.  Results beyond the type are infinities there, as for any rounding."""
    from hackable_lm_b200 import ops

    g = torch.Generator().manual_seed(tokens)
    q, _ = codes((tokens, 16), seed=tokens)
    scale = least * (most / least) ** torch.rand(tokens, generator=g, dtype=torch.float64)
    scale = scale.clamp(max=most).float()
    scale[tokens // 2] = most
    grad = (torch.randn(tokens, 8, generator=g) * reach / tokens ** 0.5).to(dtype)
    y = ops.weight_grad_q8(grad.to(cuda_device), q.to(cuda_device), scale.to(cuda_device)).cpu().double()
    e = quant8.weight_grad_q8(grad, q, scale)
    size = grad.double().abs().t() @ quant8.read_back(q, scale).abs()
    E = half_step(dtype)
    unit = most * 2.0 ** -7 if dtype == torch.float16 else 0.0
    bound = size * (2 * E * E + (2 * tokens + 4) * U) + grad.double().abs().sum(dim=0).unsqueeze(1) * unit * 2.0 ** -24
    most_out = torch.finfo(dtype).max
    inside = e.abs() + bound <= most_out
    beyond = e.abs() - bound >= most_out * (1 + E)
    err = (y - e).abs()
    assert bool((err <= bound + (e.abs() + bound) * E + half_subnormal(dtype))[inside].all()), float((err - bound)[inside].max())
    assert torch.equal(y[beyond], e[beyond].sign() * float("inf"))
    assert bool((inside | beyond).any())


def test_weight_grad_q8_infinite_gradients(cuda_device):
    """An infinity in the gradient gives infinities of the products' signs, not NaN, and NaN where
    the value read back is zero; with scales whose values one 16-bit number holds, too."""
    from hackable_lm_b200 import ops

    for dtype in (torch.bfloat16, torch.float16):
        q, scale = codes((40, 32), seed=1)
        scale[3:5] = 0.25
        grad = values((40, 16), dtype, seed=2)
        grad[3, 5], grad[4, 6] = float("inf"), float("-inf")
        q[3, 7] = 0
        q[4, :8] = 1
        y = ops.weight_grad_q8(grad.to(cuda_device), q.to(cuda_device), scale.to(cuda_device)).cpu()
        e = quant8.weight_grad_q8(grad, q, scale).to(dtype)
        assert torch.equal(torch.isnan(y), torch.isnan(e)) and torch.equal(torch.isinf(y), torch.isinf(e))
        bad = torch.isinf(e)
        assert torch.equal(y[bad], e[bad])


def test_weight_grad_q8_same_bits_every_time(cuda_device):
    from hackable_lm_b200 import ops

    q, scale = (t.to(cuda_device) for t in codes((20000, 272), seed=1))
    grad = values((20000, 264), torch.bfloat16, seed=2).to(cuda_device)
    first = ops.weight_grad_q8(grad, q, scale)
    for _ in range(5):
        assert torch.equal(ops.weight_grad_q8(grad, q, scale), first)


def test_weight_grad_q8_empty_and_nonfinite(cuda_device):
    from hackable_lm_b200 import ops

    q, scale = (t.to(cuda_device) for t in codes((100, 48), seed=1))
    grad = values((100, 24), torch.bfloat16, seed=2).to(cuda_device)
    zero = ops.weight_grad_q8(grad[:0], q[:0], scale[:0])
    assert zero.shape == (24, 48) and not zero.any()
    assert ops.weight_grad_q8(grad[:, :0], q, scale).shape == (0, 48)
    grad[3, 5] = float("inf")
    y = ops.weight_grad_q8(grad, q, scale)
    assert bool((~torch.isfinite(y[5])).all()) and bool(torch.isfinite(y[:5]).all()) and bool(torch.isfinite(y[6:]).all())
    scale[50] = float("nan")
    assert bool(torch.isnan(ops.weight_grad_q8(grad, q, scale)).all())


def test_weight_grad_q8_leaves_rows_behind_the_last_token(cuda_device):
    """A padded batch handed over as a view: the rows behind it (NaN here) take no part."""
    from hackable_lm_b200 import ops

    q, scale = (t.to(cuda_device) for t in codes((256, 48), seed=1))
    grad = values((256, 24), torch.bfloat16, seed=2).to(cuda_device)
    expect = ops.weight_grad_q8(grad[:131].clone(), q[:131].clone(), scale[:131].clone())
    grad[131:] = float("nan")
    scale[131:] = float("nan")
    assert torch.equal(ops.weight_grad_q8(grad[:131], q[:131], scale[:131]), expect)


def test_weight_grad_q8_offsets_past_32_bits(cuda_device):
    from hackable_lm_b200 import ops

    grad = torch.zeros(70000, 32768, dtype=torch.bfloat16, device=cuda_device)
    tail = values((5, 32768), torch.bfloat16, seed=1)
    grad[-5:] = tail.to(cuda_device)
    q, scale = codes((70000, 16), seed=2)
    y = ops.weight_grad_q8(grad, q.to(cuda_device), scale.to(cuda_device))
    small = ops.weight_grad_q8(tail.to(cuda_device), q[-5:].to(cuda_device), scale[-5:].to(cuda_device))
    e = quant8.weight_grad_q8(tail, q[-5:], scale[-5:])
    size = tail.double().abs().t() @ quant8.read_back(q[-5:], scale[-5:]).abs()
    E = half_step(torch.bfloat16)
    bound = size * (E + 16 * U) * (1 + 2 * E) + e.abs() * E
    assert_within(y, e, bound, "grad_w")
    assert_within(small, e, bound, "grad_w of the last rows alone")


def test_linear_ckpt8_gradients(cuda_device):
    """y and grad_x are F.linear's; grad_w is the product with the values read back."""
    from hackable_lm_b200 import kernels

    x = values((3, 50, 48), torch.bfloat16, seed=1)
    w = values((24, 48), torch.bfloat16, seed=2, scale=0.1)
    d = values((3, 50, 24), torch.bfloat16, seed=3, scale=0.1)
    xd, wd = x.to(cuda_device).requires_grad_(True), w.to(cuda_device).requires_grad_(True)
    y = kernels.linear_ckpt8(xd, wd)
    gx, gw = torch.autograd.grad(y, (xd, wd), d.to(cuda_device))
    xr, wr = x.to(cuda_device).requires_grad_(True), w.to(cuda_device).requires_grad_(True)
    yr = torch.nn.functional.linear(xr, wr)
    gxr, gwr = torch.autograd.grad(yr, (xr, wr), d.to(cuda_device))
    assert torch.equal(y, yr) and torch.equal(gx, gxr)
    q, scale = quant8.quantize_rows(x)
    flat = d.reshape(150, 24)
    e = quant8.weight_grad_q8(flat, q.reshape(150, 48), scale.reshape(150))
    size = flat.double().abs().t() @ quant8.read_back(q, scale).reshape(150, 48).abs()
    E = half_step(torch.bfloat16)
    assert_within(gw, e, size * (E + 154 * U) * (1 + 2 * E) + e.abs() * E, "grad_w")
    # and against the whole gradient: half a scale per value of x, times the gradients' magnitudes
    half = (scale.double() / 2).reshape(150, 1).expand(150, 48)
    exact = flat.double().t() @ x.double().reshape(150, 48)
    bound = flat.double().abs().t() @ half * (1 + 4 * U) + size * (E + 160 * U) * (1 + 2 * E) + e.abs() * E
    assert_within(gw, exact, bound, "grad_w against the unquantised gradient")
    # a weight that needs no gradient, and no gradient at all
    assert torch.equal(kernels.linear_ckpt8(xd, w.to(cuda_device)), yr)
    with torch.no_grad():
        assert torch.equal(kernels.linear_ckpt8(xd, wd), yr)


# ---------------------------------------------------------------------------
# streams, graphs, other ways to call
# ---------------------------------------------------------------------------
def _all_operators(device, seed=0):
    """Every operator once on fresh inputs: a function that runs them and returns their outputs."""
    from hackable_lm_b200 import kernels, ops

    x = values((150, 256), torch.bfloat16, seed=seed).to(device)
    r = values((150, 256), torch.bfloat16, seed=seed + 1).to(device)
    w, w_scale = (t.to(device) for t in codes((384, 256), seed=seed))
    wl, wl_scale = (t.to(device) for t in codes((64, 192), seed=seed + 1))
    d = values((150, 384), torch.bfloat16, seed=seed + 2).to(device)
    dh = values((150, 192), torch.bfloat16, seed=seed + 3).to(device)

    def run():
        out, q, s = kernels.residual_rms_norm_q8(r, x, 1e-6)
        gate_up = kernels.linear_q8(q, s, w, w_scale)
        h, cq, cs = ops.swiglu_ckpt8(gate_up)
        hq, hs = kernels.quantize_rows(h)
        few = kernels.linear_q8(hq[:20], hs[:20], wl, wl_scale)
        one = kernels.linear_q8(hq[:1], hs[:1], wl, wl_scale, torch.float32)
        return [out, q, s, gate_up, h, cq, cs, hq, hs, few, one, ops.swiglu_ckpt8_backward(cq, cs, dh),
                ops.weight_grad_q8(d, q, s), kernels.dequantize_rows(q, s)]

    return run, (x, r)


def test_side_stream_and_two_streams_at_once(cuda_device):
    a, _ = _all_operators(cuda_device, 0)
    b, _ = _all_operators(cuda_device, 50)
    ea, eb = a(), b()
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(sa):
            ga = a()
        with torch.cuda.stream(sb):
            gb = b()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ea, ga)) and all(torch.equal(p, q) for p, q in zip(eb, gb))


def test_two_threads_at_once(cuda_device):
    """The calls release the interpreter lock: threads with a stream each get their own results."""
    import threading

    runs = [_all_operators(cuda_device, seed)[0] for seed in (0, 50)]
    expected = [run() for run in runs]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = runs[i]()
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for e, g in zip(expected, got):
        assert g is not None and all(torch.equal(p, q) for p, q in zip(e, g))


def test_captured_and_replayed_with_other_inputs(cuda_device):
    a, (x, r) = _all_operators(cuda_device, 0)
    b, _ = _all_operators(cuda_device, 50)
    a(), b()
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        oa = a()
    with torch.cuda.graph(gb):
        ob = b()
    x.copy_(values((150, 256), torch.bfloat16, seed=77).to(cuda_device))
    expect_a, expect_b = a(), b()
    for _ in range(3):
        ga.replay()
        gb.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(oa, expect_a))
    assert all(torch.equal(p, q) for p, q in zip(ob, expect_b))
    # on two streams at once
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(sa):
            ga.replay()
        with torch.cuda.stream(sb):
            gb.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(oa, expect_a))
    assert all(torch.equal(p, q) for p, q in zip(ob, expect_b))


@pytest.mark.parametrize("captured", [False, True])
def test_neighbours_of_other_kinds_in_the_stream(captured, cuda_device):
    """The kernels are set up while the work before them in the stream still runs.  Whatever that is
    (a copy, a fill, a torch kernel, a join of another stream) is waited for, and what follows waits
    for them; run many times over the same buffers, eagerly and captured."""
    from hackable_lm_b200 import kernels, ops

    rows, cols = 3000, 768
    src = [values((rows, cols), torch.bfloat16, seed=i).to(cuda_device) for i in range(4)]
    w, ws = kernels.quantize_rows(values((384, cols), torch.bfloat16, seed=9).to(cuda_device))
    x, r = torch.empty_like(src[0]), torch.empty_like(src[0])
    side = torch.cuda.Stream()

    def run(i):
        main = torch.cuda.current_stream()
        x.copy_(src[i % 4])                       # a device copy, then a kernel that reads it
        r.fill_(0.5)                              # a fill
        out, q, s = kernels.residual_rms_norm_q8(r, x, 1e-6)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            y = kernels.linear_q8(q, s, w, ws)    # on another stream
        main.wait_stream(side)
        h, cq, cs = ops.swiglu_ckpt8(y)           # after the join
        g = h.mul(2.0)                            # a torch kernel between two of the library's
        x.zero_()                                 # overwrites what the first kernel read
        grad = ops.swiglu_ckpt8_backward(cq, cs, g)
        gw = ops.weight_grad_q8(grad, q, s)
        few = kernels.linear_q8(q[:7], s[:7], w, ws, torch.float32)
        back = kernels.dequantize_rows(q, s)
        return [t.clone() for t in (out, y, h, grad, gw, few, back)]

    torch.cuda.synchronize()
    expect = []
    for i in range(4):
        expect.append(run(i))
        torch.cuda.synchronize()
    runs = []
    if captured:
        for i in range(4):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = run(i)
            runs.append((graph, got))
    for _ in range(20):
        for i in range(4):
            if captured:
                runs[i][0].replay()
                got = runs[i][1]
            else:
                got = run(i)
            checks = [torch.equal(a, b) for a, b in zip(got, expect[i])] if _ % 5 == 4 else []
            assert all(checks), (i, checks)
    torch.cuda.synchronize()


def test_backward_captured_while_an_eager_graph_lives(cuda_device):
    """The checkpoint operators' backward, captured with its forward on a side stream, beside an
    eager graph of the same leaves made on that stream.  (One made on the default stream keeps the
    leaves' accumulation nodes there, and autograd then waits on the default stream inside the
    capture, which CUDA refuses for any differentiable operator.)"""
    from hackable_lm_b200 import kernels

    x = values((64, 48), torch.bfloat16, seed=1).to(cuda_device).requires_grad_(True)
    w = values((96, 48), torch.bfloat16, seed=2, scale=0.1).to(cuda_device).requires_grad_(True)

    def step():
        h = kernels.swiglu_ckpt8(kernels.linear_ckpt8(x, w))
        return torch.autograd.grad(h.float().sum(), (x, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        live = kernels.swiglu_ckpt8(kernels.linear_ckpt8(x, w))  # an eager graph of the same leaves
        for _ in range(2):
            expect = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, expect))
    with torch.cuda.stream(side):
        again = torch.autograd.grad(live.float().sum(), (x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(again, expect))


def test_first_calls_of_a_process_inside_a_capture(cuda_device, tmp_path):
    """A process whose first call of each operator is captured: it works, or it is refused with an
    error; the process goes on and the next, uncaptured call gives the right result."""
    import subprocess
    import sys
    from pathlib import Path

    script = tmp_path / "first.py"
    script.write_text(
        "import sys, torch\n"
        f"sys.path.insert(0, {str(Path(__file__).resolve().parents[1])!r})\n"
        "from hackable_lm_b200 import kernels, ops\n"
        "x = torch.randn(200, 256, device='cuda', dtype=torch.bfloat16)\n"
        "def run():\n"
        "    q, s = kernels.quantize_rows(x)\n"
        "    y = kernels.linear_q8(q, s, q, s)\n"
        "    one = kernels.linear_q8(q[:1], s[:1], q, s)\n"
        "    out, nq, ns = kernels.residual_rms_norm_q8(x, x, 1e-6)\n"
        "    h, cq, cs = ops.swiglu_ckpt8(x)\n"
        "    return y, one, out, ns, ops.swiglu_ckpt8_backward(cq, cs, h), ops.weight_grad_q8(x, q, s), kernels.dequantize_rows(q, s)\n"
        "torch.cuda.synchronize()\n"
        "g = torch.cuda.CUDAGraph()\n"
        "try:\n"
        "    with torch.cuda.graph(g):\n"
        "        got = run()\n"
        "    g.replay()\n"
        "    torch.cuda.synchronize()\n"
        "    print('captured')\n"
        "except RuntimeError as e:\n"
        "    got = None\n"
        "    print('refused', str(e)[:200])\n"
        "expect = run()\n"
        "torch.cuda.synchronize()\n"
        "assert got is None or all(torch.equal(a, b) for a, b in zip(got, expect))\n"
        "print('done')\n")
    out = subprocess.run([sys.executable, str(script)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip().endswith("done"), out.stdout + out.stderr
    print(out.stdout)


def test_gradient_asked_of_an_integer_output_is_refused(cuda_device):
    from hackable_lm_b200 import kernels

    x = values((4, 32), torch.bfloat16).to(cuda_device).requires_grad_(True)
    _, scale = kernels.quantize_rows(x)
    with pytest.raises(RuntimeError):
        scale.sum().backward()
    out, _, _ = kernels.residual_rms_norm_q8(x, x.detach(), 1e-6)
    with pytest.raises(RuntimeError):
        out.sum().backward()


@pytest.mark.parametrize("name", sorted(bad_calls("meta")))
def test_argument_checks(name, cuda_device):
    from hackable_lm_b200 import _lib

    before = _lib.launch_count()
    with pytest.raises(RuntimeError):
        bad_calls(cuda_device)[name]()
    assert _lib.launch_count() == before


def test_unsupported_sizes_raise_the_library_error(cuda_device):
    """K that is no multiple of 16, or too long; N of the gradient no multiple of 8."""
    from hackable_lm_b200 import _lib, kernels, ops

    def c(rows, cols):
        return torch.zeros(rows, cols, dtype=torch.int8, device=cuda_device), torch.ones(rows, device=cuda_device)

    for k in (24, 131072):
        with pytest.raises(_lib.HlmError, match="unsupported"):
            kernels.linear_q8(*c(2, k), *c(3, k))
    g = torch.zeros(5, 12, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(_lib.HlmError, match="unsupported"):
        ops.weight_grad_q8(g, *c(5, 32))
    with pytest.raises(_lib.HlmError, match="unsupported"):
        ops.weight_grad_q8(g[:, :8], *c(5, 24))
    with pytest.raises(RuntimeError):
        kernels.linear_ckpt8(g.float().requires_grad_(True), torch.zeros(8, 12, device=cuda_device, requires_grad=True))


def test_linear_ckpt8_keeps_its_type_under_autocast(cuda_device):
    from hackable_lm_b200 import kernels

    x = values((20, 48), torch.bfloat16, seed=1).to(cuda_device).requires_grad_(True)
    w = values((24, 48), torch.bfloat16, seed=2, scale=0.1).to(cuda_device).requires_grad_(True)
    y = kernels.linear_ckpt8(x, w)
    grads = torch.autograd.grad(y.sum(), (x, w))
    with torch.autocast("cuda", dtype=torch.float16):
        y2 = kernels.linear_ckpt8(x, w)
        with torch.no_grad():
            assert torch.equal(y, kernels.linear_ckpt8(x, w))
    assert y2.dtype == torch.bfloat16 and torch.equal(y, y2)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(y2.sum(), (x, w))))


def test_modes_and_transforms_see_the_operators(cuda_device):
    """Under a dispatch mode the registered operator runs (and is seen); the result is the same."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from hackable_lm_b200 import kernels

    seen = []

    class Recorder(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    x = values((5, 64), torch.bfloat16).to(cuda_device)
    q, scale = kernels.quantize_rows(x)
    with Recorder():
        q2, scale2 = kernels.quantize_rows(x)
    assert any("hackable_lm_b200.quantize_rows" in s for s in seen)
    assert torch.equal(q, q2) and torch.equal(scale, scale2)
    neg = torch._neg_view(x)  # a lazily negated view: its storage holds the other sign
    q3, scale3 = kernels.quantize_rows(neg)
    assert torch.equal(q3, -q) and torch.equal(scale3, scale)


def test_traced_operators_are_recorded(cuda_device):
    """torch.jit.trace records the operators, not the values of the traced call."""
    from hackable_lm_b200 import kernels

    x, y = values((5, 64), torch.bfloat16, seed=1).to(cuda_device), values((5, 64), torch.bfloat16, seed=2).to(cuda_device)
    traced = torch.jit.trace(lambda t: kernels.dequantize_rows(*kernels.quantize_rows(t)), x, check_trace=False)
    assert torch.equal(traced(y), kernels.dequantize_rows(*kernels.quantize_rows(y)))


def test_forward_mode_derivatives_are_refused(cuda_device):
    """A tangent is never dropped in silence."""
    import torch.autograd.forward_ad as fw

    from hackable_lm_b200 import kernels, ops

    x = values((4, 64), torch.bfloat16, seed=1).to(cuda_device)
    w = values((16, 64), torch.bfloat16, seed=2).to(cuda_device)
    q, scale = kernels.quantize_rows(x)
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        ds = fw.make_dual(scale, torch.ones_like(scale))
        for call in (lambda: kernels.quantize_rows(d), lambda: kernels.rms_norm_q8(d, None, 1e-6),
                     lambda: kernels.residual_rms_norm_q8(x, d, 1e-6), lambda: kernels.dequantize_rows(q, ds),
                     lambda: kernels.linear_q8(q, ds, q, scale), lambda: ops.swiglu_ckpt8(d),
                     lambda: kernels.linear_ckpt8(d, w.requires_grad_(True))):
            with pytest.raises(RuntimeError, match="forward"):
                call()


@pytest.mark.parametrize("name", ["quantize_rows", "dequantize_rows", "rms_norm_q8", "residual_rms_norm_q8", "linear_q8",
                                  "swiglu_ckpt8", "swiglu_ckpt8_backward", "weight_grad_q8", "linear_ckpt8"])
def test_opcheck(name, cuda_device):
    x = values((5, 64), torch.bfloat16).to(cuda_device)
    q, s = (t.to(cuda_device) for t in codes((5, 64), seed=1))
    w, ws = (t.to(cuda_device) for t in codes((24, 64), seed=2))
    gs = torch.rand(5, 2, device=cuda_device)
    args = {
        "quantize_rows": (x,), "dequantize_rows": (q, s, torch.float16), "rms_norm_q8": (x, None, 1e-6),
        "residual_rms_norm_q8": (x, x.clone(), x[0].clone(), 1e-6), "linear_q8": (q, s, w, ws, torch.bfloat16),
        "swiglu_ckpt8": (x.clone().requires_grad_(True),), "swiglu_ckpt8_backward": (q, gs, x[:, :32].contiguous()),
        "weight_grad_q8": (x, q, s),
        "linear_ckpt8": (x.clone().requires_grad_(True), x[:, :64].repeat(5, 1)[:24].clone().requires_grad_(True)),
    }[name]
    torch.library.opcheck(getattr(torch.ops.hackable_lm_b200, name).default, args)


def test_chain_of_8_bit_operators(cuda_device):
    """norm -> projection -> SwiGLU -> quantise -> projection, as the int8 model runs them, against
    the same chain in 64 bits.  Each link is checked on the values that the link before gave."""
    from hackable_lm_b200 import kernels

    for rows in (1, 6, 40, 300):
        r, x = values((rows, 256), torch.bfloat16, seed=1), values((rows, 256), torch.bfloat16, seed=2)
        w1, s1 = quant8.quantize_rows(values((512, 256), torch.float32, seed=3, scale=0.05))
        w2, s2 = quant8.quantize_rows(values((256, 256), torch.float32, seed=4, scale=0.05))
        dev = [t.to(cuda_device) for t in (r, x, w1, s1, w2, s2)]
        out, q, s = kernels.residual_rms_norm_q8(dev[0], dev[1], 1e-6)
        gate_up = kernels.linear_q8(q, s, dev[2], dev[3])
        h = kernels.swiglu_ckpt8(gate_up)
        hq, hs = kernels.quantize_rows(h)
        y = kernels.linear_q8(hq, hs, dev[4], dev[5])
        eo, eq, es = quant8.rms_norm_q8(r, x, None, 1e-6)
        e1 = quant8.linear_q8(eq, s.cpu(), w1, s1)
        E = half_step(torch.bfloat16)
        assert_within(gate_up, e1, e1.abs() * (3 * U + E), "gate_up")
        g, u = gate_up.cpu().double().chunk(2, dim=-1)
        eh = g * torch.sigmoid(g) * u
        assert_within(h, eh, eh.abs() * ((2 * g.abs() + 16) * U + E) + 2.0 ** -126, "h")
        ehq, ehs = quant8.quantize_rows(h.cpu())
        assert torch.equal(hq.cpu(), ehq) and torch.equal(hs.cpu(), ehs)
        e2 = quant8.linear_q8(ehq, ehs, w2, s2)
        assert_within(y, e2, e2.abs() * (3 * U + E), "y")
