"""Host side of the 8-bit operators: refusals, shapes on meta tensors, and the oracle itself."""
from __future__ import annotations

import ctypes

import pytest
import torch

from hackable_lm_b200 import _lib, kernels, ops
from oracle import quant8


def test_c_entry_points_refuse_bad_arguments_before_any_launch():
    lib = _lib.load()
    V, BF, F32, F16 = ctypes.c_void_p(16), _lib.HLM_BF16, _lib.HLM_F32, _lib.HLM_F16
    odd = ctypes.c_void_p(24)
    assert lib.hlm_quantize_rows(V, V, V, -1, 8, BF, None) == -1
    assert lib.hlm_quantize_rows(V, V, V, 4, 0, BF, None) == -1
    assert lib.hlm_quantize_rows(None, V, V, 4, 8, BF, None) == -1
    assert lib.hlm_quantize_rows(V, V, V, 4, 8, 7, None) == -2
    assert lib.hlm_quantize_rows(None, None, None, 0, 8, BF, None) == 0
    assert lib.hlm_dequantize_rows(V, None, V, 4, 8, BF, None) == -1
    assert lib.hlm_dequantize_rows(V, V, V, 4, 8, 9, None) == -2
    assert lib.hlm_residual_rms_norm_q8(V, V, None, None, V, V, 4, 8, 1e-6, BF, None) == -1  # residual without out
    assert lib.hlm_residual_rms_norm_q8(None, V, None, None, V, V, 4, 0, 1e-6, BF, None) == -1
    assert lib.hlm_residual_rms_norm_q8(None, V, None, None, V, V, 4, 8, 1e-6, 5, None) == -2
    assert lib.hlm_linear_q8(V, V, V, V, V, -1, 8, 16, BF, None) == -1
    assert lib.hlm_linear_q8(V, V, V, V, None, 1, 8, 16, BF, None) == -1
    assert lib.hlm_linear_q8(V, V, V, V, V, 1, 8, 0, BF, None) == -2
    assert lib.hlm_linear_q8(V, V, V, V, V, 1, 8, 24, BF, None) == -2
    assert lib.hlm_linear_q8(V, V, V, V, V, 1, 8, 131056 + 16, BF, None) == -2
    assert lib.hlm_linear_q8(V, V, V, V, V, 1, 8, 16, 4, None) == -2
    assert lib.hlm_linear_q8(odd, V, V, V, V, 1, 8, 16, BF, None) == -2
    assert lib.hlm_linear_q8(V, V, odd, V, V, 1, 8, 16, F16, None) == -2
    assert lib.hlm_linear_q8(None, None, None, None, None, 0, 8, 16, F32, None) == 0
    assert lib.hlm_swiglu_ckpt8_fwd(V, V, V, V, -1, 8, BF, None) == -1
    assert lib.hlm_swiglu_ckpt8_fwd(V, V, None, V, 1, 8, BF, None) == -1
    assert lib.hlm_swiglu_ckpt8_fwd(V, V, V, V, 1, 8, 3, None) == -2
    assert lib.hlm_swiglu_ckpt8_bwd(V, V, V, None, 1, 8, BF, None) == -1
    assert lib.hlm_swiglu_ckpt8_bwd(None, None, None, None, 0, 8, BF, None) == 0
    assert lib.hlm_weight_grad_q8(V, V, V, V, None, 0, -1, 8, 16, BF, None) == -1
    assert lib.hlm_weight_grad_q8(V, V, V, None, None, 0, 4, 8, 16, BF, None) == -1
    assert lib.hlm_weight_grad_q8(V, V, V, V, None, 0, 4, 12, 16, BF, None) == -2
    assert lib.hlm_weight_grad_q8(V, V, V, V, None, 0, 4, 8, 24, BF, None) == -2
    assert lib.hlm_weight_grad_q8(V, V, V, V, None, 0, 4, 8, 16, F32, None) == -2
    assert lib.hlm_weight_grad_q8(V, odd, V, V, None, 0, 4, 8, 16, BF, None) == -2


def test_plan_queries():
    lib = _lib.load()
    a, b = ctypes.c_int(-7), ctypes.c_int(-7)
    assert lib.hlm_linear_q8_plan(1, 4096, 768, _lib.HLM_BF16, None) == -1
    assert lib.hlm_linear_q8_plan(0, 4096, 768, _lib.HLM_BF16, a) == -1
    assert lib.hlm_linear_q8_plan(1, 4096, 24, _lib.HLM_BF16, a) == -2
    assert lib.hlm_linear_q8_plan(1, 4096, 131072, _lib.HLM_BF16, a) == -2
    assert lib.hlm_linear_q8_plan(1, 4096, 768, 5, a) == -2
    assert lib.hlm_weight_grad_q8_plan(0, 8, 16, a, b) == -1
    assert lib.hlm_weight_grad_q8_plan(1, 8, 16, None, b) == -1
    assert a.value == b.value == -7
    assert lib.hlm_linear_q8_plan(1, 4096, 768, _lib.HLM_BF16, a) == 0 and a.value == 0
    assert lib.hlm_linear_q8_plan(32768, 4096, 768, _lib.HLM_F32, a) == 0 and a.value == -256
    assert lib.hlm_weight_grad_q8_plan(32768, 4096, 768, a, b) == 0 and a.value == 256 and b.value > 1
    for tokens, N, K in ((1, 8, 16), (1003, 520, 272), (32768, 768, 2048)):
        assert lib.hlm_weight_grad_q8_plan(tokens, N, K, a, b) == 0 and b.value >= 1
        parts = 4 * N * K * b.value if b.value > 1 else 0
        need = lib.hlm_weight_grad_q8_workspace_bytes(tokens, N, K)
        assert need >= 4 * tokens * K + parts


def test_cpu_tensors_are_rejected():
    x = torch.randn(4, 32, dtype=torch.bfloat16)
    q, s = torch.zeros(4, 32, dtype=torch.int8), torch.ones(4)
    calls = [lambda: kernels.quantize_rows(x), lambda: kernels.dequantize_rows(q, s), lambda: kernels.rms_norm_q8(x, None, 1e-6),
             lambda: kernels.residual_rms_norm_q8(x, x, 1e-6), lambda: kernels.linear_q8(q, s, q, s),
             lambda: kernels.swiglu_ckpt8(x), lambda: kernels.linear_ckpt8(x, x), lambda: ops.weight_grad_q8(x, q, s),
             lambda: ops.swiglu_ckpt8_backward(q, torch.ones(4, 2), x[:, :16]), lambda: ops.quantize_rows(x)]
    for call in calls:
        with pytest.raises(RuntimeError):
            call()


def bad_calls(device):
    """Calls whose shapes or types do not fit together."""
    def t(shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device=device)

    x, q, s = t((4, 32)), t((4, 32), torch.int8), t(4, torch.float32)
    return {
        "other K": lambda: ops.linear_q8(q, s, q[:, :16], s), "weight of one dimension": lambda: ops.linear_q8(q, s, q[0], s[0]),
        "scales of other rows": lambda: ops.linear_q8(q, s[:3], q, s), "not codes": lambda: ops.linear_q8(x, s, q, s),
        "weight scales of other rows": lambda: ops.linear_q8(q, s, q, s[:2]),
        "output type": lambda: ops.linear_q8(q, s, q, s, torch.int32), "scales in 16 bits": lambda: ops.linear_q8(q, s.half(), q, s),
        "codes again": lambda: ops.quantize_rows(q), "no columns": lambda: ops.quantize_rows(t((4, 0))),
        "a number": lambda: ops.quantize_rows(t(())), "read back type": lambda: ops.dequantize_rows(q, s, torch.float64),
        "read back scales": lambda: ops.dequantize_rows(q, s.half(), torch.float32),
        "norm rows": lambda: ops.residual_rms_norm_q8(x, x[:2], None, 1e-6),
        "norm types": lambda: ops.residual_rms_norm_q8(x, x.float(), None, 1e-6),
        "norm weight": lambda: ops.rms_norm_q8(x, t(5), 1e-6), "norm of doubles": lambda: ops.rms_norm_q8(x.double(), None, 1e-6),
        "odd width": lambda: ops.swiglu_ckpt8(t((2, 7))), "gate_up type": lambda: ops.swiglu_ckpt8(q),
        "scales of another width": lambda: ops.swiglu_ckpt8_backward(q, t((4, 4), torch.float32), x[:, :16]),
        "gradient of another width": lambda: ops.swiglu_ckpt8_backward(q, t((4, 2), torch.float32), x),
        "gradient in 32 bits": lambda: ops.weight_grad_q8(x.float(), q, s),
        "gradient of other rows": lambda: ops.weight_grad_q8(x[:3], q, s),
    }


@pytest.mark.parametrize("name", sorted(bad_calls("meta")))
def test_argument_checks_on_meta_tensors(name):
    with pytest.raises(RuntimeError):
        bad_calls("meta")[name]()


def test_shapes_on_meta_tensors():
    x = torch.empty(2, 3, 64, device="meta", dtype=torch.bfloat16)
    q, s = kernels.quantize_rows(x)
    assert q.shape == x.shape and q.dtype == torch.int8 and s.shape == (2, 3) and s.dtype == torch.float32
    assert kernels.dequantize_rows(q, s, torch.float16).dtype == torch.float16
    out, q, s = kernels.residual_rms_norm_q8(x, x, 1e-6)
    assert out.dtype == torch.bfloat16 and q.shape == x.shape
    w, ws = torch.empty(40, 64, device="meta", dtype=torch.int8), torch.empty(40, device="meta")
    assert kernels.linear_q8(q, s, w, ws).shape == (2, 3, 40)
    gu = torch.empty(2, 3, 400, device="meta", dtype=torch.bfloat16, requires_grad=True)
    h = kernels.swiglu_ckpt8(gu)
    h.sum().backward()
    assert h.shape == (2, 3, 200) and gu.grad.shape == gu.shape
    assert ops.swiglu_ckpt8(gu)[2].shape == (2, 3, 4)
    xw = torch.empty(2, 3, 64, device="meta", dtype=torch.bfloat16, requires_grad=True)
    wf = torch.empty(40, 64, device="meta", dtype=torch.bfloat16, requires_grad=True)
    kernels.linear_ckpt8(xw, wf).sum().backward()
    assert xw.grad.shape == xw.shape and wf.grad.shape == wf.shape


def test_oracle_codes_are_within_half_a_scale():
    v = torch.randn(50, 300, generator=torch.Generator().manual_seed(0)) * 3
    q, s = quant8.quantize(v)
    err = (quant8.read_back(q, s) - v.double()).abs()
    # half a scale, and the roundings of 127 / a, the product (each 127 u of a code at most) and a / 127
    assert bool((err <= s.double().unsqueeze(-1) * (0.5 + 4 * 127 * 2.0 ** -24)).all())
    assert int(q.abs().max()) == 127


def test_oracle_swiglu_gradient_against_differences():
    """The checkpoint's gradient is the derivative of silu(gate) * up at the values read back."""
    g = torch.Generator().manual_seed(1)
    gate_up = torch.randn(3, 2 * 200, generator=g)
    d = torch.randn(3, 200, generator=g)
    _, q, s = quant8.swiglu_ckpt8(gate_up)
    grad = quant8.swiglu_ckpt8_backward(q, s, d)
    qg, qu = q.chunk(2, dim=-1)
    sg, su = s.chunk(2, dim=-1)
    gate, up = quant8.group_read_back(qg, sg), quant8.group_read_back(qu, su)
    f = lambda a, b: d.double() * a * torch.sigmoid(a) * b  # noqa: E731
    e = 1e-5  # central differences: error e^2 / 6 * third derivative (below 1.5 |d u|) + 1e-16 / e
    dg = (f(gate + e, up) - f(gate - e, up)) / (2 * e)
    du = (f(gate, up + e) - f(gate, up - e)) / (2 * e)
    tol = 1e-9 * (1 + (d.double() * up).abs().max() + (d.double() * gate).abs().max())
    assert (grad - torch.cat((dg, du), dim=-1)).abs().max() <= tol


def test_activation_checkpoint_config():
    from hackable_lm_b200.config import model_config_for_depth
    from hackable_lm_b200.model import LanguageModel

    assert model_config_for_depth(2).activation_checkpoint == "none"
    assert model_config_for_depth(2, activation_checkpoint="INT8").activation_checkpoint == "int8"
    with pytest.raises(ValueError):
        model_config_for_depth(2, activation_checkpoint="int4")
    with pytest.raises(RuntimeError):
        LanguageModel(model_config_for_depth(2, vocab_size=64, backend="torch", activation_checkpoint="int8"))
    with pytest.raises(RuntimeError):
        LanguageModel(model_config_for_depth(2, vocab_size=64)).quantize_int8()


def test_config_without_the_checkpoint_field():
    """A config object of the reference's fields alone builds the model, as before the field was there."""
    from types import SimpleNamespace

    from hackable_lm_b200.config import model_config_for_depth
    from hackable_lm_b200.model import LanguageModel

    fields = model_config_for_depth(2, vocab_size=64, sequence_len=32, backend="torch", attention_backend="torch").to_dict()
    del fields["activation_checkpoint"], fields["extra"]
    model = LanguageModel(SimpleNamespace(**fields))
    idx = torch.zeros(1, 8, dtype=torch.long)
    _, loss = model(idx, idx)
    loss.backward()
    assert bool(torch.isfinite(loss)) and not model.blocks[0].mlp.keep_int8


def test_int8_model_refuses_a_negative_loss_chunk():
    from hackable_lm_b200.config import model_config_for_depth
    from hackable_lm_b200.model import LanguageModel

    with torch.device("meta"):
        model = LanguageModel(model_config_for_depth(2, vocab_size=64, sequence_len=32, loss_chunk_size=-1))
    with pytest.raises(RuntimeError, match="nonnegative"):
        model.quantize_int8()


def test_int8_linear_keeps_its_scales_in_32_bits():
    from hackable_lm_b200.quantized import Int8Linear

    lin = Int8Linear(torch.empty(24, 32, device="meta", dtype=torch.bfloat16))
    lin = lin.to_empty(device="cpu")
    scale = torch.rand(24)
    lin.weight.zero_()
    lin.weight_scale.copy_(scale)
    for move in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.float()):
        move(lin)
        assert lin.weight.dtype == torch.int8
        assert lin.weight_scale.dtype == torch.float32 and torch.equal(lin.weight_scale, scale)
    assert torch.equal(lin.state_dict()["weight_scale"], scale)


def test_models_on_meta_tensors_reach_the_operators():
    from hackable_lm_b200.config import model_config_for_depth
    from hackable_lm_b200.model import LanguageModel

    with torch.device("meta"):
        model = LanguageModel(model_config_for_depth(2, vocab_size=64, sequence_len=128, activation_checkpoint="int8"))
        model = model.to(torch.bfloat16)
        idx = torch.zeros(2, 128, dtype=torch.long)
        kinds = []

        def keep(t):
            kinds.append(t.dtype)
            return t

        with torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t):
            _, loss = model(idx, idx)
        loss.backward()
        assert torch.int8 in kinds and all(p.grad is not None for p in model.parameters())
        logits, _ = model.quantize_int8()(idx)
        assert logits.shape == (2, 128, 64) and logits.dtype == torch.bfloat16
