"""The model on the 8-bit operators: int8 inference and 8-bit activation checkpoints in training."""
from __future__ import annotations

import pytest
import torch

from hackable_lm_b200.config import model_config_for_depth
from hackable_lm_b200.model import LanguageModel

pytestmark = pytest.mark.gpu


def _model(device, depth=4, **kw):
    torch.manual_seed(0)
    cfg = model_config_for_depth(depth, vocab_size=512, sequence_len=256, **kw)
    return LanguageModel(cfg).to(device).to(torch.bfloat16)


def _tokens(device, batch=2, length=256, vocab=512):
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, vocab, (batch, length + 1), generator=g).to(device)
    return ids[:, :-1].contiguous(), ids[:, 1:].contiguous()


def _rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("length", [1, 37, 256])
@pytest.mark.parametrize("window", [None, 64])
def test_int8_model_against_bf16_model(length, window, cuda_device):
    """Rounding a row to 8 bits moves it by a / 127 / sqrt(12) for a magnitude a of about four times
    its rms: 0.9% of its norm; a projection whose input and weight are both rounded is 1.3% off,
    and four of them in each of four blocks and the LM head add up to at most sqrt(17) 1.3% = 5.4%
    of the logits (less: the residual stream carries most).  Held to twice that."""
    model = _model(cuda_device, attention_window=window)
    x, y = _tokens(cuda_device, length=length)
    quantized = model.quantize_int8()
    with torch.no_grad():
        logits, none = model(x)
    got, none8 = quantized(x)
    assert none is None and none8 is None and got.shape == logits.shape and got.dtype == logits.dtype
    assert not got.requires_grad
    assert _rel(got, logits) < 0.11
    # logits this far apart move the loss by at most their largest difference, on average far less
    _, loss = quantized(x, y)
    with torch.no_grad():
        _, loss16 = model(x, y)
    assert abs(float(loss) - float(loss16)) <= float((got.float() - logits.float()).abs().max()) + 1e-2
    y2 = y.clone()
    y2[0, 0] = -100
    _, ignored = quantized(x, y2)
    per = torch.nn.functional.cross_entropy(got.float().reshape(-1, 512), y2.reshape(-1))
    assert torch.isnan(per) == torch.isnan(ignored) and (torch.isnan(per) or abs(float(per) - float(ignored)) < 1e-2)


def test_int8_model_targets_like_the_bf16_models(cuda_device):
    """32-bit targets are taken; targets outside the vocabulary are left out of the mean, as the bf16
    model's fused loss leaves them out."""
    model = _model(cuda_device, depth=2)
    quantized = model.quantize_int8()
    x, y = _tokens(cuda_device)
    assert torch.equal(quantized(x, y.to(torch.int32))[1], quantized(x, y)[1])
    ignored, odd = y.clone(), y.clone()
    ignored[0, :5] = -100
    odd[0, :5] = torch.tensor([-1, 512, 2 ** 40, -2 ** 40, -100], device=cuda_device)
    expect = quantized(x, ignored)[1]
    assert torch.equal(quantized(x, odd)[1], expect) and bool(torch.isfinite(expect))
    with torch.no_grad():
        assert torch.equal(model(x, odd)[1], model(x, ignored)[1])
        none = torch.full_like(y, -1)
        assert bool(torch.isnan(model(x, none)[1])) and bool(torch.isnan(quantized(x, none)[1]))


def test_int8_model_weights_and_state(cuda_device):
    model = _model(cuda_device, depth=2)
    quantized = model.quantize_int8()
    w = quantized.dequantized_weights()
    assert len(w) == 2 * 4 + 1
    got, weight = w["blocks.1.gate_up_proj"], model.blocks[1].mlp.gate_up.gate_up_proj.weight
    step = weight.float().abs().amax(dim=1, keepdim=True) / 127
    # half a step, and the rounding of the value read back to bf16
    assert bool(((got.float() - weight.float()).abs() <= 0.5001 * step + weight.float().abs() * 2 ** -8).all())
    state = quantized.state_dict()
    assert state["lm_head.weight"].dtype == torch.int8 and state["lm_head.weight_scale"].dtype == torch.float32
    other = _model(cuda_device, depth=2)
    with torch.no_grad():
        for p in other.parameters():
            p.zero_()
    other = other.quantize_int8()
    other.load_state_dict(state)
    x, _ = _tokens(cuda_device)
    assert torch.equal(other(x)[0], quantized(x)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_int8_model_in_another_type(dtype, cuda_device):
    """A move to another type is for the stream between the projections: the codes and their scales
    stay.  A wider or other 16-bit stream moves each of its roundings by at most two half steps of
    bf16, 2^-7 of a value, well inside the 5.4% that the 8-bit rounding itself is given above."""
    quantized = _model(cuda_device, depth=2).quantize_int8()
    x, y = _tokens(cuda_device)
    logits, (_, loss) = quantized(x)[0], quantized(x, y)
    scales = {n: b.clone() for n, b in quantized.named_buffers() if n.endswith("weight_scale")}
    moved = quantized.to(dtype)
    assert moved is quantized and quantized.tok_emb.weight.dtype == dtype
    for n, b in quantized.named_buffers():
        if n.endswith("weight_scale"):
            assert b.dtype == torch.float32 and torch.equal(b, scales[n])
        elif n.endswith("weight"):
            assert b.dtype == torch.int8
    got, _ = quantized(x)
    _, got_loss = quantized(x, y)
    assert got.dtype == dtype and _rel(got, logits) < 0.054
    assert abs(float(got_loss) - float(loss)) <= float((got.double() - logits.double()).abs().max()) + 1e-2
    back, _ = quantized.to("cpu").to(cuda_device)(x)
    assert torch.equal(back, got)
    if dtype == torch.bfloat16:
        assert torch.equal(got, logits)


def test_int8_model_is_a_snapshot(cuda_device):
    """What happens to the model afterwards does not reach the 8-bit one."""
    model = _model(cuda_device, depth=2)
    quantized = model.quantize_int8()
    x, _ = _tokens(cuda_device)
    before = quantized(x)[0]
    with torch.no_grad():
        for p in model.parameters():
            p.mul_(0.5)
    model.to("cpu")
    assert torch.equal(quantized(x)[0], before)


def test_int8_model_compiled(cuda_device):
    """torch.compile of the 8-bit model runs the registered operators: the same bits where the
    surrounding operations are the same kernels."""
    quantized = _model(cuda_device, depth=2).quantize_int8()
    x, _ = _tokens(cuda_device)
    eager = quantized(x)[0]
    compiled = torch.compile(quantized, fullgraph=True, dynamic=False)(x)[0]
    assert compiled.shape == eager.shape and compiled.dtype == eager.dtype
    assert torch.equal(compiled, eager)


def test_int8_model_captured_and_replayed(cuda_device):
    quantized = _model(cuda_device, depth=2).quantize_int8()
    x, _ = _tokens(cuda_device, batch=1, length=16)
    quantized(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = quantized(x)
    x.copy_(x.flip(1))
    expect, _ = quantized(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, expect)


def test_training_with_8_bit_checkpoints(cuda_device):
    """The forward is that of the bf16 path up to its roundings; each gradient is off by the 8-bit
    rounding of what was kept: 0.9% of a row's norm for the projections' inputs, 0.7% for gate_up
    (groups of 128: a is about 2.8 rms), on independent tokens, so below 2% in all, beside the
    bf16 roundings of two different kernel sequences (below 2% of a gradient, as for the other
    paths of the model): held to 5%."""
    x, y = _tokens(cuda_device)
    plain, kept = _model(cuda_device), _model(cuda_device, activation_checkpoint="int8")
    kept.load_state_dict(plain.state_dict())
    _, loss = plain(x, y)
    _, loss8 = kept(x, y)
    loss.backward()
    loss8.backward()
    loss, loss8 = float(loss.detach()), float(loss8.detach())
    assert abs(loss - loss8) <= 1e-3 * abs(loss)
    for (name, p), (_, p8) in zip(plain.named_parameters(), kept.named_parameters()):
        assert p8.grad is not None and _rel(p8.grad, p.grad) < 0.05, name
    # the same model in evaluation keeps nothing and runs the usual path
    with torch.no_grad():
        assert torch.equal(kept(x)[0], plain(x)[0])


def test_8_bit_checkpoints_halve_what_the_mlp_keeps(cuda_device):
    x = torch.randn(8, 512, 256, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    held = {}
    for mode in ("none", "int8"):
        mlp = _model(cuda_device, depth=4, activation_checkpoint=mode).blocks[0].mlp
        saved = {}

        def keep(t):
            saved[t.data_ptr()] = t.numel() * t.element_size()
            return t

        with torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t):
            out, norm = mlp(x, x)
        weights = {p.data_ptr() for p in mlp.parameters()}
        held[mode] = sum(n for ptr, n in saved.items() if ptr not in weights)
        (out.float().sum() + norm.float().square().sum()).backward()
    rows, C, H = 8 * 512, 256, 768
    assert held["none"] == rows * 2 * (C + 2 * H + H + C)  # x, gate_up, h, and out for the norm
    assert held["int8"] == rows * (C + 2 * H + H + 4 * (1 + 12 + 1) + 2 * C)


@pytest.mark.parametrize("keep", ["none", "int8"])
def test_bench_counts_the_calls_of_a_step(keep, cuda_device):
    """The bench's table of calls in a micro-step of twelve layers, by which it averages, is what runs."""
    import bench
    from hackable_lm_b200 import _lib

    model = _model(cuda_device, depth=12, activation_checkpoint=keep)
    x, y = _tokens(cuda_device)
    calls = bench.d12_kernels(keep)
    timers = {k: _lib.KernelTimer(k, 4 * n) for k, n in calls.items()}
    for t in timers.values():
        t.__enter__()
    try:
        model(x, y)[1].backward()
    finally:
        for t in timers.values():
            t.__exit__(None, None, None)
    torch.cuda.synchronize()
    one_launch = {"gate_up", "proj_norm", "rmsnorm_fwd", "quant_rows", "dequant_rows", "swiglu_ckpt8_fwd",
                  "swiglu_ckpt8_bwd", "weight_grad_q8"}
    for k, n in calls.items():
        if k in one_launch:
            assert timers[k].launches == n, k
        else:  # a call may be two launches; the unfused SwiGLU does not run here
            assert n <= timers[k].launches <= 2 * n or (k in ("swiglu_fwd", "swiglu_bwd") and timers[k].launches == 0), k


def test_train_step_with_8_bit_checkpoints(cuda_device):
    from hackable_lm_b200 import train

    s = train.build(cuda_device, depth=2, vocab=512, seq_len=256, micro_batch=2, global_tokens=1024,
                    activation_checkpoint="int8")
    assert s.config.activation_checkpoint == "int8"
    batches = train.synthetic_batches(2, 2, 256, 512, 0, cuda_device)
    loss = train.train_step(s, batches)
    assert bool(torch.isfinite(loss))


def test_compiled_model_with_8_bit_checkpoints(cuda_device):
    """torch.compile(fullgraph=True) traces the operators.  The compiler's fusions round elsewhere, which
    moves the gradients of the bf16 model too; the checkpoints, taken of such values, may differ by their
    own rounding on both sides, sqrt(2) 0.9% of a row's norm: 2% on top of what the bf16 model moves by."""
    from hackable_lm_b200 import kernels
    from parity import assert_loss_close

    x, y = _tokens(cuda_device)
    moved = {}
    for mode in ("none", "int8"):
        torch._dynamo.reset()
        eager = _model(cuda_device, depth=2, activation_checkpoint=mode)
        twin = _model(cuda_device, depth=2, activation_checkpoint=mode)
        twin.load_state_dict(eager.state_dict())
        _, le = eager(x, y)
        le.backward()
        _, lc = kernels.compile_training_model(twin, True)(x, y)
        lc.backward()
        assert_loss_close(lc.detach(), le.detach(), tol=1e-4, what="compiled loss")
        moved[mode] = {n: _rel(p.grad, q.grad) for (n, p), (_, q) in zip(twin.named_parameters(), eager.named_parameters())}
    for n, r in moved["int8"].items():
        assert r <= moved["none"][n] + 0.02, (n, r, moved["none"][n])
