"""Cases of the 8-bit operators: row quantisation, RMSNorm with an 8-bit output,
the 8-bit integer projection, and the 8-bit activation checkpoints of the MLP.

Every pass runs either in its plain form (elementary torch operations in 32 bits,
rounded once) or through the framework's entry points (``own``).

The 8-bit format, for a group of values v (a whole row, or 128 columns):

    a = max(max|v|, 2^-110),  q = rint(v * (127 / a)),  scale = a / 127,  v ~ q * scale

with the two divisions and the product in 32-bit IEEE arithmetic: the codes are
defined by them, so a code next to a rounding border is the same everywhere.
"""
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
FLOOR = 2.0 ** -110
GROUP = 128


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # quantising a projection's input and reading it back: one short prompt, one
        # training micro-batch (16 sequences of 2048 tokens, the depth-12 MLP width)
        {"name": "rows short", "op": "rows", "rows": 67, "cols": 768, "type": "bf16"},
        {"name": "rows batch", "op": "rows", "rows": 32768, "cols": 2048, "type": "bf16"},
        # the norm before a projection: a few tokens of odd width with a weight, and the
        # whole micro-batch of the depth-12 model (weightless, as its norms are)
        {"name": "norm few", "op": "norm", "rows": 5, "cols": 1000, "type": "fp16", "weight": True},
        {"name": "norm batch", "op": "norm", "rows": 32768, "cols": 768, "type": "bf16", "weight": False},
        # 8-bit projections: one token through gate_up, a handful through the down
        # projection, ragged sizes with a 32-bit result, the micro-batch through gate_up
        {"name": "linear token", "op": "linear", "rows": 1, "n": 4096, "k": 768, "type": "bf16"},
        {"name": "linear few", "op": "linear", "rows": 24, "n": 768, "k": 2048, "type": "fp16"},
        {"name": "linear ragged", "op": "linear", "rows": 777, "n": 1111, "k": 1360, "type": "fp32"},
        {"name": "linear batch", "op": "linear", "rows": 32768, "n": 4096, "k": 768, "type": "bf16"},
        # SwiGLU that keeps its input in 8 bits, forward and backward: a ragged short
        # batch in 32 bits, the depth-12 micro-batch
        {"name": "swiglu short", "op": "swiglu", "rows": 333, "hidden": 1000, "type": "fp32"},
        {"name": "swiglu batch", "op": "swiglu", "rows": 32768, "hidden": 2048, "type": "bf16"},
        # weight gradient of a projection from its input kept in 8 bits: a small layer on a
        # ragged batch, the depth-12 gate_up projection on the micro-batch
        {"name": "wgrad small", "op": "wgrad", "rows": 1003, "n": 520, "k": 272, "type": "fp16"},
        {"name": "wgrad batch", "op": "wgrad", "rows": 32768, "n": 4096, "k": 768, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _steps(rng, lo, hi, step):
    return step * _log(rng, lo // step, hi // step)


def draw(rng):
    op = rng.choice(["rows", "norm", "linear", "swiglu", "wgrad"])
    if op in ("rows", "norm"):
        cols = _log(rng, 16, 8192)
        if rng.random() < 0.5:
            cols = max(16, cols // 16 * 16)
        rows = _log(rng, 1, min(32768, (32768 * (2048 if op == "rows" else 768)) // cols))
        case = {"op": op, "rows": rows, "cols": cols, "type": rng.choice(["bf16", "fp16", "fp32"])}
        if case["type"] == "fp32":
            case["rows"] = max(1, rows // 2)
        if op == "norm":
            case["weight"] = rng.random() < 0.5
        return case
    if op == "linear":
        n, k = _log(rng, 16, 8192), _steps(rng, 64, 8192, 16)
        most = 32768 * 4096 * 768
        rows = _log(rng, 1, max(1, min(32768, most // (n * k), 32768 * 4096 // (2 * n))))
        return {"op": op, "rows": rows, "n": n, "k": k, "type": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "swiglu":
        hidden = _log(rng, 16, 8192)
        if rng.random() < 0.5:
            hidden = max(16, hidden // 16 * 16)
        rows = _log(rng, 1, min(32768, 32768 * 1024 // hidden))
        return {"op": op, "rows": rows, "hidden": hidden, "type": rng.choice(["bf16", "fp16", "fp32"])}
    n, k = _steps(rng, 64, 8192, 8), _steps(rng, 64, 8192, 16)
    rows = _log(rng, 1, max(1, min(32768, 32768 * 4096 * 768 // (n * k))))
    return {"op": op, "rows": rows, "n": n, "k": k, "type": rng.choice(["bf16", "fp16"])}


def _normal(shape, seed, stream):
    g = torch.Generator(device="cuda").manual_seed(seed * 16 + stream)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(rows, cols, seed, stream):
    """Activations: normal values whose columns differ in size (factors e^(0.5 z))."""
    return _normal((rows, cols), seed, stream).mul_(torch.exp(0.5 * _normal((cols,), seed, stream + 1)))


def _codes(x):
    a = x.abs().amax(dim=-1, keepdim=True).clamp(min=FLOOR)
    most = torch.full_like(a, 127.0)
    return torch.round(x * (most / a)).to(torch.int8), (a / most).squeeze(-1)


def prepare(case, seed):
    op, dtype = case["op"], TYPES[case["type"]]
    state = {"op": op, "dtype": dtype}
    if op == "rows":
        state["x"] = _activations(case["rows"], case["cols"], seed, 0).to(dtype)
    elif op == "norm":
        # the residual stream is several times the size of one layer's branch
        state["residual"] = _activations(case["rows"], case["cols"], seed, 0).mul_(4.0).to(dtype)
        state["branch"] = _normal((case["rows"], case["cols"]), seed, 2).to(dtype)
        state["weight"] = (1.0 + 0.1 * _normal((case["cols"],), seed, 3)).to(dtype) if case["weight"] else None
    elif op == "linear":
        # the projection's input as the norm leaves it; the weights, quantised once
        state["q"], state["scale"] = _codes(_activations(case["rows"], case["k"], seed, 0))
        state["w"], state["w_scale"] = _codes(_normal((case["n"], case["k"]), seed, 2).mul_(0.02))
    elif op == "swiglu":
        state["gate_up"] = _activations(case["rows"], 2 * case["hidden"], seed, 0).to(dtype)
        state["grad"] = _normal((case["rows"], case["hidden"]), seed, 2).mul_(0.1).to(dtype)
    else:
        state["x"] = _activations(case["rows"], case["k"], seed, 0).to(dtype)
        state["grad"] = _normal((case["rows"], case["n"]), seed, 2).mul_(0.1).to(dtype)
    return state


def run(state):
    return _run_own(state) if own else PLAIN[state["op"]](state)


def _run_own(state):
    from hackable_lm_b200 import kernels, ops

    op = state["op"]
    if op == "rows":
        q, scale = kernels.quantize_rows(state["x"])
        return kernels.dequantize_rows(q, scale, state["dtype"])
    if op == "norm":
        out, q, scale = kernels.residual_rms_norm_q8(state["residual"], state["branch"], EPS, state["weight"])
        return out, kernels.dequantize_rows(q, scale, state["dtype"])
    if op == "linear":
        return kernels.linear_q8(state["q"], state["scale"], state["w"], state["w_scale"], state["dtype"])
    if op == "swiglu":
        h, q, scale = ops.swiglu_ckpt8(state["gate_up"])
        return h, ops.swiglu_ckpt8_backward(q, scale, state["grad"])
    q, scale = kernels.quantize_rows(state["x"])
    return ops.weight_grad_q8(state["grad"], q, scale)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _round(x):
    """x as 8-bit codes (held in 32 bits) and the scale of each row (last dimension)."""
    a = torch.clamp(torch.amax(torch.abs(x), dim=-1, keepdim=True), min=FLOOR)
    most = torch.full_like(a, 127.0)  # a tensor: with a number, torch multiplies by a rounded reciprocal
    return torch.round(x * (most / a)), a / most


def _plain_rows(state):
    q, scale = _round(state["x"].float())
    return (q * scale).to(state["dtype"])


def _plain_norm(state):
    out = (state["residual"].float() + state["branch"].float()).to(state["dtype"])
    x = out.float()
    rstd = 1.0 / torch.sqrt(torch.sum(x * x, dim=-1, keepdim=True) / x.shape[-1] + EPS)
    # 1/rms is common to the row: it scales the row's step and leaves its codes alone
    q, scale = _round(x if state["weight"] is None else x * state["weight"].float())
    return out, (q * (scale * rstd)).to(state["dtype"])


def _plain_linear(state):
    acc = state["q"].float() @ state["w"].float().t()
    return (acc * state["scale"][:, None] * state["w_scale"][None, :]).to(state["dtype"])


def _grouped(x):
    """x read back from 8 bits with one scale for each row and 128 columns."""
    rows, cols = x.shape
    pad = -cols % GROUP
    groups = torch.cat((x, x.new_zeros((rows, pad))), dim=1).reshape(rows, -1, GROUP)
    q, scale = _round(groups)
    return (q * scale).reshape(rows, cols + pad)[:, :cols]


def _plain_swiglu(state):
    hidden = state["grad"].shape[-1]
    x, grad = state["gate_up"].float(), state["grad"].float()
    gate, up = x[:, :hidden], x[:, hidden:]
    h = gate / (1.0 + torch.exp(-gate)) * up
    gate, up = _grouped(gate), _grouped(up)
    s = 1.0 / (1.0 + torch.exp(-gate))
    grad_gate = grad * up * s * (1.0 + gate * (1.0 - s))
    grad_up = grad * gate * s
    return h.to(state["dtype"]), torch.cat((grad_gate, grad_up), dim=1).to(state["dtype"])


def _plain_wgrad(state):
    q, scale = _round(state["x"].float())
    return (state["grad"].float().t() @ (q * scale)).to(state["dtype"])


PLAIN = {"rows": _plain_rows, "norm": _plain_norm, "linear": _plain_linear, "swiglu": _plain_swiglu,
         "wgrad": _plain_wgrad}


# ---------------------------------------------------------------------------
# work and the exact values
# ---------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["type"]]
    op, rows = case["op"], case["rows"]
    if op == "rows":  # x in; codes and scales out and in; values out
        n = rows * case["cols"]
        return {"bytes": n * (2 * size + 2) + 8 * rows, "flops": 4 * n}
    if op == "norm":  # residual, branch in; sum, codes, scales out; codes, scales in; values out
        n = rows * case["cols"]
        return {"bytes": n * (4 * size + 2) + 8 * rows, "flops": 8 * n}
    if op == "linear":
        n, k = case["n"], case["k"]
        return {"bytes": rows * k + n * k + rows * n * size + 4 * (rows + n), "flops": 2 * rows * n * k}
    if op == "swiglu":  # gate_up in, h out, codes out and in, grad in, grad_gate_up out
        n = rows * case["hidden"]
        return {"bytes": n * (6 * size + 4) + 16 * rows * -(-case["hidden"] // GROUP), "flops": 30 * n}
    n, k = case["n"], case["k"]  # x in, codes out and in, grad in, grad_w out
    return {"bytes": rows * k * (size + 2) + rows * n * size + n * k * size + 8 * rows, "flops": 2 * rows * n * k}


def _step_of(largest):
    """The step (scale) of groups whose largest magnitudes are given, as the format defines it."""
    return torch.maximum(largest, torch.full_like(largest, FLOOR)).div(torch.full_like(largest, 127.0))


def _read_back(values, factor=None):
    """Exact values that 8-bit codes of the last dimension stand for, times `factor`."""
    v32 = values.to(torch.float32)
    largest = v32.abs().max(dim=-1).values.unsqueeze(-1)
    per_step = torch.full_like(largest, 127.0).div(torch.maximum(largest, torch.full_like(largest, FLOOR)))
    back = v32.mul(per_step).round().to(torch.float64).mul(_step_of(largest).to(torch.float64))
    return back if factor is None else back.mul(factor)


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if s["op"] == "rows":
        return _read_back(s["x"])
    if s["op"] == "norm":
        # the sum is rounded to the type once, and the norm is that of the rounded sum
        total = s["residual"].to(f64).add(s["branch"].to(f64))
        kept = s["residual"].float().add(s["branch"].float()).to(s["dtype"])
        rms = kept.to(f64).square().mean(dim=-1, keepdim=True).add(EPS).sqrt()
        v = kept.float() if s["weight"] is None else kept.float().mul(s["weight"].float())
        return total, _read_back(v, rms.reciprocal())
    if s["op"] == "linear":
        left = s["q"].to(f64).mul(s["scale"].to(f64).unsqueeze(1))
        return left.matmul(s["w"].to(f64).mul(s["w_scale"].to(f64).unsqueeze(1)).T)
    if s["op"] == "swiglu":
        gate, up = s["gate_up"].to(f64).chunk(2, dim=-1)
        h = gate.mul(torch.sigmoid(gate)).mul(up)
        back = [torch.cat([_read_back(p) for p in half.float().split(GROUP, dim=-1)], dim=-1) for half in (gate, up)]
        d, sig = s["grad"].to(f64), torch.sigmoid(back[0])
        slope = sig.add(back[0].mul(sig).mul(1 - sig))
        return h, torch.cat((d.mul(back[1]).mul(slope), d.mul(back[0]).mul(sig)), dim=-1)
    return s["grad"].to(f64).T.matmul(_read_back(s["x"]))
