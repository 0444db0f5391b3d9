"""What a training step of a norm, a layer of experts and their optimizer state
costs: the cases that the framework's operators for it are measured on.

Three operators, each with a plain form in 32-bit torch operations:

* products grouped by expert: ``out[r] = left[r] @ right[e]`` for the rows r of
  expert e (``ends[e - 1] <= r < ends[e]``; rows past the last end are zero), and
  the gradients of both factors;
* layer norm, forward and backward with the weight's and bias's gradients;
* AdamW over many tensors, states in 32 bits or in 8 (e4m3 values with one
  32-bit scale for each block of 256 elements).
"""

import math

import numpy as np
import torch

own = False

BLOCK = 256  # elements that share a scale of the 8-bit states
TOP = 448.0  # largest e4m3 value
TINY = 2.0**-9  # smallest e4m3 value above zero
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One token routed to 8 of 64 experts (the batch of 64 matrices of 1024 x 4096 that
        # the framework's benchmark orthogonalises): reading 8 weights is all there is.
        {"name": "experts: one token", "op": "experts", "rows": 8, "tail": 0, "experts": 64, "k": 1024, "n": 4096,
         "type": "bf16", "skew": -1.0},
        # A decoding batch of 96 sequences with 2 experts each: every expert has a few rows.
        {"name": "experts: decoding batch", "op": "experts", "rows": 192, "tail": 0, "experts": 64, "k": 4096,
         "n": 1024, "type": "bf16", "skew": 0.5},
        # Odd sizes in half precision, with empty experts and rows that nobody owns.
        {"name": "experts: odd sizes", "op": "experts", "rows": 777, "tail": 13, "experts": 5, "k": 1000, "n": 1501,
         "type": "f16", "skew": 2.0},
        # A training batch through few wide experts (4096 x 14336, the benchmark's MLP shape).
        {"name": "experts: wide", "op": "experts", "rows": 16384, "tail": 0, "experts": 8, "k": 4096, "n": 14336,
         "type": "bf16", "skew": 0.3},
        # Gradients of rows and weights for a small batch, ragged.
        {"name": "expert gradients: small", "op": "expert_gradients", "rows": 1003, "tail": 0, "experts": 16, "k": 512,
         "n": 1024, "type": "bf16", "skew": 1.0},
        # Gradients of a training batch over 64 experts.
        {"name": "expert gradients: training", "op": "expert_gradients", "rows": 32768, "tail": 0, "experts": 64,
         "k": 1024, "n": 4096, "type": "bf16", "skew": 0.5},
        # 16 bias vectors of 4096 (the optimizer benchmark's AdamW group): launches and host time.
        {"name": "adamw: vectors, 8 bits", "op": "adamw", "tensors": 16, "elements": 4096, "spread": 0.0, "bits": 8,
         "type": "f32", "gradient": "f32", "packed": False},
        # Embedding-sized tensors beside vectors, bf16 with 8-bit states.
        {"name": "adamw: embeddings, 8 bits", "op": "adamw", "tensors": 24, "elements": 67108864, "spread": 3.0,
         "bits": 8, "type": "bf16", "gradient": "bf16", "packed": False},
        # The same in 32-bit states for bf16 parameters, odd sizes.
        {"name": "adamw: mixed, 32 bits", "op": "adamw", "tensors": 40, "elements": 7777777, "spread": 3.0, "bits": 32,
         "type": "bf16", "gradient": "bf16", "packed": False},
        # One sequence step through a norm: a few rows, latency.
        {"name": "norm: few rows", "op": "norm", "rows": 7, "columns": 4096, "type": "bf16", "weight": "bf16",
         "backward": False},
        # A training batch: forward and backward, weights in 32 bits.
        {"name": "norm: training", "op": "norm", "rows": 16384, "columns": 4096, "type": "bf16", "weight": "f32",
         "backward": True},
        # Odd row length in 32 bits.
        {"name": "norm: odd columns", "op": "norm", "rows": 4099, "columns": 1111, "type": "f32", "weight": "f32",
         "backward": True},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _inner(rng, low, high):
    """A width: a usual one, an odd multiple of 8, or an odd number."""
    usual = [n for n in (64, 128, 256, 512, 768, 1024, 1536, 2048, 4096, 5120, 8192, 14336, 16384) if low <= n <= high]
    size = _log_uniform(rng, low, high - 16)
    return rng.choice([rng.choice(usual), rng.choice(usual), size // 16 * 16 + 8, size | 1])


def draw(rng):
    op = rng.choice(["experts", "experts", "expert_gradients", "adamw", "adamw", "norm", "norm"])
    if op in ("experts", "expert_gradients"):
        while True:
            case = {"op": op, "rows": _log_uniform(rng, 1, 32768), "tail": rng.choice([0, 0, rng.randrange(1, 40)]),
                    "experts": _log_uniform(rng, 2, 96), "k": _inner(rng, 64, 8192), "n": _inner(rng, 64, 8192),
                    "type": rng.choice(["bf16", "bf16", "f16"]), "skew": round(rng.uniform(0.0, 1.5), 2)}
            weights = case["experts"] * case["k"] * case["n"]
            if weights <= 64 * 1024 * 4096 and case["rows"] * case["k"] * case["n"] <= 32768 * 1024 * 4096:
                return case
    if op == "adamw":
        while True:
            kind = rng.choice(["bf16", "bf16", "f32", "f16"])
            case = {"op": op, "tensors": _log_uniform(rng, 1, 200), "elements": _log_uniform(rng, 100, 4000000),
                    "spread": round(rng.uniform(0.0, 3.0), 2), "bits": rng.choice([8, 8, 32]), "type": kind,
                    "gradient": rng.choice([kind, kind, "f32"]), "packed": rng.random() < 0.2}
            if case["tensors"] * case["elements"] <= 48 * 2097152:
                return case
    while True:
        case = {"op": op, "rows": _log_uniform(rng, 1, 32768), "columns": _inner(rng, 64, 16384),
                "type": rng.choice(["bf16", "f16", "f32"]), "weight": rng.choice(["same", "f32"]),
                "backward": rng.random() < 0.7}
        if case["weight"] == "same":
            case["weight"] = case["type"]
        if case["rows"] * case["columns"] <= 16384 * 4096:
            return case


# ------------------------------------------------------------------- inputs
def _counts(case, rng):
    """Rows of each expert: a random share for each, its logarithm spread by ``skew``
    (negative: one row for each of the first experts, as one token has)."""
    experts, rows = case["experts"], case["rows"]
    if case["skew"] < 0:
        counts = np.zeros(experts, dtype=np.int64)
        counts[rng.permutation(experts)[:rows]] = 1
        return counts
    share = np.exp(case["skew"] * rng.standard_normal(experts))
    return rng.multinomial(rows, share / share.sum())


def _sizes(case):
    """Elements of each tensor, the same for every seed: ``elements`` at most, smaller by
    factors of up to ``10 ** spread``, odd ones among them."""
    rng = np.random.RandomState(case["tensors"] * 7919 + case["elements"])
    sizes = [case["elements"] / 10 ** (case["spread"] * u) for u in rng.uniform(0.0, 1.0, case["tensors"])]
    sizes[0] = case["elements"]
    return [max(1, int(s)) for s in sizes]


def _round_up(value, unit):
    return (value + unit - 1) // unit * unit


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    dtype = TYPES[case["type"]]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(shape, generator=gen, device=device) * scale).to(to)

    if case["op"] in ("experts", "expert_gradients"):
        counts = _counts(case, rng)
        total = case["rows"] + case["tail"]
        state = {
            "case": case,
            "x": normal(total, case["k"]),
            "weight": normal(case["experts"], case["n"], case["k"], scale=0.02),
            "ends": torch.tensor(np.cumsum(counts), dtype=torch.int32, device=device),
            "largest": max(1, int(counts.max())),
        }
        if case["op"] == "expert_gradients":
            state["grad"] = normal(total, case["n"], scale=1e-2)
        return state
    if case["op"] == "norm":
        weight = TYPES[case["weight"]]
        rows, columns = case["rows"], case["columns"]
        # Activations of a residual stream: rows of differing size, columns with an offset.
        x = torch.randn((rows, columns), generator=gen, device=device)
        x = x * torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device=device))
        x = x + 0.5 * torch.randn((1, columns), generator=gen, device=device)
        return {
            "case": case,
            "x": x.to(dtype),
            "weight": (1.0 + 0.1 * torch.randn(columns, generator=gen, device=device)).to(weight),
            "bias": normal(columns, scale=0.1, to=weight),
            "grad": normal(rows, columns, scale=1e-2) if case["backward"] else None,
            "epsilon": 1e-5,
        }
    # AdamW: the tensors are slices of flat buffers, as a bucket of gradients is; each starts on a
    # multiple of 256 elements, zeros between, or right after its neighbour (packed).
    sizes = _sizes(case)
    pitch = sizes if case["packed"] else [_round_up(n, BLOCK) for n in sizes]
    starts = [0, *np.cumsum(pitch).tolist()]
    total = starts[-1]
    held = torch.zeros(total, dtype=torch.bool, device=device)
    for start, n in zip(starts, sizes):
        held[start:start + n] = True
    flat = {
        "parameter": normal(total, scale=0.02) * held,
        "gradient": normal(total, scale=1e-3, to=TYPES[case["gradient"]]) * held,
    }
    # Moments as they stand after some steps: of the gradients' size.
    first = normal(total, scale=3e-4, to=torch.float32) * held
    second = (normal(total, scale=1e-3, to=torch.float32).square() * 0.5 + 1e-9) * held
    state = {"case": case, "sizes": sizes, "starts": starts[:-1], "flat": flat, "step": 100}
    if case["bits"] == 32:
        flat["exp_avg"], flat["exp_avg_sq"] = first, second
    else:
        blocks = [_round_up(n, BLOCK) // BLOCK for n in sizes]
        state["block_starts"] = [0, *np.cumsum(blocks).tolist()][:-1]
        state["blocks"] = blocks
        count = sum(blocks)
        # Codes over their whole range, scales of the moments' size.
        flat["exp_avg"] = (first * (TOP / 1.2e-3)).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
        flat["exp_avg_sq"] = ((second * (TOP / 8e-6)).clamp(TINY, TOP) * held).to(torch.float8_e4m3fn)
        spread = 0.5 + torch.rand((2, count), generator=gen, device=device)
        flat["exp_avg_scale"] = spread[0] * (1.2e-3 / TOP)
        flat["exp_avg_sq_scale"] = spread[1] * (8e-6 / TOP)
    # The optimizer's per-tensor views of these buffers.
    for role in ("parameter", "gradient", "exp_avg", "exp_avg_sq"):
        state[role] = [flat[role][a:a + n] for a, n in zip(state["starts"], sizes)]
    if case["bits"] == 8:
        for role in ("exp_avg_scale", "exp_avg_sq_scale"):
            state[role] = [flat[role][a:a + n] for a, n in zip(state["block_starts"], state["blocks"])]
    return state


HYPER = {"learning_rate": 1e-3, "beta1": 0.9, "beta2": 0.95, "epsilon": 1e-8, "weight_decay": 0.1}


# ---------------------------------------------------------------- the passes
def run(state):
    op = state["case"]["op"]
    if op == "experts":
        return _experts(state)
    if op == "expert_gradients":
        return _expert_gradients(state)
    if op == "norm":
        return _norm(state)
    return _adamw(state)


def _row_table(state):
    """[experts, largest] row numbers of each expert, and which of them exist."""
    ends = state["ends"].long()
    starts = torch.cat([ends.new_zeros(1), ends[:-1]])
    rows = starts[:, None] + torch.arange(state["largest"], device=ends.device)
    return rows, rows < ends[:, None]


def _by_expert(x, rows, valid):
    """x's rows in 32 bits, [experts, largest, columns], zeros where there is no row."""
    picked = x[torch.where(valid, rows, 0)].float()
    return torch.where(valid[..., None], picked, 0.0)


def _back(y, rows, valid, total, dtype):
    """The rows of [experts, largest, columns] at their places, the others zero."""
    out = torch.zeros((total + 1, y.shape[-1]), dtype=dtype, device=y.device)
    out[torch.where(valid, rows, total)] = y.to(dtype)
    return out[:total]


def _experts(state):
    x, weight = state["x"], state["weight"]
    if own:
        from gram_newton_schulz_ampere_b200 import ops

        return ops.grouped_gemm(x, weight.transpose(1, 2), state["ends"])
    rows, valid = _row_table(state)
    y = torch.bmm(_by_expert(x, rows, valid), weight.float().transpose(1, 2))
    return _back(y, rows, valid, x.shape[0], x.dtype)


def _expert_gradients(state):
    x, weight, grad = state["x"], state["weight"], state["grad"]
    if own:
        from gram_newton_schulz_ampere_b200 import ops

        return {"x": ops.grouped_gemm(grad, weight, state["ends"]),
                "weight": ops.grouped_gemm_reduce(grad, x, state["ends"])}
    rows, valid = _row_table(state)
    grads = _by_expert(grad, rows, valid)
    dx = torch.bmm(grads, weight.float())
    dweight = torch.bmm(grads.transpose(1, 2), _by_expert(x, rows, valid))
    return {"x": _back(dx, rows, valid, x.shape[0], x.dtype), "weight": dweight.to(weight.dtype)}


def _norm(state):
    x, weight, bias, grad, eps = (state[k] for k in ("x", "weight", "bias", "grad", "epsilon"))
    if own:
        from gram_newton_schulz_ampere_b200 import ops

        y, mean, rstd = ops.layer_norm(x, weight, bias, eps)
        if grad is None:
            return y
        dx, dweight, dbias = ops.layer_norm_backward(grad, x, weight, mean, rstd)
        return {"y": y, "x": dx, "weight": dweight, "bias": dbias}
    x32, w32 = x.float(), weight.float()
    centred = x32 - x32.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + eps)
    unit = centred * rstd
    y = (unit * w32 + bias.float()).to(x.dtype)
    if grad is None:
        return y
    g32 = grad.float()
    a = g32 * w32
    dx = rstd * (a - a.mean(1, keepdim=True) - unit * (a * unit).mean(1, keepdim=True))
    return {"y": y, "x": dx.to(x.dtype), "weight": (g32 * unit).sum(0).to(weight.dtype),
            "bias": g32.sum(0).to(bias.dtype)}


def _adamw(state):
    """One step in place; the flat parameter and state buffers are the outputs."""
    state["step"] += 1
    flat, bits = state["flat"], state["case"]["bits"]
    if own:
        from gram_newton_schulz_ampere_b200 import ops

        if "handle" not in state:  # what an optimizer keeps from step to step
            state["handle"] = ops.AdamWStates(
                state["parameter"], bits, state["exp_avg"], state["exp_avg_sq"],
                state.get("exp_avg_scale"), state.get("exp_avg_sq_scale"))
        state["handle"].step(state["gradient"], step=state["step"], **HYPER)
    else:
        _plain_adamw(state)
    return {k: v for k, v in flat.items() if k != "gradient"}


def _plain_adamw(state):
    lr, b1, b2 = HYPER["learning_rate"], HYPER["beta1"], HYPER["beta2"]
    flat, t = state["flat"], state["step"]
    p, g = flat["parameter"].float(), flat["gradient"].float()
    if state["case"]["bits"] == 8:
        m, v = _decode(state, "exp_avg"), _decode(state, "exp_avg_sq")
    else:
        m, v = flat["exp_avg"], flat["exp_avg_sq"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    denominator = torch.sqrt(v) * (1 / math.sqrt(1 - b2**t)) + HYPER["epsilon"]
    p = p * (1 - lr * HYPER["weight_decay"]) - m / denominator * (lr / (1 - b1**t))
    flat["parameter"].copy_(p)
    if state["case"]["bits"] == 8:
        _encode(state, "exp_avg", m)
        _encode(state, "exp_avg_sq", v)
    else:
        flat["exp_avg"].copy_(m)
        flat["exp_avg_sq"].copy_(v)


def _blocks(state, flat):
    """[blocks, 256]: each tensor's elements from a block's start on, zeros behind its end."""
    if not state["case"]["packed"]:
        return flat.view(-1, BLOCK)
    return torch.cat([torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)) for t in flat.split(state["sizes"])]).view(-1, BLOCK)


def _flat(state, blocks):
    """The inverse of _blocks."""
    if not state["case"]["packed"]:
        return blocks.view(-1)
    parts = blocks.view(-1).split([n * BLOCK for n in state["blocks"]])
    return torch.cat([part[:n] for part, n in zip(parts, state["sizes"])])


def _decode(state, role):
    values = _blocks(state, state["flat"][role].float()) * state["flat"][role + "_scale"][:, None]
    return _flat(state, values)


def _encode(state, role, values):
    values = _blocks(state, values)
    top = values.abs().amax(1)
    state["flat"][role + "_scale"].copy_(top * (1 / TOP))
    scaled = values * torch.where(top > 1e-30, torch.reciprocal(top) * TOP, 0.0)[:, None]
    if role == "exp_avg_sq":  # a second moment above zero stays above zero
        scaled = torch.where(values > 0, scaled.clamp_min(TINY), scaled)
    state["flat"][role].copy_(_flat(state, scaled.clamp(-TOP, TOP)).to(torch.float8_e4m3fn))


# ----------------------------------------------------------------- the floor
def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    es = _size(case["type"])
    if case["op"] in ("experts", "expert_gradients"):
        rows, total, k, n = case["rows"], case["rows"] + case["tail"], case["k"], case["n"]
        touched = min(case["experts"], rows)  # at most: an expert without rows is not read
        weights = case["experts"] * k * n if case["op"] == "expert_gradients" else 0
        if case["op"] == "experts":
            return {"bytes": es * (rows * k + touched * k * n + total * n), "flops": 2 * rows * k * n}
        return {"bytes": es * (rows * (k + n) + touched * k * n + total * k + weights), "flops": 4 * rows * k * n}
    if case["op"] == "norm":
        cells = case["rows"] * case["columns"]
        ws = _size(case["weight"])
        if not case["backward"]:
            return {"bytes": 2 * es * cells + 2 * ws * case["columns"], "flops": 8 * cells}
        return {"bytes": 4 * es * cells + 4 * ws * case["columns"], "flops": 20 * cells}
    elements = sum(_sizes(case))
    held = 2 if case["bits"] == 8 else 8
    scales = 16 * sum(_round_up(n, BLOCK) // BLOCK for n in _sizes(case)) if case["bits"] == 8 else 0
    each = 2 * es + _size(case["gradient"]) + 2 * held
    return {"bytes": each * elements + scales, "flops": 16 * elements}


# ------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op in ("experts", "expert_gradients"):
        x, weight = state["x"].double(), state["weight"]
        ends = [0, *state["ends"].tolist()]
        if op == "experts":
            y = x.new_zeros((x.shape[0], case["n"]))
            for e, (a, b) in enumerate(zip(ends, ends[1:])):
                y[a:b] = x[a:b] @ weight[e].double().T
            return y
        grad = state["grad"].double()
        dx = torch.zeros_like(x)
        dweight = torch.empty(weight.shape, dtype=torch.float64, device=x.device)
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            dx[a:b] = grad[a:b] @ weight[e].double()
            dweight[e] = grad[a:b].T @ x[a:b]
        return {"x": dx, "weight": dweight}
    if op == "norm":
        x, w = state["x"].double(), state["weight"].double()
        mu = x.sum(1) / case["columns"]
        var = ((x - mu[:, None]) ** 2).sum(1) / case["columns"]
        xh = (x - mu[:, None]) / torch.sqrt(var + state["epsilon"])[:, None]
        y = xh * w + state["bias"].double()
        if not case["backward"]:
            return y
        dy = state["grad"].double()
        n = case["columns"]
        inner = dy * w
        dx = (n * inner - inner.sum(1, keepdim=True) - xh * (inner * xh).sum(1, keepdim=True))
        dx = dx / (n * torch.sqrt(var + state["epsilon"])[:, None])
        return {"y": y, "x": dx, "weight": (dy * xh).sum(0), "bias": dy.sum(0)}
    return _exact_adamw(state, case)


def _nearest(values):
    """Each value's nearest e4m3 value, in 64 bits."""
    table = torch.arange(127, dtype=torch.uint8, device=values.device).view(torch.float8_e4m3fn).double()
    middle = (table[1:] + table[:-1]) / 2
    return torch.sign(values) * table[torch.bucketize(values.abs(), middle)]


def _exact_adamw(state, case):
    lr, b1, b2 = HYPER["learning_rate"], HYPER["beta1"], HYPER["beta2"]
    t = state["step"] + 1
    out = {k: v.double() for k, v in state["flat"].items() if k != "gradient"}
    for i, (a, n) in enumerate(zip(state["starts"], state["sizes"])):
        p, g = (state["flat"][k][a:a + n].double() for k in ("parameter", "gradient"))
        m, v = (state["flat"][k][a:a + n].double() for k in ("exp_avg", "exp_avg_sq"))
        scales = {}
        if case["bits"] == 8:
            c, count = state["block_starts"][i], state["blocks"][i]
            here = torch.arange(n, device=p.device) // BLOCK
            m = m * state["flat"]["exp_avg_scale"][c:c + count].double()[here]
            v = v * state["flat"]["exp_avg_sq_scale"][c:c + count].double()[here]
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g**2
        out["parameter"][a:a + n] = p - lr * HYPER["weight_decay"] * p - lr * (m / (1 - b1**t)) / (
            torch.sqrt(v / (1 - b2**t)) + HYPER["epsilon"])
        if case["bits"] == 8:
            for name, values in (("exp_avg", m), ("exp_avg_sq", v)):
                filled = torch.nn.functional.pad(values, (0, count * BLOCK - n)).view(count, BLOCK)
                scales[name] = filled.abs().amax(1) / TOP
                codes = filled / scales[name].clamp_min(1e-300)[:, None]
                if name == "exp_avg_sq":
                    codes = torch.where(filled > 0, codes.clamp_min(TINY), codes)
                out[name][a:a + n] = _nearest(codes).reshape(-1)[:n]
                out[name + "_scale"][c:c + count] = scales[name]
        else:
            out["exp_avg"][a:a + n] = m
            out["exp_avg_sq"][a:a + n] = v
    return out
