"""What the output end of a language model costs in training and serving: the cases that the
framework's operators for it are measured on.

Four operators, each with a plain form in 32-bit torch operations:

* products of 8-bit matrices: ``left [m, k] @ right [k, n]``, both e4m3 with 32-bit scales, one
  for each 128 of k of every row of ``left``, one for each 128 x 128 block of ``right``;
* a linear layer that multiplies so: its activations, weights and output gradients are brought
  into 8 bits within the call; forward and both gradients (the weight's from 16-bit factors);
* root-mean-square norm of a residual stream: the sum of the stream and a layer's output, its
  norm in the stream's type or in 8 bits with a scale for each 128 columns, and the gradients;
* distillation from a teacher's top logits: ``T^2 sum_j p_j (log p_j - log q_j)`` with p the
  softmax of the teacher's top logits over T and q the student's over the whole vocabulary,
  and the gradient of the student's logits.
"""

import math

import torch

own = False

BLOCK = 128  # elements along the contraction that share a scale
TOP = 448.0  # largest e4m3 value
LEAST = TOP * 2.0**-126  # a block's largest magnitude counts as this at least, so that its scale is a normal number
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One token through a wide layer (4096 x 14336, the benchmark's MLP shape): reading the weights is all there is.
        {"name": "product: one token", "op": "product", "m": 1, "k": 4096, "n": 14336, "turned": False, "type": "bf16"},
        # A decoding batch through the layer back (14336 x 4096).
        {"name": "product: decoding batch", "op": "product", "m": 96, "k": 14336, "n": 4096, "turned": False,
         "type": "bf16"},
        # Odd sizes in half precision, the gradient's orientation of the weights.
        {"name": "product: odd sizes", "op": "product", "m": 777, "k": 1000, "n": 1501, "turned": True, "type": "f16"},
        # A prompt, or a training batch, through the wide layer.
        {"name": "product: prompt", "op": "product", "m": 16384, "k": 4096, "n": 14336, "turned": False, "type": "bf16"},
        # A small training batch through a linear layer: forward, both gradients.
        {"name": "linear: small batch", "op": "linear", "m": 1003, "k": 1024, "n": 4096, "type": "bf16"},
        # A training batch through a square layer (4096 x 4096, the benchmark's attention matrices).
        {"name": "linear: training", "op": "linear", "m": 16384, "k": 4096, "n": 4096, "type": "bf16"},
        # One token's norm ahead of an 8-bit product: latency.
        {"name": "norm: one token, 8 bits", "op": "norm", "rows": 1, "columns": 4096, "type": "bf16", "weight": "bf16",
         "residual": True, "bits": 8, "backward": False},
        # A training batch: the stream's sum, the 8-bit norm, and the gradients.
        {"name": "norm: training, 8 bits", "op": "norm", "rows": 16384, "columns": 4096, "type": "bf16",
         "weight": "f32", "residual": True, "bits": 8, "backward": True},
        # Odd row length in 32 bits, the first norm of a model (no layer's output to add yet).
        {"name": "norm: odd columns", "op": "norm", "rows": 4099, "columns": 1111, "type": "f32", "weight": "f32",
         "residual": False, "bits": 32, "backward": True},
        # A few tokens' loss, as an evaluation of a short answer has them: latency.
        {"name": "loss: few rows", "op": "loss", "rows": 5, "vocabulary": 32000, "top": 32, "type": "bf16",
         "indices": "i64", "temperature": 1.0, "pass": "loss"},
        # An odd vocabulary in 32 bits: the loss, and the gradient in a call of its own, as autograd makes it.
        {"name": "loss: odd vocabulary", "op": "loss", "rows": 1021, "vocabulary": 50001, "top": 20, "type": "f32",
         "indices": "i32", "temperature": 2.0, "pass": "two"},
        # A training batch over a large vocabulary: loss and gradient in one call.
        {"name": "loss: training", "op": "loss", "rows": 4096, "vocabulary": 131072, "top": 64, "type": "bf16",
         "indices": "i64", "temperature": 2.0, "pass": "one"},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _inner(rng, low, high):
    """A width: a usual one, an odd multiple of 8, or an odd number."""
    usual = [n for n in (128, 256, 512, 768, 1024, 1536, 2048, 4096, 5120, 8192, 14336) if low <= n <= high]
    size = _log_uniform(rng, low, high - 16)
    return rng.choice([rng.choice(usual), rng.choice(usual), size // 16 * 16 + 8, size | 1])


def draw(rng):
    op = rng.choice(["product", "product", "linear", "norm", "norm", "loss", "loss"])
    if op in ("product", "linear"):
        while True:
            case = {"op": op, "m": _log_uniform(rng, 1, 16384), "k": _inner(rng, 128, 14336), "n": _inner(rng, 128, 14336)}
            if op == "product":
                case["turned"] = rng.random() < 0.4
            case["type"] = rng.choice(["bf16", "bf16", "f16"])
            if case["m"] * case["k"] * case["n"] <= 16384 * 4096 * (14336 if op == "product" else 4096):
                return case
    if op == "norm":
        while True:
            case = {"op": op, "rows": _log_uniform(rng, 1, 32768), "columns": _inner(rng, 128, 14336),
                    "type": rng.choice(["bf16", "bf16", "f16", "f32"]), "weight": rng.choice(["same", "f32"]),
                    "residual": rng.random() < 0.7, "bits": rng.choice([8, 0]), "backward": rng.random() < 0.6}
            case["weight"] = case["type"] if case["weight"] == "same" else case["weight"]
            case["bits"] = case["bits"] or 8 * _size(case["type"])
            if case["rows"] * case["columns"] <= 16384 * 4096:
                return case
    while True:
        case = {"op": op, "rows": _log_uniform(rng, 1, 8192), "vocabulary": _log_uniform(rng, 1000, 160000),
                "top": _log_uniform(rng, 1, 128), "type": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "indices": rng.choice(["i32", "i64"]), "temperature": rng.choice([1.0, 1.0, 2.0, 0.7, 4.0]),
                "pass": rng.choice(["loss", "two", "one", "one"])}
        if rng.random() < 0.5:
            case["vocabulary"] = max(1024, case["vocabulary"] // 128 * 128)
        if case["rows"] * case["vocabulary"] * _size(case["type"]) <= 4096 * 131072 * 2:
            return case


# ------------------------------------------------------------------- inputs
def _round_up(value, unit):
    return (value + unit - 1) // unit * unit


def _quantized(x, block_rows):
    """Codes and scales of a matrix held in 32 bits, as the framework lays them out: rows of codes
    start on multiples of 16 bytes, scales of one block column follow one another."""
    rows, cols = x.shape
    tall = _round_up(rows, block_rows)
    padded = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, tall - rows))
    blocks = padded.view(tall // block_rows, block_rows, -1, BLOCK)
    top = blocks.abs().amax((1, 3)).clamp_min(LEAST)
    whole = torch.full_like(top, TOP)  # a tensor: a plain number over one is divided with two roundings
    scaled = (blocks * (whole / top)[:, None, :, None]).clamp(-TOP, TOP).view(tall, -1)
    codes = torch.zeros((rows, _round_up(cols, 16)), dtype=torch.float8_e4m3fn, device=x.device)[:, :cols]
    codes.copy_(scaled[:rows, :cols].to(torch.float8_e4m3fn))
    return codes, (top / whole).t().contiguous().t()


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(shape, generator=gen, device=device) * scale).to(to)

    def activations(rows, columns):
        """Activations of a residual stream: rows of differing size, columns with an offset."""
        x = torch.randn((rows, columns), generator=gen, device=device)
        x = x * torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device=device))
        return x + 0.5 * torch.randn((1, columns), generator=gen, device=device)

    state = {"case": case}
    if case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        left = activations(m, k) if not case["turned"] else normal(m, k, scale=1e-3, to=torch.float32)
        state["left"], state["left_scales"] = _quantized(left, 1)
        # The layer's weights [out, in]: the forward product takes their transpose, the gradient of
        # the input the weights as they are.
        shape = (k, n) if case["turned"] else (n, k)
        codes, scales = _quantized(normal(*shape, scale=0.02, to=torch.float32), BLOCK)
        state["right"], state["right_scales"] = (codes, scales) if case["turned"] else (codes.t(), scales.t())
    elif case["op"] == "linear":
        state["x"] = activations(case["m"], case["k"]).to(dtype).requires_grad_()
        state["weight"] = normal(case["n"], case["k"], scale=0.02).requires_grad_()
        state["grad"] = normal(case["m"], case["n"], scale=1e-2)
    elif case["op"] == "norm":
        rows, columns, weight = case["rows"], case["columns"], TYPES[case["weight"]]
        state["x"] = activations(rows, columns).to(dtype)
        state["residual"] = normal(rows, columns) if case["residual"] else None
        state["weight"] = (1.0 + 0.1 * torch.randn(columns, generator=gen, device=device)).to(weight)
        state["grad"] = normal(rows, columns, scale=1e-2) if case["backward"] else None
        # The stream's own gradient, from the layers behind.
        state["grad_total"] = normal(rows, columns, scale=1e-2) if case["backward"] and case["residual"] else None
        state["epsilon"] = 1e-5
    else:
        rows, v, top = case["rows"], case["vocabulary"], case["top"]
        logits = torch.randn((rows, v), generator=gen, device=device) * 2.0
        start = torch.randint(0, v, (rows, 1), generator=gen, device=device)
        apart = torch.randint(1, max(2, v // top), (rows, 1), generator=gen, device=device)
        indices = (start + apart * torch.arange(top, device=device)) % v
        teacher = (8.0 + 2.0 * torch.randn((rows, top), generator=gen, device=device)).sort(1, descending=True).values
        # The student has learnt part of it.
        logits.scatter_add_(1, indices, 0.5 * teacher + normal(rows, top, to=torch.float32))
        # Some rows have fewer entries, and some none (tokens of the prompt).
        kept = torch.randint(0, top + 1, (rows, 1), generator=gen, device=device)
        kept = torch.where(torch.rand((rows, 1), generator=gen, device=device) < 0.7, top, kept)
        kept = torch.where(torch.rand((rows, 1), generator=gen, device=device) < 0.1, 0, kept)
        indices = torch.where(torch.arange(top, device=device) < kept, indices, -1)
        state["logits"] = logits.to(dtype)
        state["indices"] = indices.to(torch.int32 if case["indices"] == "i32" else torch.int64)
        state["teacher"] = teacher
        answered = (kept[:, 0] > 0).float()
        # The mean over the rows that count; half precision trains with a scaled loss.
        state["grad"] = answered / answered.sum().clamp_min(1.0) * (4096.0 if case["type"] == "f16" else 1.0)
    return state


# ---------------------------------------------------------------- the passes
def run(state):
    return {"product": _product, "linear": _linear, "norm": _norm, "loss": _loss}[state["case"]["op"]](state)


def _spread(scales, block_rows, block_columns, rows, columns):
    """Scales as a matrix of the codes' size."""
    return scales.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(block_columns, 1)[:, :columns]


def _product(state):
    case, left, right = state["case"], state["left"], state["right"]
    dtype = TYPES[case["type"]]
    if own:
        from gram_newton_schulz_ampere_b200 import ops

        return ops.gemm_8bit(left, state["left_scales"], right, state["right_scales"], out_dtype=dtype)
    m, k, n = case["m"], case["k"], case["n"]
    a = left.float() * _spread(state["left_scales"], 1, BLOCK, m, k)
    b = right.float() * _spread(state["right_scales"], BLOCK, BLOCK, k, n)
    return (a @ b).to(dtype)


def _rounded(x, block_rows):
    """A matrix as its codes and scales hold it, in 32 bits."""
    codes, scales = _quantized(x.float(), block_rows)
    return codes.float() * _spread(scales, block_rows, BLOCK, *x.shape)


def _linear(state):
    x, weight, grad = state["x"], state["weight"], state["grad"]
    if own:
        from gram_newton_schulz_ampere_b200 import training

        y = training.linear_8bit(x, weight)
        dx, dweight = torch.autograd.grad(y, (x, weight), grad)
        return {"y": y.detach(), "x": dx, "weight": dweight}
    with torch.no_grad():
        w8 = _rounded(weight, BLOCK)
        y = _rounded(x, 1) @ w8.t()
        dx = _rounded(grad, 1) @ w8
        dweight = grad.float().t() @ x.float()
        return {"y": y.to(x.dtype), "x": dx.to(x.dtype), "weight": dweight.to(weight.dtype)}


def _norm(state):
    x, residual, weight, grad, eps = (state[k] for k in ("x", "residual", "weight", "grad", "epsilon"))
    eight = state["case"]["bits"] == 8
    if own:
        from gram_newton_schulz_ampere_b200 import ops

        if eight:
            codes, scales, total, rstd = ops.rms_norm_8bit(x, weight, residual, eps)
            out = {"codes": codes, "scales": scales}
        else:
            y, total, rstd = ops.rms_norm(x, weight, residual, eps)
            out = {"y": y}
        if residual is not None:
            out["total"] = total
        if grad is not None:
            out["x"], out["weight"] = ops.rms_norm_backward(grad, total, weight, rstd, state["grad_total"])
        return out
    total = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    h, w = total.float(), weight.float()
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + eps)
    y = h * rstd * w
    out = dict(zip(("codes", "scales"), _quantized(y, 1))) if eight else {"y": y.to(x.dtype)}
    if residual is not None:
        out["total"] = total
    if grad is not None:
        dy, unit = grad.float(), h * rstd
        inner = dy * w
        dx = rstd * (inner - unit * (inner * unit).mean(1, keepdim=True))
        if state["grad_total"] is not None:
            dx = dx + state["grad_total"].float()
        out["x"], out["weight"] = dx.to(x.dtype), (dy * unit).sum(0).to(weight.dtype)
    return out


def _loss(state):
    case, logits, indices, teacher, grad = (state[k] for k in ("case", "logits", "indices", "teacher", "grad"))
    t = case["temperature"]
    if own:
        from gram_newton_schulz_ampere_b200 import ops

        if case["pass"] == "one":
            loss, dlogits = ops.distillation_loss_gradient(grad, logits, indices, teacher, t)
            return {"loss": loss, "logits": dlogits}
        loss, statistics = ops.distillation_loss(logits, indices, teacher, t)
        if case["pass"] == "loss":
            return loss
        return {"loss": loss,
                "logits": ops.distillation_loss_backward(grad, logits, indices, teacher, statistics, t)}
    there = (indices >= 0) & (indices < case["vocabulary"])
    at = torch.where(there, indices, 0).long()
    counts = there.any(1)
    log_p = teacher.float() / t
    log_p = torch.where(there, log_p, -math.inf)
    log_p = log_p - torch.where(counts, log_p.amax(1), 0.0)[:, None]
    log_p = log_p - torch.where(counts, log_p.exp().sum(1).log(), 0.0)[:, None]
    p = log_p.exp()
    z = logits.float() / t
    z = z - z.amax(1, keepdim=True)
    e = z.exp()
    total = e.sum(1, keepdim=True)
    log_q = z.gather(1, at) - total.log()
    loss = t * t * torch.where(there, p * (log_p - log_q), 0.0).sum(1)
    if case["pass"] == "loss":
        return loss
    scale = torch.where(counts, grad * t, 0.0)[:, None]
    dlogits = (e / total).scatter_add_(1, at, torch.where(there, -p, 0.0)) * scale
    return {"loss": loss, "logits": dlogits.to(logits.dtype)}


# ----------------------------------------------------------------- the floor
def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    es = _size(case["type"])
    if case["op"] in ("product", "linear"):
        m, k, n = case["m"], case["k"], case["n"]
        blocks = _round_up(k, BLOCK) // BLOCK
        if case["op"] == "product":
            scales = 4 * blocks * (m + _round_up(n, BLOCK) // BLOCK)
            return {"bytes": m * k + k * n + scales + es * m * n, "flops": 2 * m * k * n}
        return {"bytes": es * (2 * m * k + 2 * m * n + 2 * k * n), "flops": 6 * m * k * n}
    if case["op"] == "norm":
        cells, ws = case["rows"] * case["columns"], _size(case["weight"])
        moved = es * (1 + 2 * case["residual"]) + (1 + 4 / BLOCK if case["bits"] == 8 else es)
        flops = 8
        if case["backward"]:
            moved += es * (2 + case["residual"])
            flops += 12
        return {"bytes": moved * cells + ws * case["columns"] * (1 + case["backward"]), "flops": flops * cells}
    cells, entries = case["rows"] * case["vocabulary"], case["rows"] * case["top"]
    moved = es * cells * (1 if case["pass"] == "loss" else 2)
    return {"bytes": moved + entries * (8 if case["indices"] == "i32" else 12) + 8 * case["rows"],
            "flops": (4 if case["pass"] == "loss" else 8) * cells}


# ------------------------------------------------------- the same in 64 bits
def _nearest(values):
    """Each value's nearest e4m3 value, in 64 bits, ties to the even one, at most 448."""
    table = torch.arange(127, dtype=torch.uint8, device=values.device).view(torch.float8_e4m3fn).double()
    middle = (table[1:] + table[:-1]) / 2
    size = values.abs()
    low = torch.bucketize(size, middle)  # the lower one at a tie
    tie = (low < 126) & (size == middle[low.clamp_max(125)]) & (low % 2 == 1)
    return torch.sign(values) * table[torch.where(tie, low + 1, low)]


def _exact_blocks(x, block_rows):
    """Codes and scales of a matrix, both in 64 bits, a block row at a time."""
    codes, scales = torch.empty_like(x), []
    for b in range(0, x.shape[1], BLOCK):
        part = x[:, b:b + BLOCK]
        if block_rows == 1:
            top = part.abs().amax(1)
            every = top[:, None]
        else:
            top = torch.stack([r.abs().max() for r in part.split(block_rows)])
            every = top.repeat_interleave(block_rows)[:x.shape[0], None]
        codes[:, b:b + BLOCK] = _nearest(part * TOP / every.clamp_min(LEAST))
        scales.append(top.clamp_min(LEAST) / TOP)
    return codes, torch.stack(scales, 1)


def _exact_values(x, block_rows):
    codes, scales = _exact_blocks(x.double(), block_rows)
    for b in range(scales.shape[1]):
        by_row = scales[:, b].repeat_interleave(block_rows)[:x.shape[0], None]
        codes[:, b * BLOCK:(b + 1) * BLOCK] *= by_row
    return codes


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "product":
        out = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        left, right = state["left"].to(torch.float64), state["right"].to(torch.float64)
        for i in range(state["left_scales"].shape[1]):
            here = slice(i * BLOCK, (i + 1) * BLOCK)
            by_column = state["right_scales"][i].double().repeat_interleave(BLOCK)[:case["n"]]
            out.addmm_(left[:, here] * state["left_scales"][:, i:i + 1].double(), right[here] * by_column)
        return out
    if case["op"] == "linear":
        with torch.no_grad():
            x, weight, grad = state["x"].detach(), state["weight"].detach(), state["grad"]
            w = _exact_values(weight, BLOCK)
            return {"y": torch.einsum("mk,nk->mn", _exact_values(x, 1), w),
                    "x": torch.einsum("mn,nk->mk", _exact_values(grad, 1), w),
                    "weight": torch.einsum("mn,mk->nk", grad.double(), x.double())}
    if case["op"] == "norm":
        h = state["x"]
        out = {}
        if state["residual"] is not None:
            summed = state["x"].double() + state["residual"].double()
            out["total"] = summed
            h = summed.to(h.dtype)  # the stream is kept in its type, and the norm is of what is kept
        h, w = h.double(), state["weight"].double()
        size = torch.sqrt(h.square().sum(1) / case["columns"] + state["epsilon"])
        y = h / size[:, None] * w
        if case["bits"] == 8:
            out["codes"], out["scales"] = _exact_blocks(y, 1)
        else:
            out["y"] = y
        if case["backward"]:
            dy = state["grad"].double()
            inner = (dy * w * h).sum(1) / case["columns"]
            dx = dy * w / size[:, None] - h * (inner / size**3)[:, None]
            out["x"] = dx if state["grad_total"] is None else dx + state["grad_total"].double()
            out["weight"] = (dy * h / size[:, None]).sum(0)
        return out
    t, v = case["temperature"], case["vocabulary"]
    loss = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    dlogits = None if case["pass"] == "loss" else torch.empty((case["rows"], v), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // v)
    for first in range(0, case["rows"], step):
        rows = slice(first, first + step)
        z, teacher = state["logits"][rows].double() / t, state["teacher"][rows].double() / t
        index = state["indices"][rows].long()
        there = (index >= 0) & (index < v)
        some = there.any(1)
        share = torch.where(there, torch.exp(teacher - teacher.amax(1, keepdim=True)), 0.0)
        share = share / torch.where(some, share.sum(1), 1.0)[:, None]
        log_share = torch.log(torch.where(share > 0, share, 1.0))
        lse = torch.logsumexp(z, 1, keepdim=True)
        log_q = torch.gather(z, 1, index.clamp(0, v - 1)) - lse
        loss[rows] = t * t * (share * torch.where(there, log_share - log_q, 0.0)).sum(1)
        if dlogits is not None:
            q = torch.exp(z - lse)
            q.scatter_add_(1, index.clamp(0, v - 1), -share)
            dlogits[rows] = q * (t * state["grad"][rows].double() * some)[:, None]
    return loss if dlogits is None else {"loss": loss, "logits": dlogits}
