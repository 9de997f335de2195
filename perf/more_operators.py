"""A model's projections in 8-bit integers with one scale for each token and one for each output channel, and the loss of a prompt's tokens on such an
output projection (nihilus_amd.i8).

product   rows of activations brought to 8 bits, each with its own scale (as they are, behind an RMS norm, or as silu(gate) * up), times a matrix
          whose rows have a scale each, and a residual added
loss      softmax cross entropy of each row's next token over the whole vocabulary, and the log of the softmax's sum, without the logits
train     the same with the gradient of the rows

The number x stands for is round(x / s) * s, s = max |x| / 127 of its row as a 32-bit float; sums of such products are whole numbers, and exact.  A gradient
is taken with respect to the rounded rows.  Sizes are those of the LLaMA-3-8B and 70B shapes (4096 and 8192 values, 14336 and 28672 in the
feed-forward part, 128256 tokens) and, in draw(), any.
"""
import math
import random

import torch

own = False

V = 128256
EPS = 1e-5
SCALED = 127.0


def listed():
    return [
        # One token through a query projection: the smallest call there is, between two launches of a decode step.
        {"name": "product_one_token", "op": "product", "rows": 1, "k": 4096, "n": 4096, "front": "plain", "residual": False, "type": "float32"},
        # One token through the gate projection, behind the norm.
        {"name": "product_one_token_gate", "op": "product", "rows": 1, "k": 4096, "n": 14336, "front": "norm", "residual": False, "type": "float32"},
        # A decode step of 13 sequences through the output projection of a 70B attention.
        {"name": "product_13_rows", "op": "product", "rows": 13, "k": 8192, "n": 8192, "front": "plain", "residual": True, "type": "bfloat16"},
        # A short prompt of an odd length, 32-bit activations, behind the norm.
        {"name": "product_prompt_117", "op": "product", "rows": 117, "k": 4096, "n": 14336, "front": "norm", "residual": False, "type": "float32"},
        # Sizes that no tile divides.
        {"name": "product_odd_1001", "op": "product", "rows": 1001, "k": 1507, "n": 5003, "front": "plain", "residual": True, "type": "float16"},
        # An ordinary prompt through the down projection, behind silu(gate) * up.
        {"name": "product_down_512", "op": "product", "rows": 512, "k": 14336, "n": 4096, "front": "silu", "residual": True, "type": "bfloat16"},
        # A server's batch of prompts through a 70B gate projection.
        {"name": "product_prompt_8192", "op": "product", "rows": 8192, "k": 8192, "n": 28672, "front": "norm", "residual": False, "type": "bfloat16"},
        # What a decode step's tokens were worth: a row for each of three sequences.
        {"name": "loss_3_rows", "op": "loss", "rows": 3, "k": 4096, "n": V, "front": "norm", "type": "float32"},
        # A prompt scored, an odd number of rows.
        {"name": "loss_prompt_2047", "op": "loss", "rows": 2047, "k": 4096, "n": V, "front": "norm", "type": "float32"},
        # A few rows of a short text, 32-bit gradients.
        {"name": "train_5_rows", "op": "train", "rows": 5, "k": 4096, "n": V, "front": "plain", "type": "float32"},
        # Rows of an ordinary text on a smaller vocabulary of an odd size.
        {"name": "train_300_rows", "op": "train", "rows": 300, "k": 2048, "n": 32003, "front": "plain", "type": "float32"},
        # A batch of a learner that trains what is in front of a frozen model's output projection.
        {"name": "train_2048_rows", "op": "train", "rows": 2048, "k": 4096, "n": V, "front": "plain", "type": "bfloat16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["product", "product", "product", "loss", "loss", "train", "train"])
    kind = rng.choice(["float32", "float16", "bfloat16"])
    if op == "product":
        case = {"op": op, "rows": _log_int(rng, 1, 8192), "k": _log_int(rng, 64, 16384), "n": _log_int(rng, 64, 32768), "front": rng.choice(["plain", "norm", "silu"]), "residual": rng.random() < 0.5}
        if case["front"] == "silu" and kind == "float32":
            kind = "bfloat16"
    else:
        case = {"op": op, "rows": _log_int(rng, 1, 2048), "k": _log_int(rng, 256, 8192), "n": _log_int(rng, 1000, 131072), "front": rng.choice(["plain", "norm"]) if op == "loss" else "plain"}
        most = 2048 * 4096 * V
        case["rows"] = max(1, min(case["rows"], most // (case["k"] * case["n"])))
    if rng.random() < 0.5:  # sizes that models have, in the other half any
        case["k"], case["n"] = max(64, case["k"] // 64 * 64), max(64, case["n"] // 64 * 64)
    case["type"] = kind
    return case


class _Source:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.generator = torch.Generator(device="cuda")
        self.generator.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, std=1.0):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=self.generator)

    def uniform(self, *shape):
        return torch.empty(shape, dtype=torch.float32, device="cuda").uniform_(0.0, 1.0, generator=self.generator)


def _weight(source, n, k, std):
    """[n, k] in 8 bits with a scale for each row, rows of different sizes as trained ones are."""
    quants = torch.empty((n, k), dtype=torch.int8, device="cuda")
    scales = torch.empty(n, dtype=torch.float32, device="cuda")
    for at in range(0, n, 16384):
        part = min(16384, n - at)
        w = source.normal(part, k, std=std) * (0.5 + source.uniform(part, 1))
        scales[at : at + part] = w.abs().amax(dim=1) / SCALED
        quants[at : at + part] = (w / scales[at : at + part, None]).round()
    return quants, scales


def prepare(case, seed):
    source = _Source(seed)
    rows, k, n, op = case["rows"], case["k"], case["n"], case["op"]
    kind = getattr(torch, case["type"])
    quants, scales = _weight(source, n, k, 0.02 if op == "product" else 0.05)
    state = {"op": op, "case": case, "quants": quants, "scales": scales}
    if case["front"] == "silu":
        state["gate"], state["up"] = source.normal(rows, k, dtype=kind, std=2.0), source.normal(rows, k, dtype=kind)
    elif op == "product":
        # a few of the values are far larger than the others, as they are between a model's layers
        x = source.normal(rows, k) * torch.exp(0.5 * source.normal(1, k))
        state["x"] = x.to(kind)
    if case["front"] == "norm":
        state["norm"] = 1.0 + 0.2 * source.normal(k)
    if op == "product":
        state["residual"] = source.normal(rows, n, dtype=kind) if case["residual"] else None
    else:
        # rows lean towards the token that follows, most of them clearly; one in ten is not scored
        targets = (source.uniform(rows) * n).long().clamp(max=n - 1)
        row = quants[targets].float()
        lean = row / row.norm(dim=1, keepdim=True).clamp(min=1.0)
        state["x"] = (source.normal(rows, k) + (3.0 + source.normal(rows, 1)) * lean).to(kind)
        state["targets"] = torch.where(source.uniform(rows) < 0.1, -1, targets).to(torch.int32)
        if op == "train":
            state["grad"] = source.uniform(rows) / rows
    if own:
        from nihilus_amd import i8

        state["w"] = i8.tile(quants, scales)
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------------------


def _front(s):
    """The rows that are brought to 8 bits, 32-bit floats."""
    front = s["case"]["front"]
    if front == "silu":
        gate = s["gate"].to(torch.float64)
        return (gate / (1.0 + torch.exp(-gate)) * s["up"].to(torch.float64)).to(torch.float32)
    x = s["x"].to(torch.float32)
    if front == "norm":
        wide = x.to(torch.float64)
        x = x * torch.rsqrt((wide * wide).mean(dim=1, keepdim=True) + EPS).to(torch.float32) * s["norm"]
    return x


def _rounded(x):
    """Whole numbers (as 32-bit floats) and the rows' scales; quotients in 64 bits, where none that is not a half rounds to one."""
    scale = (x.abs().amax(dim=1, keepdim=True).to(torch.float64) / SCALED).to(torch.float32)
    return (x.to(torch.float64) / scale.to(torch.float64)).nan_to_num_(0.0).round_().clamp_(-SCALED, SCALED).to(torch.float32), scale


def _logits(s):
    x, scale = _rounded(_front(s))
    return torch.matmul(x, s["quants"].to(torch.float32).t()).mul_(scale).mul_(s["scales"])


def _softmax(s, logits):
    """(losses, logs of the sums, weights in the logits' place, which rows are scored)"""
    scored = s["targets"] >= 0
    at = s["targets"].long().clamp(min=0)[:, None]
    hit = logits.gather(1, at)
    top = logits.amax(dim=1, keepdim=True)
    weights = logits.sub_(top).exp_()
    total = weights.sum(dim=1, keepdim=True)
    lse = top + total.log()
    return torch.where(scored, (lse - hit)[:, 0], 0.0), lse[:, 0], weights.div_(total), scored


def _plain(s):
    logits = _logits(s)
    if s["op"] == "product":
        if s["residual"] is not None:
            logits += s["residual"].to(torch.float32)
        return logits.to(getattr(torch, s["case"]["type"]))
    losses, lse, weights, scored = _softmax(s, logits)
    if s["op"] == "loss":
        return {"losses": losses, "lse": lse}
    weights.scatter_add_(1, s["targets"].long().clamp(min=0)[:, None], torch.full((len(scored), 1), -1.0, device=weights.device))
    weights.mul_(torch.where(scored, s["grad"], 0.0)[:, None]).mul_(s["scales"])
    dx = torch.matmul(weights, s["quants"].to(torch.float32))
    return {"losses": losses, "lse": lse, "dx": dx.to(s["x"].dtype)}


def run(state):
    s = state
    if not own:
        return _plain(s)
    from nihilus_amd import i8

    case, w = s["case"], s["w"]
    rows, n, k = case["rows"], case["n"], case["k"]
    if s["op"] == "product":
        if case["front"] == "silu":
            return i8.gemm(w, i8.silu_mul_quantize(s["gate"], s["up"]), rows, n, k, dtype=s["gate"].dtype, residual=s["residual"])
        if case["front"] == "norm":
            return i8.mul_mat(w, s["x"], n, k, residual=s["residual"], norm_weight=s["norm"], eps=EPS)
        return i8.mul_mat(w, s["x"], n, k, residual=s["residual"])
    xq = i8.rms_norm_quantize(s["x"], s["norm"], EPS) if case["front"] == "norm" else i8.quantize(s["x"])
    losses, lse = i8.token_losses(w, xq, s["targets"], n, k)
    if s["op"] == "loss":
        return {"losses": losses, "lse": lse}
    return {"losses": losses, "lse": lse, "dx": i8.token_losses_grad(w, xq, s["targets"], losses, lse, n, k, grad=s["grad"], dtype=s["x"].dtype)}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------


def work(case):
    rows, n, k = case["rows"], case["n"], case["k"]
    wide = 4 if case["type"] == "float32" else 2
    moved = n * k + 4 * n + rows * k * wide * (2 if case["front"] == "silu" else 1) + (4 * k if case["front"] == "norm" else 0)
    if case["op"] == "product":
        return {"bytes": moved + rows * n * wide * (2 if case["residual"] else 1), "flops": 2 * rows * n * k}
    if case["op"] == "loss":
        return {"bytes": moved + 12 * rows, "flops": 2 * rows * n * k}
    return {"bytes": moved + 16 * rows + rows * k * wide, "flops": 4 * rows * n * k}


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------------------


def _exact_rows(s, case):
    """What each value stands for once it is rounded, in 64 bits.  Rows are 32-bit floats, and so are their scales: that rounding is the definition's."""
    def single(v):
        return v.float().double()

    if case["front"] == "silu":
        rows = single(s["gate"].double() * torch.sigmoid(s["gate"].double()) * s["up"].double())
    else:
        rows = s["x"].double()
        if case["front"] == "norm":
            size = single(1.0 / torch.sqrt(torch.linalg.vector_norm(rows, dim=1).square() / case["k"] + EPS))
            rows = single(single(rows * size[:, None]) * s["norm"].double())
    step = single(torch.linalg.vector_norm(rows, ord=math.inf, dim=1) / 127)
    step = torch.where(step == 0, 1.0, step)[:, None]
    return torch.clamp(torch.round(rows / step), -127, 127) * step


def exact(case, seed):
    s = prepare(case, seed)
    w = s["quants"].double()
    w *= s["scales"].double()[:, None]
    x = _exact_rows(s, case)
    if case["op"] == "product":
        y = torch.mm(x, w.t())
        return y if s["residual"] is None else y + s["residual"].double()
    found = {name: [] for name in ("losses", "lse", "dx")}
    for at in range(0, case["rows"], 512):  # so many rows at a time
        part = x[at : at + 512]
        logits = torch.mm(part, w.t())
        lse = torch.logsumexp(logits, dim=1)
        targets = s["targets"][at : at + 512].long()
        kept = targets >= 0
        row = torch.arange(len(part), device=x.device)
        found["lse"].append(lse)
        found["losses"].append((lse - logits[row, targets.clamp(min=0)]) * kept)
        if case["op"] == "train":
            slope = torch.exp(logits - lse[:, None])
            slope[row[kept], targets[kept]] -= 1.0
            found["dx"].append(torch.mm(slope * (s["grad"][at : at + 512].double() * kept)[:, None], w))
    return {name: torch.cat(parts) for name, parts in found.items() if parts}
