"""The definitions of nihilus_amd/i8.py in 64 bits, with the roundings to 32 that they name, on the CPU or the GPU."""
import torch

U = 2.0**-24  # half a step of fp32, relative
HALF = {torch.float32: U, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}  # half a step relative to the value


def rows_of(x, norm_weight=None, eps=0.0):
    """The fp32 values that are quantized, as fp64."""
    x = x.double()
    if norm_weight is None:
        return x
    r = (1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + torch.tensor(eps, dtype=torch.float32).double().item())).float()
    return ((x.float() * r) * norm_weight.float()).double()


def quantize(v):
    """fp64 rows that hold fp32 values -> (int8, fp32 scales)"""
    top = v.abs().amax(dim=1) if v.shape[1] else v.new_zeros(v.shape[0])
    finite = torch.isfinite(v).all(dim=1)
    scales = (torch.where(finite, top, 0.0) / 127.0).float()
    step = scales.double()[:, None]
    q = torch.where((step > 0) & finite[:, None], torch.round(v / torch.where(step > 0, step, 1.0)), 0.0).clamp(-127, 127)
    return q.to(torch.int8), torch.where(finite, scales, float("nan"))


def product(wq, ws, xq, xs, kind, residual=None):
    """Bit for bit: the whole-number sums, then fp32 operations one at a time, then one rounding."""
    sums = xq.double() @ wq.double().t()  # exact: whole numbers below 2^31
    y = (sums.float() * xs[:, None]) * ws[None, :]
    if residual is not None:
        y = y + residual.float()
    return y.to(kind)


def logits(wq, ws, xq, xs):
    return (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()[None, :]


def losses(l, targets):
    lse = torch.logsumexp(l, dim=1)
    scored = (targets >= 0) & (targets < l.shape[1])
    hit = l.gather(1, targets.long().clamp(0, l.shape[1] - 1)[:, None])[:, 0]
    return torch.where(scored, lse - hit, 0.0), lse


def logit_bound(l):
    """How far a logit of fp32 may be off: a whole number brought to fp32 and two products, three roundings."""
    return 3 * U * l.abs().amax(dim=1)


def lse_bound(l):
    """... and lse: the sum's terms have three more roundings and the exponential's two ulp, (l - maximum) log2 e among them (relative to itself, so U times the
    spread twice), the sums are chains of at most 32 + 2, count / 64 and 64 additions and joins of four roundings each, and lse is a maximum plus a logarithm (two ulp)."""
    spread = l.amax(dim=1) - l.amin(dim=1)
    count = (l.shape[1] + 31) // 32
    return logit_bound(l) + U * (3 * spread + 10 + 34 + 4 * (count / 64 + 1) + 4 * 64) + 6 * U * torch.logsumexp(l, dim=1).abs()


def slopes(l, targets, grad=None):
    lse = torch.logsumexp(l, dim=1)
    d = torch.exp(l - lse[:, None])
    scored = (targets >= 0) & (targets < l.shape[1])
    row = torch.arange(l.shape[0], device=l.device)
    d[row[scored], targets[scored].long()] -= 1.0
    d = torch.where(scored[:, None], d, 0.0)
    return d if grad is None else d * grad.double()[:, None]


def gradient(l, targets, wq, ws, grad=None):
    return slopes(l, targets, grad) @ (wq.double() * ws.double()[:, None])


def gradient_bound(l, targets, wq, ws, kind, grad=None):
    """Per element.  A slope's exponential is off by the logit's and lse's errors and four roundings (relative to itself, so by that times the softmax), the slope by two more; as one fp16 number
    by half a step of it (2^-12 ulp of a normal number, an absolute 2^-25 below 2^-14 of the row's lift of at least 2^12 / most), as two by 2^-22; sums of fp32 over n."""
    w = wq.double().abs() * ws.double().abs()[:, None]
    p = torch.exp(l - torch.logsumexp(l, dim=1)[:, None])
    d = slopes(l, targets).abs()
    g = 1.0 if grad is None else grad.double().abs()[:, None]
    off = (logit_bound(l) + lse_bound(l) + 8 * U)[:, None] * p
    terms = 2.0**-11 if kind != torch.float32 else 2.0**-21
    most = d.amax(dim=1, keepdim=True).clamp(min=2.0**-16)
    sums = (l.shape[1] + 64) * U
    total = (off + d * (terms + sums + 8 * U) + 2.0**-25 * 2.0**-12 * most) @ w + 2.0**-25 * 2.0**-12 * most * ws.abs().max().double() * l.shape[1]
    exact = gradient(l, targets, wq, ws, grad).abs()
    return total * g + exact * (HALF[kind] + 4 * U) + (2.0**-25 if kind == torch.float16 else 0.0)
