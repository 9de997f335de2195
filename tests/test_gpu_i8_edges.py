"""GPU: the ends of what int8 rows, the losses on them and their gradient are given: result types against each other, rows that are sure of their target, logits and gates of any size."""
import pytest
import torch

import i8_reference as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def i8():
    from nihilus_amd import i8

    i8._lib.lib()
    return i8


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, dtype=torch.float32, std=1.0):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=g)


def _matrix(g, rows, k):
    q = torch.randint(-127, 128, (rows, k), device="cuda", dtype=torch.int8, generator=g)
    return q, torch.empty(rows, device="cuda").uniform_(0.5, 1.5, generator=g) / (127.0 * max(k, 1) ** 0.5)


# ---- gates of any size


def _silu_rows(gate, up):
    """silu(gate) up in 64 bits (exp(-gate) of gates far down is past them: gate exp(gate) there)"""
    g = gate.double()
    return torch.where(g < -600, g * torch.exp(g.clamp(max=-600)), g / (1.0 + torch.exp(-g.clamp(min=-600)))) * up.double()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("k", [70, 9000, 40000])
def test_silu_of_gates_of_any_size(i8, k, kind):
    most = torch.finfo(kind).max
    tops = [60.0, 79.0, 81.0, 88.0, 104.0, 1000.0, 65504.0, 1e30, 2.3e38, 2.4e38, 3.3e38]
    tops = torch.tensor([t for t in tops if t <= most] + [most], device="cuda")
    g = _gen(k)
    # rows of gates that are all far up, all far down (what is left of them, or nothing), of either sign, and a single one among ordinary ones
    size = tops[:, None] * torch.empty(len(tops), k, device="cuda").uniform_(0.95, 1.0, generator=g)
    size[:, 0] = tops
    ordinary = _normal(g, len(tops), k, std=3.0)
    single, down = ordinary.clone(), ordinary.clone()
    single[:, 3], down[:, k - 2] = tops, -tops
    signs = torch.randint(0, 2, (len(tops), k), device="cuda", generator=g) * 2 - 1
    gate = torch.cat([size, -size, size * signs, single, down]).to(kind)
    up = _normal(g, *gate.shape, dtype=kind).clamp(-1, 1)
    q, s = i8.untile(i8.silu_mul_quantize(gate, up), *gate.shape)
    v = _silu_rows(gate, up)
    # v within 3 units of 2^-23 of itself, or of the smallest number; the scale is rounded once more, and the whole number is one of the two next to the quotient
    top = v.abs().amax(dim=1)
    assert torch.isfinite(s).all() and ((s.double() - top / 127).abs() <= 8 * R.U * top / 127 + 4 * 2.0**-149).all()
    few = 2.0**-149 * 4 / s.double().clamp(min=2.0**-149)[:, None]  # (units of the smallest number in a scale: more than a few bits only far below the normal numbers)
    off = (q.double() * s.double()[:, None] - v).abs()
    assert (off <= s.double()[:, None] * (0.5 + 127 * (16 * R.U + few)) + 4 * 2.0**-149).all()
    far = (gate[:, 1:] < -140).all(dim=1)
    assert far.sum() >= 2 and (s[far] == 0).all() and (q[far] == 0).all()


def test_silu_of_gates_that_are_not_finite(i8):
    gate, up = torch.zeros(5, 100, device="cuda"), torch.ones(5, 100, device="cuda")
    gate[0, 7], gate[1, 8], gate[2, 9] = float("nan"), float("inf"), -float("inf")  # (an infinity over an infinity)
    gate[3, 0] = 3e38
    gate[4] = 1.0
    q, s = i8.untile(i8.silu_mul_quantize(gate, up), 5, 100)
    assert torch.isnan(s[:3]).all() and (q[:3] == 0).all() and torch.isfinite(s[3:]).all() and q[3, 0] == 127


# ---- gradients of every type


# (one pass over the vocabulary, and tiles; pieces of it at 8192 rows)
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 1000, 64), (5, 4099, 576), (16, 600, 4096), (3, 900, 4160), (17, 700, 130), (160, 3008, 1280), (310, 2001, 300), (8192, 4200, 64)])
def test_a_gradient_in_16_bits_is_the_one_of_32_rounded(i8, m, n, k, kind):
    g = _gen(m + n + k)
    (wq, ws), x = _matrix(g, n, k), _normal(g, m, k)
    w, xq = i8.tile(wq, 4.0 * ws), i8.quantize(x)
    targets = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32, generator=g)
    losses, lse = i8.token_losses(w, xq, targets, n, k)
    grad = torch.rand(m, device="cuda", generator=g)
    wide, narrow = (i8.token_losses_grad(w, xq, targets, losses, lse, n, k, grad=grad, dtype=t) for t in (torch.float32, kind))
    # The last product (a row's grad) may be rounded to fp16 at once, which leaves another number only where fp32 rounds it to the middle of two: both are as far from it then, exactly.
    far = [(t.double() - wide.double()).abs() for t in (narrow, wide.to(kind))]
    assert wide.abs().max() > 0 and torch.equal(*far) and (kind != torch.bfloat16 or torch.equal(narrow, wide.to(kind)))


# ---- rows that are sure of their target, at logits of any size


def _exact_logits(wanted, fine):
    """wanted [m, n] fp64, multiples of 2^-fine[i] in row i and below 2^18 of them: int8 operands and scales (powers of two, of three sizes) whose products are exactly those, row i in 64 values of its own.

    A row's 62 values of 127 and one of 1 are met by 62 values whose sum is a token's number / 127, and the rest."""
    m, n = wanted.shape
    steps = (wanted * torch.tensor([2.0**f for f in fine], dtype=torch.float64)[:, None]).round().long()
    ws = torch.tensor([2.0 ** -(j % 3) for j in range(n)])
    whole = steps * (1.0 / ws).long()[None]  # of 2^-fine ws
    assert whole.abs().max() <= 62 * 127 * 127
    most = (whole.abs() + 63) // 127
    places = torch.arange(62)
    wq, xq = torch.zeros(n, 64 * m, dtype=torch.int8), torch.zeros(m, 64 * m, dtype=torch.int8)
    for i in range(m):
        part = ((most[i][:, None] - 127 * places).clamp(0, 127) * whole[i].sign()[:, None]).to(torch.int8)
        wq[:, 64 * i : 64 * i + 62] = part
        wq[:, 64 * i + 62] = (whole[i] - 127 * part.long().sum(1)).to(torch.int8)
        xq[i, 64 * i : 64 * i + 62], xq[i, 64 * i + 62] = 127, 1
    xs = torch.tensor([2.0**-f for f in fine])
    wq, ws, xq, xs = (t.cuda() for t in (wq, ws, xq, xs))
    l = R.logits(wq, ws, xq, xs)
    assert torch.equal(l.cpu(), steps.double() / torch.tensor([2.0**f for f in fine], dtype=torch.float64)[:, None])
    return wq, ws, xq, xs, l


# largest logit, how fine the logits are
SIZES = [(25.0, 11), (300.0, 9), (4000.0, 5), (20000.0, 2), (-20000.0, 2), (30000.0, 2), (120000.0, 0)]


def _sure_case(m, n, seed=0):
    """Rows of every size of logits, with a few tokens from 1/4 to 14 below the target's (which is theirs in one row of five), all others 40 to 90 below."""
    g = torch.Generator().manual_seed(seed + m)
    wanted, fine, targets = torch.empty(m, n, dtype=torch.float64), [], torch.empty(m, dtype=torch.int32)
    for i in range(m):
        top, f = SIZES[i % len(SIZES)]
        fine.append(f)
        gaps = 40.0 + 50.0 * torch.rand(n, generator=g, dtype=torch.float64)
        order = torch.randperm(n, generator=g)
        near = 1 + i % 3
        gaps[order[0]] = 0.0
        gaps[order[1 : 1 + near]] = [0.25, 1.0, 3.0, 6.0, 8.0, 9.0, 11.0, 14.0][i // 2 % 8] + torch.randint(0, 2, (near,), generator=g).double()
        wanted[i] = ((top - gaps) * 2**f).round() / 2**f
        targets[i] = order[1] if i % 5 == 3 else order[0]
    return (*_exact_logits(wanted, fine), targets.cuda())


def _sum_bound(l):
    """How far the log of a row's sum of exponentials, over the largest, may be off.  The differences are exact here.  An addition rounds by U of the sum: 32 of a lane and two among lanes in a stretch, one to a thread
    (stretches are fewer than threads), six among lanes, and one of the two waves or three of more.  An exponential below the largest is off by twice its exponent's and the two ulp (4 U): 6 U where it is most, and so
    again wherever it is joined to a larger one, seven times at most."""
    s = torch.exp(l - l.amax(dim=1, keepdim=True)).sum(dim=1)
    return R.U * (44 + 48 * (1 - 1 / s))


SURE = [(5, 331), (16, 600), (40, 331), (300, 250)]


@pytest.mark.parametrize("m,n", SURE)
def test_losses_of_rows_that_are_sure(i8, m, n):
    wq, ws, xq, xs, l, targets = _sure_case(m, n)
    losses, lse = i8.token_losses(i8.tile(wq, ws), i8.tile(xq, xs), targets, n, 64 * m)
    want, want_lse = R.losses(l, targets)
    # the target's distance from the largest is exact; a logarithm of two ulp, and a sum
    assert ((losses.double() - want).abs() <= _sum_bound(l) + 6 * R.U * want).all()
    assert ((lse.double() - want_lse).abs() <= _sum_bound(l) + 6 * R.U * want + R.U * want_lse.abs()).all()


def _sure_bound(l, targets, wq, ws, kind, grad):
    n = l.shape[1]
    losses, lse = R.losses(l, targets)
    want, d = R.gradient(l, targets, wq, ws, grad), R.slopes(l, targets)
    own = torch.zeros_like(d, dtype=torch.bool).scatter_(1, targets.long()[:, None], True)
    # The target's slope, exp(-loss) - 1: as exact as the loss, and two ulp.  The others, exp(l - lse): lse's rounding and its sum's, a difference and a product by log2 e (3 U of the exponent), two ulp.
    off_own = (torch.exp(-losses) * (_sum_bound(l) + 6 * R.U * losses))[:, None] + 4 * R.U * d.abs()
    off = torch.where(own, off_own, d.abs() * (R.U * lse.abs() + _sum_bound(l) + 6 * R.U * losses)[:, None] + d.abs() * R.U * (3 * (lse[:, None] - l) + 4))
    # two products, two fp16 numbers (2^-22 of a slope, or half of the smallest number, 2^-25, where the largest is 2^12 or more), sums over n in fp32
    off = off + d.abs() * (2 * R.U + 2.0**-22 + (n + 64) * R.U)
    least = 2.0**-25 * 2.0**-12 * (-torch.expm1(-losses)).clamp(min=2.0**-16)[:, None] * 2 * ws.max().double() * wq.double().abs().sum(0)[None]
    return (off @ (wq.double().abs() * ws.double()[:, None]) + least) * grad.double()[:, None] + want.abs() * (R.HALF[kind] + 2 * R.U) + (2.0**-25 if kind == torch.float16 else 0.0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n", SURE)
def test_gradient_of_rows_that_are_sure(i8, m, n, kind):
    wq, ws, xq, xs, l, targets = _sure_case(m, n)
    w, x = i8.tile(wq, ws), i8.tile(xq, xs)
    losses, lse = i8.token_losses(w, x, targets, n, 64 * m)
    grad = torch.rand(m, device="cuda", generator=_gen(m))
    dx = i8.token_losses_grad(w, x, targets, losses, lse, n, 64 * m, grad=grad, dtype=kind).double()
    want, bound = R.gradient(l, targets, wq, ws, grad), _sure_bound(l, targets, wq, ws, kind, grad)
    assert torch.isfinite(dx).all() and ((dx - want).abs() <= bound).all()
    # ... which says something of every row whose loss is above 1e-4, whatever its logits
    told = R.losses(l, targets)[0] > 1e-4
    assert told.sum() >= m // 2 and ((bound.amax(1) < 0.2 * want.abs().amax(1)) | ~told).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m", [8, 24])
def test_gradient_of_two_tokens_far_up(i8, m, kind):
    # A loss in steps of lse's last place was nothing here, and the other token's slope, which lse does not hide, past fp16 in units of the smallest.
    n = 40
    sizes = [(9000.0, 8.0, 4), (20000.0, 7.75, 2), (20000.0, 6.25, 2), (50000.0, 9.0, 1), (100000.0, 7.0, 0), (-100000.0, 8.0, 0), (2.0**22, 32.0, -5), (2.0**29, 2.0**12, -12)]
    wanted, fine = torch.empty(m, n, dtype=torch.float64), [sizes[i % 8][2] for i in range(m)]
    targets = torch.tensor([(7 * i + 3) % n for i in range(m)], dtype=torch.int32)
    for i in range(m):
        top, gap, f = sizes[i % 8]
        wanted[i] = top - max(64.0, 2.0**-f)
        wanted[i, targets[i]], wanted[i, (7 * i + 3 + i) % n if i % n else 0] = top, top - gap
    wq, ws, xq, xs, l = _exact_logits(wanted, fine)
    targets = targets.cuda()
    w, x, grad = i8.tile(wq, ws), i8.tile(xq, xs), torch.ones(m, device="cuda")
    losses, lse = i8.token_losses(w, x, targets, n, 64 * m)
    dx = i8.token_losses_grad(w, x, targets, losses, lse, n, 64 * m, dtype=kind).double()
    assert torch.isfinite(dx).all()
    assert ((dx - R.gradient(l, targets, wq, ws, grad)).abs() <= _sure_bound(l, targets, wq, ws, kind, grad)).all()


@pytest.mark.parametrize("m", [3, 40, 300])
def test_losses_of_logits_past_fp32(i8, m):
    # a row's scale is so large that some logits, or all of a stretch, are infinite: the sums' scale takes the first 128 tokens there, the others' takes them back
    n, k = 700, 64
    g = _gen(m)
    wq, ws = _matrix(g, n, k)
    xq = torch.randint(1, 128, (m, k), device="cuda", dtype=torch.int8, generator=g)
    xs = torch.full((m,), 2.0**100, device="cuda")
    ws[:128] = 2.0**30
    ws[128:] *= 2.0**-100
    wq[:128] = -wq[:128].abs() - 1  # -infinity
    wq[:128].clamp_(min=-127)
    targets = torch.randint(128, n, (m,), device="cuda", dtype=torch.int32, generator=g)
    w, x = i8.tile(wq, ws), i8.tile(xq, xs)
    losses, lse = i8.token_losses(w, x, targets, n, k)
    want, want_lse = R.losses(R.logits(wq[128:], ws[128:], xq, xs), targets - 128)
    l = R.logits(wq[128:], ws[128:], xq, xs)
    assert ((lse.double() - want_lse).abs() <= R.lse_bound(l)).all()
    assert ((losses.double() - want).abs() <= R.lse_bound(l) + R.logit_bound(l) + 4 * R.U * want.abs()).all()
    targets[0] = 5  # a target at -infinity
    losses, lse = i8.token_losses(w, x, targets, n, k)
    assert losses[0] == float("inf") and torch.isfinite(losses[1:]).all() and torch.isfinite(lse).all()
    wq[9] = 127  # and one of all tokens at +infinity
    losses, lse = i8.token_losses(i8.tile(wq, ws), x, targets, n, k)
    assert (lse == float("inf")).all() and (losses == float("inf")).all()
    targets[0] = 9  # infinity less infinity
    losses, _ = i8.token_losses(i8.tile(wq, ws), x, targets, n, k)
    assert torch.isnan(losses[0]) and (losses[1:] == float("inf")).all()
    ws[9] = float("nan")
    losses, lse = i8.token_losses(i8.tile(wq, ws), x, targets, n, k)
    assert torch.isnan(lse).all() and torch.isnan(losses).all()


# ---- memory


# (one pass over the vocabulary; tiles of an odd last strip, several heights and splits; two pieces of the vocabulary; rows past 8192, cut as the first ones)
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(5, 50, 70), (16, 2001, 1000), (33, 2001, 130), (310, 2001, 130), (129, 16404, 200), (40, 33, 5000), (8192, 4200, 64), (8217, 700, 64)])
def test_workspaces_of_the_losses_are_enough(i8, m, n, k, kind):
    g = _gen(m + n)
    w, x = i8.tile(*_matrix(g, n, k)), i8.quantize(_normal(g, m, k))
    targets = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32, generator=g)
    losses, lse = i8.token_losses(w, x, targets, n, k)
    dx = i8.token_losses_grad(w, x, targets, losses, lse, n, k, dtype=kind)
    for need, call, want in ((i8._need("nh_i8_token_losses_workspace_bytes", m, n, k), lambda ws: i8.token_losses(w, x, targets, n, k, workspace=ws), (losses, lse)),
                             (i8._need("nh_i8_token_losses_grad_workspace_bytes", m, n, k, i8._TYPES[kind]), lambda ws: (i8.token_losses_grad(w, x, targets, losses, lse, n, k, dtype=kind, workspace=ws),), (dx,))):
        for fill in (77, 255):  # (what is there before means nothing: 255 is NaN in every type)
            memory = torch.full((need + 4096,), fill, device="cuda", dtype=torch.uint8)
            assert all(torch.equal(a, b) for a, b in zip(call(memory[:need]), want)) and (memory[need:] == fill).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 77, 100), (1, 4096, 4096), (2, 333, 1000), (4, 515, 1507), (5, 515, 1507), (117, 1003, 512)])
def test_mul_mat_onto_its_residual(i8, m, n, k, kind):
    g = _gen(m + n + k)
    w, x, norm, r = i8.tile(*_matrix(g, n, k)), _normal(g, m, k, dtype=kind), 1.0 + 0.2 * _normal(g, k), _normal(g, m, n, dtype=kind)
    for weight, eps in ((None, 0.0), (norm, 1e-5)):
        want, onto = i8.mul_mat(w, x, n, k, residual=r, norm_weight=weight, eps=eps), r.clone()
        assert i8.mul_mat(w, x, n, k, residual=onto, norm_weight=weight, eps=eps, out=onto) is onto and torch.equal(onto, want)


@pytest.mark.parametrize("m", [5, 40])
def test_targets_at_the_ends_of_their_type(i8, m):
    n, k = 300, 64
    g = _gen(m)
    w, x = i8.tile(*_matrix(g, n, k)), i8.quantize(_normal(g, m, k))
    targets = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32, generator=g)
    losses, lse = i8.token_losses(w, x, targets, n, k)
    dx = i8.token_losses_grad(w, x, targets, losses, lse, n, k)
    targets[0], targets[1], targets[2], targets[3] = -(2**31), 2**31 - 1, -1, n
    some, some_lse = i8.token_losses(w, x, targets, n, k)
    assert (some[:4] == 0).all() and torch.equal(some[4:], losses[4:]) and torch.equal(some_lse, lse)
    some = i8.token_losses_grad(w, x, targets, some, some_lse, n, k)
    assert (some[:4] == 0).all() and torch.equal(some[4:], dx[4:])


@pytest.mark.parametrize("m,n,k", [(5, 700, 300), (40, 700, 300), (300, 2001, 130)])
def test_workspaces_anywhere_at_16_bytes(i8, m, n, k):
    g = _gen(m + n)
    w, x = i8.tile(*_matrix(g, n, k)), _normal(g, m, k)
    xq = i8.quantize(x)
    targets = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32, generator=g)
    losses, lse = i8.token_losses(w, xq, targets, n, k)
    needs = (i8._need("nh_i8_mul_mat_workspace_bytes", m, k), i8._need("nh_i8_token_losses_workspace_bytes", m, n, k), i8._need("nh_i8_token_losses_grad_workspace_bytes", m, n, k, 0))
    for need, call in zip(needs, (lambda ws: (i8.mul_mat(w, x, n, k, workspace=ws),), lambda ws: i8.token_losses(w, xq, targets, n, k, workspace=ws),
                                  lambda ws: (i8.token_losses_grad(w, xq, targets, losses, lse, n, k, workspace=ws),))):
        memory = torch.full((need + 1024,), 77, device="cuda", dtype=torch.uint8)
        for by in (16, 240):
            assert all(torch.equal(a, b) for a, b in zip(call(memory[by : by + need]), call(None))) and (memory[by + need :] == 77).all()
            memory.fill_(77)
