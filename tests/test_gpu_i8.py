"""GPU: int8 products with a scale per row of either operand, the losses of a vocabulary projection and their gradient, against the definitions in 64 bits."""
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


# ---- quantizers


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 64), (2, 63), (3, 65), (15, 16), (16, 1000), (17, 4096), (33, 130), (130, 257), (5, 16385), (1, 20000), (1100, 8200), (1030, 5000), (3, 40000)])
def test_quantize(i8, rows, k, kind):
    x = _normal(_gen(rows * k), rows, k, dtype=kind)
    x[:, ::7] *= 5.0
    q, s = i8.untile(i8.quantize(x), rows, k)
    want_q, want_s = R.quantize(x.double())
    assert torch.equal(s, want_s) and torch.equal(q, want_q)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,k,eps", [(1, 64, 1e-5), (2, 63, 0.0), (17, 4096, 1e-5), (33, 130, 1e-6), (4, 16401, 1e-5), (1040, 9000, 1e-5), (2, 33000, 1e-6)])
def test_rms_norm_quantize(i8, rows, k, eps, kind):
    g = _gen(rows + k)
    x, w = _normal(g, rows, k, dtype=kind, std=3.0), 1.0 + 0.3 * _normal(g, k)
    q, s = i8.untile(i8.rms_norm_quantize(x, w, eps), rows, k)
    want_q, want_s = R.quantize(R.rows_of(x, w, eps))
    assert torch.equal(s, want_s) and torch.equal(q, want_q)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 64), (3, 65), (17, 14336), (40, 130), (2, 28672)])
def test_silu_mul_quantize(i8, rows, k, kind):
    g = _gen(rows + k)
    gate, up = _normal(g, rows, k, dtype=kind, std=3.0), _normal(g, rows, k, dtype=kind)
    q, s = i8.untile(i8.silu_mul_quantize(gate, up), rows, k)
    v = gate.double() / (1.0 + torch.exp(-gate.double())) * up.double()
    # v within 3 units (of 2 U) in the last place, so the scale within that and its own rounding, and the whole number one of those next to the quotient
    top = v.abs().amax(dim=1)
    assert ((s.double() - top / 127).abs() <= 8 * R.U * top / 127).all()
    assert ((q.double() * s.double()[:, None] - v).abs() <= s.double()[:, None] * (0.5 + 127 * 16 * R.U)).all()


@pytest.mark.parametrize("kind", TYPES)
def test_rows_apart_and_not_aligned(i8, kind):
    g = _gen(3)
    wide = _normal(g, 40, 301, dtype=kind)
    w = 1.0 + 0.3 * _normal(g, 100)
    for x in (wide[:, :100], wide[:, 1:101], wide[::2, 3:103], wide[:1, 5:105]):
        rows = x.shape[0]
        q, s = i8.untile(i8.quantize(x), rows, 100)
        want_q, want_s = R.quantize(x.double())
        assert torch.equal(s, want_s) and torch.equal(q, want_q)
        q, s = i8.untile(i8.rms_norm_quantize(x, w, 1e-5), rows, 100)
        want_q, want_s = R.quantize(R.rows_of(x, w, 1e-5))
        assert torch.equal(s, want_s) and torch.equal(q, want_q)
        assert torch.equal(i8.untile(i8.silu_mul_quantize(x, x), rows, 100)[0], i8.untile(i8.silu_mul_quantize(x.contiguous(), x.contiguous()), rows, 100)[0])
    one = wide[7]
    q, s = i8.untile(i8.quantize(one), 1, 301)
    want_q, want_s = R.quantize(one[None].double())
    assert torch.equal(s, want_s) and torch.equal(q, want_q)


def test_rows_of_nothing_of_borders_and_of_what_is_not_finite(i8):
    k = 200
    x = torch.zeros(12, k, device="cuda")
    x[1, 3] = float("inf")
    x[2, 199] = float("nan")
    x[3, 0] = -float("inf")
    x[4] = torch.arange(k, device="cuda") * 2.0**-149  # below the normal numbers: scales of a unit or none
    x[5] = torch.arange(k, device="cuda") * 1e-38
    x[6] = 3.4e38
    x[6, ::2] *= -1
    x[7] = torch.arange(k, device="cuda") - 100.0
    x[7, 0] = 127.0  # scale 1: halves are ties, and go to the even side
    x[7, 1:20] = torch.arange(19, device="cuda") - 9.5
    x[8] = 2.0**-149
    x[9] = torch.linspace(-254, 254, k, device="cuda")
    x[10, 0], x[10, 1] = 1e30, 1e-30
    q, s = i8.untile(i8.quantize(x), 12, k)
    want_q, want_s = R.quantize(x.double())
    assert torch.equal(torch.isnan(s), torch.isnan(want_s)) and torch.isnan(s).sum() == 3
    assert torch.equal(s.nan_to_num(), want_s.nan_to_num()) and torch.equal(q, want_q)
    wq, ws = _matrix(_gen(1), 33, k)
    y = i8.gemm(i8.tile(wq, ws), i8.quantize(x), 12, 33, k)
    bad = torch.isnan(s)
    assert torch.isnan(y[bad]).all() and (y[0] == 0).all()
    # (row 6: a sum of some thousands times a scale of 2.7e36 is past fp32, before w's scale is there)
    assert torch.equal(y[~bad], R.product(wq, ws, q[~bad], s[~bad], torch.float32))


def test_rows_below_the_normal_numbers(i8):
    # a scale of few bits: 190 units / 127 is one unit, and values past 127 of it are held there; a scale of none for rows below 64
    units = torch.tensor([190, -190, 128, 127, 126, 64, 63, 1, -1, 0], dtype=torch.float64, device="cuda")
    x = torch.stack([(units * u * 2.0**-149).float() for u in (1, 2, 3, 1000, 2**20, 2**24)] + [(units.clamp(-63, 63) * 2.0**-149).float()])
    q, s = i8.untile(i8.quantize(x), *x.shape)
    want_q, want_s = R.quantize(x.double())
    assert torch.equal(s, want_s) and torch.equal(q, want_q)
    assert q[0, 0] == 127 and q[0, 1] == -127 and s[0] > 0 and s[-1] == 0


def test_quotients_next_to_halves(i8):
    # numbers around (n + 1/2) scales, one unit in the last place apart: the true quotient decides, not a rounded one
    g = _gen(11)
    top = torch.empty(64, 1, device="cuda").uniform_(0.1, 10.0, generator=g)
    scale = (top.double() / 127).float().double()
    half = torch.arange(-126, 126, device="cuda").double() + 0.5
    near = (half[None] * scale).float()
    x = torch.cat([top, near, torch.nextafter(near, torch.full_like(near, 1e9)), torch.nextafter(near, torch.full_like(near, -1e9))], dim=1)
    q, s = i8.untile(i8.quantize(x), *x.shape)
    want_q, want_s = R.quantize(x.double())
    assert torch.equal(s, want_s) and torch.equal(q, want_q)


@pytest.mark.parametrize("rows,k", [(1, 1), (16, 64), (17, 65), (100, 1000)])
def test_tile_and_back(i8, rows, k):
    q, s = _matrix(_gen(rows), rows, k)
    q[0, 0] = -128
    tiled = i8.tile(q, s)
    assert tiled.numel() == i8.tiled_bytes(rows, k)
    back_q, back_s = i8.untile(tiled, rows, k)
    assert torch.equal(back_q, q) and torch.equal(back_s, s)
    # the layout that the header states
    steps = (k + 63) // 64
    strips = (rows + 15) // 16
    fragments = tiled[: strips * steps * 1024].view(torch.int8).view(strips, steps, 4, 16, 16)  # [strip][step][c][r][j]
    plain = fragments.permute(0, 3, 1, 2, 4).reshape(strips * 16, steps * 64)
    assert torch.equal(plain[:rows, :k], q) and (plain[:rows, k:] == 0).all()


# ---- products

SHAPES = [(1, 1, 1), (1, 33, 64), (1, 4096, 4096), (2, 5, 65), (3, 250, 1000), (13, 1003, 8192), (16, 64, 130), (17, 31, 63), (32, 1000, 500), (33, 257, 192), (64, 64, 64), (65, 300, 1030), (117, 515, 4100),
          (128, 512, 320), (200, 130, 257), (256, 256, 256), (300, 33000, 130), (513, 17001, 64), (1001, 5003, 1507), (1030, 8190, 100), (2, 70000, 130), (5000, 3, 66)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm_bit_for_bit(i8, m, n, k, kind):
    g = _gen(m + n + k)
    (wq, ws), (xq, xs) = _matrix(g, n, k), _matrix(g, m, k)
    w, x = i8.tile(wq, ws), i8.tile(xq, xs)
    assert torch.equal(i8.gemm(w, x, m, n, k, dtype=kind), R.product(wq, ws, xq, xs, kind))
    r = _normal(g, m, n, dtype=kind)
    want = R.product(wq, ws, xq, xs, kind, r)
    assert torch.equal(i8.gemm(w, x, m, n, k, dtype=kind, residual=r), want)
    assert i8.gemm(w, x, m, n, k, dtype=kind, residual=r, out=r) is r and torch.equal(r, want)


# (rows that are a little less than 96, 160 and 192, n for several hundred tiles, K of one step to ten)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k", [(90, 20003, 64), (81, 16400, 577), (150, 16400, 130), (157, 20003, 577), (145, 33002, 400), (180, 16400, 60), (190, 20003, 130), (177, 16402, 577), (310, 20001, 200)])
def test_gemm_in_tiles_of_other_heights(i8, m, n, k, kind):
    test_gemm_bit_for_bit(i8, m, n, k, kind)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_sums_up_to_the_last_bit(i8, m):
    # the longest K with the largest values: whole numbers just below 2^31
    n, k = 40, 131008
    wq = torch.full((n, k), -128, device="cuda", dtype=torch.int8)
    xq = torch.full((m, k), -128, device="cuda", dtype=torch.int8)
    wq[1::2] = 127
    ones = torch.ones(max(m, n), device="cuda")
    y = i8.gemm(i8.tile(wq, ones[:n]), i8.tile(xq, ones[:m]), m, n, k)
    assert (y[:, 0::2] == 16384.0 * k).all() and (y[:, 1::2] == -16256.0 * k).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (1, 14336, 4096), (1, 77, 100), (1, 1, 1), (1, 33, 63), (1, 1000, 4097), (1, 500, 16384), (1, 515, 14336), (1, 9000, 8191), (1, 100, 16385), (1, 20, 5000), (2, 1000, 4096), (2, 33, 8191), (2, 9001, 8192), (2, 300, 8193), (3, 1001, 4095), (4, 515, 1507), (4, 9004, 4096), (4, 40, 4097), (5, 64, 64), (13, 8192, 8192), (117, 1000, 512), (600, 13000, 96)])
def test_mul_mat_is_quantize_and_gemm(i8, m, n, k, kind):
    g = _gen(m + n + k)
    wq, ws = _matrix(g, n, k)
    w, x, norm, r = i8.tile(wq, ws), _normal(g, m, k, dtype=kind), 1.0 + 0.2 * _normal(g, k), _normal(g, m, n, dtype=kind)
    for weight, eps in ((None, 0.0), (norm, 1e-5)):
        xq, xs = R.quantize(R.rows_of(x, weight, eps))
        assert torch.equal(i8.mul_mat(w, x, n, k, norm_weight=weight, eps=eps), R.product(wq, ws, xq, xs, kind))
        assert torch.equal(i8.mul_mat(w, x, n, k, residual=r, norm_weight=weight, eps=eps), R.product(wq, ws, xq, xs, kind, r))
    if m == 1:
        assert torch.equal(i8.mul_mat(w, x[0], n, k), i8.mul_mat(w, x, n, k))
    apart = torch.zeros(m, k + 3, device="cuda", dtype=kind)[:, 1 : k + 1].copy_(x)
    assert torch.equal(i8.mul_mat(w, apart, n, k), i8.mul_mat(w, x, n, k))


# ---- losses


def _loss_case(i8, m, n, k, seed=0, spread=1.0):
    g = _gen(seed + m + n + k)
    wq, ws = _matrix(g, n, k)
    ws = ws * 8.0 * spread
    xq, xs = _matrix(g, m, k)
    xs = xs * k**0.5 / 40.0
    targets = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32, generator=g)
    if m > 2:
        targets[1], targets[2] = -1, n
    return wq, ws, xq, xs, targets


LOSSES = [(1, 1, 64), (1, 2, 1), (1, 1000, 64), (2, 33, 65), (3, 4097, 256), (16, 128, 100), (17, 5000, 130), (64, 250, 64), (65, 1003, 200), (130, 257, 64), (300, 2000, 128), (700, 9001, 64), (1, 128256, 512), (16, 6001, 1030), (9, 4099, 2050), (5, 4100, 4096), (4, 515, 3000)]


@pytest.mark.parametrize("m,n,k", LOSSES)
def test_losses(i8, m, n, k):
    wq, ws, xq, xs, targets = _loss_case(i8, m, n, k)
    losses, lse = i8.token_losses(i8.tile(wq, ws), i8.tile(xq, xs), targets, n, k)
    l = R.logits(wq, ws, xq, xs)
    want, want_lse = R.losses(l, targets)
    bound = R.lse_bound(l)
    assert ((lse.double() - want_lse).abs() <= bound).all()
    assert ((losses.double() - want).abs() <= bound + R.logit_bound(l) + 4 * R.U * want.abs()).all()
    if m > 2:
        assert losses[1] == 0 and losses[2] == 0


@pytest.mark.parametrize("m", [2, 70])
def test_losses_of_logits_far_apart_and_of_rows_that_are_not_finite(i8, m):
    n, k = 1500, 128
    wq, ws, xq, xs, targets = _loss_case(i8, m, n, k, spread=60.0)
    xs[0] = float("nan")
    targets[0] = 5
    losses, lse = i8.token_losses(i8.tile(wq, ws), i8.tile(xq, xs), targets, n, k)
    assert torch.isnan(losses[0]) and torch.isnan(lse[0])
    l = R.logits(wq, ws, xq[1:], xs[1:])
    want, want_lse = R.losses(l, targets[1:])
    assert ((lse[1:].double() - want_lse).abs() <= R.lse_bound(l)).all()
    assert ((losses[1:].double() - want).abs() <= R.lse_bound(l) + R.logit_bound(l) + 4 * R.U * want.abs()).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k", LOSSES + [(5, 3000, 4160), (2, 40, 1030)])
def test_gradient(i8, m, n, k, kind):
    wq, ws, xq, xs, targets = _loss_case(i8, m, n, k)
    w, x = i8.tile(wq, ws), i8.tile(xq, xs)
    losses, lse = i8.token_losses(w, x, targets, n, k)
    l = R.logits(wq, ws, xq, xs)
    grad = _normal(_gen(1), m)
    for g in (None, grad):
        dx = i8.token_losses_grad(w, x, targets, losses, lse, n, k, grad=g, dtype=kind)
        off = (dx.double() - R.gradient(l, targets, wq, ws, g)).abs()
        assert (off <= R.gradient_bound(l, targets, wq, ws, kind, g)).all()
    if m > 2:
        assert (dx[1] == 0).all() and (dx[2] == 0).all()


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(90, 16400, 130), (150, 20003, 64), (157, 16400, 330), (180, 16403, 200), (310, 20001, 130)])
def test_losses_and_gradient_in_tiles_of_other_heights(i8, m, n, k, kind):
    test_losses(i8, m, n, k)
    test_gradient(i8, m, n, k, kind)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(700, 130), (1056, 580)])
@pytest.mark.parametrize("m", [17, 32, 33, 49, 66, 81, 97, 113, 129, 145, 177, 209, 241, 257, 310])
def test_gradient_of_rows_in_tiles_of_every_height(i8, m, n, k, kind):
    wq, ws, xq, xs, targets = _loss_case(i8, m, n, k)
    w, x = i8.tile(wq, ws), i8.tile(xq, xs)
    losses, lse = i8.token_losses(w, x, targets, n, k)
    l = R.logits(wq, ws, xq, xs)
    grad = _normal(_gen(m), m)
    dx = i8.token_losses_grad(w, x, targets, losses, lse, n, k, grad=grad, dtype=kind)
    assert ((dx.double() - R.gradient(l, targets, wq, ws, grad)).abs() <= R.gradient_bound(l, targets, wq, ws, kind, grad)).all()


@pytest.mark.parametrize("m,n,k", [(3, 600, 512), (12, 6001, 576), (5, 3000, 4160), (40, 1500, 300), (160, 3008, 1280), (310, 2001, 130)])
def test_gradient_in_fp16_is_off_by_its_rounding_alone(i8, m, n, k):
    # what fp32 is off by, and half a step of the result (2^-11 of a normal number, 2^-25 of the smallest)
    wq, ws, xq, xs, targets = _loss_case(i8, m, n, k)
    w, x = i8.tile(wq, ws), i8.tile(xq, xs)
    losses, lse = i8.token_losses(w, x, targets, n, k)
    l = R.logits(wq, ws, xq, xs)
    dx = i8.token_losses_grad(w, x, targets, losses, lse, n, k, dtype=torch.float16)
    want = R.gradient(l, targets, wq, ws)
    assert ((dx.double() - want).abs() <= R.gradient_bound(l, targets, wq, ws, torch.float32) + want.abs() * 2.0**-11 + 2.0**-25).all()


@pytest.mark.parametrize("m", [3, 80])
def test_gradient_of_rows_that_are_sure_and_of_rows_that_are_not_finite(i8, m):
    n, k = 1100, 256
    wq, ws, xq, xs, targets = _loss_case(i8, m, n, k)
    w, rows = wq.double() * ws.double()[:, None], torch.arange(m, device="cuda")
    targets = targets.clamp(0, n - 1)
    x = torch.randn(m, k, device="cuda", generator=_gen(5)) + w[targets.long()].float() * torch.linspace(0, 40, m, device="cuda")[:, None]
    x[2, 7] = float("nan")
    tiled = i8.quantize(x)
    xq, xs = i8.untile(tiled, m, k)
    wt = i8.tile(wq, ws)
    losses, lse = i8.token_losses(wt, tiled, targets, n, k)
    dx = i8.token_losses_grad(wt, tiled, targets, losses, lse, n, k)
    assert torch.isnan(dx[2]).all()
    keep = rows[rows != 2]
    l = R.logits(wq, ws, xq[keep], xs[keep])
    assert ((dx[keep].double() - R.gradient(l, targets[keep], wq, ws)).abs() <= R.gradient_bound(l, targets[keep], wq, ws, torch.float32)).all()
    targets[2] = -1  # not scored: nothing of it
    losses, lse = i8.token_losses(wt, tiled, targets, n, k)
    assert losses[2] == 0 and (i8.token_losses_grad(wt, tiled, targets, losses, lse, n, k)[2] == 0).all()


def test_gradient_against_differences(i8):
    # the loss of the rows that x stands for, in 64 bits, along random directions
    m, n, k, h = 4, 300, 96, 1e-5
    wq, ws, xq, xs, targets = _loss_case(i8, m, n, k)
    grad = torch.rand(m, device="cuda", generator=_gen(2))
    w, x = i8.tile(wq, ws), i8.tile(xq, xs)
    losses, lse = i8.token_losses(w, x, targets, n, k)
    dx = i8.token_losses_grad(w, x, targets, losses, lse, n, k, grad=grad).double()
    rows, weights = xq.double() * xs.double()[:, None], wq.double() * ws.double()[:, None]

    def value(r):
        return (R.losses(r @ weights.t(), targets)[0] * grad.double()).sum()

    l = R.logits(wq, ws, xq, xs)
    bound = R.gradient_bound(l, targets, wq, ws, torch.float32, grad)
    for seed in range(5):
        v = torch.randn(m, k, device="cuda", dtype=torch.float64, generator=_gen(seed))
        slope = (value(rows + h * v) - value(rows - h * v)) / (2 * h)
        # the difference itself: third derivatives of a loss are below 8 |w v|^3, and a 64-bit value of some 10 has 2e-15
        wide = (v @ weights.t()).abs().amax()
        assert (slope - (dx * v).sum()).abs() <= (bound * v.abs()).sum() + m * 8 * wide**3 * h * h / 6 + 4e-15 * 10 * m / h


def test_pieces_of_the_vocabulary_and_splits(i8):
    # rows so many that the vocabulary goes in several pieces (2 ^ 27 / (4 bytes 8192 rows): 4096 tokens each)
    m, n, k = 8192, 9000, 64
    wq, ws, xq, xs, targets = _loss_case(i8, m, n, k)
    w, x = i8.tile(wq, ws), i8.tile(xq, xs)
    losses, lse = i8.token_losses(w, x, targets, n, k)
    dx = i8.token_losses_grad(w, x, targets, losses, lse, n, k)
    some = torch.arange(0, m, 37, device="cuda")
    l = R.logits(wq, ws, xq[some], xs[some])
    assert ((losses[some].double() - R.losses(l, targets[some])[0]).abs() <= R.lse_bound(l) + R.logit_bound(l) + 4 * R.U * 30).all()
    assert ((dx[some].double() - R.gradient(l, targets[some], wq, ws)).abs() <= R.gradient_bound(l, targets[some], wq, ws, torch.float32)).all()


@pytest.mark.parametrize("m,n,k", [(8200, 600, 64), (16500, 40, 130), (9001, 130000, 64)])
def test_rows_so_many_that_they_go_in_parts(i8, m, n, k):
    wq, ws, xq, xs, targets = _loss_case(i8, m, n, k)
    w, x = i8.tile(wq, ws), i8.tile(xq, xs)
    losses, lse = i8.token_losses(w, x, targets, n, k)
    grad = torch.rand(m, device="cuda", generator=_gen(3))
    dx = i8.token_losses_grad(w, x, targets, losses, lse, n, k, grad=grad, dtype=torch.bfloat16)
    some = torch.cat([torch.arange(0, m, 211, device="cuda"), torch.arange(8180, 8200, device="cuda"), torch.arange(m - 10, m, device="cuda")])
    l = R.logits(wq, ws, xq[some], xs[some])
    want, want_lse = R.losses(l, targets[some])
    assert ((lse[some].double() - want_lse).abs() <= R.lse_bound(l)).all()
    assert ((losses[some].double() - want).abs() <= R.lse_bound(l) + R.logit_bound(l) + 4 * R.U * want.abs()).all()
    assert ((dx[some].double() - R.gradient(l, targets[some], wq, ws, grad[some])).abs() <= R.gradient_bound(l, targets[some], wq, ws, torch.bfloat16, grad[some])).all()


# ---- as they are used


def test_a_feed_forward_part_and_the_loss_behind_it(i8):
    m, k, ff, vocab, eps = 37, 512, 1400, 3001, 1e-5
    g = _gen(9)
    gate, up, down, head = (i8.quantize(_normal(g, n, kk, std=kk**-0.5)) for n, kk in ((ff, k), (ff, k), (k, ff), (vocab, k)))
    x, norm = _normal(g, m, k), 1.0 + 0.1 * _normal(g, k)
    targets = torch.randint(0, vocab, (m,), device="cuda", dtype=torch.int32, generator=g)

    def step():
        h = i8.rms_norm_quantize(x, norm, eps)
        a, b = i8.gemm(gate, h, m, ff, k, dtype=torch.bfloat16), i8.gemm(up, h, m, ff, k, dtype=torch.bfloat16)
        y = i8.gemm(down, i8.silu_mul_quantize(a, b), m, k, ff, residual=x)
        rows = i8.rms_norm_quantize(y, norm, eps)
        losses, lse = i8.token_losses(head, rows, targets, vocab, k)
        return a, b, y, losses, lse, i8.token_losses_grad(head, rows, targets, losses, lse, vocab, k, dtype=torch.float16)

    a, b, y, losses, lse, dx = step()
    (gq, gs), (dq, ds), (hq, hs) = i8.untile(gate, ff, k), i8.untile(down, k, ff), i8.untile(head, vocab, k)
    assert torch.equal(a, R.product(gq, gs, *R.quantize(R.rows_of(x, norm, eps)), torch.bfloat16))
    mid = i8.untile(i8.silu_mul_quantize(a, b), m, ff)
    assert torch.equal(y, R.product(dq, ds, *mid, torch.float32, x))
    rows = R.quantize(R.rows_of(y, norm, eps))
    l = R.logits(hq, hs, *rows)
    assert ((losses.double() - R.losses(l, targets)[0]).abs() <= R.lse_bound(l) + R.logit_bound(l) + 4 * R.U * 30).all()
    assert ((dx.double() - R.gradient(l, targets, hq, hs)).abs() <= R.gradient_bound(l, targets, hq, hs, torch.float16)).all()

    # captured, and replayed among the program's own calls
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
    torch.cuda.current_stream().wait_stream(stream)
    for seed in range(4):
        x.copy_(_normal(_gen(100 + seed), m, k))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


def test_two_streams_at_once(i8):
    g = _gen(4)
    m, n, k = 70, 3000, 512
    w = i8.tile(*_matrix(g, n, k))
    xs = [_normal(g, m, k) for _ in range(2)]
    targets = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32, generator=g)

    def step(x):
        q = i8.quantize(x)
        losses, lse = i8.token_losses(w, q, targets, n, k)
        return i8.mul_mat(w, x, n, k), losses, i8.token_losses_grad(w, q, targets, losses, lse, n, k)

    alone = [step(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(step(x))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_what_is_behind_results_and_workspaces_is_left_alone(i8):
    m, n, k = 5, 50, 70
    g = _gen(6)
    w, x = i8.tile(*_matrix(g, n, k)), _normal(g, m, k)
    for need, call in ((i8._need("nh_i8_mul_mat_workspace_bytes", m, k), lambda ws: i8.mul_mat(w, x, n, k, workspace=ws)),):
        memory = torch.full((need + 512,), 77, device="cuda", dtype=torch.uint8)
        assert torch.equal(call(memory[:need]), call(None)) and (memory[need:] == 77).all()
    held = torch.full((m + 2, n), 3.0, device="cuda")
    i8.mul_mat(w, x, n, k, out=held[:m])
    assert (held[-1] == 3).all()
    targets = torch.zeros(m, device="cuda", dtype=torch.int32)
    xq = i8.quantize(x)
    losses, lse = i8.token_losses(w, xq, targets, n, k)
    need = i8._need("nh_i8_token_losses_grad_workspace_bytes", m, n, k, 0)
    memory = torch.full((need + 512,), 77, device="cuda", dtype=torch.uint8)
    assert torch.equal(i8.token_losses_grad(w, xq, targets, losses, lse, n, k, workspace=memory[:need]), i8.token_losses_grad(w, xq, targets, losses, lse, n, k))
    assert (memory[need:] == 77).all()


def test_weights_from_q8_0(i8, q8):
    n, k = 96, 256
    blocks = q8.fill_weight_blocks(1, n, k)
    tiled = q8.tile(blocks, n, k)
    values = q8.get_rows(tiled, torch.arange(n, dtype=torch.int32, device="cuda"), n, k, tiled=True)
    q, s = i8.untile(i8.from_q8_0(tiled, n, k), n, k)
    want_q, want_s = R.quantize(values.double())
    assert torch.equal(q, want_q) and torch.equal(s, want_s)


def test_the_native_calls_and_the_python_way(i8, monkeypatch):
    assert i8._calls is not None
    g = _gen(8)
    m, n, k = 6, 90, 200
    w, norm, r = i8.tile(*_matrix(g, n, k)), 1.0 + 0.1 * _normal(g, k), _normal(g, m, n, dtype=torch.float16)
    wide = _normal(g, m, k + 7, dtype=torch.float16)
    x = wide[:, 3 : k + 3]
    targets, grad = torch.randint(0, n, (m,), device="cuda", dtype=torch.int32, generator=g), _normal(g, m)

    def both(call):
        out = []
        for native in (i8._calls, None):
            monkeypatch.setattr(i8, "_calls", native)
            try:
                out.append(call())
            except Exception as e:  # noqa: BLE001
                out.append((type(e), str(e)))
        monkeypatch.undo()
        return out

    xq = i8.quantize(x)
    losses, lse = i8.token_losses(w, xq, targets, n, k)
    for call in (lambda: i8.untile(i8.quantize(x), m, k), lambda: i8.untile(i8.quantize(x[0]), 1, k), lambda: i8.untile(i8.rms_norm_quantize(x, norm, 1e-5), m, k), lambda: i8.untile(i8.silu_mul_quantize(x, x), m, k),
                 lambda: (i8.gemm(w, xq, m, n, k, dtype=torch.bfloat16), i8.gemm(w, xq, m, n, k, dtype=torch.float16, residual=r)), lambda: (i8.mul_mat(w, x, n, k, residual=r), i8.mul_mat(w, x[:1], n, k, norm_weight=norm, eps=1e-5)),
                 lambda: i8.token_losses(w, xq, targets, n, k), lambda: (i8.token_losses_grad(w, xq, targets, losses, lse, n, k, grad=grad), i8.token_losses_grad(w, xq, targets, losses, lse, n, k, dtype=torch.float16))):
        native, python = both(call)
        assert all(torch.equal(a, b) for a, b in zip(native, python))
    for call in (lambda: i8.quantize(x.t()), lambda: i8.quantize(x.double()), lambda: i8.quantize(x.expand(3, m, k)), lambda: i8.quantize(x[:1].expand(3, k)), lambda: i8.rms_norm_quantize(x, norm[1:], 1e-5),
                 lambda: i8.rms_norm_quantize(x, norm, -1.0), lambda: i8.silu_mul_quantize(x, x[1:]), lambda: i8.silu_mul_quantize(x, x.float()), lambda: i8.gemm(w[:-1], xq, m, n, k), lambda: i8.gemm(w, xq, m + 16, n, k),
                 lambda: i8.gemm(w, xq, m, n, k, dtype=torch.float64), lambda: i8.gemm(w, xq, m, n, k, residual=r), lambda: i8.gemm(w, xq, m, n, 0), lambda: i8.mul_mat(w, x, n, k - 1), lambda: i8.mul_mat(w, x, n + 16, k),
                 lambda: i8.mul_mat(w, x, n, k, residual=r[1:]), lambda: i8.token_losses(w, xq, targets.long(), n, k), lambda: i8.token_losses(w, xq, targets[None], n, k), lambda: i8.token_losses(w, xq[64:], targets, n, k),
                 lambda: i8.token_losses_grad(w, xq, targets, losses[1:], lse, n, k), lambda: i8.token_losses_grad(w, xq, targets, losses, lse, n, k, grad=grad.double()),
                 lambda: i8.token_losses_grad(w, xq, targets, losses, lse, n, k, dtype=torch.int32)):
        native, python = both(call)
        assert isinstance(native, tuple) and issubclass(native[0], Exception) and native == python, native


def test_empty_calls(i8):
    w = i8.tile(*_matrix(_gen(1), 32, 64))
    x = torch.empty(0, 64, device="cuda")
    assert i8.mul_mat(w, x, 32, 64).shape == (0, 32)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    losses, lse = i8.token_losses(w, i8.quantize(x), none, 32, 64)
    assert losses.numel() == 0 and i8.token_losses_grad(w, i8.quantize(x), none, losses, lse, 32, 64).shape == (0, 64)
    assert i8.mul_mat(i8.tile(torch.empty(0, 64, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda")), torch.ones(3, 64, device="cuda"), 0, 64).shape == (3, 0)
