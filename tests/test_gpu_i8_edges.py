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
