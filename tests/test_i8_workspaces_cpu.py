"""CPU: workspaces of the calls on int8 matrices with a scale per row are aligned as every pointer there, to 16 bytes."""
import pytest

P = 1 << 32
Q = [P + (i << 34) for i in range(8)]  # pointers that nothing follows, far from each other


@pytest.fixture(scope="module")
def lib():
    from nihilus_amd import _lib

    return _lib.lib()


def _calls(lib, workspace, rows=5):
    a, b, c, d, e, f, _, _ = Q
    return [lib.nh_i8_mul_mat(a, c, 0, 64, None, 0.0, None, b, rows, 32, 64, workspace, 1 << 24, None), lib.nh_i8_token_losses(a, b, c, d, e, rows, 32, 64, workspace, 1 << 24, None),
            lib.nh_i8_token_losses_grad(a, b, c, d, e, None, f, 0, rows, 32, 64, workspace, 1 << 24, None)]


@pytest.mark.parametrize("by", [1, 4, 8, 24])
def test_less_than_16_bytes_is_refused(lib, by):
    assert _calls(lib, Q[7] + by) == [-2] * 3


@pytest.mark.parametrize("by", [16, 48, 240])
def test_multiples_of_16_bytes_are_not(lib, by):
    import torch

    if torch.cuda.is_available():
        pytest.skip("would run")
    assert _calls(lib, Q[7] + by) == [-4] * 3  # no device: the check behind the others
