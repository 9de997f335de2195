"""CPU: the calls on int8 matrices with a scale per row: every declared function is exported and bound, sizes, and the calls that end before any device work."""
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000  # a pointer that nothing follows
Q = [P << (4 * i) for i in range(8)]  # ... and others far from it


@pytest.fixture(scope="module")
def lib():
    from nihilus_amd import _lib

    return _lib.lib()


def test_every_declared_function_is_exported_and_bound(lib):
    from nihilus_amd import _lib

    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "nihilus_amd", "i8_abi.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(nh_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(_lib.I8_SIGNATURES) and all(hasattr(lib, n) for n in names)


@pytest.mark.parametrize("rows,k", [(0, 1), (1, 1), (1, 16385), (2, 8192), (2, 8193), (3, 4096), (4, 4097), (5, 64), (16, 64), (17, 65), (128256, 4096), (4096, 14336)])
def test_bytes_of_a_tiled_matrix(lib, rows, k):
    strips = (rows + 15) // 16
    assert lib.nh_i8_tiled_bytes(rows, k) == strips * ((k + 63) // 64 * 1024 + 64)
    # (one row of up to 16384 values is quantized inside the product)
    assert lib.nh_i8_mul_mat_workspace_bytes(rows, k) == (0 if rows == 1 and k <= 16384 else lib.nh_i8_tiled_bytes(rows, k))


def test_sizes_that_are_refused(lib):
    assert lib.nh_i8_tiled_bytes(-1, 64) == -3 and lib.nh_i8_tiled_bytes(1, 0) == -3 and lib.nh_i8_tiled_bytes(1, -5) == -3
    assert lib.nh_i8_tiled_bytes((1 << 22) + 1, 64) == -5 and lib.nh_i8_tiled_bytes(1, 131009) == -5 and lib.nh_i8_tiled_bytes(1 << 22, 131008) == -5
    assert lib.nh_i8_token_losses_workspace_bytes(1 << 22, 1 << 22, 64) == -5 and lib.nh_i8_token_losses_workspace_bytes(-1, 4, 64) == -3
    assert lib.nh_i8_token_losses_grad_workspace_bytes(4, 4, 64, 3) == -6 and lib.nh_i8_token_losses_grad_workspace_bytes(4, 4, 0, 0) == -3
    assert lib.nh_i8_token_losses_grad_workspace_bytes(0, 4, 64, 0) == 0


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (5, 128256, 4096), (2048, 128256, 4096), (65, 1000, 64), (100000, 128256, 4096), (1 << 20, 1000, 64), (1, 1 << 22, 64)])
def test_a_workspace_holds_no_logits(lib, m, n, k):
    # stretches of 64 MiB; slopes of 128 MiB, or of 1024 tokens for 8192 rows, and sums of at most 256 tiles of 512 x 128, or one set for 8192 rows
    for kind, terms in ((0, 2), (1, 1), (2, 1)):
        need = lib.nh_i8_token_losses_grad_workspace_bytes(m, n, k, kind)
        rows = min((m + 15) // 16 * 16, 8192)
        assert 0 < need <= max(1 << 27, rows * 2048 * terms) + max(256 * 512 * 128 * 4, rows * (k + 64) * 4) + 4096
    assert lib.nh_i8_token_losses_workspace_bytes(m, n, k) <= (1 << 26) + 4 * min(m, 1 << 21) + 4096


def _calls(lib):
    """name -> (function, good arguments, which are pointers)"""
    a, b, c, d, e, f, g, _ = Q
    return {
        "quantize": (lib.nh_i8_quantize, [a, 0, 64, b, 2, 64, None], [0, 3]),
        "norm": (lib.nh_i8_rms_norm_quantize, [a, 0, 64, c, 1e-5, b, 2, 64, None], [0, 3, 5]),
        "silu": (lib.nh_i8_silu_mul_quantize, [a, c, 0, 64, 64, b, 2, 64, None], [0, 1, 5]),
        "tile": (lib.nh_i8_tile, [a, c, b, 2, 64, None], [0, 1, 2]),
        "untile": (lib.nh_i8_untile, [b, a, c, 2, 64, None], [0, 1, 2]),
        "gemm": (lib.nh_i8_gemm, [a, c, None, b, 0, 2, 32, 64, None], [0, 1, 3]),
        "mul_mat": (lib.nh_i8_mul_mat, [a, c, 0, 64, None, 0.0, None, b, 5, 32, 64, d, 1 << 20, None], [0, 1, 7, 11]),
        "losses": (lib.nh_i8_token_losses, [a, b, c, d, e, 2, 32, 64, f, 1 << 20, None], [0, 1, 2, 3, 4, 8]),
        "grad": (lib.nh_i8_token_losses_grad, [a, b, c, d, e, None, f, 0, 2, 32, 64, g, 1 << 30, None], [0, 1, 2, 3, 4, 6, 11]),
    }


NAMES = ["quantize", "norm", "silu", "tile", "untile", "gemm", "mul_mat", "losses", "grad"]


def _call(lib, name, **over):
    fn, args, _ = _calls(lib)[name]
    args = list(args)
    for i, v in over.items():
        args[int(i[1:])] = v
    return fn(*args)


@pytest.mark.parametrize("name", NAMES)
def test_a_pointer_that_is_not_there(lib, name):
    for i in _calls(lib)[name][2]:
        assert _call(lib, name, **{f"a{i}": None}) == -1, i


@pytest.mark.parametrize("name,at", [("quantize", 0), ("quantize", 3), ("norm", 3), ("norm", 5), ("silu", 1), ("silu", 5), ("tile", 1), ("tile", 2), ("untile", 0), ("gemm", 0), ("gemm", 1), ("gemm", 2), ("gemm", 3),
                                     ("mul_mat", 0), ("mul_mat", 1), ("mul_mat", 4), ("mul_mat", 6), ("mul_mat", 7), ("mul_mat", 11), ("losses", 1), ("losses", 2), ("losses", 3), ("losses", 8), ("grad", 5), ("grad", 6), ("grad", 11)])
def test_a_pointer_that_is_not_aligned(lib, name, at):
    assert _call(lib, name, **{f"a{at}": Q[7] + 2}) == -2


# (rows, k) of the quantizers, (M, N, K) of the products
SIZES = {"quantize": (4, 5), "norm": (6, 7), "silu": (6, 7), "tile": (3, 4), "untile": (3, 4), "gemm": (5, 6, 7), "mul_mat": (8, 9, 10), "losses": (5, 6, 7), "grad": (8, 9, 10)}


@pytest.mark.parametrize("name", NAMES)
def test_shapes(lib, name):
    at = SIZES[name]
    stride = {"quantize": ["a2"], "norm": ["a2"], "silu": ["a3", "a4"], "mul_mat": ["a3"]}.get(name, [])
    wide = {s: 1 << 20 for s in stride}
    for i in at[:-1]:
        assert _call(lib, name, **{f"a{i}": -1}) == -3
        assert _call(lib, name, **{f"a{i}": (1 << 22) + 1}) == -5
    for bad, code in ((0, -3), (-64, -3), (131009, -5)):
        assert _call(lib, name, **{f"a{at[-1]}": bad}, **wide) == code
    for s in stride:
        assert _call(lib, name, **{s: 63}) == -3 and _call(lib, name, **{s: 1 << 41}) == -5
    assert _call(lib, name, **{f"a{at[0]}": 0}) == 0  # nothing to do
    if len(at) == 3:
        assert _call(lib, name, **{f"a{at[0]}": 1 << 22, f"a{at[1]}": 1 << 22}) == -5
        assert _call(lib, name, **{f"a{at[1]}": 0}) == (0 if name in ("gemm", "mul_mat") else -3)


def test_types_and_eps(lib):
    for name, at in (("quantize", 1), ("norm", 1), ("silu", 2), ("gemm", 4), ("mul_mat", 2), ("grad", 7)):
        for bad in (-1, 3):
            assert _call(lib, name, **{f"a{at}": bad}) == -6
    for name, at in (("norm", 4), ("mul_mat", 5)):
        for bad in (-1e-5, float("inf"), float("nan")):
            assert _call(lib, name, **{f"a{at}": bad}) == -6


def test_a_workspace_that_is_too_small(lib):
    assert _call(lib, "mul_mat", a12=lib.nh_i8_mul_mat_workspace_bytes(5, 64) - 1) == -6
    assert _call(lib, "losses", a9=lib.nh_i8_token_losses_workspace_bytes(2, 32, 64) - 1) == -6
    assert _call(lib, "grad", a12=lib.nh_i8_token_losses_grad_workspace_bytes(2, 32, 64, 0) - 1) == -6


# name -> which arguments are written, which are read
USES = {"quantize": ([3], [0]), "norm": ([5], [0, 3]), "silu": ([5], [0, 1]), "tile": ([2], [0, 1]), "untile": ([1, 2], [0]), "gemm": ([3], [0, 1]), "mul_mat": ([7, 11], [0, 1]), "losses": ([3, 4, 8], [0, 1, 2]),
        "grad": ([6, 11], [0, 1, 2, 3, 4])}


@pytest.mark.parametrize("name", NAMES)
def test_results_over_what_is_read_or_over_each_other(lib, name):
    args, (written, read) = _calls(lib)[name][1], USES[name]
    for i, w in enumerate(written):
        for other in read + written[:i]:
            assert _call(lib, name, **{f"a{w}": args[other]}) == -6, (w, other)
    if name in ("gemm", "mul_mat"):  # the residual: the result itself, or apart from it
        at, y = (2, 3) if name == "gemm" else (6, 7)
        assert _call(lib, name, **{f"a{at}": args[y] + 16}) == -6 and _call(lib, name, **{f"a{at}": args[y] - 16}) == -6
    if name == "mul_mat":
        assert _call(lib, name, a6=args[11]) == -6 and _call(lib, name, a4=args[7]) == -6


@pytest.mark.skipif(torch.cuda.is_available(), reason="would run")
@pytest.mark.parametrize("name", NAMES)
def test_good_calls_want_a_device(lib, name):
    assert _call(lib, name) == -4


def test_tensors_that_the_wrappers_refuse():
    from nihilus_amd import i8

    x = torch.zeros(2, 64)
    for call in (lambda: i8.quantize(x), lambda: i8.rms_norm_quantize(x, x[0], 0.0), lambda: i8.silu_mul_quantize(x, x), lambda: i8.tile(x.to(torch.int8), x[:, 0]), lambda: i8.untile(x, 2, 64),
                 lambda: i8.gemm(x, x, 2, 2, 64), lambda: i8.mul_mat(x, x, 2, 64), lambda: i8.token_losses(x, x, x, 2, 64), lambda: i8.token_losses_grad(x, x, x, x, x, 2, 64)):
        with pytest.raises(TypeError):
            call()
