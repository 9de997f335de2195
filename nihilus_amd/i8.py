"""Products in 8-bit integers with one scale for each row of either operand (each token, each output channel), and the softmax cross entropy of a vocabulary
projection with its gradient, for callers that hold torch tensors.

torch is used for device memory and streams only; every operation is calls through the C ABI (``include/nihilus_amd/i8_abi.h``, which says what each one
computes), on the current stream of the tensors' device.  Names follow q8_0.py, whose weights have a scale for each 32 values: more exact, and a fifth of the rate where a prompt's rows are many.

A tiled matrix is a ``torch.uint8`` tensor of ``tiled_bytes(rows, k)``, for weights and activations alike: quantize() makes one of either.
"""
from __future__ import annotations

import torch

from . import _lib
from .attention import _TYPES, _call, _own_memory
from .q8_0 import _calls, _holds, _native


def tiled_bytes(rows: int, k: int) -> int:
    n = _lib.lib().nh_i8_tiled_bytes(rows, k)
    _lib.check("nh_i8_tiled_bytes", n if n < 0 else 0)
    return n


def _x(t: torch.Tensor, name: str) -> tuple[torch.Tensor, int]:
    """[rows, k] of fp32, fp16 or bf16 (a vector is one row), values of a row side by side, and the elements from one row to the next."""
    if not t.is_cuda or t.dtype not in _TYPES:
        raise TypeError(f"{name} must be a float32, float16 or bfloat16 tensor on the GPU")
    if t.dim() not in (1, 2):
        raise ValueError(f"{name} must be [rows, k] or [k]")
    if t.dim() == 1:
        t = t[None]
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the values of a row must lie side by side")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{name}: rows must not overlap")
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _plain(t: torch.Tensor, dtype: torch.dtype, device: torch.device, shape, name: str) -> torch.Tensor:
    if t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous {dtype} tensor on the operands' GPU")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    return t


def _tiled(t: torch.Tensor, device: torch.device, rows: int, k: int, name: str) -> torch.Tensor:
    if t.dtype != torch.uint8 or t.device != device:
        raise TypeError(f"{name} must be a uint8 tensor on the operands' GPU")
    _holds(t, tiled_bytes(rows, k), name)
    return t


def _bytes(n: int, device: torch.device) -> torch.Tensor:
    return torch.empty(n, dtype=torch.uint8, device=device)


def _need(fn: str, *sizes) -> int:
    n = getattr(_lib.lib(), fn)(*sizes)
    _lib.check(fn, n if n < 0 else 0)
    return n


def _workspace(workspace: torch.Tensor | None, n: int, device: torch.device) -> tuple[torch.Tensor | None, int | None, int]:
    if n == 0 and workspace is None:
        return None, None, 0
    if workspace is None:
        _own_memory(n, device)
        workspace = _bytes(n, device)
    elif workspace.dtype != torch.uint8 or workspace.device != device or not workspace.is_contiguous():
        raise TypeError("workspace must be a contiguous uint8 tensor on the operands' GPU")
    return workspace, workspace.data_ptr(), workspace.numel()


def quantize(x: torch.Tensor) -> torch.Tensor:
    """x [rows, k] (or [k]) of fp32, fp16 or bf16, rows apart by any stride -> a tiled matrix with a scale of max |x| / 127 for each row."""
    if _calls is not None:
        r = _native(_calls.i8_quantize(x), "nh_i8_quantize")
        if r is not None:
            return r
    x, stride = _x(x, "x")
    out = _bytes(tiled_bytes(*x.shape), x.device)
    _call("nh_i8_quantize", x.device, x.data_ptr(), _TYPES[x.dtype], stride, out.data_ptr(), *x.shape)
    return out


def rms_norm_quantize(x: torch.Tensor, norm_weight: torch.Tensor, eps: float) -> torch.Tensor:
    """quantize((x * 1/rms(x)) * norm_weight), one kernel; norm_weight fp32 [k]."""
    if _calls is not None:
        r = _native(_calls.i8_rms_norm_quantize(x, norm_weight, eps), "nh_i8_rms_norm_quantize")
        if r is not None:
            return r
    x, stride = _x(x, "x")
    _plain(norm_weight, torch.float32, x.device, x.shape[1:], "norm_weight")
    out = _bytes(tiled_bytes(*x.shape), x.device)
    _call("nh_i8_rms_norm_quantize", x.device, x.data_ptr(), _TYPES[x.dtype], stride, norm_weight.data_ptr(), eps, out.data_ptr(), *x.shape)
    return out


def silu_mul_quantize(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """quantize(silu(gate) * up), one kernel."""
    if _calls is not None:
        r = _native(_calls.i8_silu_mul_quantize(gate, up), "nh_i8_silu_mul_quantize")
        if r is not None:
            return r
    (gate, gate_stride), (up, up_stride) = _x(gate, "gate"), _x(up, "up")
    if gate.dtype != up.dtype or gate.device != up.device:
        raise TypeError("gate and up must be of the same type, on the same GPU")
    if gate.shape != up.shape:
        raise ValueError("gate and up must have the same shape")
    out = _bytes(tiled_bytes(*gate.shape), gate.device)
    _call("nh_i8_silu_mul_quantize", gate.device, gate.data_ptr(), up.data_ptr(), _TYPES[gate.dtype], gate_stride, up_stride, out.data_ptr(), *gate.shape)
    return out


def tile(q: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """int8 [rows, k] with scales fp32 [rows] -> tiled."""
    if not q.is_cuda or q.dim() != 2:
        raise TypeError("q must be an int8 matrix on the GPU")
    rows, k = _plain(q, torch.int8, q.device, q.shape, "q").shape
    _plain(scales, torch.float32, q.device, (rows,), "scales")
    out = _bytes(tiled_bytes(rows, k), q.device)
    _call("nh_i8_tile", q.device, q.data_ptr(), scales.data_ptr(), out.data_ptr(), rows, k)
    return out


def untile(tiled: torch.Tensor, rows: int, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """tiled -> (int8 [rows, k], scales fp32 [rows])."""
    if not tiled.is_cuda:
        raise TypeError("tiled must be a uint8 tensor on the GPU")
    _tiled(tiled, tiled.device, rows, k, "tiled")
    q = torch.empty((rows, k), dtype=torch.int8, device=tiled.device)
    scales = torch.empty(rows, dtype=torch.float32, device=tiled.device)
    _call("nh_i8_untile", tiled.device, tiled.data_ptr(), q.data_ptr(), scales.data_ptr(), rows, k)
    return q, scales


def _gemm(w, xq, m, n, k, kind, residual, out):
    if residual is not None:
        _plain(residual, kind, w.device, (m, n), "residual")
    if out is None:
        return torch.empty((m, n), dtype=kind, device=w.device)
    return _plain(out, kind, w.device, (m, n), "out")


def gemm(w: torch.Tensor, xq: torch.Tensor, m: int, n: int, k: int, dtype: torch.dtype = torch.float32, residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Tiled activations [m, k] x tiled weight [n, k] (+ residual [m, n]) -> [m, n] of `dtype` (out may be the residual tensor itself: in-place accumulate)."""
    if out is None and _calls is not None:
        r = _native(_calls.i8_gemm(w, xq, m, n, k, _TYPES.get(dtype), residual), "nh_i8_gemm")
        if r is not None:
            return r
    if not w.is_cuda or dtype not in _TYPES:
        raise TypeError("w must be a uint8 tensor on the GPU, dtype float32, float16 or bfloat16")
    _tiled(w, w.device, n, k, "w")
    _tiled(xq, w.device, m, k, "xq")
    out = _gemm(w, xq, m, n, k, dtype, residual, out)
    _call("nh_i8_gemm", w.device, w.data_ptr(), xq.data_ptr(), None if residual is None else residual.data_ptr(), out.data_ptr(), _TYPES[dtype], m, n, k)
    return out


def mul_mat(w: torch.Tensor, x: torch.Tensor, n: int, k: int, residual: torch.Tensor | None = None, norm_weight: torch.Tensor | None = None, eps: float = 0.0,
            out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Activations [m, k] (or [k]) x tiled weight [n, k] -> [m, n] of x's type: quantize (behind the RMS norm, with norm_weight), product, + residual [m, n] if given.

    workspace: nh_i8_mul_mat_workspace_bytes(m, k) bytes; without one the call has its own."""
    if out is None and workspace is None and _calls is not None:
        r = _native(_calls.i8_mul_mat(w, x, n, k, residual, norm_weight, eps), "nh_i8_mul_mat")
        if r is not None:
            return r
    x, stride = _x(x, "x")
    m = x.shape[0]
    if x.shape[1] != k:
        raise ValueError(f"x must be [rows, {k}]")
    _tiled(w, x.device, n, k, "w")
    if norm_weight is not None:
        _plain(norm_weight, torch.float32, x.device, (k,), "norm_weight")
    out = _gemm(x, x, m, n, k, x.dtype, residual, out)
    workspace, ws, ws_bytes = _workspace(workspace, _need("nh_i8_mul_mat_workspace_bytes", m, k), x.device)
    _call("nh_i8_mul_mat", x.device, w.data_ptr(), x.data_ptr(), _TYPES[x.dtype], stride, None if norm_weight is None else norm_weight.data_ptr(), eps,
          None if residual is None else residual.data_ptr(), out.data_ptr(), m, n, k, ws, ws_bytes)
    return out


def token_losses(w: torch.Tensor, xq: torch.Tensor, targets: torch.Tensor, n: int, k: int, workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Softmax cross entropy of tiled rows [m, k] on a tiled projection [n, k]: (losses, lse), fp32 [m]; targets int32 [m], rows with a target outside [0, n) are not
    scored: their loss is 0.  lse is the log of the sum of the exponentials; the log-probability of a row's target is -loss.

    workspace: nh_i8_token_losses_workspace_bytes(m, n, k) bytes; without one the call has its own."""
    if workspace is None and _calls is not None:
        r = _native(_calls.i8_token_losses(w, xq, targets, n, k), "nh_i8_token_losses")
        if r is not None:
            return r
    if not w.is_cuda:
        raise TypeError("w must be a uint8 tensor on the GPU")
    m = targets.numel()
    _plain(targets, torch.int32, w.device, (m,), "targets")
    _tiled(w, w.device, n, k, "w")
    _tiled(xq, w.device, m, k, "xq")
    losses, lse = (torch.empty(m, dtype=torch.float32, device=w.device) for _ in range(2))
    workspace, ws, ws_bytes = _workspace(workspace, _need("nh_i8_token_losses_workspace_bytes", m, n, k), w.device)
    _call("nh_i8_token_losses", w.device, w.data_ptr(), xq.data_ptr(), targets.data_ptr(), losses.data_ptr(), lse.data_ptr(), m, n, k, ws, ws_bytes)
    return losses, lse


def token_losses_grad(w: torch.Tensor, xq: torch.Tensor, targets: torch.Tensor, losses: torch.Tensor, lse: torch.Tensor, n: int, k: int, grad: torch.Tensor | None = None,
                      dtype: torch.dtype = torch.float32, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of (grad * losses).sum() with respect to the rows that xq stands for, [m, k] of `dtype`; losses and lse as token_losses gave them, grad fp32 [m] (ones if not given).

    A quantizer in front passes it on as it is (straight through).  workspace: nh_i8_token_losses_grad_workspace_bytes(m, n, k, type) bytes; without one the call has its own."""
    if workspace is None and _calls is not None:
        r = _native(_calls.i8_token_losses_grad(w, xq, targets, losses, lse, n, k, grad, _TYPES.get(dtype)), "nh_i8_token_losses_grad")
        if r is not None:
            return r
    if not w.is_cuda or dtype not in _TYPES:
        raise TypeError("w must be a uint8 tensor on the GPU, dtype float32, float16 or bfloat16")
    m = targets.numel()
    _plain(targets, torch.int32, w.device, (m,), "targets")
    _tiled(w, w.device, n, k, "w")
    _tiled(xq, w.device, m, k, "xq")
    for name, t in ("losses", losses), ("lse", lse), ("grad", grad):
        if t is not None:
            _plain(t, torch.float32, w.device, (m,), name)
    dx = torch.empty((m, k), dtype=dtype, device=w.device)
    workspace, ws, ws_bytes = _workspace(workspace, _need("nh_i8_token_losses_grad_workspace_bytes", m, n, k, _TYPES[dtype]), w.device)
    _call("nh_i8_token_losses_grad", w.device, w.data_ptr(), xq.data_ptr(), targets.data_ptr(), losses.data_ptr(), lse.data_ptr(), None if grad is None else grad.data_ptr(), dx.data_ptr(),
          _TYPES[dtype], m, n, k, ws, ws_bytes)
    return dx


def from_q8_0(w_tiled: torch.Tensor, n: int, k: int) -> torch.Tensor:
    """A tiled Q8_0 weight [n, k] (q8_0.tile) with one scale per row instead of one per 32 values: each row is rounded once more, to max |w| / 127 of the whole row."""
    from . import q8_0

    return quantize(q8_0.get_rows(w_tiled, torch.arange(n, dtype=torch.int32, device=w_tiled.device), n, k, tiled=True))
