"""What stands between a block's projections, for callers that hold torch tensors: rope and the write into a paged key / value cache, causal
attention over it, and the cache's pages from one step to the next.

torch is used for device memory and streams only; every operation is one call through the C ABI (``include/nihilus_amd/attention_abi.h``,
which says what each one computes), on the current stream of the tensors' device.  In the reference these are nodes of the mega cores whose
GPU bodies are empty (infra/core_traits.hpp:596-616, :743-766).

The cache of a model is two tensors, ``k_pages`` [layers, pages, kv_heads, page_size, head_dim] and ``v_pages`` [layers, pages, kv_heads, head_dim,
page_size], fp16 or bf16; a layer's own, ``k_pages[layer]`` and ``v_pages[layer]``, is what append_rope and the attentions take.  A batch is
``page_table`` int32 [sequences, width], ``lengths`` int32 [sequences] (tokens of each sequence, those of this call among them) and, where sequences have other
than one row each, ``starts`` int32 [sequences + 1]: rows starts[b] .. starts[b + 1] - 1 are the last tokens of sequence b.  Tables live on the GPU and
are checked where they are used: a key on a page that the cache does not have is not written, and left out of attention.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .q8_0 import _calls, _native, _stream

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)


def empty_cache(layers: int, pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.float16, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """The K and V pages of a model, not initialised (nothing that was not written is ever part of a result)."""
    if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS or dtype not in (torch.float16, torch.bfloat16) or min(layers, pages, kv_heads) < 1:
        raise ValueError(f"a cache has pages of {PAGE_SIZES} tokens, heads of {HEAD_DIMS} values in float16 or bfloat16, and at least one layer, page and head")
    return (torch.empty((layers, pages, kv_heads, page_size, head_dim), dtype=dtype, device=device), torch.empty((layers, pages, kv_heads, head_dim, page_size), dtype=dtype, device=device))


def rope_turns(head_dim: int, base: float = 500000.0, factors=None, rotary: int | None = None, device="cuda") -> torch.Tensor:
    """Turns per position of each pair of values, fp64 [rotary / 2]: base^(-2i / rotary) / (2 pi), divided by factors[i] if given (the model's rope_freqs)."""
    rotary = head_dim if rotary is None else rotary
    if rotary % 16 or not 0 <= rotary <= head_dim:
        raise ValueError("rotary must be a multiple of 16, head_dim at most")
    turns = torch.tensor([base ** (-2.0 * i / rotary) / (2.0 * math.pi) for i in range(rotary // 2)], dtype=torch.float64)
    if factors is not None:
        turns /= torch.as_tensor(factors, dtype=torch.float64).cpu().reshape(rotary // 2)
    return turns.to(device)


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, dims: int):
    if not (k_pages.is_cuda and k_pages.is_contiguous() and v_pages.is_contiguous()) or k_pages.dtype not in (torch.float16, torch.bfloat16) or v_pages.dtype != k_pages.dtype:
        raise TypeError("k_pages and v_pages must be contiguous float16 or bfloat16 tensors on the GPU")
    if v_pages.device != k_pages.device:
        raise TypeError("k_pages and v_pages must be on the same GPU")
    if k_pages.dim() != dims or v_pages.shape != (*k_pages.shape[:-2], k_pages.shape[-1], k_pages.shape[-2]):
        raise ValueError(f"k_pages must be [{'layers, ' if dims == 5 else ''}pages, kv_heads, page_size, head_dim], v_pages the same with its last two the other way round")
    layers, (pages, kv_heads, page_size, head_dim) = (k_pages.shape[0] if dims == 5 else 1), k_pages.shape[-4:]
    return _lib.AttnCache(k_pages.data_ptr(), v_pages.data_ptr(), layers, pages, kv_heads, page_size, head_dim, _TYPES[k_pages.dtype])


def _ints(t: torch.Tensor, like: torch.Tensor, shape, name: str) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != like.device or not t.is_contiguous():
        raise TypeError(f"{name} must be a contiguous int32 tensor on the cache's GPU")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    return t


def _batch(page_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor | None, like: torch.Tensor):
    if page_table.dim() != 2:
        raise ValueError("page_table must be [sequences, width]")
    n, width = page_table.shape
    _ints(page_table, like, (n, width), "page_table")
    _ints(lengths, like, (n,), "lengths")
    if starts is not None:
        _ints(starts, like, (n + 1,), "starts")
    return _lib.AttnBatch(page_table.data_ptr(), lengths.data_ptr(), None if starts is None else starts.data_ptr(), n, width)


def _rows(t: torch.Tensor, like: torch.Tensor, heads: int | None, name: str) -> int:
    """Elements from one row to the next of [rows, heads, head_dim]."""
    if t.device != like.device or t.dtype not in (torch.float32, like.dtype):
        raise TypeError(f"{name} must be float32 or of the cache's type, on the cache's GPU")
    dim = like.shape[-1]
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [rows, {'heads' if heads is None else heads}, {dim}]")
    least = t.shape[1] * dim
    if (t.shape[2] > 1 and t.stride(2) != 1) or (t.shape[1] > 1 and t.stride(1) != dim):
        raise ValueError(f"{name}: the heads of a row must lie side by side")
    return t.stride(0) if t.shape[0] > 1 else least


def _out(out: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape, type and device")
    return out


def _call(fn: str, device: torch.device, *args) -> None:
    """One call on the current stream of `device`, whichever device is current."""
    if device.index == torch.cuda.current_device():
        _lib.check(fn, getattr(_lib.lib(), fn)(*args, _stream()))
        return
    with torch.cuda.device(device):
        _lib.check(fn, getattr(_lib.lib(), fn)(*args, _stream()))


def append_rope(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, turns: torch.Tensor,
                starts: torch.Tensor | None = None, interleaved: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rope on q and k at the rows' positions; k and v go into a layer's pages, the rotated q is returned (out may be q itself).

    q [rows, q_heads, head_dim], k and v [rows, kv_heads, head_dim], rows apart by any multiple of 16 bytes; turns as rope_turns gives them, for the first
    2 * len(turns) values of a head: pairs are neighbours if interleaved, else half of those values apart.  Rows that no sequence has are left alone
    (in `out` too)."""
    if out is None and _calls is not None:
        r = _native(_calls.append_rope(q, k, v, k_pages, v_pages, page_table, lengths, turns, starts, int(interleaved)), "nh_attn_append_rope")
        if r is not None:
            return r
    cache, batch = _pages(k_pages, v_pages, 4), _batch(page_table, lengths, starts, k_pages)
    strides = _rows(q, k_pages, None, "q"), _rows(k, k_pages, k_pages.shape[1], "k"), _rows(v, k_pages, k_pages.shape[1], "v")
    if not (q.dtype == k.dtype == v.dtype) or not (q.shape[0] == k.shape[0] == v.shape[0]):
        raise ValueError("q, k and v must have the same type and the same number of rows")
    if turns.dtype != torch.float64 or turns.device != q.device or turns.dim() != 1 or not turns.is_contiguous():
        raise TypeError("turns must be a contiguous float64 vector on the cache's GPU")
    out = _out(out, q)
    _call("nh_attn_append_rope", q.device, C.byref(cache), C.byref(batch), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _TYPES[q.dtype], q.shape[0], q.shape[1], *strides,
          turns.data_ptr(), turns.numel(), int(interleaved))
    return out


class Workspace:
    """Memory for the attentions' own use, for callers that keep it: of one stream, or one captured graph, at a time."""

    def __init__(self, nbytes: int, counter_bytes: int, device):
        self.memory = torch.empty(nbytes, dtype=torch.uint8, device=device)
        self.counters = torch.zeros(counter_bytes // 4, dtype=torch.int32, device=device)  # every call leaves them zero

    def args(self, like: torch.Tensor):
        if self.memory.device != like.device:
            raise TypeError("the workspace must be on the cache's GPU")
        return self.memory.data_ptr(), self.memory.numel(), self.counters.data_ptr(), 4 * self.counters.numel()


_PER_THREAD = 2  # hipStreamPerThread: the handle that names the calling thread's own default stream


def _own_memory(nbytes: int, device: torch.device) -> None:
    """Refuses memory of the call's own where torch's allocator would give it to another thread's call while this one runs: it tells streams apart by their handles."""
    if nbytes and (_stream() if device.index == torch.cuda.current_device() else torch.cuda.current_stream(device).cuda_stream) == _PER_THREAD:
        raise ValueError("the per-thread default stream is another one in each thread: give a workspace, or use a stream of torch's")


def _needs(fn: str, *sizes) -> tuple[int, int]:
    n, c = C.c_int64(), C.c_int64()
    _lib.check(fn, getattr(_lib.lib(), fn)(*sizes, C.byref(n), C.byref(c)))
    return n.value, c.value


def prompt_workspace(rows: int, sequences: int, q_heads: int, kv_heads: int, head_dim: int, device="cuda") -> Workspace:
    return Workspace(*_needs("nh_attn_prompt_needs", rows, sequences, q_heads, kv_heads, head_dim), device)


def decode_workspace(sequences: int, q_heads: int, kv_heads: int, head_dim: int, prefix_pages: int = 0, page_size: int = 64, device="cuda") -> Workspace:
    return Workspace(*_needs("nh_attn_decode_needs", sequences, q_heads, kv_heads, head_dim, prefix_pages, page_size), device)


def attention_prompt(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor, scale: float | None = None,
                     out: torch.Tensor | None = None, workspace: Workspace | None = None) -> torch.Tensor:
    """Causal attention of packed rows [rows, q_heads, head_dim] over what their sequences' pages hold, keys and values of these rows among it.

    scale is 1 / sqrt(head_dim) unless given.  Rows that no sequence has are not written (in `out` they keep what they held).  workspace: see
    prompt_workspace; without one the call has its own."""
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if out is None and workspace is None and _calls is not None:
        r = _native(_calls.attention_prompt(q, k_pages, v_pages, page_table, lengths, starts, scale), "nh_attn_prompt")
        if r is not None:
            return r
    cache, batch = _pages(k_pages, v_pages, 4), _batch(page_table, lengths, starts, k_pages)
    stride = _rows(q, k_pages, None, "q")
    out = _out(out, q)
    if workspace is None:
        workspace = prompt_workspace(q.shape[0], page_table.shape[0], q.shape[1], k_pages.shape[1], k_pages.shape[3], q.device)
        _own_memory(workspace.memory.numel(), q.device)
    _call("nh_attn_prompt", q.device, C.byref(cache), C.byref(batch), q.data_ptr(), out.data_ptr(), _TYPES[q.dtype], q.shape[0], q.shape[1], stride, scale, *workspace.args(k_pages))
    return out


def attention_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, prefix_pages: torch.Tensor | None = None,
                     scale: float | None = None, out: torch.Tensor | None = None, workspace: Workspace | None = None) -> torch.Tensor:
    """Attention of one row per sequence, q [sequences, q_heads, head_dim], over all of its keys.

    prefix_pages, int32: pages whose keys every sequence begins with; they are read once for the whole batch where that is faster, and that many entries at the front of
    each page_table row are not looked at here (cache_step and cache_compact do: to them a page that no row names is free).  A sequence of no tokens gives zeros.  workspace: see decode_workspace; without one the call has its own."""
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if out is None and workspace is None and _calls is not None:
        r = _native(_calls.attention_decode(q, k_pages, v_pages, page_table, lengths, prefix_pages, scale), "nh_attn_decode")
        if r is not None:
            return r
    cache, batch = _pages(k_pages, v_pages, 4), _batch(page_table, lengths, None, k_pages)
    stride = _rows(q, k_pages, None, "q")
    if q.shape[0] != page_table.shape[0]:
        raise ValueError("q must have a row for each sequence")
    count = 0
    if prefix_pages is not None:
        count = prefix_pages.numel()
        _ints(prefix_pages, k_pages, (count,), "prefix_pages")
    out = _out(out, q)
    if workspace is None:
        _, kv_heads, page_size, head_dim = k_pages.shape
        workspace = decode_workspace(q.shape[0], q.shape[1], kv_heads, head_dim, count, page_size, q.device)
        _own_memory(workspace.memory.numel(), q.device)
    _call("nh_attn_decode", q.device, C.byref(cache), C.byref(batch), prefix_pages.data_ptr() if count else None, count, q.data_ptr(), out.data_ptr(), _TYPES[q.dtype], q.shape[1], stride, scale,
          *workspace.args(k_pages))
    return out


def _pages_workspace(pages: int, sequences: int, width: int, device) -> torch.Tensor:
    n = _lib.lib().nh_attn_pages_workspace_bytes(pages, sequences, width)
    _lib.check("nh_attn_pages_workspace_bytes", n if n < 0 else 0)
    _own_memory(n, device)
    return torch.empty(n, dtype=torch.uint8, device=device)


def cache_step(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor,
               grow: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The cache's next state: new sequence i goes on where sequence parents[i] stands (-1: it is empty), grow[i] tokens longer or shorter.

    Returns (page_table, lengths, info): the new tables, whose lengths count the tokens to come (what append_rope takes next), and int32 [3]: pages held now,
    pages copied, pages missing.  Full pages are shared, a page that several would go on writing into is copied (keys and values, all layers), sequences
    that nobody goes on with are ended and their pages free.  The old tables stay as they are."""
    if _calls is not None:
        r = _native(_calls.cache_step(k_pages, v_pages, page_table, lengths, parents, grow), "nh_attn_cache_step")
        if r is not None:
            return r
    cache, batch = _pages(k_pages, v_pages, 5), _batch(page_table, lengths, None, k_pages)
    if parents.dim() != 1:
        raise ValueError("parents must be a vector")
    n, width = parents.numel(), page_table.shape[1]
    _ints(parents, k_pages, (n,), "parents")
    _ints(grow, k_pages, (n,), "grow")
    table, now, info = (torch.empty(s, dtype=torch.int32, device=k_pages.device) for s in ((n, width), (n,), (3,)))
    ws = _pages_workspace(k_pages.shape[1], n, width, k_pages.device)
    _call("nh_attn_cache_step", k_pages.device, C.byref(cache), C.byref(batch), parents.data_ptr(), grow.data_ptr(), n, table.data_ptr(), now.data_ptr(), info.data_ptr(), ws.data_ptr(), ws.numel())
    return table, now, info


def cache_compact(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Moves the pages that hold the sequences' tokens to the front of the cache, in all layers.

    Returns (page_table, info): where they are then, and int32 [3]: pages in use (from that index on nothing is held), pages moved, entries that named no page."""
    if _calls is not None:
        r = _native(_calls.cache_compact(k_pages, v_pages, page_table, lengths), "nh_attn_cache_compact")
        if r is not None:
            return r
    cache, batch = _pages(k_pages, v_pages, 5), _batch(page_table, lengths, None, k_pages)
    n, width = page_table.shape
    table, info = (torch.empty(s, dtype=torch.int32, device=k_pages.device) for s in ((n, width), (3,)))
    ws = _pages_workspace(k_pages.shape[1], n, width, k_pages.device)
    _call("nh_attn_cache_compact", k_pages.device, C.byref(cache), C.byref(batch), table.data_ptr(), info.data_ptr(), ws.data_ptr(), ws.numel())
    return table, info
