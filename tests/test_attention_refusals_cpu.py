"""CPU: calls of attention and the paged cache that end before any device work, beside those of test_attention_cpu.py."""
import ctypes as C

import pytest
import torch

from test_attention_cpu import BOGUS, _append, _batch, _cache, _compact, _decode, _prompt, _step  # noqa: F401


class _On:
    """A tensor that says it is on some device."""

    def __init__(self, tensor, device):
        self._tensor, self.device = tensor, torch.device(device)
        self.is_cuda = self.device.type == "cuda"

    def __getattr__(self, name):
        return getattr(self._tensor, name)


@pytest.mark.parametrize("where", ["cpu", "cuda:1"])
@pytest.mark.parametrize("dims", [4, 5])
def test_value_pages_of_another_device_are_refused(where, dims):
    from nihilus_amd import attention as A

    k, v = A.empty_cache(1, 4, 2, 16, 64, device="cpu")
    if dims == 4:
        k, v = k[0], v[0]
    cache = A._pages(_On(k, "cuda:0"), _On(v, "cuda:0"), dims)
    assert (cache.pages, cache.kv_heads, cache.page_size, cache.head_dim) == (4, 2, 16, 64)
    with pytest.raises(TypeError):
        A._pages(_On(k, "cuda:0"), _On(v, where), dims)


@pytest.mark.parametrize("page_size,count", [(16, 1), (64, 4), (256, 1 << 22)])
def test_a_prefix_that_no_sequence_shares(page_size, count):
    from nihilus_amd import _lib

    n, c = C.c_int64(), C.c_int64()
    assert _lib.lib().nh_attn_decode_needs(0, 4, 2, 64, 0, page_size, C.byref(n), C.byref(c)) == 0
    without = n.value, c.value
    assert _lib.lib().nh_attn_decode_needs(0, 4, 2, 64, count, page_size, C.byref(n), C.byref(c)) == 0
    assert (n.value, c.value) == without
    assert _decode(cache=_cache(page_size=page_size), batch=_batch(sequences=0), prefix=BOGUS, count=count, q=None, out=None, ws=None, counters=None) == 0


# where the calls on a cache's pages find what they read, and where they put what they write; far from each other
READ = {"page_table": BOGUS * 2, "lengths": BOGUS * 3, "parents": BOGUS * 4, "grow": BOGUS * 5, "k_pages": BOGUS * 16, "v_pages": BOGUS * 32}
SIZE = {"page_table": 48, "lengths": 12, "parents": 12, "grow": 12, "k_pages": 32768, "v_pages": 32768, "new_table": 48, "new_lengths": 12, "info": 12}
WRITTEN = {"new_table": BOGUS * 6, "new_lengths": BOGUS * 7, "info": BOGUS * 8}


def _pages_call(which, **over):
    at = {**READ, **WRITTEN, **over}
    cache, batch = _cache(k_pages=at["k_pages"], v_pages=at["v_pages"]), _batch(page_table=at["page_table"], lengths=at["lengths"])
    if which == "compact":
        return _compact(cache, batch, at["new_table"], at["info"], None, 0)
    return _step(cache, batch, at["parents"], at["grow"], 3, at["new_table"], at["new_lengths"], at["info"], None, 0)


def _overlapping(which):
    results = ["new_table", "info"] if which == "compact" else list(WRITTEN)
    inputs = [n for n in READ if which == "step" or n not in ("parents", "grow")]
    return [(r, other) for i, r in enumerate(results) for other in inputs + results[:i]]


@pytest.mark.parametrize("which,result,other", [(w, *pair) for w in ("step", "compact") for pair in _overlapping(w)])
def test_results_of_the_page_calls_over_what_they_read_are_refused(which, result, other):
    # every workgroup plans from the inputs while the first one writes the results
    there = {**READ, **WRITTEN}[other]
    for at in (there, there + SIZE[other] - 4, there - SIZE[result] + 4):
        assert _pages_call(which, **{result: at}) == -6, at
    if torch.cuda.is_available():
        return  # (what is not refused would run)
    for at in (there + SIZE[other], there - SIZE[result]):
        assert _pages_call(which, **{result: at}) == -4, at


@pytest.mark.parametrize("name", [*READ, *WRITTEN])
def test_a_workspace_of_the_page_calls_over_anything_else_is_refused(name):
    from nihilus_amd import _lib

    pages, ws = 100000, 1 << 40
    need = _lib.lib().nh_attn_pages_workspace_bytes(pages, 3, 4)
    far = {**WRITTEN, "parents": READ["parents"], "grow": READ["grow"], "k_pages": 1 << 41, "v_pages": 1 << 42}
    size = {**SIZE, "k_pages": pages * 4096, "v_pages": pages * 4096}[name]
    for at in (ws, ws + need - 16, ws - size + 16 if size > 48 else ws + 256):
        here = {**far, name: at}
        batch = _batch(page_table=here.get("page_table", READ["page_table"]), lengths=here.get("lengths", READ["lengths"]))
        cache = _cache(pages=pages, k_pages=here["k_pages"], v_pages=here["v_pages"])
        assert _step(cache, batch, here["parents"], here["grow"], 3, here["new_table"], here["new_lengths"], here["info"], ws, need) == -6, at
        if name not in ("parents", "grow", "new_lengths"):
            assert _compact(cache, batch, here["new_table"], here["info"], ws, need) == -6, at


# A launch has fewer than 2^32 threads along its grid: what the kernels would need more for is refused ahead of it.


def _fits(status):
    """What is not refused ends at the missing GPU; with one it would run."""
    return status == -4


@pytest.mark.parametrize("rows,heads,kv_heads,fits", [((1 << 24) - 270000, 1, 1, True), ((1 << 24) - 250000, 1, 1, False), (1 << 24, 2, 1, False), (1 << 28, 4, 2, False), (1 << 30, 1, 1, False),
                                                       (1 << 14, 65535, 65535, False), (8191, 65535, 65535, True)])
def test_rows_of_append_that_no_launch_has_workgroups_for(rows, heads, kv_heads, fits):
    # a workgroup of 256 threads for each row, and one for 64 rows of a head's values
    assert (rows + -(-rows // 64) * kv_heads < 1 << 24) == fits
    if fits and torch.cuda.is_available():
        return
    far = dict(q=1 << 44, out=1 << 45, k=1 << 46, v=(1 << 46) + (1 << 45), batch=_batch(starts=BOGUS), cache=_cache(kv_heads=kv_heads))
    status = _append(rows=rows, heads=heads, strides=(heads * 64, kv_heads * 64, kv_heads * 64), **far)
    assert _fits(status) if fits else status == -5


@pytest.mark.parametrize("rows,sequences,heads,kv_heads,fits", [(5 << 20, 1 << 20, 32, 8, True), (5 << 20, 1 << 20, 64, 16, False), (1 << 20, 200000, 256, 64, True), (1 << 21, 1 << 18, 256, 64, False)])
def test_tiles_of_a_prompt_that_no_launch_has_workgroups_for(rows, sequences, heads, kv_heads, fits):
    from nihilus_amd import _lib

    tiles = (rows * (heads // kv_heads) // 128 + sequences) * kv_heads
    assert (tiles < 1 << 24) == fits and _lib.lib().nh_attn_debug_prompt_kernel(rows, sequences, heads, kv_heads, -1) == 2
    n, c = C.c_int64(), C.c_int64()
    assert _lib.lib().nh_attn_prompt_needs(rows, sequences, heads, kv_heads, 64, C.byref(n), C.byref(c)) == (0 if fits else -5)
    if fits and torch.cuda.is_available():
        return
    status = _prompt(cache=_cache(kv_heads=kv_heads), batch=_batch(starts=BOGUS, sequences=sequences), q=1 << 44, out=1 << 45, rows=rows, heads=heads, stride=heads * 64, bytes=1 << 60, counter_bytes=1 << 60)
    assert _fits(status) if fits else status == -5


def test_tiles_of_a_prefix_that_no_launch_has_workgroups_for():
    from nihilus_amd import _lib

    n, c = C.c_int64(), C.c_int64()
    for sequences, status in [((1 << 20) - 8, 0), (1 << 20, -5)]:  # 1024 query heads of one kv head: eight tiles of 512 threads each
        assert _lib.lib().nh_attn_decode_needs(sequences, 1024, 1, 64, 1, 16, C.byref(n), C.byref(c)) == status
        assert _lib.lib().nh_attn_decode_needs(sequences, 1024, 1, 64, 0, 16, C.byref(n), C.byref(c)) == 0
    assert _decode(cache=_cache(kv_heads=1), batch=_batch(sequences=1 << 20, table_width=1), prefix=BOGUS, count=1, q=1 << 44, out=1 << 45, heads=1024, stride=65536, bytes=1 << 60, counter_bytes=1 << 60) == -5


def test_more_table_entries_than_a_step_can_count():
    # 2^31 pages could be wanted at once, one more than the counts of `info` hold
    sequences, width = 1 << 20, 1 << 11
    batch = _batch(page_table=1 << 40, sequences=sequences, table_width=width)
    assert _step(batch=batch, children=sequences, parents=1 << 41, grow=1 << 42, table=1 << 43, lengths=1 << 44) == -5
    assert _compact(batch=batch, table=1 << 43) == -5
    if not torch.cuda.is_available():
        assert _fits(_step(batch=_batch(page_table=1 << 40, lengths=1 << 39, sequences=sequences, table_width=width), children=sequences - 1, parents=1 << 41, grow=1 << 42, table=1 << 43, lengths=1 << 44, ws=1 << 45))


def test_the_customisation_points_as_calls_of_this_abi_compile():
    import os
    import subprocess

    from nihilus_amd.build import hipcc
    from test_attention_cpu import ROOT

    cxx = os.path.join(os.path.dirname(hipcc()), "amdclang++")
    src = os.path.join(ROOT, "tests", "cpp", "attention_customisation_points.cpp")
    res = subprocess.run([cxx, "-std=c++23", "-Wall", "-Wextra", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), src], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
