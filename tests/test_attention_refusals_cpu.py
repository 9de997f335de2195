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
