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
