"""CPU: the C ABI of attention and the paged cache is exported as declared and refuses bad calls before any device work; the wrappers refuse tensors that do not fit."""
import ctypes as C
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BOGUS = 0x10000  # never dereferenced: every call below ends in validation


def _cache(**over):
    from nihilus_amd import _lib

    v = dict(k_pages=BOGUS, v_pages=BOGUS, layers=1, pages=8, kv_heads=2, page_size=16, head_dim=64, type=1)
    v.update(over)
    return _lib.AttnCache(*v.values())


def _batch(**over):
    from nihilus_amd import _lib

    v = dict(page_table=BOGUS, lengths=BOGUS, starts=None, sequences=3, table_width=4)
    v.update(over)
    return _lib.AttnBatch(*v.values())


def test_header_and_bindings_name_the_same_functions():
    from nihilus_amd import _lib

    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "nihilus_amd", "attention_abi.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(nh_attn_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(_lib.ATTENTION_SIGNATURES)
    assert all(hasattr(_lib.lib(), n) for n in names)


def test_the_header_is_plain_c():
    import subprocess

    res = subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), "-x", "c", os.path.join(ROOT, "include", "nihilus_amd", "attention_abi.h")],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr


def _append(cache=None, batch=None, q=BOGUS, k=BOGUS, v=BOGUS, out=BOGUS * 2, type=0, rows=3, heads=4, strides=(256, 128, 128), turns=BOGUS, pairs=32):
    from nihilus_amd import _lib

    return _lib.lib().nh_attn_append_rope(C.byref(cache or _cache()), C.byref(batch or _batch()), q, k, v, out, type, rows, heads, *strides, turns, pairs, 1, None)


MEMORY = dict(ws=BOGUS, bytes=1 << 30, counters=BOGUS, counter_bytes=1 << 30)


def _prompt(cache=None, batch=None, q=BOGUS, out=BOGUS * 2, type=0, rows=3, heads=4, stride=256, scale=0.125, **memory):
    from nihilus_amd import _lib

    return _lib.lib().nh_attn_prompt(C.byref(cache or _cache()), C.byref(batch or _batch(starts=BOGUS)), q, out, type, rows, heads, stride, scale, *{**MEMORY, **memory}.values(), None)


def _decode(cache=None, batch=None, prefix=None, count=0, q=BOGUS, out=BOGUS * 2, type=0, heads=4, stride=256, scale=0.125, **memory):
    from nihilus_amd import _lib

    return _lib.lib().nh_attn_decode(C.byref(cache or _cache()), C.byref(batch or _batch()), prefix, count, q, out, type, heads, stride, scale, *{**MEMORY, **memory}.values(), None)


def _step(cache=None, batch=None, parents=BOGUS, grow=BOGUS, children=3, table=BOGUS * 2, lengths=BOGUS * 3, info=BOGUS * 4, ws=BOGUS, bytes=1 << 30):
    from nihilus_amd import _lib

    return _lib.lib().nh_attn_cache_step(C.byref(cache or _cache()), C.byref(batch or _batch()), parents, grow, children, table, lengths, info, ws, bytes, None)


def _compact(cache=None, batch=None, table=BOGUS * 2, info=BOGUS * 4, ws=BOGUS, bytes=1 << 30):
    from nihilus_amd import _lib

    return _lib.lib().nh_attn_cache_compact(C.byref(cache or _cache()), C.byref(batch or _batch()), table, info, ws, bytes, None)


@pytest.mark.parametrize("call", [_append, _prompt, _decode, _step, _compact])
def test_caches_and_batches_that_are_refused(call):
    starts = {"starts": BOGUS} if call is _prompt else {}
    for status, over in [(-1, {"k_pages": None}), (-1, {"v_pages": None}), (-2, {"k_pages": BOGUS + 8}), (-2, {"v_pages": BOGUS + 2}), (-3, {"layers": 0}), (-3, {"pages": 0}),
                         (-3, {"kv_heads": 0}), (-3, {"kv_heads": -2}), (-3, {"page_size": 8}), (-3, {"page_size": 48}), (-3, {"page_size": 512}), (-3, {"head_dim": 96}), (-3, {"head_dim": 256}),
                         (-6, {"type": 0}), (-6, {"type": 3}), (-5, {"pages": 1 << 40})]:
        assert call(cache=_cache(**over)) == status, over
    for status, over in [(-3, {"sequences": -1}), (-3, {"table_width": -1}), (-1, {"lengths": None}), (-1, {"page_table": None}), (-5, {"sequences": 1 << 21}), (-5, {"table_width": 1 << 27})]:
        assert call(batch=_batch(**{**starts, **over})) == status, over


@pytest.mark.parametrize("call", [_append, _prompt, _decode])
def test_rows_that_are_refused(call):
    assert call(cache=_cache(layers=2)) == -3
    assert call(type=2) == -6 and call(type=7) == -6  # an fp16 cache takes fp32 and fp16
    assert call(heads=3) == -3 and call(heads=0) == -3
    assert call(q=None) == -1 and call(out=None) == -1
    assert call(q=BOGUS + 4) == -2 and call(out=BOGUS + 8) == -2


def test_append_refusals():
    assert _append(strides=(255, 128, 128)) == -3 and _append(strides=(256, 120, 128)) == -3 and _append(strides=(256, 128, 64)) == -3
    assert _append(strides=(257, 128, 128)) == -2 and _append(type=1, strides=(260, 128, 128)) == -2  # rows start on 16 bytes
    assert _append(pairs=12) == -3 and _append(pairs=40) == -3 and _append(pairs=-8) == -3
    assert _append(turns=None) == -1 and _append(k=None) == -1 and _append(v=None) == -1
    assert _append(rows=2) == -6  # without starts: a row per sequence
    assert _append(rows=-1, batch=_batch(starts=BOGUS)) == -3 and _append(rows=1 << 29, batch=_batch(starts=BOGUS)) == -5
    assert _append(q=BOGUS, out=BOGUS, strides=(512, 128, 128)) == -6  # in place only without gaps
    assert _append(rows=0, batch=_batch(starts=BOGUS), q=None, k=None, v=None, out=None) == 0
    assert _append(rows=0, batch=_batch(sequences=0), q=None, k=None, v=None, out=None) == 0


def test_attention_refusals():
    for call in (_prompt, _decode):
        assert call(stride=128) == -3 and call(stride=258) == -2
        for scale in (0.0, -1.0, float("inf"), float("nan")):
            assert call(scale=scale) == -6
    assert _prompt(batch=_batch()) == -1  # starts
    assert _prompt(rows=-1) == -3 and _prompt(rows=1 << 29) == -5
    assert _prompt(rows=0, q=None, out=None) == 0 and _prompt(batch=_batch(starts=BOGUS, sequences=0), q=None, out=None) == 0
    assert _decode(batch=_batch(starts=BOGUS)) == -6
    for call in (_prompt, _decode):
        assert call(ws=None) == -1 and call(ws=BOGUS + 16) == -2 and call(bytes=100) == -6
        assert call(counters=None) == -1 and call(counters=BOGUS + 64) == -2 and call(counter_bytes=8) == -6
    assert _decode(count=1) == -1 and _decode(count=-1) == -3 and _decode(count=1 << 40) == -5
    assert _decode(batch=_batch(sequences=0), q=None, out=None, ws=None, counters=None) == 0


def test_pages_refusals():
    for call in (_step, _compact):
        assert call(info=None) == -1 and call(table=None) == -1
        large = dict(cache=_cache(pages=100000))  # (a small one needs no workspace)
        assert call(ws=None, **large) == -1 and call(ws=BOGUS + 128) == -2 and call(bytes=64, **large) == -6
        assert call(table=BOGUS + 16) == -6  # the old table, in part
    assert _step(parents=None) == -1 and _step(grow=None) == -1 and _step(lengths=None) == -1
    assert _step(children=-1) == -3 and _step(children=1 << 21) == -5
    assert _step(lengths=BOGUS) == -6 and _step(lengths=BOGUS * 5, parents=BOGUS * 5 + 8) == -6 and _step(lengths=BOGUS * 5, grow=BOGUS * 5 - 8) == -6


def test_workspace_sizes():
    from nihilus_amd import _lib

    lib = _lib.lib()
    n, c = C.c_int64(), C.c_int64()

    def decode(*sizes):
        status = lib.nh_attn_decode_needs(*sizes, C.byref(n), C.byref(c))
        return status or n.value

    def prompt(*sizes):
        status = lib.nh_attn_prompt_needs(*sizes, C.byref(n), C.byref(c))
        return status or n.value

    assert decode(64, 32, 8, 128, 0, 64) >= 64 * 32 * 128 * 4 and c.value >= 64 * 8 * 4
    assert decode(64, 32, 8, 128, 128, 64) > decode(64, 32, 8, 128, 0, 64)
    assert decode(4, 33, 8, 128, 0, 64) == -3 and decode(4, 32, 0, 128, 0, 64) == -3 and decode(4, 32, 8, 80, 0, 64) == -3 and decode(4, 32, 8, 128, 0, 24) == -3 and decode(-1, 32, 8, 128, 0, 64) == -3
    assert decode(1 << 21, 32, 8, 128, 0, 64) == -5 and decode(4, 32, 8, 128, -1, 64) == -3
    assert prompt(20, 2, 32, 8, 128) > 0 and c.value > 0 and prompt(8192, 1, 64, 8, 128) == 0 and c.value == 0  # many rows: the tile kernel, which needs nothing
    assert prompt(-1, 2, 32, 8, 128) == -3 and prompt(20, 2, 32, 8, 96) == -3 and prompt(1 << 29, 2, 32, 8, 128) == -5
    assert lib.nh_attn_prompt_needs(20, 2, 32, 8, 128, None, C.byref(c)) == -1 and lib.nh_attn_decode_needs(4, 32, 8, 128, 0, 64, C.byref(n), None) == -1
    g = lib.nh_attn_pages_workspace_bytes
    assert g(1, 0, 0) == 0 and g(1000, 64, 10) == 0 and g(100000, 64, 10) >= 100000 * 8 and g(5000, 20000, 1) >= 20000 * 8 and g(0, 1, 1) == -3 and g(1, -1, 1) == -3 and g(1 << 40, 1, 1) == -5


def test_results_over_inputs_are_refused():
    size = 3 * 6 * 64 * 4  # rows, heads, values of fp32
    for call in (_prompt, _decode):
        for out in (BOGUS, BOGUS + size - 16, BOGUS - size + 16):
            assert call(out=out, heads=6, stride=384) == -6, (call, out)
        for out in (BOGUS + size, BOGUS - size):
            assert call(out=out, heads=6, stride=384) != -6, (call, out)
    far = {"k": BOGUS * 4, "v": BOGUS * 6, "heads": 6}
    assert _append(out=BOGUS, strides=(384, 128, 128), **far) != -6  # in place
    assert _append(out=BOGUS, strides=(512, 128, 128), **far) == -6 and _append(out=BOGUS + 16, strides=(384, 128, 128), **far) == -6
    assert _append(out=BOGUS * 4, strides=(384, 128, 128), **far) == -6 and _append(out=BOGUS * 6 - size + 16, strides=(384, 128, 128), **far) == -6
    assert _append(out=BOGUS * 6 - size, strides=(384, 128, 128), **far) != -6


def test_which_kernel_a_prompt_takes(monkeypatch):
    from nihilus_amd import _lib

    f = _lib.lib().nh_attn_debug_prompt_kernel
    assert f(117, 1, 32, 8, -1) == 1 and f(8192, 1, 64, 8, -1) == 2
    monkeypatch.delenv("NH_Q8_0_DEBUG_HOOKS", raising=False)
    assert f(117, 1, 32, 8, 2) == -6
    monkeypatch.setenv("NH_Q8_0_DEBUG_HOOKS", "1")
    assert f(117, 1, 32, 8, 2) == 2 and f(117, 1, 32, 8, -1) == 2 and f(117, 1, 32, 8, 3) == -6 and f(117, 1, 32, 8, 0) == 1


def test_without_a_gpu_calls_fail_loudly():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert _append() == -4 and _prompt() == -4 and _decode() == -4 and _step() == -4 and _compact() == -4


def test_wrappers_refuse_tensors_on_the_cpu():
    import torch

    from nihilus_amd import attention as A

    k, v = A.empty_cache(1, 4, 2, 16, 64, device="cpu")
    table, lengths, q = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros((1, 2, 64))
    with pytest.raises(TypeError):
        A.attention_decode(q, k[0], v[0], table, lengths)
    with pytest.raises(TypeError):
        A.cache_compact(k, v, table, lengths)
    for bad in (dict(page_size=24), dict(head_dim=80), dict(dtype=torch.float32), dict(pages=0)):
        with pytest.raises(ValueError):
            A.empty_cache(**{**dict(layers=1, pages=4, kv_heads=2, page_size=16, head_dim=64, device="cpu"), **bad})


def test_turns():
    import math

    import torch

    from nihilus_amd import attention as A

    t = A.rope_turns(128, base=10000.0, device="cpu")
    assert t.dtype == torch.float64 and t.shape == (64,) and t[0] == 1 / (2 * math.pi) and abs(float(t[63]) - 10000 ** (-126 / 128) / (2 * math.pi)) < 1e-18
    f = A.rope_turns(64, rotary=32, factors=[2.0] * 16, device="cpu")
    assert f.shape == (16,) and float(f[0]) == 0.5 / (2 * math.pi)
    with pytest.raises(ValueError):
        A.rope_turns(64, rotary=24, device="cpu")
    with pytest.raises(ValueError):
        A.rope_turns(64, rotary=80, device="cpu")
