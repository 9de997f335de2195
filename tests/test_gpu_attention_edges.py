"""GPU: attention and the paged cache where a call stands on the edge of what it takes, beside test_gpu_attention.py and test_gpu_cache_pages.py: tensors of
another device, batches of nobody, peaked scores across the pieces of a row's keys, streams of other owners, the forms that only large calls take."""
import pytest
import torch

from test_gpu_attention import A, BF16, F16, F32, INF, KINDS, NAN, Batch, _check, _check_prompt, _check_with_odd_values, _starts, kernel  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_value_pages_on_the_host_are_refused(A, monkeypatch, native):  # noqa: F811
    if not native:
        monkeypatch.setattr(A, "_calls", None)
    b = Batch(3, [20, 5], 16, 2, 64, F16)
    k, v, table, dl = b.device()
    q, kv = b.rows(2, 4, F32).cuda(), b.rows(2, 2, F32).cuda()
    ints, starts = torch.zeros(2, dtype=torch.int32).cuda(), torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    host = v.cpu()
    for call in (lambda: A.append_rope(q, kv, kv, k, host, table, dl, A.rope_turns(64)), lambda: A.attention_prompt(q, k, host, table, dl, starts), lambda: A.attention_decode(q, k, host, table, dl),
                 lambda: A.cache_step(k[None], host[None], table, dl, ints, ints), lambda: A.cache_compact(k[None], host[None], table, dl)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("native", [True, False])
def test_calls_for_nobody(A, monkeypatch, native):  # noqa: F811
    if not native:
        monkeypatch.setattr(A, "_calls", None)
    b = Batch(5, [70], 16, 2, 64, F16, shared=4)
    k, v, table, dl = b.device()
    prefix = torch.tensor(b.common, dtype=torch.int32).cuda()
    q, kv, none = torch.empty(0, 8, 64, device="cuda"), torch.empty(0, 2, 64, device="cuda"), dl[:0]
    assert A.attention_decode(q, k, v, table[:0], none, prefix_pages=prefix).shape == (0, 8, 64)
    assert A.attention_decode(q, k, v, table[:0], none, prefix_pages=prefix, workspace=A.decode_workspace(0, 8, 2, 64, prefix_pages=4, page_size=16)).shape == (0, 8, 64)
    assert A.attention_decode(q, k, v, table[:0], none).shape == (0, 8, 64)
    assert A.attention_prompt(q, k, v, table[:0], none, torch.zeros(1, dtype=torch.int32).cuda()).shape == (0, 8, 64)
    assert A.append_rope(q, kv, kv, k, v, table[:0], none, A.rope_turns(64)).shape == (0, 8, 64)
    new, lengths, info = A.cache_step(k[None], v[None], table, dl, none, none)  # everybody has ended
    assert new.shape == (0, table.shape[1]) and lengths.shape == (0,) and info.tolist() == [0, 0, 0]
    new, info = A.cache_compact(k[None], v[None], table[:0], none)
    assert new.shape == (0, table.shape[1]) and info.tolist() == [0, 0, 0]


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("length", [150, 3000])
def test_odd_values_far_below_the_largest_score(A, kernel, dtype, cache, dim, page, length):  # noqa: F811
    # One key's score is thousands above all others, so that what any other part of the keys adds up to is joined with a factor that is too small for fp32. An
    # infinite value there stays infinite all the same, wherever the keys are cut: over waves, groups of waves, workgroups, a prefix and its pieces.
    pages = 1280 // page if length == 3000 else 64 // page
    for top in (5, length // 2, length - 10):
        b = Batch(41, [length], page, 2, dim, cache, shared=pages)
        ahead = torch.sign(torch.randn(2, dim, generator=b.g))  # the direction that the largest score has, for each kv head
        b.k[b.table[0][top // page], :, top % page] = (8 * ahead).to(cache)
        for i, j in enumerate(range(3, length - 6, max(1, length // 40))):
            if j != top:
                b.v[b.table[0][j // page], i % 2, i, j % page] = (INF, -INF, INF, NAN)[i % 4]
        q = (60 * ahead.repeat_interleave(4, 0) + b.rows(5, 8, F32)).to(dtype)
        k, v, table, lengths = b.device()
        keys, values, there = b.keys(0, length)
        out = A.attention_prompt(q.cuda(), k, v, table, lengths, torch.tensor([0, 5], dtype=torch.int32).cuda()).cpu()
        for i in range(5):
            seen = length - 4 + i
            _check_with_odd_values(out[i], q[i], keys[:, :seen], values[:, :seen], there[:seen], dim**-0.5, dtype, ("prompt", top, i))
        for prefix in (None, torch.tensor(b.common, dtype=torch.int32).cuda()):
            out = A.attention_decode(q[:1].cuda(), k, v, table, lengths, prefix_pages=prefix).cpu()
            _check_with_odd_values(out[0], q[0], keys, values, there, dim**-0.5, dtype, ("decode", top, prefix is not None))


PER_THREAD = 2  # the handle that names the calling thread's own default stream, whichever thread that is


@pytest.mark.parametrize("native", [True, False])
def test_the_stream_that_is_another_one_in_each_thread(A, monkeypatch, native):  # noqa: F811
    # Memory that a call takes for itself goes to the next call on a stream of the same handle, here another thread's, which does not wait for this one.
    if not native:
        monkeypatch.setattr(A, "_calls", None)
    b = Batch(43, [700, 33], 32, 2, 64, F16)
    q = b.rows(2, 8, F32)
    k, v, table, dl = b.device()
    x, starts = q.cuda(), torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    large = tuple(t[0] for t in A.empty_cache(1, 50000, 1, 16, 64))
    ints = torch.zeros(2, dtype=torch.int32).cuda()
    spaces = A.decode_workspace(2, 8, 2, 64), A.prompt_workspace(2, 2, 8, 2, 64)
    want = A.attention_decode(x, k, v, table, dl), A.attention_prompt(x, k, v, table, dl, starts)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(PER_THREAD)):
        for call in (lambda: A.attention_decode(x, k, v, table, dl), lambda: A.attention_prompt(x, k, v, table, dl, starts), lambda: A.cache_step(large[0][None], large[1][None], table, dl, ints, ints),
                     lambda: A.cache_compact(large[0][None], large[1][None], table, dl)):
            with pytest.raises(ValueError):
                call()
        got = A.attention_decode(x, k, v, table, dl, workspace=spaces[0]), A.attention_prompt(x, k, v, table, dl, starts, workspace=spaces[1])
        A.cache_step(k[None], v[None], table, dl, ints, ints)  # (a small cache's step needs no memory)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_streams_of_other_owners_leave_nothing_behind(A):  # noqa: F811
    # the handle of a stream that somebody else made and destroyed may be given out again: nothing is kept under it
    import ctypes

    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    hip = ctypes.CDLL(path)
    b = Batch(47, [3000, 50, 900], 64, 2, 128, F16)
    k, v, table, dl = b.device()
    q = b.rows(3, 8, F32).cuda()
    want = A.attention_decode(q, k, v, table, dl)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(6):
        handle = ctypes.c_void_p()
        assert hip.hipStreamCreate(ctypes.byref(handle)) == 0
        with torch.cuda.stream(torch.cuda.ExternalStream(handle.value)):
            for _ in range(3):
                got = A.attention_decode(q, k, v, table, dl)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del got
        assert torch.cuda.memory_allocated() == before
        assert hip.hipStreamDestroy(handle) == 0


@pytest.mark.parametrize("heads", [4, 64])
def test_starts_that_descend(A, kernel, heads):  # noqa: F811
    # the same rows in half of 2048 sequences of 64000 keys: more work, in steps, than 32 bits hold, also of the sequences that a wave adds up at once
    rows, n, pages = 1 << 18, 2048, 250
    rows = rows * 4 // heads
    k, v = (t[0].zero_() for t in A.empty_cache(1, pages, heads // 4, 256, 64))
    memory = torch.full((rows + 256, heads, 64), 7.0, dtype=F16, device="cuda")
    q = torch.zeros(rows, heads, 64, dtype=F16, device="cuda")
    table = torch.arange(pages, dtype=torch.int32).repeat(n, 1).cuda()
    lengths = torch.full((n,), 64000, dtype=torch.int32).cuda()
    starts = torch.tensor([0, rows] * (n // 2) + [0], dtype=torch.int32).cuda()
    A.attention_prompt(q, k, v, table, lengths, starts, out=memory[128:-128])
    assert bool((memory[:128] == 7).all()) and bool((memory[-128:] == 7).all())
    if kernel == 1:
        assert bool((memory == 7).all())
