"""GPU: attention and the paged cache where a call stands on the edge of what it takes, beside test_gpu_attention.py and test_gpu_cache_pages.py: tensors of
another device, batches of nobody, peaked scores across the pieces of a row's keys, streams of other owners, the forms that only large calls take."""
import pytest
import torch

import attention_reference as R

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


def _spoilt(b, seq, missing, odd):
    """Pages that the cache does not have and values that are not finite, past the keys whose pages a wave holds at once."""
    for j, d, x in odd:
        b.v[b.table[seq][j // b.page], :, d, j % b.page] = x
    for j in missing:
        b.table[seq][j // b.page] = (-1, len(b.k), 2**31 - 1)[j % 3]


def _keys(b, seq, n, prefix=()):
    """As Batch.keys, for many keys at a time."""
    row = torch.tensor(list(prefix) + b.table[seq][len(prefix) :])
    j = torch.arange(n)
    id = row[j // b.page]
    there = (id >= 0) & (id < len(b.k))
    id = torch.where(there, id, 0)
    k, v = b.k[id, :, j % b.page].double(), b.v[id, :, :, j % b.page].double()  # [n, kv heads, dim]
    return torch.where(there[:, None, None], k, 0.0).transpose(0, 1), torch.where(there[:, None, None], v, 0.0).transpose(0, 1), there


def _check_rows_of_long_prompts(b, out, q, new, heads, dtype):
    starts, out = _starts(new), out.cpu()
    for seq, n in enumerate(new):
        keys, values, there = _keys(b, seq, b.lengths[seq])
        for i in sorted({0, 1, 127, 128, n // 3, n // 2, n - 129, n - 2, n - 1} & set(range(n))):
            seen = b.lengths[seq] - n + i + 1
            _check_with_odd_values(out[starts[seq] + i], q[starts[seq] + i], keys[:, :seen], values[:, :seen], there[:seen], b.dim**-0.5, dtype, (seq, i))


# what the sizes choose (plan_tiles in attention_prompt.hip): tiles * kv heads above 320 one group of waves per workgroup, above 160 two, below that pieces of the keys too; parts
# and pieces of more than sixteen tiles of 64 keys, so that the pages of the next 1024 keys are taken up on the way
@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (128, 16)])
@pytest.mark.parametrize("new,cached,heads,kv_heads,many", [([2600, 300, 1], [700, 1500, 2500], 16, 16, (321, 1 << 20)), ([700], [4500], 32, 8, (161, 320)), ([300], [10000], 32, 8, (1, 160))],
                         ids=["one_group_of_waves", "two", "pieces"])
def test_tiles_past_a_thousand_keys(A, dtype, cache, dim, page, new, cached, heads, kv_heads, many):  # noqa: F811
    tiles = (sum(new) * (heads // kv_heads) // 128 + len(new)) * kv_heads
    assert many[0] <= tiles <= many[1] and A._lib.lib().nh_attn_debug_prompt_kernel(sum(new), len(new), heads, kv_heads, -1) == 2
    b = Batch(61, [a + c for a, c in zip(new, cached)], page, kv_heads, dim, cache)
    last = b.lengths[0] - 1
    _spoilt(b, 0, [1024, 1153, 2050, last - 200], [(1000, 0, INF), (1100, 1, NAN), (2047, 2, -INF), (2200, 3, INF), (2900, 4, NAN), (last - 1, 5, INF), (last, 6, NAN)])
    q = b.rows(sum(new), heads, dtype)
    k, v, table, lengths = b.device()
    out = A.attention_prompt(q.cuda(), k, v, table, lengths, torch.tensor(_starts(new), dtype=torch.int32).cuda())
    _check_rows_of_long_prompts(b, out, q, new, heads, dtype)


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_pieces_of_a_prefix_past_a_thousand_keys(A, dtype, cache, dim, page):  # noqa: F811
    n, prefix = 9, 16384  # nine tiles of rows and eight kv heads: three pieces of 5504 keys, two parts each, apart from the sequences' own keys
    own = [0, 40, 1, 7, 64, 130, 17, -prefix + 2500, 3]  # the last one ends inside the prefix
    b = Batch(67, [prefix + x for x in own], page, 8, dim, cache, shared=prefix // page)
    for j, d, x in [(900, 0, INF), (1500, 1, NAN), (2100, 2, -INF), (3000, 3, INF), (6000, 4, NAN), (12000, 5, -INF), (16383, 6, INF)]:
        b.v[b.common[j // page], :, d, j % page] = x
    common = list(b.common)
    common[1200 // page], common[7000 // page] = -1, len(b.k) + 3
    q = b.rows(n, 1024, dtype)
    k, v, table, lengths = b.device()
    out = A.attention_decode(q.cuda(), k, v, table, lengths, prefix_pages=torch.tensor(common, dtype=torch.int32).cuda()).cpu()
    for seq in (0, 5, 7):
        keys, values, there = _keys(b, seq, prefix + own[seq], common)
        for h in range(0, 1024, 301):  # (of four kv heads)
            _check_with_odd_values(out[seq, h : h + 1], q[seq, h : h + 1], keys[h // 128 : h // 128 + 1], values[h // 128 : h // 128 + 1], there, dim**-0.5, dtype, (seq, h))


@pytest.mark.parametrize("cache", [F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_few_rows_of_16_bits_lose_nothing_but_their_own_rounding(A, cache, dim, page):  # noqa: F811
    # Weights in two terms of 8 (11) bits and rounding to nearest: off by 2^-18 (2^-22) at most, beside the errors of attention_reference.py for fp32 rows
    lengths = [700, 90, 33, 260]
    b = Batch(71, lengths, page, 2, dim, cache)
    q = b.rows(8, 8, cache)
    k, v, table, dl = b.device()
    one, several = A.attention_decode(q[:4].cuda(), k, v, table, dl).cpu(), A.attention_prompt(q.cuda(), k, v, table, dl, torch.tensor([0, 2, 4, 6, 8], dtype=torch.int32).cuda()).cpu()

    def check(got, row, seq, seen):
        keys, values, there = b.keys(seq, seen)
        ref, mean, d, n = R.attend(row, keys, values, there, dim**-0.5)
        inner = mean * (2 * (torch.expm1(d)[:, None] + 4 * R.U + 2.0**-18) + (2 * n + 12) * R.U)
        most = inner + R.half_step(cache) * (ref.abs() + inner) + R.tiny(cache)
        off = (got.double() - ref).abs()
        assert bool((off <= most).all()), (seq, seen, float((off / most).max()))

    for s, n in enumerate(lengths):
        check(one[s], q[s], s, n)
        check(several[2 * s], q[2 * s], s, n - 1)
        check(several[2 * s + 1], q[2 * s + 1], s, n)


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_scores_that_just_have_bits_behind_the_point(A, kernel, dtype, cache):  # noqa: F811
    # One key far above the others, at 7e6 of a score: the row's weights are formed below a number of that size, in fp16 too. Its value comes out, off by the weight's
    # rounding (half a step of 16 bits, 2^-20 in terms) and the result's own.
    length, top, dim = 300, 170, 64
    b = Batch(73, [length], 16, 1, dim, cache)
    ahead = torch.sign(torch.randn(dim, generator=b.g))
    b.k[b.table[0][top // 16], :, top % 16] = (4 * ahead).to(cache)
    q = (4 * ahead + 0.25 * b.rows(4, 4, F32)).to(dtype)
    k, v, table, dl = b.device()
    scale = 7e6 / float((4 * ahead).double() @ (4 * ahead).double())
    want = b.v[b.table[0][top // 16], :, :, top % 16].double().expand(4, dim)
    most = want.abs() * (R.half_step(dtype) + 2.0**-20 + (R.half_step(cache) if dtype == cache else 0.0)) * 1.01
    outs = A.attention_prompt(q.cuda(), k, v, table, dl, torch.tensor([0, 4], dtype=torch.int32).cuda(), scale=scale), A.attention_decode(q[:1].cuda(), k, v, table, dl, scale=scale)
    for out in outs:
        for row in out.cpu().double():
            assert bool(((row - want).abs() <= most).all()), float(((row - want).abs() / most).max())
