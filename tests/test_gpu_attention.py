"""GPU: rope + cache write, prompt and decode attention over a paged cache, against their definitions in 64 bits (attention_reference.py, which
derives the bounds), where they can go wrong: lengths around tiles, pages and pieces, ragged batches, every type, grouping and page size, pages that the
cache does not have, garbage behind a sequence's end, strides, rows of nobody."""
import math
import random

import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
KINDS = [(F32, F16), (F16, F16), (F32, BF16), (BF16, BF16)]
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def A():
    from nihilus_amd import attention

    attention._lib.lib()
    return attention


@pytest.fixture(params=[1, 2], ids=["rows", "tiles"])
def kernel(A, request, monkeypatch):
    """Each of the two kernels that a prompt may take, and each of the two ways over a decode step's shared prefix, whatever the sizes."""
    monkeypatch.setenv("NH_Q8_0_DEBUG_HOOKS", "1")
    force = A._lib.lib().nh_attn_debug_prompt_kernel
    assert force(1, 1, 1, 1, request.param) == request.param
    yield request.param
    assert force(1, 1, 1, 1, 0) in (1, 2)


class Batch:
    """A cache with sequences in scattered pages; what lies outside the sequences is NaN."""

    def __init__(self, seed, lengths, page, kv_heads, dim, cache, extra_width=1, spare=3, shared=0):
        self.g = torch.Generator().manual_seed(seed)
        self.lengths, self.page, self.kv_heads, self.dim = lengths, page, kv_heads, dim
        need = [-(-max(n, 0) // page) for n in lengths]
        total = shared + sum(max(0, n - shared) for n in need) + spare
        order = torch.randperm(total, generator=self.g).tolist()
        common, order = order[:shared], order[shared:]
        self.table = []
        width = max(need + [0]) + extra_width
        for n in need:
            mine = common[:n] + [order.pop() for _ in range(max(0, n - shared))]
            self.table.append(mine + [-1] * (width - n))
        self.common = common
        self.k = torch.full((total, kv_heads, page, dim), NAN, dtype=cache)
        self.v = torch.full((total, kv_heads, dim, page), NAN, dtype=cache)
        for row, n in zip(self.table, lengths):
            for j, id in enumerate(row):
                here = min(page, n - j * page)
                if here > 0:
                    self.k[id, :, :here] = torch.randn(kv_heads, here, dim, generator=self.g).to(cache)
                    self.v[id, :, :, :here] = torch.randn(kv_heads, dim, here, generator=self.g).to(cache)

    def rows(self, n, heads, dtype, std=1.5):
        return (torch.randn(n, heads, self.dim, generator=self.g) * std).to(dtype)

    def device(self):
        return (self.k.cuda(), self.v.cuda(), torch.tensor(self.table, dtype=torch.int32).reshape(len(self.table), -1).cuda(), torch.tensor(self.lengths, dtype=torch.int32).cuda())

    def keys(self, seq, n, prefix=None):
        row = self.table[seq]
        if prefix is not None:
            row = list(prefix) + row[len(prefix) :]
        return R.keys_of(self.k, self.v, row, n)


def _check(got, ref, mean, d, n, dtype, what):
    got = got.double()
    assert bool(torch.isfinite(got).all()), what
    off, most = (got - ref).abs(), R.bound(ref, mean, d, n, dtype)
    assert bool((off <= most).all()), (what, float((off / most).max()))


def _check_prompt(b, out, q, starts, new, dtype, scale):
    """Every row of every sequence; few rows of long sequences."""
    got = out.cpu()
    for seq, n_new in enumerate(new):
        length = b.lengths[seq]
        k, v, there = b.keys(seq, max(length, 0))
        rows = range(n_new) if n_new <= 40 else sorted({0, 1, 31, 32, 33, n_new // 2, n_new - 2, n_new - 1})
        for i in rows:
            seen = max(0, length - n_new + i + 1)
            ref = R.attend(q[starts[seq] + i], k[:, :seen], v[:, :seen], there[:seen], scale)
            _check(got[starts[seq] + i], *ref, dtype, (seq, i))


def _starts(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_prompt_ragged(A, kernel, dtype, cache, dim, page):
    new, cached = [1, 0, 33, 64, 5, 130, 0, 1], [0, 70, 0, 1, 200, 31, 0, 64]
    b = Batch(1, [a + c for a, c in zip(new, cached)], page, 2, dim, cache)
    starts = _starts(new)
    q = b.rows(sum(new), 8, dtype)
    k, v, table, lengths = b.device()
    out = A.attention_prompt(q.cuda(), k, v, table, lengths, torch.tensor(starts, dtype=torch.int32).cuda())
    assert out.dtype == dtype
    _check_prompt(b, out, q, starts, new, dtype, dim**-0.5)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (6, 2), (7, 1), (40, 2), (5, 5), (129, 1)])
def test_prompt_groupings_and_pages(A, kernel, heads, kv_heads, page):
    new, cached = [67, 3], [0, 300]
    b = Batch(heads + page, [a + c for a, c in zip(new, cached)], page, kv_heads, 64, F16)
    q = b.rows(sum(new), heads, F32)
    k, v, table, lengths = b.device()
    out = A.attention_prompt(q.cuda(), k, v, table, lengths, torch.tensor(_starts(new), dtype=torch.int32).cuda(), scale=0.2)
    _check_prompt(b, out, q, _starts(new), new, F32, 0.2)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257])
def test_prompt_lengths(A, kernel, n):
    b = Batch(n, [n], 32, 1, 128, F16)
    q = b.rows(n, 4, F16)
    k, v, table, lengths = b.device()
    out = A.attention_prompt(q.cuda(), k, v, table, lengths, torch.tensor([0, n], dtype=torch.int32).cuda())
    _check_prompt(b, out, q, [0, n], [n], F16, 128**-0.5)


def test_prompt_of_many_sequences(A, kernel):
    rng = random.Random(5)  # more than the 64 that a wave adds up at a time, empty ones among them
    new = [rng.choice([0, 0, 1, 2, 40]) for _ in range(150)]
    b = Batch(5, [n + rng.choice([0, 17]) for n in new], 16, 1, 64, F16)
    q = b.rows(sum(new), 2, F32)
    k, v, table, lengths = b.device()
    out = A.attention_prompt(q.cuda(), k, v, table, lengths, torch.tensor(_starts(new), dtype=torch.int32).cuda())
    _check_prompt(b, out, q, _starts(new), new, F32, 0.125)


def test_rows_of_nobody_stay_as_they_are(A, kernel):
    new = [3, 0, 4]
    b = Batch(7, [20, 5, 4], 16, 2, 64, F16)
    k, v, table, lengths = b.device()
    starts = torch.tensor([2, 5, 5, 9], dtype=torch.int32).cuda()  # two rows in front, three behind
    q = b.rows(12, 4, F32)
    q[:2], q[9:] = NAN, NAN
    out = torch.full((12, 4, 64), 7.0, device="cuda")
    A.attention_prompt(q.cuda(), k, v, table, lengths, starts, out=out)
    assert bool((out[:2] == 7).all()) and bool((out[9:] == 7).all())
    _check_prompt(b, out, q, [2, 5, 5], new, F32, 0.125)
    # ... and in append_rope: neither the rotated q nor the cache
    k2, v2 = k.clone(), v.clone()
    out.fill_(7.0)
    kk, vv = b.rows(12, 2, F32), b.rows(12, 2, F32)
    A.append_rope(q.cuda(), kk.cuda(), vv.cuda(), k2, v2, table, lengths, A.rope_turns(64), starts=starts, out=out)
    assert bool((out[:2] == 7).all()) and bool((out[9:] == 7).all())
    same = (k2.cpu() == b.k) | (k2.cpu().isnan() & b.k.isnan())
    same_v = (v2.cpu() == b.v) | (v2.cpu().isnan() & b.v.isnan())
    written = [(b.table[s][p // 16], p % 16) for s, n in enumerate(new) for p in range(b.lengths[s] - n, b.lengths[s])]
    for id in range(len(b.k)):
        for at in range(16):
            if (id, at) not in written:
                assert bool(same[id, :, at].all()) and bool(same_v[id, :, :, at].all())


@pytest.mark.parametrize("call", ["prompt", "decode"])
def test_pages_that_the_cache_does_not_have(A, kernel, call):
    lengths = [100, 40, 16, 90]
    b = Batch(9, lengths, 16, 2, 64, F16, extra_width=0)
    total = len(b.k)
    b.table[0][2], b.table[0][5], b.table[1][0], b.table[2][0], b.table[3][1] = -1, total, 2**31 - 1, -(2**31), total + 5
    b.lengths = lengths = [100, 40, 16, 16 * len(b.table[0]) + 50]  # the last one ends behind its table
    n = 3 if call == "prompt" else 1
    q = b.rows(4 * n, 4, F32)
    k, v, table, dl = b.device()
    if call == "prompt":
        out = A.attention_prompt(q.cuda(), k, v, table, dl, torch.tensor([0, 3, 6, 9, 12], dtype=torch.int32).cuda())
    else:
        out = A.attention_decode(q.cuda(), k, v, table, dl)
    # what lies on the pages of the fourth sequence behind its 90 keys was never written: NaN there, so leave it out of the test
    out = out.cpu()
    for s in range(3):
        kk, vv, there = b.keys(s, lengths[s])
        for i in range(n):
            seen = lengths[s] - n + i + 1
            _check(out[s * n + i], *R.attend(q[s * n + i], kk[:, :seen], vv[:, :seen], there[:seen], 0.125), F32, (s, i))
    assert bool((out[2 * n : 3 * n] == 0).all())  # no key at all


@pytest.mark.parametrize("length", [0, -5])
def test_sequences_without_keys_give_zeros(A, kernel, length):
    b = Batch(11, [10, 0, 40], 16, 1, 64, F16)
    b.lengths[1] = length
    k, v, table, lengths = b.device()
    q = b.rows(3, 4, F32)
    out = A.attention_decode(q.cuda(), k, v, table, lengths).cpu()
    assert bool((out[1] == 0).all())
    out = A.attention_prompt(q.cuda(), k, v, table, lengths, torch.arange(4, dtype=torch.int32).cuda()).cpu()
    assert bool((out[1] == 0).all())
    # a table without a single entry
    out = A.attention_decode(q.cuda(), k, v, table[:, :0].contiguous(), lengths)
    assert bool((out == 0).all())
    # rows in front of a sequence's first token
    out = A.attention_prompt(q.cuda(), k, v, table[:1].contiguous(), torch.tensor([1], dtype=torch.int32).cuda(), torch.tensor([0, 3], dtype=torch.int32).cuda()).cpu()
    assert bool((out[:2] == 0).all()) and bool((out[2] != 0).any())


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 64)])
def test_decode_ragged(A, dtype, cache, dim, page):
    lengths = [1, 2, 31, 32, 33, 0, 64, 127, 128, 129, 300, 700]
    b = Batch(13, lengths, page, 2, dim, cache)
    q = b.rows(len(lengths), 8, dtype)
    k, v, table, dl = b.device()
    out = A.attention_decode(q.cuda(), k, v, table, dl)
    assert out.dtype == dtype
    for s, n in enumerate(lengths):
        _check(out[s].cpu(), *R.attend(q[s], *b.keys(s, n), dim**-0.5), dtype, s)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (6, 2), (16, 1), (17, 1), (80, 2)])
def test_decode_groupings_and_pages(A, heads, kv_heads, page):
    lengths = [260, 5, 90]
    b = Batch(heads * page, lengths, page, kv_heads, 64, F16)
    q = b.rows(3, heads, F32)
    k, v, table, dl = b.device()
    out = A.attention_decode(q.cuda(), k, v, table, dl, scale=0.3)
    for s, n in enumerate(lengths):
        _check(out[s].cpu(), *R.attend(q[s], *b.keys(s, n), 0.3), F32, s)


@pytest.mark.parametrize("sequences", [65, 300])
def test_decode_of_many_sequences(A, sequences):
    rng = random.Random(sequences)
    lengths = [rng.choice([0, 1, 17, 64, 150]) for _ in range(sequences)]
    lengths[3] = 2000  # beside one that is much longer: cut into pieces
    b = Batch(17, lengths, 32, 1, 64, F16)
    q = b.rows(sequences, 4, F32)
    k, v, table, dl = b.device()
    out = A.attention_decode(q.cuda(), k, v, table, dl).cpu()
    for s in sorted({0, 3, 62, 63, 64, sequences - 1, *range(5, sequences, 17)}):
        _check(out[s], *R.attend(q[s], *b.keys(s, lengths[s]), 0.125), F32, s)


def test_decode_of_a_long_sequence(A):
    b = Batch(19, [30011], 256, 1, 64, F16)
    q = b.rows(1, 2, F32)
    k, v, table, dl = b.device()
    out = A.attention_decode(q.cuda(), k, v, table, dl).cpu()
    _check(out[0], *R.attend(q[0], *b.keys(0, 30011), 0.125), F32, 0)


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("dim,page,pages", [(64, 16, 1), (64, 16, 9), (128, 64, 3), (128, 256, 1)])
def test_decode_behind_a_shared_prefix(A, kernel, dtype, cache, dim, page, pages):
    prefix = page * pages
    own = [1, 0, 40, 100, 5, 33, 300, -3, -prefix, 64]  # negative: a sequence that ends inside the prefix, or has nothing
    b = Batch(23, [prefix + n for n in own], page, 2, dim, cache, shared=pages)
    q = b.rows(len(own), 8, dtype)
    k, v, table, dl = b.device()
    table[:, :pages] = 123456  # these entries are not looked at
    out = A.attention_decode(q.cuda(), k, v, table, dl, prefix_pages=torch.tensor(b.common, dtype=torch.int32).cuda()).cpu()
    plain = A.attention_decode(q.cuda(), k, v, torch.tensor(b.table, dtype=torch.int32).cuda(), dl).cpu()
    for s, n in enumerate(own):
        ref = R.attend(q[s], *b.keys(s, prefix + n, prefix=b.common), dim**-0.5)
        _check(out[s], *ref, dtype, s)
        _check(plain[s], *ref, dtype, ("not shared", s))


def test_prefix_of_many_rows_in_pieces(A, kernel):
    page, pages, n = 32, 40, 70  # 560 rows: five tiles; 1280 keys: several pieces
    own = [i % 37 for i in range(n)]
    b = Batch(29, [page * pages + x for x in own], page, 1, 64, F16, shared=pages)
    q = b.rows(n, 8, F32)
    k, v, table, dl = b.device()
    prefix = torch.tensor(b.common, dtype=torch.int32).cuda()
    out = A.attention_decode(q.cuda(), k, v, table, dl, prefix_pages=prefix).cpu()
    for s in range(0, n, 9):
        _check(out[s], *R.attend(q[s], *b.keys(s, page * pages + own[s]), 0.125), F32, s)
    # a prefix page that the cache does not have is left out
    broken = list(b.common)
    broken[7] = -1
    out = A.attention_decode(q.cuda(), k, v, table, dl, prefix_pages=torch.tensor(broken, dtype=torch.int32).cuda()).cpu()
    for s in (0, 33, 69):
        _check(out[s], *R.attend(q[s], *b.keys(s, page * pages + own[s], prefix=broken), 0.125), F32, s)
    # ... and an empty list shares nothing
    same = A.attention_decode(q.cuda(), k, v, table, dl, prefix_pages=prefix[:0])
    assert torch.equal(same, A.attention_decode(q.cuda(), k, v, table, dl))


@pytest.mark.parametrize("std", [1e-30, 1e-6, 300.0, 1e6])
def test_sizes_of_q(A, kernel, std):
    # fp32 q goes through fp16 terms: neither what fp16 cannot hold nor its small numbers may show
    b = Batch(31, [150], 16, 1, 64, F16)
    q = b.rows(150, 4, F32, std=std)
    k, v, table, dl = b.device()
    scale = 0.125 / max(std, 1.0)
    out = A.attention_prompt(q.cuda(), k, v, table, dl, torch.tensor([0, 150], dtype=torch.int32).cuda(), scale=scale)
    _check_prompt(b, out, q, [0, 150], [150], F32, scale)
    out = A.attention_decode(q[:1].cuda(), k, v, table, dl, scale=scale).cpu()
    _check(out[0], *R.attend(q[0], *b.keys(0, 150), scale), F32, 0)


@pytest.mark.parametrize("cache", [F16, BF16])
def test_peaked_and_flat_scores(A, kernel, cache):
    b = Batch(37, [400], 32, 1, 64, cache)
    k, v, table, dl = b.device()
    for std, dtype in ((60.0, F32), (0.0, F32), (60.0, cache)):
        q = b.rows(400, 2, dtype, std=std)
        out = A.attention_prompt(q.cuda(), k, v, table, dl, torch.tensor([0, 400], dtype=torch.int32).cuda())
        _check_prompt(b, out, q, [0, 400], [400], dtype, 0.125)
        out = A.attention_decode(q[:1].cuda(), k, v, table, dl).cpu()
        _check(out[0], *R.attend(q[0], *b.keys(0, 400), 0.125), dtype, std)


def test_strided_rows_and_in_place(A, kernel):
    # q, k and v as parts of one fused projection
    b = Batch(41, [50, 20], 16, 2, 64, F16)
    k, v, table, dl = b.device()
    starts = torch.tensor([0, 30, 45], dtype=torch.int32).cuda()
    fused = torch.randn(45, 8 + 2 + 2, 64, generator=b.g).cuda()
    q, kk, vv = fused[:, :8], fused[:, 8:10], fused[:, 10:]
    turns = A.rope_turns(64)
    k2, v2 = k.clone(), v.clone()
    got = A.append_rope(q, kk, vv, k, v, table, dl, turns, starts=starts)
    whole = A.append_rope(q.contiguous(), kk.contiguous(), vv.contiguous(), k2, v2, table, dl, turns, starts=starts)
    assert torch.equal(got, whole) and torch.equal(k.view(torch.int16), k2.view(torch.int16)) and torch.equal(v.view(torch.int16), v2.view(torch.int16))
    mine = q.contiguous()
    assert A.append_rope(mine, kk, vv, k2, v2, table, dl, turns, starts=starts, out=mine) is mine and torch.equal(mine, whole)
    assert torch.equal(A.attention_prompt(q, k, v, table, dl, starts), A.attention_prompt(q.contiguous(), k, v, table, dl, starts))
    assert torch.equal(A.attention_decode(q[:2], k, v, table, dl), A.attention_decode(q[:2].contiguous(), k, v, table, dl))
    for bad in (fused.transpose(0, 1), fused[:, ::2], fused[..., :32], fused.double()):
        with pytest.raises((TypeError, ValueError)):
            A.attention_prompt(bad, k, v, table, dl, starts)
    from nihilus_amd import Q8Error

    with pytest.raises(Q8Error):  # rows that do not start on 16 bytes
        A.attention_prompt(torch.zeros(45 * 513, device="cuda").as_strided((45, 8, 64), (513, 64, 1)), k, v, table, dl, starts)


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (128, 128), (128, 32), (64, 0)])
def test_append_rope(A, dtype, cache, interleaved, dim, rotary):
    new, cached = [1, 0, 70, 5], [0, 9, 13, 100000]
    b = Batch(43, [n + min(c, 100) for n, c in zip(new, cached)], 16, 2, dim, cache)
    # the last sequence stands at a far position: its table has the last pages only
    lengths = [n + c for n, c in zip(new, cached)]
    width = -(-max(lengths) // 16)
    table = torch.full((4, width), -1, dtype=torch.int32)
    for s in range(4):
        for j in range(-(-lengths[s] // 16)):
            table[s, j] = b.table[s][j % len(b.table[s])] if s < 3 else b.table[s][j - (-(-lengths[s] // 16)) + 2] if j >= -(-lengths[s] // 16) - 2 else -1
    rows = sum(new)
    q, k, v = b.rows(rows, 6, dtype), b.rows(rows, 2, dtype), b.rows(rows, 2, dtype)
    kp, vp, _, _ = b.device()
    base, factors = 500000.0, [1.0 + 0.5 * i for i in range(rotary // 2)]
    turns = A.rope_turns(dim, base=base, factors=factors, rotary=rotary)
    out = A.append_rope(q.cuda(), k.cuda(), v.cuda(), kp, vp, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), turns,
                        starts=torch.tensor(_starts(new), dtype=torch.int32).cuda(), interleaved=interleaved)
    assert out.dtype == dtype
    out, kp, vp = out.cpu().double(), kp.cpu().double(), vp.cpu().double()
    inverse = [base ** (-2.0 * i / max(rotary, 1)) / factors[i] for i in range(rotary // 2)]

    def check(got, x, pos, kind):
        ref, size = R.rope(x, pos, inverse, interleaved)
        # angle 2 pi 2^-26, sine and cosine 2 ulp, two products and a sum: 4e-7 < 2^-21 of |a| + |b|; then one rounding
        most = size * 2.0**-21
        most = most + R.half_step(kind) * (ref.abs() + most) + R.tiny(kind)
        assert bool(((got - ref).abs() <= most).all()), (pos, float(((got - ref).abs() - most).max()))

    for s, n in enumerate(new):
        for i in range(n):
            r, pos = _starts(new)[s] + i, lengths[s] - n + i
            id, at = int(table[s, pos // 16]), pos % 16
            check(out[r], q[r], pos, dtype)
            check(kp[id, :, at], k[r], pos, cache)
            assert torch.equal(vp[id, :, :, at], v[r].to(cache).double())


def test_append_one_row_per_sequence(A):
    lengths = [1, 16, 17, 33, 0, 64]  # the fifth has no place for its row
    b = Batch(47, lengths, 16, 8, 128, F16)
    q, k, v = b.rows(6, 32, F32), b.rows(6, 8, F32), b.rows(6, 8, F32)
    kp, vp, table, dl = b.device()
    turns = A.rope_turns(128)
    out = A.append_rope(q.cuda(), k.cuda(), v.cuda(), kp, vp, table, dl, turns)
    kp2, vp2, _, _ = b.device()
    same = A.append_rope(q.cuda(), k.cuda(), v.cuda(), kp2, vp2, table, dl, turns, starts=torch.arange(7, dtype=torch.int32).cuda())
    assert torch.equal(out, same) and torch.equal(kp.view(torch.int16), kp2.view(torch.int16)) and torch.equal(vp.view(torch.int16), vp2.view(torch.int16))
    for s, n in enumerate(lengths):
        if n:
            id, at = b.table[s][(n - 1) // 16], (n - 1) % 16
            assert torch.equal(vp[id, :, :, at].cpu(), v[s].to(F16))
    changed = (vp.cpu().view(torch.int16) != b.v.view(torch.int16)).flatten(1).any(1)
    assert sorted(torch.nonzero(changed).flatten().tolist()) == sorted(b.table[s][(n - 1) // 16] for s, n in enumerate(lengths) if n)


def test_offsets_past_32_bits(A, kernel):
    # pages behind 2^32 bytes and 2^31 values of the cache
    pages, page, heads, dim = 20000, 256, 8, 128  # 2^18 values of K each: 10.5 GB
    k, v = A.empty_cache(1, pages, heads, page, dim)
    k, v = k[0], v[0]
    ids = torch.tensor([[19999, 9000, 16500]], dtype=torch.int32).cuda()
    gen = torch.Generator(device="cuda").manual_seed(1)
    for id in ids[0].tolist():
        k[id].normal_(generator=gen)
        v[id].normal_(generator=gen)
    q = torch.randn(3, 8, dim, generator=gen, device="cuda")
    lengths = torch.tensor([700], dtype=torch.int32).cuda()
    out = A.attention_decode(q[:1], k, v, ids, lengths)
    small = A.attention_decode(q[:1], k[ids[0].long()].contiguous(), v[ids[0].long()].contiguous(), torch.arange(3, dtype=torch.int32).cuda()[None], lengths)
    assert torch.equal(out, small)
    starts = torch.tensor([0, 3], dtype=torch.int32).cuda()
    out = A.attention_prompt(q, k, v, ids, lengths, starts)
    small = A.attention_prompt(q, k[ids[0].long()].contiguous(), v[ids[0].long()].contiguous(), torch.arange(3, dtype=torch.int32).cuda()[None], lengths, starts)
    assert torch.equal(out, small)
    x = torch.randn(3, 8, dim, generator=gen, device="cuda")
    A.append_rope(q, x, x, k, v, ids, lengths, A.rope_turns(dim), starts=starts)
    assert torch.equal(v[16500, :, :, 697 - 512 : 700 - 512], x.to(F16).permute(1, 2, 0))


def test_streams_and_captured_graphs(A, kernel):
    # replays with new inputs, eager calls between them, a second graph with a workspace of its own on another stream
    lengths = [700, 33, 1, 260]
    b = Batch(53, lengths, 32, 2, 128, F16, shared=0)
    k, v, table, dl = b.device()
    starts = torch.tensor([0, 3, 4, 5, 9], dtype=torch.int32).cuda()
    q, kk, vv = (torch.empty(n, h, 128, device="cuda") for n, h in ((9, 8), (9, 2), (9, 2)))
    turns = A.rope_turns(128)

    def step(ws):
        r = A.append_rope(q, kk, vv, k, v, table, dl, turns, starts=starts)
        return r, A.attention_prompt(r, k, v, table, dl, starts), A.attention_decode(r[:4].contiguous(), k, v, table, dl, workspace=ws), *A.cache_step(k[None], v[None], table, dl, parents, grow)

    parents, grow = torch.tensor([0, 0, 3, -1], dtype=torch.int32).cuda(), torch.tensor([1, 1, 1, 1], dtype=torch.int32).cuda()

    def fill(seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for t in (q, kk, vv):
            t.normal_(generator=gen)

    spaces = [A.decode_workspace(4, 8, 2, 128, page_size=32) for _ in range(3)]
    fill(0)
    step(spaces[0])
    torch.cuda.synchronize()
    graphs = []
    for ws in spaces[1:]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(ws)
        graphs.append((g, outs))
    side = torch.cuda.Stream()
    for seed in range(1, 5):
        fill(seed)
        torch.cuda.synchronize()
        graphs[0][0].replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        side.synchronize()
        want = step(spaces[0])
        torch.cuda.synchronize()
        for _, outs in graphs:
            for got, ref in zip(outs, want):
                assert torch.equal(got, ref), seed


def test_two_streams_at_once(A):
    b = Batch(59, [3000, 50, 900], 64, 2, 128, F16)
    k, v, table, dl = b.device()
    q = [b.rows(3, 8, F32).cuda() for _ in range(2)]
    want = [A.attention_decode(x, k, v, table, dl) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in q]
    got = [[] for _ in q]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(A.attention_decode(q[i], k, v, table, dl))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_the_two_prompt_kernels_agree(A, monkeypatch):
    # a chunk of few rows behind long cached parts: pieces on one side, tiles on the other
    new, cached = [5, 1, 40, 0], [3000, 0, 700, 50]
    b = Batch(73, [n + c for n, c in zip(new, cached)], 32, 2, 128, F16)
    q = b.rows(sum(new), 8, F32).cuda()
    k, v, table, dl = b.device()
    starts = torch.tensor(_starts(new), dtype=torch.int32).cuda()
    monkeypatch.setenv("NH_Q8_0_DEBUG_HOOKS", "1")
    force = A._lib.lib().nh_attn_debug_prompt_kernel
    got = []
    try:
        for which in (1, 2):
            force(1, 1, 1, 1, which)
            got.append(A.attention_prompt(q, k, v, table, dl, starts))
    finally:
        force(1, 1, 1, 1, 0)
    _check_prompt(b, got[0], q.cpu(), _starts(new), new, F32, 128**-0.5)
    _check_prompt(b, got[1], q.cpu(), _starts(new), new, F32, 128**-0.5)


@pytest.mark.parametrize("graph", [False, True])
def test_counters_are_left_zero(A, graph):
    b = Batch(79, [3000, 900, 1, 0, 257], 32, 2, 64, F16)
    k, v, table, dl = b.device()
    q = b.rows(5, 8, F32).cuda()
    ws = A.decode_workspace(5, 8, 2, 64)
    want = A.attention_decode(q, k, v, table, dl)
    if graph:
        A.attention_decode(q, k, v, table, dl, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = A.attention_decode(q, k, v, table, dl, workspace=ws)
            own = A.attention_decode(q, k, v, table, dl)
        for _ in range(4):
            out.zero_(), own.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(own, want) and not bool(ws.counters.any())
    for _ in range(3):
        assert torch.equal(A.attention_decode(q, k, v, table, dl, workspace=ws), want)
    assert not bool(ws.counters.any())


def test_same_bits_every_time(A):
    b = Batch(61, [2500, 700, 31], 16, 2, 128, F16)
    k, v, table, dl = b.device()
    q = b.rows(3, 8, F32).cuda()
    first = A.attention_decode(q, k, v, table, dl)
    assert all(torch.equal(first, A.attention_decode(q, k, v, table, dl)) for _ in range(10))
    # a sequence's result does not hang on how the rows of the table behind its pages look
    table[1, -1] = 5
    assert torch.equal(first, A.attention_decode(q, k, v, table, dl))


def test_prompt_and_decode_agree(A, kernel):
    # a sequence written token by token and decoded gives what the same sequence in one prompt gives
    n, heads, kv_heads, dim, page = 70, 4, 2, 64, 16
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(n, h, dim, generator=gen, device="cuda") for h in (heads, kv_heads, kv_heads))
    turns = A.rope_turns(dim)
    table = torch.randperm(8, generator=torch.Generator().manual_seed(1)).to(torch.int32)[None].cuda()
    caches = [tuple(t[0] for t in A.empty_cache(1, 8, kv_heads, page, dim)) for _ in range(2)]
    starts = torch.tensor([0, n], dtype=torch.int32).cuda()
    full = torch.tensor([n], dtype=torch.int32).cuda()
    whole = A.attention_prompt(A.append_rope(q, k, v, *caches[0], table, full, turns, starts=starts), *caches[0], table, full, starts)
    for i in range(n):
        at = torch.tensor([i + 1], dtype=torch.int32).cuda()
        r = A.append_rope(q[i : i + 1], k[i : i + 1], v[i : i + 1], *caches[1], table, at, turns)
        one = A.attention_decode(r, *caches[1], table, at)
        # each is within 1e-5 of the exact result (fp32, 70 keys, scores of a few units: the bound of attention_reference.py)
        assert float((one[0] - whole[i]).abs().max()) < 2e-5 * float(v.abs().max()), i
    used = [int(p) for p in table[0, : -(-n // page)]]
    for id in used[:-1]:
        assert torch.equal(caches[0][0][id], caches[1][0][id]) and torch.equal(caches[0][1][id], caches[1][1][id])


def test_native_calls_and_the_python_way_agree(A, monkeypatch):
    # the same bits either way, and the native calls are the ones that run
    b = Batch(67, [50, 0, 90], 16, 2, 64, F16)
    q, kk, vv = (b.rows(40, h, F32).cuda() for h in (8, 2, 2))
    starts, turns = torch.tensor([0, 30, 30, 40], dtype=torch.int32).cuda(), A.rope_turns(64)
    parents, grow = torch.tensor([0, 0, 2], dtype=torch.int32).cuda(), torch.tensor([1, 1, -2], dtype=torch.int32).cuda()
    k0, v0, table, dl = b.device()

    def calls():
        k, v = k0.clone(), v0.clone()
        r = A.append_rope(q, kk, vv, k, v, table, dl, turns, starts=starts, interleaved=False)
        res = [r, A.attention_prompt(r, k, v, table, dl, starts, scale=0.2), A.attention_decode(r[:3], k, v, table, dl), A.attention_decode(r[:3], k, v, table, dl, prefix_pages=table[0, :1].contiguous()),
               *A.cache_step(k[None], v[None], table, dl, parents, grow), *A.cache_compact(k[None], v[None], table, dl)]
        return [*res, k.view(torch.int16), v.view(torch.int16)]

    names = ["append_rope", "attention_prompt", "attention_decode", "cache_step", "cache_compact"]
    ran = []
    real = A._calls
    assert real is not None

    class Seen:
        def __getattr__(self, name):
            def call(*args):
                r = getattr(real, name)(*args)
                ran.append((name, r is not None))
                return r

            return call

    monkeypatch.setattr(A, "_calls", Seen())
    native = calls()
    assert {n for n, ok in ran if ok} == set(names) and all(ok for _, ok in ran)
    monkeypatch.setattr(A, "_calls", None)
    assert all(torch.equal(x, y) for x, y in zip(native, calls()))


@pytest.mark.parametrize("native", [True, False])
def test_tensors_that_are_refused(A, monkeypatch, native):
    if not native:
        monkeypatch.setattr(A, "_calls", None)
    b = Batch(71, [20, 5], 16, 2, 64, F16)
    k, v, table, dl = b.device()
    q, turns, starts = b.rows(2, 4, F32).cuda(), A.rope_turns(64), torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    kv = b.rows(2, 2, F32).cuda()
    A.attention_decode(q, k, v, table, dl)
    errors = (TypeError, ValueError, RuntimeError)
    for args in [(q, k, v.float(), table, dl), (q, k, v.transpose(-1, -2), table, dl), (q, k, v[:-1], table, dl), (q, k, k, table, dl), (q, k, v, table.long(), dl), (q, k, v, table[0], dl),
                 (q, k, v, table, dl[:1]), (q, k, v, table.cpu(), dl), (q, k, v, table, dl.cpu()), (q.cpu(), k, v, table, dl), (q.to(BF16), k, v, table, dl), (q[:1], k, v, table, dl),
                 (q[:, :3], k, v, table, dl), (q[:, :, :32], k, v, table, dl), (q.reshape(2, -1), k, v, table, dl), (q, k[None], v[None], table, dl), (q, k.to(BF16), v, table, dl),
                 (q, k, v, table.t().contiguous().t(), dl)]:
        with pytest.raises(errors):
            A.attention_decode(*args)
        if args[0].shape[0] == 2:  # (rows that are not there are nobody's for a prompt)
            with pytest.raises(errors):
                A.attention_prompt(*args, starts)
    for s in (starts[:2], starts.long(), starts.cpu(), None):
        with pytest.raises(errors + (AttributeError,)):
            A.attention_prompt(q, k, v, table, dl, s)
    for scale in (0.0, -0.1, float("inf"), float("nan")):
        with pytest.raises(errors):
            A.attention_decode(q, k, v, table, dl, scale=scale)
    with pytest.raises(errors):
        A.attention_decode(q, k, v, table, dl, prefix_pages=table[0].long())
    with pytest.raises(errors):
        A.attention_decode(q, k, v, table, dl, workspace=A.decode_workspace(1, 2, 2, 64))  # too small
    for out in (q[:1], q.half(), q.cpu(), torch.empty(2, 64, 4, device="cuda").transpose(1, 2)):
        with pytest.raises(errors):
            A.attention_decode(q, k, v, table, dl, out=out)
    for bad in [(q, kv[:1], kv), (q, kv, kv.half()), (q, kv[:, :1], kv), (q, kv, kv.cpu()), (q.half(), kv, kv)]:
        with pytest.raises(errors):
            A.append_rope(*bad, k, v, table, dl, turns)
    for t in (turns.float(), turns.cpu(), turns[:12], turns[None], A.rope_turns(128)):
        with pytest.raises(errors):
            A.append_rope(q, kv, kv, k, v, table, dl, t)
    parents = torch.zeros(2, dtype=torch.int32).cuda()
    for args in [(k, v, table, dl, parents, parents), (k[None], v[None], table, dl, parents, parents[:1]), (k[None], v[None], table, dl, parents.long(), parents),
                 (k[None], v[None], table, dl, parents[None], parents)]:
        with pytest.raises(errors):
            A.cache_step(*args)
    with pytest.raises(errors):
        A.cache_compact(k, v, table, dl)


def _check_with_odd_values(got, q, k, v, there, scale, dtype, what):
    """Values that are infinite or NaN reach the rows that see their keys, in their column, and no others."""
    clean = torch.where(torch.isfinite(v), v, 0.0)
    ref, mean, d, n = R.attend(q, k, clean, there, scale)
    group = q.shape[0] // k.shape[0]
    odd = torch.where(torch.isfinite(v), 0.0, v)[:, there].sum(1).repeat_interleave(group, 0)  # [heads, dim]: 0, an infinity or NaN
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(odd)) and torch.equal(torch.isinf(got), torch.isinf(odd)), what
    assert torch.equal(got[torch.isinf(odd)], odd[torch.isinf(odd)]), what
    _check(torch.where(odd == 0, got, ref), ref, mean, d, n, dtype, what)


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_odd_values_of_later_rows(A, kernel, dtype, cache, dim, page):
    new, cached = [70, 3, 200], [20, 0, 65]
    b = Batch(17, [a + c for a, c in zip(new, cached)], page, 2, dim, cache)
    for seq, places in enumerate([[(25, 0, INF), (26, 0, -INF), (40, 1, NAN), (63, 5, INF), (64, 6, -INF), (89, 7, NAN)], [(2, 3, INF)], [(66, 9, -INF), (200, 9, INF), (201, 40, NAN), (264, 63, INF)]]):
        for j, d, x in places:
            b.v[b.table[seq][j // page], seq % 2, d, j % page] = x
    starts = _starts(new)
    q = b.rows(sum(new), 4, dtype)
    k, v, table, lengths = b.device()
    out = A.attention_prompt(q.cuda(), k, v, table, lengths, torch.tensor(starts, dtype=torch.int32).cuda()).cpu()
    for seq, n in enumerate(new):
        keys, values, there = b.keys(seq, b.lengths[seq])
        for i in range(n):
            seen = cached[seq] + i + 1
            _check_with_odd_values(out[starts[seq] + i], q[starts[seq] + i], keys[:, :seen], values[:, :seen], there[:seen], dim**-0.5, dtype, (seq, i))


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_odd_values_in_a_prefix_that_some_rows_see_in_part(A, kernel, dtype, cache, dim):
    page, pages = 16, 9
    lengths = [300, 144, 150, 17, 40, 100, 0, -(2**31), 129, 128]
    b = Batch(23, lengths, page, 2, dim, cache, shared=pages)
    for j, d, x in [(16, 0, INF), (30, 0, -INF), (39, 2, NAN), (40, 3, INF), (99, 4, -INF), (128, 5, NAN), (143, 6, INF)]:
        b.v[b.common[j // page], j % 2, d, j % page] = x
    q = b.rows(len(lengths), 8, dtype)
    k, v, table, n = b.device()
    out = A.attention_decode(q.cuda(), k, v, table, n, prefix_pages=torch.tensor(b.common, dtype=torch.int32).cuda()).cpu()
    for seq, length in enumerate(lengths):
        keys, values, there = b.keys(seq, max(length, 0), b.common)
        _check_with_odd_values(out[seq], q[seq], keys, values, there, dim**-0.5, dtype, seq)


def test_a_stretch_of_many_small_pages(A):
    lengths = [20011, 3]  # pages of 16 keys: a workgroup's stretch has more of them than a wave holds in a register
    b = Batch(29, lengths, 16, 64, 64, F16)
    q = b.rows(2, 64, F16)
    k, v, table, n = b.device()
    out = A.attention_decode(q.cuda(), k, v, table, n).cpu()
    for seq, length in enumerate(lengths):
        ref = R.attend(q[seq], *b.keys(seq, length), 0.125)
        _check(out[seq], *ref, F16, seq)


def test_decode_behind_a_prefix_replayed(A, kernel):
    lengths = [700, 64, 65, 130, 256]
    b = Batch(31, lengths, 64, 2, 128, F16, shared=1)
    q = b.rows(5, 8, F32)
    k, v, table, n = b.device()
    x, prefix = q.cuda(), torch.tensor(b.common, dtype=torch.int32).cuda()
    out = torch.empty_like(x)
    space = A.decode_workspace(5, 8, 2, 128, prefix_pages=1, page_size=64)
    A.attention_decode(x, k, v, table, n, prefix_pages=prefix, out=out, workspace=space)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.attention_decode(x, k, v, table, n, prefix_pages=prefix, out=out, workspace=space)
    for turn in range(3):
        q = b.rows(5, 8, F32)
        x.copy_(q)
        out.fill_(NAN)
        graph.replay()
        got = out.cpu()
        eager = A.attention_decode(x, k, v, table, n, prefix_pages=prefix).cpu()
        assert torch.equal(got, eager)
        for seq, length in enumerate(lengths):
            _check(got[seq], *R.attend(q[seq], *b.keys(seq, length, b.common), 128**-0.5), F32, (turn, seq))


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_few_rows_behind_long_caches(A, kernel, dtype, cache, dim, page):
    # tiles whose keys are cut into pieces, and others, in one call; twice, for the counters; the same bits each time
    new, cached = [5, 40, 1, 130, 0], [4000, 0, 700, 1100, 2000]
    b = Batch(37, [a + c for a, c in zip(new, cached)], page, 1, dim, cache)
    b.v[b.table[0][3990 // page], 0, 7, 3990 % page] = -INF
    b.v[b.table[3][1200 // page], 0, 9, 1200 % page] = NAN
    starts = _starts(new)
    q = b.rows(sum(new), 4, dtype)
    k, v, table, lengths = b.device()
    x, at = q.cuda(), torch.tensor(starts, dtype=torch.int32).cuda()
    space = A.prompt_workspace(sum(new), len(new), 4, 1, dim)
    first = A.attention_prompt(x, k, v, table, lengths, at, workspace=space)
    for _ in range(3):
        again = A.attention_prompt(x, k, v, table, lengths, at, workspace=space)
        assert torch.equal(again.view(torch.int16), first.view(torch.int16))
        assert int(space.counters.abs().sum()) == 0
    first = first.cpu()
    for seq, n in enumerate(new):
        keys, values, there = b.keys(seq, b.lengths[seq])
        for i in sorted({0, n // 2, n - 1} & set(range(n))):
            seen = cached[seq] + i + 1
            _check_with_odd_values(first[starts[seq] + i], q[starts[seq] + i], keys[:, :seen], values[:, :seen], there[:seen], dim**-0.5, dtype, (seq, i))
