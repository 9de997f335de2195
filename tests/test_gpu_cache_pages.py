"""GPU: the paged cache from one step to the next and its compaction, against the bookkeeping of attention_reference.py (plain Python on page numbers): tables,
counts and the bytes of every page."""
import random

import pytest
import torch

import attention_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A():
    from nihilus_amd import attention

    attention._lib.lib()
    return attention


def _cache(A, seed, layers, pages, heads, page, dim, dtype=torch.float16):
    k, v = A.empty_cache(layers, pages, heads, page, dim, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    k.view(torch.int16).random_(-30000, 30000, generator=g)
    v.view(torch.int16).random_(-30000, 30000, generator=g)
    return k, v


def _dev(x, shape=None):
    t = torch.tensor(x, dtype=torch.int32)
    return (t if shape is None else t.reshape(shape)).cuda()


def _moved(t, moves):
    t = t.clone()
    for src, dst in moves:
        t[:, dst] = t[:, src]
    return t


def _bits(t):
    return t.view(torch.int16)


def _step(A, k, v, table, lengths, parents, grow):
    width = len(table[0]) if table else 0
    pages, page = k.shape[1], k.shape[3]
    want = R.step(table, lengths, parents, grow, pages, page)
    k0, v0 = k.clone(), v.clone()
    d_table, d_lengths = _dev(table, (len(table), width)), _dev(lengths)
    new, now, info = A.cache_step(k, v, d_table, d_lengths, _dev(parents), _dev(grow))
    assert new.tolist() == want[0] and now.tolist() == want[1] and info.tolist() == want[2]
    assert torch.equal(_bits(k), _bits(_moved(k0, want[3]))) and torch.equal(_bits(v), _bits(_moved(v0, want[3])))
    assert d_table.tolist() == table and d_lengths.tolist() == lengths
    return new.tolist(), now.tolist(), info.tolist()


def _state(rng, sequences, page, longest, pages, width=None):
    lengths = [rng.randint(0, longest) for _ in range(sequences)]
    order = list(range(pages))
    rng.shuffle(order)
    width = -(-longest // page) + 2 if width is None else width
    table = []
    for n in lengths:
        c = -(-n // page)
        table.append([order.pop() for _ in range(c)] + [-1] * (width - c))
    return table, lengths


@pytest.mark.parametrize("seed", range(12))
def test_step_over_many_steps(A, seed):
    # sequences that go on, fork, end, shrink and grow, step after step on the tables that the last step gave; now and then no page is left
    rng = random.Random(seed)
    page = rng.choice([16, 32, 64])
    sequences, longest = rng.choice([1, 3, 17, 40]), rng.choice([10, 100, 300])
    need = sequences * (-(-longest // page))
    pages = need + rng.choice([0, 3, 50])
    k, v = _cache(A, seed, rng.choice([1, 3]), max(pages, 1), rng.choice([1, 2]), page, 64)
    table, lengths = _state(rng, sequences, page, longest, max(pages, 1))
    for _ in range(6):
        children = rng.choice([sequences, sequences, 1, 2 * sequences])
        parents = [rng.choice([-1, rng.randrange(len(table)), rng.randrange(len(table)), rng.randrange(len(table)), len(table), -7]) if rng.random() < 0.3 else rng.randrange(len(table))
                   for _ in range(children)]
        grow = [rng.choice([1, 1, 1, 0, -1, -20, 5, 70]) for _ in range(children)]
        table, lengths, _ = _step(A, k, v, table, lengths, parents, grow)


def test_step_shares_full_pages_and_copies_the_open_one(A):
    k, v = _cache(A, 1, 2, 12, 2, 16, 64)
    # one sequence of 40 tokens: pages 5, 6 full, 7 open
    new, now, info = _step(A, k, v, [[5, 6, 7, -1]], [40], [0, 0, 0], [1, 1, 0])
    assert new == [[5, 6, 7, -1], [5, 6, 0, -1], [5, 6, 1, -1]] and now == [41, 41, 40] and info == [5, 2, 0]
    # a child that goes back into a page that another holds in full gets a copy of it
    new, _, info = _step(A, k, v, [[5, 6, 7, -1]], [40], [0, 0], [1, -30])
    assert new == [[5, 6, 7, -1], [0, -1, -1, -1]] and info == [4, 1, 0]
    # exactly full pages: nothing is open, growth takes a page of its own
    new, _, info = _step(A, k, v, [[5, 6, -1]], [32], [0, 0], [1, 1])
    assert new == [[5, 6, 0], [5, 6, 1]] and info == [4, 0, 0]
    # two sequences that share an open page from before (by hand): the lower one keeps it
    new, _, info = _step(A, k, v, [[5, 6], [5, 6]], [20, 20], [1, 0], [1, 1])
    assert new == [[5, 6], [5, 0]] and info == [3, 1, 0]


def test_step_edges(A):
    k, v = _cache(A, 2, 1, 5, 1, 16, 64)
    # nobody goes on: everything is free
    assert _step(A, k, v, [[0, 1], [2, -1]], [20, 3], [-1, -1], [5, 5])[2] == [0, 0, 0]
    # no children, no sequences
    assert _step(A, k, v, [[0, 1]], [20], [], [])[2] == [0, 0, 0]
    new, now, info = A.cache_step(k, v, torch.empty((0, 4), dtype=torch.int32, device="cuda"), _dev([]), _dev([0, -1]), _dev([9, 9]))
    assert new.tolist() == [[-1] * 4] * 2 and now.tolist() == [0, 0] and info.tolist() == [0, 0, 0]
    # too few pages: the lowest children get theirs; growth stops at the table's end
    new, now, info = _step(A, k, v, [[0, 1, -1, -1]], [32], [0, 0, 0], [32, 32, 1000])
    assert info[2] == 3 and now == [64, 64, 64] and new[0] == [0, 1, 2, 3] and new[1] == [0, 1, 4, -1]
    # pages that the cache does not have are counted and stay missing
    new, _, info = _step(A, k, v, [[0, 9, -4, -1]], [40], [0, 0], [1, 1])
    assert new == [[0, -1, -1, -1]] * 2 and info == [1, 0, 4]
    # lengths that are none
    _step(A, k, v, [[0, 1], [2, 3]], [-5, 1000], [0, 1, 1], [3, -2, 2**31 - 1])
    _step(A, k, v, [[0, 1], [2, 3]], [20, 32], [0, 1], [-(2**31), -(2**31)])
    # a sequence that names a page twice
    _step(A, k, v, [[3, 3, 3]], [40], [0, 0], [1, 1])


@pytest.mark.parametrize("pages", [9000, 70000])
def test_step_of_a_large_cache_and_many_children(A, pages):
    rng = random.Random(pages)
    k, v = _cache(A, 3, 1, pages, 1, 16, 64)
    table, lengths = _state(rng, 1200, 16, 100, pages)
    parents = [rng.randrange(1200) for _ in range(1500)]
    _step(A, k, v, table, lengths, parents, [rng.choice([1, 0, 16, -3]) for _ in parents])


@pytest.mark.parametrize("seed", range(8))
def test_compact(A, seed):
    rng = random.Random(seed)
    page = rng.choice([16, 64])
    sequences = rng.choice([1, 5, 30])
    pages = sequences * 8 + rng.choice([1, 20])
    k, v = _cache(A, seed, 3, pages, 2, page, 128 if seed % 2 else 64, dtype=torch.bfloat16)
    table, lengths = _state(rng, sequences, page, 8 * page, pages)
    for s in range(0, sequences, 3):
        lengths[s] = rng.choice([0, lengths[s] // 2])  # ended or cut short: what the table still names is not held
    if sequences > 4:  # shared pages
        lengths[1] = lengths[2] = 5 * page
        table[1][:5] = table[2][:5] = [p for p in range(pages - 1, -1, -1) if not any(p in row for row in table)][:5]
    want = R.compact(table, lengths, pages, page)
    k0, v0 = k.clone(), v.clone()
    new, info = A.cache_compact(k, v, _dev(table), _dev(lengths))
    assert new.tolist() == want[0] and info.tolist() == want[1]
    assert torch.equal(_bits(k), _bits(_moved(k0, want[2]))) and torch.equal(_bits(v), _bits(_moved(v0, want[2])))
    again, info = A.cache_compact(k, v, new, _dev(lengths))  # nothing is left to move
    assert again.tolist() == want[0] and info.tolist() == [want[1][0], 0, 0]


def test_compact_edges(A):
    k, v = _cache(A, 4, 2, 6, 1, 16, 64)
    k0 = k.clone()
    new, info = A.cache_compact(k, v, _dev([[3, 9, -1]]), _dev([48]))
    assert new.tolist() == [[0, -1, -1]] and info.tolist() == [1, 1, 2] and torch.equal(_bits(k[:, 0]), _bits(k0[:, 3]))
    new, info = A.cache_compact(k, v, torch.empty((0, 3), dtype=torch.int32, device="cuda"), _dev([]))
    assert new.shape == (0, 3) and info.tolist() == [0, 0, 0]
    new, info = A.cache_compact(k, v, _dev([[5, 4, 3, 2, 1, 0]]), _dev([96]))  # full: nothing moves
    assert new.tolist() == [[5, 4, 3, 2, 1, 0]] and info.tolist() == [6, 0, 0]
    new, info = A.cache_compact(k, v, _dev([[5, 4]]), _dev([-3]))
    assert new.tolist() == [[-1, -1]] and info.tolist() == [0, 0, 0]


def test_a_large_cache_is_compacted(A):
    rng = random.Random(9)
    pages = 40000
    k, v = _cache(A, 5, 1, pages, 1, 16, 64)
    table, lengths = _state(rng, 700, 16, 600, pages)
    want = R.compact(table, lengths, pages, 16)
    k0, v0 = k.clone(), v.clone()
    new, info = A.cache_compact(k, v, _dev(table), _dev(lengths))
    assert new.tolist() == want[0] and info.tolist() == want[1] and want[1][1] > 1000
    src, dst = _dev([m[0] for m in want[2]]).long(), _dev([m[1] for m in want[2]]).long()
    k0[:, dst], v0[:, dst] = k0[:, src], v0[:, src]
    assert torch.equal(_bits(k), _bits(k0)) and torch.equal(_bits(v), _bits(v0))


def test_generation_with_forks_and_compaction(A, q8):
    """The operators together, as a program that runs a model calls them: prompts, a decode loop whose sequences fork and end, a compaction in between, the
    projections by the Q8_0 mat-muls; every attention against the definition, on the tokens that the sequences consist of."""
    heads, kv_heads, dim, page, layers, embd = 8, 2, 64, 16, 2, 512
    g = torch.Generator(device="cuda").manual_seed(7)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    weights = [{n: q8.quantize_row_q8_0(randn(rows, embd) * 0.05, tiled=True) for n, rows in (("q", heads * dim), ("k", kv_heads * dim), ("v", kv_heads * dim), ("o", embd))} for _ in range(layers)]
    k_pages, v_pages = A.empty_cache(layers, 64, kv_heads, page, dim)
    k_pages.fill_(float("nan"))
    v_pages.fill_(float("nan"))
    turns = A.rope_turns(dim)
    inverse = [500000.0 ** (-2.0 * i / dim) for i in range(dim // 2)]
    new = [37, 16, 5]
    parents, grow = _dev([-1, -1, -1]), _dev([0, 0, 0])
    table, lengths = torch.full((3, 8), -1, dtype=torch.int32, device="cuda"), _dev([0, 0, 0])
    # (a sequence starts as the empty one: a parent of no tokens)
    table, lengths, info = A.cache_step(k_pages, v_pages, table, lengths, _dev([0, 1, 2]), _dev(new))
    assert info.tolist()[2] == 0 and lengths.tolist() == new
    # what each sequence's keys and values are, kept beside the cache: [layer][sequence] -> lists of (k, v) rows as projected
    history = [[[] for _ in new] for _ in range(layers)]

    def layer_pass(layer, x, starts):
        w = weights[layer]
        q = q8.mul_mat(w["q"], x, heads * dim, embd).view(-1, heads, dim)
        k = q8.mul_mat(w["k"], x, kv_heads * dim, embd).view(-1, kv_heads, dim)
        v = q8.mul_mat(w["v"], x, kv_heads * dim, embd).view(-1, kv_heads, dim)
        r = A.append_rope(q, k, v, k_pages[layer], v_pages[layer], table, lengths, turns, starts=starts)
        if starts is None:
            attn = A.attention_decode(r, k_pages[layer], v_pages[layer], table, lengths)
        else:
            attn = A.attention_prompt(r, k_pages[layer], v_pages[layer], table, lengths, starts)
        ends = lengths.tolist()
        begin = list(range(len(ends) + 1)) if starts is None else starts.tolist()
        for s, n in enumerate(ends):
            rows = range(begin[s], begin[s + 1])
            history[layer][s] += [(k[i].cpu(), v[i].cpu()) for i in rows] if n else []
            if not n:
                continue
            assert len(history[layer][s]) == n
            # the keys as the cache has to hold them: rotated, rounded once (differences of a unit in the last place of fp16 from the fp32 rotation are in the bound below)
            kk = torch.stack([R.rope(kv[0], j, inverse, True)[0].to(torch.float16).double() for j, kv in enumerate(history[layer][s])], dim=1)
            vv = torch.stack([kv[1].to(torch.float16).double() for kv in history[layer][s]], dim=1)
            i = rows[-1]
            qq = R.rope(q[i].cpu(), n - 1, inverse, True)[0]
            ref, mean, d, count = R.attend(qq, kk, vv, torch.ones(n, dtype=torch.bool), dim**-0.5)
            # q off by 2^-21, a key now and then by a unit of fp16 (2^-10) where the fp32 rotation lies on the other side of a tie: S (2^-21 + 2^-10) more in a score
            big = dim**-0.5 * torch.stack([(kk[h // (heads // kv_heads)].abs() @ qq[h].abs()).max() for h in range(heads)])
            most = R.bound(ref, mean, d + big * (2.0**-21 + 2.0**-10), count, torch.float32)
            off = (attn[i].cpu().double() - ref).abs()
            assert bool((off <= most).all()), (layer, s, n)
        return q8.mul_mat(w["o"], attn.reshape(-1, heads * dim), embd, embd, residual=x)

    x = randn(sum(new), embd)
    starts = _dev([0, 37, 53, 58])
    for layer in range(layers):
        x = layer_pass(layer, x, starts)
    plans = [[0, 1, 2], [0, 0, 1, 2], [3, 1, 1, 0, 0], [0, 1, 2, 3, 4], [4, 4, -1, 2, 2], [0, 1, 3, 4]]
    for t, plan in enumerate(plans):
        table, lengths, info = A.cache_step(k_pages, v_pages, table, lengths, _dev(plan), _dev([1] * len(plan)))
        assert info.tolist()[2] == 0
        history[:] = [[list(h[p]) if p >= 0 else [] for p in plan] for h in history]
        if t == 3:
            table, info = A.cache_compact(k_pages, v_pages, table, lengths)
            assert info.tolist()[2] == 0 and int(table.max()) == info.tolist()[0] - 1
            k_pages[:, info.tolist()[0] :] = float("nan")  # nothing is held there
            v_pages[:, info.tolist()[0] :] = float("nan")
        x = randn(len(plan), embd)
        for layer in range(layers):
            x = layer_pass(layer, x, None)
