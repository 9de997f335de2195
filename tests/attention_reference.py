"""Attention over a paged cache, rope and page bookkeeping from their definitions, in 64 bits and plain Python, for the tests of nihilus_amd.attention.

Bounds.  With u = 2^-24 (half a step of fp32) an fp32 sum of n products is off by at most (n + 2) u times the sum of their magnitudes.  For a row with
scores s_j = scale q.k_j, S = scale max_j sum |q||k_j| and s = max |s_j| that gives, with 2^-21 for q as a sum of 16-bit terms (22 bits and more), an error of a score of at most
    d = S ((dim + 4) u + 2^-21) + 4 s u
(the last for scores brought into powers of two and for the exponent's rounding), so a relative error of a weight of e^d - 1 + 4 u, of a weighted
sum over n keys of as much plus (n + 2) u, of the sum of the weights likewise, and of the joining of partial results (each a product with a
power of two and an addition) 8 u more.  A 16-bit q has its weights rounded once: half a step.  All of these are relative to sum p |v| / sum p.
The result is rounded once to its type: half a step of its own size (and half the smallest subnormal).
"""
import math

import torch

U = 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def keys_of(k_pages, v_pages, row, length):
    """[kv heads, length, dim] keys and values of one sequence in 64 bits, and which of them exist; pages that the cache does not have give zeros that do not."""
    pages, heads, page, dim = k_pages.shape
    k, v = torch.zeros(heads, length, dim, dtype=torch.float64), torch.zeros(heads, length, dim, dtype=torch.float64)
    there = torch.zeros(length, dtype=torch.bool)
    for j in range(length):
        slot = j // page
        if slot < len(row) and 0 <= row[slot] < pages:
            k[:, j], v[:, j], there[j] = k_pages[row[slot], :, j % page].double(), v_pages[row[slot], :, :, j % page].double(), True
    return k, v, there


def attend(q, k, v, there, scale):
    """q [heads, dim] over k, v [kv heads, n, dim] where there: the result [heads, dim] and sum p |v| / sum p, and per head d and n (see above)."""
    heads, dim = q.shape
    group = heads // k.shape[0]
    out, mean, d = torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dtype=torch.float64)
    k, v = k[:, there], v[:, there]
    if k.shape[1] == 0:
        return out, mean, d, 0
    for h in range(heads):
        x = q[h].double()
        s = scale * (k[h // group] @ x)
        w = torch.exp(s - s.max())
        w = w / w.sum()
        out[h], mean[h] = w @ v[h // group], w @ v[h // group].abs()
        big = scale * float((k[h // group].abs() @ x.abs()).max())
        d[h] = big * ((dim + 4) * U + 2.0**-21) + 4 * float(s.abs().max()) * U
    return out, mean, d, k.shape[1]


def bound(ref, mean, d, n, dtype):
    """How far a result may be off, element by element."""
    weight = torch.expm1(d)[..., None] + 4 * U + (half_step(dtype) if dtype != torch.float32 else 0.0)
    inner = mean * (2 * weight + (2 * n + 4 + 8) * U)
    return inner + half_step(dtype) * (ref.abs() + inner) + tiny(dtype)


def rope(x, pos, inverse, interleaved):
    """x [heads, dim] in 64 bits turned by pos * inverse[i]; (result, |a| + |b| of each value's pair)."""
    x = x.double().clone()
    r = 2 * len(inverse)
    out, size = x.clone(), torch.zeros_like(x)
    for i, w in enumerate(inverse):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        t = math.fmod(pos * w, 2.0 * math.pi)
        c, s = math.cos(t), math.sin(t)
        out[:, a], out[:, b] = x[:, a] * c - x[:, b] * s, x[:, a] * s + x[:, b] * c
        size[:, a] = size[:, b] = x[:, a].abs() + x[:, b].abs()
    return out, size


def step(table, lengths, parents, grow, pages, page):
    """The next tables, lengths, info and moves of a cache, from the definition: what a child keeps, who owns a page that is written on, what is given."""
    width = len(table[0]) if table else 0
    kept, after, full, owner, lost = [], [], set(), {}, 0
    for i, (p, g) in enumerate(zip(parents, grow)):
        alive = 0 <= p < len(table)
        had = min(max(lengths[p], 0), width * page) if alive else 0
        now = min(max(had + g, 0), width * page) if alive else 0
        keep = min(had, now)
        row = table[p][: -(-keep // page)] if alive else []
        for j, id in enumerate(row):
            if not 0 <= id < pages:
                lost += 1
            elif j == len(row) - 1 and keep % page:
                owner.setdefault(id, i)
            else:
                full.add(id)
        kept.append((row, keep))
        after.append(now)
    free = [p for p in range(pages) if p not in full and p not in owner]
    n_free, given, missing, moves, new = len(free), 0, 0, [], []
    for i, (row, keep) in enumerate(kept):
        row, out = list(row), []
        last = len(row) - 1 if keep % page else None
        for j in range(-(-after[i] // page)):
            if j < len(row) and not 0 <= row[j] < pages:
                out.append(-1)
                continue
            if j < len(row) and (j != last or (row[j] not in full and owner[row[j]] == i)):
                out.append(row[j])
                continue
            if free:
                got, given = free.pop(0), given + 1
            else:
                got, missing = -1, missing + 1
            if j < len(row) and got >= 0:
                moves.append((row[j], got))
            out.append(got)
        new.append(out + [-1] * (width - len(out)))
    return new, after, [pages - n_free + given, len(moves), missing + lost], moves


def compact(table, lengths, pages, page):
    width = len(table[0]) if table else 0
    rows, lost, live = [], 0, set()
    for row, n in zip(table, lengths):
        row = row[: -(-min(max(n, 0), width * page) // page)]
        lost += sum(not 0 <= id < pages for id in row)
        live.update(id for id in row if 0 <= id < pages)
        rows.append(row)
    holes = [p for p in range(len(live)) if p not in live]
    moves = list(zip(sorted(p for p in live if p >= len(live)), holes))
    to = dict(moves)
    new = [[to.get(id, id) if 0 <= id < pages else -1 for id in row] + [-1] * (width - len(row)) for row in rows]
    return new, [len(live), len(moves), lost], moves
