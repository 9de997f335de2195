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
