"""Shared pages where they can go wrong: lists that are filled anew, queries that do not see all of a segment, pages whose scale
is not finite where nobody looks, sequences without tokens of their own, four levels; against the numpy oracle in float64
with the bounds of test_shared_gpu."""

import numpy as np
import pytest
import torch

from test_shared_gpu import check, clean_status, family, ints, on_gpu      # noqa: F401

pytestmark = pytest.mark.gpu


def test_the_list_may_be_filled_anew(cuda_dev):
    """A buffer of slots that a server fills again before it attends: the plan and its sequences stay together, in single calls
    and in a graph whose replays read the buffer as it is then."""
    rng = np.random.default_rng(1)
    pool, slots = family(rng, 100, [40, 64, 200], 3, [5] * 9, 2, 64, 16)
    g = on_gpu(pool)
    lists = [slots[:6], slots[[8, 1, 7, 0, 6, 2]]]
    q = torch.from_numpy(rng.standard_normal((6, 4, 1, 64))).to(torch.float16).cuda()
    wants = [check(g, pool, q, x) for x in lists]
    buffer = ints(lists[0])
    s = g.share(buffer)
    buffer.copy_(ints(lists[1]))
    assert s.slots.tolist() == [int(x) for x in lists[0]]
    assert torch.equal(g.attend_shared(q, s), wants[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t = g.share(buffer)
        out = g.attend_shared(q, t)
    for i in (0, 1, 0):
        buffer.copy_(ints(lists[i]))
        graph.replay()
        buffer.fill_(-1)
        assert torch.equal(out, wants[i]) and torch.equal(g.attend_shared(q, t), wants[i])


@pytest.mark.parametrize("side,value", [("ks", float("nan")), ("vs", float("inf"))])
@pytest.mark.parametrize("page,tq,samples", [(16, 40, 3), (32, 70, 2), (64, 66, 4)])
def test_scales_of_pages_that_a_query_does_not_see(cuda_dev, side, value, page, tq, samples):
    """Queries among the last tq positions, all of them on shared pages: a scale that is not finite concerns the queries that see its
    page, and no others."""
    rng = np.random.default_rng(2)
    n = 2 * samples
    pool, slots = family(rng, 4 * page, [4 * page, 5 * page], samples, [0] * n, 2, 64, page)
    q = torch.from_numpy(rng.standard_normal((n, 4, tq, 64))).to(torch.float16).cuda()
    g = on_gpu(pool)
    s = g.share(ints(slots))
    assert s.own.tolist() == [int(pool["lens"][x]) for x in slots]                  # nothing of their own
    clean = g.attend_shared(q, s)
    back = 1 if tq <= 2 * page else 2                                               # the page that far from the end
    hurt = torch.zeros(clean.shape[:3], dtype=torch.bool, device="cuda")
    for first in (0, samples):                                                      # a page of either family
        blocks = int(pool["lens"][slots[first]]) // page
        pool[side][pool["table"][slots[first], blocks - back], 1] = value
        for i in range(first, first + samples):
            begins = (blocks - back) * page                                         # its first token
            hurt[i, torch.arange(tq, device="cuda") + int(pool["lens"][slots[i]]) - tq >= begins, 2:] = True
    g = on_gpu(pool)
    got = g.attend_shared(q, g.share(ints(slots)))
    assert not hurt.all() and hurt.any()
    assert torch.equal(got[~hurt], clean[~hurt]) and torch.isnan(got[hurt]).all()
    if side == "ks":
        assert torch.equal(torch.isnan(g.attend(q, ints(slots))).any(-1), hurt)


@pytest.mark.parametrize("dtype,d,page,tq,samples,own", [
    (torch.float16, 64, 16, 5, 3, [0, 1, 4]), (torch.bfloat16, 128, 64, 3, 4, [0, 2, 0, 1]), (torch.bfloat16, 64, 32, 100, 2, [0, 7]),
    (torch.float16, 128, 128, 200, 3, [0, 0, 50]), (torch.bfloat16, 128, 16, 1, 40, [0] * 40), (torch.float16, 128, 16, 31, 9, [0, 1, 2, 3, 4, 5, 6, 7, 8])])
def test_queries_that_do_not_see_all_of_a_segment(cuda_dev, dtype, d, page, tq, samples, own):
    """Fewer tokens of their own than queries, down to none: the first queries stand on shared pages."""
    rng = np.random.default_rng(3)
    pool, slots = family(rng, 2 * page, [page, 3 * page], samples, own * 2, 2, d, page)
    g = on_gpu(pool)
    n = 2 * samples
    q = torch.from_numpy(rng.standard_normal((n, 6, tq, d))).to(dtype).cuda()
    s = g.share(ints(slots))
    assert (s.depth.cpu() == 2).all() and any(int(pool["lens"][x]) - tq < o for x, o in zip(slots, s.own.tolist()))
    check(g, pool, q, slots, shared=s)
    check(g, pool, q, slots, -0.07, shared=s)


@pytest.mark.parametrize("d,page,tq,many", [(64, 16, 1, 1), (128, 32, 2, 1), (128, 16, 1, 5)])
def test_four_levels(cuda_dev, d, page, tq, many):
    """Sequences that part in twos four times over, and `many` such trees that share nothing: every level's part of a row is
    joined with its own tokens."""
    from oracle import paged as O
    rng = np.random.default_rng(4)
    held, n = [3, 2, 4, 1], 16 * many                                               # blocks of a class on each level
    pool = O.empty_pool(200 * many, 1, d, page, n, 14)
    fresh = iter(rng.permutation(200 * many))
    pages = {}
    for i in range(n):
        row = [pages.setdefault((level, i >> 4 - level, b), next(fresh)) for level in range(4) for b in range(held[level])]
        own = int(rng.integers(tq, 3 * page))
        row += [next(fresh) for _ in range(O.blocks(own, page))]
        pool["table"][i, :len(row)] = row
        pool["lens"][i] = sum(held) * page + own
    for x in ("kc", "vc"):
        pool[x][:] = rng.integers(1, 256, pool[x].shape)
    for x in ("ks", "vs"):
        pool[x][:] = 0.02 * np.exp(0.3 * rng.standard_normal(pool[x].shape))
    g = on_gpu(pool)
    order = rng.permutation(n)
    s = g.share(ints(order))
    assert s.depth.tolist() == [4] * n and s.count.tolist() == [15 * many]
    check(g, pool, torch.from_numpy(rng.standard_normal((n, 4, tq, d))).to(torch.bfloat16).cuda(), order, shared=s)


def test_a_wide_table_of_short_sequences(cuda_dev):
    """Rows for 65536 pages: the results of a narrow table, bit for bit."""
    rng = np.random.default_rng(5)
    pool, slots = family(rng, 64, [70] * 75, 8, [20] * 600, 2, 64, 64)
    g = on_gpu(pool)
    q = torch.from_numpy(rng.standard_normal((600, 16, 16, 64), np.float32)).to(torch.float16).cuda()
    want = g.attend_shared(q, g.share(ints(slots)))
    pool["table"] = np.pad(pool["table"], ((0, 0), (0, 65536 - pool["table"].shape[1])), constant_values=-1)
    g = on_gpu(pool)
    assert torch.equal(g.attend_shared(q, g.share(ints(slots))), want)
    check(g, pool, q[:4, :, :2].contiguous(), slots[:4])
