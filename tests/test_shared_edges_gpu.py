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
