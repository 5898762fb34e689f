"""Several host threads on one stream: each call's results are those of one thread, bit for bit."""

import threading

import numpy as np
import pytest
import torch

from test_shared_gpu import family, ints, on_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(cuda_dev):
    import kvb
    kvb.device_status()
    yield
    assert kvb.device_status() == 0, "a test left the device status word set"


def together(jobs, times):
    """jobs: (call, wanted outputs).  Each by a thread of its own on the default stream, compared at the end."""
    gate, same, failed = threading.Barrier(len(jobs)), [None] * len(jobs), []

    def work(i, call, want):
        try:
            ok = torch.ones((), dtype=torch.bool, device="cuda")
            gate.wait()
            for _ in range(times):
                for x, y in zip(call(), want):
                    ok &= (x == y).all()
            same[i] = ok
        except Exception as e:                                          # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i, *job)) for i, job in enumerate(jobs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert all(bool(x) for x in same)


def test_cross_attention(cuda_dev):
    """Calls of few rows and of many, over states of other lengths, the same workspace."""
    import kvb
    g = torch.Generator(device="cuda").manual_seed(1)
    jobs = []
    for queries, keys in (([300, 40], [3000, 77]), ([1000], [900]), ([1, 2], [5000, 30]), ([20], [4000])):
        cu = [torch.tensor([0] + list(np.cumsum(x)), dtype=torch.int32, device="cuda") for x in (queries, keys)]
        q, k, v = (torch.randn(n, h, 128, generator=g, device="cuda").bfloat16() for n, h in ((sum(queries), 8), (sum(keys), 2), (sum(keys), 2)))
        call = lambda q=q, k=k, v=v, cu=cu: kvb.cross_attention(q, k, v, *cu, return_lse=True)       # noqa: E731
        jobs.append((call, call()))
    torch.cuda.synchronize()
    together(jobs, 300)


def test_attend_shared(cuda_dev):
    """Calls of two layers of a pool over batches of other sizes."""
    rng = np.random.default_rng(2)
    pool, slots = family(rng, 300, [40, 500, 64], 8, rng.integers(1, 200, 24), 2, 128, 64)
    g = on_gpu(pool)
    layers = [g, g.add_layer(*[getattr(g, x).flip(0).contiguous() for x in ("kc", "vc", "ks", "vs")])]
    jobs = []
    for n, tq in ((24, 1), (7, 3), (16, 2), (2, 1)):
        q = torch.from_numpy(rng.standard_normal((n, 8, tq, 128))).to(torch.bfloat16).cuda()
        s, p = g.share(ints(slots[rng.permutation(24)[:n]])), layers[n % 2]
        call = lambda p=p, q=q, s=s: p.attend_shared(q, s, return_lse=True)                         # noqa: E731
        jobs.append((call, call()))
    torch.cuda.synchronize()
    together(jobs, 300)


def test_a_pool_that_two_threads_change(cuda_dev):
    """One thread grows and frees its sequences, the other forks, frees and compacts: what is held is told by the table, and the
    sequences that stay keep their rows."""
    import kvb
    g = torch.Generator(device="cuda").manual_seed(3)
    pool = kvb.PagePool.create(400, 2, 64, 16, n_slots=40, max_blocks=40)
    layer = pool.add_layer()
    stay, mine, forks = ints(range(8)), ints(range(8, 16)), ints(range(16, 24))
    lens = [100 + 7 * i for i in range(8)]
    cu = ints(np.concatenate([[0], np.cumsum(lens)]))
    start = pool.extend(stay, ints(lens))
    for p in (pool, layer):
        p.write(stay, start, cu, *(torch.randn(sum(lens), 2, 64, generator=g, device="cuda").half() for _ in "kv"))
    zero, before = ints([0] * 8), []
    for p in (pool, layer):
        before += p.read(stay, zero, cu, sum(lens))
    add, ca = ints([21] * 8), ints(np.arange(9) * 21)
    k, v = (torch.randn(8 * 21, 2, 64, generator=g, device="cuda").half() for _ in "kv")

    def grow():
        at = pool.extend(mine, add)
        for p in (pool, layer):
            p.write(mine, at, ca, k, v)
        pool.free(mine)
        return ()

    def move():
        pool.fork(stay, forks)
        pool.free(stay[:4])
        pool.fork(forks[:4], stay[:4])
        pool.free(forks)
        pool.compact()
        return ()

    torch.cuda.synchronize()
    together([(grow, ()), (move, ())], 200)
    after = []
    for p in (pool, layer):
        after += p.read(stay, zero, cu, sum(lens))
    assert all(torch.equal(x, y) for x, y in zip(before, after))
    held = torch.bincount(pool.table[pool.table >= 0].long(), minlength=400)
    assert torch.equal(held, pool.refs.long()) and pool.lens.tolist() == lens + [0] * 32
