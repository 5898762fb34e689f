"""Pages that several sequences hold: the search for them (whole numbers, exact) and the attention that computes them once
for all, against the numpy oracle in float64.

Bound of an output: that of attend (the weights rounded to float16, the output to its type, float32 sums), because the parts
of a row are joined in float32 (a few 2^-24, inside the 2^-13 that stands for the sums and exponentials):
|o - exact| <= (u_out + 2^-11 + 2^-13 + 2 e) sum p|v| / l + keys 2^-24 max|v|, e the logits' round-off."""

import numpy as np
import pytest
import torch

from oracle import paged as O

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
NAMES = ("kc", "vc", "ks", "vs", "table", "lens", "refs")


@pytest.fixture(autouse=True)
def clean_status(cuda_dev):
    import kvb
    kvb.device_status()
    yield
    assert kvb.device_status() == 0, "a test left the device status word set"


def status():
    import kvb
    return kvb.device_status()


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def on_gpu(pool):
    import kvb
    return kvb.PagePool(*[torch.from_numpy(pool[x].copy()).cuda() for x in NAMES])


def family(rng, system, prompts, samples, own, hkv=2, d=64, page=16, scale=1.0):
    """A pool of sequences forked from forked prompts: every full page of the system prompt is held by all, of a request by
    its samples.  Sequence i: request i // samples, system + prompts[..] + own[i] tokens."""
    n = len(prompts) * samples
    before = [system + p for p in prompts]
    lens = [before[i // samples] + own[i] for i in range(n)]
    nb = [O.blocks(x, page) for x in lens]
    pool = O.empty_pool(sum(nb) + 5, hkv, d, page, n + 2, max(nb) + 2)
    perm, at, slots = rng.permutation(sum(nb) + 5), 0, rng.permutation(n + 2)[:n]
    for i, s in enumerate(slots):
        first = slots[i // samples * samples]
        held = 0
        if i:
            held = system // page
            pool["table"][s, :held] = pool["table"][slots[0], :held]
        if i % samples:
            held = before[i // samples] // page
            pool["table"][s, :held] = pool["table"][first, :held]
        pool["table"][s, held:nb[i]] = perm[at:at + nb[i] - held]
        at += nb[i] - held
        for b in range(nb[i]):
            pool["refs"][pool["table"][s, b]] += 1
        pool["lens"][s] = lens[i]
    for x in ("kc", "vc"):
        pool[x][:] = np.clip(np.rint(rng.standard_normal(pool[x].shape) * 40), -127, 127) + 128
    for x in ("ks", "vs"):
        pool[x][:] = scale * 0.025 * np.exp(0.3 * rng.standard_normal(pool[x].shape))
    return pool, slots


def check_share(g, pool, slots):
    s = g.share(ints(slots))
    want = O.share(pool, slots)
    n, segments = len(slots), want["segments"]
    assert s.order.tolist() == want["order"] and s.own.tolist() == want["own"] and s.depth.tolist() == want["depth"]
    assert s.count.tolist() == [len(segments)]
    assert s.segments.tolist() == segments + [[0] * 5] * (n - len(segments))
    return s


FAMILIES = [    # system, prompts, samples, page
    (0, [100], 2, 16), (0, [40, 7, 64, 129], 3, 16), (70, [5, 100, 33, 16, 1], 4, 32), (200, [64] * 9, 1, 64),
    (0, [15], 4, 16), (128, [128, 128], 8, 128), (16, list(range(1, 60, 3)), 5, 16)]


@pytest.mark.parametrize("system,prompts,samples,page", FAMILIES)
def test_share(cuda_dev, system, prompts, samples, page):
    rng = np.random.default_rng(1)
    n = len(prompts) * samples
    pool, slots = family(rng, system, prompts, samples, rng.integers(0, 3 * page, n), page=page)
    g = on_gpu(pool)
    for order in (np.arange(n), rng.permutation(n), rng.integers(0, n, 2 * n)):       # any order, the same sequence twice
        check_share(g, pool, slots[order])


@pytest.mark.parametrize("n", [1, 2, 31, 33, 300, 1000, 1024])
def test_share_of_random_tables(cuda_dev, n):
    """Rows over a few page numbers: many levels, classes that part anywhere, pages held in different blocks, entries that
    are no page, lengths that do not fit."""
    rng = np.random.default_rng(n)
    for width, ids in ((3, 2), (40, 3), (7, 40), (300, 2)):
        pool = O.empty_pool(ids + 3, 1, 64, 16, n, width)
        base = rng.integers(0, ids, (max(1, n // 5), width))
        keep = rng.integers(0, width + 1, n)
        rows = base[rng.integers(0, len(base), n)]
        pool["table"][:] = np.where(np.arange(width) < keep[:, None], rows, rng.integers(-1, ids + 4, (n, width)))
        pool["lens"][:] = rng.integers(-5, 16 * width + 40, n)
        check_share(on_gpu(pool), pool, rng.permutation(n))


def test_share_refusals(cuda_dev):
    rng = np.random.default_rng(3)
    pool, slots = family(rng, 0, [100], 3, [1, 2, 3])
    g = on_gpu(pool)
    bad = np.array([slots[0], 99, slots[1], -1])
    check_share(g, pool, bad)
    assert status() == 2
    s = g.share(ints([]))
    assert s.count.tolist() == [0] and s.order.shape == (0,) and s.segments.shape == (0, 5)
    with pytest.raises(ValueError):
        g.share(ints(np.zeros(1025)))
    for slots in (torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int32), ints(np.zeros(6))[::2]):
        with pytest.raises(ValueError):
            g.share(slots)


def check(g, pool, q, slots, scaling=None, shared=None, **kw):
    d = q.shape[-1]
    sc = d ** -0.5 if scaling is None else scaling
    s = g.share(ints(slots)) if shared is None else shared
    out, lse = g.attend_shared(q, s, scaling, return_lse=True, **kw)
    want, wl, mean_abs = O.attend(pool, q.float().cpu().numpy(), slots, sc)
    rows = [O.rows(pool, x, 0, pool["lens"][x]) for x in slots]
    vmax = max([float(np.abs(r[1]).max(initial=0)) for r in rows])
    kmax = max([float(np.abs(r[0]).sum(-1).max(initial=0)) for r in rows])
    keys = int(max(pool["lens"][list(slots)]))
    logit = d * 2.0 ** -24 * kmax * float(q.float().abs().max()) * abs(sc)
    tol = (U[q.dtype] + 2.0 ** -11 + 2.0 ** -13 + 2 * logit) * mean_abs + keys * 2.0 ** -24 * vmax
    got = out.double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) - tol).max()), [int(x) for x in np.argwhere(bad)[0]])
    gl = lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(gl), np.isneginf(wl))
    seen = ~np.isneginf(wl)
    assert (np.abs(gl[seen] - wl[seen]) <= logit + 2.0 ** -16 + 2.0 ** -22 * np.abs(wl[seen])).all()
    assert (got[~seen] == 0).all()
    assert torch.equal(g.attend_shared(q, s, scaling), out)             # the same call gives the same bits
    return out


ATTENDS = [     # dtype, d, page, hkv, rep, tq, system, prompts, samples, longest
    (torch.bfloat16, 128, 64, 2, 4, 1, 0, [500], 2, 40),
    (torch.float16, 64, 16, 1, 1, 1, 0, [33, 7, 64], 2, 20),
    (torch.bfloat16, 128, 32, 2, 4, 1, 100, [300, 64, 1], 8, 50),
    (torch.float16, 128, 64, 1, 8, 1, 1000, [64, 200], 16, 130),
    (torch.float16, 64, 16, 2, 4, 4, 50, [100, 31], 5, 30),
    (torch.bfloat16, 64, 128, 3, 3, 2, 129, [256] * 3, 3, 200),
    (torch.bfloat16, 128, 16, 1, 5, 3, 3000, [20, 1, 700], 7, 90),
    (torch.float16, 64, 32, 1, 16, 1, 320, [1] * 40, 1, 33),
    (torch.bfloat16, 128, 64, 4, 1, 7, 64, [64], 9, 3)]


@pytest.mark.parametrize("dtype,d,page,hkv,rep,tq,system,prompts,samples,longest", ATTENDS)
def test_attend_shared(cuda_dev, dtype, d, page, hkv, rep, tq, system, prompts, samples, longest):
    rng = np.random.default_rng(5)
    n = len(prompts) * samples
    pool, slots = family(rng, system, prompts, samples, rng.integers(tq, longest + tq, n), hkv, d, page)
    slots = rng.permutation(slots)
    q = torch.from_numpy(rng.standard_normal((n, hkv * rep, tq, d))).to(dtype).cuda()
    g = on_gpu(pool)
    check(g, pool, q, slots)
    check(g, pool, q, slots, -0.03)
