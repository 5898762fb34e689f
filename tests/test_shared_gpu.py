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


def reference(g, q, slots, scaling):
    """The same attention in float64 on the GPU, from the pool's tensors: out, lse and the attended mean of |v|."""
    n, hq, tq, d = q.shape
    outs, lses, means = [], [], []
    for i, s in enumerate(slots):
        m = int(g.lens[s])
        pages = g.table[s, :-(-m // g.page)].long()

        def side(c, scale):
            return ((c[pages].double() - 128) * scale[pages].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :m]

        k, v = side(g.kc, g.ks), side(g.vc, g.vs)
        x = torch.einsum("hrtd,hnd->hrtn", q[i].double().unflatten(0, (g.Hkv, -1)), k) * scaling
        last = m - tq + torch.arange(tq, device="cuda")
        x = x.masked_fill(torch.arange(m, device="cuda") > last[:, None], -torch.inf)
        lses.append(torch.logsumexp(x, -1).permute(2, 0, 1).flatten(1))
        w = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        outs.append(torch.einsum("hrtn,hnd->thrd", w, v).flatten(1, 2))
        means.append(torch.einsum("hrtn,hnd->thrd", w, v.abs()).flatten(1, 2))
    return torch.stack(outs), torch.stack(lses), torch.stack(means)


def check_large(g, q, slots, scaling=None, shared=None):
    d = q.shape[-1]
    sc = d ** -0.5 if scaling is None else scaling
    out, lse = g.attend_shared(q, shared or g.share(ints(slots)), scaling, return_lse=True)
    want, wl, mean_abs = reference(g, q, slots, sc)
    logit = d * 2.0 ** -24 * 127 * d * float(g.ks.max()) * float(q.float().abs().max()) * abs(sc)
    tol = (U[q.dtype] + 2.0 ** -11 + 2.0 ** -13 + 2 * logit) * mean_abs + int(g.lens.max()) * 2.0 ** -24 * 127 * float(g.vs.max())
    bad = (out.double() - want).abs() > tol
    assert torch.isfinite(out).all() and not bad.any(), (int(bad.sum()), float(((out.double() - want).abs() - tol).max()), [int(x) for x in bad.nonzero()[0]])
    seen = wl > -torch.inf
    assert torch.equal(lse > -torch.inf, seen) and (out[~seen] == 0).all()
    assert ((lse.double() - wl).abs()[seen] <= logit + 2.0 ** -16 + 2.0 ** -22 * wl.abs()[seen]).all()
    return out


LARGE = [       # dtype, d, page, hkv, rep, tq, system, prompts, samples: items cut over many blocks, whole ones, several groups of rows
    (torch.bfloat16, 128, 64, 1, 4, 1, 30000, [1], 3), (torch.float16, 64, 16, 2, 8, 3, 2000, [300, 20], 40),
    (torch.bfloat16, 128, 128, 8, 4, 1, 4000, [20] * 64, 1), (torch.float16, 128, 32, 2, 16, 5, 0, [64, 1000, 128], 20),
    (torch.bfloat16, 64, 64, 4, 2, 1, 64, [500] * 30, 20)]


@pytest.mark.parametrize("dtype,d,page,hkv,rep,tq,system,prompts,samples", LARGE)
def test_attend_shared_large(cuda_dev, dtype, d, page, hkv, rep, tq, system, prompts, samples):
    rng = np.random.default_rng(6)
    n = len(prompts) * samples
    pool, slots = family(rng, system, prompts, samples, rng.integers(tq, 150 + tq, n), hkv, d, page)
    g = on_gpu(pool)
    q = torch.from_numpy(rng.standard_normal((n, hkv * rep, tq, d))).to(dtype).cuda()
    check_large(g, q, rng.permutation(slots))


def test_attend_shared_of_what_attend_gives(cuda_dev):
    """Nothing shared, one sequence, the same sequence several times, sequences that are empty or shorter than their
    queries; the results of attend up to the bound of both."""
    rng = np.random.default_rng(7)
    pool, slots = family(rng, 0, [40, 33, 16], 1, [5, 0, 3], page=16)
    pool["lens"][slots[1]] = 0
    pool["lens"][slots[2]] = 2
    g = on_gpu(pool)
    for pick in ([0], [0, 1, 2], [0, 0], [2, 0, 0, 1, 0]):
        for tq in (1, 4):
            q = torch.from_numpy(rng.standard_normal((len(pick), 4, tq, 64))).to(torch.float16).cuda()
            check(g, pool, q, slots[pick])


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64)])
def test_attend_shared_scales_far_apart(cuda_dev, d, page):
    """Shared pages of zeros, of tiny and huge key and value scales."""
    rng = np.random.default_rng(8)
    pool, slots = family(rng, 600, [1], 6, [3] * 6, 1, d, page)
    for i, b in enumerate(pool["table"][slots[0], :600 // page]):
        pool["vs"][b] = [0.02, 2.0 ** -60, 2.0 ** 40, 0.0][i % 4]
        pool["ks"][b] = [0.02, 0.0, 0.05, 2.0 ** -40][(i // 4) % 4]
    g = on_gpu(pool)
    q = torch.from_numpy(rng.standard_normal((6, 4, 1, d))).to(torch.bfloat16).cuda()
    check(g, pool, q, slots)
    for i, b in enumerate(pool["table"][slots[0], :600 // page]):       # value scales that pass 2^100 of one another
        pool["vs"][b] = 2.0 ** -90 if i % 2 else 2.0 ** 50
        pool["ks"][b] = 0.05 if i % 2 else 1e-6
    check(on_gpu(pool), pool, q, slots)


@pytest.mark.parametrize("scaling", [0.0, 2.0, -1.0])
def test_attend_shared_any_scaling(cuda_dev, scaling):
    rng = np.random.default_rng(9)
    pool, slots = family(rng, 300, [30, 5], 3, [2] * 6, 2, 64, 16)
    q = torch.from_numpy(rng.standard_normal((6, 4, 2, 64))).to(torch.float16).cuda()
    check(on_gpu(pool), pool, q, slots, scaling)


def test_a_row_that_is_not_finite_stays_alone(cuda_dev):
    rng = np.random.default_rng(10)
    pool, slots = family(rng, 500, [64, 1], 4, [30] * 8, 2, 128, 64)
    g = on_gpu(pool)
    q = torch.from_numpy(rng.standard_normal((8, 8, 1, 128))).to(torch.bfloat16).cuda()
    s = g.share(ints(slots))
    clean = g.attend_shared(q, s)
    for at, value in (((0, 3, 0, 5), float("nan")), ((7, 0, 0, 0), float("inf"))):
        p = q.clone()
        p[at] = value
        got = g.attend_shared(p, s)
        hurt = torch.zeros(got.shape[:3], dtype=torch.bool, device="cuda")
        hurt[at[0], 0, at[1]] = True
        assert torch.equal(got[~hurt], clean[~hurt]) and torch.isnan(got[hurt]).all()


@pytest.mark.parametrize("side,value", [("ks", float("nan")), ("vs", float("inf"))])
def test_a_scale_that_is_not_finite_is_that_of_its_head(cuda_dev, side, value):
    """No write makes such a scale; where one is, attend_shared is not finite where attend is not, and nowhere else."""
    rng = np.random.default_rng(18)
    pool, slots = family(rng, 500, [64, 1], 4, [30] * 8, 2, 128, 64)
    q = torch.from_numpy(rng.standard_normal((8, 8, 1, 128))).to(torch.bfloat16).cuda()
    g = on_gpu(pool)
    clean = g.attend_shared(q, g.share(ints(slots)))
    pool[side][pool["table"][slots[0], 3], 1] = value
    g = on_gpu(pool)
    got = g.attend_shared(q, g.share(ints(slots)))
    assert torch.isnan(g.attend(q, ints(slots))[:, :, 4:]).all() and torch.isnan(got[:, :, 4:]).all()
    assert torch.equal(got[:, :, :4], clean[:, :, :4])


@pytest.mark.parametrize("samples", [2, 16])
def test_pages_whose_offsets_pass_32_bits(cuda_dev, samples):
    """The last pages of a pool of 4.3 GB a side: the results of a small pool, bit for bit."""
    import kvb
    rng = np.random.default_rng(19)
    pool, slots = family(rng, 700, [64, 1], samples, [30] * (2 * samples), 2, 128, 64)
    small, pages = on_gpu(pool), len(pool["refs"])
    before = (1 << 32) // (2 * 64 * 128)
    far = {x: torch.empty((before + pages, *getattr(small, x).shape[1:]), dtype=getattr(small, x).dtype, device="cuda")
           for x in ("kc", "vc", "ks", "vs", "refs")}
    for x, to in far.items():
        to[before:] = getattr(small, x)
    table = torch.where(small.table >= 0, small.table + before, small.table)
    large = kvb.PagePool(far["kc"], far["vc"], far["ks"], far["vs"], table, small.lens.clone(), far["refs"])
    q = torch.from_numpy(rng.standard_normal((2 * samples, 8, 1, 128))).to(torch.bfloat16).cuda()
    a, b = small.share(ints(slots)), large.share(ints(slots))
    assert torch.equal(a.plan, b.plan) and int(a.count) > 0
    for x, y in zip(small.attend_shared(q, a, return_lse=True), large.attend_shared(q, b, return_lse=True)):
        assert torch.equal(x, y)


def test_a_plan_stays_good_while_sequences_grow(cuda_dev):
    rng = np.random.default_rng(11)
    pool, slots = family(rng, 100, [40, 64], 3, [1, 2, 3, 4, 5, 6], 2, 64, 16)
    g = on_gpu(pool)
    s = g.share(ints(slots))
    for new in (1, 30):
        cu = np.arange(7) * new
        k, v = (torch.randn(6 * new, 2, 64, device="cuda") for _ in "kv")
        small = dict(pool)
        start = O.extend(small, slots, [new] * 6)
        if start[0] < 0:                                        # the pool's spare pages are used up
            break
        assert np.array_equal(g.extend(ints(slots), ints([new] * 6)).cpu().numpy(), start)
        O.write(small, slots, start, cu, k.cpu().numpy(), v.cpu().numpy())
        g.write(ints(slots), ints(start), ints(cu), k, v)
        q = torch.from_numpy(rng.standard_normal((6, 4, 1, 64))).to(torch.float16).cuda()
        check(g, small, q, slots, shared=s)


def test_plans_that_are_none(cuda_dev):
    """Whatever a plan holds, no address is formed from it that does not fit; the status word tells."""
    rng = np.random.default_rng(12)
    pool, slots = family(rng, 200, [40, 64], 3, [9] * 6, 2, 64, 16)
    g = on_gpu(pool)
    q = torch.from_numpy(rng.standard_normal((6, 8, 2, 64))).to(torch.float16).cuda()
    good = g.share(ints(slots))
    want, plan = g.attend_shared(q, good), good.plan.clone()
    n = 6
    for at, value in ((0, -1), (3, 2 ** 31 - 1), (3 * n, -5), (3 * n, 6), (3 * n + 1, 0), (3 * n + 1, 1000), (3 * n + 2, 8), (3 * n + 2, -16),
                      (3 * n + 3, 2 ** 31 - 1), (3 * n + 4, 4), (3 * n + 4, -1)):
        good.plan[at] = value
        g.attend_shared(q, good)
        assert status() == 2, (at, value)
        good.plan.copy_(plan)
    for at, value in ((n, 2 ** 31 - 1), (n, -7), (2 * n, 100), (2 * n, -100), (8 * n, -3), (8 * n, 2 ** 30)):      # clamped
        good.plan[at] = value
        g.attend_shared(q, good)
        status()
        good.plan.copy_(plan)
    for seed in range(20):
        good.plan.copy_(ints(np.random.default_rng(seed).integers(-2 ** 31, 2 ** 31, 8 * n + 1, dtype=np.int64).astype(np.int32)))
        g.attend_shared(q, good)
        good.plan.copy_(ints(np.random.default_rng(seed).integers(0, 300, 8 * n + 1)))
        g.attend_shared(q, good)
    status()
    good.plan.copy_(plan)
    assert torch.equal(g.attend_shared(q, good), want)          # and leaves the workspace sound


def test_table_entries_that_are_no_page(cuda_dev):
    """They are nobody's: what is behind them is not shared, and tokens without a page are left out, as attend does."""
    rng = np.random.default_rng(13)
    pool, slots = family(rng, 200, [40], 4, [9] * 4, 2, 64, 16)
    pool["table"][slots, 5] = [-1, 10 ** 6, -1, -7]
    g = on_gpu(pool)
    s = check_share(g, pool, slots)
    assert s.own.tolist() == [80] * 4
    q = torch.from_numpy(rng.standard_normal((4, 4, 1, 64))).to(torch.float16).cuda()
    got, want = g.attend_shared(q, s), g.attend(q, ints(slots))
    assert status() == 2
    # both round weights and outputs: twice the bound of one, the values being below 0.025 127 e
    assert float((got - want).abs().max()) <= 2 * (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -13 + 2.0 ** -12) * 9


def test_more_sequences_than_one_launch_takes(cuda_dev):
    rng = np.random.default_rng(14)
    pool, slots = family(rng, 32, [16] * 75, 8, rng.integers(1, 40, 600), 1, 64, 16)
    g = on_gpu(pool)
    for tq in (1, 3):
        q = torch.from_numpy(rng.standard_normal((600, 2, tq, 64))).to(torch.float16).cuda()
        check_large(g, q, slots)


def test_refusals(cuda_dev):
    rng = np.random.default_rng(15)
    pool, slots = family(rng, 64, [20], 3, [1, 2, 3])
    g, other = on_gpu(pool), on_gpu(pool)
    s = g.share(ints(slots))
    q = torch.randn(3, 4, 1, 64, device="cuda").half()
    empty = g.share(ints([]))
    assert g.attend_shared(q[:0], empty).shape == (0, 1, 4, 64)
    for a in (dict(q=q[:2]), dict(q=q[..., :32]), dict(q=q.cpu()), dict(q=q[:, :3]), dict(out=q), dict(out=torch.empty(3, 1, 4, 64, device="cuda")),
              dict(scaling=float("inf"))):
        with pytest.raises(ValueError):
            g.attend_shared(**dict(dict(q=q, shared=s), **a))
    with pytest.raises(NotImplementedError):
        g.attend_shared(q.float(), s)
    with pytest.raises(ValueError, match="another table"):
        other.attend_shared(q, s)
    out = torch.empty(3, 1, 4, 64, device="cuda", dtype=torch.float16)
    assert g.attend_shared(q, s, out=out) is out
    shifted = torch.empty(3 * 256 + 2, device="cuda", dtype=torch.float16)[2:].view(3, 1, 4, 64)       # a 4-byte boundary will do
    assert torch.equal(g.attend_shared(q, s, out=shifted), out)
    wide = torch.randn(3, 4, 2, 64, device="cuda").half()
    wide[:, :, 1:] = q
    assert torch.equal(g.attend_shared(wide[:, :, 1:], s), out)


def test_streams_and_graphs(cuda_dev):
    """Steps of growing sequences in a captured graph (extend, write, share, attend_shared of two layers); two graphs replayed
    at once; calls on two streams."""
    rng = np.random.default_rng(16)
    pool, slots = family(rng, 100, [40, 70], 4, [1] * 8, 2, 64, 16)
    extra = O.empty_pool(len(pool["refs"]) + 200, 2, 64, 16, 10, 40)
    for x in ("kc", "vc", "ks", "vs", "refs"):
        extra[x][:len(pool[x])] = pool[x]
    extra["table"][:, :pool["table"].shape[1]] = pool["table"]
    extra["lens"][:] = pool["lens"]
    g = on_gpu(extra)
    h = g.add_layer()
    slot, one, cu = ints(slots), ints([1] * 8), ints(np.arange(9))
    q, k, v = torch.randn(8, 4, 1, 64, device="cuda").half(), torch.randn(8, 2, 64, device="cuda").half(), torch.randn(8, 2, 64, device="cuda").half()
    outs = [torch.empty(8, 1, 4, 64, device="cuda", dtype=torch.float16) for _ in "gh"]
    plans = []

    def step():
        start = g.extend(slot, one)
        s = g.share(slot)
        plans.append(s)
        for p, out in zip((g, h), outs):
            p.write(slot, start, cu, k, v)
            p.attend_shared(q, s, out=out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(40):
        q.normal_()
        k.normal_()
        v.normal_()
        graph.replay()
        if i % 13 == 0:
            torch.cuda.synchronize()
            want = {x: getattr(g, x).cpu().numpy() for x in NAMES}
            assert plans[-1].depth.tolist() == O.share(want, slots)["depth"]
            check(g, want, q, slots)
            for p, out in zip((g, h), outs):
                assert torch.equal(out, p.attend_shared(q, p.share(slot)))
    side = torch.cuda.Stream()
    s, want = g.share(slot), g.attend_shared(q, g.share(slot))
    two = []
    for _ in range(2):
        two.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(two[-1]):
            two.append([g.attend_shared(q, s) for _ in range(3)])
    side.wait_stream(torch.cuda.current_stream())
    here, there = [], []
    for _ in range(20):
        two[0].replay()
        here.append(g.attend_shared(q, s))
        with torch.cuda.stream(side):
            two[2].replay()
            there.append(g.attend_shared(q, s))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in here + there + two[1] + two[3])


@pytest.mark.parametrize("samples", [3, 30])
def test_many_calls_give_the_same_bits(cuda_dev, samples):
    rng = np.random.default_rng(17)
    n = 3 * samples
    pool, slots = family(rng, 300, [40, 500, 64], samples, rng.integers(1, 200, n), 2, 128, 64)
    g = on_gpu(pool)
    q = torch.from_numpy(rng.standard_normal((n, 8, 1, 128))).to(torch.bfloat16).cuda()
    s = g.share(ints(slots))
    want, same = g.attend_shared(q, s), torch.ones((), dtype=torch.bool, device="cuda")
    for _ in range(1000):
        t = g.share(s.slots)
        same &= (t.plan == s.plan).all() & (g.attend_shared(q, t) == want).all()
    assert bool(same)


def test_a_serving_step_with_an_encoder(cuda_dev):
    """As a decoder over an encoder's states would run: prompts prefilled, forked into samples, steps whose self-attention
    shares the prompts' pages and whose cross attention takes all samples of a prompt in one go over its states."""
    import kvb
    rng = np.random.default_rng(18)
    lens, states, samples, hq, hkv, d = [70, 33, 129], [500, 1, 77], 4, 8, 2, 64
    g = kvb.PagePool.create(80, hkv, d, 16, n_slots=15, max_blocks=30)
    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda").half()        # noqa: E731
    parents, children = ints([0, 1, 2]), ints(np.arange(3, 15))
    cu, ck = ints(cu_all := np.concatenate([[0], np.cumsum(lens)])), ints(np.concatenate([[0], np.cumsum(states)]))
    q, k, v = rand(sum(lens), hq, d), rand(sum(lens), hkv, d), rand(sum(lens), hkv, d)
    g.write(parents, g.extend(parents, ints(lens)), cu, k, v)
    kvb.prefill_attention(q, k, v, cu)
    ek, ev = rand(sum(states), hkv, d), rand(sum(states), hkv, d)
    first = kvb.cross_attention(q, ek, ev, cu, ck)
    g.fork(parents.repeat_interleave(samples), children)
    g.free(parents)
    per = ints(np.arange(4) * samples)
    for _ in range(20):
        start = g.extend(children, ints([1] * 12))
        s = g.share(children)
        g.write(children, start, ints(np.arange(13)), rand(12, hkv, d), rand(12, hkv, d))
        x = rand(12, hq, 1, d)
        out = g.attend_shared(x, s)
        y = kvb.cross_attention(out[:, 0], ek, ev, per, ck)
    assert s.count.tolist() == [3] and s.segments[:3, 1].tolist() == [4, 4, 4]
    pool = {x: getattr(g, x).cpu().numpy() for x in NAMES}
    check(g, pool, x, list(range(3, 15)), shared=s)
    for a, rows, lo, hi in ((out[:, 0], y, per.tolist(), ck.tolist()), (q, first, cu_all.tolist(), ck.tolist())):
        for i in range(3):
            for head in range(hq):
                kk, vv = ek[hi[i]:hi[i + 1], head // 4].double(), ev[hi[i]:hi[i + 1], head // 4].double()
                p = torch.softmax(a[lo[i]:lo[i + 1], head].double() @ kk.t() * d ** -0.5, -1)
                # 2 u + 2^-13 of the attended |v|, and 2^-24 max|v| per key
                tol = (2.0 ** -10 + 2.0 ** -12) * (p @ vv.abs()) + states[i] * 2.0 ** -24 * 6
                assert ((rows[lo[i]:lo[i + 1], head].double() - p @ vv).abs() <= tol).all()
