"""The 8-bit page pool on the GPU against the numpy oracle: codes, scales, tables, lengths and reference counts
exact, attention within a derived bound of the float64 result, and the refusals.

Bound of an attention output (u the unit roundoff of a type: 2^-11 for float16, 2^-8 for bfloat16): the weights
are rounded to float16 (2^-11, and 2^-25 absolutely where that is subnormal, once per key), the output to its
type, and the logits carry float32 sums: |o - exact| <= (u_out + 2^-11 + 2^-13) sum p|v| / l + keys 2^-24 max|v|.
The log-sum-exp: the logits' sums of d products (d 2^-24 max sum |q k| scaling) and the float32 softmax sum (2^-16)."""

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


def same(g, pool, names=NAMES):
    for x in names:
        assert np.array_equal(getattr(g, x).cpu().numpy(), pool[x]), x


def cu_of(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)


def random_pool(rng, lens, hkv=2, d=64, page=16, spare=5, n_slots=None, scale=1.0):
    """A pool whose sequences have shuffled pages and codes of N(0, scale^2) rows."""
    n_slots = n_slots or len(lens) + 2
    nb = [O.blocks(n, page) for n in lens]
    n_pages = sum(nb) + spare
    pool = O.empty_pool(n_pages, hkv, d, page, n_slots, max(nb + [1]) + 2)
    perm, at = rng.permutation(n_pages), 0
    for s, (n, b) in enumerate(zip(lens, nb)):
        pool["table"][s, :b] = perm[at:at + b]
        pool["refs"][perm[at:at + b]] = 1
        pool["lens"][s] = n
        at += b
    # rows past a sequence's end and unused pages hold what earlier sequences left there
    pool["kc"][:] = rng.integers(1, 256, pool["kc"].shape)
    pool["vc"][:] = rng.integers(1, 256, pool["vc"].shape)
    pool["ks"][:] = pool["vs"][:] = 1e20
    cu = cu_of(lens)
    x = [(rng.standard_normal((cu[-1], hkv, d)) * scale).astype(np.float32) for _ in range(2)]
    O.write(pool, range(len(lens)), [0] * len(lens), cu, *x)
    return pool


# ------------------------------------------------------------------------------------------------
# write and read
# ------------------------------------------------------------------------------------------------
WRITES = [      # page, d, hkv, dtype, starts, new
    (64, 128, 8, torch.bfloat16, [0], [1000]),
    (16, 64, 2, torch.float16, [0, 5, 16, 31, 100], [1, 1, 16, 50, 0]),
    (32, 128, 3, torch.float32, [31, 0, 64], [1, 129, 31]),
    (128, 64, 1, torch.bfloat16, [127, 129, 0], [2, 300, 128]),
    (128, 128, 2, torch.float32, [3], [256]),
    (16, 128, 1, torch.float16, list(range(40)), [(7 * i) % 23 + 1 for i in range(40)]),
]


@pytest.mark.parametrize("page,d,hkv,dtype,starts,new", WRITES)
def test_write_codes_and_scales_are_exact(cuda_dev, page, d, hkv, dtype, starts, new):
    rng = np.random.default_rng(11)
    lens = [a + b for a, b in zip(starts, new)]
    pool = random_pool(rng, lens, hkv, d, page)
    g, cu = on_gpu(pool), cu_of(new)
    rows = rng.standard_normal((cu[-1], hkv, d)) * np.exp(rng.standard_normal((cu[-1], 1, 1)))
    k = torch.from_numpy(rows).to(dtype).cuda()
    # strided rows: every second head of a wider tensor
    wide = torch.zeros(cu[-1], 2 * hkv, d, dtype=dtype, device="cuda")
    wide[:, ::2] = k.flip(0)
    v = wide[:, ::2]
    slots = rng.permutation(len(lens))
    pool["table"][:len(lens)] = pool["table"][:len(lens)][np.argsort(slots)]
    pool["lens"][:len(lens)] = pool["lens"][:len(lens)][np.argsort(slots)]
    g = on_gpu(pool)
    O.write(pool, slots, starts, cu, k.float().cpu().numpy(), v.float().cpu().numpy())
    g.write(ints(slots), ints(starts), ints(cu), k, v)
    same(g, pool)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        gk, gv = g.read(ints(slots), ints(starts), ints(cu), int(cu[-1]), out)
        for i, s in enumerate(slots):
            if new[i]:
                for got, want in zip((gk, gv), O.rows(pool, s, starts[i], new[i])):
                    assert torch.equal(got[cu[i]:cu[i + 1]].cpu(), torch.from_numpy(want).to(out))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page,d", [(16, 64), (64, 128), (128, 128)])
def test_write_odd_values_of_16_bits_and_odd_addresses(cuda_dev, dtype, page, d):
    """Non-finite values among 16-bit rows, the largest and smallest magnitudes, rows off any 16-byte boundary."""
    rng = np.random.default_rng(19)
    n = 3 * page + 5
    pool = O.empty_pool(4, 1, d, page, 1, 4)
    O.extend(pool, [0], [n])
    g = on_gpu(pool)
    x = torch.from_numpy(rng.standard_normal((n, 1, d)) * np.exp(2 * rng.standard_normal((n, 1, 1)))).to(dtype)
    y = x.flip(0).clone()
    x[2, 0, 3], x[page, 0, 1], x[page + 1, 0, 2], x[2 * page:3 * page] = float("nan"), float("inf"), -float("inf"), 0
    y[:page] *= torch.finfo(dtype).tiny
    y[page:2 * page, 0, 7] = torch.finfo(dtype).max
    y[2 * page:3 * page] = float("nan")
    odd = torch.empty(n * (d + 3) + 1, dtype=dtype, device="cuda")[1:].view(n, 1, d + 3)[:, :, :d]
    odd.copy_(y)
    O.write(pool, [0], [0], [0, n], x.float().numpy(), y.float().numpy())
    for v in (y.cuda(), odd):
        g.write(ints([0]), ints([0]), ints([0, n]), x.cuda(), v)
        same(g, pool)


def test_write_takes_odd_values(cuda_dev):
    """NaN and infinities, rows of zeros, values near the smallest and largest magnitudes, a larger scale later."""
    pool = O.empty_pool(3, 1, 64, 16, 1, 3)
    O.extend(pool, [0], [40])
    g = on_gpu(pool)
    rng = np.random.default_rng(5)
    x = rng.standard_normal((40, 1, 64)).astype(np.float32)
    x[3, 0, 5], x[4, 0, 6], x[5, 0, 7] = np.nan, np.inf, -np.inf
    x[16:32] = 0
    y = np.zeros_like(x)
    y[:16] = 1e-35 * rng.standard_normal((16, 1, 64))
    y[16:] = 3e38 * rng.uniform(-1, 1, (24, 1, 64))
    for a, b in ((0, 1), (1, 2), (2, 18), (18, 40)):
        O.write(pool, [0], [a], [0, b - a], x[a:b], y[a:b])
        g.write(ints([0]), ints([a]), ints([0, b - a]), torch.from_numpy(x[a:b]).cuda(), torch.from_numpy(y[a:b]).cuda())
        same(g, pool)
    inf = torch.full((1, 1, 64), float("inf"), device="cuda")
    g.write(ints([0]), ints([39]), ints([0, 1]), inf, -inf)
    O.write(pool, [0], [39], [0, 1], inf.cpu().numpy(), -inf.cpu().numpy())
    same(g, pool)


def test_write_leaves_out_what_it_may_not_touch(cuda_dev):
    rng = np.random.default_rng(6)
    pool = random_pool(rng, [20, 20], n_slots=2)
    pool["refs"][pool["table"][1, 1]] = 2               # shared
    g = on_gpu(pool)
    x = torch.randn(4, 2, 64, device="cuda")
    for slots, start, bits in (([0], [-1], 0), ([2], [0], 2), ([-1], [0], 2), ([1], [16], 2), ([0], [60], 2), ([0], [1 << 30], 2)):
        g.write(ints(slots), ints(start), ints([0, 4]), x, x)
        assert status() == bits
        same(g, pool)
    g.write(ints([0]), ints([0]), ints([0, 5]), x, x)   # offsets past the rows
    assert status() == 2
    same(g, pool)
    g.write(ints([]), ints([]), ints([0]), x, x)
    g.write(ints([0]), ints([0]), ints([0, 0]), x[:0], x[:0])
    same(g, pool)


# ------------------------------------------------------------------------------------------------
# page tables
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n_pages", [40, 1024, 33000, 70001])
def test_extend_takes_the_lowest_free_pages(cuda_dev, n_pages):
    rng = np.random.default_rng(7)
    pool = O.empty_pool(n_pages, 1, 64, 16, 50, 4000)
    pool["refs"][:] = rng.random(n_pages) < 0.6
    pool["refs"][-1] = 0
    g = on_gpu(pool)
    slots = rng.permutation(50)[:33]
    limit = (n_pages - pool["refs"].sum()) * 16 // 2 // 33
    for _ in range(2):
        add = rng.integers(0, limit, 33)
        add[3] = 0
        got, want = g.extend(ints(slots), ints(add)), O.extend(pool, slots, add)
        assert np.array_equal(got.cpu().numpy(), want) and status() == (16 if want[0] < 0 else 0)
        same(g, pool)


def test_extend_refuses_as_a_whole(cuda_dev):
    pool = O.empty_pool(10, 1, 64, 16, 4, 8)
    g = on_gpu(pool)
    for slots, add, bits in (([0, 1], [100, 65], 16), ([0], [129], 2), ([4], [1], 2), ([0, -1], [1, 1], 2), ([0], [-1], 2)):
        got = g.extend(ints(slots), ints(add))
        assert (got.cpu().numpy() == -1).all() and status() == bits
        same(g, pool)
    O.extend(pool, [0, 1], [100, 48])                   # exactly all
    assert (g.extend(ints([0, 1]), ints([100, 48])).cpu().numpy() == 0).all()
    same(g, pool)


FORKS = [       # lens, src, dst
    ([40, 16, 1, 77, 0, 5, 0, 0], [0, 3, 4], [5, 6, 7]),
    ([40, 33, 17, 64], [1, 0, 0, 2], [0, 1, 2, 3]),            # permuted, one parent twice, one dropped
    ([40, 33, 17], [0, 0, 2], [0, 1, 2]),                      # kept as they are
    ([200, 0, 0, 0, 0, 0, 0, 0, 0], [0] * 8, list(range(1, 9))),
]


@pytest.mark.parametrize("lens,src,dst", FORKS)
@pytest.mark.parametrize("page,d,hkv", [(16, 64, 2), (64, 128, 8), (128, 64, 3)])
def test_fork_free_compact_follow_the_oracle(cuda_dev, lens, src, dst, page, d, hkv):
    rng = np.random.default_rng(8)
    pool = random_pool(rng, lens, hkv, d, page, spare=23)
    g = on_gpu(pool)
    for _ in range(3):
        assert O.fork(pool, src, dst)
        g.fork(ints(src), ints(dst))
        same(g, pool)
    gone = [dst[0], dst[0]]                                    # a slot named twice is freed once
    O.free(pool, gone[:1])
    g.free(ints(gone))
    same(g, pool)
    n = O.compact(pool)
    assert int(g.compact()) == n
    same(g, pool)
    assert int(g.compact()) == n
    same(g, pool)


@pytest.mark.parametrize("n_pages", [100, 33000, 70001])
def test_compact_large_pools(cuda_dev, n_pages):
    rng = np.random.default_rng(9)
    pool = O.empty_pool(n_pages, 1, 64, 16, 8, n_pages // 10 + 1)
    perm = rng.permutation(n_pages)
    for s in range(8):
        n = n_pages // 20 + s % 3
        pool["table"][s, :n] = perm[s * (n_pages // 10):][:n]
        pool["lens"][s] = n * 16 - s
        pool["refs"][pool["table"][s, :n]] = 1
    pool["kc"][:, 0, 0, 0] = np.arange(n_pages) % 251 + 1
    pool["vs"][:, 0] = np.arange(n_pages)
    g = on_gpu(pool)
    assert int(g.compact()) == O.compact(pool)
    same(g, pool)


def test_layers_of_one_table(cuda_dev):
    """fork, compact and copy_pages on the first pool move the pages of every layer and change the table once."""
    rng = np.random.default_rng(20)
    pool = random_pool(rng, [40, 33, 64, 0], 2, 64, 16, spare=9)
    other = {x: pool[x].copy() for x in NAMES}
    other["kc"], other["vs"] = rng.integers(1, 256, pool["kc"].shape).astype(np.uint8), rng.random(pool["vs"].shape, np.float32)
    g = on_gpu(pool)
    h = g.add_layer(*[torch.from_numpy(other[x].copy()).cuda() for x in ("kc", "vc", "ks", "vs")])
    for p in (pool, other):
        O.fork(p, [0, 1], [3, 4])
        O.free(p, [0, 2])
        O.compact(p)
        O.copy_page(p, 1, len(p["refs"]) - 1)
    g.fork(ints([0, 1]), ints([3, 4]))
    g.free(ints([0, 2]))
    g.compact()
    g.copy_pages(ints([1]), ints([len(pool["refs"]) - 1]))
    same(g, pool)
    same(h, other)
    with pytest.raises(ValueError):
        g.add_layer(*[x[:-1] for x in (h.kc, h.vc, h.ks, h.vs)])
    q = torch.randn(1, 4, 1, 64, device="cuda", dtype=torch.float16)
    check_attend(h, other, q, [4])


def test_fork_and_free_refusals(cuda_dev):
    rng = np.random.default_rng(10)
    pool = random_pool(rng, [20, 33, 0], spare=1)
    g = on_gpu(pool)
    for src, dst, bits in (([0, 1], [2, 3], 16), ([0], [5], 2), ([-1], [2], 2), ([9], [2], 2)):
        g.fork(ints(src), ints(dst))
        assert status() == bits
        same(g, pool)
    g.free(ints([5, -1]))
    assert status() == 2
    g.copy_pages(ints([0]), ints([99]))
    assert status() == 2
    same(g, pool)
    g.copy_pages(ints([0, 2]), ints([1, 3]))
    O.copy_page(pool, 0, 1)
    O.copy_page(pool, 2, 3)
    same(g, pool)


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
def check_attend(g, pool, q, slots, scaling=None, **kw):
    d = q.shape[-1]
    sc = d ** -0.5 if scaling is None else scaling
    out, lse = g.attend(q, ints(slots), scaling, return_lse=True, **kw)
    want, wl, mean_abs = O.attend(pool, q.float().cpu().numpy(), slots, sc)
    vmax = max([float(np.abs(O.rows(pool, s, 0, pool["lens"][s])[1]).max(initial=0)) for s in slots] + [0])
    kmax = max([float(np.abs(O.rows(pool, s, 0, pool["lens"][s])[0]).sum(-1).max(initial=0)) for s in slots] + [0])
    keys = int(max(pool["lens"][list(slots)]))
    logit = d * 2.0 ** -24 * kmax * float(q.float().abs().max()) * sc
    tol = (U[q.dtype] + 2.0 ** -11 + 2.0 ** -13 + 2 * logit) * mean_abs + keys * 2.0 ** -24 * vmax
    got = out.double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all()
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) - tol).max()))
    gl = lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(gl), np.isneginf(wl))
    seen = ~np.isneginf(wl)
    assert (np.abs(gl[seen] - wl[seen]) <= logit + 2.0 ** -16 + 2.0 ** -22 * np.abs(wl[seen])).all()
    assert (got[~seen] == 0).all()
    assert torch.equal(g.attend(q, ints(slots), scaling), out)          # the same call gives the same bits
    return out


ATTENDS = [     # dtype, d, page, hkv, rep, tq, lens
    (torch.float16, 128, 64, 2, 4, 1, [1, 15, 16, 17, 63, 64, 65, 200]),
    (torch.bfloat16, 128, 16, 1, 8, 1, [4097, 0, 1]),
    (torch.bfloat16, 64, 32, 4, 1, 1, [31, 32, 33, 1000]),
    (torch.float16, 64, 128, 2, 3, 1, [127, 128, 129, 777]),
    (torch.float16, 128, 32, 2, 4, 3, [1, 2, 3, 4, 100, 515]),          # rows before the sequence's start: empty
    (torch.bfloat16, 64, 16, 2, 5, 7, [6, 7, 8, 1030, 0]),
    (torch.float16, 128, 128, 1, 16, 4, [900, 2049]),
    (torch.bfloat16, 128, 64, 3, 2, 40, [39, 41, 350]),
    (torch.float16, 128, 64, 8, 8, 1, [3000] * 5 + [7]),
]


@pytest.mark.parametrize("dtype,d,page,hkv,rep,tq,lens", ATTENDS)
def test_attend(cuda_dev, dtype, d, page, hkv, rep, tq, lens):
    rng = np.random.default_rng(12)
    pool = random_pool(rng, lens, hkv, d, page)
    g = on_gpu(pool)
    slots = rng.permutation(len(lens))
    q = torch.from_numpy(rng.standard_normal((len(lens), hkv * rep, tq, d))).to(dtype).cuda()
    check_attend(g, pool, q, slots)
    check_attend(g, pool, q, slots, 0.02)


def test_attend_long_context(cuda_dev):
    """One long sequence over many blocks of work, and a batch of one: the split over the cache and its joining."""
    rng = np.random.default_rng(13)
    pool = random_pool(rng, [30001, 5], 1, 128, 64)
    q = torch.from_numpy(rng.standard_normal((1, 4, 1, 128))).half().cuda()
    check_attend(on_gpu(pool), pool, q, [0])
    check_attend(on_gpu(pool), pool, 3 * q, [0])


@pytest.mark.parametrize("d", [64, 128])
def test_attend_pages_of_very_different_scales(cuda_dev, d):
    """Keys and values of 1e-6, 1 and 30 in one sequence, pages of zeros, a query of large and small entries."""
    rng = np.random.default_rng(14)
    pool = O.empty_pool(64, 2, d, 16, 1, 64)
    O.extend(pool, [0], [640])
    x = rng.standard_normal((2, 640, 2, d)).astype(np.float32)
    mag = np.repeat([1e-6, 1, 30, 0, 1e-12, 2, 0.1, 5], 80)[None, :, None, None].astype(np.float32)
    kk, vv = x[0] * np.minimum(mag[0], 2), x[1] * mag[0, ::-1]
    O.write(pool, [0], [0], [0, 640], kk, vv)
    q = torch.from_numpy(rng.standard_normal((1, 8, 2, d)) * np.array([1, 1e-3, 3, 1e-5, 1, 0, 2, 1])[None, :, None, None]).half().cuda()
    check_attend(on_gpu(pool), pool, q, [0])


def test_attend_peaked_and_flat(cuda_dev):
    rng = np.random.default_rng(15)
    pool = random_pool(rng, [2000], 1, 128, 32)
    g = on_gpu(pool)
    k, _ = O.rows(pool, 0, 0, 2000)
    q = torch.from_numpy(np.stack([k[1234, 0] * 2, k[3, 0] * 2, k[1999, 0] * 2, 0 * k[0, 0]]))[None, :, None].to(torch.bfloat16).cuda()
    check_attend(g, pool, q, [0], 0.5)


@pytest.mark.parametrize("scaling", [-0.1, 0.0, 1e-30])
def test_attend_any_scaling(cuda_dev, scaling):
    rng = np.random.default_rng(21)
    pool = random_pool(rng, [333, 20], 2, 64, 16)
    q = torch.from_numpy(rng.standard_normal((2, 4, 3, 64))).half().cuda()
    out, lse = on_gpu(pool).attend(q, ints([0, 1]), scaling, return_lse=True)
    want, wl, mean_abs = O.attend(pool, q.float().cpu().numpy(), [0, 1], scaling)
    assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -9 * mean_abs + 1e-4).all()
    assert np.abs(lse.double().cpu().numpy() - wl).max() <= 1e-3


def test_attend_more_sequences_than_one_launch_takes(cuda_dev):
    rng = np.random.default_rng(22)
    lens = [(i * 7) % 50 for i in range(1100)]
    pool = random_pool(rng, lens, 1, 64, 16)
    slots = rng.permutation(1100)
    q = torch.from_numpy(rng.standard_normal((1100, 2, 1, 64))).half().cuda()
    check_attend(on_gpu(pool), pool, q, slots)


def test_attend_rows_do_not_touch_each_other(cuda_dev):
    """NaN and infinities in one query leave the other rows as they are."""
    rng = np.random.default_rng(23)
    pool = random_pool(rng, [700, 90], 2, 128, 32)
    g = on_gpu(pool)
    q = torch.from_numpy(rng.standard_normal((2, 8, 2, 128))).half().cuda()
    clean = g.attend(q, ints([0, 1]))
    for bad in (float("nan"), float("inf")):
        p = q.clone()
        p[0, 3, 1, 7] = bad
        got = g.attend(p, ints([0, 1]))
        assert not torch.isfinite(got[0, 1, 3]).any()
        got[0, 1, 3] = clean[0, 1, 3]
        assert torch.equal(got, clean)


def test_attend_reports_a_workspace_that_was_not_zero(cuda_dev):
    rng = np.random.default_rng(24)
    g = on_gpu(random_pool(rng, [30000], 1, 64, 64))
    q = torch.randn(1, 2, 1, 64, device="cuda", dtype=torch.float16)
    g.attend(q, ints([0]))
    for ws in g._ws.values():
        ws[:1024] = 77
    g.attend(q, ints([0]))
    assert status() == 8


def test_many_sequences_in_one_call(cuda_dev):
    rng = np.random.default_rng(25)
    n = 1500
    pool = O.empty_pool(5000, 1, 64, 16, 2 * n, 4)
    g = on_gpu(pool)
    slots, add = rng.permutation(2 * n)[:n], rng.integers(0, 30, n)
    got = g.extend(ints(slots), ints(add))
    assert np.array_equal(got.cpu().numpy(), O.extend(pool, slots, add))
    same(g, pool)
    dst = rng.permutation(2 * n)[:n]
    assert O.fork(pool, slots, dst)
    g.fork(ints(slots), ints(dst))
    same(g, pool)
    O.free(pool, slots[:700])
    g.free(ints(slots[:700]))
    assert int(g.compact()) == O.compact(pool)
    same(g, pool)


def test_attend_refuses_what_does_not_fit(cuda_dev):
    rng = np.random.default_rng(16)
    pool = random_pool(rng, [100, 50])
    g = on_gpu(pool)
    q = torch.randn(1, 4, 1, 64, device="cuda", dtype=torch.float16)
    for bad in ([4], [-1]):
        g.attend(q, ints(bad))
        assert status() == 2
    hurt = {x: pool[x].copy() for x in NAMES}
    hurt["table"][0, 2] = len(pool["refs"])
    h = on_gpu(hurt)
    h.attend(q, ints([0]))
    assert status() == 2
    check_attend(h, hurt, q, [1])                       # the other sequence, and the workspace, are sound
    assert g.attend(q[:0], ints([])).shape == (0, 1, 4, 64)


def test_attend_on_another_stream_and_strided_queries(cuda_dev):
    rng = np.random.default_rng(17)
    pool = random_pool(rng, [1000, 300], 2, 128, 64)
    g = on_gpu(pool)
    base = torch.randn(2, 3, 8, 128, device="cuda", dtype=torch.float16)
    q = base.transpose(1, 2)                            # (2, 8, 3, 128), strided
    want = check_attend(g, pool, q, [0, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    with torch.cuda.stream(side):
        for _ in range(20):
            outs.append(g.attend(q, ints([0, 1])))
    here = [g.attend(q, ints([0, 1])) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs + here)


def test_decode_steps_in_a_captured_graph(cuda_dev):
    """extend, write and attend are captured once; replays serve the growing sequences."""
    rng = np.random.default_rng(18)
    pool = random_pool(rng, [30, 15, 0], 2, 64, 16, spare=40, n_slots=3)
    pool["table"] = np.pad(pool["table"], ((0, 0), (0, 12)), constant_values=-1)
    g = on_gpu(pool)
    slots, one, cu = ints([2, 0, 1]), ints([1, 1, 1]), ints([0, 1, 2, 3])
    k, v = (torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q, out = torch.zeros(3, 4, 1, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(3, 1, 4, 64, device="cuda", dtype=torch.bfloat16)

    def step():
        start = g.extend(slots, one)
        g.write(slots, start, cu, k, v)
        g.attend(q, slots, out=out)

    with torch.cuda.stream(torch.cuda.Stream()):
        start = torch.full((3,), -1, dtype=torch.int32, device="cuda")
        g.write(slots, start, cu, k, v)                 # loads the kernels and the workspaces: changes nothing
        g.extend(slots, torch.zeros_like(one))
        stream = torch.cuda.current_stream()
        g.attend(q, slots, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for i in range(20):
        x = torch.from_numpy(rng.standard_normal((2, 3, 2, 64))).to(torch.bfloat16)
        k.copy_(x[0]), v.copy_(x[1])
        q.copy_(torch.from_numpy(rng.standard_normal((3, 4, 1, 64))))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        start = O.extend(pool, [2, 0, 1], [1, 1, 1])
        O.write(pool, [2, 0, 1], start, [0, 1, 2, 3], x[0].float().numpy(), x[1].float().numpy())
        same(g, pool)
        want, _, mean_abs = O.attend(pool, q.float().cpu().numpy(), [2, 0, 1], 64 ** -0.5)
        assert (np.abs(out.double().cpu().numpy() - want) <= (2.0 ** -8 + 2.0 ** -10) * mean_abs + 1e-4).all()
