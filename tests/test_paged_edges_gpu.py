"""The paged path at the edges of what a caller may hand it: outputs of the wrong place, lengths that do not fit, graphs
that outlive a workspace, scales at the ends of their range."""

import numpy as np
import pytest
import torch

from oracle import paged as O

pytestmark = pytest.mark.gpu
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


def filled(rng, lens, hkv=1, d=64, page=16, spare=8, max_blocks=None, n_slots=None):
    """A pool of sequences 0 .. with rows of N(0, 1)."""
    nb = [O.blocks(n, page) for n in lens]
    pool = O.empty_pool(sum(nb) + spare, hkv, d, page, n_slots or len(lens), max_blocks or max(nb) + 2)
    O.extend(pool, range(len(lens)), lens)
    cu = np.concatenate([[0], np.cumsum(lens)])
    O.write(pool, range(len(lens)), [0] * len(lens), cu, *(rng.standard_normal((cu[-1], hkv, d)).astype(np.float32) for _ in "kv"))
    return pool


def test_outputs_and_inputs_of_another_place_are_refused(cuda_dev):
    """Refused on the host, nothing is launched."""
    import kvb
    rng = np.random.default_rng(1)
    g = on_gpu(filled(rng, [40, 7]))
    q, slots = torch.randn(2, 4, 1, 64, device="cuda", dtype=torch.float16), ints([0, 1])
    odd = torch.zeros(2 * 4 * 64 + 1, device="cuda", dtype=torch.float16)[1:].view(2, 1, 4, 64)
    for out in (torch.zeros(2, 1, 4, 64, dtype=torch.float16), odd):
        with pytest.raises(ValueError):
            g.attend(q, slots, out=out)
    for args in ((q.cpu(), slots), (q, slots.cpu())):
        with pytest.raises(ValueError):
            g.attend(*args)
    rows, start, cu = torch.zeros(2, 1, 64, device="cuda"), ints([40, 7]), ints([0, 1, 2])
    for args in ((slots, start, cu, rows.cpu(), rows), (slots, start, cu, rows, rows.cpu()), (slots, start.cpu(), cu, rows, rows)):
        with pytest.raises(ValueError):
            g.write(*args)
    p, cu = torch.zeros(8, 2, 64, device="cuda", dtype=torch.float16), ints([0, 8])
    for args, kw in (((p, p, p, cu), dict(out=p.cpu())), ((p, p.cpu(), p, cu), {}), ((p, p, p.cpu(), cu), {}), ((p, p, p, cu, cu.cpu()), {})):
        with pytest.raises(ValueError):
            kvb.prefill_attention(*args, **kw)
    assert not odd.any()


@pytest.mark.parametrize("length", [-1, -2 ** 31, 5 * 16 + 1, 2 ** 31 - 1])
def test_lengths_that_no_row_holds_are_refused_as_a_whole(cuda_dev, length):
    """The pool takes the caller's lengths: extend, and fork from and onto such a sequence, change nothing."""
    rng = np.random.default_rng(2)
    pool = filled(rng, [40, 7, 0], max_blocks=5, n_slots=4)
    pool["lens"][3] = length
    g = on_gpu(pool)
    for slots, add in (([3], [1]), ([0, 3], [1, 0]), ([3, 1], [0, 1])):
        assert (g.extend(ints(slots), ints(add)).cpu().numpy() == -1).all() and status() == 2
        same(g, pool)
    for src, dst in (([3], [2]), ([0], [3]), ([0, 3], [2, 1]), ([0, 1], [2, 3]), ([3], [3])):
        g.fork(ints(src), ints(dst))
        assert status() == 2
        same(g, pool)
    assert O.fork(pool, [0], [2])                       # the others go on
    g.fork(ints([0]), ints([2]))
    same(g, pool)


@pytest.mark.parametrize("n", [16, 17, 32])
def test_extend_refuses_needs_whose_sum_passes_32_bits(cuda_dev, n):
    """n sequences of 2^27 - 1 pages each: the sum is just below 2^31, above it, and just below 2^32."""
    import kvb
    blocks = 2 ** 27 - 1
    table = torch.empty(n, blocks, dtype=torch.int32, device="cuda")        # rows that the call may not touch
    z = dict(device="cuda")
    codes, scales = torch.full((40, 1, 16, 64), 128, dtype=torch.uint8, **z), torch.zeros(40, 1, **z)
    lens, refs = torch.zeros(n, dtype=torch.int32, **z), torch.zeros(40, dtype=torch.int32, **z)
    g = kvb.PagePool(codes, codes.clone(), scales, scales.clone(), table, lens, refs)
    start = g.extend(ints(range(n)), ints([blocks * 16] * n))
    assert status() == 16 and (start == -1).all() and not lens.any() and not refs.any()
    del g, table
    torch.cuda.empty_cache()


def test_a_captured_fork_and_compact_outlive_larger_calls(cuda_dev):
    """A later, larger fork takes another workspace; what the graph holds is still its own."""
    rng = np.random.default_rng(3)
    pool = filled(rng, [40, 33, 5] + [20] * 30, spare=80, n_slots=40)
    g = on_gpu(pool)
    src, dst = ints([0, 1]), ints([33, 34])
    with torch.cuda.stream(torch.cuda.Stream()):
        stream = torch.cuda.current_stream()
        g.fork(src, dst)
        g.compact()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            g.fork(src, dst)
            live = g.compact()
        many = list(range(3, 33))
        held = {ws.data_ptr(): ws.numel() for ws in g._ws.values()}
        g.fork(ints(many), ints(many))                  # larger: sequences kept as they are
    torch.cuda.synchronize()
    assert held.keys() - {ws.data_ptr() for ws in g._ws.values()}           # the workspace was replaced
    others = [torch.full((n,), 9, dtype=torch.uint8, device="cuda") for n in held.values() for _ in range(8)]
    assert not held.keys() & {x.data_ptr() for x in others}
    assert O.fork(pool, [0, 1], [33, 34])
    O.compact(pool)
    same(g, pool)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert O.fork(pool, [0, 1], [33, 34])
        assert int(live) == O.compact(pool)
        same(g, pool)
    assert all((x == 9).all() for x in others)


def test_attention_keeps_one_workspace_a_stream(cuda_dev):
    """Whatever the batches are, and for all layers of a table: they attend one after the other."""
    rng = np.random.default_rng(4)
    pool = filled(rng, [40, 33, 5, 20], hkv=2, d=64)
    g = on_gpu(pool)
    layers = [g] + [g.add_layer(*(x.clone() for x in (g.kc, g.vc, g.ks, g.vs))) for _ in range(3)]
    z = dict(device="cuda")
    wide = g.add_layer(torch.full((g.n_pages, 1, 16, 128), 128, dtype=torch.uint8, **z), torch.full((g.n_pages, 1, 16, 128), 128, dtype=torch.uint8, **z),
                       torch.zeros(g.n_pages, 1, **z), torch.zeros(g.n_pages, 1, **z))
    outs = []
    for n in (1, 2, 4, 3):
        for hq, tq in ((2, 1), (4, 3)):
            q = torch.from_numpy(rng.standard_normal((n, hq, tq, 64))).half().cuda()
            outs.append([p.attend(q, ints(range(n))) for p in layers])
    assert len(layers[-1]._ws) == 1 and sum(ws.numel() for ws in g._ws.values()) < 4 << 20
    assert all(torch.equal(x, row[0]) for row in outs for x in row)
    wide.attend(torch.zeros(1, 4, 1, 128, dtype=torch.float16, **z), ints([0]))         # needs a larger one
    assert len(g._ws) == 1 and torch.equal(layers[2].attend(q, ints(range(n))), outs[-1][0])


def check_scales(pool, g, q, slot, n):
    """One sequence against float64.  Beside the relative terms (bfloat16 output 2^-8, float16 weights 2^-11, float32 sums and
    exponentials 2^-13) a weight may be subnormal: 2^-25 of the largest p_j s_j a key, s_j = 127 scales being the most that the
    key's page can hold; the reference may lag behind by 2^8 and halve nothing, as the weights then only grow."""
    out, lse = g.attend(q, ints([slot]), 1.0, return_lse=True)
    out, lse = out.double().cpu().numpy()[0, 0], lse.double().cpu().numpy()[0, 0]
    k, v = (x.astype(np.float64) for x in O.rows(pool, slot, 0, n))
    page, rep = pool["kc"].shape[2], q.shape[1] // k.shape[1]
    most = 127.0 * pool["vs"][pool["table"][slot, np.arange(n) // page]].astype(np.float64)         # (n, Hkv)
    for a in range(q.shape[1]):
        h, qa = a // rep, q[0, a, 0].double().cpu().numpy()
        s = k[:, h] @ qa
        e = k.shape[2] * 2.0 ** -24 * float((np.abs(k[:, h]) @ np.abs(qa)).max())
        p = np.exp(s - s.max())
        p, want_lse = p / p.sum(), s.max() + np.log(p.sum())
        tol = (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -13 + 2 * e) * (p @ np.abs(v[:, h])) + n * 2.0 ** -25 * (p * most[:, h]).max()
        bad = np.abs(out[a] - p @ v[:, h]) > tol
        assert not bad.any(), (a, int(bad.sum()), out[a][bad][:4], (p @ v[:, h])[bad][:4])
        assert abs(lse[a] - want_lse) <= e + 2.0 ** -16 + 2.0 ** -22 * abs(want_lse)


SCALES = [      # magnitude of the values of each run of tokens; 0: pages of zeros
    [1e-6, 0, 1e-6, 1e-6],
    [1e-3, 1e-3, 0, 1e-3, 0],
    [0, 0, 1e-20],
    [2.0 ** -98, 1e12, 1],
    [1e12, 2.0 ** -98, 0, 1e-6],
    [2.0 ** -98],
    [1e30, 1e-28, 1e30],
]


@pytest.mark.parametrize("d,hq,run", [(64, 2, 48), (128, 4, 160), (128, 32, 200)])
@pytest.mark.parametrize("mags", SCALES)
def test_attention_over_values_of_any_scale(cuda_dev, mags, d, hq, run):
    """Pages of zeros take their mass and give no values; pages of tiny values keep both beside large ones."""
    rng = np.random.default_rng(5)
    n = run * len(mags) - 3
    nb = O.blocks(n, 16)
    pool = O.empty_pool(nb + 2, 2, d, 16, 1, nb)
    O.extend(pool, [0], [n])
    mag = np.repeat(mags, run)[:n, None, None]
    v = (rng.uniform(0.5, 1, (n, 2, d)) * rng.choice([-1, 1], (n, 1, 1)) * mag).astype(np.float32)
    k = rng.standard_normal((n, 2, d)).astype(np.float32)
    O.write(pool, [0], [0], [0, n], k, v)
    g = on_gpu(pool)
    for size in (0.03, 0.5):
        q = torch.from_numpy(size * rng.standard_normal((1, hq, 1, d))).bfloat16().cuda()
        check_scales(pool, g, q, 0, n)


def test_all_values_zero(cuda_dev):
    rng = np.random.default_rng(6)
    pool = O.empty_pool(8, 1, 64, 16, 1, 8)
    O.extend(pool, [0], [100])
    k = rng.standard_normal((100, 1, 64)).astype(np.float32)
    O.write(pool, [0], [0], [0, 100], k, 0 * k)
    out, lse = on_gpu(pool).attend(torch.randn(1, 2, 3, 64, device="cuda").half(), ints([0]), return_lse=True)
    assert (out == 0).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("page,gone", [(16, [1]), (16, [0, 4]), (64, [2]), (32, [0]), (16, list(range(13)))])
def test_pages_that_are_not_there_are_left_out(cuda_dev, page, gone):
    """Tokens whose page number does not fit have no mass: the others' mean is the result, the status word says so."""
    rng = np.random.default_rng(7)
    n = 200
    pool = filled(rng, [n], hkv=2, d=64, page=page, max_blocks=O.blocks(n, page))
    q = rng.standard_normal((1, 4, 1, 64)).astype(np.float32)
    q = torch.from_numpy(q).half().cuda()
    k, v = O.rows(pool, 0, 0, n)
    keep = ~np.isin(np.arange(n) // page, gone)
    hurt = {x: pool[x].copy() for x in NAMES}
    hurt["table"][0, gone] = [-1 if i % 2 else len(pool["refs"]) for i in range(len(gone))]
    out, lse = on_gpu(hurt).attend(q, ints([0]), return_lse=True)
    assert status() == 2
    for a in range(4):
        s = k[keep, a // 2].astype(np.float64) @ q[0, a, 0].double().cpu().numpy() / 8
        if not keep.any():
            assert (out == 0).all() and torch.isneginf(lse).all()
            break
        p = np.exp(s - s.max())
        want = p @ v[keep, a // 2] / p.sum()
        assert np.abs(out[0, 0, a].double().cpu().numpy() - want).max() <= 4 * 2.0 ** -10         # values below 4, weights and output of float16
        assert abs(float(lse[0, 0, a]) - (s.max() + np.log(p.sum()))) <= 1e-4


@pytest.mark.parametrize("page,tq,hq,lens", [(16, 150, 4, [300, 7, 0, 1000]), (128, 1, 2, [500] * 5), (16, 40, 32, [129])])
def test_attention_over_a_table_of_the_longest_rows(cuda_dev, page, tq, hq, lens):
    """Rows of 2^31 tokens: the call is divided over launches whose work fits 32 bits at any lengths, with the same bits."""
    import kvb
    rng = np.random.default_rng(8)
    pool = filled(rng, lens, hkv=2, d=64, page=page)
    g = on_gpu(pool)
    q = torch.from_numpy(rng.standard_normal((len(lens), hq, tq, 64))).half().cuda()
    want, lse = g.attend(q, ints(range(len(lens))), return_lse=True)
    table = torch.empty(len(lens), (2 ** 31 - 1) // page, dtype=torch.int32, device="cuda")
    table[:, :pool["table"].shape[1]] = g.table
    h = kvb.PagePool(g.kc, g.vc, g.ks, g.vs, table, g.lens, g.refs)
    got, gl = h.attend(q, ints(range(len(lens))), return_lse=True)
    err = (got.float() - want.float()).abs().max()
    assert err <= 2.0 ** -8 and torch.equal(torch.isneginf(gl), torch.isneginf(lse))       # other shares, other order of joining
    seen = ~torch.isneginf(lse)
    assert (gl - lse)[seen].abs().max() <= 2.0 ** -16 * 20


def test_attention_whose_work_passes_32_bits(cuda_dev):
    """Many query rows over a long sequence: 2^31 units of (token, row group) and more.  The last positions' rows are looked at."""
    rng = np.random.default_rng(9)
    n, tq, hq = 36000, 2 ** 19, 64
    pool = filled(rng, [n], hkv=1, d=64, page=128)
    g = on_gpu(pool)
    q = torch.zeros(1, hq, tq, 64, dtype=torch.float16, device="cuda")
    q[0, :, -3:] = torch.randn(hq, 3, 64, device="cuda")
    out = torch.full((1, tq, hq, 64), 7.0, dtype=torch.float16, device="cuda")
    got, lse = g.attend(q, ints([0]), out=out, return_lse=True)
    assert status() == 0 and (got[0, :tq - n] == 0).all() and torch.isneginf(lse[0, :tq - n]).all()
    k, v = (torch.from_numpy(x[:, 0]).double().cuda() for x in O.rows(pool, 0, 0, n))
    for t in range(3):
        seen = n - 2 + t
        s = q[0, :, tq - 3 + t].double() @ k[:seen].t() / 8
        want = torch.softmax(s, -1) @ v[:seen]
        assert (got[0, tq - 3 + t].double() - want).abs().max() <= 1e-3
    mean = v[:n - 1000].mean(0)
    assert (got[0, tq - 1001].double() - mean).abs().max() <= 1e-3                          # a query of zeros: the mean of what it sees
