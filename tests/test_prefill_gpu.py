"""Causal attention of packed prompts on the GPU against float64, and its refusals.

Bound (u the unit roundoff, 2^-11 for float16 and 2^-8 for bfloat16): the weights are rounded to the inputs' type
before the product with the values (u, and 2^-25 absolutely per key where a float16 weight is subnormal), the
output once more (u); float32 sums and the exponential stay below 2^-13: |o - exact| <= (2 u + 2^-13 + 2 e) sum p|v| / l +
keys 2^-24 max|v|, e = d 2^-24 max sum |q k| scaling being the logits' round-off.  The log-sum-exp: e + 2^-14 (the
float32 sum and the exponential's relative error) + 2^-22 |lse|."""

import math

import numpy as np
import pytest
import torch

from oracle import paged as O

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def clean_status(cuda_dev):
    import kvb
    kvb.device_status()
    yield
    assert kvb.device_status() == 0, "a test left the device status word set"


def cu_of(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def exact(q, k, v, cu_q, cu_k, scaling):
    """The oracle's prefill in float64 on the GPU (tied to it by test_exact_is_the_oracle)."""
    hq, hkv = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mean_abs, lse = torch.zeros_like(out), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for a0, a1, b0, b1 in zip(cq, cq[1:], ck, ck[1:]):
        if a1 == a0 or b1 == b0:
            continue
        for a in range(hq):
            kk, vv = k[b0:b1, a * hkv // hq].double(), v[b0:b1, a * hkv // hq].double()
            s = q[a0:a1, a].double() @ kk.t() * scaling
            seen = torch.arange(b1 - b0, device="cuda") <= torch.arange(a1 - a0, device="cuda")[:, None] + (b1 - b0) - (a1 - a0)
            s = torch.where(seen, s, -math.inf)
            m = s.amax(1, keepdim=True)
            p = torch.where(seen, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
            l = p.sum(1, keepdim=True)
            vz = torch.where(torch.isfinite(vv), vv, 0.0)
            out[a0:a1, a] = torch.where(l > 0, p @ vz / l, 0.0)
            mean_abs[a0:a1, a] = torch.where(l > 0, p @ vz.abs() / l, 0.0)
            lse[a0:a1, a] = (m + l.log())[:, 0]
    return out, lse, mean_abs


def check(q, k, v, cu_q, cu_k, scaling=None, out_rows=slice(None), **kw):
    import kvb
    sc = q.shape[2] ** -0.5 if scaling is None else scaling
    out, lse = kvb.prefill_attention(q, k, v, cu_q, cu_k, scaling, return_lse=True, **kw)
    want, wl, mean_abs = exact(q, k, v, cu_q, cu_k, sc)
    u, d = U[q.dtype], q.shape[2]
    fin = torch.where(torch.isfinite(k.float()), k.float(), 0.0)
    e = d * 2.0 ** -24 * float(fin.abs().sum(-1).max() if k.numel() else 0) * float(q.float().abs().max()) * abs(sc)
    vmax = float(torch.where(torch.isfinite(v.float()), v.float(), 0.0).abs().max()) if v.numel() else 0.0
    keys = int((cu_k[1:] - cu_k[:-1]).max())
    tol = (2 * u + 2.0 ** -13 + 2 * e) * mean_abs + keys * 2.0 ** -24 * vmax
    got, gl = out.double()[out_rows], lse.double()[out_rows]
    want, wl, tol = want[out_rows], wl[out_rows], tol[out_rows]
    assert torch.isfinite(got).all()
    bad = (got - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() - tol).max()), [int(x) for x in bad.nonzero()[0]])
    seen = wl > -math.inf
    assert torch.equal(gl > -math.inf, seen) and (got[~seen] == 0).all()
    assert ((gl[seen] - wl[seen]).abs() <= e + 2.0 ** -14 + 2.0 ** -22 * wl[seen].abs()).all()
    assert torch.equal(kvb.prefill_attention(q, k, v, cu_q, cu_k, scaling), out)      # the same call, the same bits
    return out


def rand(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def test_exact_is_the_oracle(cuda_dev):
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((n, h, 16)) for n, h in ((9, 4), (12, 2), (12, 2)))
    a = O.prefill(q, k, v, [0, 3, 9], [0, 2, 12], 0.4)
    b = exact(*(torch.from_numpy(x).cuda() for x in (q, k, v)), cu_of([3, 6]), cu_of([2, 10]), 0.4)
    for x, y in zip(a, b):
        np.testing.assert_allclose(y.cpu().numpy(), x, rtol=1e-12, atol=1e-14)


CASES = [       # dtype, d, hkv, rep, query lengths, key lengths (None: the same)
    (torch.bfloat16, 128, 2, 4, [1], None),
    (torch.bfloat16, 128, 2, 4, [33, 1, 128, 7, 64, 0, 300], None),
    (torch.float16, 128, 1, 1, [127, 128, 129, 257, 513], None),
    (torch.float16, 64, 2, 4, [500, 31, 32, 33, 63, 65], None),
    (torch.bfloat16, 64, 1, 8, [1000, 16, 17], None),
    (torch.bfloat16, 64, 3, 1, [129, 640], None),
    (torch.float16, 128, 2, 3, [43, 42, 85, 400], None),                      # 128 is no multiple of the group
    (torch.bfloat16, 128, 1, 7, [37, 200], None),
    (torch.float16, 64, 1, 16, [9, 100], None),
    (torch.bfloat16, 128, 1, 64, [5, 40], None),
    (torch.float16, 128, 1, 80, [6, 21], None),
    (torch.bfloat16, 128, 2, 4, [1, 5, 64, 100], [4000, 77, 64, 1111]),       # chunks after their prefixes
    (torch.float16, 64, 2, 2, [130, 3], [2130, 515]),
    (torch.float16, 128, 2, 4, [50, 200, 10, 7], [20, 0, 10, 129]),           # rows that see nothing
    (torch.bfloat16, 64, 1, 4, [300], [5]),
    (torch.bfloat16, 128, 8, 4, [2500, 1500], None),
    (torch.float16, 64, 4, 2, [3001], [5000]),
]


@pytest.mark.parametrize("dtype,d,hkv,rep,ql,kl", CASES)
def test_prefill(cuda_dev, dtype, d, hkv, rep, ql, kl):
    g = torch.Generator(device="cuda").manual_seed(21)
    kl = kl or ql
    q, k, v = rand(g, sum(ql), hkv * rep, d, dtype=dtype), rand(g, sum(kl), hkv, d, dtype=dtype), rand(g, sum(kl), hkv, d, dtype=dtype)
    check(q, k, v, cu_of(ql), cu_of(kl))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prefill_many_short_sequences(cuda_dev, dtype):
    g = torch.Generator(device="cuda").manual_seed(22)
    ql = [(i * 7) % 41 for i in range(150)]
    q, k, v = rand(g, sum(ql), 8, 64, dtype=dtype), rand(g, sum(ql), 2, 64, dtype=dtype), rand(g, sum(ql), 2, 64, dtype=dtype)
    check(q, k, v, cu_of(ql), cu_of(ql))


def test_prefill_strided_views(cuda_dev):
    """Views of one projection's output, a (heads, tokens, d) layout, and rows that belong to no sequence."""
    g = torch.Generator(device="cuda").manual_seed(23)
    x = rand(g, 400, 4 + 2 + 2, 128, dtype=torch.bfloat16)
    cu = cu_of([150, 250])
    a = check(x[:, :4], x[:, 4:6], x[:, 6:], cu, cu)
    t = [y.transpose(0, 1).contiguous().transpose(0, 1) for y in (x[:, :4], x[:, 4:6], x[:, 6:])]
    assert torch.equal(check(*t, cu, cu), a)
    out = torch.full((400, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    import kvb
    kvb.prefill_attention(x[:, :4], x[:, 4:6], x[:, 6:], cu[:2], out=out)
    assert torch.equal(out[:150], a[:150]) and (out[150:] == 7).all()


@pytest.mark.parametrize("scale", [30.0, 1e-3])
def test_prefill_peaked_and_flat(cuda_dev, scale):
    """Logits whose running maximum jumps, and rows that attend to everything alike."""
    g = torch.Generator(device="cuda").manual_seed(24)
    q, k, v = rand(g, 700, 4, 128, dtype=torch.bfloat16), rand(g, 700, 1, 128, dtype=torch.bfloat16), rand(g, 700, 1, 128, dtype=torch.bfloat16)
    k *= torch.linspace(0.01, 2, 700, device="cuda")[:, None, None].to(torch.bfloat16)
    check(q * (scale ** 0.5), k, v, cu_of([700]), cu_of([700]))


def test_prefill_extreme_logits(cuda_dev):
    """Logits of thousands, keys that give -inf, all of them equal."""
    g = torch.Generator(device="cuda").manual_seed(25)
    q, v = rand(g, 300, 2, 64, dtype=torch.bfloat16), rand(g, 300, 1, 64, dtype=torch.bfloat16)
    k = torch.sign(rand(g, 300, 1, 64, dtype=torch.bfloat16)) * 0.5
    q2 = torch.sign(q) * 16
    check(q2, k, v, cu_of([300]), cu_of([300]), scaling=64.0)
    check(torch.zeros_like(q), k, v, cu_of([300]), cu_of([300]))


@pytest.mark.parametrize("scaling", [-0.1, 0.0, 1e-30])
def test_prefill_any_scaling(cuda_dev, scaling):
    g = torch.Generator(device="cuda").manual_seed(28)
    q, k, v = rand(g, 300, 4, 64, dtype=torch.float16), rand(g, 300, 2, 64, dtype=torch.float16), rand(g, 300, 2, 64, dtype=torch.float16)
    check(q, k, v, cu_of([100, 200]), cu_of([100, 200]), scaling)


SPLIT = [       # few rows over long keys: their items are computed in pieces
    (torch.float16, 64, 4, 4, [500, 1100], [7500, 1433]),
    (torch.bfloat16, 128, 1, 8, [1, 70, 3], [9001, 4000, 129]),
    (torch.bfloat16, 128, 2, 1, [200], [20000]),
    (torch.float16, 128, 1, 3, [5, 2000], [12345, 2000]),
    (torch.bfloat16, 64, 2, 2, [64] * 40, [1100 + 37 * i for i in range(40)]),
]


@pytest.mark.parametrize("dtype,d,hkv,rep,ql,kl", SPLIT)
def test_prefill_in_pieces(cuda_dev, dtype, d, hkv, rep, ql, kl):
    g = torch.Generator(device="cuda").manual_seed(29)
    q, k, v = rand(g, sum(ql), hkv * rep, d, dtype=dtype), rand(g, sum(kl), hkv, d, dtype=dtype), rand(g, sum(kl), hkv, d, dtype=dtype)
    check(q, k, v, cu_of(ql), cu_of(kl))
    check(3 * q, k, v, cu_of(ql), cu_of(kl))


def test_pieces_keep_non_finite_values_where_they_are_seen(cuda_dev):
    import kvb
    g = torch.Generator(device="cuda").manual_seed(30)
    q, k, v = rand(g, 40, 4, 128, dtype=torch.bfloat16), rand(g, 9000, 1, 128, dtype=torch.bfloat16), rand(g, 9000, 1, 128, dtype=torch.bfloat16)
    cu_q, cu_k = cu_of([40]), cu_of([9000])
    clean = check(q, k, v, cu_q, cu_k)
    for key in (100, 5000, 8965, 8999):
        p = v.clone()
        p[key, 0, 9] = float("nan")
        got = kvb.prefill_attention(q, k, p, cu_q, cu_k)
        first = max(0, key - 8960)                       # the first query that sees the key
        assert torch.equal(got[:first], clean[:first]) and torch.isnan(got[first:, :, 9]).all()
        assert torch.equal(got[..., :9], clean[..., :9]) and torch.equal(got[..., 10:], clean[..., 10:])


def test_prefill_reports_a_workspace_that_was_not_zero(cuda_dev):
    import kvb
    from kvb import paged
    q, k = torch.randn(40, 4, 64, device="cuda", dtype=torch.float16), torch.randn(9000, 1, 64, device="cuda", dtype=torch.float16)
    cu_q, cu_k = cu_of([40]), cu_of([9000])
    want = kvb.prefill_attention(q, k, k, cu_q, cu_k)
    for ws in paged._PREFILL_WS.values():
        ws[:16384] = 77
    kvb.prefill_attention(q, k, k, cu_q, cu_k)
    assert kvb.device_status() == 8
    for ws in paged._PREFILL_WS.values():
        ws[:16384] = 0
    assert torch.equal(kvb.prefill_attention(q, k, k, cu_q, cu_k), want) and kvb.device_status() == 0


@pytest.mark.parametrize("keys", [40, 2000])
def test_prefill_refuses_a_stream_capture(cuda_dev, keys):
    """Whether the call would make its workspace (many keys) or not; the stream works on afterwards."""
    import kvb
    q, k = torch.randn(40, 4, 64, device="cuda", dtype=torch.float16), torch.randn(keys, 2, 64, device="cuda", dtype=torch.float16)
    out = torch.zeros_like(q)
    cu_q, cu_k = cu_of([40]), cu_of([keys])
    want = kvb.prefill_attention(q, k, k, cu_q, cu_k)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for made in range(2):                                # without and with the stream's workspace
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=torch.cuda.current_stream()):
                with pytest.raises(NotImplementedError):
                    kvb.prefill_attention(q, k, k, cu_q, cu_k, out=out)
                q.mul_(1)
            assert torch.equal(kvb.prefill_attention(q, k, k, cu_q, cu_k), want)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,d", [(torch.float16, 128), (torch.bfloat16, 64)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_masked_places_do_not_matter(cuda_dev, dtype, d, poison):
    """Non-finite rows of other sequences and of a sequence's own later tokens leave the rows before them alone."""
    import kvb
    g = torch.Generator(device="cuda").manual_seed(26)
    ql = [70, 45, 200]
    q, k, v = rand(g, 315, 4, d, dtype=dtype), rand(g, 315, 2, d, dtype=dtype), rand(g, 315, 2, d, dtype=dtype)
    clean = check(q, k, v, cu_of(ql), cu_of(ql))
    kp, vp = k.clone(), v.clone()
    kp[70:115] = poison
    vp[70:115] = poison
    got = kvb.prefill_attention(q, kp, vp, cu_of(ql), cu_of(ql))
    assert torch.equal(got[:70], clean[:70]) and torch.equal(got[115:], clean[115:])
    assert not torch.isfinite(got[70:115].float()).any()
    for row in (115 + 3, 115 + 150):
        kp, vp = k.clone(), v.clone()
        kp[row, 0], vp[row, 1, 5] = poison, poison
        got = kvb.prefill_attention(q, kp, vp, cu_of(ql), cu_of(ql))
        assert torch.equal(got[:row], clean[:row])
        assert not torch.isfinite(got[row:, 2:, 5].float()).any()                    # a value that they all see
        assert torch.equal(got[row:, 2:, :5], clean[row:, 2:, :5]) and torch.equal(got[row:, 2:, 6:], clean[row:, 2:, 6:])


def test_prefill_refusals(cuda_dev):
    import kvb
    z = dict(device="cuda")
    q, k = torch.zeros(8, 4, 128, dtype=torch.bfloat16, **z), torch.zeros(8, 2, 128, dtype=torch.bfloat16, **z)
    cu = cu_of([8])
    bad = [
        (ValueError, (q.cpu(), k, k, cu)), (ValueError, (q, k.half(), k, cu)), (ValueError, (q[0], k, k, cu)),
        (ValueError, (q, k, k[:4], cu)), (ValueError, (q[:, :3], k, k, cu)), (ValueError, (q, k, k, cu.long())),
        (ValueError, (q, k, k, cu.cpu())), (ValueError, (q, k, k, cu, cu_of([4, 4]))), (ValueError, (q, k, k, cu[:0])),
        (NotImplementedError, (q.float(), k.float(), k.float(), cu)),
        (NotImplementedError, (q[:, :, :32].contiguous(), k[:, :, :32].contiguous(), k[:, :, :32].contiguous(), cu)),
        (ValueError, (q.transpose(1, 2), k.transpose(1, 2), k.transpose(1, 2), cu)),
    ]
    for kind, args in bad:
        with pytest.raises(kind):
            kvb.prefill_attention(*args)
    odd = torch.zeros(8 * 4 * 128 + 1, dtype=torch.bfloat16, **z)[1:].view(8, 4, 128)
    with pytest.raises(ValueError):
        kvb.prefill_attention(odd, k, k, cu)                          # rows off their 16-byte boundary
    with pytest.raises(ValueError):
        kvb.prefill_attention(q, k, k, cu, out=torch.zeros(8, 4, 128, **z))
    assert kvb.prefill_attention(q[:0], k[:0], k[:0], cu_of([0])).shape == (0, 4, 128)
    assert kvb.prefill_attention(q[:0], k[:0], k[:0], torch.zeros(1, dtype=torch.int32, **z)).shape == (0, 4, 128)
    out, lse = kvb.prefill_attention(q, k[:0], k[:0], cu, cu_of([0]), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    kvb.prefill_attention(q, k, k, cu, cu_of([9]))                    # keys past the rows
    assert kvb.device_status() == 2


def test_prefill_on_another_stream(cuda_dev):
    import kvb
    g = torch.Generator(device="cuda").manual_seed(27)
    q, k, v = rand(g, 900, 8, 128, dtype=torch.float16), rand(g, 900, 2, 128, dtype=torch.float16), rand(g, 900, 2, 128, dtype=torch.float16)
    cu = cu_of([300, 600])
    want = check(q, k, v, cu, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = [kvb.prefill_attention(q, k, v, cu) for _ in range(10)]
    b = [kvb.prefill_attention(q, k, v, cu) for _ in range(10)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in a + b)
