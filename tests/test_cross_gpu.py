"""Attention of packed queries to keys of another length on the GPU against float64, and its refusals.

Bound (u the unit roundoff, 2^-11 for float16 and 2^-8 for bfloat16): the weights are rounded to the inputs' type before the
product with the values (u, and 2^-25 absolutely per key where a float16 weight is subnormal), the output once more (u); float32
sums and the exponential stay below 2^-13: |o - exact| <= (2 u + 2^-13 + 2 e) sum p|v| / l + keys 2^-24 max|v|, e = d 2^-24
max sum |q k| scaling being the logits' round-off.  The log-sum-exp: e + 2^-14 (the float32 sum and the exponential's
relative error) + 2^-22 |lse|."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def clean_status(cuda_dev):
    import kvb
    kvb.device_status()
    yield
    assert kvb.device_status() == 0, "a test left the device status word set"


def status():
    import kvb
    return kvb.device_status()


def cu_of(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def exact(q, k, v, cu_q, cu_k, scaling):
    """The definition in float64: out, lse and the attended mean of |v|."""
    hq, hkv = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mean_abs, lse = torch.zeros_like(out), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for a0, a1, b0, b1 in zip(cq, cq[1:], ck, ck[1:]):
        if a1 <= a0 or b1 <= b0:
            continue
        for a in range(hq):
            kk, vv = k[b0:b1, a * hkv // hq].double(), v[b0:b1, a * hkv // hq].double()
            s = q[a0:a1, a].double() @ kk.t() * scaling
            lse[a0:a1, a] = torch.logsumexp(s, 1)
            p = torch.softmax(s, 1)
            out[a0:a1, a], mean_abs[a0:a1, a] = p @ vv, p @ vv.abs()
    return out, lse, mean_abs


def check(q, k, v, cu_q, cu_k, scaling=None, rows=slice(None), **kw):
    import kvb
    sc = q.shape[2] ** -0.5 if scaling is None else scaling
    out, lse = kvb.cross_attention(q, k, v, cu_q, cu_k, scaling, return_lse=True, **kw)
    want, wl, mean_abs = exact(q, k, v, cu_q, cu_k, sc)
    u, d = U[q.dtype], q.shape[2]
    e = d * 2.0 ** -24 * float(k.float().abs().sum(-1).max() if k.numel() else 0) * float(q.float().abs().max()) * abs(sc)
    vmax = float(v.float().abs().max()) if v.numel() else 0.0
    keys = int((cu_k[1:] - cu_k[:-1]).max())
    tol = (2 * u + 2.0 ** -13 + 2 * e) * mean_abs + keys * 2.0 ** -24 * vmax
    got, gl = out.double()[rows], lse.double()[rows]
    want, wl, tol = want[rows], wl[rows], tol[rows]
    assert torch.isfinite(got).all()
    bad = (got - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() - tol).max()), [int(x) for x in bad.nonzero()[0]])
    seen = wl > -math.inf
    assert torch.equal(gl > -math.inf, seen) and (got[~seen] == 0).all()
    assert ((gl[seen] - wl[seen]).abs() <= e + 2.0 ** -14 + 2.0 ** -22 * wl[seen].abs()).all()
    assert torch.equal(kvb.cross_attention(q, k, v, cu_q, cu_k, scaling), out)      # the same call, the same bits
    return out


def rand(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def states(g, nk, hkv, d, dtype):
    """Keys and values as views of one projection, keys with strong channels."""
    kv = torch.randn(nk, 2 * hkv, d, generator=g, device="cuda")
    kv[:, :hkv] *= torch.exp(0.5 * torch.randn(hkv, d, generator=g, device="cuda"))
    kv = kv.to(dtype)
    return kv[:, :hkv], kv[:, hkv:]


CASES = [       # dtype, d, hkv, rep, queries, keys
    (torch.bfloat16, 128, 2, 4, [1], [1]),
    (torch.float16, 64, 3, 1, [1, 1, 1, 1], [31, 32, 33, 1000]),
    (torch.bfloat16, 128, 2, 4, [1] * 9, [15, 16, 17, 0, 127, 128, 129, 2000, 1]),
    (torch.float16, 128, 1, 8, [1, 0, 3, 2], [700, 50, 0, 1]),
    (torch.bfloat16, 64, 2, 5, [4, 1, 7], [64, 4097, 130]),
    (torch.float16, 128, 2, 2, [8, 5, 8, 1], [577, 1025, 33, 3001]),
    (torch.bfloat16, 128, 2, 4, [300], [200]),
    (torch.float16, 64, 1, 16, [129, 1, 64], [513, 100, 255]),
    (torch.bfloat16, 128, 1, 3, [43, 86, 200], [128, 127, 129]),
    (torch.float16, 128, 4, 1, [1000, 17, 0, 640], [63, 2049, 77, 640]),
    (torch.bfloat16, 64, 2, 4, [33, 64, 65], [1, 0, 1000]),
    (torch.float16, 128, 1, 128, [2, 1], [300, 77]),
    (torch.bfloat16, 128, 8, 4, [1] * 40, [(i * 37) % 300 for i in range(40)])]


@pytest.mark.parametrize("dtype,d,hkv,rep,queries,keys", CASES)
def test_cross(cuda_dev, dtype, d, hkv, rep, queries, keys):
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = states(g, sum(keys), hkv, d, dtype)
    q = rand(g, sum(queries), hkv * rep, d, dtype=dtype)
    check(q, k, v, cu_of(queries), cu_of(keys))
    check(3 * q, k, v, cu_of(queries), cu_of(keys), -0.11)
