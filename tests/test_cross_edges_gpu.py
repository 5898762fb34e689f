"""Cross attention at the ends of its ranges; bounds as in test_cross_gpu."""

import pytest
import torch

from test_cross_gpu import clean_status, cu_of, rand, status      # noqa: F401

pytestmark = pytest.mark.gpu


def wide_keys(g, used, rows, hkv):
    """Rows for many more keys than the sequences have, one head for all KV heads; NaN where no sequence is."""
    one = torch.full((rows, 1, 64), float("nan"), dtype=torch.float16, device="cuda")
    one[:used] = rand(g, used, 1, 64, dtype=torch.float16)
    return one.expand(-1, hkv, -1)


def test_many_sequences_over_many_rows(cuda_dev):
    """1100 single queries, states in a buffer of four million rows: the product of all of both passes 32 bits, the work does not."""
    import kvb
    g = torch.Generator(device="cuda").manual_seed(1)
    keys = [(i * 7) % 40 for i in range(1100)]
    k = wide_keys(g, sum(keys), 1 << 22, 16)
    q = rand(g, 1100, 16, 64, dtype=torch.float16)
    want = kvb.cross_attention(q, k[:sum(keys)], k[:sum(keys)], cu_of([1] * 1100), cu_of(keys))
    assert torch.equal(kvb.cross_attention(q, k, k, cu_of([1] * 1100), cu_of(keys)), want)


@pytest.mark.parametrize("rows", [1 << 20, 4])
def test_a_sequence_of_too_much_work_is_left_out(cuda_dev, rows):
    """4096 x 16 groups of rows by 65534 units of keys, and one that fits beside it; few rows: 32768 heads by 131069 units."""
    import kvb
    g = torch.Generator(device="cuda").manual_seed(2)
    many = rows > 4
    heads, nk = (16, 1 << 22) if many else (32768, 1 << 22)
    k = wide_keys(g, 100, nk, heads)
    q = rand(g, 1, heads, 64, dtype=torch.float16).expand(rows + 2, -1, -1)
    cq = torch.tensor([0, 2, rows + 2], dtype=torch.int32, device="cuda")
    ck = torch.tensor([0, 100, nk], dtype=torch.int32, device="cuda")
    out = torch.full((rows + 2, heads, 64), 3, dtype=torch.float16, device="cuda")
    kvb.cross_attention(q, k, k, cq, ck, out=out)
    assert status() == 2 and (out[2:] == 3).all()
    want = kvb.cross_attention(q[:2], k[:100], k[:100], cu_of([2]), cu_of([100]))
    # the first sequence may run on the kernel for many rows here and on that for few alone: twice the bound of one, the attended
    # mean of |v| below its maximum
    top = float(k[:100, 0].float().abs().max())
    e = 64 * 2.0 ** -24 * float(k[:100, 0].float().abs().sum(-1).max()) * float(q[0].float().abs().max()) / 8
    assert ((out[:2].float() - want.float()).abs() <= 2 * (2.0 ** -10 + 2.0 ** -13 + 2 * e + 100 * 2.0 ** -24) * top).all()


def rows_of_digits(units, dtype):
    """256 queries whose logits are 0 for the first key of every 64 and -x for the others, x from 0 to 1.5 in steps that either
    type holds: (x, the exact log-sum-exp over `units` such 64 keys, the bound of its error).  Of the weights 2^(-x log2 e) a
    quarter comes from the polynomial (2.8e-6), the rest from ex2.approx (2^-22), each from an argument that was rounded twice
    (2 2^-24 x relatively); a unit's sum has at most 32 roundings in a row, the sum over units one each; the logarithm and its product
    with the maximum 2^-22 |lse|."""
    x = torch.arange(256, dtype=torch.float64, device="cuda") * (2.0 ** -7 if dtype == torch.bfloat16 else 1.5 / 256)
    if dtype == torch.bfloat16:                                 # eight digits: from 1 on every second one
        x = torch.where(x < 1, x, 1 + (x - 1).mul(64).floor() / 64).clamp(max=1.5)
    lse = torch.log(units * (1 + 63 * torch.exp(-x)))
    argument = 2 * 2.0 ** -24 * x
    tol = (2.8e-6 + argument) / 4 + (2.0 ** -22 + argument) * 3 / 4 + (32 + units) * 2.0 ** -24 + 2.0 ** -22 * lse.abs()
    return x, lse, tol


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,units", [(64, 16), (128, 3)])
def test_the_log_sum_exp_keeps_the_digits_of_float32(cuda_dev, dtype, d, units):
    import kvb
    x, lse, tol = rows_of_digits(units, dtype)
    q = torch.zeros(256, 1, d, dtype=dtype, device="cuda")
    q[:, 0, 0] = -x
    assert torch.equal(q[:, 0, 0].double(), -x) and float(tol.max()) < 1e-5
    k = torch.zeros(64 * units, 1, d, dtype=dtype, device="cuda")
    k[torch.arange(64 * units, device="cuda") % 64 > 0, 0, 0] = 1
    _, got = kvb.cross_attention(q, k, k, cu_of([256]), cu_of([64 * units]), 1.0, return_lse=True)
    bad = (got[:, 0].double() - lse).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got[:, 0].double() - lse).abs() / tol).max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_log_sum_exp_of_shared_pages_keeps_the_digits_of_float32(cuda_dev, dtype):
    import kvb
    x, lse, tol = rows_of_digits(16, dtype)
    pool = kvb.PagePool.create(20, 1, 64, 64, n_slots=32, max_blocks=16)
    pool.table[:] = torch.arange(16, dtype=torch.int32, device="cuda")
    pool.lens.fill_(1024)
    pool.refs[:16] = 32
    pool.kc[:, :, 1:, 0] = 129
    pool.ks.fill_(1)
    pool.vs.fill_(0.01)
    q = torch.zeros(256, 64, dtype=dtype, device="cuda")
    q[:, 0] = -x
    s = pool.share(torch.arange(32, dtype=torch.int32, device="cuda"))
    assert s.segments[0].tolist() == [0, 32, 0, 1024, 0]
    _, got = pool.attend_shared(q.view(32, 8, 1, 64), s, 1.0, return_lse=True)
    bad = (got.view(256).double() - lse).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.view(256).double() - lse).abs() / tol).max()))
