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
