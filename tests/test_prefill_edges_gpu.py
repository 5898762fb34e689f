"""Prefill attention where a call could trust what an earlier one left, or an offset that does not ascend."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(cuda_dev):
    import kvb
    kvb.device_status()
    yield
    assert kvb.device_status() == 0, "a test left the device status word set"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("left", [1, 2, 7, 0x7FFFFFFF])
def test_counters_left_by_an_unfinished_call_are_reported_and_do_not_count(cuda_dev, left):
    """Fewer arrivals than an item has pieces are the dangerous ones: they would pass for pieces of this call."""
    import kvb
    from kvb import paged
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(40, 4, 64, generator=g, device="cuda").half()
    k, v = (torch.randn(9000, 1, 64, generator=g, device="cuda").half() for _ in range(2))
    cu_q, cu_k = ints([0, 40]), ints([0, 9000])
    want, lse = kvb.prefill_attention(q, k, v, cu_q, cu_k, return_lse=True)
    assert kvb.device_status() == 0
    ws = paged._PREFILL_WS[(0, torch.cuda.current_stream().cuda_stream, 64)]
    ws[16384:] = 255                                    # partials of no call: NaN
    ws[:16384].view(torch.int32).fill_(left)
    got, gl = kvb.prefill_attention(q, k, v, cu_q, cu_k, return_lse=True)
    assert kvb.device_status() == 8
    assert torch.equal(got, want) and torch.equal(gl, lse)
    assert torch.equal(kvb.prefill_attention(q, k, v, cu_q, cu_k), want)             # its words are in order again
    assert kvb.device_status() == 0
    ws[:16384] = 0


def test_offsets_that_do_not_ascend_are_reported(cuda_dev):
    """More rows named than there are: nothing is read or written past the tensors, and the status word says so."""
    import kvb
    q = torch.randn(300, 2, 64, device="cuda", dtype=torch.float16)
    cu = ints([0, 300] * 40 + [0])
    out = torch.zeros(301, 2, 64, device="cuda", dtype=torch.float16)
    kvb.prefill_attention(q, q, q, cu, out=out[:300])
    assert kvb.device_status() == 2 and (out[300] == 0).all()


def test_many_calls_in_a_row_give_the_same_bits(cuda_dev):
    """Whole items, pieces and empty rows, calls queued behind one another."""
    import kvb
    g = torch.Generator(device="cuda").manual_seed(2)
    cases = []
    for ql, kl, d in (([700, 1, 0, 129], [700, 1, 0, 129], 128), ([30, 5], [6000, 3], 64), ([9], [2500], 128)):
        q = torch.randn(sum(ql), 8, d, generator=g, device="cuda").bfloat16()
        k, v = (torch.randn(sum(kl), 2, d, generator=g, device="cuda").bfloat16() for _ in range(2))
        cu = [ints([0] + torch.tensor(x).cumsum(0).tolist()) for x in (ql, kl)]
        cases.append((q, k, v, *cu))
    want = [kvb.prefill_attention(*c) for c in cases]
    outs = [[kvb.prefill_attention(*c) for c in cases] for _ in range(30)]
    assert all(torch.equal(o, w) for row in outs for o, w in zip(row, want))


@pytest.mark.parametrize("dtype,d,hkv", [(torch.float16, 128, 2), (torch.bfloat16, 64, 1)])
@pytest.mark.parametrize("poison", [float("nan"), -float("inf")])
def test_non_finite_values_in_cut_items(cuda_dev, dtype, d, hkv, poison):
    """Rows before a non-finite value keep their bits, rows from it on are not finite in its channel only, whichever piece
    of the keys it lies in."""
    import kvb
    g = torch.Generator(device="cuda").manual_seed(3)
    ql, kl = [70, 3], [6000, 2500]
    q = torch.randn(sum(ql), 4 * hkv, d, generator=g, device="cuda").to(dtype)
    k, v = (torch.randn(sum(kl), hkv, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    cu_q, cu_k = ints([0, 70, 73]), ints([0, 6000, 8500])
    clean = kvb.prefill_attention(q, k, v, cu_q, cu_k)
    assert torch.isfinite(clean).all()
    for key in (0, 3000, 5930, 5995, 5999):
        p = v.clone()
        p[key, -1, 11] = poison
        got = kvb.prefill_attention(q, k, p, cu_q, cu_k)
        first, heads = max(0, key - 5930), slice(4 * (hkv - 1), None)
        assert not torch.isfinite(got[first:70, heads, 11]).any()
        got[first:70, heads, 11] = clean[first:70, heads, 11]
        assert torch.equal(got, clean)


def test_broadcast_rows_and_heads(cuda_dev):
    """Strides of zero: one key head expanded over all, one query row for every token."""
    import kvb
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(1, 8, 64, generator=g, device="cuda").half().expand(90, 8, 64)
    k, v = (torch.randn(90, 1, 64, generator=g, device="cuda").half().expand(90, 4, 64) for _ in range(2))
    cu = ints([0, 33, 90])
    assert torch.equal(kvb.prefill_attention(q, k, v, cu), kvb.prefill_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu))
