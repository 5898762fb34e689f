"""The serving example end to end: it repeats itself bit for bit, its samples agree where their prompts and first tokens
do, and its decode steps agree with attention over the rows read back."""

import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


def test_serving_example_repeats(cuda_dev):
    import kvb
    import paged_serving as ex
    kvb.device_status()
    a = ex.serve(layers=2, steps=6, lens=(130, 1, 64, 300), samples=3)
    b = ex.serve(layers=2, steps=6, lens=(130, 1, 64, 300), samples=3)
    assert a[0].shape == (12, 6) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_decode_steps_agree_with_a_chunk_after_the_prefix(cuda_dev):
    """The same new tokens once step by step through attend and once as one chunk over the rows read back."""
    import kvb
    pool = kvb.PagePool.create(64, 2, 128, 32, n_slots=2, max_blocks=32)
    g = torch.Generator(device="cuda").manual_seed(3)
    n, new = 500, 9
    q = torch.randn(new, 8, 128, generator=g, device="cuda").half()
    k, v = (torch.randn(n + new, 2, 128, generator=g, device="cuda").half() for _ in range(2))
    i32 = dict(dtype=torch.int32, device="cuda")
    slot, zero, one = torch.tensor([1], **i32), torch.tensor([0], **i32), torch.tensor([1], **i32)
    pool.write(slot, pool.extend(slot, torch.tensor([n], **i32)), torch.tensor([0, n], **i32), k[:n], v[:n])
    outs = []
    for t in range(new):
        start = pool.extend(slot, one)
        pool.write(slot, start, torch.tensor([0, 1], **i32), k[n + t:n + t + 1], v[n + t:n + t + 1])
        kk, vv = pool.read(slot, zero, torch.tensor([0, n + t + 1], **i32), n + t + 1, torch.float16)
        cu = torch.tensor([0, 1], **i32), torch.tensor([0, n + t + 1], **i32)
        a, la = pool.attend(q[t][None, :, None], slot, return_lse=True)
        b, lb = kvb.prefill_attention(q[t:t + 1], kk, vv, *cu, return_lse=True)
        outs.append(a[0, 0])
        # both round weights and outputs to float16, and the rows read back are rounded once more: 4 x 2^-11 of values
        # below 5, and as much of logits below 16 in the log-sum-exp
        assert (a[0, 0].float() - b[0].float()).abs().max() <= 5 * 2.0 ** -9
        assert (la[0, 0] - lb[0]).abs().max() <= 16 * 2.0 ** -9
    assert kvb.device_status() == 0
