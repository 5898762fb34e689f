"""The paged oracle itself: attention against a direct softmax, codes against their definition, and the page
operations against what they have to keep (every sequence's stored rows and the reference counts)."""

import numpy as np
import pytest

from oracle import paged as O


def _counts(pool):
    page = pool["kc"].shape[2]
    n = np.zeros_like(pool["refs"])
    for s in range(len(pool["lens"])):
        for b in range(O.blocks(pool["lens"][s], page)):
            n[pool["table"][s, b]] += 1
    return n


def _filled(rng, lens, page=16, hkv=2, d=64, n_pages=60, n_slots=8):
    pool = O.empty_pool(n_pages, hkv, d, page, n_slots, 12)
    slots = np.arange(len(lens))
    start = O.extend(pool, slots, lens)
    cu = np.concatenate([[0], np.cumsum(lens)])
    O.write(pool, slots, start, cu, *(rng.standard_normal((cu[-1], hkv, d)).astype(np.float32) for _ in range(2)))
    return pool


def test_prefill_equals_masked_softmax():
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((7, h, 8)) for h in (4, 2, 2))
    out, lse, _ = O.prefill(q, k, v, [0, 3, 7], [0, 3, 7], 0.3)
    for a in range(4):
        s = q[3:, a] @ k[3:, a // 2].T * 0.3
        s[np.triu_indices(4, 1)] = -np.inf
        p = np.exp(s - s.max(1, keepdims=True))
        np.testing.assert_allclose(out[3:, a], p / p.sum(1, keepdims=True) @ v[3:, a // 2], rtol=1e-12, atol=1e-14)
        np.testing.assert_allclose(lse[3:, a], np.log(np.exp(s).sum(1)), rtol=1e-12, atol=1e-13)


def test_prefill_rows_without_keys():
    q, k = np.ones((5, 1, 4)), np.ones((2, 1, 4))
    out, lse, _ = O.prefill(q, k, k, [0, 5], [0, 2], 1.0)
    assert (out[:3] == 0).all() and np.isneginf(lse[:3]).all() and (out[3:] == 1).all()


@pytest.mark.parametrize("page", [16, 64])
def test_write_is_within_half_a_step(page):
    rng = np.random.default_rng(2)
    pool = O.empty_pool(8, 1, 64, page, 1, 8)
    O.extend(pool, [0], [100])
    x = rng.standard_normal((100, 1, 64)).astype(np.float32)
    O.write(pool, [0], [0], [0, 100], x, 2 * x)
    k, v = O.rows(pool, 0, 0, 100)
    step = pool["ks"][pool["table"][0, np.arange(100) // page]][:, :, None]
    assert (np.abs(k - x) <= 0.5001 * step).all() and (np.abs(v - 2 * x) <= 1.0002 * step).all()


def test_write_grows_the_scale_once():
    pool = O.empty_pool(1, 1, 64, 16, 1, 1)
    O.extend(pool, [0], [2])
    one = np.ones((1, 1, 64), np.float32)
    O.write(pool, [0], [0], [0, 1], one, one)
    O.write(pool, [0], [1], [0, 1], 4 * one, one / 2)
    k, v = O.rows(pool, 0, 0, 2)
    assert np.allclose(k[0], 1, atol=2 / 127) and np.allclose(k[1], 4) and (pool["kc"][0, 0, 0] == 128 + 32).all()
    assert np.allclose(v[0], 1) and np.allclose(v[1], 0.5, atol=0.5 / 127)


def test_page_operations_keep_the_sequences():
    rng = np.random.default_rng(3)
    pool = _filled(rng, [40, 16, 1, 77, 0])
    want = {s: O.rows(pool, s, 0, pool["lens"][s]) for s in range(5)}
    assert O.fork(pool, [0, 3, 3, 4], [5, 6, 3, 7])
    want.update({5: want[0], 6: want[3], 7: want[4]})
    O.free(pool, [1, 0])
    del want[0], want[1]
    n = O.compact(pool)
    assert (pool["refs"][:n] > 0).all() and (pool["refs"][n:] == 0).all()
    assert (pool["refs"] == _counts(pool)).all()
    for s, (k, v) in want.items():
        gk, gv = O.rows(pool, s, 0, pool["lens"][s])
        assert np.array_equal(gk, k) and np.array_equal(gv, v)


def test_fork_permutes_and_refuses():
    rng = np.random.default_rng(4)
    pool = _filled(rng, [20, 33])
    a, b = O.rows(pool, 0, 0, 20), O.rows(pool, 1, 0, 33)
    assert O.fork(pool, [1, 0], [0, 1])
    assert np.array_equal(O.rows(pool, 0, 0, 33)[0], b[0]) and np.array_equal(O.rows(pool, 1, 0, 20)[1], a[1])
    pool["refs"][pool["refs"] == 0] = 1
    before = {x: pool[x].copy() for x in pool}
    assert not O.fork(pool, [0], [2])
    assert all(np.array_equal(pool[x], before[x]) for x in pool)
