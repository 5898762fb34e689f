"""What the entry points for shared pages and cross attention refuse and let through, checked on the host before any CUDA call."""

import ctypes as C

import pytest

from test_shared_cpu import A, call, pages


@pytest.mark.parametrize("change,word", [(dict(slots=None), "null"), (dict(plan=None), "null"), (dict(kept=None), "null"), (dict(n=-1), "n <="),
                                         (dict(n=1025), "n <=")])
def test_share_kept(change, word):
    a = dict(slots=A, n=3, plan=A, kept=A, stream=None)
    a.update(change)
    st, msg = call("kvb_page_share_kept", C.byref(pages()), *a.values())
    assert st == 1 and word in msg and "page_share" in msg, (st, msg)


@pytest.mark.parametrize("pool,n,Hq,Tq,fits", [
    (dict(max_blocks=65536, Hkv=8), 512, 64, 4, True), (dict(max_blocks=1 << 20, Hkv=1, page=16), 1024, 128, 1, True),
    (dict(max_blocks=1 << 24, Hkv=1), 100, 1, 1, True), (dict(max_blocks=1 << 24, Hkv=8), 100, 8, 1, False),
    (dict(max_blocks=8), 1000, 2 * 32767, 1000, False), (dict(max_blocks=65536, Hkv=8), 1024, 64, 64, True)])
def test_width_of_a_table(pool, n, Hq, Tq, fits):
    """What is refused goes by the segments' own work, 64 tokens by 256 rows: the next check is that of the workspace."""
    st, msg = call("kvb_page_attend_shared", C.byref(pages(**pool)), A, 1, Hq, Tq, A, n, A, 0.1, A, None, A, 64, None)
    assert (st, "workspace" in msg) == (1, True) if fits else (st, "too many" in msg) == (4, True), (st, msg)


@pytest.mark.parametrize("n,nq,nk,Hq,Hkv,d,fits", [
    (1000, 1000, 4000000, 32, 8, 128, True), (2000, 2000, 3000000, 16, 16, 64, True), (128, 1 << 20, 1 << 22, 32, 8, 128, True),
    (1, 1 << 20, 1 << 22, 32, 8, 128, False), (1, 1 << 16, 1 << 20, 32, 8, 128, True), (128, 1 << 30, 1 << 22, 32, 8, 128, False)])
def test_size_of_a_batch(n, nq, nk, Hq, Hkv, d, fits):
    """What is refused is what one sequence alone could not hold, not the product of all queries and all keys: the next check is
    that of the workspace."""
    st, msg = call("kvb_cross_attention", A, A, A, 2, nq, nk, Hq, Hkv, d, Hq * d, d, Hkv * d, d, Hkv * d, d, A, A, n, 0.1, A, None, A, 64, None)
    assert (st, "workspace" in msg) == (1, True) if fits else (st, "too many" in msg) == (4, True), (st, msg)
