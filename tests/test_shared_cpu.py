"""Refusals of the C entry points for shared pages, checked on the host before any CUDA call."""

import ctypes as C

import pytest

A, B = 4096, 1 << 30        # stand-ins for aligned device addresses: never read


def pages(**kw):
    from kvb import _lib
    f = dict(kc=A, vc=A, ks=A, vs=A, table=A, lens=A, refs=A, n_pages=10, Hkv=2, d=128, page=64, n_slots=4, max_blocks=8)
    f.update(kw)
    return _lib.Pages(*[f[n] for n, _ in _lib.Pages._fields_])


def call(name, *args):
    from kvb import _lib
    lib = _lib.lib()
    st = getattr(lib, name)(*args)
    return st, lib.kvb_last_error().decode()


@pytest.mark.parametrize("change,status,word", [
    (dict(slots=None), 1, "null"), (dict(plan=None), 1, "null"), (dict(n=-1), 1, "n <="), (dict(n=1025), 1, "n <=")])
def test_share(change, status, word):
    a = dict(slots=A, n=3, plan=A, stream=None)
    a.update(change)
    st, msg = call("kvb_page_share", C.byref(pages()), *a.values())
    assert st == status and word in msg and "page_share" in msg, (st, msg)


@pytest.mark.parametrize("pool,change,status,word", [
    ({}, dict(q=None), 1, "null"), ({}, dict(plan=None), 1, "null"), ({}, dict(slots=None), 1, "null"), ({}, dict(workspace=None), 1, "null"),
    ({}, dict(Hq=3), 1, "Hq"), ({}, dict(Tq=0), 1, "Tq"), ({}, dict(dtype=0), 4, "float16"), ({}, dict(n=-1), 1, "n >="),
    ({}, dict(n=1025), 1, "n <="), ({}, dict(q=A + 8), 1, "alignment"), ({}, dict(out=A + 2), 1, "alignment"),
    ({}, dict(scaling=float("inf")), 1, "finite"), ({}, dict(workspace_bytes=64), 1, "workspace"), ({}, dict(workspace=A + 16), 1, "workspace"),
    (dict(max_blocks=1 << 20), dict(n=1000, Hq=64, Tq=8), 4, "too many"), (dict(page=48), {}, 4, "pages"), (dict(d=96), {}, 4, "d 64")])
def test_attend_shared(pool, change, status, word):
    a = dict(q=A, dtype=1, Hq=4, Tq=1, slots=A, n=3, plan=A, scaling=0.1, out=A, lse=None, workspace=A, workspace_bytes=B, stream=None)
    a.update(change)
    st, msg = call("kvb_page_attend_shared", C.byref(pages(**pool)), *a.values())
    assert st == status and word in msg and "page_attend_shared" in msg, (st, msg)


def test_sizes():
    from kvb import _lib
    f = _lib.lib().kvb_page_attend_shared_workspace
    p = C.byref(pages())
    one = _lib.lib().kvb_page_attend_workspace(p, 1, 4, 1)
    assert f(p, 1, 4, 1) >= one and f(p, 3, 4, 2) >= one + 2 * 3 * 8 * 130 * 4 and f(p, 100, 4, 1) >= one + 4 * 400 * 130 * 4
    assert f(p, 1025, 4, 1) == f(p, -1, 4, 1) == f(p, 3, 0, 1) == f(C.byref(pages(d=96)), 3, 4, 1) == 0


def test_oracle_finds_what_forks_share():
    """Hand-made rows: two levels, a sequence that ends inside a page, one that shares nothing."""
    from oracle import paged as O
    pool = O.empty_pool(20, 1, 64, 16, 5, 6)
    pool["table"][0, :5] = [3, 4, 5, 6, 7]
    pool["table"][1, :5] = [3, 4, 5, 9, 10]
    pool["table"][2, :5] = [1, 2, 5, 6, 7]
    pool["table"][3, :5] = [3, 4, 8, 11, 12]
    pool["table"][4, :3] = [3, 4, 5]
    pool["lens"][:] = [80, 75, 80, 80, 47]
    s = O.share(pool, [2, 0, 3, 4, 1])
    assert s["order"] == [0, 1, 4, 2, 3]
    assert s["segments"] == [[1, 4, 0, 32, 0], [1, 2, 32, 48, 1]]
    assert s["own"] == [0, 48, 32, 32, 48] and s["depth"] == [0, 2, 1, 1, 2]
    assert O.share(pool, [2])["own"] == [0]


@pytest.mark.parametrize("change,status,word", [
    (dict(q=None), 1, "null"), (dict(cu_k=None), 1, "null"), (dict(workspace=None), 1, "null"), (dict(nq=-1), 1, "n >= 0"),
    (dict(nk=1 << 31), 1, "row counts"), (dict(Hq=5), 1, "Hq"), (dict(Hkv=0), 1, "Hq"), (dict(dtype=0), 4, "float16"), (dict(d=32), 4, "d 64"),
    (dict(q_row=516), 1, "strides"), (dict(v_head=-128), 1, "strides"), (dict(k_row=0), 4, "rows of their own"), (dict(q=A + 8), 1, "alignment"),
    (dict(out=A + 16), 1, "alignment"), (dict(scaling=float("nan")), 1, "finite"), (dict(workspace=A + 8), 1, "workspace"),
    (dict(workspace_bytes=64), 1, "workspace"), (dict(nq=1 << 30, Hq=64, Hkv=1, k_head=0), 4, "too many"),
    (dict(nq=1 << 24, nk=1 << 30, n=1), 4, "too many")])
def test_cross(change, status, word):
    a = dict(q=A, k=A, v=A, dtype=2, nq=10, nk=10, Hq=4, Hkv=2, d=128, q_row=512, q_head=128, k_row=256, k_head=128, v_row=256,
             v_head=128, cu_q=A, cu_k=A, n=1, scaling=0.1, out=A, lse=None, workspace=A, workspace_bytes=B, stream=None)
    a.update(change)
    st, msg = call("kvb_cross_attention", *a.values())
    assert st == status and word in msg and "cross_attention" in msg, (st, msg)


def test_cross_sizes():
    from kvb import _lib
    f = _lib.lib().kvb_cross_workspace
    assert f(32) == f(0) == 0 and 8192 < f(64) < f(128)
    assert call("kvb_cross_attention", *[None] * 3, 2, 0, 0, 4, 2, 128, *[0] * 6, None, None, 0, 0.1, None, None, None, 0, None)[0] == 0


def test_calls_run_on_the_device_of_their_tensors(monkeypatch):
    """With device 0 current, calls on device 1 begin again with that one current, and the first is back afterwards."""
    import torch
    from kvb import paged
    now = [0]

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *exc):
            now[0] = self.before

    class Tensor:
        def get_device(self):
            return 1

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    names = ("share", "attend_shared")
    Pool = type("Pool", (paged.PagePool,), {x: (lambda x: lambda self, *args: (x, now[0], args))(x) for x in names})
    pool = Pool.__new__(Pool)
    pool._index = 1
    assert paged.PagePool.share(pool, 5) == ("share", 1, (5,)) and now == [0]
    assert paged.PagePool.attend_shared(pool, 5, 6, 0.5, 7, True) == ("attend_shared", 1, (5, 6, 0.5, 7, True)) and now == [0]
    whole = paged.cross_attention
    monkeypatch.setattr(paged, "cross_attention", lambda *args: (args, now[0]))
    q = Tensor()
    assert whole(q, 1, 2, 3, 4, return_lse=True) == ((q, 1, 2, 3, 4, None, None, True), 1) and now == [0]
