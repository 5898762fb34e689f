"""Host threads on one stream: a call of several launches holds its workspace until they are enqueued.  The library is a
stand-in whose calls give way between two of their steps, as the real ones let the interpreter's lock go."""

import threading
import time

import pytest
import torch


class Tensor:
    """What the calls ask of a tensor of CUDA device 0."""
    is_cuda, device = True, torch.device("cuda", 0)

    def __init__(self, *shape, dtype=torch.float16, at=4096):
        self.shape, self.dtype, self.at = torch.Size(shape), dtype, at

    def dim(self):
        return len(self.shape)

    def stride(self):
        return tuple(self.shape[i + 1:].numel() for i in range(len(self.shape)))

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.at

    def numel(self):
        return self.shape.numel()


class Library:
    """Records which thread took which step of a call on which workspace (the argument before the last two), or all on one."""

    def __init__(self):
        self.steps, self.one = [], False

    def __getattr__(self, name):
        if name.endswith("_workspace"):
            return lambda *args: 1 << 16

        def call(*args):
            for step in ("begins", "ends"):
                self.steps.append((0 if self.one else args[-3], step, threading.get_ident()))
                time.sleep(0.002)
            return 0
        return call


@pytest.fixture
def paged(monkeypatch):
    from kvb import paged
    library, made = Library(), iter(range(1 << 20, 1 << 30, 1 << 20))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)
    monkeypatch.setattr(paged, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(paged, "_new", lambda shape, strides, dtype, device: Tensor(*shape, dtype=dtype))
    monkeypatch.setattr(paged, "_fresh_workspace", lambda size, zeroed, device: Tensor(size, at=next(made)))
    monkeypatch.setattr(torch, "empty_like", lambda x: Tensor(*x.shape, dtype=x.dtype))
    monkeypatch.setattr(torch, "empty", lambda shape, dtype, device: Tensor(*shape, dtype=dtype))
    monkeypatch.setattr(torch, "zeros", lambda size, **kw: Tensor(size, at=next(made)))
    monkeypatch.setattr(paged, "_not_capturing", lambda who: None)
    monkeypatch.setattr(paged, "_CROSS_WS", {})
    monkeypatch.setattr(paged.L, "lib", lambda: library)
    return paged, library


def pool_of(paged):
    import ctypes as C
    pool = paged.PagePool.__new__(paged.PagePool)
    pool._index, pool.device, pool.d, pool.table, pool._p = 0, Tensor.device, 64, Tensor(8, 8, dtype=torch.int32), C.c_void_p()
    pool._ws, pool._replaced, pool._lock = {}, [], threading.Lock()
    pool.Hkv, pool._layers, pool._n = 2, None, 1
    return pool


def together(library, *calls):
    """Each call by a thread of its own, several times; the steps of one workspace are whole calls one after the other."""
    gate, failed = threading.Barrier(len(calls)), []

    def work(call):
        try:
            gate.wait()
            for _ in range(5):
                call()
        except Exception as e:                                          # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert len(library.steps) == 10 * len(calls)
    for at in {x[0] for x in library.steps}:
        mine = [x for x in library.steps if x[0] == at]
        for first, last in zip(mine[::2], mine[1::2]):
            assert (first[1], last[1]) == ("begins", "ends") and first[2] == last[2], mine


def test_cross_attention(paged):
    paged, library = paged
    q, k, cu = Tensor(5, 4, 64), Tensor(9, 2, 64), Tensor(2, dtype=torch.int32)
    paged.cross_attention(q, k, k, cu, cu)
    library.steps.clear()
    together(library, *[lambda: paged.cross_attention(q, k, k, cu, cu)] * 4)
    assert len({x[0] for x in library.steps}) == 1                      # they did use one workspace


def test_attend_shared(paged):
    """Of one pool and of another of its layers, which share their workspaces."""
    paged, library = paged
    one, two = pool_of(paged), pool_of(paged)
    two._ws, two._replaced, two._lock = one._ws, one._replaced, one._lock
    shared = paged.SharedPages(Tensor(3, dtype=torch.int32), Tensor(25, dtype=torch.int32), one.table)
    two.table = one.table
    q = Tensor(3, 4, 1, 64)
    together(library, *[lambda p=p: p.attend_shared(q, shared) for p in (one, two, one, two)])
    assert len({x[0] for x in library.steps}) == 1


def test_calls_that_change_table_or_pages(paged):
    """fork and compact plan with the table before they write it: nothing that changes it or the pages comes in between."""
    paged, library = paged
    library.one = True
    pool, ints = pool_of(paged), lambda n: Tensor(n, dtype=torch.int32)
    shared, q, k = paged.SharedPages(ints(3), ints(25), pool.table), Tensor(3, 4, 1, 64), Tensor(9, 2, 64)
    together(library, lambda: pool.fork(ints(3), ints(3)), pool.compact, lambda: pool.extend(ints(3), ints(3)), lambda: pool.free(ints(3)),
             lambda: pool.write(ints(3), ints(3), ints(4), k, k), lambda: pool.copy_pages(ints(3), ints(3)),
             lambda: pool.attend_shared(q, shared))


def test_a_finalizer_may_call_the_pool_inside_a_call(paged):
    """As the collection of garbage would have it: the object whose end frees a sequence goes while a call holds the lock."""
    paged, library = paged
    library.one = True
    pool, ints = pool_of(paged), lambda n: Tensor(n, dtype=torch.int32)
    pool._lock, whole = paged.threading.RLock(), pool._workspace

    class Handle:
        def __del__(self):
            pool.free(ints(3))

    def workspace(*args):
        Handle()
        return whole(*args)

    pool._workspace = workspace
    t = threading.Thread(target=lambda: pool.fork(ints(3), ints(3)), daemon=True)
    t.start()
    t.join(10)
    assert not t.is_alive()
    assert [x[1] for x in library.steps] == ["begins", "ends"] * 2


def test_locks_are_reentrant(paged):
    paged, _ = paged
    cu = Tensor(2, dtype=torch.int32)
    paged.cross_attention(Tensor(5, 4, 64), Tensor(9, 2, 64), Tensor(9, 2, 64), cu, cu)
    (_, lock), = paged._CROSS_WS.values()
    assert type(lock) is type(threading.RLock())


def test_layers_share_the_lock(paged, monkeypatch):
    paged, _ = paged
    monkeypatch.setattr(paged.PagePool, "__init__", lambda self, *ts: vars(self).update(vars(pool_of(paged)), n_pages=1, page=16, _c=paged.L.Pages(), _n=1, _layers=(paged.L.Pages * 1)()))
    first = paged.PagePool()
    for x in ("lens", "refs"):
        setattr(first, x, None)
    other = first.add_layer(1, 2, 3, 4)
    assert other._lock is first._lock and other._ws is first._ws
