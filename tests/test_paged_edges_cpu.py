"""What the paged path refuses on the host, beside the descriptors and sizes: addresses and devices."""

import ctypes as C

import pytest

A, B = 4096, 1 << 30        # stand-ins for aligned device addresses: never read


def pages(**kw):
    from kvb import _lib
    f = dict(kc=A, vc=A, ks=A, vs=A, table=A, lens=A, refs=A, n_pages=10, Hkv=2, d=128, page=64, n_slots=4, max_blocks=8)
    f.update(kw)
    return _lib.Pages(*[f[n] for n, _ in _lib.Pages._fields_])


@pytest.mark.parametrize("out,lse", [(A + 1, None), (A + 2, None), (A, A + 2), (A, A + 1)])
def test_attend_refuses_outputs_off_their_words(out, lse):
    """Outputs are stored two 16-bit values at a time, the log-sum-exp as float32."""
    from kvb import _lib
    lib = _lib.lib()
    st = lib.kvb_page_attend(C.byref(pages()), A, 1, 4, 1, A, 1, 0.1, out, lse, A, B, None)
    assert st == 1 and "alignment" in lib.kvb_last_error().decode()


@pytest.mark.parametrize("lse", [A + 1, A + 2])
def test_prefill_refuses_a_log_sum_exp_off_its_words(lse):
    from kvb import _lib
    lib = _lib.lib()
    st = lib.kvb_prefill_attention(A, A, A, 2, 10, 10, 4, 2, 128, 512, 128, 256, 128, 256, 128, A, A, 1, 0.1, A, lse, None, 0, None)
    assert st == 1 and "alignment" in lib.kvb_last_error().decode()


class _Ints:
    """Looks like an int32 tensor of n entries on a device."""

    def __init__(self, n, index):
        import torch
        self.dtype, self.shape, self._index = torch.int32, (n,), index

    def get_device(self):
        return self._index

    def is_contiguous(self):
        return True


def test_whole_numbers_of_another_device_are_refused():
    from kvb import paged
    paged._check_ints("call", 3, 1, _Ints(3, 1), _Ints(3, 1))
    paged._check_on("call", 1, _Ints(3, 1))
    for other in (0, 2, -1):
        with pytest.raises(ValueError, match="CUDA device 1"):
            paged._check_ints("call", 3, 1, _Ints(3, 1), _Ints(3, other))
        with pytest.raises(ValueError, match="CUDA device 1"):
            paged._check_on("call", 1, _Ints(3, 1), _Ints(3, other))


def test_calls_run_on_the_device_of_their_tensors(monkeypatch):
    """With device 0 current, a pool of device 1 switches for the call and back; one of device 0 does not switch."""
    import torch
    from kvb import paged
    now, switched = [0], []

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, now[0] = now[0], self.index
            switched.append(self.index)

        def __exit__(self, *exc):
            now[0] = self.before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)

    def again(name):
        return lambda self, *args: (name, now[0], args)

    calls = dict(extend=2, write=5, read=5, attend=5, fork=2, free=1, compact=0, copy_pages=2)
    Pool = type("Pool", (paged.PagePool,), {name: again(name) for name in calls})
    pool = Pool.__new__(Pool)
    pool._index = 1
    for name, n in calls.items():                       # each begins again with device 1 current, then the first is back
        given = tuple(range(n - (name == "read")))
        got = getattr(paged.PagePool, name)(pool, *given)
        assert got[:2] == (name, 1) and got[2][:len(given)] == given and now == [0]
    assert switched == [1] * len(calls)
    pool._index = 0
    with pytest.raises(AttributeError):                 # device 0 is current: no switch, the call itself begins
        paged.PagePool.free(pool, None)
    assert switched == [1] * len(calls)

    class Tensor:
        def get_device(self):
            return 1

    def seen(*args):
        return args, now[0]

    # the call begins again with device 1 current
    whole = paged.prefill_attention
    monkeypatch.setattr(paged, "prefill_attention", seen)
    q = Tensor()
    assert whole(q, 2, 3, 4, scaling=5) == ((q, 2, 3, 4, None, 5, None, False), 1) and now == [0]


def test_attend_refuses_more_rows_a_head_than_32_bits():
    from kvb import _lib
    lib = _lib.lib()
    st = lib.kvb_page_attend(C.byref(pages(Hkv=1)), A, 1, 4096, 1 << 20, A, 1, 0.1, A, None, A, B, None)
    assert st == 1 and "2^31" in lib.kvb_last_error().decode()
