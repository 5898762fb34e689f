"""Refusals of the paged path's C entry points, checked on the host before any CUDA call."""

import ctypes as C

import pytest

A, B = 4096, 1 << 20        # stand-ins for aligned device addresses: never read


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


@pytest.mark.parametrize("field,value,status", [
    ("kc", 0, 1), ("refs", 0, 1), ("n_pages", 0, 1), ("n_pages", 1 << 31, 1), ("Hkv", 0, 1), ("n_slots", 0, 1),
    ("max_blocks", 0, 1), ("max_blocks", 1 << 26, 1), ("kc", 8, 1), ("vc", 4097, 1), ("page", 48, 4), ("page", 256, 4),
    ("d", 96, 4), ("d", 256, 4)])
def test_pool_descriptor(field, value, status):
    p = C.byref(pages(**{field: value}))
    calls = [("kvb_page_extend", (p, A, A, 1, A, None)), ("kvb_page_write", (p, A, A, A, 1, A, A, 2, 5, 256, 128, 256, 128, None)),
             ("kvb_page_read", (p, A, A, A, 1, A, A, 2, 5, None)), ("kvb_page_free", (p, A, 1, None)),
             ("kvb_page_copy", (p, 1, A, A, 1, None)), ("kvb_page_fork", (p, 1, A, A, 1, A, B, None)),
             ("kvb_page_compact", (p, 1, A, A, B, None)), ("kvb_page_attend", (p, A, 1, 4, 1, A, 1, 0.1, A, None, A, B, None))]
    for name, args in calls:
        st, msg = call(name, *args)
        assert st == status and name[4:] in msg, (name, st, msg)
    assert call("kvb_page_fork_workspace", p, 1)[0] == call("kvb_page_compact_workspace", p)[0] == 0
    assert call("kvb_page_attend_workspace", p, 1, 4, 1)[0] == 0


@pytest.mark.parametrize("name,args,status,word", [
    ("kvb_page_extend", (0, A, 1, A, None), 1, "null"), ("kvb_page_extend", (A, A, -1, A, None), 1, "n <="),
    ("kvb_page_extend", (A, A, 1 << 20, A, None), 1, "n <="),
    ("kvb_page_write", (A, A, 0, 1, A, A, 2, 5, 256, 128, 256, 128, None), 1, "null"),
    ("kvb_page_write", (A, A, A, 1, A, A, 3, 5, 256, 128, 256, 128, None), 1, "dtype"),
    ("kvb_page_write", (A, A, A, 1, A, A, 2, 1 << 31, 256, 128, 256, 128, None), 1, "rows"),
    ("kvb_page_read", (A, A, A, -1, A, A, 2, 5, None), 1, "n >= 0"),
    ("kvb_page_free", (0, 1, None), 1, "null"), ("kvb_page_copy", (1, A, 0, 1, None), 1, "null"), ("kvb_page_copy", (0, A, A, 1, None), 1, "null"),
    ("kvb_page_fork", (1, A, A, 1, A, 16, None), 1, "workspace"), ("kvb_page_fork", (1, A, A, 1, A + 16, B, None), 1, "alignment"),
    ("kvb_page_compact", (1, A, A, 16, None), 1, "workspace"), ("kvb_page_compact", (1, 0, A, B, None), 1, "null"),
    ("kvb_page_attend", (A, 1, 3, 1, A, 1, 0.1, A, None, A, B, None), 1, "Hq"),
    ("kvb_page_attend", (A, 1, 4, 0, A, 1, 0.1, A, None, A, B, None), 1, "Tq"),
    ("kvb_page_attend", (A, 0, 4, 1, A, 1, 0.1, A, None, A, B, None), 4, "float16"),
    ("kvb_page_attend", (A, 1, 4, 1, 0, 1, 0.1, A, None, A, B, None), 1, "null"),
    ("kvb_page_attend", (A, 1, 4, 1, A, 1, 0.1, A, None, A, 0, None), 1, "workspace")])
def test_page_calls(name, args, status, word):
    st, msg = call(name, C.byref(pages()), *args)
    assert st == status and word in msg, (st, msg)


def test_layers_share_their_table():
    from kvb import _lib
    two = (_lib.Pages * 2)(pages(), pages(table=2 * A))
    for name, args in (("kvb_page_copy", (A, A, 1, None)), ("kvb_page_fork", (A, A, 1, A, B, None)), ("kvb_page_compact", (A, A, B, None))):
        st, msg = call(name, two, 2, *args)
        assert st == 1 and "share" in msg


@pytest.mark.parametrize("change,status,word", [
    (dict(q=0), 1, "null"), (dict(cu_q=0), 1, "null"), (dict(nq=-1), 1, "n >= 0"), (dict(nk=1 << 31), 1, "row counts"),
    (dict(Hq=5), 1, "Hq"), (dict(Hkv=0), 1, "Hq"), (dict(dtype=0), 4, "float16"), (dict(d=32), 4, "d 64"),
    (dict(q_row=516), 1, "strides"), (dict(v_head=-128), 1, "strides"), (dict(q=A + 8), 1, "alignment"),
    (dict(out=A + 2), 1, "alignment"), (dict(workspace=A, workspace_bytes=64), 1, "workspace"), (dict(workspace=A + 8, workspace_bytes=1 << 30), 1, "workspace")])
def test_prefill_call(change, status, word):
    a = dict(q=A, k=A, v=A, dtype=2, nq=10, nk=10, Hq=4, Hkv=2, d=128, q_row=512, q_head=128, k_row=256, k_head=128, v_row=256,
             v_head=128, cu_q=A, cu_k=A, n=1, scaling=0.1, out=A, lse=None, workspace=None, workspace_bytes=0, stream=None)
    a.update(change)
    st, msg = call("kvb_prefill_attention", *a.values())
    assert st == status and word in msg, (st, msg)
