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
