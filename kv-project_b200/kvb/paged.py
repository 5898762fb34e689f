"""The paged path: causal attention of packed prompts, and a pool of 8-bit pages that many sequences share.

  prefill_attention   attention of whole prompts packed without padding, or of chunks after their prefixes
                      (chunked_attention over a prompt, STRATA_KV.py:641-675)
  cross_attention     attention of packed queries to keys of another length (an encoder's states), from single tokens to
                      whole prompts
  PagePool            keys and values of growing sequences in 8-bit pages (one scale per page, KV head and
                      side): extend, write, attend, read, fork, free, compact, copy_pages; share and attend_shared for
                      batches whose sequences hold pages in common.  It stands where the reference's per-sequence
                      buffers do (LayerState, STRATA_KV.py:682-720), for a batch.

Every call enqueues on the current stream of its tensors' device and never synchronises.  Whole numbers (slots, lengths,
page numbers) are int32 tensors on the device, so a captured graph of a pool's calls serves any lengths (one call of each
kind on the stream first: workspaces are not made inside a capture; share, attend_shared and cross_attention need none, a
graph holds workspaces of its own for them); prefill_attention is not captured, it raises NotImplementedError.  Ranges that do not fit are left out and raise the device status word (``kvb.device_status``: bit 1 a
range, bit 4 a pool without enough free pages); rows that are left out of a result are not written.  Several threads may
use one stream: the launches of a call follow one another.
"""

from __future__ import annotations

import ctypes as C
import threading

import torch

from . import _lib as L
from .ops import _DT

_I32 = torch.int32
# a new dense tensor by its strides: 1.6 us where torch.empty takes 2.4
_new = torch.empty_strided
# the current stream's handle without building a Stream object, which costs as much as the launch (4.5 against 0.1 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _elsewhere(index: int) -> bool:
    """Whether a call on tensors of CUDA device `index` needs that device made current first (< 0: it will be refused):
    launches, attributes and the workspaces' sizes are those of the current device, whatever the addresses are.  (Asked in
    each call: a decorator's two more frames cost 0.4 us.)"""
    return index >= 0 and index != torch._C._cuda_getDevice()


def _check_on(who: str, index: int, *ts):
    """Tensors of CUDA device `index`: an address of the host or of another device would be read or written as one of this."""
    for t in ts:
        if t.get_device() != index:
            raise ValueError(f"{who}: every tensor must live on CUDA device {index}")


def _check_ints(who: str, n: int, index: int, *ts):
    """int32, contiguous, one-dimensional tensors of n entries on CUDA device `index`."""
    for t in ts:
        if t.dtype is not _I32 or t.shape != (n,) or t.get_device() != index or not t.is_contiguous():
            raise ValueError(f"{who}: slots, starts, counts and offsets must be contiguous int32 tensors of {n} entries on "
                             f"CUDA device {index}")


def _not_capturing(who: str):
    """A workspace's zeros would only be written when the graph is replayed."""
    if torch.cuda.is_current_stream_capturing():
        raise NotImplementedError(f"{who}: the first call on a stream makes a workspace, which a stream capture cannot")


_COUNTS = 8192                                                  # bytes at such a workspace's start that are counters


def _fresh_workspace(size: int, zeroed: int, device) -> torch.Tensor:
    """A workspace with its counters zeroed.  Inside a stream capture it comes from the graph's own memory: two graphs never
    share one, and each replay zeroes the counters."""
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    ws[:zeroed].zero_()
    return ws


_PREFILL_WS = {}
_UNSPLIT_KEYS = 1024


def _prefill_workspace(lib, device, stream: int, d: int) -> torch.Tensor:
    """The zero-filled workspace of one stream (40 MB at d 128), made at the first call that may need it."""
    ws = _PREFILL_WS.get((device.index, stream, d))
    if ws is None:
        _not_capturing("prefill_attention")
        ws = _PREFILL_WS[(device.index, stream, d)] = torch.zeros(lib.kvb_prefill_workspace(d), dtype=torch.uint8, device=device)
    return ws


def prefill_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor = None,
                      scaling: float = None, out: torch.Tensor = None, return_lse: bool = False):
    """Causal attention of packed sequences: q (Nq, Hq, d), k and v (Nk, Hkv, d) float16 / bfloat16, any row and head
    strides (d contiguous); sequence s has the query rows cu_q[s] .. cu_q[s + 1] - 1 and the key rows of cu_k (default:
    cu_q).  Query i of a sequence sees its keys j <= i + (keys - queries): with as many keys as queries the usual causal
    mask, with more the queries are the last positions.  Query head a reads KV head a // (Hq // Hkv).  scaling defaults
    to d ** -0.5.  Returns out (Nq, Hq, d), with return_lse also the log-sum-exp (Nq, Hq) float32; a row that sees no
    key gives zeros and -inf."""
    if _elsewhere(q.get_device()):
        with torch.cuda.device(q.get_device()):
            return prefill_attention(q, k, v, cu_q, cu_k, scaling, out, return_lse)
    if cu_k is None:
        cu_k = cu_q
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise ValueError("prefill_attention: q (Nq, Hq, d), k and v (Nk, Hkv, d)")
    if not q.is_cuda:
        raise ValueError("kvb: tensors must live on a CUDA device")
    index = q.get_device()
    _check_on("prefill_attention", index, k, v)
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("prefill_attention: q, k and v of one dtype")
    nq, hq, d = q.shape
    nk, hkv, _ = k.shape
    n = cu_q.shape[0] - 1 if cu_q.dim() == 1 else -1
    if n < 0:
        raise ValueError("prefill_attention: cu_q and cu_k hold n + 1 offsets each")
    _check_ints("prefill_attention", n + 1, index, cu_q, cu_k)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if d and not qs[2] == ks[2] == vs[2] == 1:
        raise ValueError("prefill_attention: d must be contiguous")
    if out is None:
        out = _new((nq, hq, d), (hq * d, d, 1), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != index or not out.is_contiguous():
        raise ValueError("prefill_attention: out must be contiguous (Nq, Hq, d) in q's dtype and on its device")
    lse = _new((nq, hq), (hq, 1), dtype=torch.float32, device=q.device) if return_lse else None
    # only query tiles of more than 16 steps of 64 keys are ever cut into pieces
    lib, stream = L.lib(), _raw_stream(index)
    ws = _prefill_workspace(lib, q.device, stream, d) if nk > _UNSPLIT_KEYS else None
    st = lib.kvb_prefill_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _DT.get(q.dtype, -1), nq, nk, hq, hkv, d, qs[0], qs[1], ks[0], ks[1],
        vs[0], vs[1], cu_q.data_ptr(), cu_k.data_ptr(), n, d ** -0.5 if scaling is None else scaling, out.data_ptr(),
        lse.data_ptr() if return_lse else None, None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), stream)
    if st:
        L.check(st, "kvb_prefill_attention")
    return (out, lse) if return_lse else out


_CROSS_WS = {}


def _cross_workspace(lib, device, stream: int, d: int):
    """The workspace of one stream (40 MB at d 128), its counters zeroed, and the lock of the calls that use it: a call's
    launches hand partial sums to one another through it, and the library's calls run without the interpreter's lock."""
    own = None if torch._C._cuda_isCurrentStreamCapturing() else _CROSS_WS.get((device.index, stream, d))
    if own is None:
        own = _fresh_workspace(max(lib.kvb_cross_workspace(d), 256), _COUNTS, device), threading.RLock()
        if not torch._C._cuda_isCurrentStreamCapturing():
            _CROSS_WS[(device.index, stream, d)] = own
    return own


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor,
                    scaling: float = None, out: torch.Tensor = None, return_lse: bool = False):
    """Attention of packed queries to keys of another length (an encoder's states): q (Nq, Hq, d), k and v (Nk, Hkv, d)
    float16 / bfloat16, any row and head strides of 16 bytes (d contiguous; an expanded head is read once); sequence s has the
    query rows cu_q[s] .. cu_q[s + 1] - 1 and sees all of the key rows cu_k[s] .. cu_k[s + 1] - 1.  Query head a reads KV
    head a // (Hq // Hkv).  scaling defaults to d ** -0.5.  Returns out (Nq, Hq, d), with return_lse also the log-sum-exp (Nq,
    Hq) float32; rows of a sequence without keys are zeros and -inf, rows of no sequence are not written."""
    if _elsewhere(q.get_device()):
        with torch.cuda.device(q.get_device()):
            return cross_attention(q, k, v, cu_q, cu_k, scaling, out, return_lse)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise ValueError("cross_attention: q (Nq, Hq, d), k and v (Nk, Hkv, d)")
    if not q.is_cuda:
        raise ValueError("kvb: tensors must live on a CUDA device")
    index = q.get_device()
    _check_on("cross_attention", index, k, v)
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("cross_attention: q, k and v of one dtype")
    nq, hq, d = q.shape
    nk, hkv, _ = k.shape
    n = cu_q.shape[0] - 1 if cu_q.dim() == 1 else -1
    if n < 0:
        raise ValueError("cross_attention: cu_q and cu_k hold n + 1 offsets each")
    _check_ints("cross_attention", n + 1, index, cu_q, cu_k)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if d > 1 and not qs[2] == ks[2] == vs[2] == 1:
        raise ValueError("cross_attention: d must be contiguous")
    if out is None:
        out = _new((nq, hq, d), (hq * d, d, 1), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != index or not out.is_contiguous():
        raise ValueError("cross_attention: out must be contiguous (Nq, Hq, d) in q's dtype and on its device")
    lse = _new((nq, hq), (hq, 1), dtype=torch.float32, device=q.device) if return_lse else None
    lib, stream = L.lib(), _raw_stream(index)
    ws, lock = _cross_workspace(lib, q.device, stream, d)
    with lock:
        st = lib.kvb_cross_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _DT.get(q.dtype, -1), nq, nk, hq, hkv, d, qs[0], qs[1], ks[0], ks[1],
            vs[0], vs[1], cu_q.data_ptr(), cu_k.data_ptr(), n, d ** -0.5 if scaling is None else scaling, out.data_ptr(),
            lse.data_ptr() if return_lse else None, ws.data_ptr(), ws.numel(), stream)
    if st:
        L.check(st, "kvb_cross_attention")
    return (out, lse) if return_lse else out


class SharedPages:
    """What PagePool.share found for n sequences, int32 tensors on the device (views of one): order (n), the sequences'
    places in the list, those of a segment together; own (n), the first token of each that no segment covers; depth (n), how
    many segments cover it; segments (n, 5): first place in order, members, first token, end, level; count (1) of them.
    slots (n) are the sequences as they were listed then: a copy, so that the list may be filled anew.  It stays good while the
    sequences only grow; fork, free, compact and copy_pages make it stale."""

    __slots__ = ("n", "table", "_whole", "_slots", "_plan", "_views")

    def __init__(self, slots, plan, table):
        self._whole, self._slots, self._plan, self.n, self.table, self._views = None, slots, plan, slots.shape[0], table, None

    @classmethod
    def _of(cls, whole, n, table):
        """Of one tensor, the plan and the slots behind it; views of it are made when they are asked for."""
        self = cls.__new__(cls)
        self._whole, self._slots, self._plan, self.n, self.table, self._views = whole, None, None, n, table, None
        return self

    @property
    def plan(self):
        if self._plan is None:
            self._plan = self._whole[:8 * self.n + 1]
        return self._plan

    @property
    def slots(self):
        return (self._views or self._split())[5] if self._slots is None else self._slots

    def _addresses(self, index: int):
        """Of plan and slots, on CUDA device `index`."""
        if self._whole is None:
            _check_on("attend_shared", index, self._plan, self._slots)
            return self._plan.data_ptr(), self._slots.data_ptr()
        _check_on("attend_shared", index, self._whole)
        at = self._whole.data_ptr()
        return at, at + 4 * (8 * self.n + 1)

    def _split(self):
        """The parts, in one call: 3 us where five take 6."""
        n, whole = self.n, self._whole
        self._views = self._plan.split_with_sizes((n, n, n, 5 * n, 1)) if whole is None else whole.split_with_sizes((n, n, n, 5 * n, 1, n))
        return self._views

    @property
    def order(self):
        return (self._views or self._split())[0]

    @property
    def own(self):
        return (self._views or self._split())[1]

    @property
    def depth(self):
        return (self._views or self._split())[2]

    @property
    def segments(self):
        return (self._views or self._split())[3].view(self.n, 5)

    @property
    def count(self):
        return (self._views or self._split())[4]


class PagePool:
    """Pages of ``page`` tokens for Hkv KV heads: codes kc, vc (n_pages, Hkv, page, d) uint8 and scales ks, vs (n_pages,
    Hkv) float32 (a stored value is (code - 128) * scale), table (n_slots, max_blocks) int32 with each sequence's pages,
    lens (n_slots) int32, refs (n_pages) int32.  The pool works on the tensors it is given.  The other layers of a model are
    pools of their own over the same table (add_layer): write, read and attend go to each, the calls that change the table
    (extend, fork, free, compact, copy_pages) once to the first pool, which moves the pages of all."""

    def __init__(self, kc, vc, ks, vs, table, lens, refs):
        ts = (kc, vc, ks, vs, table, lens, refs)
        if kc.dim() != 4 or not all(t.is_cuda and t.is_contiguous() and t.device == kc.device for t in ts):
            raise ValueError("PagePool: contiguous CUDA tensors of one device, kc (n_pages, Hkv, page, d)")
        n_pages, hkv, page, d = kc.shape
        if vc.shape != kc.shape or kc.dtype != torch.uint8 or vc.dtype != torch.uint8:
            raise ValueError("PagePool: kc and vc uint8 (n_pages, Hkv, page, d)")
        if ks.shape != (n_pages, hkv) or vs.shape != ks.shape or ks.dtype != torch.float32 or vs.dtype != torch.float32:
            raise ValueError("PagePool: ks and vs float32 (n_pages, Hkv)")
        if table.dim() != 2 or lens.shape != (table.shape[0],) or refs.shape != (n_pages,) or \
                any(t.dtype != _I32 for t in (table, lens, refs)):
            raise ValueError("PagePool: table (n_slots, max_blocks), lens (n_slots), refs (n_pages) int32")
        self.kc, self.vc, self.ks, self.vs, self.table, self.lens, self.refs = ts
        self.n_pages, self.Hkv, self.page, self.d = n_pages, hkv, page, d
        self.device, self._index = kc.device, kc.device.index
        self._c = L.Pages(*[t.data_ptr() for t in ts], n_pages, hkv, d, page, *table.shape)
        self._p = C.byref(self._c)
        self._layers, self._n = (L.Pages * 1)(self._c), 1
        self._ws, self._replaced = {}, []
        # held while a call's launches are enqueued: they hand data to one another through a workspace, which another thread's
        # launches between them on the same stream would overwrite (the library's calls run without the interpreter's lock); and
        # what plans with the table, then moves pages and writes it (fork, compact) must not be met halfway by what changes
        # table or pages.  Reentrant: a finalizer that frees a sequence may run inside (never between a call's launches, which are
        # one call of the library)
        self._lock = threading.RLock()
        self._attend_ws = {}                                            # stream: address and bytes
        self._attend_bytes = L.lib().kvb_page_attend_workspace(self._p, 1, hkv, 1)      # the same for any call

    @classmethod
    def create(cls, n_pages: int, Hkv: int, d: int, page: int = 64, n_slots: int = 64, max_blocks: int = None, device="cuda"):
        """An empty pool (max_blocks: pages of the longest sequence; all of the pool by default)."""
        z = dict(device=device)
        return cls(torch.full((n_pages, Hkv, page, d), 128, dtype=torch.uint8, **z),
                   torch.full((n_pages, Hkv, page, d), 128, dtype=torch.uint8, **z),
                   torch.zeros((n_pages, Hkv), **z), torch.zeros((n_pages, Hkv), **z),
                   torch.full((n_slots, n_pages if max_blocks is None else max_blocks), -1, dtype=_I32, **z),
                   torch.zeros(n_slots, dtype=_I32, **z), torch.zeros(n_pages, dtype=_I32, **z))

    def add_layer(self, kc=None, vc=None, ks=None, vs=None) -> "PagePool":
        """The pool of another layer over this pool's table (empty codes and scales of the same shape by default)."""
        if kc is None:
            kc, vc = torch.full_like(self.kc, 128), torch.full_like(self.vc, 128)
            ks, vs = torch.zeros_like(self.ks), torch.zeros_like(self.vs)
        other = PagePool(kc, vc, ks, vs, self.table, self.lens, self.refs)
        if (other.n_pages, other.page) != (self.n_pages, self.page):
            raise ValueError("add_layer: as many pages of as many tokens as the first pool has")
        other._lock = self._lock
        other._ws, other._replaced = self._ws, self._replaced           # one workspace a stream for all layers: their calls take turns
        self._layers = (L.Pages * (self._n + 1))(*self._layers, other._c)
        self._n += 1
        return other

    def _workspace(self, kind: str, stream: int, size: int) -> torch.Tensor:
        """A zero-filled buffer for one kind of call on one stream.  One that became too small stays allocated, because a
        captured graph may hold its address; each is twice the one before at least, so that they do not add up."""
        ws = self._ws.get((kind, stream))
        if ws is None or ws.numel() < size:
            _not_capturing(kind)
            if ws is not None:
                self._replaced.append(ws)
                size = max(size, 2 * ws.numel())
            ws = self._ws[(kind, stream)] = torch.zeros(max(size, 256), dtype=torch.uint8, device=self.device)
        return ws

    def _attend_workspace(self, stream: int):
        with self._lock:                                                # the address kept is that of the buffer kept
            ws = self._workspace("attend", stream, self._attend_bytes)
            self._attend_ws[stream] = at = (ws.data_ptr(), ws.numel())
        return at

    def extend(self, slots: torch.Tensor, add: torch.Tensor) -> torch.Tensor:
        """Pages for add[i] more tokens of sequence slots[i]; returns the positions (n,) int32 where they go (-1: the call
        was refused, nothing changed)."""
        if _elsewhere(self._index):
            with torch.cuda.device(self._index):
                return self.extend(slots, add)
        n = slots.shape[0]
        _check_ints("extend", n, self._index, slots, add)
        start = torch.empty_like(slots)
        with self._lock:
            st = L.lib().kvb_page_extend(self._p, slots.data_ptr(), add.data_ptr(), n, start.data_ptr(), _raw_stream(self._index))
        if st:
            L.check(st, "kvb_page_extend")
        return start

    def write(self, slots, start, cu, k, v) -> None:
        """Codes of the packed rows k, v (N, Hkv, d): rows cu[i] .. cu[i + 1] - 1 go to the positions start[i] ... of
        sequence slots[i] (as extend returned them; distinct slots, as two ranges of one page would be written at once)."""
        if _elsewhere(self._index):
            with torch.cuda.device(self._index):
                return self.write(slots, start, cu, k, v)
        n = slots.shape[0]
        _check_ints("write", n, self._index, slots, start)
        _check_ints("write", n + 1, self._index, cu)
        if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (self.Hkv, self.d) or k.dtype != v.dtype:
            raise ValueError("write: k and v (N, Hkv, d) of one dtype")
        _check_on("write", self._index, k, v)
        a, b = k.stride(), v.stride()
        if a[2] != 1 or b[2] != 1:
            raise ValueError("write: d must be contiguous")
        with self._lock:
            st = L.lib().kvb_page_write(self._p, slots.data_ptr(), start.data_ptr(), cu.data_ptr(), n, k.data_ptr(), v.data_ptr(),
                                        _DT.get(k.dtype, -1), k.shape[0], a[0], a[1], b[0], b[1], _raw_stream(self._index))
        if st:
            L.check(st, "kvb_page_write")

    def read(self, slots, start, cu, rows: int, dtype=torch.bfloat16):
        """The stored keys and values (rows, Hkv, d) of the positions start[i] ... of sequence slots[i], packed as in
        write (rows = cu[-1]); rows of a range that is left out (start[i] < 0, or one that does not fit) are not written."""
        if _elsewhere(self._index):
            with torch.cuda.device(self._index):
                return self.read(slots, start, cu, rows, dtype)
        n = slots.shape[0]
        _check_ints("read", n, self._index, slots, start)
        _check_ints("read", n + 1, self._index, cu)
        k, v = (_new((rows, self.Hkv, self.d), (self.Hkv * self.d, self.d, 1), dtype=dtype, device=self.device) for _ in "kv")
        st = L.lib().kvb_page_read(self._p, slots.data_ptr(), start.data_ptr(), cu.data_ptr(), n, k.data_ptr(), v.data_ptr(),
                                   _DT.get(dtype, -1), rows, _raw_stream(self._index))
        if st:
            L.check(st, "kvb_page_read")
        return k, v

    def attend(self, q, slots, scaling: float = None, out=None, return_lse: bool = False):
        """Attention of q (n, Hq, Tq, d), the last Tq positions of each sequence, over its pages -> (n, Tq, Hq, d) in q's
        dtype (float16 / bfloat16); with return_lse also the log-sum-exp (n, Tq, Hq) float32."""
        if _elsewhere(self._index):
            with torch.cuda.device(self._index):
                return self.attend(q, slots, scaling, out, return_lse)
        if q.dim() != 4 or q.shape[3] != self.d:
            raise ValueError("attend: q (n, Hq, Tq, d) on the pool's device")
        _check_on("attend", self._index, q)
        n, hq, tq, d = q.shape
        _check_ints("attend", n, self._index, slots)
        if not q.is_contiguous():
            q = q.contiguous()
        if out is None:
            out = _new((n, tq, hq, d), (tq * hq * d, hq * d, d, 1), dtype=q.dtype, device=q.device)
        elif out.shape != (n, tq, hq, d) or out.dtype != q.dtype or out.get_device() != self._index or not out.is_contiguous():
            raise ValueError("attend: out must be contiguous (n, Tq, Hq, d) in q's dtype on the pool's device")
        lse = _new((n, tq, hq), (tq * hq, hq, 1), dtype=torch.float32, device=q.device) if return_lse else None
        lib, stream = L.lib(), _raw_stream(self._index)
        ws, size = self._attend_ws.get(stream) or self._attend_workspace(stream)
        st = lib.kvb_page_attend(self._p, q.data_ptr(), _DT.get(q.dtype, -1), hq, tq, slots.data_ptr(), n,
                                 d ** -0.5 if scaling is None else scaling, out.data_ptr(), lse.data_ptr() if return_lse else None,
                                 ws, size, stream)
        if st:
            L.check(st, "kvb_page_attend")
        return (out, lse) if return_lse else out

    def share(self, slots) -> SharedPages:
        """Which leading full pages the sequences hold in common (at most 1024; forked ones share their parents'), in up to
        four levels: once a step, for the attend_shared of all layers (which says when that pays)."""
        if _elsewhere(self._index):
            with torch.cuda.device(self._index):
                return self.share(slots)
        n = slots.shape[0]
        _check_ints("share", n, self._index, slots)
        whole = _new((9 * n + 1,), (1,), dtype=_I32, device=self.device)
        at = whole.data_ptr()
        st = L.lib().kvb_page_share_kept(self._p, slots.data_ptr(), n, at, at + 4 * (8 * n + 1), _raw_stream(self._index))
        if st:
            L.check(st, "kvb_page_share_kept")
        return SharedPages._of(whole, n, self.table)

    def attend_shared(self, q, shared: SharedPages, scaling: float = None, out=None, return_lse: bool = False):
        """attend for the sequences of `shared`: the same results up to rounding, the pages that several of them hold read
        and multiplied once for all.  q (n, Hq, Tq, d) -> (n, Tq, Hq, d), with return_lse also (n, Tq, Hq) float32.
        Its three launches take 25 us where attend takes 8 for two short sequences: it is for batches whose sequences hold much in
        common.  With 8 KV heads of 128 channels it is the faster one from about 100 000 tokens on, counted once per sequence, in groups
        of 8 sequences and more (attend_shared and attend: 16 behind one prompt of 4096 tokens 32 us and 31, 64 of them 37 and 94, 64
        behind 16384 55 and 310)."""
        if _elsewhere(self._index):
            with torch.cuda.device(self._index):
                return self.attend_shared(q, shared, scaling, out, return_lse)
        if q.dim() != 4 or q.shape[3] != self.d or q.shape[0] != shared.n:
            raise ValueError("attend_shared: q (n, Hq, Tq, d) on the pool's device, n the sequences of `shared`")
        if shared.table.data_ptr() != self.table.data_ptr() or shared.table.shape != self.table.shape:
            raise ValueError("attend_shared: `shared` is of another table")
        _check_on("attend_shared", self._index, q)
        plan, slots = shared._addresses(self._index)
        n, hq, tq, d = q.shape
        if not q.is_contiguous():
            q = q.contiguous()
        if out is None:
            out = _new((n, tq, hq, d), (tq * hq * d, hq * d, d, 1), dtype=q.dtype, device=q.device)
        elif out.shape != (n, tq, hq, d) or out.dtype != q.dtype or out.get_device() != self._index or not out.is_contiguous():
            raise ValueError("attend_shared: out must be contiguous (n, Tq, Hq, d) in q's dtype on the pool's device")
        lse = _new((n, tq, hq), (tq * hq, hq, 1), dtype=torch.float32, device=q.device) if return_lse else None
        lib, stream = L.lib(), _raw_stream(self._index)
        size = lib.kvb_page_attend_shared_workspace(self._p, n, hq, tq)
        with self._lock:
            if torch._C._cuda_isCurrentStreamCapturing():
                ws = _fresh_workspace(max(size, _COUNTS), _COUNTS, self.device)
            else:
                ws = self._workspace("attend_shared", stream, size)
            st = lib.kvb_page_attend_shared(self._p, q.data_ptr(), _DT.get(q.dtype, -1), hq, tq, slots, n, plan,
                                            d ** -0.5 if scaling is None else scaling, out.data_ptr(),
                                            lse.data_ptr() if return_lse else None, ws.data_ptr(), ws.numel(), stream)
        if st:
            L.check(st, "kvb_page_attend_shared")
        return (out, lse) if return_lse else out

    def fork(self, src, dst) -> None:
        """Sequence dst[i] becomes a copy of src[i] (full pages shared, a partial last page copied); what it held is
        released.  All sources are taken as they were before the call."""
        if _elsewhere(self._index):
            with torch.cuda.device(self._index):
                return self.fork(src, dst)
        n = src.shape[0]
        _check_ints("fork", n, self._index, src, dst)
        lib, stream = L.lib(), _raw_stream(self._index)
        with self._lock:
            ws = self._workspace("fork", stream, lib.kvb_page_fork_workspace(self._p, n))
            st = lib.kvb_page_fork(self._layers, self._n, src.data_ptr(), dst.data_ptr(), n, ws.data_ptr(), ws.numel(), stream)
        if st:
            L.check(st, "kvb_page_fork")

    def free(self, slots) -> None:
        """Drops the sequences and their references to pages."""
        if _elsewhere(self._index):
            with torch.cuda.device(self._index):
                return self.free(slots)
        n = slots.shape[0]
        _check_ints("free", n, self._index, slots)
        with self._lock:
            st = L.lib().kvb_page_free(self._p, slots.data_ptr(), n, _raw_stream(self._index))
        if st:
            L.check(st, "kvb_page_free")

    def compact(self) -> torch.Tensor:
        """Moves the live pages to the pool's start; returns their number (one int32 on the device)."""
        if _elsewhere(self._index):
            with torch.cuda.device(self._index):
                return self.compact()
        lib, stream = L.lib(), _raw_stream(self._index)
        live = torch.empty((), dtype=_I32, device=self.device)
        with self._lock:
            ws = self._workspace("compact", stream, lib.kvb_page_compact_workspace(self._p))
            st = lib.kvb_page_compact(self._layers, self._n, live.data_ptr(), ws.data_ptr(), ws.numel(), stream)
        if st:
            L.check(st, "kvb_page_compact")
        return live

    def copy_pages(self, src, dst) -> None:
        """Page src[i] over page dst[i], codes and scales."""
        if _elsewhere(self._index):
            with torch.cuda.device(self._index):
                return self.copy_pages(src, dst)
        n = src.shape[0]
        _check_ints("copy_pages", n, self._index, src, dst)
        with self._lock:
            st = L.lib().kvb_page_copy(self._layers, self._n, src.data_ptr(), dst.data_ptr(), n, _raw_stream(self._index))
        if st:
            L.check(st, "kvb_page_copy")
