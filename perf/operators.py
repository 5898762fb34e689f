"""The operators of the paged path, as a program that serves many sequences from one pool calls them.

  prefill  causal attention of packed prompts (or of chunks after their prefixes) with grouped heads
  decode   one decode step of a layer: the step's keys and values go into the 8-bit pages, the queries
           attend over them
  write    packed keys and values into the pages, and the sequences read back from them
  fork     sequences become copies of others (shared full pages, the last partial page copied)
  churn    finished sequences are freed, the pool is compacted, new sequences get their pages

`run` computes an operator in its plain form (elementary torch operations in 32 bits), or, where `own` is
true, through this repository's package.  `exact` is the definition in 64 bits.

The pool: codes kc, vc (n_pages, Hkv, page, d) uint8 and scales ks, vs (n_pages, Hkv) float32, a stored
value being (code - 128) * scale; table (n_slots, max_blocks) int32 holds each sequence's pages (-1 past its
last), lens (n_slots) int32 its tokens, refs (n_pages) int32 how many sequences hold a page.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
TINY = 2.0 ** -100          # a page whose largest magnitude is below this is stored as zeros


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _blocks(n, page):
    return -(-n // page)


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # a short question typed into a chat: one prompt of an odd length, where the call's latency counts
        dict(name="prefill_short", op="prefill", dtype="bf16", hq=32, hkv=8, d=128, q="77", prefix="0", lse=False),
        # a batch of prompts of very different lengths packed without padding
        dict(name="prefill_packed", op="prefill", dtype="bf16", hq=32, hkv=8, d=128,
             q="1,3001,129,640,2048,17,1023,350", prefix="0,0,0,0,0,0,0,0", lse=True),
        # the longest prompt: a whole context of 16384 tokens
        dict(name="prefill_long", op="prefill", dtype="bf16", hq=32, hkv=8, d=128, q="16384", prefix="0", lse=False),
        # chunks of two prompts whose earlier tokens are already there, small heads, no lengths that fit a tile
        dict(name="prefill_chunk", op="prefill", dtype="f16", hq=16, hkv=4, d=64, q="500,1100", prefix="7000,333",
             lse=True),
        # one sequence of 4096 tokens decoding alone: latency
        dict(name="decode_one", op="decode", dtype="f16", hq=32, hkv=8, d=128, page=64, tq=1, lens="4096"),
        # a full batch at the long context: bandwidth
        dict(name="decode_batch", op="decode", dtype="bf16", hq=32, hkv=8, d=128, page=64, tq=1,
             lens=_text([32768] * 8)),
        # continuous batching: sequences at every stage, from the first token on, 8 query heads per KV head
        dict(name="decode_ragged", op="decode", dtype="bf16", hq=64, hkv=8, d=128, page=32, tq=1,
             lens=_text([1 + (i * i * 37) % 7919 for i in range(48)])),
        # four drafted tokens per sequence checked in one step, small heads, small pages
        dict(name="decode_drafts", op="decode", dtype="f16", hq=16, hkv=4, d=64, page=16, tq=4,
             lens="4,1000,2049,5003,777,3333"),
        # a whole prompt into empty pages, and read back for the next chunk's attention
        dict(name="write_prompt", op="write", dtype="bf16", hkv=8, d=128, page=64, start="0", new="16384"),
        # short turns of running conversations appended where their last pages end
        dict(name="write_turns", op="write", dtype="f16", hkv=4, d=64, page=16,
             start=_text([(i * 211) % 1500 for i in range(24)]), new=_text([1 + (i * 67) % 300 for i in range(24)])),
        # four prompts sampled eight times each: 32 children share their parents' pages
        dict(name="fork_samples", op="fork", hkv=8, d=128, page=64, lens="4000,1777,8100,2048", children=8),
        # a server's housekeeping: a quarter of the sequences end, the pool closes its holes, others start
        dict(name="churn_pool", op="churn", hkv=8, d=128, page=64,
             lens=_text([64 + (i * 523) % 4001 for i in range(64)])),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _some_lens(rng, n, hi, total):
    lens = [_log_int(rng, 1, hi) for _ in range(n)]
    while sum(lens) > total:
        lens[lens.index(max(lens))] //= 2
    return [max(1, x) for x in lens]


def draw(rng):
    op = rng.choice(["prefill", "prefill", "decode", "decode", "write", "fork", "churn"])
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([2, 4, 8])
    rep = rng.choice([1, 2, 3, 4, 4, 8]) if hkv < 8 else rng.choice([1, 2, 4])
    dtype = rng.choice(["bf16", "f16"])
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "prefill":
        n = rng.choice([1, 1, 2, 5, 12])
        q = _some_lens(rng, n, _log_int(rng, 2, 12000), 12000)
        if n == 1:
            q = [_log_int(rng, 1, 12000)]
        prefix = [_log_int(rng, 1, 4000) if rng.random() < 0.3 else 0 for _ in q]
        return dict(op="prefill", dtype=dtype, hq=hkv * rep, hkv=hkv, d=d, q=_text(q), prefix=_text(prefix),
                    lse=rng.random() < 0.5)
    if op == "decode":
        n = _log_int(rng, 1, 64)
        lens = _some_lens(rng, n, _log_int(rng, 8, 32768), 260000)
        lens[0] = max(lens[0], _log_int(rng, 8, 32768))
        lens = [min(x, 500000 // n) for x in lens]
        tq = rng.choice([1, 1, 1, 2, 3, 5])
        return dict(op="decode", dtype=dtype, hq=hkv * rep, hkv=hkv, d=d, page=page, tq=tq,
                    lens=_text(max(x, tq) for x in lens))
    n = _log_int(rng, 1, 32)
    if op == "write":
        new = _some_lens(rng, n, _log_int(rng, 2, 12000), 12000)
        start = [rng.choice([0, _log_int(rng, 1, 2000)]) if n > 1 else 0 for _ in new]
        while sum(start) + sum(new) > 16384:
            start = [x // 2 for x in start]
        return dict(op="write", dtype=dtype, hkv=hkv, d=d, page=page, start=_text(start), new=_text(new))
    lens = _some_lens(rng, n, _log_int(rng, 8, 8000), 40000)
    if op == "fork":
        return dict(op="fork", hkv=hkv, d=d, page=page, lens=_text(lens[:8]), children=_log_int(rng, 1, 8))
    lens += [_log_int(rng, 1, 500) for _ in range(max(0, 4 - n))]
    return dict(op="churn", hkv=hkv, d=d, page=page, lens=_text(lens))


def _pairs(q, prefix):
    """(query, key) pairs that the causal mask leaves."""
    return sum(n * p + n * (n + 1) // 2 for n, p in zip(q, prefix))


def work(case):
    op, d, hkv = case["op"], case["d"], case["hkv"]
    if op == "prefill":
        q, prefix = _ints(case["q"]), _ints(case["prefix"])
        nq, nk = sum(q), sum(q) + sum(prefix)
        return {"bytes": 2 * d * (2 * nq * case["hq"] + 2 * nk * hkv) + (4 * nq * case["hq"] if case["lse"] else 0),
                "flops": 4 * d * case["hq"] * _pairs(q, prefix)}
    page = case["page"]
    if op == "decode":
        lens, tq = _ints(case["lens"]), case["tq"]
        pages = sum(_blocks(n, page) for n in lens)
        kv = sum(lens) * hkv * d * 2 + pages * (hkv * 8 + 4)
        io = len(lens) * tq * d * 2 * (2 * case["hq"] + 2 * hkv) + len(lens) * tq * hkv * d * 2
        return {"bytes": kv + io, "flops": 4 * d * case["hq"] * _pairs([tq] * len(lens), [n - tq for n in lens])}
    if op == "write":
        start, new = _ints(case["start"]), _ints(case["new"])
        n, m = sum(new), sum(new) + sum(start)
        pages = sum(_blocks(a + b, page) for a, b in zip(start, new))
        return {"bytes": n * hkv * d * 2 * (2 + 1) + m * hkv * d * 2 * (1 + 2) + pages * hkv * 16, "flops": 0}
    lens = _ints(case["lens"])
    page_bytes = 2 * hkv * (page * d + 4)
    if op == "fork":
        part = sum(1 for n in lens if n % page) * case["children"]
        blocks = sum(_blocks(n, page) for n in lens) * case["children"]
        return {"bytes": 2 * part * page_bytes + blocks * 16, "flops": 0}
    # churn: a quarter of the pages are freed and their holes filled from the pool's end, then given out again
    blocks = [_blocks(n, page) for n in lens]
    freed = sum(blocks) // 4
    moved = freed * (sum(blocks) - freed) // sum(blocks)
    return {"bytes": 2 * moved * page_bytes + 8 * sum(blocks) + 16 * freed, "flops": 0}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _i32(values):
    return torch.tensor([int(v) for v in values], dtype=torch.int32, device=DEV)


def _cu(lens):
    return torch.cat([_i32([0]), torch.cumsum(_i32(lens), 0, dtype=torch.int32)])


def _key_scale(g, hkv, d):
    """Keys have a few strong channels: a lognormal scale per KV head and channel."""
    return torch.exp(0.5 * torch.randn(hkv, d, generator=g, device=DEV))


def _pool(g, lens, room, hkv, d, page, n_slots, spare):
    """A pool in use: the pages of `lens` (with room for `room` more tokens each) are scattered over it and
    hold coded keys and values."""
    blocks = [_blocks(n + r, page) for n, r in zip(lens, room)]
    n_pages = sum(blocks) + spare
    perm = torch.randperm(n_pages, generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    mb = max(blocks) + 2
    b = _i32(blocks)[:, None]
    at = (torch.cumsum(b, 0) - b) + torch.arange(mb, device=DEV)
    rows = torch.where(torch.arange(mb, device=DEV) < b, perm[at.clamp(max=n_pages - 1).long()], -1).to(torch.int32)
    table = torch.full((n_slots, mb), -1, dtype=torch.int32, device=DEV)
    slots = torch.randperm(n_slots, generator=g, device=DEV)[:len(lens)].to(torch.int32)
    table[slots.long()] = rows
    length = torch.zeros(n_slots, dtype=torch.int32, device=DEV)
    length[slots.long()] = _i32(lens)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
    refs[perm[:sum(blocks)].long()] = 1

    def coded(scale):
        x = torch.randn(n_pages, hkv, page, d, generator=g, device=DEV)
        if scale is not None:
            x *= scale[None, :, None, :]
        s = x.abs().amax((2, 3)) / 127
        return (x.mul_((1 / s)[..., None, None]).round_().clamp_(-127, 127) + 128).to(torch.uint8), s

    kc, ks = coded(_key_scale(g, hkv, d))
    vc, vs = coded(None)
    return dict(kc=kc, vc=vc, ks=ks, vs=vs, table=table, lens=length, refs=refs), slots


def prepare(case, seed):
    g = _gen(seed)
    op, d, hkv = case["op"], case["d"], case["hkv"]
    st = {"case": dict(case), "op": op}
    if op == "prefill":
        dt, hq = DTYPES[case["dtype"]], case["hq"]
        ql, prefix = _ints(case["q"]), _ints(case["prefix"])
        kl = [a + b for a, b in zip(ql, prefix)]
        nq, nk = sum(ql), sum(kl)
        scale = _key_scale(g, hkv, d)
        if nq == nk:        # q, k and v are views of one projection's output
            x = torch.randn(nq, hq + 2 * hkv, d, generator=g, device=DEV)
            x[:, hq:hq + hkv] *= scale
            x = x.to(dt)
            q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        else:
            q = torch.randn(nq, hq, d, generator=g, device=DEV).to(dt)
            k = (torch.randn(nk, hkv, d, generator=g, device=DEV) * scale).to(dt)
            v = torch.randn(nk, hkv, d, generator=g, device=DEV).to(dt)
        st.update(q=q, k=k, v=v, cu_q=_cu(ql), cu_k=_cu(kl), max_q=max(ql), max_k=max(kl), scaling=d ** -0.5)
        return st
    page = case["page"]
    if op == "decode":
        dt, hq, tq = DTYPES[case["dtype"]], case["hq"], case["tq"]
        lens = _ints(case["lens"])
        n = len(lens)
        pool, slots = _pool(g, lens, [0] * n, hkv, d, page, n + 3, 7)
        st.update(pool=pool, slots=slots, max_len=max(lens), scaling=d ** -0.5,
                  start=_i32([x - tq for x in lens]), cu=_cu([tq] * n),
                  q=torch.randn(n, hq, tq, d, generator=g, device=DEV).to(dt),
                  k=(torch.randn(n * tq, hkv, d, generator=g, device=DEV) * _key_scale(g, hkv, d)).to(dt),
                  v=torch.randn(n * tq, hkv, d, generator=g, device=DEV).to(dt))
        return st
    if op == "write":
        dt = DTYPES[case["dtype"]]
        start, new = _ints(case["start"]), _ints(case["new"])
        lens = [a + b for a, b in zip(start, new)]
        n = sum(new)
        pool, slots = _pool(g, lens, [0] * len(lens), hkv, d, page, len(lens) + 1, 5)
        # new rows of every magnitude: some pages have to take a larger scale for them
        grow = torch.exp(0.7 * torch.randn(n, 1, 1, generator=g, device=DEV))
        st.update(pool=pool, slots=slots, start=_i32(start), cu=_cu(new), zero=_i32([0] * len(lens)),
                  cu_all=_cu(lens), rows=sum(lens),
                  k=(torch.randn(n, hkv, d, generator=g, device=DEV) * _key_scale(g, hkv, d) * grow).to(dt),
                  v=(torch.randn(n, hkv, d, generator=g, device=DEV) * grow).to(dt))
        return st
    lens = _ints(case["lens"])
    n = len(lens)
    if op == "fork":
        c = case["children"]
        pool, parents = _pool(g, lens, [0] * n, hkv, d, page, n * (1 + c) + 2, 2 * n * c + 9)
        free = torch.ones(n * (1 + c) + 2, dtype=torch.bool, device=DEV)
        free[parents.long()] = False
        st.update(pool=pool, src=parents.repeat_interleave(c),
                  dst=torch.nonzero(free).flatten()[:n * c].to(torch.int32))
        return st
    pool, slots = _pool(g, lens, [0] * n, hkv, d, page, n + 2, 16 + sum(lens) // page // 8)
    st.update(pool=pool, turn=0, subsets=[slots[i::4].contiguous() for i in range(4)],
              again=[_i32(lens[i::4]) for i in range(4)])
    return st


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(st):
    return (_run_own if own else _run_plain)(st)


def _kvb():
    root = str(Path(__file__).resolve().parents[1] / "kv-project_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import kvb
    return kvb


def _run_own(st):
    kvb = sys.modules.get("kvb") or _kvb()
    op = st["op"]
    if op == "prefill":
        if st["case"]["lse"]:
            out, lse = kvb.prefill_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], st["scaling"],
                                             return_lse=True)
            return {"out": out, "lse": lse}
        return {"out": kvb.prefill_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], st["scaling"])}
    p = st["pool"]
    pool = st.get("handle")
    if pool is None:        # the handle that a program keeps beside its pool
        pool = st["handle"] = kvb.PagePool(p["kc"], p["vc"], p["ks"], p["vs"], p["table"], p["lens"], p["refs"])
    if op == "decode":
        pool.write(st["slots"], st["start"], st["cu"], st["k"], st["v"])
        return {"out": pool.attend(st["q"], st["slots"], st["scaling"]), "ks": p["ks"], "vs": p["vs"]}
    if op == "write":
        pool.write(st["slots"], st["start"], st["cu"], st["k"], st["v"])
        k, v = pool.read(st["slots"], st["zero"], st["cu_all"], st["rows"], st["k"].dtype)
        return {"k": k, "v": v, "ks": p["ks"], "vs": p["vs"]}
    if op == "fork":
        pool.fork(st["src"], st["dst"])
        return dict(p)
    i = st["turn"]
    st["turn"] = (i + 1) % 4
    pool.free(st["subsets"][i])
    pool.compact()
    start = pool.extend(st["subsets"][i], st["again"][i])
    return dict(p, start=start)


def _run_plain(st):
    op = st["op"]
    if op == "prefill":
        return _plain_prefill(st)
    p = st["pool"]
    if op == "decode":
        _plain_write(p, st["slots"], st["start"], st["cu"], st["k"], st["v"])
        out = _plain_attend(p, st["q"], st["slots"], st["scaling"], st["max_len"])
        return {"out": out, "ks": p["ks"], "vs": p["vs"]}
    if op == "write":
        _plain_write(p, st["slots"], st["start"], st["cu"], st["k"], st["v"])
        k, v = _plain_read(p, st["slots"], st["zero"], st["cu_all"], st["rows"], st["k"].dtype)
        return {"k": k, "v": v, "ks": p["ks"], "vs": p["vs"]}
    if op == "fork":
        _plain_fork(p, st["src"], st["dst"])
        return dict(p)
    i = st["turn"]
    st["turn"] = (i + 1) % 4
    _plain_free(p, st["subsets"][i])
    _plain_compact(p)
    return dict(p, start=_plain_extend(p, st["subsets"][i], st["again"][i]))


def _masked_attention(q, k, v, visible):
    """q (S, H, R, T, d), k and v (S, H, L, d) float32, visible (S, T, L): outputs and log-sum-exp; a row
    that sees nothing gives zeros and -inf."""
    S, H, R, T, d = q.shape
    s = torch.matmul(q.reshape(S, H, R * T, d), k.transpose(-1, -2)).view(S, H, R, T, -1)
    s.masked_fill_(~visible[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    s.sub_(m).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(S, H, R * T, -1), v).view(S, H, R, T, d)
    return torch.where(total > 0, o / total, 0.0), (m + total.log())[..., 0]


def _plain_prefill(st):
    q, k, v, cu_q, cu_k = (st[x] for x in ("q", "k", "v", "cu_q", "cu_k"))
    nq, hq, d = q.shape
    hkv = k.shape[1]
    rep = hq // hkv

    def padded(x, cu, n):
        i = cu[:-1, None] + torch.arange(n, device=DEV)
        ok = i < cu[1:, None]
        return torch.where(ok[..., None, None], x.float()[i.clamp(max=x.shape[0] - 1)], 0.0)

    qp = (padded(q, cu_q, st["max_q"]) * st["scaling"]).unflatten(2, (hkv, rep)).permute(0, 2, 3, 1, 4)
    kp, vp = (padded(x, cu_k, st["max_k"]).transpose(1, 2) for x in (k, v))
    ql, kl = cu_q.diff(), cu_k.diff()
    i, j = torch.arange(st["max_q"], device=DEV), torch.arange(st["max_k"], device=DEV)
    visible = (j[None, None, :] <= i[None, :, None] + (kl - ql)[:, None, None]) & (j < kl[:, None])[:, None, :]
    o, lse = _masked_attention(qp, kp, vp, visible)
    token = torch.arange(nq, device=DEV)
    seq = torch.searchsorted(cu_q[1:], token.int(), right=True)
    at = token - cu_q[seq]
    out = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, at].to(q.dtype)
    if not st["case"]["lse"]:
        return {"out": out}
    return {"out": out, "lse": lse.permute(0, 3, 1, 2).flatten(2, 3)[seq, at]}


def _token_places(p, slots, start, cu, rows):
    """(page, row in the page) of every packed token."""
    page = p["kc"].shape[2]
    token = torch.arange(rows, device=DEV, dtype=torch.int32)
    seq = torch.searchsorted(cu[1:], token, right=True)
    pos = start[seq] + token - cu[seq]
    return p["table"][slots[seq].long(), (pos // page).long()].long(), (pos % page).long()


def _plain_write(p, slots, start, cu, k, v):
    page = p["kc"].shape[2]
    pg, row = _token_places(p, slots, start, cu, k.shape[0])
    first = p["table"][slots.long(), (start // page).long()].long()
    held = start % page
    for codes, scales, x in ((p["kc"], p["ks"], k.float()), (p["vc"], p["vs"], v.float())):
        a = torch.where(torch.isfinite(x), x, 0.0).abs().amax(-1)
        a = torch.zeros_like(scales).scatter_reduce_(0, pg[:, None].expand_as(a), a, "amax")
        touched = torch.zeros(scales.shape[0], dtype=torch.bool, device=DEV)
        touched[pg] = True
        base = torch.zeros_like(scales)
        base[first] = torch.where((held > 0)[:, None], scales[first], 0.0)
        new = torch.maximum(base, torch.where(a < TINY, 0.0, a / 127))
        ratio = torch.where(new > 0, base / new, 0.0)
        old = codes[first]
        again = ((old.float() - 128) * ratio[first][..., None, None]).round() + 128
        keep = torch.arange(page, device=DEV) < held[:, None]
        codes[first] = torch.where(keep[:, None, :, None], again.to(torch.uint8), old)
        c = x * torch.where(new > 0, 1 / new, 0.0)[pg][..., None]
        c = torch.where(torch.isnan(c), 0.0, c.round().clamp(-127, 127))
        codes[pg, :, row] = (c + 128).to(torch.uint8)
        scales.copy_(torch.where(touched[:, None], new, scales))


def _plain_read(p, slots, start, cu, rows, dtype):
    pg, row = _token_places(p, slots, start, cu, rows)
    return tuple(((c[pg, :, row].float() - 128) * s[pg][..., None]).to(dtype)
                 for c, s in ((p["kc"], p["ks"]), (p["vc"], p["vs"])))


def _plain_attend(p, q, slots, scaling, max_len):
    n, hq, tq, d = q.shape
    hkv, page = p["kc"].shape[1:3]
    nb = _blocks(max_len, page)
    pages = p["table"][slots.long(), :nb].clamp(min=0).long()
    k, v = (((c[pages].float() - 128) * s[pages][..., None, None]).transpose(1, 2).flatten(2, 3)
            for c, s in ((p["kc"], p["ks"]), (p["vc"], p["vs"])))
    length = p["lens"][slots.long()]
    j, t = torch.arange(nb * page, device=DEV), torch.arange(tq, device=DEV)
    visible = j[None, None, :] <= (length[:, None] - tq + t[None, :])[:, :, None]
    o, _ = _masked_attention((q.float() * scaling).unflatten(1, (hkv, hq // hkv)), k, v, visible)
    return o.flatten(1, 2).transpose(1, 2).to(q.dtype)


def _free_pages(p):
    """All pages, the free ones first, each part in ascending order."""
    return torch.argsort((p["refs"] != 0).to(torch.int8), stable=True)


def _plain_extend(p, slots, new):
    page, mb = p["kc"].shape[2], p["table"].shape[1]
    at = slots.long()
    start = p["lens"][at]
    have, want = (start + page - 1) // page, (start + new + page - 1) // page
    need = want - have
    order = _free_pages(p)
    b = torch.arange(mb, device=DEV)
    i = (torch.cumsum(need, 0) - need - have)[:, None] + b
    fresh = order[i.clamp(0, order.numel() - 1)].to(torch.int32)
    p["table"][at] = torch.where((b >= have[:, None]) & (b < want[:, None]), fresh, p["table"][at])
    p["refs"][order] = torch.where(torch.arange(order.numel(), device=DEV) < need.sum(), 1, p["refs"][order])
    p["lens"][at] = start + new
    return start


def _held(p, rows, count):
    """How often each page occurs in the first `count` entries of table rows."""
    used = torch.arange(rows.shape[1], device=DEV) < count[:, None]
    out = torch.zeros_like(p["refs"])
    return out.index_add_(0, rows.clamp(min=0).flatten().long(), used.flatten().to(torch.int32))


def _plain_free(p, slots):
    page, at = p["kc"].shape[2], slots.long()
    p["refs"].sub_(_held(p, p["table"][at], (p["lens"][at] + page - 1) // page))
    p["table"][at] = -1
    p["lens"][at] = 0


def _plain_fork(p, src, dst):
    page = p["kc"].shape[2]
    s, t = src.long(), dst.long()
    length, rows, old = p["lens"][s], p["table"][s], p["table"][t]
    old_blocks = (p["lens"][t] + page - 1) // page
    blocks = (length + page - 1) // page
    same = src == dst
    part = (length % page != 0) & ~same
    last = (blocks - 1).clamp(min=0)[:, None].long()
    before = rows.gather(1, last)[:, 0]
    fresh = _free_pages(p)[(torch.cumsum(part, 0) - 1).clamp(min=0)].to(torch.int32)
    rows = rows.scatter(1, last, torch.where(part, fresh, before)[:, None])
    p["refs"].add_(_held(p, rows, blocks)).sub_(_held(p, old, old_blocks))
    to, come = torch.where(part, fresh, before).clamp(min=0).long(), before.clamp(min=0).long()
    for x in ("kc", "vc", "ks", "vs"):
        p[x][to] = p[x][come]
    p["table"][t] = rows
    p["lens"][t] = length


def _plain_compact(p):
    refs = p["refs"]
    n = refs.numel()
    ids = torch.arange(n, device=DEV)
    live = refs > 0
    count = live.sum()
    mover, hole = live & (ids >= count), ~live & (ids < count)          # as many of the one as of the other
    come, to = (torch.argsort((~x).to(torch.int8), stable=True) for x in (mover, hole))
    taken = torch.where(hole, come[(torch.cumsum(hole, 0) - 1).clamp(min=0)], ids)
    new_id = torch.where(mover, to[(torch.cumsum(mover, 0) - 1).clamp(min=0)], ids)
    for x in ("kc", "vc", "ks", "vs"):
        p[x].copy_(p[x][taken])
    p["table"].copy_(torch.where(p["table"] >= 0, new_id[p["table"].clamp(min=0).long()].to(torch.int32), -1))
    refs.copy_(torch.where(ids < count, refs[taken], 0))


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op in ("fork", "churn"):
        return None         # bytes and whole numbers are moved, nothing is computed
    st = prepare(case, seed)
    if op == "prefill":
        return _exact_prefill(st)
    p = st["pool"]
    kc, ks = _exact_write(st, p["kc"], p["ks"], st["k"])
    vc, vs = _exact_write(st, p["vc"], p["vs"], st["v"])
    page = kc.shape[2]
    table, slots = p["table"].tolist(), st["slots"].tolist()

    def sequence(c, s, slot, n):
        pages = torch.tensor(table[slot][:_blocks(n, page)], device=DEV)
        return (c[pages] * s[pages][..., None, None]).transpose(1, 2).flatten(0, 1)[:n]      # (n, Hkv, d)

    if op == "write":
        lens = st["cu_all"].diff().tolist()
        return {"k": torch.cat([sequence(kc, ks, a, n) for a, n in zip(slots, lens)]),
                "v": torch.cat([sequence(vc, vs, a, n) for a, n in zip(slots, lens)]), "ks": ks, "vs": vs}
    q = st["q"].double()
    hkv, tq = kc.shape[1], q.shape[2]
    outs = []
    for b, slot in enumerate(slots):
        n = int(p["lens"][slot])
        k, v = sequence(kc, ks, slot, n), sequence(vc, vs, slot, n)
        heads = [_exact_rows(q[b, a], k[:, a * hkv // q.shape[1]], v[:, a * hkv // q.shape[1]], n - tq, st["scaling"])[0]
                 for a in range(q.shape[1])]
        outs.append(torch.stack(heads, 1))
    return {"out": torch.stack(outs), "ks": ks, "vs": vs}


def _exact_rows(q, k, v, before, scaling):
    """Rows q (T, d) at positions before, before + 1, ... over keys (L, d): outputs and log-sum-exp."""
    s = q @ k.t() * scaling
    seen = torch.arange(k.shape[0], device=DEV) <= torch.arange(q.shape[0], device=DEV)[:, None] + before
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    return torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[:, None]) @ v, lse


def _exact_prefill(st):
    cu_q, cu_k = st["cu_q"].tolist(), st["cu_k"].tolist()
    hq, hkv = st["q"].shape[1], st["k"].shape[1]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(st["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for a0, a1, b0, b1 in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        for h in range(hq):
            k, v = (st[x][b0:b1, h * hkv // hq].double() for x in ("k", "v"))
            for r in range(a0, a1, 4096):
                e = min(a1, r + 4096)
                out[r:e, h], lse[r:e, h] = _exact_rows(st["q"][r:e, h].double(), k, v, (b1 - b0) - (a1 - a0) + r - a0,
                                                       st["scaling"])
    return {"out": out, "lse": lse} if st["case"]["lse"] else {"out": out}


def _exact_write(st, codes, scales, x):
    """Codes less 128 and scales of the pool after the write, in 64 bits."""
    c, s = codes.double() - 128, scales.double()
    page, table = codes.shape[2], st["pool"]["table"].tolist()
    start, cu, slots = st["start"].tolist(), st["cu"].tolist(), st["slots"].tolist()
    x = x.double()
    for i, slot in enumerate(slots):
        pos, row = start[i], cu[i]
        while row < cu[i + 1]:
            pg, off = table[slot][pos // page], pos % page
            n = min(page - off, cu[i + 1] - row)
            rows = x[row:row + n].transpose(0, 1)                                            # (Hkv, n, d)
            old = s[pg] if off else torch.zeros_like(s[pg])
            new = torch.maximum(old, rows.abs().amax((1, 2)) / 127)
            c[pg, :, :off] = torch.round(c[pg, :, :off] * (old / new)[:, None, None])
            c[pg, :, off:off + n] = torch.round(rows / new[:, None, None])
            s[pg] = new
            pos, row = pos + n, row + n
    return c, s
