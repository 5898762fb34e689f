"""Attention over states that many queries share, as a program that serves many sequences calls it.

  share   which leading pages the sequences of a batch have in common (samples of one prompt, requests behind
          one system prompt), found on the GPU from the pool's table
  shared  one decode step's attention of such a batch over the 8-bit pages, the common pages computed once
          for all that hold them
  cross   attention of packed queries to an encoder's states of another length (16-bit keys and values, no
          causal mask): a decoder's prompts, its single tokens, several samples over one encoder's states

`run` computes an operator in its plain form (elementary torch operations in 32 bits), or, where `own` is
true, through this repository's package.  `exact` is the definition in 64 bits.

The pool: codes kc, vc (n_pages, Hkv, page, d) uint8 and scales ks, vs (n_pages, Hkv) float32, a stored
value being (code - 128) * scale; table (n_slots, max_blocks) int32 holds each sequence's pages (-1 past its
last), lens (n_slots) int32 its tokens, refs (n_pages) int32 how many sequences hold a page.

What `share` gives, for the n listed sequences: in up to LEVELS rounds, the sequences of one class (at first
all of them) that hold the same page in the block behind their common ones are a class of the next round; a
class of two or more gets a segment, from the blocks before to the last that all its members hold in full.
order (n): the sequences' places in the list, members of a class together, classes by their first member;
own (n): the first token of a sequence that no segment covers; depth (n): how many segments cover it;
segments (n, 5): first member in `order`, members, first token, end, level, by level and then by first
member (zeros behind the last); count (1): how many there are.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LEVELS = 4


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
        # four questions answered twice each: a small batch, where the call's latency counts
        dict(name="share_pairs", op="share", page=64, system=0, prompts="700,129,64,1023", samples=2, longest=60),
        # a full server: 480 sequences, a system prompt before 60 requests of 8 samples each
        dict(name="share_server", op="share", page=64, system=2048, samples=8, longest=700,
             prompts=_text([100 + (i * 997) % 6000 for i in range(60)])),
        # two samples of one short prompt decoding: latency
        dict(name="shared_pair", op="shared", dtype="bf16", hq=32, hkv=8, d=128, page=64, tq=1, system=0, prompts="700",
             samples=2, longest=60),
        # four prompts sampled eight times each
        dict(name="shared_samples", op="shared", dtype="bf16", hq=32, hkv=8, d=128, page=64, tq=1, system=0,
             prompts="4000,1777,8100,2048", samples=8, longest=500),
        # 64 requests behind one long document that all of them ask about
        dict(name="shared_document", op="shared", dtype="bf16", hq=32, hkv=8, d=128, page=64, tq=1, system=16384,
             prompts=_text([20 + (i * 131) % 400 for i in range(64)]), samples=1, longest=300),
        # a system prompt, requests of several lengths, samples of each: sharing on two levels, 8 query heads per KV head
        dict(name="shared_tree", op="shared", dtype="f16", hq=64, hkv=8, d=128, page=32, tq=1, system=2500,
             prompts="1500,333,4097,2048,801,64", samples=8, longest=400),
        # four drafted tokens per sample checked in one step, small heads, small pages
        dict(name="shared_drafts", op="shared", dtype="f16", hq=16, hkv=4, d=64, page=16, tq=4, system=0,
             prompts="5003,777", samples=5, longest=200),
        # one token of one sequence over an encoder's states: latency
        dict(name="cross_one", op="cross", dtype="f16", hq=16, hkv=16, d=64, q="1", k="1500", lse=False),
        # a decode step of a full batch, every sequence with states of its own length: bandwidth
        dict(name="cross_decode", op="cross", dtype="bf16", hq=32, hkv=8, d=128, q=_text([1] * 48),
             k=_text([257 + (i * i * 53) % 7001 for i in range(48)]), lse=False),
        # several samples of each sequence over the same states, one sequence without states
        dict(name="cross_samples", op="cross", dtype="bf16", hq=32, hkv=8, d=128, q="8,5,8,1,8,7",
             k="4097,1025,0,577,8191,2305", lse=True),
        # packed prompts over image and document states
        dict(name="cross_prompts", op="cross", dtype="f16", hq=32, hkv=8, d=128, q="700,33,1500,1,129,640,2048,250",
             k="1601,4100,577,1025,63,6404,2048,17", lse=True),
        # the longest: a whole context of queries over a long document's states
        dict(name="cross_long", op="cross", dtype="bf16", hq=32, hkv=8, d=128, q="8192", k="16384", lse=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _some_lens(rng, n, hi, total):
    lens = [_log_int(rng, 1, hi) for _ in range(n)]
    while sum(lens) > total:
        lens[lens.index(max(lens))] //= 2
    return [max(1, x) for x in lens]


def draw(rng):
    op = rng.choice(["share", "shared", "shared", "shared", "cross", "cross", "cross"])
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "share":
        requests, samples = _log_int(rng, 4, 60), rng.choice([2, 3, 5, 8])
        return dict(op="share", page=page, system=rng.choice([0, _log_int(rng, 1, 4000)]), samples=samples,
                    prompts=_text(_some_lens(rng, requests, _log_int(rng, 8, 6000), 200000)),
                    longest=_log_int(rng, 1, 700))
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([2, 4, 8])
    rep = rng.choice([1, 2, 3, 4, 4, 8]) if hkv < 8 else rng.choice([1, 2, 4])
    dtype = rng.choice(["bf16", "f16"])
    if op == "shared":
        requests, samples = _log_int(rng, 1, 16), rng.choice([1, 2, 3, 5, 8])
        system = rng.choice([0, _log_int(rng, 1, 12000)])
        prompts = _some_lens(rng, requests, _log_int(rng, 8, 12000), 40000)
        longest = _log_int(rng, 1, 500)
        while requests * samples * (system + max(prompts) + longest) > 1000000:
            system, prompts = system // 2, [max(1, x // 2) for x in prompts]
        return dict(op="shared", dtype=dtype, hq=hkv * rep, hkv=hkv, d=d, page=page, tq=rng.choice([1, 1, 1, 2, 3, 5]),
                    system=system, prompts=_text(prompts), samples=samples, longest=longest)
    n = _log_int(rng, 1, 48)
    if rng.random() < 0.5:
        q = [rng.choice([1, 1, 1, 2, 4, 7]) for _ in range(n)]
    else:
        q = _some_lens(rng, n, _log_int(rng, 2, 4000), 12000)
    k = [0 if rng.random() < 0.05 else x for x in _some_lens(rng, n, _log_int(rng, 8, 16384), 200000)]
    k[0] = max(k[0], 1)
    while n * max(q) * max(k) * hkv * rep > 2 ** 31:
        if max(q) > max(k):
            q[q.index(max(q))] //= 2
        else:
            k[k.index(max(k))] //= 2
    return dict(op="cross", dtype=dtype, hq=hkv * rep, hkv=hkv, d=d, q=_text(q), k=_text(k), lse=rng.random() < 0.5)


def _family(case):
    """Of a pool whose requests stand behind one system prompt and are sampled several times: per sequence its
    request and length, per request the tokens before its samples part."""
    prompts, samples = _ints(case["prompts"]), case["samples"]
    before = [case["system"] + p for p in prompts]
    request = [i // samples for i in range(len(prompts) * samples)]
    lens = [before[j] + max(1 + (i * i * 37) % case["longest"], case.get("tq", 1)) for i, j in enumerate(request)]
    return request, lens, before


def work(case):
    op = case["op"]
    if op == "cross":
        d, hq, hkv = case["d"], case["hq"], case["hkv"]
        q, k = _ints(case["q"]), _ints(case["k"])
        return {"bytes": 2 * d * (2 * sum(q) * hq + 2 * sum(k) * hkv) + (4 * sum(q) * hq if case["lse"] else 0),
                "flops": 4 * d * hq * sum(a * b for a, b in zip(q, k))}
    page = case["page"]
    request, lens, before = _family(case)
    n, all_blocks = len(lens), case["system"] // page
    pages = all_blocks + sum(b // page - all_blocks for b in before) + sum(
        _blocks(x, page) - before[j] // page for x, j in zip(lens, request))
    if op == "share":
        # every table entry of a full block once, slots and lengths; order, own, depth and segments out
        return {"bytes": 4 * sum(x // page for x in lens) + 8 * n + 4 * (8 * n + 1), "flops": 0}
    d, hq, hkv, tq = case["d"], case["hq"], case["hkv"], case["tq"]
    tokens = all_blocks * page + sum((b // page - all_blocks) * page for b in before) + sum(
        x - before[j] // page * page for x, j in zip(lens, request))
    pairs = sum(tq * (x - tq) + tq * (tq + 1) // 2 for x in lens)
    return {"bytes": tokens * hkv * d * 2 + pages * (hkv * 8 + 4) + n * tq * hq * d * 4, "flops": 4 * d * hq * pairs}


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


def _family_pool(case, seed, g, hkv, d):
    """A pool whose sequences were forked: full pages of the system prompt held by all, those of a request by its
    samples, the rest by each alone; pages scattered over the pool, sequences listed in any order."""
    page = case["page"]
    request, lens, before = _family(case)
    n, rng = len(lens), np.random.default_rng(int(seed))
    spare, n_slots = 5, n + 3
    all_blocks = case["system"] // page
    mine = [b // page - all_blocks for b in before]                      # blocks that a request's samples share
    alone = [_blocks(x, page) - before[j] // page for x, j in zip(lens, request)]
    n_pages = all_blocks + sum(mine) + sum(alone) + spare
    ids = rng.permutation(n_pages).astype(np.int32)
    at = all_blocks
    prompt_pages = []
    for m in mine:
        prompt_pages.append(ids[at:at + m])
        at += m
    table = np.full((n_slots, max(_blocks(x, page) for x in lens) + 1), -1, np.int32)
    refs, length = np.zeros(n_pages, np.int32), np.zeros(n_slots, np.int32)
    slots = rng.permutation(n_slots)[:n].astype(np.int32)
    for i in rng.permutation(n):
        row = np.concatenate([ids[:all_blocks], prompt_pages[request[i]], ids[at:at + alone[i]]])
        at += alone[i]
        table[slots[i], :len(row)] = row
        refs[row] += 1
        length[slots[i]] = lens[i]
    slots = slots[rng.permutation(n)]

    def coded(scale):
        x = torch.randn(n_pages, hkv, page, d, generator=g, device=DEV)
        if scale is not None:
            x *= scale[None, :, None, :]
        s = x.abs().amax((2, 3)) / 127
        return (x.mul_((1 / s)[..., None, None]).round_().clamp_(-127, 127) + 128).to(torch.uint8), s

    kc, ks = coded(_key_scale(g, hkv, d))
    vc, vs = coded(None)
    pool = dict(kc=kc, vc=vc, ks=ks, vs=vs, **{k: torch.from_numpy(x).to(DEV) for k, x in (("table", table), ("lens", length), ("refs", refs))})
    return pool, torch.from_numpy(slots).to(DEV), max(lens)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    st = {"case": dict(case), "op": op}
    if op == "share":
        # the table alone matters: the smallest pages that there are
        st["pool"], st["slots"], _ = _family_pool(case, seed, g, 1, 64)
        return st
    dt, hq, hkv, d = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"]
    st["scaling"] = d ** -0.5
    if op == "shared":
        st["pool"], st["slots"], st["max_len"] = _family_pool(case, seed, g, hkv, d)
        st["q"] = torch.randn(st["slots"].shape[0], hq, case["tq"], d, generator=g, device=DEV).to(dt)
        return st
    ql, kl = _ints(case["q"]), _ints(case["k"])
    # keys and values are views of one projection of the encoder's states
    kv = torch.randn(sum(kl), 2 * hkv, d, generator=g, device=DEV)
    kv[:, :hkv] *= _key_scale(g, hkv, d)
    kv = kv.to(dt)
    st.update(q=torch.randn(sum(ql), hq, d, generator=g, device=DEV).to(dt), k=kv[:, :hkv], v=kv[:, hkv:], cu_q=_cu(ql),
              cu_k=_cu(kl), max_q=max(ql), max_k=max(kl))
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
    if op == "cross":
        if st["case"]["lse"]:
            out, lse = kvb.cross_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], st["scaling"], return_lse=True)
            return {"out": out, "lse": lse}
        return {"out": kvb.cross_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], st["scaling"])}
    p = st["pool"]
    pool = st.get("handle")
    if pool is None:        # the handle that a program keeps beside its pool
        pool = st["handle"] = kvb.PagePool(p["kc"], p["vc"], p["ks"], p["vs"], p["table"], p["lens"], p["refs"])
    if op == "share":
        s = pool.share(st["slots"])
        return {"order": s.order, "own": s.own, "depth": s.depth, "segments": s.segments, "count": s.count}
    shared = st.get("shared")
    if shared is None:      # found once a step, for all layers
        shared = st["shared"] = pool.share(st["slots"])
    return {"out": pool.attend_shared(st["q"], shared, st["scaling"])}


def _run_plain(st):
    op = st["op"]
    if op == "cross":
        return _plain_cross(st)
    if op == "share":
        return _plain_share(st["pool"], st["slots"])
    return {"out": _plain_attend(st["pool"], st["q"], st["slots"], st["scaling"], st["max_len"])}


def _plain_share(p, slots):
    page, n = p["kc"].shape[2], slots.shape[0]
    rows = p["table"][slots.long()]
    b, i = torch.arange(rows.shape[1], device=DEV), torch.arange(n, device=DEV)
    good = (b < (p["lens"][slots.long()] // page)[:, None]) & (rows >= 0) & (rows < p["refs"].shape[0])
    held = good.to(torch.int8).cumprod(1).sum(1)                        # leading full blocks
    end, cls, alive = torch.zeros_like(i), torch.zeros_like(i), torch.ones_like(i, dtype=torch.bool)
    depth = torch.zeros_like(i)
    leaders, spans = [], []
    for _ in range(LEVELS):
        key = rows.gather(1, end.clamp(max=rows.shape[1] - 1)[:, None])[:, 0].long()
        more = alive & (end < held)
        same = (cls[:, None] == cls) & (key[:, None] == key) & more[:, None] & more
        same |= i[:, None] == i
        leader, size = same.to(torch.int8).argmax(1), same.sum(1)
        common = ((rows == rows[leader]) & good & good[leader]).to(torch.int8).cumprod(1).sum(1)
        stop = torch.full_like(i, rows.shape[1]).scatter_reduce_(0, leader, common, "amin")[leader]
        alive = size > 1
        spans.append((end, torch.where(alive, stop, end), size, alive & (leader == i)))
        leaders.append(leader)
        end, cls, depth = torch.where(alive, stop, end), leader, depth + alive
    order = i
    for leader in reversed(leaders):
        order = order[torch.argsort(leader[order], stable=True)]
    place = torch.empty_like(i).scatter_(0, order, i)
    table = []
    for level, ((a, e, size, first), leader) in enumerate(zip(spans, leaders)):
        where = torch.full_like(i, n).scatter_reduce_(0, leader, place, "amin")[leader]
        rank = torch.where(first, level * n + where, LEVELS * n)
        table.append((rank, torch.stack([where, size, a * page, e * page, torch.full_like(i, level)], 1), first))
    rank, values, first = (torch.cat(x) for x in zip(*table))
    at = torch.argsort(rank, stable=True)[:n]
    count = first.sum().reshape(1)
    segments = torch.where(torch.arange(n, device=DEV)[:, None] < count, values[at], 0)
    out = {"order": order, "own": end * page, "depth": depth, "segments": segments, "count": count}
    return {k: x.to(torch.int32) for k, x in out.items()}


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


def _plain_cross(st):
    q, k, v, cu_q, cu_k = (st[x] for x in ("q", "k", "v", "cu_q", "cu_k"))
    nq, hq, d = q.shape
    hkv = k.shape[1]

    def padded(x, cu, n):
        i = cu[:-1, None] + torch.arange(n, device=DEV)
        ok = i < cu[1:, None]
        return torch.where(ok[..., None, None], x.float()[i.clamp(max=x.shape[0] - 1)], 0.0)

    qp = (padded(q, cu_q, st["max_q"]) * st["scaling"]).unflatten(2, (hkv, hq // hkv)).permute(0, 2, 3, 1, 4)
    kp, vp = (padded(x, cu_k, st["max_k"]).transpose(1, 2) for x in (k, v))
    j = torch.arange(st["max_k"], device=DEV)
    visible = (j < cu_k.diff()[:, None])[:, None, :].expand(-1, st["max_q"], -1)
    o, lse = _masked_attention(qp, kp, vp, visible)
    token = torch.arange(nq, device=DEV)
    seq = torch.searchsorted(cu_q[1:], token.int(), right=True)
    at = token - cu_q[seq]
    out = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, at].to(q.dtype)
    if not st["case"]["lse"]:
        return {"out": out}
    return {"out": out, "lse": lse.permute(0, 3, 1, 2).flatten(2, 3)[seq, at]}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op == "share":
        return None         # whole numbers
    st = prepare(case, seed)
    if op == "cross":
        return _exact_cross(st)
    p, q = st["pool"], st["q"].double()
    page, hkv = case["page"], case["hkv"]
    table, outs = p["table"].cpu(), []
    for b, slot in enumerate(st["slots"].tolist()):
        n = int(p["lens"][slot])
        pages = table[slot, :_blocks(n, page)].long().to(DEV)

        def side(c, s):
            return ((c[pages].double() - 128) * s[pages].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n]

        k, v = side(p["kc"], p["ks"]), side(p["vc"], p["vs"])                               # (Hkv, n, d)
        rows = q[b].unflatten(0, (hkv, -1))                                                 # (Hkv, rep, Tq, d)
        s = torch.einsum("hrtd,hnd->hrtn", rows, k) * st["scaling"]
        last = n - case["tq"] + torch.arange(case["tq"], device=DEV)
        w = torch.softmax(s.masked_fill(torch.arange(n, device=DEV) > last[:, None], -math.inf), -1)
        outs.append(torch.einsum("hrtn,hnd->thrd", w, v).flatten(1, 2))
    return {"out": torch.stack(outs)}


def _exact_cross(st):
    cu_q, cu_k = st["cu_q"].tolist(), st["cu_k"].tolist()
    hq, hkv = st["q"].shape[1], st["k"].shape[1]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(st["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for a0, a1, b0, b1 in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        if b1 == b0:
            continue
        for h in range(hq):
            k, v = (st[x][b0:b1, h * hkv // hq].double() for x in ("k", "v"))
            for r in range(a0, a1, 4096):
                e = min(a1, r + 4096)
                s = st["q"][r:e, h].double() @ k.t() * st["scaling"]
                lse[r:e, h] = torch.logsumexp(s, -1)
                out[r:e, h] = torch.exp(s - lse[r:e, h, None]) @ v
    return {"out": out, "lse": lse} if st["case"]["lse"] else {"out": out}
