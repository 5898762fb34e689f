"""Oracle of the paged path: causal attention of packed sequences in float64, and the 8-bit page pool as plain
numpy state (a dict of kc, vc, ks, vs, table, lens, refs).  Writes follow the code's definition one float32
operation at a time, so codes and scales are exact; page operations move whole numbers and bytes."""

from __future__ import annotations

import numpy as np

TINY = np.float32(2.0 ** -100)


def causal_rows(q, k, v, scaling, before):
    """q (T, d) over k, v (L, d) in float64, query i sees keys j <= i + before.  Returns out (T, d), lse (T,) and
    the attended mean of |v| (T, d), which error bounds are stated in.  Rows that see nothing: 0, -inf, 0."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    T, L = q.shape[0], k.shape[0]
    out, mean_abs, lse = np.zeros((T, v.shape[1])), np.zeros((T, v.shape[1])), np.full(T, -np.inf)
    for i in range(T):
        n = min(max(i + before + 1, 0), L)
        if n == 0:
            continue
        s = k[:n] @ q[i] * scaling
        m = s.max()
        p = np.exp(s - m)
        lse[i] = m + np.log(p.sum())
        out[i], mean_abs[i] = p @ v[:n] / p.sum(), p @ np.abs(v[:n]) / p.sum()
    return out, lse, mean_abs


def prefill(q, k, v, cu_q, cu_k, scaling):
    """q (Nq, Hq, d), k, v (Nk, Hkv, d): out, lse, mean_abs in float64 (see causal_rows)."""
    hq, hkv = q.shape[1], k.shape[1]
    out, mean_abs = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full(q.shape[:2], -np.inf)
    for a0, a1, b0, b1 in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        for a in range(hq):
            h = a * hkv // hq
            out[a0:a1, a], lse[a0:a1, a], mean_abs[a0:a1, a] = causal_rows(
                q[a0:a1, a], k[b0:b1, h], v[b0:b1, h], scaling, (b1 - b0) - (a1 - a0))
    return out, lse, mean_abs


def empty_pool(n_pages, hkv, d, page, n_slots, max_blocks):
    return dict(kc=np.full((n_pages, hkv, page, d), 128, np.uint8), vc=np.full((n_pages, hkv, page, d), 128, np.uint8),
                ks=np.zeros((n_pages, hkv), np.float32), vs=np.zeros((n_pages, hkv), np.float32),
                table=np.full((n_slots, max_blocks), -1, np.int32), lens=np.zeros(n_slots, np.int32),
                refs=np.zeros(n_pages, np.int32))


def blocks(n, page):
    return -(-int(n) // page)


def code8(x, inv):
    with np.errstate(invalid="ignore", over="ignore"):
        c = np.asarray(x, np.float32) * np.float32(inv)
        c = np.where(np.isnan(c), np.float32(0), np.clip(np.rint(c), -127, 127))
    return (c + 128).astype(np.uint8)


def write(pool, slots, start, cu, k, v):
    """k, v (N, Hkv, d) float32 values."""
    page = pool["kc"].shape[2]
    for slot, st, a, b in zip(slots, start, cu, cu[1:]):
        pos, row = int(st), int(a)
        while st >= 0 and row < b:
            pg, off = pool["table"][slot, pos // page], pos % page
            n = min(page - off, int(b) - row)
            for codes, scales, x in ((pool["kc"], pool["ks"], k), (pool["vc"], pool["vs"], v)):
                for h in range(codes.shape[1]):
                    r = np.asarray(x[row:row + n, h], np.float32)
                    amax = np.abs(np.where(np.isfinite(r), r, np.float32(0))).max()
                    old = scales[pg, h] if off else np.float32(0)
                    s = max(old, np.float32(0) if amax < TINY else np.float32(amax / np.float32(127)))
                    if s > old > 0:
                        c = codes[pg, h, :off].astype(np.float32) - np.float32(128)
                        codes[pg, h, :off] = (np.rint(c * np.float32(old / s)) + 128).astype(np.uint8)
                    codes[pg, h, off:off + n] = code8(r, np.float32(1) / s if s > 0 else 0)
                    scales[pg, h] = s
            pos, row = pos + n, row + n


def rows(pool, slot, start, n):
    """Stored keys and values (n, Hkv, d) float32 of the positions start .. of a sequence."""
    page = pool["kc"].shape[2]
    at = np.arange(start, start + n)
    pg = pool["table"][slot, at // page]
    return tuple((c[pg, :, at % page].astype(np.float32) - np.float32(128)) * s[pg][..., None]
                 for c, s in ((pool["kc"], pool["ks"]), (pool["vc"], pool["vs"])))


def attend(pool, q, slots, scaling):
    """q (n, Hq, Tq, d): out (n, Tq, Hq, d), lse (n, Tq, Hq), mean_abs in float64."""
    n, hq, tq, d = q.shape
    hkv = pool["kc"].shape[1]
    out, mean_abs, lse = np.zeros((n, tq, hq, d)), np.zeros((n, tq, hq, d)), np.full((n, tq, hq), -np.inf)
    for i, slot in enumerate(slots):
        length = int(pool["lens"][slot])
        k, v = rows(pool, slot, 0, length)
        for a in range(hq):
            h = a * hkv // hq
            out[i, :, a], lse[i, :, a], mean_abs[i, :, a] = causal_rows(q[i, a], k[:, h], v[:, h], scaling, length - tq)
    return out, lse, mean_abs


def _free(pool):
    return np.flatnonzero(pool["refs"] == 0)


def extend(pool, slots, add):
    page, mb = pool["kc"].shape[2], pool["table"].shape[1]
    lens = [int(pool["lens"][s]) for s in slots]
    need = [blocks(n + a, page) - blocks(n, page) for n, a in zip(lens, add)]
    free = _free(pool)
    if sum(need) > len(free) or any(blocks(n + a, page) > mb for n, a in zip(lens, add)):
        return np.full(len(lens), -1, np.int32)
    at = 0
    for s, n, a, m in zip(slots, lens, add, need):
        have = blocks(n, page)
        pool["table"][s, have:have + m] = free[at:at + m]
        pool["refs"][free[at:at + m]] = 1
        pool["lens"][s] = n + a
        at += m
    return np.array(lens, np.int32)


def free(pool, slots):
    page = pool["kc"].shape[2]
    for s in slots:
        for b in range(blocks(pool["lens"][s], page)):
            pool["refs"][pool["table"][s, b]] -= 1
            pool["table"][s, b] = -1
        pool["lens"][s] = 0


def copy_page(pool, a, b):
    for x in ("kc", "vc", "ks", "vs"):
        pool[x][b] = pool[x][a]


def fork(pool, src, dst):
    """False (and nothing changed) when the pool has too few free pages."""
    page = pool["kc"].shape[2]
    lens = [int(pool["lens"][s]) for s in src]
    table = [pool["table"][s].copy() for s in src]
    part = [s != t and n % page != 0 for s, t, n in zip(src, dst, lens)]
    fresh = list(_free(pool))
    if sum(part) > len(fresh):
        return False
    for i, n in enumerate(lens):
        if part[i]:
            to = fresh.pop(0)
            copy_page(pool, table[i][blocks(n, page) - 1], to)
            table[i][blocks(n, page) - 1] = to
    for i, (s, t) in enumerate(zip(src, dst)):
        if s == t:
            continue
        for b in range(blocks(pool["lens"][t], page)):
            pool["refs"][pool["table"][t, b]] -= 1
        nb = blocks(lens[i], page)
        pool["table"][t] = -1
        pool["table"][t, :nb] = table[i][:nb]
        for b in range(nb):
            pool["refs"][table[i][b]] += 1
        pool["lens"][t] = lens[i]
    return True


def compact(pool):
    live = np.flatnonzero(pool["refs"] > 0)
    n = len(live)
    movers, holes = live[live >= n], np.flatnonzero(pool["refs"][:n] == 0)
    for a, b in zip(movers, holes):
        copy_page(pool, a, b)
        pool["refs"][b], pool["refs"][a] = pool["refs"][a], 0
        pool["table"][pool["table"] == a] = b
    return n


SHARE_LEVELS = 4


def share(pool, slots, levels=SHARE_LEVELS):
    """Which leading full pages the listed sequences hold in common: order, own, depth, segments (first place in order,
    members, first token, end, level).  A class of two or more sequences that hold the same page behind the blocks they had in
    common before gets a segment up to the last block that all its members hold in full; what is left of it is divided by the
    next block's page, `levels` times at most.  Classes, and the order, go by their first member."""
    n, page, n_pages = len(slots), pool["kc"].shape[2], len(pool["refs"])
    full, rows = [], []
    for s in slots:
        ok = 0 <= s < len(pool["lens"])
        ids = [int(x) for x in pool["table"][s]] if ok else []
        k = min(max(int(pool["lens"][s]), 0) // page, len(ids)) if ok else 0
        bad = [b for b in range(k) if not 0 <= ids[b] < n_pages]
        full.append(bad[0] if bad else k)
        rows.append(ids)
    own, depth, found = [0] * n, [0] * n, []

    def divide(members, at, level):
        """Members in order of the list -> their order; segments as (level, first member's index, ...)."""
        if level == levels:
            return members
        classes = {}
        for i in members:
            classes.setdefault(rows[i][at] if at < full[i] else ("alone", i), []).append(i)
        order = []
        for group in sorted(classes.values()):
            if len(group) == 1:
                order += group
                continue
            end = at
            while all(end < full[i] and rows[i][end] == rows[group[0]][end] for i in group):
                end += 1
            for i in group:
                own[i], depth[i] = end * page, level + 1
            found.append((level, group[0], len(group), at * page, end * page))
            order += divide(group, end, level + 1)
        return order

    order = divide(list(range(n)), 0, 0)
    place = {i: p for p, i in enumerate(order)}
    segments = [[place[f], m, a, e, level] for level, f, m, a, e in sorted(found, key=lambda x: (x[0], place[x[1]]))]
    return dict(order=order, own=own, depth=depth, segments=segments)
