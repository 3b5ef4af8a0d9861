"""A plain restatement of the KV cache in pages: the order of a page's values, RoPE, attention in
float64, and forks, growth and compaction as loops over the tables."""
import math

import numpy as np
import torch

BLOCK = 16


def rope(x, cos, sin):
    """rotate_half in f32, every product and sum rounded."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    c, s = np.asarray(cos, np.float32), np.asarray(sin, np.float32)
    return np.concatenate([a * c - b * s, b * c + a * s], axis=-1).astype(np.float32)


def rounded(x, dtype):
    """f32 values rounded to the pages' type (to nearest even), as a tensor of it."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(dtype)


def put(pool, page, head, slot, k, v):
    """One slot's K and V rows [hd] (of the pool's type) into a CPU pool [n, 2, kv, page, hd]."""
    pool[page, 0, head, slot] = k
    hd = k.shape[-1]
    pool[page, 1, head].view(-1, hd, BLOCK)[slot // BLOCK, :, slot % BLOCK] = v


def get(pool, page, head, slot):
    hd = pool.shape[-1]
    return (pool[page, 0, head, slot],
            pool[page, 1, head].reshape(-1, hd, BLOCK)[slot // BLOCK, :, slot % BLOCK])


def rows(pool, table, n, head):
    """Slots 0 .. n - 1 of a KV head in float64 (zeros where there is no page) and whether each
    has a page."""
    n_pages, _, _, page, hd = pool.shape
    ids = np.asarray(table)[:-(-n // page)].astype(np.int64)
    ok = (ids >= 0) & (ids < n_pages)
    got = pool[torch.from_numpy(np.where(ok, ids, 0))][:, :, head].double()
    k = got[:, 0].reshape(-1, hd).numpy()
    v = got[:, 1].reshape(-1, page // BLOCK, hd, BLOCK).transpose(-1, -2).reshape(-1, hd).numpy()
    there = np.repeat(ok, page)
    return np.where(there[:, None], k, 0)[:n], np.where(there[:, None], v, 0)[:n], there[:n]


def attend(q, k, v, there):
    """softmax(q k / sqrt(hd)) v of the rows that are there, and sum p |v| per channel."""
    k, v = k[there], v[there]
    s = k @ q / math.sqrt(q.shape[-1])
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v, p @ np.abs(v)


def fork(tables, lengths, refs, parents):
    t, n, r = tables.copy(), lengths.copy(), refs.copy()
    for s, p in enumerate(parents):
        ok = 0 <= p < len(parents)
        t[s] = tables[p] if ok else -1
        n[s] = lengths[p] if ok else 0
        for old, new in zip(tables[s], t[s]):
            if old != new:
                if 0 <= old < len(refs):
                    r[old] -= 1
                if 0 <= new < len(refs):
                    r[new] += 1
    return t, n, r


def grow(tables, lengths, refs, rows_, page):
    """(tables, refs, room, copies [(src, dst, blocks)]) after room for rows_ more rows."""
    t, r = tables.copy(), refs.copy()
    columns, room, copies = t.shape[1], [], []
    for s, (n, m) in enumerate(zip(lengths.tolist(), rows_)):
        end = max(n, 0)
        if n >= 0 and m > 0 and n < columns * page:
            for c in range(n // page, min((n + m - 1) // page, columns - 1) + 1):
                p = t[s, c]
                none = not 0 <= p < len(r)
                if none or r[p] > 1:
                    free = np.flatnonzero(r <= 0)
                    if not len(free):
                        break
                    f = free[0]
                    t[s, c], r[f] = f, 1
                    if not none:
                        r[p] -= 1
                        if c == n // page and n % page:
                            copies.append((int(p), int(f), -(-(n % page) // BLOCK)))
                end = (c + 1) * page
        room.append(max(end, n, 0))
    return t, r, np.array(room), copies


def compact(tables, refs):
    """(tables, refs, live, moves [(src, dst)])."""
    live = int((refs > 0).sum())
    at = np.arange(len(refs))
    src, dst = at[(refs > 0) & (at >= live)], at[(refs <= 0) & (at < live)]
    to, r = at.copy(), refs.copy()
    to[src], r[dst], r[src] = dst, refs[src], 0
    ok = (tables >= 0) & (tables < len(refs))
    return (np.where(ok, to[np.where(ok, tables, 0)], tables), r, live,
            list(zip(src.tolist(), dst.tolist())))


def shared_tables(rng, n_seq, columns, n_pages, used, shared):
    """Random tables: the first ``shared`` columns of all sequences name the same pages, the rest
    of each its own, up to ``used[s]`` columns; and the counts of the pages."""
    ids = rng.permutation(n_pages)
    t = np.full((n_seq, columns), -1, np.int32)
    at = shared
    for s in range(n_seq):
        u = used[s]
        t[s, :min(shared, u)] = ids[:min(shared, u)]
        if u > shared:
            t[s, shared:u] = ids[at:at + u - shared]
            at += u - shared
    assert at <= n_pages
    return t, np.bincount(t[t >= 0], minlength=n_pages).astype(np.int32)
