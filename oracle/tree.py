"""Decoding on drafted trees, in 64 bits and step by step: blocks and slots, attention, sampling, acceptance."""
from __future__ import annotations

import numpy as np

BLOCK = 16


def ancestor_bits(parents, words: int) -> np.ndarray:
    """uint32 [nodes, words]: each node's ancestors and itself."""
    out = np.zeros((len(parents), words), np.uint32)
    for j, p in enumerate(parents):
        if p >= 0:
            out[j] = out[p]
        if j < 32 * words:
            out[j, j // 32] |= np.uint32(1 << (j % 32))
    return out


def depths(parents) -> list[int]:
    out = []
    for p in parents:
        out.append(out[p] + 1 if p >= 0 else 0)
    return out


def reserve(tables, lens, counts, ring, *, block=BLOCK, rows=None, offset=None, parents=None, words=0):
    """Tables [R, cols] and ring [2 + n] are changed in place; returns slots, positions, cu, granted and
    masks of the packed tokens."""
    head, have, ids = int(ring[0]), int(ring[1]), ring[2:]
    cap = tables.shape[1] * block
    slots, pos, cu, granted, masks = [], [], [0], [], []
    stopped, seen = False, set()
    for i, n in enumerate(counts):
        n = max(int(n), 0)
        row = i if rows is None else int(rows[i])
        known = 0 <= row < len(tables)
        start = int(lens[row]) if known else 0
        ok = known and row not in seen and start >= 0 and start + n <= cap
        if known:
            seen.add(row)
        if ok and n:
            want = [j for j in range(start // block, (start + n - 1) // block + 1) if tables[row, j] < 0]
            if want and len(want) > have:
                stopped = True
            if want and stopped:
                ok = False
            for j in want if ok else []:
                tables[row, j] = ids[head]
                head, have = (head + 1) % len(ids), have - 1
        granted.append(n if ok else 0)
        up = [-1] * n if parents is None else list(parents[cu[-1]:cu[-1] + n])
        deep = depths(up) if parents is not None else list(range(n))
        if parents is not None:
            masks.append(ancestor_bits(up, words))
        base = start + (int(offset[row]) if offset is not None and known else 0)
        for j in range(n):
            b = tables[row, (start + j) // block] if ok else -1
            slots.append(int(b) * block + (start + j) % block if b >= 0 else -1)
            pos.append(base + deep[j] if known else deep[j])
        cu.append(cu[-1] + n)
    ring[0], ring[1] = head, have
    return (np.array(slots, np.int64), np.array(pos, np.int32), np.array(cu, np.int32),
            np.array(granted, np.int32), np.concatenate(masks) if masks else None)


def release(tables, keep, ring, *, block=BLOCK, rows=None) -> None:
    head, have, ids = int(ring[0]), int(ring[1]), ring[2:]
    for i, n in enumerate(keep):
        row = i if rows is None else int(rows[i])
        if not 0 <= row < len(tables):
            continue
        for j in range(-(-int(n) // block), tables.shape[1]):
            if tables[row, j] >= 0:
                ids[(head + have) % len(ids)] = tables[row, j]
                have += 1
                tables[row, j] = -1
    ring[1] = have


def attention(q, k_cache, v_cache, tables, ctx, cu, masks=None, rows=None):
    """q [T, NH, D], caches [NB, KVH, 16, D] (any float type), masks uint32 [T, words].  Returns out and
    lse of the trees' rows, and for each row the sum of p |v| and the largest sum of |q k| / sqrt(D)."""
    q = np.asarray(q, np.float64)
    T, NH, D = q.shape
    KVH = k_cache.shape[1]
    out, lse = np.zeros((T, NH, D)), np.full((T, NH), -np.inf)
    size, big = np.zeros((T, NH, D)), np.zeros((T, NH))
    for i, c in enumerate(ctx):
        n = int(cu[i + 1] - cu[i])
        row = i if rows is None else int(rows[i])
        pos = np.arange(int(c) + n)
        ids = tables[row][pos // BLOCK] if n else np.zeros(0, np.int64)
        live = (ids >= 0) & (ids < len(k_cache))
        for j in range(n):
            t = int(cu[i]) + j
            see = live.copy()
            x = pos - int(c)
            if masks is None:
                see &= x <= j
            else:
                bit = np.array([x_ < 0 or (x_ < 32 * masks.shape[1] and
                                           (int(masks[t, x_ // 32]) >> (x_ % 32)) & 1 == 1) for x_ in x])
                see &= bit
            if not see.any():
                continue
            at = ids[see], pos[see] % BLOCK
            for h in range(NH):
                kv = h // (NH // KVH)
                k = np.asarray(k_cache[at[0], kv, at[1]], np.float64)
                v = np.asarray(v_cache[at[0], kv, at[1]], np.float64)
                z = k @ q[t, h] / np.sqrt(D)
                m = z.max()
                e = np.exp(z - m)
                p = e / e.sum()
                out[t, h] = p @ v
                lse[t, h] = m + np.log(e.sum())
                size[t, h] = p @ np.abs(v)
                big[t, h] = (np.abs(k) @ np.abs(q[t, h])).max() / np.sqrt(D)
    return out, lse, size, big


def sample(x, t, u, k=0, p=1.0, m=0.0):
    """Token and log probability of one row of logits."""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf
    if not t > 0:
        return int(np.argmax(x)), 0.0
    order = np.argsort(-x, kind="stable")
    v = x[order]
    if 0 < k < len(v):
        v = v[v >= v[k - 1]]
    with np.errstate(invalid="ignore"):
        w = np.where(v == top, 1.0, np.exp((v - top) / float(t)))
    w = np.where(v == -np.inf, 0.0, w)
    c = np.cumsum(w)
    n = int((w > 0).sum())
    if p < 1:
        n = min(n, int(np.searchsorted(c, max(float(p), 0.0) * c[-1], side="right")) + 1)
    if m > 0:
        n = min(n, int((w >= min(float(m), 1.0)).sum()))
    j = min(n - 1, int(np.searchsorted(c[:n], min(max(float(u), 0.0), 1 - 2.0 ** -24) * c[n - 1], side="right")))
    return int(order[j]), float(np.log(w[j]) - np.log(c[n - 1]))


def accept(tokens, parents, targets, cu, deep: int):
    """Each tree's path and the draws at its nodes."""
    paths, new = [], []
    for a, b in zip(cu[:-1], cu[1:]):
        path = [0] if b > a else []
        while path and len(path) < deep:
            cur = path[-1]
            nxt = [c for c in range(cur + 1, b - a)
                   if parents[a + c] == cur and tokens[a + c] == targets[a + cur]]
            if not nxt:
                break
            path.append(nxt[0])
        paths.append(path)
        new.append([int(targets[a + c]) for c in path])
    return paths, new
