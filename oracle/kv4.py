"""The 4-bit KV cache's format and operators in 64 bits (numpy): the statement that
``tiny_infra_b200.kv4`` is tested against.  No counterpart in the reference project.

Pool [NB, KVH, 18 D] bytes, blocks of 16 tokens; a tile is K codes [16, D/2], V codes [16, D/2],
K scales [D/16, 16], V scales [D/16, 16].
"""
from __future__ import annotations

import numpy as np

BLOCK = 16
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scale_values(b: np.ndarray) -> np.ndarray:
    """Scale bytes -> values: the half-precision number with bits b << 7."""
    return (b.astype(np.uint16) << 7).view(np.float16).astype(np.float64)


def quantize(x: np.ndarray):
    """x [..., D] (values of a 16-bit type) -> (codes uint8 [..., D], scale bytes [..., D/16])."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 16)
    finite = np.isfinite(g).all(-1)
    g = np.where(finite[..., None], g, 0.0)
    a = np.abs(g).max(-1) / 6.0
    e = np.maximum(np.frexp(a)[1] - 1, -14)
    s = np.minimum(np.rint(np.ldexp(a, 3 - e)) * np.ldexp(1.0, e - 3), 10240.0)
    t = np.where(s > 0, s, 1.0)[..., None]
    y = np.abs(g) / t
    mid = (MAGNITUDES[1:] + MAGNITUDES[:-1]) / 2
    code = np.zeros(y.shape, np.uint8)
    for i, m in enumerate(mid):                   # a tie goes to the even code
        code += (y > m) if i % 2 == 0 else (y >= m)
    code = np.where(s[..., None] > 0, code, 0)
    code = np.where((g < 0) & (code > 0), code | 8, code).astype(np.uint8)
    sb = (s.astype(np.float16).view(np.uint16) >> 7).astype(np.uint8)
    sb = np.where(finite, sb, 0xFF).astype(np.uint8)
    return code.reshape(x.shape), sb


def values(code: np.ndarray, scale_bytes: np.ndarray) -> np.ndarray:
    v = MAGNITUDES[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = scale_values(scale_bytes)[..., None]
    return (v.reshape(*scale_bytes.shape, 16) * s).reshape(code.shape)


def untile(tiles: np.ndarray):
    """Tiles [..., 18 D] -> K, V [..., 16, D] in 64 bits."""
    d = tiles.shape[-1] // 18
    lead, h = tiles.shape[:-1], 8 * d

    def one(c, s):
        codes = np.stack([c & 15, c >> 4], -1).reshape(*lead, BLOCK, d)
        return values(codes, np.swapaxes(s.reshape(*lead, d // 16, BLOCK), -1, -2))
    return (one(tiles[..., :h], tiles[..., 2 * h:2 * h + d]),
            one(tiles[..., h:2 * h], tiles[..., 2 * h + d:]))


def put(pool: np.ndarray, k: np.ndarray, v: np.ndarray, slots: np.ndarray) -> None:
    """Append tokens k, v [T, KVH, D] at their slots, in place."""
    d = pool.shape[-1] // 18
    for which, x in ((0, k), (1, v)):
        code, sb = quantize(x)
        packed = code[..., 0::2] | (code[..., 1::2] << 4)
        for t, slot in enumerate(slots):
            if slot < 0 or slot >= pool.shape[0] * BLOCK:
                continue
            b, o = divmod(int(slot), BLOCK)
            at = which * 8 * d + o * (d // 2)
            pool[b, :, at:at + d // 2] = packed[t]
            at = 16 * d + which * d + o
            pool[b, :, at:16 * d + (which + 1) * d:BLOCK] = sb[t]


def positions(table_row: np.ndarray, n: int, num_blocks: int):
    """Positions < n whose table entry holds a block, and their blocks."""
    pos = np.arange(min(n, len(table_row) * BLOCK))
    blk = table_row[pos // BLOCK]
    ok = (blk >= 0) & (blk < num_blocks)
    return pos[ok], blk[ok]


def cached(pool: np.ndarray, table_row: np.ndarray, n: int):
    """K, V [KVH, tokens, D] of the row's first n tokens (those with a block)."""
    pos, _ = positions(table_row, n, pool.shape[0])
    lb, i = np.unique(pos // BLOCK, return_inverse=True)
    k, v = untile(pool[table_row[lb].astype(np.int64)])           # [blocks, KVH, 16, D]
    return (np.swapaxes(k[i, :, pos % BLOCK], 0, 1), np.swapaxes(v[i, :, pos % BLOCK], 0, 1))


def decode(q: np.ndarray, pool: np.ndarray, tables: np.ndarray, ctx: np.ndarray, rows=None):
    """Returns out, lse, and what error bounds need: the weighted mean of |v|, the plain sum of |v|
    over the sum of p (p relative to the row's largest; both out's shape), and the largest sum of
    |q k| / sqrt(D) of each (sequence, head).  Rows with ctx 0 are NaN here."""
    B, NH, D = q.shape
    kvh = pool.shape[1]
    out, mean, flat = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros(q.shape)
    lse, big = np.full((B, NH), -np.inf), np.zeros((B, NH))
    for b in range(B):
        k, v = cached(pool, tables[b if rows is None else rows[b]], int(ctx[b]))
        if ctx[b] <= 0 or k.shape[1] == 0:
            continue
        for h in range(NH):
            kk, vv = k[h * kvh // NH], v[h * kvh // NH]
            s = kk @ q[b, h] / np.sqrt(D)
            m = s.max()
            p = np.exp(s - m)
            out[b, h], mean[b, h] = p @ vv / p.sum(), p @ np.abs(vv) / p.sum()
            flat[b, h] = np.abs(vv).sum(0) / p.sum()
            lse[b, h] = m + np.log(p.sum())
            big[b, h] = (np.abs(kk) @ np.abs(q[b, h])).max() / np.sqrt(D)
    return out, lse, mean, flat, big


def weights(w: np.ndarray, q, lse, pool, tables, ctx, rows=None):
    """(new totals, bound factor per token: sum over heads of p * (1 + |s| + |lse| + sum|qk|))."""
    B, NH, D = q.shape
    kvh = pool.shape[1]
    new, slack = w.astype(np.float64).copy(), np.zeros(w.shape)
    for b in range(B):
        row = tables[b if rows is None else rows[b]]
        pos, blk = positions(row, int(ctx[b]), pool.shape[0])
        k, _ = cached(pool, row, int(ctx[b]))
        for h in range(NH):
            kk = k[h * kvh // NH]
            s = kk @ q[b, h] / np.sqrt(D)
            p = np.exp(s - lse[b, h])
            new[blk, h * kvh // NH, pos % BLOCK] += p
            slack[blk, h * kvh // NH, pos % BLOCK] += p * (
                1 + np.abs(s) + abs(lse[b, h]) + np.abs(kk) @ np.abs(q[b, h]) / np.sqrt(D))
    return new, slack


def survivors(w: np.ndarray, keep: int, recent: int) -> np.ndarray:
    """Positions that stay of one sequence and kv head with totals w [n]."""
    n = len(w)
    if n <= keep:
        return np.arange(n)
    key = np.where(np.isnan(w), np.inf, w.astype(np.float64))
    nan = np.isnan(w)
    old = np.arange(n - recent)
    order = np.lexsort((old, -key[old], ~nan[old]))     # NaN first, then by weight, then by place
    return np.sort(np.concatenate([order[:keep - recent], np.arange(n - recent, n)]))


def evict(pool, w, tables, ctx, keep, recent, out_tables=None, rows=None):
    """In place on pool [L, NB, KVH, 18 D] and w [L, NB, KVH, 16]; returns kept positions
    {(layer, b, head): array}."""
    out_tables = tables if out_tables is None else out_tables
    L, NB, KVH, tile = pool.shape
    d, kept = tile // 18, {}
    codes = np.concatenate([np.arange(d // 2), 8 * d + np.arange(d // 2)])
    scales = 16 * d + BLOCK * np.arange(d // 8)
    for la in range(L):
        for b in range(len(ctx)):
            r, n = (b if rows is None else rows[b]), int(ctx[b])
            if n <= 0:
                continue
            for h in range(KVH):
                pos = np.arange(n)
                idx = survivors(w[la, tables[r, pos // BLOCK], h, pos % BLOCK], keep, recent)
                kept[la, b, h] = idx
                sb, so = tables[r, idx // BLOCK], idx % BLOCK
                to = np.arange(len(idx))
                db, do = out_tables[r, to // BLOCK], to % BLOCK
                c = pool[la, sb[:, None], h, codes + so[:, None] * (d // 2)]
                s = pool[la, sb[:, None], h, scales + so[:, None]]
                ww = w[la, sb, h, so].copy()
                pool[la, db[:, None], h, codes + do[:, None] * (d // 2)] = c
                pool[la, db[:, None], h, scales + do[:, None]] = s
                w[la, db, h, do] = ww
    return kept


def prefill(q, pool, tables, starts, counts, rows=None):
    """out and the bounds' terms as ``decode`` gives them; causal over positions 0 .. start + i."""
    out, mean, flat, big = (np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape),
                            np.zeros(q.shape[:2]))
    at = 0
    for i, (s, n) in enumerate(zip(starts, counts)):
        for j in range(n):
            r = i if rows is None else rows[i]
            o, _, m, f, g = decode(q[at:at + 1], pool, tables[r:r + 1], np.array([s + j + 1]))
            out[at], mean[at], flat[at], big[at] = o[0], m[0], f[0], g[0]
            at += 1
    return out, mean, flat, big
