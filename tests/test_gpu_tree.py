"""The operators of a step on drafted trees (paging, tree, sampler.sample) against 64-bit step-by-step
forms, and run together as a step runs them."""
import numpy as np
import pytest
import torch

from oracle import tree as oracle

pytestmark = pytest.mark.gpu


def _status():
    from tiny_infra_b200 import _native as N
    return N.device_status()


def _dev(a, dtype=None):
    t = torch.as_tensor(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def _random_parents(rng, n, wide=4):
    return [-1] + [int(rng.integers(max(0, j - wide), j)) for j in range(1, n)] if n else []


# ---- reserve and release ---------------------------------------------------------------------------
def _layout(rng, lens, cols, extra, rows=None, block=16):
    """Tables [R, cols] with the cached tokens' blocks, and a ring that has gone round with `extra` blocks."""
    R = len(lens)
    need = [-(-int(n) // block) for n in lens]
    ids = rng.permutation(sum(need) + extra + 5).astype(np.int32)
    tables = np.full((R, cols), -1, np.int32)
    at = 0
    for r, n in enumerate(need):
        tables[r, :n] = ids[at:at + n]
        at += n
    ring = np.zeros(2 + sum(need) + extra + 3, np.int32)
    size = len(ring) - 2
    ring[0], ring[1] = max(0, size - 3), extra
    ring[2 + (ring[0] + np.arange(extra)) % size] = ids[at:at + extra]
    return tables, ring


def _reserve(tables, lens, counts, ring, cap, *, block=16, rows=None, offset=None, parents=None, words=0):
    from tiny_infra_b200 import paging
    d = dict(tables=_dev(tables), ring=_dev(ring), slots=torch.full((cap,), 77, dtype=torch.int64, device="cuda"),
             pos=torch.full((cap,), 77, dtype=torch.int32, device="cuda"),
             cu=torch.full((len(counts) + 1,), 77, dtype=torch.int32, device="cuda"),
             granted=torch.full((len(counts),), 77, dtype=torch.int32, device="cuda"), masks=None)
    kw = {}
    if rows is not None:
        kw["row_index"] = _dev(rows, torch.int32)
    if offset is not None:
        kw["pos_offset"] = _dev(offset, torch.int32)
    if parents is not None:
        full = np.zeros(cap, np.int32)
        full[:len(parents)] = parents
        kw["parents"] = _dev(full)
        if words:
            d["masks"] = kw["masks"] = torch.full((cap, words), 77, dtype=torch.int32, device="cuda")
    paging.reserve(d["tables"], _dev(lens, torch.int32), _dev(counts, torch.int32), d["ring"], d["slots"], d["pos"],
                   d["cu"], block_size=block, granted=d["granted"], **kw)
    return {k: None if v is None else v.cpu().numpy() for k, v in d.items()}


def _check_reserve(rng, lens, counts, extra, *, cols=None, block=16, rows=None, offset=None, tree=False, words=0,
                   behind=3):
    cols = cols or max(-(-(int(n) + 300) // block) for n in lens) if cols is None else cols
    tables, ring = _layout(rng, lens, cols, extra, block=block)
    parents = sum((_random_parents(rng, n) for n in counts), []) if tree else None
    total = int(sum(counts))
    got = _reserve(tables, lens, counts, ring, total + behind, block=block, rows=rows, offset=offset,
                   parents=parents, words=words)
    slots, pos, cu, granted, masks = oracle.reserve(tables, lens, counts, ring, block=block, rows=rows,
                                                    offset=offset, parents=parents, words=words)
    np.testing.assert_array_equal(got["granted"], granted)
    np.testing.assert_array_equal(got["tables"], tables)
    np.testing.assert_array_equal(got["cu"], cu)
    np.testing.assert_array_equal(got["slots"], np.concatenate([slots, np.full(behind, -1)]))
    np.testing.assert_array_equal(got["pos"], np.concatenate([pos, np.zeros(behind, np.int32)]))
    np.testing.assert_array_equal(got["ring"][:2], ring[:2])
    if words:
        np.testing.assert_array_equal(got["masks"].view(np.uint32),
                                      np.concatenate([masks, np.zeros((behind, words), np.uint32)]))
    return got


@pytest.mark.parametrize("seqs", [1, 2, 31, 33, 257, 4096])
def test_reserve_one_token_each(seqs):
    rng = np.random.default_rng(seqs)
    _check_reserve(rng, rng.integers(0, 200, seqs), [1] * seqs, extra=seqs)
    assert _status() == 0


@pytest.mark.parametrize("seqs,most,extra", [(1, 1, 1), (3, 700, 500), (40, 900, 1200), (70, 33, 60), (1300, 70, 900),
                                             (9, 40000, 9000)])
def test_reserve_ragged(seqs, most, extra):
    """Counts from none to many, the pool short in some; the last case takes the second launch."""
    rng = np.random.default_rng(most)
    lens, counts = rng.integers(0, 100, seqs), rng.integers(0, most + 1, seqs)
    _check_reserve(rng, lens, counts, extra, cols=-(-(100 + most) // 16))
    assert _status() == 0


@pytest.mark.parametrize("nodes,words", [(1, 1), (31, 1), (32, 1), (33, 2), (64, 2), (129, 5), (200, 7)])
def test_reserve_trees(nodes, words):
    rng = np.random.default_rng(nodes)
    counts = [nodes, 1, 0, max(1, nodes // 2), nodes, 3 % (nodes + 1)]
    rows = rng.permutation(9)[:6].astype(np.int32)
    _check_reserve(rng, rng.integers(0, 400, 9), counts, extra=200, rows=rows, offset=rng.integers(0, 9, 9), tree=True,
                   words=words)
    _check_reserve(rng, rng.integers(0, 400, 9), counts, extra=200, rows=rows, tree=True)
    assert _status() == 0


def test_reserve_other_block_sizes():
    rng = np.random.default_rng(4)
    for block in (1, 5, 32):
        _check_reserve(rng, rng.integers(0, 90, 12), rng.integers(0, 60, 12), extra=100, block=block)


def test_reserve_short_pool_serves_in_order():
    """The first that does not fit ends it; those behind that need no block are still served."""
    rng = np.random.default_rng(5)
    got = _check_reserve(rng, [0, 15, 16, 3, 3, 31], [40, 1, 20, 5, 20, 2], extra=4)
    assert got["granted"].tolist() == [40, 1, 0, 5, 0, 0]
    assert _status() == 0


def test_reserve_bad_rows_are_left_out():
    """A row named twice, one outside the table, a length beyond the row: no blocks for them, the status
    bit for the caller; padding rows (-1) in silence."""
    from tiny_infra_b200 import _native as N
    rng = np.random.default_rng(6)
    for rows, bad in (([2, 0, 2, 1], True), ([2, 0, 7, 1], True), ([2, 0, -1, 1], False)):
        _check_reserve(rng, [3, 3, 3], [20, 20, 20, 20], extra=30, rows=np.array(rows, np.int32), cols=10)
        assert _status() == (N.TI_DEVERR_BAD_INPUT if bad else 0)
    _check_reserve(rng, [3, 150, 3], [20, 20, 20], extra=30, cols=10)
    assert _status() == N.TI_DEVERR_BAD_INPUT


def test_reserve_buffers_too_small():
    """More tokens than places: what fits is written, and the status says so."""
    from tiny_infra_b200 import _native as N
    rng = np.random.default_rng(7)
    tables, ring = _layout(rng, [0, 5, 9], 20, 40)
    got = _reserve(tables, [0, 5, 9], [30, 30, 30], ring, 50)
    slots, pos, cu, _, _ = oracle.reserve(tables, [0, 5, 9], [30, 30, 30], ring)
    np.testing.assert_array_equal(got["slots"], slots[:50])
    np.testing.assert_array_equal(got["tables"], tables)
    assert got["cu"].tolist() == [0, 30, 60, 90] and _status() == N.TI_DEVERR_BAD_INPUT


def test_reserve_parent_behind_its_child():
    from tiny_infra_b200 import _native as N
    rng = np.random.default_rng(8)
    tables, ring = _layout(rng, [4], 4, 3)
    assert _reserve(tables, [4], [4], ring, 4, parents=[-1, 3, 1, 2])["pos"].tolist() == [4, 4, 5, 6]
    assert _status() == N.TI_DEVERR_BAD_INPUT
    tables, ring = _layout(rng, [4], 4, 3)
    got = _reserve(tables, [4], [4], ring, 4, parents=[-1, 3, 1, 2], words=1)
    assert got["masks"].ravel().tolist() == [1, 2, 6, 14]      # node 1 is taken for a root
    assert got["pos"].tolist() == [4, 4, 5, 6] and _status() == N.TI_DEVERR_BAD_INPUT


@pytest.mark.parametrize("seqs", [1, 7, 40, 600])
def test_release(seqs):
    from tiny_infra_b200 import paging
    rng = np.random.default_rng(seqs)
    lens = rng.integers(0, 700, seqs)
    tables, ring = _layout(rng, lens, 50, 9)
    rows = rng.permutation(seqs)[:max(1, seqs - 2)].astype(np.int32)
    keep = (lens[rows] * rng.random(len(rows))).astype(np.int32) * rng.integers(0, 2, len(rows)).astype(np.int32)
    dt, dr = _dev(tables), _dev(ring)
    paging.release(dt, _dev(keep), dr, row_index=_dev(rows))
    oracle.release(tables, keep, ring, rows=rows)
    np.testing.assert_array_equal(dt.cpu().numpy(), tables)
    assert paging.free_ids(dr) == paging.free_ids(torch.from_numpy(ring))
    assert _status() == 0


def test_release_row_twice_and_full_ring():
    from tiny_infra_b200 import _native as N
    from tiny_infra_b200 import paging
    tables = _dev(np.array([[4, 5, 6], [7, -1, 8]], np.int32))
    ring = paging.free_list([1], capacity=6)
    paging.release(tables, _dev([0, 16, 0], torch.int32), ring, row_index=_dev([1, 0, 1], torch.int32))
    assert paging.free_ids(ring) == [1, 7, 8, 5, 6] and tables.cpu().tolist() == [[4, -1, -1], [-1, -1, -1]]
    assert _status() == N.TI_DEVERR_BAD_INPUT
    tables[1, 0] = 9
    tables[1, 1] = 10
    paging.release(tables, _dev([0, 0], torch.int32), ring)       # three blocks, room for one
    assert paging.free_ids(ring) == [1, 7, 8, 5, 6] and tables.cpu().tolist() == [[4, -1, -1], [9, 10, -1]]
    assert _status() == N.TI_DEVERR_BAD_INPUT


def test_reserve_as_the_host_allocator():
    """The same requests through BlockAllocator and on the device hand out the same blocks."""
    from tiny_infra_b200 import paging
    from tiny_infra_b200.cache_manager import BlockAllocator
    rng = np.random.default_rng(9)
    host = BlockAllocator(12, 400, 16, num_blocks=120)
    tables = torch.full((12, 25), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(12, dtype=torch.int32, device="cuda")
    ring = paging.new_free_list(120)
    for step in range(12):
        if step % 4 == 3:
            gone = rng.permutation(12)[:4]
            for s in gone:
                host.free_slot(int(s))
            paging.release(tables, _dev(np.zeros(4, np.int32)), ring, row_index=_dev(gone, torch.int32))
            lens[_dev(gone)] = 0
        slots = rng.permutation(12)[:6]
        counts = rng.integers(0, 40, 6)
        mapping, _ = host.plan_tokens(slots, counts)
        host.advance(slots, counts)
        cap = int(counts.sum())
        sm = torch.empty(cap, dtype=torch.int64, device="cuda")
        pos = torch.empty(cap, dtype=torch.int32, device="cuda")
        cu = torch.empty(7, dtype=torch.int32, device="cuda")
        rows = _dev(slots, torch.int32)
        paging.reserve(tables, lens, _dev(counts, torch.int32), ring, sm, pos, cu, row_index=rows)
        lens[rows.long()] += _dev(counts, torch.int32)
        np.testing.assert_array_equal(sm.cpu().numpy(), mapping)
        np.testing.assert_array_equal(tables.cpu().numpy(), host.block_tables)
        assert paging.free_ids(ring) == list(host.free_blocks)
    assert _status() == 0


# ---- attention ---------------------------------------------------------------------------------------
def _scene(rng, nh, kvh, d, dtype, ctx, counts, *, cols_extra=2, rows=None, masks="tree", words=None):
    S, T = len(ctx), int(sum(counts))
    R = S if rows is None else max(rows) + 2
    table_row = list(range(S)) if rows is None else list(rows)
    cols = max(-(-(c + n) // 16) for c, n in zip(ctx, counts)) + cols_extra
    need = [-(-(c + n) // 16) for c, n in zip(ctx, counts)]
    ids = rng.permutation(sum(need) + 3)
    tables = np.full((R, cols), -1, np.int32)
    at = 0
    for r, n in zip(table_row, need):
        tables[r, :n] = ids[at:at + n]
        at += n
    nb = sum(need) + 3
    k = torch.from_numpy(rng.standard_normal((nb, kvh, 16, d)) * np.exp(0.5 * rng.standard_normal(d))).to(dtype)
    v = torch.from_numpy(rng.standard_normal((nb, kvh, 16, d))).to(dtype)
    q = torch.from_numpy(rng.standard_normal((T, nh, d))).to(dtype)
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    bits = None
    words = words or max(1, -(-max(counts) // 32))
    if masks == "tree":
        bits = [oracle.ancestor_bits(_random_parents(rng, n), words) for n in counts]
        bits = np.concatenate(bits) if T else np.zeros((0, words), np.uint32)
    elif masks == "random":
        bits = rng.integers(0, 2 ** 32, (T, words), dtype=np.uint64).astype(np.uint32)
        bits[rng.random(T) < 0.3] = 0
    return dict(q=q, k=k, v=v, tables=tables, ctx=np.array(ctx, np.int32), cu=cu, masks=bits,
                rows=None if rows is None else np.array(rows, np.int32))


def _attend(s, behind=2, strides=True):
    from tiny_infra_b200 import tree
    T, nh, d = s["q"].shape
    wide = torch.zeros(T + behind, (nh + 3) * d, dtype=s["q"].dtype, device="cuda")
    q = wide[:, :nh * d].view(T + behind, nh, d) if strides else torch.zeros(T + behind, nh, d, dtype=s["q"].dtype,
                                                                            device="cuda")
    q[:T] = s["q"].cuda()
    out = torch.full((T + behind, (nh + 1) * d), 7.0, dtype=q.dtype, device="cuda")[:, :nh * d].view(T + behind, nh, d)
    lse = torch.full((T + behind, nh), 7.0, device="cuda")
    masks = None
    if s["masks"] is not None:
        masks = torch.zeros(T + behind, s["masks"].shape[1], dtype=torch.int32, device="cuda")
        masks[:T] = _dev(s["masks"].view(np.int32))
    tree.attention(out, q, s["k"].cuda(), s["v"].cuda(), _dev(s["tables"]), _dev(s["ctx"]), _dev(s["cu"]), masks=masks,
                   row_index=None if s["rows"] is None else _dev(s["rows"]), lse=lse)
    assert (out[T:] == 7).all() and (lse[T:] == 7).all()
    return out[:T].cpu(), lse[:T].cpu()


def _limits(dtype, ref, size, big):
    """How far a result may be off.  The weights are rounded to the type (half a step each), as is the
    result; a score of n products in 32 bits is off by less than 2^-24 * 16 of the sum of their sizes (sums
    of sums of 16), which is a relative error of the weights; 2^-20 covers the exponential, the sums and
    the joins."""
    half = torch.finfo(dtype).eps / 2
    score = 2.0 ** -20 + 2.0 ** -20 * big
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return half * np.abs(ref) + (half * (1 + half) + 2 * score[..., None]) * size + tiny, score


def _check_attention(s, **kw):
    out, lse = _attend(s, **kw)
    # what no node sees does not matter to the plain form, which looks at seen tokens only
    as64 = lambda t: t.double().numpy()                                                  # noqa: E731
    ref, rl, size, big = oracle.attention(as64(s["q"]), as64(s["k"]), as64(s["v"]), s["tables"], s["ctx"], s["cu"],
                                          s["masks"], s["rows"])
    lim, score = _limits(s["q"].dtype, ref, size, big)
    off = np.abs(out.double().numpy() - ref)
    assert (off <= lim).all(), (off / np.maximum(lim, 1e-30)).max()
    none = np.isneginf(rl)
    assert (np.isneginf(lse.numpy()) == none).all()
    off = np.abs(lse.double().numpy() - np.where(none, 0, rl))[~none]
    assert (off <= (score + 2.0 ** -22 * np.abs(rl))[~none]).all()
    assert _status() == 0
    return out, lse


HEADS = [(14, 2, 64, torch.bfloat16), (8, 8, 64, torch.float16), (16, 1, 128, torch.bfloat16),
         (9, 3, 128, torch.float16), (5, 1, 64, torch.bfloat16)]


@pytest.mark.parametrize("masks", ["tree", "random", None])
@pytest.mark.parametrize("nh,kvh,d,dtype", HEADS)
def test_attention(nh, kvh, d, dtype, masks):
    """Contexts and trees from nothing to several chunks, the edges of blocks, chunks and tiles among them."""
    rng = np.random.default_rng(nh * d)
    ctx = [0, 1, 15, 16, 63, 64, 65, 130, 0, 300, 47, 127]
    counts = [1, 5, 0, 17, 1, 64, 33, 2, 40, 9, 70, 3]
    _check_attention(_scene(rng, nh, kvh, d, dtype, ctx, counts, masks=masks))


@pytest.mark.parametrize("nh,kvh,d,dtype", [HEADS[0], HEADS[3]])
def test_attention_long_contexts(nh, kvh, d, dtype):
    """Keys cut over many CTAs; one, few and many nodes."""
    rng = np.random.default_rng(d)
    for ctx, counts in (([9000], [1]), ([5003], [70]), ([4000, 17, 2500], [3, 2, 33])):
        _check_attention(_scene(rng, nh, kvh, d, dtype, ctx, counts))


@pytest.mark.parametrize("masks", ["tree", "random", None])
@pytest.mark.parametrize("nh,kvh,d,dtype", HEADS)
def test_attention_weights_in_two_parts(nh, kvh, d, dtype, masks):
    """Weights as the sum of two values of the cache's type, as in the decode and prefill attention over the same
    cache.  The first is off by half a step at most, the second is the rest and off by half a step of that:
    half^2 of the weight, and for fp16, whose weights are held times 2^7 and whose steps end at 2^-24,
    2^-25 / 2^7 of the largest (kept below 2^8 times a row's own, so 2^-32 of it).  One, two and three tiles a
    unit, one chunk and many."""
    rng = np.random.default_rng(nh + d)
    wide = 128 // (nh // kvh)
    for ctx, counts in (([0, 1, 30, 70], [3, 9, 1, 5]), ([500, 90], [2 * wide + 1, wide + 3]), ([1500], [8])):
        s = _scene(rng, nh, kvh, d, dtype, ctx, counts, masks=masks)
        out, _ = _attend(s)
        as64 = lambda t: t.double().numpy()                                              # noqa: E731
        ref, _, size, big = oracle.attention(as64(s["q"]), as64(s["k"]), as64(s["v"]), s["tables"], s["ctx"], s["cu"],
                                             s["masks"])
        half, score = torch.finfo(dtype).eps / 2, 2.0 ** -20 + 2.0 ** -20 * big
        low = 2.0 ** -32 * float(s["v"].abs().max()) * (sum(ctx) + sum(counts)) + 2.0 ** -25 if dtype == torch.float16 else 0.0
        lim = half * np.abs(ref) + (1 + half) * (half * half + 2 * score[..., None]) * size + low
        off = np.abs(out.double().numpy() - ref)
        assert (off <= lim).all(), (off / np.maximum(lim, 1e-30)).max()
    assert _status() == 0


def test_attention_many_sequences():
    rng = np.random.default_rng(3)
    n = 700
    ctx, counts = rng.integers(0, 60, n).tolist(), rng.integers(0, 4, n).tolist()
    _check_attention(_scene(rng, 2, 1, 64, torch.bfloat16, ctx, counts))


@pytest.mark.parametrize("nh,kvh,d,dtype", [HEADS[0], HEADS[2], HEADS[3]])
def test_attention_full_units_and_what_is_left(nh, kvh, d, dtype):
    """Trees of one to eleven tiles: alone, in few sequences behind long contexts, and in many."""
    rng = np.random.default_rng(nh)
    group = nh // kvh
    nodes = lambda tiles: max(1, tiles * 128 // group - int(rng.integers(0, 5)))         # noqa: E731
    for tiles in (3, 4, 5, 7):
        _check_attention(_scene(rng, nh, kvh, d, dtype, [700], [nodes(tiles)]))
    _check_attention(_scene(rng, nh, kvh, d, dtype, [2500, 0, 1300, 40], [nodes(4), 0, nodes(11), nodes(1)]))
    many = [nodes(int(n)) if n else 0 for n in rng.integers(0, 6, 37)]
    _check_attention(_scene(rng, nh, kvh, d, dtype, rng.integers(0, 300, 37).tolist(), many))


def test_attention_large_trees():
    rng = np.random.default_rng(4)
    _check_attention(_scene(rng, 7, 1, 64, torch.bfloat16, [100, 3], [300, 129]))
    _check_attention(_scene(rng, 4, 1, 128, torch.float16, [100, 3], [300, 129], masks=None))


def test_attention_rows_holes_and_words():
    """Row index, table entries that hold no block, mask rows with fewer or more bits than nodes."""
    rng = np.random.default_rng(5)
    s = _scene(rng, 14, 2, 64, torch.bfloat16, [200, 90, 33], [20, 40, 3], rows=[4, 0, 2])
    s["tables"][4, [1, 7]] = -1
    s["tables"][0, 2] = s["k"].shape[0] + 5
    _check_attention(s)
    for words in (1, 4):
        _check_attention(_scene(rng, 4, 2, 64, torch.float16, [50, 9], [40, 50], masks="random", words=words))


@pytest.mark.parametrize("nh,kvh,d,dtype", [HEADS[0], HEADS[3]])
def test_attention_sees_nothing(nh, kvh, d, dtype):
    """No context and no bits, or a table without blocks: zeros, and -inf."""
    rng = np.random.default_rng(6)
    s = _scene(rng, nh, kvh, d, dtype, [0, 20, 0], [5, 2, 3], masks="random")
    s["masks"][:] = 0
    out, lse = _check_attention(s)
    assert (out[:5] == 0).all() and torch.isneginf(lse[:5]).all()
    s["tables"][1] = -1
    out, lse = _check_attention(s)
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("nh,kvh,d,dtype", [HEADS[0], HEADS[3]])
def test_attention_unseen_values_stay_out(nh, kvh, d, dtype, bad):
    """NaN and infinities where a node does not look: behind the last token, in other blocks, in drafts on
    other branches; a node that does look gets them."""
    rng = np.random.default_rng(7)
    s = _scene(rng, nh, kvh, d, dtype, [70, 200, 5], [20, 3, 50])
    used = np.zeros((s["k"].shape[0], 16), bool)
    for i, (c, n) in enumerate(zip([70, 200, 5], [20, 3, 50])):
        pos = np.arange(c + n)
        used[s["tables"][i][pos // 16], pos % 16] = True
    for x in (s["k"], s["v"]):
        x.permute(0, 2, 1, 3)[torch.from_numpy(~used)] = bad
    clean, _ = _check_attention(s)
    # a draft whose values are bad: exactly those that have its bit are
    for i, node in ((0, 4), (2, 33)):
        p = int(s["ctx"][i]) + node
        at = int(s["tables"][i][p // 16]), p % 16
        old = s["v"][at[0], :, at[1]].clone()
        s["v"][at[0], :, at[1], 3] = bad
        out, _ = _attend(s)
        rows = range(int(s["cu"][i]), int(s["cu"][i + 1]))
        for t in range(len(out)):
            sees = t in rows and (int(s["masks"][t, node // 32]) >> (node % 32)) & 1
            if sees:
                assert not torch.isfinite(out[t, :, 3]).any()
                rest = [e for e in range(d) if e != 3]
                assert torch.equal(out[t][:, rest], clean[t][:, rest])
            else:
                assert torch.equal(out[t], clean[t])
        s["v"][at[0], :, at[1]] = old
        k_old = s["k"][at[0], :, at[1]].clone()
        s["k"][at[0], :, at[1]] = float("nan")
        out, lse = _attend(s)
        for t in range(len(out)):
            sees = t in rows and (int(s["masks"][t, node // 32]) >> (node % 32)) & 1
            assert torch.isnan(out[t]).all() if sees else torch.equal(out[t], clean[t])
        s["k"][at[0], :, at[1]] = k_old
    assert _status() == 0


def test_attention_one_token():
    """Sizes of one, and a token stride that means nothing then."""
    rng = np.random.default_rng(9)
    for ctx in (0, 16, 200):
        s = _scene(rng, 1, 1, 64, torch.bfloat16, [ctx], [1])
        _check_attention(s, behind=0, strides=False)
    from tiny_infra_b200 import tree
    q = torch.zeros(3, 1, 67, dtype=torch.bfloat16, device="cuda")[:1, :, :64].expand(1, 1, 64)
    q = q.as_strided((1, 1, 64), (67, 64, 1))
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    tree.attention(out, q, s["k"].cuda(), s["v"].cuda(), _dev(s["tables"]), _dev(s["ctx"]), _dev(s["cu"]))
    assert torch.isfinite(out).all() and _status() == 0


def test_attention_large_scores():
    """Scores of hundreds, growing along the keys, so that the running maximum moves all the time."""
    rng = np.random.default_rng(8)
    s = _scene(rng, 4, 2, 64, torch.bfloat16, [700], [6])
    for p in range(706):
        s["k"][int(s["tables"][0, p // 16]), :, p % 16] *= 1 + p / 20
    _check_attention(s)


# ---- sampling ---------------------------------------------------------------------------------------
def _draw(x, t, u, k, p, m, dtype):
    from tiny_infra_b200 import sampler
    wide = torch.zeros(x.shape[0], x.shape[1] + 3, dtype=dtype, device="cuda")
    wide[:, :x.shape[1]] = x.to(dtype).cuda()
    lp = torch.full((len(x),), 7.0, device="cuda")
    f = lambda a: _dev(np.asarray(a, np.float32))                                        # noqa: E731
    tok = sampler.sample(wide[:, :x.shape[1]], f(t), f(u), top_ks=None if k is None else _dev(k, torch.int32),
                         top_ps=None if p is None else f(p), min_ps=None if m is None else f(m), logprobs=lp)
    return tok.cpu().numpy(), lp.cpu().numpy()


def _check_draw(x, t, u, k, p, m, dtype):
    """Equal tokens; log probabilities within 2^-20 (32-bit result, and the 2^-44 steps of the weights)."""
    tok, lp = _draw(x, t, u, k, p, m, dtype)
    f32 = lambda a, i, default: default if a is None else float(np.float32(a[i]))        # noqa: E731
    xr = x.to(dtype).double().numpy()
    for i in range(len(x)):
        rt, rl = oracle.sample(xr[i], f32(t, i, 1), f32(u, i, 0), 0 if k is None else int(k[i]), f32(p, i, 1.0),
                               f32(m, i, 0.0))
        assert tok[i] == rt, (i, tok[i], rt)
        assert lp[i] == rl or abs(lp[i] - rl) <= 2.0 ** -20 * max(1.0, abs(rl)), (i, lp[i], rl)
    assert _status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 4099, 32000, 151936])
def test_sample_mixed_rows(vocab, dtype):
    rng = np.random.default_rng(vocab)
    rows = 23
    x = torch.from_numpy(rng.standard_normal((rows, vocab)) * rng.choice([0.3, 2.0, 6.0], (rows, 1)))
    t = rng.choice([0.0, 0.5, 0.8, 1.0, 1.7], rows)
    k = rng.choice([0, 1, 2, 20, 511, 700, 5000, vocab, vocab + 1], rows)
    p = rng.choice([1.0, 0.0, 0.3, 0.9, 0.99, 1.5], rows)
    m = rng.choice([0.0, 0.0, 1e-4, 0.05, 0.5, 1.0, 2.0], rows)
    u = np.concatenate([[0.0, 1 - 2.0 ** -24, 0.5], rng.random(rows - 3)])
    _check_draw(x, t, u, k, p, m, dtype)
    _check_draw(x, np.full(rows, 0.7), u, None, None, None, dtype)
    _check_draw(x, np.full(rows, 0.7), u, np.full(rows, 20), np.full(rows, 0.9), None, dtype)
    _check_draw(x, np.full(rows, 1.3), u, None, np.full(rows, 0.95), np.full(rows, 0.02), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sample_ties(dtype):
    """Few distinct values: the k-th one is shared by thousands, and draws fall among equal values."""
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.integers(-3, 2, (12, 20011)) * 0.5)
    x[5] = 1.25
    x[6, ::2] = -float("inf")
    u = rng.random(12)
    for k, p, m in ((None, None, None), (np.full(12, 30), None, None), (np.full(12, 9000), np.full(12, 0.7), None),
                    (None, np.full(12, 0.4), None), (None, None, np.full(12, 0.5))):
        _check_draw(x, np.full(12, 0.9), u, k, p, m, dtype)


def test_sample_nan_and_infinities():
    """NaN is never drawn, +inf always, a row of neither number gives -1."""
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.standard_normal((8, 3001)))
    x[0, ::3] = float("nan")
    x[1] = float("nan")
    x[2] = -float("inf")
    x[3, [5, 77, 1999]] = float("inf")
    x[4, 1:] = -float("inf")
    x[5, 10:] = float("nan")
    x[6] = float("inf")
    u = np.array([0.9, 0.5, 0.5, 0.6, 0.9, 0.99, 0.3, 0.2])
    for t in (0.0, 0.8):
        for k, p in ((None, None), (np.full(8, 20), np.full(8, 0.9)), (None, np.full(8, 0.9))):
            _check_draw(x, np.full(8, t), u, k, p, np.full(8, 0.0), torch.float32)
            _check_draw(x, np.full(8, t), u, k, p, np.full(8, 0.1), torch.bfloat16)


def test_sample_parameters_out_of_range():
    """NaN and values beyond a parameter's range keep everything, or the first of the largest (temperature)."""
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((5, 5003)) * 2)
    nan, u = float("nan"), rng.random(5)
    full = _draw(x, np.ones(5), u, None, None, None, torch.float32)
    for k, p, m in ((np.full(5, -3), np.full(5, nan), np.full(5, nan)), (np.full(5, 9000), np.full(5, 7.0), np.full(5, -1.0))):
        got = _draw(x, np.ones(5), u, k, p, m, torch.float32)
        assert (got[0] == full[0]).all() and (got[1] == full[1]).all()
    top = x.float().argmax(1).numpy()
    for t in (nan, -1.0):
        assert (_draw(x, np.full(5, t), u, None, None, None, torch.float32)[0] == top).all()
    got = _draw(x, np.ones(5), np.array([-1.0, nan, 2.0, 1.0, 0.0]), None, None, None, torch.float32)[0]
    want = _draw(x, np.ones(5), np.array([0.0, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.0]), None, None, None, torch.float32)[0]
    assert (got == want).all() and _status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [8, 4088, 4096, 4104, 12304, 20488, 150008])
def test_sample_aligned_rows(vocab, dtype):
    """Rows that wide loads can read, lengths around whole rounds of them; what lies behind a row is the next."""
    from tiny_infra_b200 import sampler
    rng = np.random.default_rng(vocab)
    rows = 9
    x = torch.from_numpy(rng.standard_normal((rows, vocab)) * 2).to(dtype)
    x[::2] += 9                                              # (the next row must not be seen)
    u, f = rng.random(rows), lambda v: torch.full((rows,), v, device="cuda")             # noqa: E731
    d, du = x.cuda(), _dev(u.astype(np.float32))
    for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (20, 0.9, 0.0), (3000, 0.8, 0.0), (0, 1.0, 0.05)):
        tok = sampler.sample(d, f(0.8), du, top_ks=torch.full((rows,), k, dtype=torch.int32, device="cuda"),
                             top_ps=f(p), min_ps=f(m)).cpu().numpy()
        for i in range(rows):
            t32 = [float(np.float32(v)) for v in (0.8, u[i], p, m)]
            assert tok[i] == oracle.sample(x[i].double().numpy(), t32[0], t32[1], k, t32[2], t32[3])[0], (k, p, m, i)
    assert _status() == 0


def test_sample_temperatures_from_tiny_to_huge():
    """Where one value is all, where all are equally likely, and logits as small as the temperature."""
    rng = np.random.default_rng(11)
    t = np.array([1e-44, 1e-40, 3e-37, 2e-36, 1e-30, 1e-6, 1e4, 1e30, 3e38], np.float32)
    u, n = rng.random(len(t)), len(t)
    plain = rng.standard_normal((n, 6007))
    near = np.clip(t.astype(np.float64)[:, None] * rng.standard_normal((n, 6007)) * 2, -3e38, 3e38)
    for x in (plain, near):
        x[:, ::5] = -float("inf")
        for p in (None, np.full(n, 0.9)):
            _check_draw(torch.from_numpy(x.astype(np.float32)), t, u, None, p, None, torch.float32)


def test_sample_equal_and_flat_rows():
    """Rows of one value (thousands of ties), rows that hardly differ, and a few large vocabularies."""
    rng = np.random.default_rng(4)
    for vocab in (9001, 151936):
        x = torch.zeros(6, vocab, dtype=torch.float64)
        x[1] = 3.5
        x[2] = torch.from_numpy(rng.standard_normal(vocab) * 1e-3)
        x[3, vocab // 2:] = -1.0
        x[4] = torch.from_numpy(np.round(rng.standard_normal(vocab)))
        x[5] = torch.linspace(-30, 30, vocab)
        u = rng.random(6)
        for k, p, m in ((None, None, None), (None, np.full(6, 0.7), None), (np.full(6, 5000), np.full(6, 0.9), None),
                        (np.full(6, 40), np.full(6, 0.9), None), (None, None, np.full(6, 0.3)),
                        (None, np.full(6, 0.999), np.full(6, 0.01))):
            _check_draw(x, np.full(6, 0.8), u, k, p, m, torch.float32)
    x = torch.from_numpy(rng.standard_normal((2, 1 << 18)) * 2)
    _check_draw(x, np.ones(2), rng.random(2), None, None, None, torch.bfloat16)
    x = torch.from_numpy(rng.standard_normal((2, (1 << 20) + 3)) * 2)
    _check_draw(x, np.ones(2), rng.random(2), np.array([0, 30]), np.full(2, 0.95), None, torch.float32)


def test_sample_far_from_the_top():
    """Draws in the thin tail, where a place is known by what is behind it; extreme temperatures."""
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((24, 151936)) * rng.choice([0.5, 1.5, 2.5], (24, 1)))
    u = 1 - 10.0 ** -rng.uniform(2, 6.5, 24)
    _check_draw(x, np.full(24, 1.1), u, None, None, None, torch.float32)
    _check_draw(x, np.full(24, 1.1), u, None, np.full(24, 0.9995), None, torch.float32)
    _check_draw(x[:6, :20000], np.array([1e-4, 1e-30, 1e3, 1e30, 30.0, 1e-2]), u[:6], None, None, None, torch.float32)


def test_sample_infinite_temperature():
    """Every finite value is equally likely, -inf and NaN still never drawn; by all ways to a token."""
    rng = np.random.default_rng(14)
    n = 12
    for vocab, scale in ((700, 1.0), (30011, 1.0), (30011, 1e38), (30011, 0.0)):
        x = np.clip(rng.standard_normal((n, vocab)) * scale, -3e38, 3e38)
        x[:, ::3] = -np.inf
        x[:, 1::11] = np.nan
        x[0, 5:] = -np.inf
        u, inf = rng.random(n), np.full(n, np.inf)
        for k, p, m in ((None, None, None), (None, np.full(n, 0.6), None), (np.full(n, 20), np.full(n, 0.9), None),
                        (np.full(n, 600), np.full(n, 0.5), None), (None, None, np.full(n, 0.3)),
                        (None, np.full(n, 0.7), np.full(n, 1.0))):
            _check_draw(torch.from_numpy(x), inf, u, k, p, m, torch.float32)


def test_sample_thin_ties_of_a_huge_vocabulary():
    """One likely token and four million of equal weights near 2^-41, of which a draw near the end takes one: its
    place from the formula (a running sum in 64 bits would lose part of each weight).  With top-p behind it too."""
    n, u = 1 << 22, 1 - 2.0 ** -21
    x = torch.full((2, n), -28.4, dtype=torch.float64)
    x[:, 5] = 0.0
    tok, lp = _draw(x, np.ones(2), np.array([u, 0.5]), None, None, None, torch.float32)
    w = np.exp(float(np.float32(-28.4)))
    # the likely token first, then the others by index: place 1 + q has the sum 1 + (q + 1) w
    q = int(np.floor(u * (n - 1) - (1 - u) / w))
    assert abs(int(tok[0]) - (q if q < 5 else q + 1)) <= 1 and tok[1] == 5
    assert abs(lp[0] - (np.log(w) - np.log1p((n - 1) * w))) < 2.0 ** -18
    tok, _ = _draw(x, np.ones(2), np.array([u, 0.5]), None, np.full(2, 1 - 2.0 ** -22), None, torch.float32)
    kept = np.floor((1 - 2.0 ** -22) * (n - 1) - 2.0 ** -22 / w) + 1             # tokens behind the likely one
    q = int(np.floor(u * kept - (1 - u) / w))
    assert abs(int(tok[0]) - (q if q < 5 else q + 1)) <= 1 and tok[1] == 5 and _status() == 0


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (40, 151936), (256, 151936), (700, 9000)])
def test_sample_min_p_same_bits_every_run(rows, vocab):
    """Several CTAs a row and one: tokens and log probabilities repeat.  Half of the rows have one likely token
    and 2000 of weights around 2^-54, whose sum is lost or not by the order in which it is taken, and
    which the likely one's log probability is."""
    from tiny_infra_b200 import sampler
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, vocab, generator=gen, device="cuda") * 2
    r = slice(0, None, 2)
    x[r] = torch.where(torch.rand(x[r].shape, generator=gen, device="cuda") < 2000 / vocab, -37.4 + 0.1 * x[r], -80.0)
    x[r, vocab // 3] = 0.0
    t, u = torch.ones(rows, device="cuda"), torch.rand(rows, generator=gen, device="cuda")
    m = torch.full((rows,), 0.01, device="cuda")
    m[r] = 1e-20
    first = None
    for _ in range(40):
        lp = torch.zeros(rows, device="cuda")
        tok = sampler.sample(x, t, u, min_ps=m, logprobs=lp)
        if first is None:
            first = tok, lp
        assert torch.equal(tok, first[0]) and torch.equal(lp, first[1])
    assert (first[1][r] <= 0).all() and (first[1][r] > -2.0 ** -40).all() and _status() == 0


def test_sample_frequencies():
    """A grid of uniforms draws each token as often as its probability says."""
    probs = np.array([0.5, 0.25, 0.125, 0.0625, 0.0625])
    x = torch.from_numpy(np.log(probs)).repeat(4096, 1)
    tok, _ = _draw(x, np.ones(4096), (np.arange(4096) + 0.5) / 4096, None, None, None, torch.float32)
    # log and its rounding to 32 bits move a border by less than a millionth: less than a grid step
    assert np.abs(np.bincount(tok, minlength=5) - 4096 * probs).max() <= 1


# ---- acceptance -------------------------------------------------------------------------------------
def _accept_scene(rng, counts, layers, kvh, d, bs, dtype, agree=0.7):
    T = int(sum(counts))
    parents = sum((_random_parents(rng, n) for n in counts), [])
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    tokens = rng.integers(0, 50, T)
    targets = rng.integers(0, 50, T)
    for i, n in enumerate(counts):
        for c in range(1, n):
            if rng.random() < agree:
                targets[cu[i] + parents[cu[i] + c]] = tokens[cu[i] + c]
    nb = -(-(T + 40) // bs)
    shape = (layers, nb, kvh, bs, d)
    return dict(tokens=tokens, parents=np.array(parents, np.int32), targets=targets, cu=cu,
                slots=rng.permutation(nb * bs)[:T].astype(np.int64),
                k=torch.from_numpy(rng.standard_normal(shape)).to(dtype),
                v=torch.from_numpy(rng.standard_normal(shape)).to(dtype))


def _check_accept(s, deep, out_slots=None, rows=None, lens=None):
    from tiny_infra_b200 import tree
    B, bs = len(s["cu"]) - 1, s["k"].shape[-2]
    k, v = s["k"].cuda(), s["v"].cuda()
    num = torch.full((B,), 7, dtype=torch.int32, device="cuda")
    path = torch.full((B, deep), 7, dtype=torch.int32, device="cuda")
    new = torch.full((B, deep), 7, dtype=torch.int32, device="cuda")
    dl = None if lens is None else _dev(lens, torch.int32)
    i32 = lambda a: _dev(a, torch.int32)                                                 # noqa: E731
    tree.accept(k, v, i32(s["tokens"]), i32(s["parents"]), i32(s["targets"]), i32(s["cu"]), _dev(s["slots"]), num, path,
                new, out_slots=None if out_slots is None else _dev(out_slots), seq_lens=dl,
                row_index=None if rows is None else i32(rows))
    paths, news = oracle.accept(s["tokens"], s["parents"], s["targets"], s["cu"].tolist(), deep)
    pad = lambda a: a + [-1] * (deep - len(a))                                           # noqa: E731
    assert num.cpu().tolist() == [len(p) for p in paths]
    assert path.cpu().tolist() == [pad(p) for p in paths] and new.cpu().tolist() == [pad(p) for p in news]
    to = s["slots"] if out_slots is None else out_slots
    limit = s["k"].shape[-4] * bs
    for old, got in ((s["k"], k.cpu()), (s["v"], v.cpu())):
        want = old.clone()
        for i, p in enumerate(paths):
            for j, c in enumerate(p):
                a, b = int(s["slots"][s["cu"][i] + c]), int(to[s["cu"][i] + j])
                if 0 <= a < limit and 0 <= b < limit:
                    want[..., b // bs, :, b % bs, :] = old[..., a // bs, :, a % bs, :]
        assert torch.equal(got, want)
    if lens is not None:
        want = np.array(lens)
        for i, p in enumerate(paths):
            want[i if rows is None else rows[i]] += len(p)
        assert dl.cpu().tolist() == want.tolist()
    return paths


@pytest.mark.parametrize("layers,kvh,d,bs,dtype", [(1, 1, 64, 16, torch.bfloat16), (3, 2, 64, 16, torch.float16),
                                                   (2, 5, 128, 16, torch.bfloat16), (2, 3, 24, 7, torch.float16)])
def test_accept(layers, kvh, d, bs, dtype):
    rng = np.random.default_rng(layers * d)
    counts = [8, 1, 0, 64, 33, 2, 130, 600]
    s = _accept_scene(rng, counts, layers, kvh, d, bs, dtype)
    rows = rng.permutation(11)[:len(counts)]
    paths = _check_accept(s, 40, rows=rows, lens=rng.integers(0, 99, 11))
    assert max(len(p) for p in paths) > 2 and min(len(p) for p in paths) == 0
    _check_accept(s, 2, lens=rng.integers(0, 99, len(counts)))
    free = np.setdiff1d(np.arange(s["k"].shape[1] * bs), s["slots"])
    s2 = _accept_scene(rng, [8, 5, 20], layers, kvh, d, bs, dtype)
    free = np.setdiff1d(np.arange(s2["k"].shape[1] * bs), s2["slots"])
    _check_accept(s2, 9, out_slots=rng.permutation(free)[:33].astype(np.int64))
    assert _status() == 0


def test_accept_long_chain_in_place():
    """A chain whose every other node is a dead end: the kept ones all move, over places of kept ones."""
    rng = np.random.default_rng(1)
    n = 301
    s = _accept_scene(rng, [n], 2, 2, 64, 16, torch.bfloat16)
    s["parents"] = np.array([-1] + [max(0, 2 * ((j - 1) // 2)) for j in range(1, n)], np.int32)
    s["tokens"] = np.arange(n)
    s["targets"] = np.minimum(np.arange(n) + 2, n)
    assert len(_check_accept(s, 400)[0]) == 151
    s["slots"] = np.arange(n)[::-1].astype(np.int64).copy()
    _check_accept(s, 400)


def test_accept_slots_outside_the_pool():
    from tiny_infra_b200 import _native as N
    rng = np.random.default_rng(2)
    s = _accept_scene(rng, [30, 9], 2, 1, 64, 16, torch.bfloat16, agree=1.0)
    s["slots"][:6] = -1
    _check_accept(s, 10)
    assert _status() == 0
    s["slots"][:6] = 1 << 40
    _check_accept(s, 10)
    assert _status() == N.TI_DEVERR_BAD_INPUT
