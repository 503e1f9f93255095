"""The 4-bit KV cache's operators (tiny_infra_b200.kv4) against the 64-bit oracle (oracle.kv4).

Tolerances.  u = half a unit in the last place of the output type relative to the value
(finfo.eps / 2).  Quantised values, moves, positions and read-backs are exact.  Attention: the
kernels multiply the exact cached values; scores are float32 sums of D products, off by at most
ds = (D + 8) 2^-24 max_t sum|q k| / sqrt(D); each exponential adds 2^-21; the weights that multiply
V may be rounded to half precision (2^-11 relative; with p = 1 for the row's largest held as
2^14, weights below 2^-28 are multiples of 2^-38, each off by at most 2^-39: without this term a
dim whose only nonzero values belong to such tokens has no error left to be in).  With
A = sum p |v| / sum p and F = sum |v| / sum p:
  |out - exact| <= max(u |exact|, u tiny) + A (2^-11 + 2 ds + 2^-20) + 2^-39 F
where tiny is the type's smallest normal number: outputs below it are multiples of 2 u tiny (fp16:
2^-24), so rounding moves them by up to u tiny whatever their size.
  |lse - exact| <= ds + 2^-20 + 2^-22 |lse|
A total of attention weight adds, per head, p * (ds + (1 + |s| + |lse|) 2^-20) and one rounding
2^-23 of the total.  Prefill: the same with p = 1 held as 2^7 (its running maximum may trail the
row's by 2^8): weights below 2^-21 are multiples of 2^-31, each off by at most 2^-32, against the
running maximum up to 2^8 times less: 2^-31 F covers what is left of them at the row's end.
"""
import numpy as np
import pytest
import torch

from oracle import kv4 as OK

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def kv4(cuda_device):
    from tiny_infra_b200 import _native, kv4
    _native.device_status()
    yield kv4
    assert _native.device_status() == 0


def half_step(x, dt):
    """Largest rounding error of storing values around x in the type."""
    f = torch.finfo(dt)
    return f.eps / 2 * np.maximum(np.abs(x), f.smallest_normal)


def dev(a, dt=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dt is None else t.to(dt)


def rounded(a, dt):
    """Values of the type, in 64 bits."""
    return torch.from_numpy(np.asarray(a)).to(dt).double().numpy()


def random_pool(rng, nb, kvh, d, amp=1.0):
    """Every byte random: codes any, scales around amp (no NaN)."""
    pool = rng.integers(0, 256, (nb, kvh, 18 * d), dtype=np.uint8)
    s = amp * np.exp(0.5 * rng.standard_normal((nb, kvh, 2 * d))) / 3
    pool[..., 16 * d:] = (s.astype(np.float16).view(np.uint16) >> 7).astype(np.uint8)
    return pool


def poison(pool, tables, lens, num):
    """Scale bytes behind each sequence's end, and of blocks in no table, become NaN or huge."""
    d = pool.shape[-1] // 18
    used = np.zeros(pool.shape[0], bool)
    for r, n in enumerate(lens):
        for j in range(min(-(-int(n) // 16), tables.shape[1])):
            if 0 <= tables[r, j] < num:
                used[tables[r, j]] = True
                left = n - 16 * j
                if left < 16:
                    sc = pool[tables[r, j], :, 16 * d:].reshape(pool.shape[1], -1, 16)
                    sc[..., left:] = 0xFF
                    pool[tables[r, j], :, 16 * d:] = sc.reshape(pool.shape[1], -1)
    pool[~used, :, 16 * d:] = 0xFF


def tables_for(rng, lens, spare=3, width=None):
    need = [-(-int(n) // 16) for n in lens]
    nb = sum(need) + spare
    width = max(max(need, default=1), 1) if width is None else width
    t = np.full((len(lens), width), -1, np.int32)
    perm, at = rng.permutation(nb), 0
    for i, n in enumerate(need):
        t[i, :n] = perm[at:at + n]
        at += n
    return t, nb


# ---- append and read back ------------------------------------------------------------------------
@pytest.mark.parametrize("dtn", ["bf16", "fp16"])
@pytest.mark.parametrize("d,kvh,tokens", [(64, 2, 1), (64, 2, 77), (64, 1, 300), (128, 3, 50),
                                          (128, 8, 513)])
def test_append_matches_the_format(kv4, dtn, d, kvh, tokens):
    rng = np.random.default_rng(tokens + d)
    dt, nb = DT[dtn], tokens // 16 + 5
    amp = np.exp2(rng.integers(-22, 15, (tokens, kvh, d // 16, 1)))
    x = [rounded((rng.standard_normal((tokens, kvh, d // 16, 16)) * amp).reshape(tokens, kvh, d), dt)
         for _ in range(2)]
    # ties: multiples of a quarter of a power of two under a group maximum of 6 (scale 1)
    x[0][0, 0, :16] = [6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -1.25, -1.75, -2.5, -3.5,
                       -5, 0]
    x[1][0, 0, :16] = 0
    if tokens > 50:
        x[0][3, 0, 5], x[1][4, 0, 20], x[1][5, 0, 0] = np.nan, np.inf, -np.inf
        if dtn == "bf16":
            x[0][6, 0, 16:32] = rounded(np.linspace(1e5, 3e38, 16), dt)      # saturates
        x[1][7, 0, :16] = rounded(np.full(16, 1e-7), dt)
    slots = rng.permutation(nb * 16)[:tokens].astype(np.int64)
    if tokens > 1:
        slots[1] = -1
    before = rng.integers(0, 256, (nb, kvh, 18 * d), dtype=np.uint8)
    pool, want = dev(before), before.copy()
    w = torch.full((nb, kvh, 16), 3.0, device="cuda")
    row = torch.zeros(tokens, 5 * kvh, d, dtype=dt, device="cuda")            # strided slices
    row[:, kvh:2 * kvh], row[:, 3 * kvh:4 * kvh] = dev(x[0], dt), dev(x[1], dt)
    kv4.append(pool, row[:, kvh:2 * kvh], row[:, 3 * kvh:4 * kvh], dev(slots), weights=w)
    OK.put(want, x[0], x[1], slots)
    got = pool.cpu().numpy()
    np.testing.assert_array_equal(got[..., 16 * d:], want[..., 16 * d:])
    gk, gv = OK.untile(got)
    wk, wv = OK.untile(want)
    live = slots[slots >= 0]
    for g, e in ((gk, wk), (gv, wv)):
        np.testing.assert_array_equal(g[live // 16, :, live % 16], e[live // 16, :, live % 16])
    rest = np.ones((nb, 16), bool)                       # every other token's bytes are as before
    rest[live // 16, live % 16] = False
    c0 = before[..., :16 * d].reshape(nb, kvh, 2, 16, d // 2)
    c1 = got[..., :16 * d].reshape(nb, kvh, 2, 16, d // 2)
    for o in range(16):
        np.testing.assert_array_equal(c1[rest[:, o], :, :, o], c0[rest[:, o], :, :, o])
    ww = w.cpu().numpy()
    assert (ww[live // 16, :, live % 16] == 0).all() and (ww[rest.nonzero()[0], :, rest.nonzero()[1]] == 3).all()
    # read back
    ko = torch.full((nb, kvh, 16, d), 7.0, dtype=dt, device="cuda")
    vo = torch.full_like(ko, 7.0)
    t = dev(rng.permutation(nb).astype(np.int32)[None])
    kv4.dequantize(pool, t, dev(np.array([nb * 16], np.int32)), t, ko, vo)
    # (the random bytes of the other tokens hold scales that append never writes: 6 times those is
    # beyond fp16, and comes back as an infinity)
    np.testing.assert_array_equal(ko.double().cpu().numpy(), rounded(gk, dt))
    np.testing.assert_array_equal(vo.double().cpu().numpy(), rounded(gv, dt))


def test_append_every_16_bit_magnitude(kv4):
    """All finite fp16 (and the bf16 that matter) under group maxima of several sizes."""
    for dt in (torch.float16, torch.bfloat16):
        bits = torch.arange(0, 0x7C00 if dt == torch.float16 else 0x7F80, dtype=torch.int16)
        v = bits.view(dt)
        pad = (-len(v)) % 15
        v = torch.cat([v, torch.zeros(pad, dtype=dt)])
        g = v.view(-1, 15)
        for mult in (1.0, 1.375, 3.3, 7.0, 40.0):
            top = (g.double().abs().amax(1, keepdim=True) * mult).clamp(max=6e4 if dt == torch.float16 else 3e38).to(dt)
            x = torch.cat([top, g], 1)
            n = -(-x.shape[0] // 4)
            x = torch.cat([x, torch.zeros(4 * n - x.shape[0], 16, dtype=dt)]).view(n, 1, 64)
            pool = kv4.new_pool(-(-n // 16), 1, 64)
            kv4.append(pool, x.cuda(), -x.cuda(), torch.arange(n, device="cuda"))
            code, sb = OK.quantize(x.double().numpy())
            want = OK.values(code, sb).reshape(n, 64)
            gk, gv = OK.untile(pool.cpu().numpy())
            np.testing.assert_array_equal(gk.reshape(-1, 64)[:n], want)
            np.testing.assert_array_equal(gv.reshape(-1, 64)[:n], -want)


def test_bad_slots_and_tables_are_flagged(cuda_device):
    from tiny_infra_b200 import _native as N
    from tiny_infra_b200 import kv4
    N.device_status()
    pool = kv4.new_pool(3, 2, 64)
    k = torch.ones(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    kv4.append(pool, k, k, torch.tensor([48, 5], device="cuda"))
    assert N.device_status() == N.TI_DEVERR_BAD_INPUT
    got = pool.cpu().numpy()
    assert got[0].any() and not got[1:].any()
    out = torch.full((2, 2, 16, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    vo = out.clone()
    t = lambda *r: torch.tensor(r, dtype=torch.int32, device="cuda")      # noqa: E731
    kv4.dequantize(pool, t([0, 7, 1]), t(40), t([1, 0, 2]), out, vo)
    assert N.device_status() == N.TI_DEVERR_BAD_INPUT                     # target block 2 of 2
    assert (out[0] == 0).all() and out[1].any()                           # source 7 holds nothing
    w = torch.rand(3, 2, 16, device="cuda")
    before, wb = pool.clone(), w.clone()
    kv4.evict(pool, w, t([0, 5]), t(20), 4, 1)
    assert N.device_status() == N.TI_DEVERR_BAD_INPUT
    kv4.evict(pool, w, t([0, 1]), t(40), 4, 1)                            # longer than its table
    assert N.device_status() == N.TI_DEVERR_BAD_INPUT
    assert torch.equal(pool, before) and torch.equal(w, wb)


# ---- decode attention and weight totals ---------------------------------------------------------------
CASES = [
    # nh, kvh, d, dt, lens
    (14, 2, 64, "bf16", [1]),
    (14, 2, 64, "fp16", [16, 17, 15, 1, 2, 33]),
    (14, 2, 64, "bf16", [512, 0, 1, 37, 100, 511, 300, 64]),
    (8, 8, 64, "fp16", [200, 31, 65]),
    (32, 8, 128, "fp16", [129, 1, 700]),
    (9, 3, 128, "bf16", [47, 48, 49, 0]),
    (16, 1, 64, "bf16", [400, 5]),
    (12, 1, 128, "fp16", [90]),
    (1, 1, 64, "bf16", [1000, 3]),
    (10, 2, 64, "bf16", [0, 0]),
    (14, 2, 64, "bf16", [20000]),
    (14, 2, 64, "fp16", list(range(0, 150, 1))),
    (4, 2, 128, "bf16", [3000, 1, 5000, 17]),
]


def make_decode(rng, nh, kvh, d, dtn, lens, qamp=1.0, width=None):
    dt = DT[dtn]
    lens = np.array(lens, np.int32)
    tables, nb = tables_for(rng, lens, width=width)
    pool = random_pool(rng, nb, kvh, d)
    poison(pool, tables, lens, nb)
    q = rounded(rng.standard_normal((len(lens), nh, d)) * qamp, dt)
    return dt, lens, tables, nb, pool, q


def check_decode(out, lse, exact, dt, d, rows):
    o, l, mean, flat, big = exact
    ds = (d + 8) * 2.0 ** -24 * big
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    tol = (half_step(o, dt) + mean * (2.0 ** -11 + 2 * ds[..., None] + 2.0 ** -20) +
           2.0 ** -39 * flat)
    bad = ~(np.abs(out - o) <= tol)
    n_bad = int(bad[rows].sum())
    assert n_bad == 0, (np.argwhere(bad)[:4].tolist(), (np.abs(out - o) - tol)[bad][:4])
    assert (np.abs(lse - l) <= ds + 2.0 ** -20 + 2.0 ** -22 * np.abs(l))[rows].all()


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{len(c[4])}x{max(c[4])}")
@pytest.mark.parametrize("wide", [False, True])
def test_decode_and_weights(kv4, case, wide):
    nh, kvh, d, dtn, lens = case
    rng = np.random.default_rng(nh * 1000 + len(lens))
    need = max(-(-max(lens) // 16), 1)
    dt, lens, tables, nb, pool, q = make_decode(rng, nh, kvh, d, dtn, lens,
                                                width=need + 200 if wide else None)
    B = len(lens)
    rows = lens > 0
    big = torch.zeros(B, nh + 3, d, dtype=dt, device="cuda")         # strided q and out
    big[:, :nh] = dev(q, dt)
    outb = torch.full((B, nh + 2, d), 5.0, dtype=dt, device="cuda")
    out, lse = outb[:, :nh], torch.full((B, nh), 5.0, device="cuda")
    dp, dtab, dl = dev(pool), dev(tables), dev(lens)
    kv4.decode_attention(out, big[:, :nh], dp, dtab, dl, lse=lse)
    exact = OK.decode(q, pool, tables, lens)
    check_decode(out, lse, exact, dt, d, rows)
    assert (out[dev(~rows)] == 5).all() and (lse[dev(~rows)] == 5).all()
    assert (outb[:, nh:] == 5).all()
    out2, lse2 = torch.empty_like(out), torch.empty_like(lse)
    kv4.decode_attention(out2, big[:, :nh], dp, dtab, dl, lse=lse2)
    assert torch.equal(out2[dev(rows)], out[dev(rows)]) and torch.equal(lse2[dev(rows)], lse[dev(rows)])
    assert torch.equal(dp.cpu(), torch.from_numpy(pool))
    # totals, with the log-sum-exp the attention gave
    w = rng.random((nb, kvh, 16)).astype(np.float32)
    dw, dn = dev(w), torch.full((nb, kvh, 16), -1.0, device="cuda")
    kv4.accumulate_weights(dw, big[:, :nh], lse, dp, dtab, dl, out=dn)
    l = np.where(rows[:, None], lse.double().cpu().numpy(), 0)
    new, slack = OK.weights(w, q, l, pool, tables, lens)
    own = np.zeros((nb, kvh, 16), bool)
    for b in range(B):
        pos, blk = OK.positions(tables[b], int(lens[b]), nb)
        own[blk, :, pos % 16] = True
    got = dn.double().cpu().numpy()
    tol = slack * (2.0 ** -20 + (d + 8) * 2.0 ** -24) + 2.0 ** -23 * np.abs(new)
    assert (np.abs(got - new) <= tol)[own].all(), np.max((np.abs(got - new) / tol)[own])
    assert (got[~own] == -1).all()
    kv4.accumulate_weights(dw, big[:, :nh], lse, dp, dtab, dl)       # in place: the same values
    assert torch.equal(dw[dev(own)], dn[dev(own)])
    assert torch.equal(dw[dev(~own)], dev(w)[dev(~own)])


@pytest.mark.parametrize("qamp", [1e-30, 1e-4, 30.0, 3000.0])
@pytest.mark.parametrize("dtn", ["bf16", "fp16"])
def test_decode_query_magnitudes(kv4, dtn, qamp):
    if dtn == "fp16" and qamp < 1e-5:
        qamp = 1e-6
    rng = np.random.default_rng(5)
    dt, lens, tables, nb, pool, q = make_decode(rng, 14, 2, 64, dtn, [300, 40, 1, 16], qamp)
    q[1, 3] = 0.0
    out, lse = torch.empty(4, 14, 64, dtype=dt, device="cuda"), torch.empty(4, 14, device="cuda")
    kv4.decode_attention(out, dev(q, dt), dev(pool), dev(tables), dev(lens), lse=lse)
    check_decode(out, lse, OK.decode(q, pool, tables, lens), dt, 64, lens > 0)


def test_decode_table_holes_row_index_and_shared_rows(kv4):
    """Entries outside the pool hold no tokens; rows picked by row_index, one of them twice."""
    rng = np.random.default_rng(9)
    dt, lens, tables, nb, pool, q = make_decode(rng, 14, 2, 64, "bf16", [400, 90, 33, 200, 48])
    pool[..., 16 * 64:][pool[..., 16 * 64:] == 0xFF] = 60
    tables[0, 3], tables[0, 24], tables[1, 0] = -1, nb, 1 << 30
    tables[2, :] = -1
    rows = np.array([3, 0, 1, 2, 0, 4], np.int32)
    ctx = np.array([200, 400, 90, 33, 177, 1000], np.int32)       # the last one: past its table
    q = q[[0, 1, 2, 3, 4, 1]]
    out = torch.zeros(6, 14, 64, dtype=dt, device="cuda")
    lse = torch.zeros(6, 14, device="cuda")
    kv4.decode_attention(out, dev(q, dt), dev(pool), dev(tables), dev(ctx), row_index=dev(rows),
                         lse=lse)
    exact = OK.decode(q, pool, tables, ctx, rows)
    check_decode(out, lse, exact, dt, 64, np.array([True, True, True, False, True, True]))
    assert torch.isnan(out[3]).all() and (lse[3] == -torch.inf).all()
    w = torch.zeros(nb, 2, 16, device="cuda")
    one = dev(rows[[0, 1, 2, 3]])
    kv4.accumulate_weights(w, dev(q, dt)[:4], lse[:4].contiguous(), dev(pool), dev(tables),
                           dev(ctx[:4]), row_index=one)
    new, slack = OK.weights(np.zeros((nb, 2, 16)), q[:4], lse[:4].double().cpu().numpy(), pool,
                            tables, ctx[:4], rows)
    tol = slack * (2.0 ** -20 + 72 * 2.0 ** -24) + 2.0 ** -23 * np.abs(new)
    assert (np.abs(w.double().cpu().numpy() - new) <= tol).all()


def test_decode_nan_keys_and_values_reach_the_output(kv4):
    """A NaN group inside the length gives NaN where the formula does, and only there."""
    rng = np.random.default_rng(3)
    dt, lens, tables, nb, pool, q = make_decode(rng, 4, 2, 64, "bf16", [100, 100, 100])
    pool[tables[0, 2], 0, 16 * 64 + 5] = 0xFF             # K group 0, token 5, head 0
    pool[tables[1, 2], 1, 16 * 64 + 64 + 16 + 3] = 0xFF   # V group 1, token 3, head 1
    out, lse = torch.empty(3, 4, 64, dtype=dt, device="cuda"), torch.empty(3, 4, device="cuda")
    kv4.decode_attention(out, dev(q, dt), dev(pool), dev(tables), dev(lens), lse=lse)
    n = torch.isnan(out).cpu()
    assert n[0, :2].all() and not n[0, 2:].any() and not n[2].any()
    assert n[1, 2:, 16:32].all() and not n[1, :2].any()
    assert not n[1, 2:, :16].any() and not n[1, 2:, 32:].any()
    assert torch.isnan(lse[0, :2]).all() and not torch.isnan(lse[1:]).any()


def test_decode_flat_tail_keeps_its_mass(kv4):
    """One heavy token and 20000 tokens of weight 2^-17 each: their sum is 15 % of the output."""
    rng = np.random.default_rng(4)
    n, d = 20001, 64
    tables, nb = tables_for(rng, [n])
    k, v = np.zeros((n, 1, d)), np.ones((n, 1, d))
    k[7, 0, 0] = 6.0
    v[7] = -2.0
    pool = np.zeros((nb, 1, 18 * d), np.uint8)
    pos = np.arange(n)
    dp = dev(pool)
    kv4.append(dp, dev(k, torch.bfloat16), dev(v, torch.bfloat16),
               dev(tables[0, pos // 16].astype(np.int64) * 16 + pos % 16))
    q = np.zeros((1, 1, d))
    q[0, 0, 0] = rounded(17 * np.log(2) * 8 / 6, torch.bfloat16)
    out, lse = torch.empty(1, 1, d, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 1, device="cuda")
    lens = np.array([n], np.int32)
    kv4.decode_attention(out, dev(q, torch.bfloat16), dp, dev(tables), dev(lens), lse=lse)
    check_decode(out, lse, OK.decode(q, dp.cpu().numpy(), tables, lens), torch.bfloat16, d,
                 np.array([True]))


def test_decode_large_batch_and_pool_offsets(kv4):
    """4096 sequences; a pool beyond 2^31 bytes with the cached blocks at its end."""
    rng = np.random.default_rng(6)
    nh, kvh, d, B = 14, 2, 64, 4096
    lens = rng.integers(0, 20, B).astype(np.int32)
    tables, nb = tables_for(rng, lens)
    pool = random_pool(rng, nb, kvh, d)
    q = rounded(rng.standard_normal((B, nh, d)), torch.bfloat16)
    far = (1 << 32) // (kvh * 18 * d) + 10
    big = torch.zeros(far + nb, kvh, 18 * d, dtype=torch.uint8, device="cuda")
    big[far:] = dev(pool)
    t = np.where(tables >= 0, tables + far, tables).astype(np.int32)
    out = torch.zeros(B, nh, d, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(B, nh, device="cuda")
    kv4.decode_attention(out, dev(q, torch.bfloat16), big, dev(t), dev(lens), lse=lse)
    pick = rng.choice(np.flatnonzero(lens), 200, replace=False)
    exact = OK.decode(q[pick], pool, tables[pick], lens[pick])
    check_decode(out[dev(pick)], lse[dev(pick)], exact, torch.bfloat16, d, np.ones(200, bool))
    w = torch.zeros(far + nb, kvh, 16, device="cuda")
    kv4.accumulate_weights(w, dev(q, torch.bfloat16), lse, big, dev(t), dev(lens))
    tot = w[far:].double().sum().item()
    assert abs(tot - nh * (lens > 0).sum()) < 1e-4 * tot and not w[:far].any()
    ko = torch.zeros(nb, kvh, 16, d, dtype=torch.bfloat16, device="cuda")
    vo = torch.zeros_like(ko)
    kv4.dequantize(big, dev(t), dev(lens), dev(tables), ko, vo)
    gk, gv = OK.untile(pool)
    b = pick[0]
    blk = tables[b, 0]
    n0 = min(int(lens[b]), 16)
    np.testing.assert_array_equal(ko[blk, :, :n0].double().cpu().numpy(), gk[blk, :, :n0])
    assert not ko[blk, :, n0:].any()


# ---- prefill ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("nh,kvh,d,dtn,starts,counts", [
    (14, 2, 64, "bf16", [0], [1]),
    (14, 2, 64, "bf16", [63, 64, 127], [1, 1, 2]),
    (14, 2, 64, "bf16", [511, 0, 100], [1, 37, 130]),
    (14, 2, 64, "fp16", [15, 16, 17, 0, 5], [16, 17, 1, 0, 33]),
    (9, 3, 128, "bf16", [0, 70], [33, 20]),
    (32, 8, 128, "fp16", [250], [9]),
    (16, 1, 64, "bf16", [31], [40]),
    (12, 1, 128, "fp16", [3], [70]),
    (4, 4, 64, "fp16", [5], [300]),
    (2, 1, 128, "bf16", [0], [260]),
    (4, 1, 64, "bf16", [40, 0], [65, 64]),
    (14, 2, 64, "bf16", [5000, 2000], [3, 20]),        # cut along the keys, and joined
    (8, 1, 128, "fp16", [3000], [33]),
])
def test_prefill(kv4, nh, kvh, d, dtn, starts, counts):
    rng = np.random.default_rng(sum(counts))
    dt = DT[dtn]
    lens = np.array([s + c for s, c in zip(starts, counts)])
    tables, nb = tables_for(rng, lens)
    pool = random_pool(rng, nb, kvh, d)
    poison(pool, tables, lens, nb)
    T = sum(counts)
    q = rounded(rng.standard_normal((T, nh, d)), dt)
    plan = kv4.PrefillPlan(starts, counts)
    if max(starts) > 1500:
        assert plan.work(nh // kvh, kvh)[2] > 1
    order = rng.permutation(len(lens)).astype(np.int32)                 # rows through row_index
    shuffled = np.empty_like(tables)
    shuffled[order] = tables
    rows = torch.zeros(T, nh + 1, d, dtype=dt, device="cuda")           # strided q and out
    rows[:, :nh] = dev(q, dt)
    big = torch.full((T, nh + 2, d), 5.0, dtype=dt, device="cuda")
    out = big[:, :nh]
    kv4.prefill_attention(out, rows[:, :nh], dev(pool), dev(shuffled), plan, row_index=dev(order))
    check_prefill(out, OK.prefill(q, pool, tables, starts, counts), dt, d)
    assert (big[:, nh:] == 5).all()
    again = torch.empty(T, nh, d, dtype=dt, device="cuda")
    kv4.prefill_attention(again, dev(q, dt), dev(pool), dev(tables), plan)
    assert torch.equal(again, out)


@pytest.mark.parametrize("nh,kvh,d,dtn,starts,counts,tiles", [
    (64, 4, 64, "bf16", [0, 100] * 19 + [2100, 1600], [24, 23] * 18 + [7, 1, 24, 20], 3),
    (36, 4, 64, "fp16", [0] * 19 + [1700], [24] * 20, 2),
    (36, 4, 128, "fp16", [50] * 19 + [1700, 0], [16] * 20 + [290], 2),
    (3, 1, 128, "bf16", [0, 1700], [70, 31], 1),
])
def test_prefill_tiles_of_an_item(kv4, nh, kvh, d, dtn, starts, counts, tiles):
    assert (kv4.PrefillPlan(starts, counts).work(nh // kvh, kvh, d)[0][:, 5] == tiles).all()
    test_prefill(kv4, nh, kvh, d, dtn, starts, counts)


def check_prefill(out, exact, dt, d, rows=slice(None)):
    o, mean, flat, big = exact
    ds = (d + 8) * 2.0 ** -24 * big[..., None]
    tol = half_step(o, dt) + mean * (2.0 ** -11 + 2 * ds + 2.0 ** -20) + 2.0 ** -31 * flat
    err = np.abs(out.double().cpu().numpy() - o)
    assert (err <= tol)[rows].all(), np.nanmax((err / tol)[rows])


def test_prefill_growing_keys_and_query_magnitudes(kv4):
    """Row maxima that keep rising along the keys (O is rescaled), and rows of very different size."""
    rng = np.random.default_rng(2)
    nh, kvh, d, n = 14, 2, 64, 400
    tables, nb = tables_for(rng, [n])
    pool = kv4.new_pool(nb, kvh, d)
    pos = np.arange(n)
    k = rounded(rng.standard_normal((n, kvh, d)) * (1 + pos[:, None, None] / 8), torch.bfloat16)
    v = rounded(rng.standard_normal((n, kvh, d)), torch.bfloat16)
    kv4.append(pool, dev(k, torch.bfloat16), dev(v, torch.bfloat16),
               dev(tables[0, pos // 16].astype(np.int64) * 16 + pos % 16))
    q = rng.standard_normal((90, nh, d)) * np.exp2(rng.integers(-40, 4, (90, nh, 1)))
    q[7, 3] = 0
    q = rounded(q, torch.bfloat16)
    out = torch.empty(90, nh, d, dtype=torch.bfloat16, device="cuda")
    kv4.prefill_attention(out, dev(q, torch.bfloat16), pool, dev(tables), kv4.PrefillPlan([310], [90]))
    check_prefill(out, OK.prefill(q, pool.cpu().numpy(), tables, [310], [90]), torch.bfloat16, d)


def test_prefill_holes_and_nan(kv4):
    """Blocks that are not there are left out; a NaN reaches the rows that attend to it and no other."""
    rng = np.random.default_rng(8)
    nh, kvh, d = 4, 2, 64
    starts, counts = [100, 30, 0], [60, 50, 40]
    lens = np.array([160, 80, 40])
    tables, nb = tables_for(rng, lens)
    pool = random_pool(rng, nb, kvh, d)
    tables[0, 2], tables[0, 7], tables[1, 3] = -1, nb + 5, -1
    q = rounded(rng.standard_normal((150, nh, d)), torch.float16)
    clean = pool.copy()
    # values: token 130 of sequence 0, head 1, dims 32-47; keys: token 50 of sequence 1, head 0
    pool[tables[0, 130 // 16], 1, 16 * d + d + 2 * 16 + 130 % 16] = 0xFF
    tables[1, 3] = tables[1, 4]
    tables[1, 4] = -1
    pool[tables[1, 50 // 16], 0, 16 * d + 0 * 16 + 50 % 16] = 0xFF
    out = torch.empty(150, nh, d, dtype=torch.float16, device="cuda")
    kv4.prefill_attention(out, dev(q, torch.float16), dev(pool), dev(tables),
                          kv4.PrefillPlan(starts, counts))
    bad = torch.isnan(out).cpu().numpy()
    want = np.zeros_like(bad)
    want[30:60, 2:, 32:48] = True                   # positions 130 and on
    want[60 + 20:110, :2] = True                    # positions 50 and on
    np.testing.assert_array_equal(bad, want)
    exact = OK.prefill(q, clean, tables, starts, counts)
    o, mean, flat, big = exact
    ds = (d + 8) * 2.0 ** -24 * big[..., None]
    tol = half_step(o, torch.float16) + mean * (2.0 ** -11 + 2 * ds + 2.0 ** -20) + 2.0 ** -31 * flat
    err = np.abs(out.double().cpu().numpy() - o)
    assert (err <= tol)[~want].all()


# ---- eviction ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("d,kvh,layers,lens,keep,recent", [
    (64, 2, 3, [100, 0, 17, 64, 33], 33, 10),
    (64, 1, 1, [5], 1, 0),
    (64, 1, 1, [5], 1, 1),
    (128, 2, 2, [300, 700, 40], 256, 256),
    (128, 3, 1, [500], 499, 0),
    (64, 2, 2, [1000, 1, 16, 2000], 16, 3),
    (64, 2, 1, [3000, 2999], 1500, 100),
    (64, 1, 1, [20000], 9000, 64),
    (64, 2, 24, [130, 5, 64, 33, 200, 77, 1, 90], 50, 7),     # many units: the small CTAs
    (128, 3, 30, [40, 120, 80, 300], 64, 0),
])
@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("wide", [False, True])
def test_evict(kv4, d, kvh, layers, lens, keep, recent, kind, in_place, wide):
    """wide: a table of more than 48 * 1024 tokens, which the kernel for long sequences serves."""
    rng = np.random.default_rng(keep)
    lens = np.array(lens, np.int32)
    tables, nb = tables_for(rng, lens, spare=sum(-(-min(n, keep) // 16) for n in lens) + 3,
                            width=3100 if wide else None)
    pool = rng.integers(0, 256, (layers, nb, kvh, 18 * d), dtype=np.uint8)
    w = (rng.random((layers, nb, kvh, 16)) ** 4).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 3, w.shape).astype(np.float32)
    if kind == "odd":
        pick = rng.random(w.shape)
        w = np.where(pick < 0.3, 0.0, np.where(pick < 0.35, np.nan, np.where(
            pick < 0.4, np.inf, np.where(pick < 0.5, -0.0, w)))).astype(np.float32)
    to = tables
    if not in_place:
        free = np.setdiff1d(np.arange(nb), tables[tables >= 0])
        to, at = np.full((len(lens), max(1, -(-keep // 16))), -1, np.int32), 0
        for i, n in enumerate(lens):
            m = -(-min(int(n), keep) // 16)
            to[i, :m] = free[at:at + m]
            at += m
    rows = rng.permutation(len(lens)).astype(np.int32)
    dp, dw = dev(pool), dev(w)
    kept = torch.full((layers, len(lens), kvh, keep + 3), -7, dtype=torch.int32, device="cuda")
    kv4.evict(dp, dw, dev(tables), dev(lens[rows]), keep, recent, row_index=dev(rows), kept=kept,
              out_block_tables=None if in_place else dev(to))
    want = OK.evict(pool, w, tables, lens[rows], keep, recent, to, rows)
    kept = kept.cpu().numpy()
    for la in range(layers):
        for b in range(len(lens)):
            for h in range(kvh):
                idx = want.get((la, b, h), np.zeros(0, int))
                np.testing.assert_array_equal(kept[la, b, h, :len(idx)], idx)
                assert (kept[la, b, h, len(idx):] == -7).all()
    gp, gw = dp.cpu().numpy(), dw.cpu().numpy()
    check = np.ones((layers, nb, kvh, 16), bool)
    for b, r in enumerate(rows):                      # places behind the survivors hold anything
        n = int(lens[r])
        m = min(n, keep)
        if in_place and n > keep:
            pos = np.arange(m, n)
            check[:, tables[r, pos // 16], :, pos % 16] = False
    gw_, w_ = np.where(np.isnan(gw), -1, gw), np.where(np.isnan(w), -1, w)
    np.testing.assert_array_equal(gw_[check], w_[check])
    gc = gp[..., :16 * d].reshape(layers, nb, kvh, 2, 16, d // 2)
    wc = pool[..., :16 * d].reshape(layers, nb, kvh, 2, 16, d // 2)
    gs = gp[..., 16 * d:].reshape(layers, nb, kvh, d // 8, 16)
    ws = pool[..., 16 * d:].reshape(layers, nb, kvh, d // 8, 16)
    np.testing.assert_array_equal(np.moveaxis(gc, 4, 3)[check], np.moveaxis(wc, 4, 3)[check])
    np.testing.assert_array_equal(np.moveaxis(gs, 4, 3)[check], np.moveaxis(ws, 4, 3)[check])


# ---- together -------------------------------------------------------------------------------------------
def test_run_together_and_in_graphs(kv4):
    """Append, attend, add up, evict, attend again, as a decode loop does; the attention also
    from two captured graphs that replay at the same time on two streams."""
    rng = np.random.default_rng(12)
    nh, kvh, d, B, dt = 14, 2, 64, 3, torch.bfloat16
    lens = np.array([130, 60, 200], np.int32)
    tables, nb = tables_for(rng, lens + 8)
    pool, w = np.zeros((nb, kvh, 18 * d), np.uint8), np.zeros((nb, kvh, 16), np.float32)
    dp, dw, dtab = dev(pool), dev(w), dev(tables)
    for b in range(B):
        pos = np.arange(lens[b])
        slots = tables[b, pos // 16].astype(np.int64) * 16 + pos % 16
        k, v = (rounded(rng.standard_normal((lens[b], kvh, d)), dt) for _ in range(2))
        kv4.append(dp, dev(k, dt), dev(v, dt), dev(slots), weights=dw)
        OK.put(pool, k, v, slots)
    keep, recent = 96, 16
    for step in range(6):
        slots = tables[np.arange(B), lens // 16].astype(np.int64) * 16 + lens % 16
        k, v = (rounded(rng.standard_normal((B, kvh, d)), dt) for _ in range(2))
        q = rounded(2 * rng.standard_normal((B, nh, d)), dt)
        kv4.append(dp, dev(k, dt), dev(v, dt), dev(slots), weights=dw)
        OK.put(pool, k, v, slots)
        lens += 1
        out, lse = torch.empty(B, nh, d, dtype=dt, device="cuda"), torch.empty(B, nh, device="cuda")
        kv4.decode_attention(out, dev(q, dt), dp, dtab, dev(lens), lse=lse)
        check_decode(out, lse, OK.decode(q, pool, tables, lens), dt, d, np.ones(B, bool))
        kv4.accumulate_weights(dw, dev(q, dt), lse, dp, dtab, dev(lens))
        w = dw.cpu().numpy()                       # the oracle's ranks use the kernel's totals
        if step in (1, 4):
            kv4.evict(dp[None], dw[None], dtab, dev(lens), keep, recent)
            OK.evict(pool[None], w[None], tables, lens, keep, recent)
            lens = np.minimum(lens, keep).astype(np.int32)
    qs = [dev(rounded(rng.standard_normal((B, nh, d)), dt), dt) for _ in range(2)]
    outs = [torch.zeros(B, nh, d, dtype=dt, device="cuda") for _ in range(2)]
    dl = dev(lens)
    plain = []
    for x in qs:
        o = torch.empty_like(x)
        kv4.decode_attention(o, x, dp, dtab, dl)
        plain.append(o)
    graphs = []
    torch.cuda.synchronize()
    for x, o in zip(qs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv4.decode_attention(o, x, dp, dtab, dl)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, p in zip(outs, plain):
            assert torch.equal(o, p)
            o.zero_()
        torch.cuda.synchronize()


@pytest.mark.parametrize("d", [64, 128])
def test_prefill_captured_and_side_by_side(kv4, d):
    """Long prefixes cut into ranges (two launches): captured and replayed, and two calls at once
    on streams of their own, give the eager result bit for bit."""
    nh, kvh, starts, counts = 14, 2, [5000, 0, 9000], [40, 3, 130]
    blocks = [-(-(s + c) // 16) for s, c in zip(starts, counts)]
    rng = np.random.default_rng(8)
    pool = kv4.new_pool(sum(blocks), kvh, d)
    pool.copy_(torch.from_numpy(rng.integers(0, 80, tuple(pool.shape), dtype=np.uint8)))
    tab = torch.full((3, max(blocks)), -1, dtype=torch.int32)
    for i, n in enumerate(blocks):
        tab[i, :n] = torch.arange(n) + sum(blocks[:i])
    tab = tab.cuda()
    plan, late = kv4.PrefillPlan(starts, counts), kv4.PrefillPlan(starts, counts)
    assert plan.work(nh // kvh, kvh)[2] > 1
    qs = [torch.from_numpy(rng.standard_normal((sum(counts), nh, d))).to("cuda", torch.bfloat16)
          for _ in range(2)]
    want, outs, graphs = [], [torch.zeros_like(q) for q in qs], []
    for q in qs:
        o = torch.zeros_like(q)
        kv4.prefill_attention(o, q, pool, tab, plan)
        want.append(o)
    torch.cuda.synchronize()
    assert not want[0].isnan().any()
    for q, o in zip(qs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            with pytest.raises(RuntimeError, match="before the capture"):
                kv4.prefill_attention(o, q, pool, tab, late)
            kv4.prefill_attention(o, q, pool, tab, plan)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for captured in (True, False):
        for _ in range(5):
            for s, g, q, o in zip(streams, graphs, qs, outs):
                with torch.cuda.stream(s):
                    if captured:
                        g.replay()
                    else:
                        kv4.prefill_attention(o, q, pool, tab, plan)
            torch.cuda.synchronize()
            for o, w in zip(outs, want):
                assert torch.equal(o, w)
                o.zero_()
            torch.cuda.synchronize()


def test_rows_that_overlap_are_refused(kv4):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")             # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")             # noqa: E731
    pool, same = kv4.new_pool(4, 2, 64), z(1, 4, 64).expand(3, 4, 64)
    slots = torch.arange(3, device="cuda")
    tables = torch.zeros(8, 32, dtype=torch.float32, device="cuda")
    for f in (lambda: kv4.decode_attention(same, z(3, 4, 64), pool, i32(3, 3), i32(3)),
              lambda: kv4.prefill_attention(same, z(3, 4, 64), pool, i32(1, 3), kv4.PrefillPlan([0], [3])),
              lambda: kv4.rope_append(pool, z(1, 8 * 64).expand(3, 8 * 64), 4, slots, tables, tables, i32(3))):
        with pytest.raises(RuntimeError, match="overlap"):
            f()
    with pytest.raises(RuntimeError, match="shape"):
        kv4.decode_attention(z(3, 256), z(3, 4, 64), pool, i32(3, 3), i32(3))
    # a query that all rows share is read, not written
    out = z(3, 4, 64)
    kv4.decode_attention(out, same, pool, i32(3, 3), i32(3) + 5)
    torch.cuda.synchronize()
    assert torch.equal(out, z(3, 4, 64))


def test_refusals(kv4):
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")      # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")             # noqa: E731
    pool, k, slots = kv4.new_pool(4, 2, 64), z(3, 2, 64), torch.arange(3, device="cuda")
    bad = [
        lambda: kv4.append(pool, z(3, 2, 128), z(3, 2, 128), slots),
        lambda: kv4.append(pool, z(3, 1, 64), z(3, 1, 64), slots),
        lambda: kv4.append(pool, k.float(), k.float(), slots),
        lambda: kv4.append(pool, k, k.half(), slots),
        lambda: kv4.append(pool, k, k, slots.int()),
        lambda: kv4.append(pool, k, k, slots[:2]),
        lambda: kv4.append(pool, k.transpose(1, 2).contiguous().transpose(1, 2), k, slots),
        lambda: kv4.append(pool[:, :1], z(3, 1, 64), z(3, 1, 64), slots),
        lambda: kv4.append(pool, k, k, slots, weights=z(4, 2, 16)),
        lambda: kv4.append(pool.float(), k, k, slots),
        lambda: kv4.decode_attention(z(2, 5, 64), z(2, 5, 64), pool, i32(2, 3), i32(2)),
        lambda: kv4.decode_attention(z(2, 34, 64), z(2, 34, 64), pool, i32(2, 3), i32(2)),
        lambda: kv4.decode_attention(z(2, 4, 64), z(2, 4, 128), pool, i32(2, 3), i32(2)),
        lambda: kv4.decode_attention(z(2, 4, 64), z(2, 4, 64).half(), pool, i32(2, 3), i32(2)),
        lambda: kv4.decode_attention(z(2, 4, 64), z(2, 4, 64), pool, i32(1, 3), i32(2)),
        lambda: kv4.decode_attention(z(2, 4, 64), z(2, 4, 64), pool, i32(2, 3), i32(3)),
        lambda: kv4.decode_attention(z(2, 4, 64), z(2, 4, 64), pool, i32(2, 3), i32(2).long()),
        lambda: kv4.decode_attention(z(2, 4, 64), z(2, 4, 64), pool, i32(2, 3), i32(2), lse=z(2, 4)),
        lambda: kv4.decode_attention(z(2, 64, 4).transpose(1, 2), z(2, 4, 64), pool, i32(2, 3), i32(2)),
        lambda: kv4.decode_attention(z(2, 4, 65)[..., :64], z(2, 4, 64), pool, i32(2, 3), i32(2)),
        lambda: kv4.decode_attention(z(5000, 4, 64), z(5000, 4, 64), pool, i32(5000, 3), i32(5000)),
        lambda: kv4.decode_attention(z(2, 4, 64), z(2, 4, 64), pool, i32(2, 0), i32(2)),
        lambda: kv4.accumulate_weights(z(4, 2, 16), z(2, 4, 64), z(2, 4, dt=torch.float32), pool, i32(2, 3), i32(2)),
        lambda: kv4.accumulate_weights(z(4, 2, 16, dt=torch.float32), z(2, 4, 64), z(2, 4), pool, i32(2, 3), i32(2)),
        lambda: kv4.evict(pool, z(4, 2, 16, dt=torch.float32), i32(1, 2), i32(1), 0, 0),
        lambda: kv4.evict(pool, z(4, 2, 16, dt=torch.float32), i32(1, 2), i32(1), 4, 5),
        lambda: kv4.evict(pool, z(3, 2, 16, dt=torch.float32), i32(1, 2), i32(1), 4, 2),
        lambda: kv4.evict(pool, z(4, 2, 16, dt=torch.float32), i32(1, 2), i32(1), 4, 2, kept=i32(1, 1, 2, 3)),
        lambda: kv4.dequantize(pool, i32(1, 2), i32(1), i32(1, 3), z(4, 2, 16, 64), z(4, 2, 16, 64)),
        lambda: kv4.dequantize(pool, i32(1, 2), i32(1), i32(1, 2), z(4, 2, 16, 128), z(4, 2, 16, 128)),
        lambda: kv4.prefill_attention(z(2, 4, 64), z(2, 4, 64), pool, i32(1, 3), kv4.PrefillPlan([0], [3])),
        lambda: kv4.prefill_attention(z(3, 4, 64), z(3, 4, 64), pool, i32(1, 3), kv4.PrefillPlan([100], [3])),
        lambda: kv4.decode_attention(z(2, 4, 64), z(2, 4, 64), pool.cpu(), i32(2, 3), i32(2)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was not refused")
    # nothing to do is not an error
    kv4.append(pool, z(0, 2, 64), z(0, 2, 64), slots[:0])
    kv4.decode_attention(z(0, 4, 64), z(0, 4, 64), pool, i32(0, 3), i32(0))
    kv4.prefill_attention(z(0, 4, 64), z(0, 4, 64), pool, i32(0, 3), kv4.PrefillPlan([], []))
