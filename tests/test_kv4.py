"""The 4-bit KV cache on the CPU: the oracle's format against a search over all its values, the
prefill plan's layout, and the C ABI's refusals (checked before any CUDA call)."""
import os

import numpy as np
import pytest
import torch

from oracle import kv4 as OK


@pytest.fixture(scope="module")
def native():
    from tiny_infra_b200 import _native
    if not os.path.exists(_native.LIB_PATH):
        from tiny_infra_b200 import build
        build.build()
    return _native


def test_format_is_exact_in_16_bits():
    """Every code times every finite scale is a bf16 and an fp16 number."""
    codes, scales = np.arange(16, dtype=np.uint8), np.arange(0xA8 + 1, dtype=np.uint8)
    assert OK.scale_values(scales[-1:])[0] >= 8.0
    sb = np.arange(256, dtype=np.uint8)
    sb = sb[OK.scale_values(sb) <= 10240.0]
    v = OK.values(np.tile(codes, len(sb)).reshape(len(sb), 16), sb[:, None])
    t = torch.from_numpy(v)
    for dt in (torch.bfloat16, torch.float16):
        assert torch.equal(t.to(dt).double(), t)


def test_quantize_takes_the_nearest_value():
    """Scale: amax / 6 to 4 significant bits; code: no magnitude is nearer, ties to the even code."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((500, 64)) * np.exp2(rng.integers(-20, 15, (500, 1)))
    x[7], x[8, :16], x[9, 3] = 0.0, 65504.0, np.nan
    x = torch.from_numpy(x).to(torch.float16).double().numpy()
    code, sb = OK.quantize(x)
    s = OK.scale_values(sb)
    assert (sb[9, 0] == 0xFF) and not np.isfinite(s[9, 0])
    ok = np.isfinite(s)
    a = np.abs(np.where(np.isnan(x), 0, x).reshape(500, 4, 16)).max(-1) / 6
    lim = np.minimum(a, 10240)
    assert (np.abs(s - lim) <= np.maximum(lim * 2.0 ** -4, 2.0 ** -18))[ok].all()
    v = OK.values(code, sb).reshape(500, 4, 16)
    g = x.reshape(500, 4, 16)
    dist = np.abs(np.abs(g)[..., None] - OK.MAGNITUDES * s[..., None, None])
    got = np.abs(np.abs(g) - np.abs(v))
    live = ok & (s > 0)
    assert (got[live] == dist[live].min(-1)).all()
    tie = (dist[live] == dist[live].min(-1, keepdims=True)).sum(-1) > 1
    assert tie.any() and (code.reshape(500, 4, 16)[live][tie] % 2 == 0).all()


def test_survivors_rule():
    w = np.array([1.0, 5.0, 5.0, np.nan, 0.0, 5.0, 9.0, 2.0], np.float32)
    np.testing.assert_array_equal(OK.survivors(w, 4, 2), [1, 3, 6, 7])
    np.testing.assert_array_equal(OK.survivors(w, 5, 2), [1, 2, 3, 6, 7])
    np.testing.assert_array_equal(OK.survivors(w, 8, 0), np.arange(8))
    np.testing.assert_array_equal(OK.survivors(w, 3, 3), [5, 6, 7])
    np.testing.assert_array_equal(OK.survivors(w, 1, 0), [3])


def test_prefill_plan_layout():
    from tiny_infra_b200.kv4 import PrefillPlan
    p = PrefillPlan([0, 511, 100, 7], [1, 33, 130, 0], device="cpu")
    assert (p.num_seqs, p.num_tokens, p.max_blocks) == (4, 164, 34)
    assert p.start_pos.tolist() == [0, 511, 100, 7]
    assert p.cu_seqlens.tolist() == [0, 1, 34, 164, 164]
    assert PrefillPlan([], [], device="cpu").work(7, 2)[2] == 0
    rng = np.random.default_rng(0)
    for group in (1, 2, 3, 7, 8, 12, 16):
        for d, most in ((64, 3), (128, 2)) * 10:
            n = int(rng.integers(1, 5))
            starts, counts = rng.integers(0, 40000, n), rng.integers(0, 900, n)
            starts[0] *= int(rng.integers(0, 2))
            items, merges, parts = PrefillPlan(starts, counts, device="cpu").work(group, 2, d)
            if not len(items):
                assert counts.sum() == 0
                continue
            tiles = int(items[0, 5])
            assert 1 <= tiles <= most and (items[:, 5] == tiles).all() and (merges[:, 4] == tiles).all()
            pair = tiles * (128 >> (group - 1).bit_length())
            length = items[:, 3] - items[:, 2]
            assert (length > 0).all() and (np.diff(length) <= 0).all() and (items[:, 2] % 64 == 0).all()
            joined = {(s, q): (f, k) for s, q, f, k, _ in merges.tolist()}
            seen = []
            for i in range(n):
                for q0 in range(0, int(counts[i]), pair):
                    keys = int(starts[i] + min(q0 + pair, counts[i]))
                    mine = sorted(items[(items[:, 0] == i) & (items[:, 1] == q0)].tolist(),
                                  key=lambda r: r[2])
                    ends = [0] + [r[3] for r in mine]                # the ranges cover the keys once
                    assert [r[2] for r in mine] == ends[:-1] and ends[-1] == keys
                    got = [r[4] for r in mine]
                    if len(mine) == 1:
                        assert got == [-1] and (i, q0) not in joined
                    else:
                        f, k = joined[i, q0]
                        assert got == list(range(f, f + k)) and k == len(mine)
                        seen += got
            assert sorted(seen) == list(range(parts))
            assert len(items) == len(seen) + sum(-(-int(c) // pair) for c in counts) - len(merges)
    for bad in (([0], [1, 2]), ([-1], [3]), ([0], [-3])):
        with pytest.raises(RuntimeError):
            PrefillPlan(*bad, device="cpu")


def test_module_refuses_host_tensors():
    from tiny_infra_b200 import kv4
    z = torch.zeros(4, 2, 18 * 64, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        kv4.append(z, torch.zeros(1, 2, 64).bfloat16(), torch.zeros(1, 2, 64).bfloat16(),
                   torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="head_dim"):
        kv4.tile_bytes(96)
    assert kv4.tile_bytes(64) == 1152 and kv4.tile_bytes(128) == 2304


FAKE = 1 << 20          # a 16-byte aligned address that is never dereferenced


def test_c_abi_refusals(native):
    lib = native.lib()

    def refused(rc, code, text):
        assert rc == code and text in lib.ti_last_error(), (rc, lib.ti_last_error())

    def append(pool=FAKE, k=FAKE, stride=128, n=4, nb=8, kvh=2, d=64, bs=16, dt=0):
        return lib.ti_kv4_append(pool, None, k, stride, 64, FAKE, 128, 64, FAKE, n, nb, kvh, d, bs,
                                 dt, None)
    assert append(n=0) == 0
    refused(append(pool=None), 1, b"null")
    refused(append(n=-1), 1, b"negative")
    refused(append(nb=0), 1, b"empty pool")
    refused(append(d=96), 2, b"head_dim")
    refused(append(bs=32), 2, b"block_size")
    refused(append(dt=2), 2, b"dtype")
    refused(append(stride=132), 1, b"aligned")
    refused(append(k=FAKE + 2), 1, b"aligned")

    def deq(out=FAKE, rows=2, mb=3, nb=8, ob=8, d=64, bs=16, dt=0):
        return lib.ti_kv4_dequantize(out, FAKE, ob, FAKE, nb, FAKE, 3, None, FAKE, FAKE, 3, rows,
                                     mb, 2, d, bs, dt, None)
    assert deq(rows=0) == 0
    refused(deq(out=None), 1, b"null")
    refused(deq(rows=-1), 1, b"negative")
    refused(deq(ob=0), 1, b"empty pool")
    refused(deq(d=80), 2, b"head_dim")
    refused(deq(dt=2), 2, b"dtype")
    refused(deq(out=FAKE + 8), 1, b"aligned")

    def att(out=FAKE, q=FAKE, qs=14 * 64, b=2, nh=14, kvh=2, d=64, bs=16, mb=4, nb=8, dt=0):
        need = lib.ti_kv4_attention_workspace_bytes(max(b, 1), nh, max(kvh, 1), d, max(mb, 1))
        return lib.ti_kv4_attention_decode(out, 14 * 64, None, q, qs, FAKE, nb, FAKE, 4, None,
                                           FAKE, b, nh, kvh, d, bs, mb, dt, FAKE, need, None)
    assert att(b=0) == 0
    refused(att(out=None), 1, b"null")
    refused(att(b=-1), 1, b"batch")
    refused(att(nh=15), 1, b"multiple")
    refused(att(kvh=0), 1, b"head counts")
    refused(att(nh=34), 2, b"16 query heads")
    refused(att(d=32), 2, b"head_dim")
    refused(att(bs=8), 2, b"block_size")
    refused(att(dt=2), 2, b"dtype")
    refused(att(b=5000), 2, b"4096")
    refused(att(qs=14 * 64 + 4), 1, b"aligned")
    refused(att(q=FAKE + 4), 1, b"aligned")

    def acc(w=FAKE, b=2, nh=14, d=64, q=FAKE):
        return lib.ti_kv4_accumulate_weights(FAKE, w, q, 14 * 64, FAKE, FAKE, 8, FAKE, 4, None,
                                             FAKE, b, nh, 2, d, 16, 4, 0, None)
    assert acc(b=0) == 0
    refused(acc(w=None), 1, b"null")
    refused(acc(nh=13), 1, b"multiple")
    refused(acc(d=256), 2, b"head_dim")
    refused(acc(q=FAKE + 4), 1, b"aligned")

    assert lib.ti_kv4_prefill_workspace_bytes(3, 2, 64) == 3 * 2 * 3 * 128 * 66 * 4
    assert lib.ti_kv4_prefill_workspace_bytes(3, 2, 128) == 3 * 2 * 2 * 128 * 130 * 4
    assert lib.ti_kv4_prefill_workspace_bytes(0, 2, 64) == 0

    def pre(out=FAKE, items=FAKE, n=2, merges=None, nm=0, parts=0, nh=14, d=64, bs=16, dt=0, mb=4,
            ws=None, wb=0, qs=14 * 64):
        return lib.ti_kv4_prefill_attention(out, 14 * 64, FAKE, qs, FAKE, 8, FAKE, 4, mb, None, FAKE,
                                            FAKE, items, n, merges, nm, parts, nh, 2, d, bs, dt, ws,
                                            wb, None)
    assert pre(n=0) == 0
    refused(pre(out=None), 1, b"null")
    refused(pre(items=None), 1, b"null")
    refused(pre(nm=1), 1, b"null")
    refused(pre(parts=2), 1, b"null")
    refused(pre(n=-1), 1, b"negative")
    refused(pre(mb=0), 1, b"table width")
    refused(pre(nh=15), 1, b"multiple")
    refused(pre(nh=34), 2, b"16 query heads")
    refused(pre(d=96), 2, b"head_dim")
    refused(pre(bs=8), 2, b"block_size")
    refused(pre(dt=2), 2, b"dtype")
    refused(pre(qs=14 * 64 + 4), 1, b"aligned")
    refused(pre(parts=2, ws=FAKE, wb=100), 4, b"workspace")

    def ev(pool=FAKE, layers=1, b=2, keep=4, recent=2, kept=None, ks=0, d=64, bs=16):
        return lib.ti_kv4_evict(pool, FAKE, layers, 8, FAKE, 4, FAKE, 4, None, FAKE, b, 4, 4, keep,
                                recent, kept, ks, 2, d, bs, None)
    assert ev(b=0) == 0 and ev(layers=0) == 0
    refused(ev(pool=None), 1, b"null")
    refused(ev(keep=0, recent=0), 1, b"keep")
    refused(ev(recent=5), 1, b"recent")
    refused(ev(recent=-1), 1, b"recent")
    refused(ev(kept=FAKE, ks=3), 1, b"kept")
    refused(ev(d=32), 2, b"head_dim")
    refused(ev(bs=32), 2, b"block_size")
    refused(ev(pool=FAKE + 8), 1, b"aligned")
    refused(ev(layers=70000), 2, b"65535")

    def rope(qkv=FAKE, stride=18 * 64, n=4, nb=8, d=64, bs=16, dt=0, nh=14, rows=32):
        return lib.ti_rope_kv4_append(qkv, stride, FAKE, None, FAKE, FAKE, FAKE, rows, FAKE, n, nb,
                                      nh, 2, d, bs, dt, None)
    assert rope(n=0) == 0
    refused(rope(qkv=None), 1, b"null")
    refused(rope(nh=0), 1, b"negative size")
    refused(rope(rows=-1), 1, b"negative size")
    refused(rope(d=32), 2, b"head_dim")
    refused(rope(dt=2), 2, b"dtype")
    refused(rope(stride=18 * 64 + 4), 1, b"aligned")


def test_allocator_truncate():
    from tiny_infra_b200.cache_manager import BlockAllocator
    a = BlockAllocator(2, 128, 16, 12)
    a.plan_tokens([0, 1], [100, 40])
    a.advance([0, 1], [100, 40])
    row = a.block_tables[0].copy()
    free = list(a.free_blocks)
    a.truncate(0, 33)
    assert (a.seq_len[0], a.pos_offset[0]) == (33, 67)
    np.testing.assert_array_equal(a.block_tables[0, :3], row[:3])
    assert (a.block_tables[0, 3:] == -1).all()
    assert list(a.free_blocks) == free + row[3:7].tolist()        # in logical order, at the back
    a.plan_tokens([0], [20])
    a.advance([0], [20])
    a.truncate(0, 48)
    assert (a.seq_len[0], a.pos_offset[0]) == (48, 72)
    a.truncate(0, 48)                                             # nothing to do
    assert (a.seq_len[0], a.pos_offset[0]) == (48, 72)
    for bad in (-1, 49):
        with pytest.raises(ValueError):
            a.truncate(0, bad)
    a.truncate(0, 0)
    assert (a.block_tables[0] == -1).all() and a.seq_len[0] == 0
    a.free_slot(0)
    a.free_slot(1)
    assert a.pos_offset[0] == 0 and sorted(a.free_blocks) == list(range(12))


def test_cache_manager_refusals():
    from tiny_infra_b200.cache_manager import KVCacheManager
    for kw in (dict(kv_bits=8), dict(track_weights=True), dict(kv_bits=4, block_size=32),
               dict(max_positions=100)):
        with pytest.raises(RuntimeError):
            KVCacheManager(2, 128, 1, 2, 64, **kw)
    with pytest.raises(RuntimeError):
        KVCacheManager(2, 128, 1, 2, 96, kv_bits=4)


def test_scheduler_evicts_before_decode():
    """Sequences at evict_above tokens are brought down before the step, and only those."""
    import asyncio

    from tests.test_scheduler_trace import _HostKV, _StandInBackend
    from tiny_infra_b200.scheduler import ContinuousBatcher, GenerationRequest
    kv = _HostKV(dict(max_batch_size=3, max_seq_len=32, block_size=16, head_dim=64))
    calls = []
    kv.seq_len_host = lambda s: int(kv.alloc.seq_len[s])

    def evict(slots, keep, recent):
        calls.append((list(slots), [kv.seq_len_host(s) for s in slots], keep, recent))
        for s in slots:
            kv.alloc.truncate(s, keep)
    kv.evict = evict
    sched = ContinuousBatcher(None, kv, backend=_StandInBackend(kv, 1000), evict_above=20,
                              evict_keep=12, evict_recent=5)

    async def run():
        for n, m in ((18, 30), (5, 9), (19, 2)):
            sched.requests_queue.put_nowait(GenerationRequest(list(range(n)), m, 0.0))
        sched._fill_active_slots()
        reqs = list(sched.active_slots)
        while sched._has_active_requests():
            sched._step_generation()
        return reqs
    reqs = asyncio.run(run())
    assert [len(r.generated_tokens) for r in reqs] == [30, 9, 2]
    assert all(r.error is None for r in reqs)
    # slot 0 reaches 20 after two steps and then again every 8 tokens
    assert [c[:2] for c in calls] == [([0], [20])] * len(calls)
    assert len(calls) == 1 + (29 - 2 - 1) // 8 and all(c[2:] == (12, 5) for c in calls)
    assert sched.stats()["evictions"] == len(calls)
    assert sorted(kv.alloc.free_blocks) == list(range(6))
    for kw in (dict(evict_keep=3), dict(evict_above=20, evict_keep=20),
               dict(evict_above=20, evict_keep=4, evict_recent=5), dict(evict_above=33)):
        with pytest.raises(ValueError):
            ContinuousBatcher(None, kv, backend=object(), **kw)
