"""The 4-bit KV cache's calls on the CPU: what a call hands to the C entry point (a stand-in library
records it), and the host logic of the cache manager and the batcher around them."""
import contextlib

import pytest
import torch


class _Recorder:
    """In the library's place: every entry point notes its arguments as C sees them, and succeeds."""

    def __init__(self, signatures):
        self.signatures, self.calls = signatures, []

    def __getattr__(self, name):
        def entry(*args):
            kinds = self.signatures[name][1]
            assert len(args) == len(kinds), name
            self.calls.append((name, [k(a).value for k, a in zip(kinds, args)]))
            return 0
        return entry


@pytest.fixture
def recorded(monkeypatch):
    """``tiny_infra_b200.kv4`` taking host tensors, its calls recorded."""
    from tiny_infra_b200 import _native, kv4
    rec = _Recorder(_native.SIGNATURES)
    monkeypatch.setattr(_native, "lib", lambda: rec)
    monkeypatch.setattr(kv4, "_device", lambda *t: 0)
    monkeypatch.setattr(kv4, "_on", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(kv4, "_stream", lambda dev: 0)
    return kv4, rec


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_dequantize_takes_the_pool_of_all_layers(recorded):
    """[layers, num_blocks, ...] is one pool of layers * num_blocks blocks, as evict leaves it."""
    kv4, rec = recorded
    out = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    for pool, blocks in ((torch.zeros(5, 2, 18 * 64, dtype=torch.uint8), 5),
                         (torch.zeros(3, 5, 2, 18 * 64, dtype=torch.uint8), 15)):
        kv4.dequantize(pool, _i32(2, 3), _i32(2), _i32(2, 3), out, out.clone())
        name, args = rec.calls.pop()
        assert name == "ti_kv4_dequantize" and args[3:5] == [pool.data_ptr(), blocks]
    with pytest.raises(RuntimeError, match="pool"):
        kv4.dequantize(torch.zeros(1, 3, 5, 2, 18 * 64, dtype=torch.uint8), _i32(2, 3), _i32(2),
                       _i32(2, 3), out, out.clone())
    assert not rec.calls


def _host_cache(**kw):
    """The scheduler's view of a cache (tests/test_scheduler_trace.py), with attributes of its own."""
    from tests.test_scheduler_trace import _HostKV
    kv = _HostKV(dict(max_batch_size=3, max_seq_len=32, block_size=16, head_dim=64))
    for name, value in kw.items():
        setattr(kv, name, value)
    return kv


def test_batcher_refuses_eviction_without_totals():
    """A cache that keeps no attention-weight totals (16-bit, or without track_weights) cannot evict:
    said when the batcher is made, not in the middle of its requests."""
    from tiny_infra_b200.scheduler import ContinuousBatcher
    with pytest.raises(ValueError, match="track_weights"):
        ContinuousBatcher(None, _host_cache(attn_weights=None), backend=object(), evict_above=20)
    for kv, kw in ((_host_cache(attn_weights=object()), dict(evict_above=20)),
                   (_host_cache(attn_weights=None), {})):
        ContinuousBatcher(None, kv, backend=object(), **kw)


def _manager(**kw):
    """A KVCacheManager's host logic without its device pool."""
    from tiny_infra_b200.cache_manager import BlockAllocator, KVCacheManager
    kv = KVCacheManager.__new__(KVCacheManager)
    kv.max_batch_size, kv.max_seq_len, kv.max_positions = 3, 32, 32
    kv.block_size, kv.head_dim, kv.device = 16, 64, torch.device("cpu")
    kv.alloc = BlockAllocator(3, 32, 16)
    kv.total_physical_blocks, kv.max_blocks_per_seq = 6, 2
    kv._seq_host, kv._bt_host, kv._evicted = kv.alloc.seq_len, kv.alloc.block_tables, False
    kv.block_tables = torch.full((3, 2), -1, dtype=torch.int32)
    kv.seq_len, kv.pos_offset = _i32(3), _i32(3)
    kv.kv4_pool = kv.attn_weights = object()
    for name, value in kw.items():
        setattr(kv, name, value)
    return kv


def test_one_sequence_at_its_last_position_ends_alone():
    """A sequence that has used up the cache's positions ends with its own error; the others go on."""
    import asyncio

    from tests.test_scheduler_trace import _StandInBackend
    from tiny_infra_b200.scheduler import ContinuousBatcher, GenerationRequest
    kv = _manager(max_positions=40)

    def evict(slots, keep, recent):              # the device part is the GPU tests'
        for s in slots:
            kv.alloc.truncate(s, keep)
        kv._evicted = True
    kv.evict = evict
    kv.free_batch_slot = kv.alloc.free_slot

    class Backend(_StandInBackend):
        def decode(self, slots, reqs):
            kv._check_positions(slots, 1)        # as KVCacheManager.plan_decode does
            return super().decode(slots, reqs)
    sched = ContinuousBatcher(None, kv, backend=Backend(kv, 1000), evict_above=20, evict_keep=12)

    async def run():
        for n, m in ((18, 60), (5, 9), (3, 30)):
            sched.requests_queue.put_nowait(GenerationRequest(list(range(n)), m, 0.0))
        sched._fill_active_slots()
        reqs = list(sched.active_slots)
        while sched._has_active_requests():
            sched._step_generation()
        return reqs
    reqs = asyncio.run(run())
    # positions 18 .. 39 are decoded: the token of the prefill and 22 more
    assert [len(r.generated_tokens) for r in reqs] == [23, 9, 30]
    assert isinstance(reqs[0].error, ValueError) and "Position" in str(reqs[0].error)
    assert reqs[1].error is None and reqs[2].error is None
    assert sched.stats()["requests_failed"] == 1 and sched.stats()["requests_finished"] == 2
    assert sorted(kv.alloc.free_blocks) == list(range(6))


@pytest.mark.parametrize("lens,cols", [((32, 0, 20), 2), ((9, 16, 5), 1)])
def test_manager_evicts_through_the_columns_in_use(monkeypatch, lens, cols):
    """The table that the kernel gets is as wide as the longest sequence that shrinks, whatever the
    cache's max_seq_len: its shared memory and its choice of a kernel go by that width."""
    from tiny_infra_b200 import kv4
    kv = _manager()
    kv.alloc.plan_tokens([0, 1, 2], lens)
    kv.alloc.advance([0, 1, 2], lens)
    kv.block_tables.copy_(torch.from_numpy(kv._bt_host))
    kv.seq_len.copy_(torch.from_numpy(kv._seq_host))
    seen = []
    monkeypatch.setattr(kv4, "evict", lambda pool, weights, tables, ctx, keep, recent, row_index: seen.append(
        (tables.clone(), tables.data_ptr(), ctx.tolist(), keep, recent, row_index.tolist())))
    before = kv.block_tables.clone()
    assert kv.evict([0, 1, 2], 8, 3) == [s for s in range(3) if lens[s] > 8]
    (tables, ptr, ctx, keep, recent, rows), = seen
    assert ptr == kv.block_tables.data_ptr() and torch.equal(tables, before[:, :cols])
    assert ctx == [lens[s] for s in rows] and (keep, recent) == (8, 3)
    assert kv._seq_host.tolist() == [min(n, 8) for n in lens] == kv.seq_len.tolist()
    assert torch.equal(kv.block_tables, torch.from_numpy(kv._bt_host))


def test_evict_sizes_beyond_32_bits(recorded):
    """keep and recent reach C as 32-bit numbers: larger ones mean that nothing is evicted, as any
    keep beyond the lengths does, not a small one."""
    kv4, rec = recorded
    pool, w = torch.zeros(5, 2, 18 * 64, dtype=torch.uint8), torch.zeros(5, 2, 16)
    for keep, recent, want in ((7, 3, [7, 3]), (2 ** 31 - 1, 0, [2 ** 31 - 1, 0]),
                               (2 ** 31, 2 ** 31, [2 ** 31 - 1] * 2),
                               (2 ** 32 + 5, 2, [2 ** 31 - 1, 2]),
                               (2 ** 40, 2 ** 33 + 1, [2 ** 31 - 1] * 2)):
        kv4.evict(pool, w, _i32(2, 3), _i32(2), keep, recent)
        name, args = rec.calls.pop()
        assert name == "ti_kv4_evict" and args[13:15] == want
    for keep, recent in ((0, 0), (2 ** 32, 2 ** 32 + 1), (4, -1)):
        with pytest.raises(RuntimeError, match="keep"):
            kv4.evict(pool, w, _i32(2, 3), _i32(2), keep, recent)
    with pytest.raises(RuntimeError, match="kept"):
        kv4.evict(pool, w, _i32(2, 3), _i32(2), 2 ** 32 + 5, 2, kept=_i32(1, 2, 2, 5))


def test_plan_is_held_for_the_streams_that_use_it(recorded, monkeypatch):
    """A plan's device tensors are its own: a call on another stream than theirs tells the allocator,
    once, so that a plan dropped behind the call does not give their memory away under it."""
    kv4, rec = recorded
    held, here = [], [0]
    monkeypatch.setattr(kv4, "_stream", lambda dev: here[0])
    monkeypatch.setattr(kv4.PrefillPlan, "_home", lambda plan: here[0], raising=False)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: held.append((t.data_ptr(), s)))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: f"stream {here[0]}")
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: capturing[0])
    capturing = [False]
    plan = kv4.PrefillPlan([0, 5000], [3, 2], device="cpu")
    q = {kvh: torch.zeros(5, 4, 64, dtype=torch.bfloat16) for kvh in (1, 2)}
    pools = {kvh: torch.zeros(3, kvh, 18 * 64, dtype=torch.uint8) for kvh in (1, 2)}

    def call(kvh, stream):
        here[0] = stream
        kv4.prefill_attention(torch.empty_like(q[kvh]), q[kvh], pools[kvh], _i32(2, 400), plan)
        out, held[:] = sorted(held), []
        return out
    base = plan.start_pos.data_ptr()
    assert call(2, 0) == []                      # the stream that made it
    first = plan._layouts[2, 2, 64][0].data_ptr()
    assert call(2, 7) == sorted([(base, "stream 7"), (first, "stream 7")])
    assert call(2, 7) == []
    assert call(1, 9) == sorted([(base, "stream 9"), (first, "stream 9")])     # a layout of 9's own
    second = plan._layouts[4, 1, 64][0].data_ptr()
    assert call(1, 7) == [(second, "stream 7")]
    assert call(1, 0) == [(second, "stream 0")]
    capturing[0] = True                          # a graph keeps the plan itself
    assert call(2, 11) == []
    capturing[0] = False
    assert len(call(2, 11)) == 3
    assert all(name.startswith("ti_kv4_prefill") for name, _ in rec.calls)


class _Untouched:
    """In a tensor's place: any use of it is an error."""

    def __getattr__(self, name):
        raise AssertionError(f"used: {name}")

    def __setitem__(self, key, value):
        raise AssertionError("written")


def test_caches_that_cannot_evict_pay_nothing_for_it():
    """Without totals nothing is ever evicted: reading the device's lengths back and freeing a slot
    do not touch the positions' offsets (a copy to the host, a fill)."""
    for totals in (None, object()):
        kv = _manager(attn_weights=totals)
        if totals is None:
            kv.pos_offset = _Untouched()
        kv.alloc.plan_tokens([1], [20])
        kv.seq_len[1] = 20
        kv.block_tables.copy_(torch.from_numpy(kv._bt_host))
        kv.sync_from_device()
        assert (kv.seq_len_host(1), kv.position_host(1)) == (20, 20)
        kv.free_batch_slot(1)
        assert kv.seq_len_host(1) == 0 and len(kv.free_blocks) == 6
    kv.pos_offset[2] = 5                         # set on the device, as the lengths may be
    kv.sync_from_device()
    assert kv.position_host(2) == 5 and kv._evicted
    kv.free_batch_slot(2)
    assert kv.pos_offset[2] == 0 and kv.position_host(2) == 0


def test_last_position_after_an_eviction_by_hand():
    """The same where the program evicts between ticks, and the batcher does not."""
    import asyncio

    from tests.test_scheduler_trace import _StandInBackend
    from tiny_infra_b200.scheduler import ContinuousBatcher, GenerationRequest
    kv = _manager(max_positions=34)
    kv.free_batch_slot = kv.alloc.free_slot

    class Backend(_StandInBackend):
        def decode(self, slots, reqs):
            kv._check_positions(slots, 1)
            return super().decode(slots, reqs)
    sched = ContinuousBatcher(None, kv, backend=Backend(kv, 1000))

    async def run():
        for n, m in ((30, 20), (5, 12)):
            sched.requests_queue.put_nowait(GenerationRequest(list(range(n)), m, 0.0))
        sched._fill_active_slots()
        reqs = list(sched.active_slots)
        sched._step_generation()                 # the prefills
        kv.alloc.truncate(0, 10)
        kv._evicted = True
        while sched._has_active_requests():
            sched._step_generation()
        return reqs
    reqs = asyncio.run(run())
    assert [None if r is None else len(r.generated_tokens) for r in reqs] == [5, 12, None]
    assert "Position" in str(reqs[0].error) and reqs[1].error is None
