"""Calls of the 4-bit KV cache's operators in the forms that programs make of them: all layers at
once, on other streams than the tensors' own, inside captures, through the model and the batcher.
Oracle and tolerances: tests/test_gpu_kv4.py."""
import numpy as np
import pytest
import torch

from oracle import kv4 as OK
from tests.test_gpu_kv4 import DT, dev, random_pool, rounded, tables_for

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv4(cuda_device):
    from tiny_infra_b200 import _native, kv4
    _native.device_status()
    yield kv4
    assert _native.device_status() == 0


@pytest.mark.parametrize("dtn", ["bf16", "fp16"])
@pytest.mark.parametrize("d,kvh,layers", [(64, 2, 3), (128, 1, 2)])
def test_evict_all_layers_and_read_them_back(kv4, dtn, d, kvh, layers):
    """The survivors of every layer, read back in one call from the pool that evict took: block
    ids count through the layers.  Exact."""
    rng = np.random.default_rng(d + layers)
    lens, keep, recent, dt = np.array([70, 16, 0, 33], np.int32), 32, 5, DT[dtn]
    new = np.minimum(lens, keep)
    tables, nb = tables_for(rng, lens)
    pool = np.stack([random_pool(rng, nb, kvh, d) for _ in range(layers)])
    w = rng.random((layers, nb, kvh, 16)).astype(np.float32)
    dp, dw = dev(pool), dev(w)
    kv4.evict(dp, dw, dev(tables), dev(lens), keep, recent)
    OK.evict(pool, w, tables, lens, keep, recent)
    most = keep // 16
    src = np.full((layers, len(lens), most), -1, np.int32)
    dst = src.copy()
    for la in range(layers):
        for i, n in enumerate(new):
            k = -(-int(n) // 16)
            src[la, i, :k] = la * nb + tables[i, :k]
            dst[la, i, :k] = (la * len(lens) + i) * most + np.arange(k)
    ko = torch.full((layers * len(lens) * most, kvh, 16, d), 9.0, dtype=dt, device="cuda")
    vo = ko.clone()
    kv4.dequantize(dp, dev(src.reshape(-1, most)), dev(np.tile(new, layers)),
                   dev(dst.reshape(-1, most)), ko, vo)
    for g, which in ((ko, 0), (vo, 1)):
        want = np.full(g.shape, 9.0)
        for la in range(layers):
            vals = OK.untile(pool[la])[which]
            for i, n in enumerate(new):
                for j in range(-(-int(n) // 16)):
                    x = vals[tables[i, j]].copy()
                    x[:, max(0, int(n) - 16 * j):] = 0
                    want[dst[la, i, j]] = x
        np.testing.assert_array_equal(g.double().cpu().numpy(), rounded(want, dt))


@pytest.fixture(scope="module")
def model(cuda_device):
    from tiny_infra_b200.config import QwenConfig
    from tiny_infra_b200.qwen2 import Qwen2ForCausalLM
    cfg = QwenConfig(num_layers=2, vocab_size=4096)
    m = Qwen2ForCausalLM(cfg).load_reference_state_dict(
        Qwen2ForCausalLM.random_state_dict(cfg, seed=2, std=0.05))
    m.deterministic = True
    return m


def manager(batch=4, max_seq=256, **kw):
    from tiny_infra_b200.cache_manager import KVCacheManager
    return KVCacheManager(batch, max_seq, 2, 2, 64, **{"kv_bits": 4, **kw})


def test_batcher_ends_one_sequence_at_its_last_position(kv4, model):
    """Two requests on a cache of 80 positions: the one that reaches them ends with its error after
    its tokens, the other completes."""
    import asyncio

    from tiny_infra_b200.scheduler import ContinuousBatcher
    kv = manager(2, 64, track_weights=True, max_positions=80)
    sched = ContinuousBatcher(model, kv, evict_above=48, evict_keep=24, evict_recent=8)

    async def main():
        loop = asyncio.create_task(sched.run_loop())

        async def one(prompt, n):
            got, error = [], None
            try:
                async for t in sched.generate_stream(prompt, n, temperature=0.0):
                    got.append(t)
            except ValueError as e:
                error = e
            return got, error
        outs = await asyncio.gather(one(list(range(40)), 100), one([5, 6, 7], 60))
        loop.cancel()
        return outs
    (long, error), (short, none) = asyncio.run(main())
    assert len(long) == 1 + 40 and "Position" in str(error)
    assert len(short) == 60 and none is None
    assert len(kv.free_blocks) == kv.total_physical_blocks


def test_model_decode_captured_first_and_twice(kv4, model):
    """A decode forward on a 4-bit cache, captured as the first call of its stream: what runs on the
    stream afterwards is right before the graph has replayed once, and two graphs captured on one
    stream replay at the same time."""
    rng = np.random.default_rng(4)
    lens = [600, 40, 333]                       # units that are cut: their joins count arrivals
    kvs = [manager(3, 2048) for _ in range(2)]
    cos, sin = model.rope_tables(2048)
    ids = rng.integers(0, 4096, sum(lens))
    pbs, want, hidden = [], [], []
    for kv in kvs:
        pb = model.plan(kv, [0, 1, 2], lens, ids)
        model.forward_packed(pb, kv, cos, sin, rows="last")
        kv.advance_device([0, 1, 2], lens)
        pbs.append(model.plan(kv, [0, 1, 2], [1, 1, 1], [7, 8, 9]))
        hidden.append(torch.randn(3, model.config.hidden_size, device="cuda",
                                  generator=torch.Generator(device="cuda").manual_seed(1)))
        # (a forward of the same token writes the same bytes into the cache again)
        want.append(model.forward_packed(pbs[-1], kv, cos, sin, hidden_in=hidden[-1], return_hidden=True))
    assert torch.equal(*want) and not torch.isnan(want[0]).any()
    torch.cuda.synchronize()
    side, replay = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for kv, pb, h in zip(kvs, pbs, hidden):
        bufs = model.scratch(3, {})             # of the graph's own
        out = torch.empty_like(h)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out.copy_(h)
            model._layers(pb, kv, cos, sin, out, side.cuda_stream, bufs=bufs)
        graphs.append((g, bufs))
        outs.append(out)
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = model.forward_packed(pbs[0], kvs[0], cos, sin, hidden_in=hidden[0], return_hidden=True)
            assert torch.equal(got, want[0])
    torch.cuda.synchronize()
    for _ in range(10):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, (g, _) in zip(replay, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_model_under_another_default_dtype(kv4, model, default):
    """Prefill with totals, decode and eviction do not depend on torch's default dtype."""
    ids, runs = np.random.default_rng(6).integers(0, 4096, 45), []
    for dt in (torch.float32, default):
        torch.set_default_dtype(dt)
        try:
            kv = manager(2, 64, track_weights=True)
            cos, sin = model.rope_tables(64)
            logits = []
            for slots, counts in (([0, 1], [40, 5]), ([0, 1], [1, 1])):
                pb = model.plan(kv, slots, counts, ids[:sum(counts)])
                logits.append(model.forward_packed(pb, kv, cos, sin, rows="last"))
                kv.advance_device(slots, counts)
            assert kv.evict([0], 20, 4) == [0]
        finally:
            torch.set_default_dtype(torch.float32)
        runs.append((*logits, kv.attn_weights, kv.kv4_pool))
    for a, b in zip(*runs):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_plan_dropped_behind_a_call_on_another_stream(kv4):
    """The plan's memory stays its own until the side stream's call, queued behind 100 ms of waiting,
    is done: allocations of the plan's stream do not get it."""
    from tiny_infra_b200 import _native as N
    nh, kvh, d, starts, counts = 14, 2, 64, [5000, 0, 9000], [40, 3, 130]
    rng = np.random.default_rng(2)
    tables, nb = tables_for(rng, [s + c for s, c in zip(starts, counts)])
    pool, tab = dev(random_pool(rng, nb, kvh, d)), dev(tables)
    q = dev(rng.standard_normal((sum(counts), nh, d)), torch.bfloat16)
    want, out = torch.empty_like(q), torch.zeros_like(q)
    side, other = torch.cuda.Stream(), kv4.PrefillPlan(starts, counts)
    for stream in (torch.cuda.current_stream(), side):     # (what a stream's first call allocates)
        with torch.cuda.stream(stream):
            kv4.prefill_attention(want, q, pool, tab, other)
        torch.cuda.synchronize()
    plan = kv4.PrefillPlan(starts, counts)
    plan.layout(nh // kvh, kvh, d)
    torch.cuda.synchronize()
    sizes = [(t.data_ptr(), t.numel()) for t, _ in plan._tensors]
    assert len(sizes) == 2
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        kv4.prefill_attention(out, q, pool, tab, plan)
    done = torch.cuda.Event()
    done.record(side)
    del plan
    fresh = [torch.empty(n, dtype=torch.int32, device="cuda") for _, n in sizes for _ in range(4)]
    early = not done.query()
    torch.cuda.synchronize()
    assert early                                # the call was still waiting
    assert not {p for p, _ in sizes} & {t.data_ptr() for t in fresh}
    assert torch.equal(out, want) and N.device_status() == 0


def test_dequantize_leaves_blocks_behind_the_length(kv4):
    """Zeros fill the last block behind a row's length; a target block that lies wholly behind it is
    neither written nor looked at, whatever its entry."""
    from tiny_infra_b200 import _native as N
    rng = np.random.default_rng(3)
    pool = random_pool(rng, 4, 2, 64)
    lens, src = np.array([17, 0, 16], np.int32), np.array([[0, 1, 2], [0, 1, 2], [3, 0, 1]], np.int32)
    dst = np.array([[4, 0, 1], [2, 3, 99], [5, 6, 2 ** 31 - 1]], np.int32)
    ko = torch.full((7, 2, 16, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    vo = ko.clone()
    kv4.dequantize(dev(pool), dev(src), dev(lens), dev(dst), ko, vo)
    assert N.device_status() == 0
    for g, vals in zip((ko, vo), OK.untile(pool)):
        want = np.full(g.shape, 9.0)
        want[4], want[0], want[5] = vals[0], vals[1], vals[3]
        want[0][:, 1:] = 0
        np.testing.assert_array_equal(g.double().cpu().numpy(), rounded(want, torch.bfloat16))


@pytest.mark.parametrize("batch", [1, 8])
def test_evict_through_tables_of_any_width(kv4, batch):
    """The same eviction, bit for bit, whatever the table's width: keys in shared memory, few CTAs to
    an SM and more units than those, and beyond shared memory."""
    rng = np.random.default_rng(batch)
    layers, kvh, d, keep, recent = 24, 2, 64, 40, 9
    lens = rng.integers(1, 200, batch).astype(np.int32)
    lens[0] = 199
    runs = []
    tables, nb = tables_for(rng, lens)
    pool = np.stack([random_pool(rng, nb, kvh, d) for _ in range(layers)])
    w = rng.integers(0, 50, (layers, nb, kvh, 16)).astype(np.float32)
    for width in (tables.shape[1], 1200, 1600, 2048, 3000, 3100):
        t = np.full((batch, width), -1, np.int32)
        t[:, :tables.shape[1]] = tables
        dp, dw = dev(pool), dev(w)
        kept = torch.full((layers, batch, kvh, keep), -7, dtype=torch.int32, device="cuda")
        kv4.evict(dp, dw, dev(t), dev(lens), keep, recent, kept=kept)
        # (places behind the survivors hold anything)
        ko = torch.zeros(layers * batch * 3, kvh, 16, d, dtype=torch.float16, device="cuda")
        vo = torch.zeros_like(ko)
        off = np.arange(layers)[:, None, None] * nb
        src = np.where(tables[:, :3] >= 0, tables[:, :3] + off, -1).astype(np.int32).reshape(-1, 3)
        new = dev(np.tile(np.minimum(lens, keep), layers).astype(np.int32))
        kv4.dequantize(dp, dev(src), new, dev(np.arange(len(src) * 3, dtype=np.int32).reshape(-1, 3)), ko, vo)
        runs.append((kept, ko, vo))
    want = OK.evict(pool, w, tables, lens, keep, recent)
    for (la, b, h), idx in want.items():
        np.testing.assert_array_equal(runs[0][0][la, b, h, :len(idx)].cpu().numpy(), idx)
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)
