"""The model, the engine and the batcher on a 4-bit KV cache (KVCacheManager(kv_bits=4)), with and
without eviction, against the 64-bit oracle of the cache's operators (oracle.kv4).

Every layer's projection rows are taken from the run itself (the ``trace`` hook), so each check is of
the cache operators as the model calls them: what the cache holds is exactly the quantised rows, and
the attention is within the operators' tolerance (tests/test_gpu_kv4.py) of the oracle on the cache's
own bytes.
"""
import asyncio

import numpy as np
import pytest
import torch

from oracle import kv4 as OK
from tiny_infra_b200 import _native as N
from tests.test_gpu_kv4 import dev, half_step, rounded

pytestmark = pytest.mark.gpu
NH, KVH, D = 14, 2, 64


@pytest.fixture(scope="module")
def model(cuda_device):
    from tiny_infra_b200 import _native
    from tiny_infra_b200.config import QwenConfig
    from tiny_infra_b200.qwen2 import Qwen2ForCausalLM
    cfg = QwenConfig(num_layers=2, vocab_size=4096)
    m = Qwen2ForCausalLM(cfg).load_reference_state_dict(
        Qwen2ForCausalLM.random_state_dict(cfg, seed=2, std=0.05))
    m.deterministic = True
    _native.device_status()
    yield m
    assert _native.device_status() == 0


def manager(batch=4, max_seq=256, **kw):
    from tiny_infra_b200.cache_manager import KVCacheManager
    return KVCacheManager(batch, max_seq, 2, KVH, D, **{"kv_bits": 4, **kw})


@pytest.mark.parametrize("dtn", ["bf16", "fp16"])
@pytest.mark.parametrize("nh,kvh,d,tokens", [(14, 2, 64, 1), (14, 2, 64, 77), (8, 8, 64, 33),
                                             (32, 8, 128, 19), (9, 3, 128, 256)])
def test_rope_append_is_rope_then_append(cuda_device, dtn, nh, kvh, d, tokens):
    from tiny_infra_b200 import custom_rope, kv4
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtn]
    g = torch.Generator(device="cuda").manual_seed(tokens)
    row = torch.randn(tokens, (nh + 2 * kvh + 1) * d, generator=g, device="cuda").to(dt)
    qkv = row[:, :(nh + 2 * kvh) * d]
    f = torch.randn(300, d // 2, generator=g, device="cuda")
    cos, sin = f.cos(), f.sin()
    pos = torch.randint(0, 300, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    nb = tokens // 16 + 3
    slots = torch.randperm(nb * 16, generator=g, device="cuda")[:tokens]
    if tokens > 2:
        slots[1] = -1
    want = qkv.clone().view(tokens, nh + 2 * kvh, d)
    q, k = want[:, :nh].contiguous(), want[:, nh:nh + kvh].contiguous()
    custom_rope.apply_inplace(q, k, cos, sin, pos)
    ref = kv4.new_pool(nb, kvh, d)
    kv4.append(ref, k, want[:, nh + kvh:], slots)
    pool, w = kv4.new_pool(nb, kvh, d), torch.ones(nb, kvh, 16, device="cuda")
    tail = row[:, (nh + 2 * kvh) * d:].clone()
    kv4.rope_append(pool, qkv, nh, slots, cos, sin, pos, weights=w)
    got = qkv.view(tokens, nh + 2 * kvh, d)
    assert torch.equal(got[:, :nh], q) and torch.equal(got[:, nh:nh + kvh], k)
    assert torch.equal(got[:, nh + kvh:], want[:, nh + kvh:])
    assert torch.equal(row[:, (nh + 2 * kvh) * d:], tail)
    assert torch.equal(pool, ref)
    live = slots[slots >= 0]
    zero = torch.zeros(nb * 16, dtype=torch.bool, device="cuda")
    zero[live] = True
    assert torch.equal(w.transpose(1, 2).reshape(nb * 16, kvh) == 0, zero[:, None].expand(-1, kvh))
    with pytest.raises(RuntimeError):
        kv4.rope_append(pool, qkv[:, :-d], nh, slots, cos, sin, pos)


def test_rope_append_checks_positions(cuda_device):
    """Tokens whose position has no row in both tables are left alone and flagged; the others go on."""
    from tiny_infra_b200 import kv4
    N.device_status()
    g = torch.Generator(device="cuda").manual_seed(3)
    nh, kvh, d = 4, 2, 64
    qkv = torch.randn(5, (nh + 2 * kvh) * d, generator=g, device="cuda").to(torch.bfloat16)
    f = torch.randn(40, d // 2, generator=g, device="cuda")
    cos, sin = f.cos(), f.sin()[:30].contiguous()
    slots = torch.arange(5, device="cuda") * 16
    for at in ([0, 29, 30, 39, 7], [-1, 3, 2 ** 31 - 1, -2 ** 31, 40]):
        pos = torch.tensor(at, dtype=torch.int32, device="cuda")
        good = (pos >= 0) & (pos < 30)
        want, ref = qkv.clone(), kv4.new_pool(5, kvh, d)
        rows = want[good].contiguous()
        kv4.rope_append(ref, rows, nh, slots[good], cos, sin, pos[good])
        want[good] = rows
        assert N.device_status() == 0
        got, pool = qkv.clone(), kv4.new_pool(5, kvh, d)
        kv4.rope_append(pool, got, nh, slots, cos, sin, pos)
        assert N.device_status() == N.TI_DEVERR_BAD_INPUT
        assert torch.equal(got, want) and torch.equal(pool, ref)
    with pytest.raises(RuntimeError):
        kv4.rope_append(pool, qkv, nh, slots, cos[:, :-1].contiguous(), sin, pos)
    with pytest.raises(RuntimeError):
        kv4.rope_append(pool, qkv, nh, slots, cos, sin, pos[:-1])


class Trace:
    """The projection rows and the attention output of every layer of one forward."""

    def __init__(self):
        self.qkv, self.attn = {}, {}

    def __call__(self, layer, stage, bufs):
        if stage == "qkv":
            self.qkv[layer] = bufs["qkv"].double().cpu().numpy()
        if stage == "attn":
            self.attn[layer] = bufs["attn"].double().cpu().numpy()


def check_step(kv, tr, slots, starts, counts, weights_before=None):
    """One forward's cache writes and attention, layer by layer; starts = cached lengths before."""
    tables = kv._bt_host
    for la in range(2):
        pool = kv.kv4_pool[la].cpu().numpy()
        rows = tr.qkv[la].reshape(-1, NH + 2 * KVH, D)
        q, k, v = rows[:, :NH], rows[:, NH:NH + KVH], rows[:, NH + KVH:]
        want = pool.copy()
        at = np.concatenate([np.arange(s, s + c) for s, c in zip(starts, counts)])
        row = np.repeat(slots, counts)
        OK.put(want, k, v, tables[row, at // 16].astype(np.int64) * 16 + at % 16)
        for g, e in zip(OK.untile(pool), OK.untile(want)):
            np.testing.assert_array_equal(g, e)
        o, mean, flat, big = OK.prefill(q, pool, tables, starts, counts, rows=slots)
        err = np.abs(tr.attn[la].reshape(o.shape) - o)
        ds = (D + 8) * 2.0 ** -24 * big[..., None]
        tol = (half_step(o, torch.bfloat16) + mean * (2.0 ** -11 + 2 * ds + 2.0 ** -20) +
               2.0 ** -31 * flat)
        assert (err <= tol).all(), (la, np.max(err / tol))


def test_prefill_and_decode_layers(model):
    kv = manager()
    cos, sin = model.rope_tables(kv.max_positions)
    rng = np.random.default_rng(0)
    slots, counts = [2, 0, 3], [5, 70, 33]
    ids = rng.integers(0, 4096, sum(counts))
    pb = model.plan(kv, slots, counts, ids)
    tr = Trace()
    model.forward_packed(pb, kv, cos, sin, rows="last", trace=tr)
    check_step(kv, tr, slots, [0, 0, 0], counts)
    kv.advance_device(slots, counts)
    # a second chunk for two of them, behind what they have
    s2, c2 = [3, 2], [40, 2]
    pb = model.plan(kv, s2, c2, rng.integers(0, 4096, 42))
    tr = Trace()
    model.forward_packed(pb, kv, cos, sin, rows="last", trace=tr)
    check_step(kv, tr, s2, [33, 5], c2)
    kv.advance_device(s2, c2)
    for _ in range(3):
        starts = [kv.seq_len_host(s) for s in slots]
        pb = model.plan(kv, slots, [1] * 3, rng.integers(0, 4096, 3))
        tr = Trace()
        model.forward_packed(pb, kv, cos, sin, rows="last", trace=tr)
        check_step(kv, tr, slots, starts, [1] * 3)
        kv.advance_device(slots, [1] * 3)
    for s in slots:
        kv.free_batch_slot(s)
    assert len(kv.free_blocks) == kv.total_physical_blocks


def test_chunked_prefill_fills_the_same_cache(model):
    rng = np.random.default_rng(1)
    ids = rng.integers(0, 4096, 90)
    pools, last = [], []
    for parts in ([90], [16, 41, 33], [1, 1, 88]):
        kv = manager(1)
        cos, sin = model.rope_tables(kv.max_positions)
        at = 0
        for n in parts:
            pb = model.plan(kv, [0], [n], ids[at:at + n])
            lg = model.forward_packed(pb, kv, cos, sin, rows="last")
            kv.advance_device([0], [n])
            at += n
        pools.append(kv.kv4_pool[0].clone())
        last.append(lg[0].float())
    # layer 0 reads only the embedding: the same rows whatever the chunks, up to the projection's
    # tile shape; a differing 16-bit rounding may move a code by one step
    a = OK.untile(pools[0].cpu().numpy())
    for other in pools[1:]:
        for x, y in zip(a, OK.untile(other.cpu().numpy())):
            differ = (x != y)
            assert differ.mean() < 2e-3
    for l in last[1:]:
        assert torch.corrcoef(torch.stack([last[0], l]))[0, 1] > 0.99


def test_engine_steps_equal_eager_forwards(model):
    """Graph-replayed decode steps produce the tokens of eager forwards on a second cache."""
    from tiny_infra_b200.engine import DecodeEngine
    rng = np.random.default_rng(3)
    kvs = [manager(4, 128, track_weights=tw) for tw in (False, False, True)]
    cos, sin = model.rope_tables(128)
    slots, counts = [0, 1, 3], [20, 3, 47]
    ids = rng.integers(0, 4096, sum(counts))
    first = None
    for kv in kvs:
        pb = model.plan(kv, slots, counts, ids)
        lg = model.forward_packed(pb, kv, cos, sin, rows="last")
        kv.advance_device(slots, counts)
        first = lg.float().argmax(-1).tolist()
    engines = [DecodeEngine(model, kvs[0]), DecodeEngine(model, kvs[2])]
    toks = [first, first, first]
    for _ in range(20):
        pb = model.plan(kvs[1], slots, [1] * 3, toks[1])
        lg = model.forward_packed(pb, kvs[1], cos, sin, rows="last")
        kvs[1].advance_device(slots, [1] * 3)
        new = [engines[0].step(slots, toks[0]).tolist(), lg.float().argmax(-1).tolist(),
               engines[1].step(slots, toks[2]).tolist()]
        assert new[0] == new[2]
        top2 = lg.float().topk(2, -1)[0]
        for i in range(3):                   # bf16 logits may tie; the epilogue compares in float32
            if new[0][i] != new[1][i]:
                assert top2[i, 0] - top2[i, 1] <= 2 ** -7 * top2[i, 0].abs()
                new[1][i] = new[0][i]
        toks = new
    for kv in kvs[1:]:
        n = [kv.seq_len_host(s) for s in slots]
        assert n == [c + 20 for c in counts]
    a, b = kvs[0].kv4_pool, kvs[2].kv4_pool
    for s in slots:
        blk = kvs[0]._bt_host[s][:-(-kvs[0].seq_len_host(s) // 16)]
        np.testing.assert_array_equal(blk, kvs[2]._bt_host[s][:len(blk)])
        assert torch.equal(a[:, blk.tolist()], b[:, blk.tolist()])


def test_weights_eviction_and_positions(model):
    """Totals are what the oracle adds up, eviction keeps what it would keep, freed blocks return,
    and the steps after it rotate at the sequences' own positions."""
    from tiny_infra_b200.engine import DecodeEngine
    from tiny_infra_b200.qwen2 import OBSERVE
    rng = np.random.default_rng(5)
    kv = manager(3, 128, track_weights=True, max_positions=400)
    eng = DecodeEngine(model, kv)
    assert eng.cos.shape[0] == 400
    slots, counts = [0, 2], [75, 5]
    pb = model.plan(kv, slots, counts, rng.integers(0, 4096, sum(counts)))
    tr = Trace()
    model.forward_packed(pb, kv, eng.cos, eng.sin, rows="last", trace=tr)
    kv.advance_device(slots, counts)
    for la in range(2):
        pool = kv.kv4_pool[la].cpu().numpy()
        q = tr.qkv[la].reshape(-1, NH + 2 * KVH, D)[:, :NH]
        w, slack = np.zeros(kv.attn_weights[la].shape), 0.0
        for i, (s, n) in enumerate(zip(slots, counts)):
            for back in range(min(OBSERVE, n)):
                r = (75 if i else 0) + n - 1 - back
                lens = np.array([n - back])
                rows = np.array([s])
                _, lse, _, _, _ = OK.decode(q[r:r + 1], pool, kv._bt_host, lens, rows)
                w, extra = OK.weights(w, q[r:r + 1], lse, pool, kv._bt_host, lens, rows)
                slack = slack + extra
        got = kv.attn_weights[la].double().cpu().numpy()
        # the kernel's own log-sum-exp: off by what the attention's scores are off, as the weights
        tol = slack * (2.0 ** -19 + 2 * (D + 8) * 2.0 ** -24) + OBSERVE * 2.0 ** -23 * w
        assert (np.abs(got - w) <= tol).all()
    toks = [7, 8]
    for _ in range(30):
        toks = eng.step(slots, toks).tolist()
    total = kv.attn_weights.double().sum((1, 3)).cpu().numpy()          # [L, KVH]
    seen = (OBSERVE + 5 + 2 * 30) * (NH // KVH)
    np.testing.assert_allclose(total, seen, rtol=1e-5)
    pool, w = kv.kv4_pool.cpu().numpy(), kv.attn_weights.cpu().numpy()
    tables, lens = kv._bt_host.copy(), np.array([105, 35], np.int32)
    free = list(kv.free_blocks)
    assert kv.evict([0, 2], 40, 10) == [0]
    OK.evict(pool, w, tables, lens[:1], 40, 10, rows=np.array([0]))
    pos = np.arange(40)
    for la in range(2):
        g, e = OK.untile(kv.kv4_pool[la].cpu().numpy()), OK.untile(pool[la])
        for x, y in zip(g, e):
            np.testing.assert_array_equal(x[tables[0, pos // 16], :, pos % 16],
                                          y[tables[0, pos // 16], :, pos % 16])
        np.testing.assert_array_equal(
            kv.attn_weights[la].cpu().numpy()[tables[0, pos // 16], :, pos % 16],
            w[la][tables[0, pos // 16], :, pos % 16])
    assert list(kv.free_blocks) == free + tables[0, 3:7].tolist()
    assert (kv.seq_len_host(0), kv.position_host(0), kv.position_host(2)) == (40, 105, 35)
    assert kv.seq_len.tolist() == [40, 0, 35] and kv.pos_offset.tolist() == [65, 0, 0]
    np.testing.assert_array_equal(kv.block_tables.cpu().numpy(), kv._bt_host)
    # decode goes on: a graph step, then a traced eager step and a traced prefill chunk
    toks = eng.step(slots, toks).tolist()
    assert eng.positions[:2].tolist() == [105, 35] and eng.ctx_lens[:2].tolist() == [41, 36]
    kv.sync_from_device()
    assert (kv.seq_len_host(0), kv.position_host(0)) == (41, 106)
    for counts in ([1, 1], [20, 3]):
        starts = [kv.seq_len_host(s) for s in slots]
        pb = model.plan(kv, slots, counts, rng.integers(0, 4096, sum(counts)))
        first = [kv.position_host(s) for s in slots]
        assert pb.positions.tolist() == [p + i for p, c in zip(first, counts) for i in range(c)]
        tr = Trace()
        model.forward_packed(pb, kv, eng.cos, eng.sin, rows="last", trace=tr)
        check_step(kv, tr, slots, starts, counts)
        kv.advance_device(slots, counts)
    # refusals
    for bad in ((0, 0), (10, 11), (10, -1)):
        with pytest.raises(ValueError):
            kv.evict([0], *bad)
    with pytest.raises(ValueError):
        kv.evict([0, 0], 10, 2)
    with pytest.raises(ValueError):
        kv.evict([3], 10, 2)
    with pytest.raises(RuntimeError):
        manager(1).evict([0], 4, 1)
    kv.alloc.pos_offset[0] = 400 - kv.seq_len_host(0)
    with pytest.raises(ValueError, match="Position"):
        kv.plan_decode([0])
    with pytest.raises(ValueError, match="Position"):
        kv.plan_tokens([2, 0], [1, 1])
    kv.free_batch_slot(0)
    assert kv.position_host(0) == 0 and kv.pos_offset[0] == 0


def test_allocate_and_insert_on_four_bits(cuda_device):
    kv = manager(2, 64)
    k, v = torch.randn(2, 2, KVH, 20, D, device="cuda").unbind(0)
    kv.allocate_and_insert(1, torch.tensor([1, 0]), k, v)
    want = np.zeros(kv.kv4_pool[1].shape, np.uint8)
    for i, s in enumerate([1, 0]):
        pos = np.arange(20)
        OK.put(want, *(rounded(x[i].permute(1, 0, 2).cpu().numpy(), torch.bfloat16) for x in (k, v)),
               kv._bt_host[s, pos // 16].astype(np.int64) * 16 + pos % 16)
    for g, e in zip(OK.untile(kv.kv4_pool[1].cpu().numpy()), OK.untile(want)):
        np.testing.assert_array_equal(g, e)
    assert not kv.kv4_pool[0].any()


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_batcher_generates_past_the_cache(model, temperature):
    """Requests longer than a slot's cache, with eviction; and the plain 4-bit cache beside them."""
    from tiny_infra_b200.scheduler import ContinuousBatcher
    rng = np.random.default_rng(9)
    prompts = [(rng.integers(0, 4096, n).tolist(), m) for n, m in ((60, 100), (5, 120), (33, 20))]

    def run(kv, prompts, **kw):
        sched = ContinuousBatcher(model, kv, prefill_chunk_tokens=32, **kw)

        async def main():
            loop = asyncio.create_task(sched.run_loop())
            outs = await asyncio.gather(*[sched.generate(p, n, temperature=temperature)
                                          for p, n in prompts])
            loop.cancel()
            return outs
        outs = asyncio.run(main())
        assert len(kv.free_blocks) == kv.total_physical_blocks
        return outs, sched.stats()
    outs, st = run(manager(3, 64, track_weights=True, max_positions=300), prompts, evict_above=64,
                   evict_keep=32, evict_recent=12)
    assert [len(o) for o in outs] == [100, 120, 20] and st["requests_failed"] == 0
    # 60 + 99 cached tokens over a cache of 64 that drops to 32, and 5 + 119
    assert st["evictions"] == 1 + (60 + 99 - 65) // 32 + 1 + (5 + 119 - 65) // 32
    assert all(0 <= t < 4096 for o in outs for t in o)
    short = [(p[:30], 12) for p, _ in prompts]
    plain, st = run(manager(3, 64), short)
    kept, st2 = run(manager(3, 64, track_weights=True, max_positions=300), short, evict_above=64)
    assert st["evictions"] == st2["evictions"] == 0
    if temperature == 0.0:
        assert plain == kept                       # below the limit nothing changes
