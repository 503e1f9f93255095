"""The operators on drafted trees in the forms that programs make of their calls: together as a step runs
them, through the model, on other streams than the tensors' own, inside captures, two at once."""
import numpy as np
import pytest
import torch

from oracle import tree as oracle
from tests.test_gpu_tree import _attend as _attend_host
from tests.test_gpu_tree import _check_attention, _dev, _limits, _random_parents, _scene, _status

pytestmark = pytest.mark.gpu


def _device_scene(s):
    d = dict(q=s["q"].cuda(), k=s["k"].cuda(), v=s["v"].cuda(), tables=_dev(s["tables"]), ctx=_dev(s["ctx"]),
             cu=_dev(s["cu"]), masks=_dev(s["masks"].view(np.int32)))
    d["out"] = torch.zeros_like(d["q"])
    d["lse"] = torch.zeros(d["q"].shape[:2], device="cuda")
    return d


def _attend(d):
    from tiny_infra_b200 import tree
    tree.attention(d["out"], d["q"], d["k"], d["v"], d["tables"], d["ctx"], d["cu"], masks=d["masks"], lse=d["lse"])


def test_attention_same_bits_every_run():
    rng = np.random.default_rng(0)
    d = _device_scene(_scene(rng, 14, 2, 64, torch.bfloat16, [3000, 900, 50], [30, 5, 64]))
    _attend(d)
    first = d["out"].clone(), d["lse"].clone()
    for _ in range(5):
        d["out"].zero_()
        _attend(d)
        assert torch.equal(d["out"], first[0]) and torch.equal(d["lse"], first[1])


@pytest.mark.parametrize("masks", ["tree", None])
@pytest.mark.parametrize("nh,kvh,d,dtype", [(2, 1, 64, torch.bfloat16), (2, 1, 128, torch.float16), (14, 2, 64, torch.float16)])
def test_attention_many_short_sequences_of_one_to_three_chunks(nh, kvh, d, dtype, masks):
    """More units than CTAs, so that a CTA has several one behind the other, and few chunks a unit, so that the
    next one may use fewer of the CTA's slots: each gets its own sums, on every run."""
    rng = np.random.default_rng(11)
    n = 500
    s = _scene(rng, nh, kvh, d, dtype, rng.choice([20, 100, 170], n).tolist(), rng.integers(1, 5, n).tolist(), masks=masks)
    first = _check_attention(s)
    for _ in range(4):
        again = _attend_host(s)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


def test_attention_on_two_streams_and_in_two_graphs():
    """Calls that cut units over CTAs, at the same time: on two streams, and replayed as two graphs that were
    captured on one stream (the first of them as that stream's first call)."""
    rng = np.random.default_rng(1)
    ds = [_device_scene(_scene(rng, 14, 2, 64, torch.bfloat16, [4000, 2100, 333], [9, 30, 2])) for _ in range(2)]
    want = []
    for d in ds:
        _attend(d)
        want.append((d["out"].clone(), d["lse"].clone()))
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs = []
    for d in ds:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[2]):
            for _ in range(5):
                _attend(d)
        graphs.append(g)
    torch.cuda.synchronize()
    for how in ("streams", "graphs"):
        for d in ds:
            d["out"].zero_()
        torch.cuda.synchronize()
        for d, g, s in zip(ds, graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(10):
                    _attend(d) if how == "streams" else g.replay()
        torch.cuda.synchronize()
        for d, (o, l) in zip(ds, want):
            assert torch.equal(d["out"], o) and torch.equal(d["lse"], l), how
    assert _status() == 0


def test_attention_behind_a_call_that_ended_early():
    """Words that a call whose waits gave up has left in the workspace are not taken for halves of joins."""
    from tiny_infra_b200 import tree
    rng = np.random.default_rng(13)
    d = _device_scene(_scene(rng, 14, 2, 64, torch.bfloat16, [4000, 2100, 333], [9, 30, 2]))
    _attend(d)
    want = d["out"].clone(), d["lse"].clone()
    for left in (1, -1):
        torch.cuda.synchronize()
        for ws in tree._ws._buf.values():
            ws[:4096].view(torch.int32).fill_(left)
        for x in (d["q"], d["k"]):
            x.neg_()                                 # (the same scores, from parts written anew)
        d["v"].mul_(2)
        d["out"].zero_()
        _attend(d)
        assert torch.equal(d["out"], want[0] * 2) and torch.equal(d["lse"], want[1])
        d["v"].div_(2)
    for ws in tree._ws._buf.values():
        ws[:4096].zero_()
    torch.cuda.synchronize()
    assert _status() == 0


def test_attention_replayed_with_other_lengths():
    """A captured call reads lengths, tables and masks when it runs: sequences grow and shrink, some to
    nothing, between replays."""
    rng = np.random.default_rng(2)
    s = _scene(rng, 8, 2, 64, torch.float16, [900, 700, 40, 0], [12, 1, 20, 3])
    d = _device_scene(s)
    _attend(d)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _attend(d)
    for lens in ([900, 700, 40, 0], [1, 0, 0, 0], [130, 64, 31, 0]):
        s["ctx"] = np.array(lens, np.int32)
        d["ctx"].copy_(_dev(s["ctx"]))
        d["out"].zero_()
        g.replay()
        as64 = lambda t: t.double().numpy()                                              # noqa: E731
        ref, rl, size, big = oracle.attention(as64(s["q"]), as64(s["k"]), as64(s["v"]), s["tables"], s["ctx"],
                                              s["cu"], s["masks"])
        lim, _ = _limits(torch.float16, ref, size, big)
        assert (np.abs(d["out"].cpu().double().numpy() - ref) <= lim).all()
    assert _status() == 0


def test_attention_offsets_beyond_32_bits():
    """Blocks at the far end of a pool of more than 2^32 elements."""
    rng = np.random.default_rng(3)
    s = _scene(rng, 8, 8, 128, torch.bfloat16, [40, 100], [5, 17])
    nb, small = (1 << 32) // (8 * 16 * 128) + 500, s["k"].shape[0]
    for x in "kv":
        big = torch.empty(nb, 8, 16, 128, dtype=torch.bfloat16, device="cuda")
        big[nb - small:] = s[x].cuda()
        s[x] = big
    tables = np.where(s["tables"] >= 0, s["tables"] + nb - small, -1)
    from tiny_infra_b200 import tree
    d = dict(q=s["q"].cuda(), out=torch.zeros_like(s["q"]).cuda())
    tree.attention(d["out"], d["q"], s["k"], s["v"], _dev(tables), _dev(s["ctx"]), _dev(s["cu"]),
                   masks=_dev(s["masks"].view(np.int32)))
    near = dict(s, k=s["k"][nb - small:].cpu(), v=s["v"][nb - small:].cpu())
    out, _ = _check_attention(near)
    assert torch.equal(d["out"].cpu(), out)
    # and their nodes moved there
    T = int(s["cu"][-1])
    slots = torch.arange(T, dtype=torch.int64) * 16 + (nb - 60) * 16
    k0 = s["k"].view(nb, 8, 16, 128)[nb - 60:].clone()
    num, path, new = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in ((2,), (2, 4), (2, 4)))
    par = torch.tensor([-1, 0, 0, 2, 3] + [-1] + [0] * 16, dtype=torch.int32).cuda()
    tok = torch.arange(T, dtype=torch.int32).cuda()
    tgt = torch.zeros(T, dtype=torch.int32).cuda()
    tgt[0], tgt[2], tgt[3] = 2, 3, 4
    tree.accept(s["k"], s["v"], tok, par, tgt, _dev(s["cu"]), slots.cuda(), num, path, new)
    assert num.tolist() == [4, 1] and path[0].tolist() == [0, 2, 3, 4]
    want = k0.clone()
    for j, c in enumerate([0, 2, 3, 4]):
        want[j, :, 0] = k0[c, :, 0]
    assert torch.equal(s["k"][nb - 60:], want) and _status() == 0


def test_calls_follow_the_current_stream():
    """Each call is queued on the current stream, behind what is there: inputs that a side stream writes late
    are seen."""
    from tiny_infra_b200 import paging, sampler
    side = torch.cuda.Stream()
    lens, counts = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    tables = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    ring = paging.new_free_list(9)
    slots = torch.zeros(60, dtype=torch.int64, device="cuda")
    pos, cu = torch.zeros(60, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.zeros(3, 50000, device="cuda")
    t, u = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        counts.fill_(20)
        paging.reserve(tables, lens, counts, ring, slots, pos, cu)
        x[:, 777] = 5.0
        tok = sampler.sample(x, t, u)
    side.synchronize()
    assert cu.tolist() == [0, 20, 40, 60] and slots[:60].min() >= 0 and tok.tolist() == [777] * 3


def test_sample_in_a_graph_and_rows_of_a_wide_buffer():
    """Captured and replayed with other parameters; row starts that are not 16-byte aligned."""
    from tiny_infra_b200 import sampler
    rng = np.random.default_rng(4)
    x = torch.from_numpy(rng.standard_normal((6, 40001)) * 3).bfloat16().cuda()
    t, u = torch.full((6,), 0.9, device="cuda"), torch.zeros(6, device="cuda")
    out = torch.zeros(6, dtype=torch.int32, device="cuda")
    k = torch.full((6,), 50, dtype=torch.int32, device="cuda")
    sampler.sample(x, t, u, top_ks=k, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sampler.sample(x, t, u, top_ks=k, out=out)
    for kk in (50, 0, 3):
        un = rng.random(6).astype(np.float32)
        u.copy_(torch.from_numpy(un))
        k.fill_(kk)
        g.replay()
        want = [oracle.sample(x[r].double().cpu().numpy(), float(np.float32(0.9)), float(un[r]), kk)[0] for r in range(6)]
        assert out.tolist() == want


def test_a_step_of_everything_together():
    """reserve -> K and V into the pool -> attention -> logits -> sample -> accept -> release, several steps,
    lengths only on the device; beside it the step-by-step forms on host copies."""
    from tiny_infra_b200 import _native as N
    from tiny_infra_b200 import paging, sampler, tree
    rng = np.random.default_rng(5)
    S, KVH, NH, D, L, V, NB, COLS, P = 5, 2, 6, 64, 2, 300, 60, 12, 6
    gen = torch.Generator(device="cuda").manual_seed(5)
    kc, vc = (torch.zeros(L, NB, KVH, 16, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    tables, ring = torch.full((S, COLS), -1, dtype=torch.int32, device="cuda"), paging.new_free_list(NB)
    lens = torch.zeros(S, dtype=torch.int32, device="cuda")
    h_tables, h_ring = tables.cpu().numpy().copy(), ring.cpu().numpy().copy()
    h_lens = np.zeros(S, np.int32)
    h_kv = np.zeros((2, L, NB, KVH, 16, D))
    head = torch.randn(NH * D, V, generator=gen, device="cuda") / 8
    for step in range(6):
        counts = rng.integers(1, 30, S).astype(np.int32)
        T, words = int(counts.sum()), 1
        parents = np.array(sum((_random_parents(rng, n) for n in counts), []), np.int32)
        tokens = rng.integers(0, 12, T).astype(np.int32)
        slots = torch.empty(T, dtype=torch.int64, device="cuda")
        pos, cu = torch.empty(T, dtype=torch.int32, device="cuda"), torch.empty(S + 1, dtype=torch.int32, device="cuda")
        masks = torch.empty(T, words, dtype=torch.int32, device="cuda")
        dp, dk = _dev(parents), _dev(tokens)
        paging.reserve(tables, lens, _dev(counts), ring, slots, pos, cu, parents=dp, masks=masks)
        q, k, v = (torch.randn(T, L, h, D, generator=gen, device="cuda").bfloat16() for h in (NH, KVH, KVH))
        out, lse = torch.empty(L, T, NH, D, dtype=torch.bfloat16, device="cuda"), torch.empty(T, NH, device="cuda")
        for la in range(L):
            kl, vl = k[:, la].contiguous(), v[:, la].contiguous()
            N.check(N.lib().ti_kv_scatter(kc[la].data_ptr(), vc[la].data_ptr(), kl.data_ptr(), KVH * D, D, vl.data_ptr(),
                                          KVH * D, D, slots.data_ptr(), T, NB, KVH, D, 16, 0,
                                          torch.cuda.current_stream().cuda_stream))
            ql = q[:, la].contiguous()
            tree.attention(out[la], ql, kc[la], vc[la], tables, lens, cu, masks=masks, lse=lse)
        # (few tokens can be drawn, so that guesses hold now and then)
        logits = out[L - 1].flatten(1).float() @ head
        logits[:, 12:] = -float("inf")
        t = torch.full((T,), 0.8 if step % 2 else 0.0, device="cuda")
        u = torch.rand(T, generator=gen, device="cuda")
        mp = torch.full((T,), 0.2, device="cuda")
        targets = sampler.sample(logits, t, u, min_ps=mp)
        num, path, new = (torch.empty(n, dtype=torch.int32, device="cuda") for n in ((S,), (S, P), (S, P)))
        start = lens.clone()
        tree.accept(kc, vc, dk, dp, targets, cu, slots, num, path, new, seq_lens=lens)
        if step == 3:
            paging.release(tables, lens, ring)
        # ---- the same, step by step
        hs, hp, hcu, granted, hm = oracle.reserve(h_tables, h_lens, counts, h_ring, parents=parents, words=words)
        assert (granted == counts).all() and slots.tolist() == hs.tolist() and pos.tolist() == hp.tolist()
        np.testing.assert_array_equal(masks.cpu().numpy().view(np.uint32), hm)
        np.testing.assert_array_equal(start.cpu().numpy(), h_lens)
        for i, x in enumerate((k, v)):
            for la in range(L):
                h_kv[i, la, hs // 16, :, hs % 16] = x[:, la].double().cpu().numpy()
        for la in range(L):
            ref, rl, size, big = oracle.attention(q[:, la].double().cpu().numpy(), h_kv[0, la], h_kv[1, la], h_tables, h_lens,
                                                  hcu, hm)
            lim, _ = _limits(torch.bfloat16, ref, size, big)
            assert (np.abs(out[la].cpu().double().numpy() - ref) <= lim).all()
        want = [oracle.sample(x, float(a), float(b), 0, 1.0, float(np.float32(0.2)))[0] for x, a, b in
                zip(logits.double().cpu().numpy(), t.tolist(), u.tolist())]
        assert targets.tolist() == want
        paths, news = oracle.accept(tokens, parents, want, hcu.tolist(), P)
        pad = lambda a: a + [-1] * (P - len(a))                                          # noqa: E731
        assert path.tolist() == [pad(p) for p in paths] and new.tolist() == [pad(p) for p in news]
        old = h_kv.copy()
        for i, p in enumerate(paths):
            for j, c in enumerate(p):
                a, b = hs[hcu[i] + c], hs[hcu[i] + j]
                h_kv[:, :, b // 16, :, b % 16] = old[:, :, a // 16, :, a % 16]
            h_lens[i] += len(p)
        if step == 3:
            oracle.release(h_tables, h_lens, h_ring)
        for i, x in enumerate((kc, vc)):
            np.testing.assert_array_equal(x.double().cpu().numpy(), h_kv[i])
        np.testing.assert_array_equal(tables.cpu().numpy(), h_tables)
        assert paging.free_ids(ring) == paging.free_ids(torch.from_numpy(h_ring))
    assert int(lens.sum()) > 6 * S and _status() == 0


@pytest.mark.parametrize("scratch", [False, True])
def test_a_pool_too_short_for_some(scratch):
    """reserve -> accept with a pool that does not reach: a sequence that was not served emits nothing, keeps its
    length and its cache, and goes on when there are blocks; the others do not notice.  scratch: the nodes
    are in blocks of their own, and the slots that the path moves to are the reserved ones."""
    from tiny_infra_b200 import paging, tree
    rng = np.random.default_rng(12)
    counts, lens0 = [20, 7, 40, 3], [30, 17, 16, 0]
    T, P, NB, L, KVH, D = sum(counts), 6, 40, 2, 2, 64
    kc, vc = (torch.from_numpy(rng.standard_normal((L, NB, KVH, 16, D))).bfloat16().cuda() for _ in range(2))
    tables = torch.full((4, 6), -1, dtype=torch.int32, device="cuda")
    tables[0, :2], tables[1, :2], tables[2, :1] = (_dev(np.arange(a, b, dtype=np.int32)) for a, b in ((0, 2), (2, 4), (4, 5)))
    # blocks needed: 2, 0, 3, 1; two are there, and the last sequence comes behind the one that ends the list
    ring, lens = paging.free_list([5, 6], capacity=20), _dev(np.array(lens0, np.int32))
    parents = np.concatenate([np.arange(-1, n - 1) for n in counts]).astype(np.int32)
    tokens = np.arange(T, dtype=np.int32)
    targets = np.where(tokens % 4 == 2, -7, tokens + 1).astype(np.int32)    # a path ends behind every fourth token
    cu, granted = torch.empty(5, dtype=torch.int32, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")
    slots, pos = torch.empty(T, dtype=torch.int64, device="cuda"), torch.empty(T, dtype=torch.int32, device="cuda")
    first = np.concatenate([[0], np.cumsum(counts)])

    def step(want_granted):
        num, path, new = (torch.full(n, 9, dtype=torch.int32, device="cuda") for n in ((4,), (4, P), (4, P)))
        paging.reserve(tables, lens, _dev(np.array(counts, np.int32)), ring, slots, pos, cu, granted=granted)
        assert granted.tolist() == [c if w else 0 for c, w in zip(counts, want_granted)]
        own = torch.arange(T, dtype=torch.int64, device="cuda") + (NB - 5) * 16 if scratch else slots
        before, was = (kc.clone(), vc.clone()), lens.tolist()
        tree.accept(kc, vc, _dev(tokens), _dev(parents), _dev(targets), cu, own, num, path, new,
                    out_slots=slots, seq_lens=lens)
        paths, news = oracle.accept(tokens, parents, targets, first.tolist(), P)
        paths = [p if w else [] for p, w in zip(paths, want_granted)]
        pad = lambda a: a + [-1] * (P - len(a))                                          # noqa: E731
        assert num.tolist() == [len(p) for p in paths] and path.tolist() == [pad(p) for p in paths]
        assert new.tolist() == [pad(n if w else []) for n, w in zip(news, want_granted)]
        assert lens.tolist() == [a + len(p) for a, p in zip(was, paths)]
        for old, now in zip(before, (kc, vc)):
            want = old.clone()
            for i, p in enumerate(paths):
                for j, c in enumerate(p):
                    a, b = int(own[first[i] + c]), int(slots[first[i] + j])
                    want[:, b // 16, :, b % 16] = old[:, a // 16, :, a % 16]
            assert torch.equal(now, want)

    step([True, True, False, False])
    ring2 = paging.free_list(paging.free_ids(ring) + list(range(10, 20)), capacity=20)
    ring.copy_(ring2)
    step([True] * 4)
    assert lens[2] > 16 and lens[3] > 0 and _status() == 0


# ---- through the model --------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def model():
    from tiny_infra_b200.config import QwenConfig
    from tiny_infra_b200.qwen2 import Qwen2ForCausalLM
    cfg = QwenConfig(num_layers=2, vocab_size=4096)
    m = Qwen2ForCausalLM(cfg).load_reference_state_dict(Qwen2ForCausalLM.random_state_dict(cfg, seed=3, std=0.05))
    m.deterministic = True
    return m


def _manager(batch=4, max_seq=512):
    from tiny_infra_b200.cache_manager import KVCacheManager
    return KVCacheManager(batch, max_seq, 2, 2, 64)


def _prompted(model, prompts):
    """A decoder whose slots hold these prompts but for their last tokens."""
    from tiny_infra_b200.speculative import TreeDecoder
    kv = _manager(len(prompts))
    dec = TreeDecoder(model, kv)
    counts = [len(p) - 1 for p in prompts]
    pb = model.plan(kv, range(len(prompts)), counts, np.concatenate([p[:-1] for p in prompts]))
    model.forward_packed(pb, kv, dec.cos, dec.sin, rows="last")
    kv.advance_device(range(len(prompts)), counts)
    return dec


def _logits_of(model, seq):
    kv = _manager(1)
    cos, sin = model.rope_tables(kv.max_positions)
    return model.forward_packed(model.plan(kv, [0], [len(seq)], np.asarray(seq)), kv, cos, sin, rows="all").float().cpu()


def test_tree_decoder_greedy(model):
    """Every emitted token is the likeliest behind the sequence so far, by a forward of its own over the whole
    sequence (to bf16 logits' noise); guesses that are right are kept, in whatever branch they are."""
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, 4096, n).tolist() for n in (30, 5, 100)]
    plain, dec = _prompted(model, prompts), _prompted(model, prompts)
    seqs = [list(p) for p in prompts]
    for _ in range(12):                          # trees of one node: one token a step
        new = plain.step([0, 1, 2], [([s[-1]], [-1]) for s in seqs])
        for s, n in zip(seqs, new):
            assert len(n) == 1
            s += n
    known = [s[len(p):] for s, p in zip(seqs, prompts)]
    got, steps = [list(p) for p in prompts], 0
    while min(len(g) - len(p) for g, p in zip(got, prompts)) < 12:
        trees = []
        for g, p, kn in zip(got, prompts, known):
            at = len(g) - len(p)
            guess = kn[at:at + 3] + rng.integers(0, 4096, 3).tolist()
            # a wrong branch first, then the right chain, then wrong tails
            toks = [g[-1], (guess[0] + 1) % 4096] + guess[:3] + [(guess[1] + 7) % 4096]
            trees.append((toks, [-1, 0, 0, 2, 3, 2]))
        steps += 1
        for g, n in zip(got, dec.step([0, 1, 2], trees)):
            g += n
    assert steps <= 8                            # (most steps keep three guesses)
    for g in got + seqs:
        lg = _logits_of(model, g)
        lg2 = lg[:-1].max(-1).values - lg[:-1].gather(1, torch.tensor(g[1:]).view(-1, 1)).squeeze(1)
        n = next(len(p) for p in prompts if g[:len(p)] == p)
        # two forwards of different shape differ by a few bf16 steps of the logits
        assert (lg2[n - 1:] <= 4 * 2.0 ** -8 * lg[n - 1:-1].abs().max()).all()
    for i, g in enumerate(got):
        assert dec.kv.seq_len_host(i) == len(g) - 1 == int(dec.kv.seq_len[i])
        held = int((dec.kv.block_tables[i] >= 0).sum())
        assert held * 16 >= len(g) - 1 and held == int((dec.kv.alloc.block_tables[i] >= 0).sum())
    np.testing.assert_array_equal(dec.kv.block_tables.cpu().numpy(), dec.kv.alloc.block_tables)
    # what is cached is what a prefill of the sequence caches
    kv = _manager(1)
    model.forward_packed(model.plan(kv, [0], [len(got[0]) - 1], np.asarray(got[0][:-1])), kv, dec.cos, dec.sin, rows="last")
    n = len(got[0]) - 1
    rows = lambda m, c: c[0][m.block_tables[0, :-(-n // 16)].long()].transpose(0, 1).reshape(2, -1, 64)[:, :n].float()  # noqa: E731
    assert torch.allclose(rows(kv, kv.key_cache), rows(dec.kv, dec.kv.key_cache), atol=0.06, rtol=0.02)
    assert _status() == 0


def test_tree_decoder_draws_and_refuses(model):
    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, 4096, n).tolist() for n in (9, 40)]
    dec = _prompted(model, prompts)
    trees = [([p[-1], 5, 6, 7], [-1, 0, 1, 0]) for p in prompts]
    new = dec.step([0, 1], trees, temperatures=[0.8, 0.0], top_ks=[0, 0], min_ps=[0.1, 0.0], top_ps=[0.9, 1.0],
                   uniforms=rng.random(8))
    assert all(1 <= len(n) <= 3 for n in new)
    for bad in ((([1, 2], [-1, 1]), "earlier"), (([1], [0]), "root"), (([], []), "token"), (([1, 2], [-1]), "per node")):
        with pytest.raises(ValueError, match=bad[1]):
            dec.step([0, 1], [bad[0], trees[1]])
    with pytest.raises(ValueError, match="distinct"):
        dec.step([0, 0], trees)
    with pytest.raises(ValueError, match="uniform"):
        dec.step([0, 1], trees, temperatures=[0.8, 0.0])
    with pytest.raises(ValueError, match="per slot"):
        dec.step([0, 1], trees, top_ks=[1])
    from tiny_infra_b200.cache_manager import KVCacheManager
    from tiny_infra_b200.speculative import TreeDecoder
    with pytest.raises(RuntimeError, match="16-bit"):
        TreeDecoder(model, KVCacheManager(2, 64, 2, 2, 64, kv_bits=4))
    assert dec.step([], []) == [] and _status() == 0
