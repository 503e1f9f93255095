"""The calls of a step on drafted trees on the CPU: what they refuse, what they hand to the C entry points
(a stand-in library records it), the C entry points' own refusals, and the step-by-step forms against the
host allocator."""
import contextlib

import numpy as np
import pytest
import torch

from oracle import tree as oracle
from tests.test_kv4_calls import _Recorder


@pytest.fixture
def recorded(monkeypatch):
    """``paging`` and ``tree`` taking host tensors, their calls recorded."""
    from tiny_infra_b200 import _native, paging, tree
    rec = _Recorder(_native.SIGNATURES)
    monkeypatch.setattr(_native, "lib", lambda: rec)
    for m in (paging, tree):
        monkeypatch.setattr(m, "_device", lambda *t: 0)
        monkeypatch.setattr(m, "_on", lambda dev: contextlib.nullcontext())
        monkeypatch.setattr(m, "_stream", lambda dev: 0)
    monkeypatch.setattr(tree, "_workspace", lambda dev, n, s: torch.zeros(64, dtype=torch.uint8))
    return paging, tree, rec


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _reserve_args(**kw):
    a = dict(block_tables=_i32(3, 5), seq_lens=_i32(3), counts=_i32(3), ring=_i32(12),
             slot_mapping=torch.zeros(9, dtype=torch.int64), positions=_i32(9), cu_seqlens=_i32(4))
    a.update(kw)
    return a


def test_reserve_hands_over_its_arguments(recorded):
    paging, _, rec = recorded
    a = _reserve_args(granted=_i32(3), parents=_i32(9), masks=_i32(9, 2), row_index=_i32(3), pos_offset=_i32(3))
    paging.reserve(**a)
    name, c = rec.calls.pop()
    p = lambda n: a[n].data_ptr()                                                        # noqa: E731
    assert name == "ti_reserve_slots"
    assert c[:-1] == [p("block_tables"), 5, 3, 5, 16, p("row_index"), p("seq_lens"), p("pos_offset"), p("counts"), 3,
                      p("ring"), 10, p("slot_mapping"), p("positions"), 9, p("cu_seqlens"), p("granted"), p("parents"),
                      p("masks"), 2]


@pytest.mark.parametrize("change,words", [
    (dict(block_tables=torch.zeros(3, 5)), "block_tables"), (dict(block_tables=_i32(2, 5)), "fewer rows"),
    (dict(block_tables=_i32(5, 3).t()), "contiguous rows"), (dict(block_tables=_i32(1, 5).expand(3, 5)), "overlap"),
    (dict(counts=_i32(3).long()), "counts"), (dict(ring=_i32(2)), "free list"), (dict(ring=_i32(4, 3)), "free list"),
    (dict(seq_lens=_i32(2)), "seq_lens"), (dict(cu_seqlens=_i32(3)), "cu_seqlens"), (dict(granted=_i32(4)), "granted"),
    (dict(slot_mapping=_i32(9)), "slot_mapping"), (dict(positions=_i32(8)), "positions"),
    (dict(parents=_i32(8)), "parents"), (dict(masks=_i32(9, 1)), "go with parents"),
    (dict(parents=_i32(9), masks=_i32(8, 1)), "masks"), (dict(parents=_i32(9), masks=_i32(9, 0)), "masks"),
    (dict(row_index=_i32(2)), "row_index"), (dict(block_size=0), "block_size"),
    (dict(counts=_i32(5000), row_index=_i32(5000)), "4096"),
    (dict(block_tables=_i32(40000, 5), row_index=_i32(3)), "32768"),
    (dict(row_index=_i32(3), seq_lens=_i32(2)), "seq_lens")])
def test_reserve_refuses(recorded, change, words):
    paging, _, rec = recorded
    with pytest.raises(RuntimeError, match=words):
        paging.reserve(**_reserve_args(**change))
    assert not rec.calls


def test_release_refuses_and_empty_calls_launch_nothing(recorded):
    paging, _, rec = recorded
    for kw, words in ((dict(keep_lens=_i32(3).long()), "keep_lens"), (dict(keep_lens=_i32(4)), "fewer rows"),
                      (dict(ring=_i32(2)), "free list"), (dict(block_size=0), "block_size"),
                      (dict(row_index=_i32(2)), "row_index")):
        with pytest.raises(RuntimeError, match=words):
            paging.release(**{**dict(block_tables=_i32(3, 5), keep_lens=_i32(3), ring=_i32(9)), **kw})
    paging.release(_i32(3, 5), _i32(0), _i32(9))
    paging.reserve(**_reserve_args(counts=_i32(0), cu_seqlens=_i32(1), positions=_i32(0),
                                   slot_mapping=torch.zeros(0, dtype=torch.int64)))
    assert not rec.calls


def test_free_list():
    from tiny_infra_b200 import paging
    ring = paging.free_list([5, 3, 9], capacity=4, device="cpu")
    assert ring.tolist() == [0, 3, 5, 3, 9, 0] and paging.free_ids(ring) == [5, 3, 9]
    ring[0] = 2
    assert paging.free_ids(ring) == [9, 0, 5]
    assert paging.free_ids(paging.new_free_list(3, device="cpu")) == [0, 1, 2]
    for bad in (dict(ids=[1, 2], capacity=1), dict(ids=[]), dict(ids=[-1])):
        with pytest.raises(RuntimeError):
            paging.free_list(**bad, device="cpu")


def _attention_args(**kw):
    b16 = torch.bfloat16
    a = dict(out=torch.zeros(7, 4, 64, dtype=b16), q=torch.zeros(7, 4, 64, dtype=b16),
             k_cache=torch.zeros(6, 2, 16, 64, dtype=b16), v_cache=torch.zeros(6, 2, 16, 64, dtype=b16),
             block_tables=_i32(3, 5), context_lens=_i32(3), cu_seqlens=_i32(4))
    a.update(kw)
    return a


def _zeros(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_attention_hands_over_its_arguments(recorded):
    _, tree, rec = recorded
    a = _attention_args(masks=_i32(7, 3), lse=torch.zeros(7, 4), q=_zeros(7, 10, 64)[:, :4], row_index=_i32(3))
    tree.attention(**a)
    name, c = [x for x in rec.calls if x[0] == "ti_tree_attention"].pop()
    p = lambda n: a[n].data_ptr()                                                        # noqa: E731
    assert c[:-3] == [p("out"), 256, p("lse"), p("q"), 640, p("k_cache"), p("v_cache"), 6, p("block_tables"), 5, 3, 5,
                      p("row_index"), p("context_lens"), p("cu_seqlens"), 3, 7, p("masks"), 3, 4, 2, 64, 16, 0]


@pytest.mark.parametrize("change,words", [
    (dict(q=_zeros(7, 4, 64, dtype=torch.float32)), "q must"), (dict(out=_zeros(6, 4, 64)), "out must"),
    (dict(out=_zeros(7, 4, 64, dtype=torch.float16)), "out must"), (dict(out=_zeros(1, 4, 64).expand(7, 4, 64)), "overlap"),
    (dict(q=_zeros(7, 64, 4).transpose(1, 2)), "contiguous"), (dict(k_cache=_zeros(6, 2, 8, 64)), "k_cache"),
    (dict(v_cache=_zeros(6, 2, 16, 128)), "v_cache"), (dict(k_cache=_zeros(6, 16, 2, 64).transpose(1, 2)), "k_cache"),
    (dict(k_cache=_zeros(6, 2, 16, 64, dtype=torch.float16), v_cache=_zeros(6, 2, 16, 64, dtype=torch.float16)), "dtype"),
    (dict(k_cache=_zeros(6, 3, 16, 64), v_cache=_zeros(6, 3, 16, 64)), "multiple"),
    (dict(q=_zeros(7, 17, 64), out=_zeros(7, 17, 64), k_cache=_zeros(6, 1, 16, 64), v_cache=_zeros(6, 1, 16, 64)), "16 per"),
    (dict(q=_zeros(7, 4, 32), out=_zeros(7, 4, 32), k_cache=_zeros(6, 2, 16, 32), v_cache=_zeros(6, 2, 16, 32)), "head_dim"),
    (dict(context_lens=_i32(3).long()), "context_lens"), (dict(cu_seqlens=_i32(3)), "cu_seqlens"),
    (dict(block_tables=_i32(2, 5)), "fewer rows"), (dict(block_tables=_i32(3, 0)), "columns"),
    (dict(row_index=_i32(4)), "row_index"), (dict(masks=_i32(6, 1)), "masks"),
    (dict(masks=_i32(7, 1).long()), "masks"), (dict(lse=torch.zeros(7, 3)), "lse")])
def test_attention_refuses(recorded, change, words):
    _, tree, rec = recorded
    with pytest.raises(RuntimeError, match=words):
        tree.attention(**_attention_args(**change))
    assert not rec.calls


def _accept_args(**kw):
    a = dict(key_cache=_zeros(3, 6, 2, 16, 64), value_cache=_zeros(3, 6, 2, 16, 64), tokens=_i32(9), parents=_i32(9),
             targets=_i32(9), cu_seqlens=_i32(4), slot_mapping=torch.zeros(9, dtype=torch.int64), num=_i32(3),
             path=_i32(3, 8), out_tokens=_i32(3, 8))
    a.update(kw)
    return a


def test_accept_hands_over_its_arguments(recorded):
    _, tree, rec = recorded
    a = _accept_args(seq_lens=_i32(11), row_index=_i32(3))
    tree.accept(**a)
    name, c = rec.calls.pop()
    p = lambda n: a[n].data_ptr()                                                        # noqa: E731
    assert name == "ti_tree_accept"
    assert c[:-1] == [p("key_cache"), p("value_cache"), 3, 6, 2, 64, 16, 2, p("tokens"), p("parents"), p("targets"),
                      p("cu_seqlens"), 3, 9, p("slot_mapping"), p("slot_mapping"), p("num"), p("path"), p("out_tokens"),
                      8, p("seq_lens"), p("row_index"), 11]


@pytest.mark.parametrize("change,words", [
    (dict(key_cache=_zeros(6, 2, 64)), "caches"), (dict(value_cache=_zeros(3, 6, 2, 16, 128)), "caches"),
    (dict(key_cache=_zeros(3, 6, 16, 2, 64).transpose(2, 3)), "contiguous"),
    (dict(key_cache=_zeros(3, 6, 2, 16, 64, dtype=torch.float32)), "bf16"),
    (dict(key_cache=_zeros(3, 6, 2, 16, 20), value_cache=_zeros(3, 6, 2, 16, 20)), "multiple of 8"),
    (dict(tokens=_i32(8)), "parents"), (dict(targets=_i32(9).long()), "targets"), (dict(num=_i32(2)), "cu_seqlens"),
    (dict(slot_mapping=_i32(9)), "slot_mapping"), (dict(out_slots=torch.zeros(8, dtype=torch.int64)), "out_slots"),
    (dict(path=_i32(3, 7)), "path"), (dict(path=_i32(3, 0), out_tokens=_i32(3, 0)), "path"),
    (dict(path=_i32(3, 1025), out_tokens=_i32(3, 1025)), "1024"), (dict(out_tokens=_i32(8, 3).t()), "out_tokens"),
    (dict(seq_lens=_i32(2)), "seq_lens"), (dict(row_index=_i32(4)), "row_index")])
def test_accept_refuses(recorded, change, words):
    _, tree, rec = recorded
    with pytest.raises(RuntimeError, match=words):
        tree.accept(**_accept_args(**change))
    assert not rec.calls


def test_host_tensors_are_refused():
    from tiny_infra_b200 import paging, sampler, tree
    for call in (lambda: paging.reserve(**_reserve_args()), lambda: tree.attention(**_attention_args()),
                 lambda: tree.accept(**_accept_args()),
                 lambda: sampler.sample(torch.zeros(2, 5), torch.zeros(2), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="rows, vocab"):
        sampler.sample(torch.zeros(2, 3, 5), torch.zeros(2), torch.zeros(2))
    with pytest.raises(RuntimeError, match="contiguous rows"):
        sampler.sample(torch.zeros(5, 2).t(), torch.zeros(2), torch.zeros(2))


def test_c_entry_points_refuse():
    """Bad sizes come back as errors before any CUDA call (the addresses are never followed)."""
    from tiny_infra_b200 import _native as N
    lib, a = N.lib(), 1 << 20

    def refused(rc, words):
        assert rc != 0 and words in lib.ti_last_error().decode(), lib.ti_last_error()

    def attention(nb=6, cols=5, rows=3, seqs=3, nh=4, kvh=2, d=64, bs=16, dt=0, q=a, ws=1 << 40, stride=256):
        return lib.ti_tree_attention(a, stride, None, q, 256, a, a, nb, a, 5, rows, cols, None, a, a, seqs, 7, None, 0, nh,
                                     kvh, d, bs, dt, a, ws, None)
    refused(attention(q=None), "null")
    refused(attention(nb=0), "pool size")
    refused(attention(nh=5), "multiple")
    refused(attention(nh=34), "16 query heads")
    refused(attention(d=96), "head_dim")
    refused(attention(bs=8), "block_size")
    refused(attention(dt=2), "dtype")
    refused(attention(q=a + 2), "aligned")
    refused(attention(stride=260), "aligned")
    refused(attention(ws=1), "workspace")
    refused(attention(rows=2), "table")
    assert lib.ti_tree_attention_workspace_bytes(14, 2, 64) > 0

    def reserve(seqs=3, rows=3, cols=5, block=16, ring=8, cap=9, words=0, parents=None, idx=None):
        return lib.ti_reserve_slots(a, 5, rows, cols, block, idx, a, None, a, seqs, a, ring, a, a, cap, a, a, parents, a,
                                    words, None)
    refused(reserve(words=1), "null")
    refused(reserve(cols=0), "size")
    refused(reserve(block=0), "size")
    refused(reserve(ring=0), "size")
    refused(reserve(seqs=5000), "4096")
    refused(reserve(rows=40000, idx=a), "32768")
    refused(reserve(rows=2), "fewer")
    refused(lib.ti_release_blocks(a, 5, 3, 5, 16, None, None, 3, a, 8, None), "null")

    def accept(d=64, eb=2, path=8, layers=3, k=a):
        return lib.ti_tree_accept(k, a, layers, 6, 2, d, 16, eb, a, a, a, a, 3, 9, a, a, a, a, a, path, None, None, 0, None)
    refused(accept(k=None), "null")
    refused(accept(d=20), "aligned")
    refused(accept(k=a + 8), "aligned")
    refused(accept(path=0), "size")
    refused(accept(path=2000), "1024")
    refused(accept(layers=0), "size")

    def draw(rows=2, vocab=10, ld=10, dt=2, logits=a):
        return lib.ti_sample_ex(logits, ld, dt, rows, vocab, a, None, None, None, a, a, None, None)
    refused(draw(logits=None), "null")
    refused(draw(vocab=0), "size")
    refused(draw(ld=9), "size")
    refused(draw(vocab=1 << 25, ld=1 << 25), "2^24")
    refused(draw(dt=7), "dtype")
    assert draw(rows=0) == 0


def test_accept_refuses_tokens_beyond_32_bits():
    """A token's K and V in 16-byte units, and a block's row of them, are counted in 32 bits."""
    from tiny_infra_b200 import _native as N
    lib, a = N.lib(), 1 << 20
    for layers, kvh, d, bs in ((1 << 20, 1 << 10, 64, 16), (1 << 30, 1 << 30, 1 << 30, 16), (1, 1, 1 << 12, 1 << 28)):
        rc = lib.ti_tree_accept(a, a, layers, 6, kvh, d, bs, 2, a, a, a, a, 3, 9, a, a, a, a, a, 8, None, None, 0, None)
        assert rc != 0 and "2^30" in lib.ti_last_error().decode()


def test_step_by_step_forms_follow_the_host_allocator():
    from tiny_infra_b200.cache_manager import BlockAllocator
    rng = np.random.default_rng(0)
    host = BlockAllocator(9, 300, 16, num_blocks=70)
    tables, lens = np.full((9, 19), -1, np.int32), np.zeros(9, np.int32)
    ring = np.concatenate([[0, 70], np.arange(70)]).astype(np.int32)
    for step in range(20):
        if step % 5 == 4:
            gone = rng.permutation(9)[:5]
            for s in gone:
                host.free_slot(int(s))
            oracle.release(tables, np.zeros(5, int), ring, rows=gone)
            lens[gone] = 0
        slots, counts = rng.permutation(9)[:5], rng.integers(0, 25, 5)
        mapping, _ = host.plan_tokens(slots, counts)
        got = oracle.reserve(tables, lens, counts, ring, rows=slots)
        host.advance(slots, counts)
        lens[slots] += counts
        np.testing.assert_array_equal(got[0], mapping)
        np.testing.assert_array_equal(tables, host.block_tables)
        assert ring[1] == len(host.free_blocks)


def test_ancestor_bits_and_sampling_forms():
    bits = oracle.ancestor_bits([-1, 0, 0, 1, 3, -1], 1).ravel().tolist()
    assert bits == [1, 3, 5, 11, 27, 32] and oracle.depths([-1, 0, 0, 1, 3, -1]) == [0, 1, 1, 2, 3, 0]
    x = np.log([0.4, 0.1, 0.3, 0.2])
    draw = lambda u, **kw: oracle.sample(x, 1.0, u, **kw)[0]                             # noqa: E731
    assert [draw(u) for u in (0.0, 0.39, 0.41, 0.71, 0.95)] == [0, 0, 2, 3, 1]
    assert draw(0.99, k=2) == 2 and draw(0.99, p=0.5) == 2 and draw(0.99, p=0.3) == 0 and draw(0.99, m=0.6) == 2
    assert oracle.sample(x, 0.0, 0.9) == (0, 0.0)


def test_tree_decoder_refuses_slots_that_are_none():
    """Before a block is assigned or anything is sent to the device."""
    from types import SimpleNamespace

    from tiny_infra_b200.speculative import TreeDecoder
    model = SimpleNamespace(device=torch.device("cpu"), rope_tables=lambda n: (None, None))
    dec = TreeDecoder(model, SimpleNamespace(kv_bits=16, max_positions=64, max_batch_size=4))
    for slots in ([-1], [4], [0, -4], [3, 1 << 40]):
        with pytest.raises(ValueError, match="from 0 to 3"):
            dec.step(slots, [([5], [-1])] * len(slots))
