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
