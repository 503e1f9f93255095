"""Drafted trees over the paged 16-bit cache: the attention of all their nodes at once, and the acceptance.

A step of speculative decoding runs the model over a tree of tokens per sequence: node 0 is the last token
the sequence emitted, every other node a guess for what follows its parent.  ``paging.reserve`` gives the
nodes' slots, positions and masks; the model appends their K and V and attends with ``attention``;
``sampler.sample`` draws a token at every node; ``accept`` keeps the path that the draws confirm.

Trees are packed: sequence i's nodes are rows ``cu_seqlens[i] .. cu_seqlens[i + 1] - 1`` (int32 [B + 1]).

* ``attention``  each node over its sequence's cached tokens and its own ancestors
* ``accept``     follow the draws down the trees; K and V of the kept nodes move together

Every call runs on the current CUDA stream of its tensors' device; argument errors raise
``RuntimeError`` before anything is launched.
"""
from __future__ import annotations

import functools

import torch

from . import _native as N
from .kv4 import (_CODE, _HALF, _cuda, _device, _fail, _head_sums, _index, _on, _out_rows, _ptr, _rows, _stream,
                  _table)

BLOCK = 16
_COUNTERS = 4096                        # bytes at a workspace's front that have to be zero before its first call
_ws = N.Workspace()


def _workspace(dev: int, nbytes: int, stream: int) -> torch.Tensor:
    """Scratch with zeroed counters, one per (device, stream); inside a stream capture one of the graph's own,
    whose counters the graph zeroes itself, so graphs that replay at the same time do not share it."""
    if torch._C._cuda_isCurrentStreamCapturing():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=_cuda(dev))
        ws[:_COUNTERS].zero_()
        return ws
    return _ws.get(_cuda(dev), nbytes, stream)


@functools.lru_cache(maxsize=256)
def _attention_bytes(dev: int, *sizes: int) -> int:
    """Workspace of an attention call on ``dev`` (the current device), asked once per sizes."""
    return int(N.lib().ti_tree_attention_workspace_bytes(*sizes))


def attention(out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              block_tables: torch.Tensor, context_lens: torch.Tensor, cu_seqlens: torch.Tensor, *,
              masks: torch.Tensor | None = None, row_index: torch.Tensor | None = None,
              lse: torch.Tensor | None = None) -> None:
    """out[t] = softmax(q[t] K^T / sqrt(head_dim)) V for every node t, over the ``context_lens[i]`` cached
    tokens of its sequence and the nodes of its tree that row t of ``masks`` has bits for (int32 [tokens,
    words], bit b of word w: node 32 w + b; itself only if its bit is set).  Without masks a node sees
    the nodes up to itself: the trees are chains, or chunks of a prompt.

    q, out: [tokens, NH, D] bf16 or fp16, D 64 or 128, at most 16 query heads per kv head.  k_cache,
    v_cache: one layer of the pool, [num_blocks, KVH, 16, D]; the nodes' K and V are in it, at positions
    ``context_lens[i]`` and on of table row ``row_index[i]`` (default i) of ``block_tables``.  ``lse``
    (float32 [tokens, NH]) receives the natural log of each row's sum of exp(scores).

    A table entry that is negative or outside the pool holds no tokens.  A node that sees nothing gets
    zeros, and -inf in ``lse``.  What a node does not see, NaN or infinite, does not reach it.  Rows behind
    the last tree are left as they were.  One launch; the same results on every run."""
    dev = _device(out, q, k_cache, v_cache, block_tables, context_lens, cu_seqlens, masks, row_index, lse)
    T, NH, d, q_stride = _rows("q", q)
    out_stride = _out_rows(out, q)
    if T == 1:
        q_stride = out_stride = NH * d              # (a single token's stride means nothing)
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape or shape[2] != BLOCK or shape[3] != d or \
            not k_cache.is_contiguous() or not v_cache.is_contiguous():
        _fail("k_cache and v_cache must be contiguous [num_blocks, num_kv_heads, 16, head_dim]")
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        _fail("q, out and the caches must share a dtype")
    nb, kvh = shape[0], shape[1]
    if d != 64 and d != 128:
        _fail("head_dim must be 64 or 128")
    if nb <= 0 or kvh <= 0 or NH <= 0 or NH % kvh or NH > 16 * kvh:
        _fail("query heads must be a multiple of the kv heads, at most 16 per kv head")
    B = context_lens.numel()
    _index("context_lens", context_lens)
    _index("cu_seqlens", cu_seqlens, B + 1)
    _index("row_index", row_index, B)
    bt_stride, cols = _table("block_tables", block_tables, B if row_index is None else None)
    words = 0
    if masks is not None:
        if masks.dtype != torch.int32 or masks.dim() != 2 or not masks.is_contiguous() or \
                masks.shape[0] != T or masks.shape[1] < 1:
            _fail("masks must be contiguous int32 [tokens, words]")
        words = masks.shape[1]
    if lse is not None:
        _head_sums("lse", lse, T, NH)
    if B == 0 or T == 0:
        return
    lib = N.lib()
    with _on(dev):
        stream = _stream(dev)
        ws = _workspace(dev, _attention_bytes(dev, NH, kvh, d), stream)
        N.check(lib.ti_tree_attention(
            out.data_ptr(), out_stride, _ptr(lse), q.data_ptr(), q_stride, k_cache.data_ptr(),
            v_cache.data_ptr(), nb, block_tables.data_ptr(), bt_stride, block_tables.shape[0], cols,
            _ptr(row_index), context_lens.data_ptr(), cu_seqlens.data_ptr(), B, T, _ptr(masks), words,
            NH, kvh, d, BLOCK, _CODE[q.dtype], ws.data_ptr(), ws.numel(), stream))


def accept(key_cache: torch.Tensor, value_cache: torch.Tensor, tokens: torch.Tensor,
           parents: torch.Tensor, targets: torch.Tensor, cu_seqlens: torch.Tensor,
           slot_mapping: torch.Tensor, num: torch.Tensor, path: torch.Tensor,
           out_tokens: torch.Tensor, *, out_slots: torch.Tensor | None = None,
           seq_lens: torch.Tensor | None = None, row_index: torch.Tensor | None = None) -> None:
    """Walk each tree from node 0: ``targets[c]`` is the token drawn at node c, and the walk goes on to the
    first later node whose parent is c and whose token (``tokens``) is that one, until there is none or
    the path is as long as ``path`` is wide.

    ``num`` [B] receives the path's length (0: the tree has no nodes, or was not run), ``path`` [B, P] its nodes and
    ``out_tokens`` [B, P] the draws at them, the sequence's new tokens: those of the guesses that held
    and the one behind them (-1 behind the path).  All int32; parents and tokens as ``paging.reserve``
    takes them.

    K and V of the path's j-th node move from its slot to that of place j, ``out_slots[cu_seqlens[i] + j]``
    (default: ``slot_mapping`` itself, so that the kept nodes follow the sequence's cached tokens;
    otherwise slots that hold none of the call's nodes; distinct either way), in every layer of ``key_cache`` / ``value_cache``
    [layers, num_blocks, KVH, block_size, D] (or of one layer).  Negative slots are skipped; slots
    outside the pool too, raising TI_DEVERR_BAD_INPUT.  ``seq_lens[row_index[i]]`` (default row i)
    advances by the path's length; where ``seq_lens`` is given, a tree whose node 0 or place 0 has a
    negative slot (``paging.reserve`` did not grant it room) counts as not run: its path is empty, its
    length stays.  Without ``seq_lens`` it is walked all the same, and leaving out what was not granted is
    the caller's part.  At most 1024 places."""
    out_slots = slot_mapping if out_slots is None else out_slots
    dev = _device(key_cache, value_cache, tokens, parents, targets, cu_seqlens, slot_mapping, num, path,
                  out_tokens, out_slots, seq_lens, row_index)
    shape = key_cache.shape
    if len(shape) not in (4, 5) or value_cache.shape != shape or not key_cache.is_contiguous() or \
            not value_cache.is_contiguous():
        _fail("the caches must be contiguous [layers, num_blocks, num_kv_heads, block_size, head_dim] or "
              "one layer of it")
    if key_cache.dtype not in _HALF or value_cache.dtype != key_cache.dtype:
        _fail("the caches must be bf16 or fp16, both the same")
    layers = shape[0] if len(shape) == 5 else 1
    nb, kvh, bs, d = shape[-4:]
    if d % 8:
        _fail("head_dim must be a multiple of 8")
    T, B = tokens.numel(), num.numel()
    for name, t in (("tokens", tokens), ("parents", parents), ("targets", targets)):
        _index(name, t, T)
    _index("num", num)
    _index("cu_seqlens", cu_seqlens, B + 1)
    for name, t in (("slot_mapping", slot_mapping), ("out_slots", out_slots)):
        if t.dtype != torch.int64 or not t.is_contiguous() or t.numel() != T:
            _fail(f"{name} must be contiguous int64 [tokens]")
    if path.dim() != 2 or path.shape[0] != B or path.shape != out_tokens.shape or \
            not 1 <= path.shape[1] <= 1024:
        _fail("path and out_tokens must be [batch, places], 1 to 1024 places")
    _index("path", path)
    _index("out_tokens", out_tokens)
    _index("row_index", row_index, B)
    _index("seq_lens", seq_lens)
    if seq_lens is not None and row_index is None and seq_lens.numel() < B:
        _fail("seq_lens has fewer entries than the batch")
    if B == 0 or layers == 0:
        return
    if min(nb, kvh, bs, d) <= 0:
        _fail("the caches are empty")
    with _on(dev):
        N.check(N.lib().ti_tree_accept(
            key_cache.data_ptr(), value_cache.data_ptr(), layers, nb, kvh, d, bs,
            key_cache.element_size(), tokens.data_ptr(), parents.data_ptr(), targets.data_ptr(),
            cu_seqlens.data_ptr(), B, T, slot_mapping.data_ptr(), out_slots.data_ptr(),
            num.data_ptr(), path.data_ptr(), out_tokens.data_ptr(), path.shape[1], _ptr(seq_lens),
            _ptr(row_index), 0 if seq_lens is None else seq_lens.numel(), _stream(dev)))
