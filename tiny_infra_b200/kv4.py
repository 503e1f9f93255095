"""Operators on a paged KV cache held in 4 bits, and its eviction by attention weight.

The pool is ``[num_blocks, num_kv_heads, 18 * head_dim]`` uint8 (``new_pool``), blocks of 16
tokens, the same block tables and slots as the 16-bit pool: 9/32 of its bytes.  One (block, kv
head) tile holds K codes, V codes, K scales, V scales; a value is an e2m1 code times the scale of
its 16 dims (an unsigned 8-bit float), exact in bf16 and fp16.  ``head_dim`` is 64 or 128.

* ``append``              quantise new tokens' K and V into their slots
* ``dequantize``          read cached tokens back as 16-bit values
* ``decode_attention``    one query token per sequence (out, and log-sum-exp on request)
* ``prefill_attention``   ragged causal chunks (``PrefillPlan`` holds their layout)
* ``accumulate_weights``  add each cached token's attention weight to its running total
* ``evict``               keep the recent tokens and the heaviest older ones, moved to the front

A block-table entry that is negative or outside the pool holds no tokens.  Every call runs on the
current CUDA stream of its tensors' device; argument errors raise ``RuntimeError`` before anything
is launched.
"""
from __future__ import annotations

import contextlib

import numpy as np
import torch

from . import _native as N

BLOCK = 16
_ws = N.Workspace()


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _cuda(**tensors) -> None:
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        _check(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
        dev = t.device if dev is None else dev
        _check(t.device == dev, f"{name} is on {t.device}, other tensors on {dev}")


def _on(t: torch.Tensor):
    """Launches go to the current device: make it the tensors' one."""
    if t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _pool_shape(pool: torch.Tensor, head_dim: int | None = None):
    _check(pool.dtype == torch.uint8 and pool.dim() == 3 and pool.is_contiguous(),
           "pool must be a contiguous uint8 [num_blocks, num_kv_heads, 18 * head_dim] tensor")
    nb, kvh, tile = pool.shape
    d = tile // 18
    _check(tile in (18 * 64, 18 * 128), "pool tiles must be 18 * head_dim bytes, head_dim 64 or 128")
    _check(head_dim is None or d == head_dim, "head_dim does not match the pool's tiles")
    _check(nb > 0 and kvh > 0, "the pool is empty")
    return nb, kvh, d


def _index(name: str, t: torch.Tensor | None, numel: int | None = None) -> None:
    if t is None:
        return
    _check(t.dtype == torch.int32 and t.is_contiguous(), f"{name} must be contiguous int32")
    _check(numel is None or t.numel() == numel, f"{name} must have {numel} entries")


def _table(name: str, t: torch.Tensor, rows: int | None) -> None:
    _check(t.dtype == torch.int32 and t.dim() == 2 and (t.shape[1] <= 1 or t.stride(1) == 1),
           f"{name} must be int32 [rows, max_blocks] with contiguous rows")
    _check(t.shape[1] > 0, f"{name} has no columns")
    _check(rows is None or t.shape[0] >= rows, f"{name} has fewer rows than the batch")


def _rows(name: str, t: torch.Tensor) -> None:
    """[T, heads, D] of a 16-bit type, each token's heads contiguous."""
    _check(t.dim() == 3 and t.dtype in (torch.bfloat16, torch.float16),
           f"{name} must be bf16 or fp16 [tokens, heads, head_dim]")
    _check(t.numel() == 0 or (t.stride(2) == 1 and t.stride(1) == t.shape[2]),
           f"{name} must have contiguous [heads, head_dim] rows")


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def tile_bytes(head_dim: int) -> int:
    """Bytes of one (block, kv head): 16 tokens' K and V codes and scales."""
    n = int(N.lib().ti_kv4_tile_bytes(int(head_dim)))
    _check(n > 0, "head_dim must be 64 or 128")
    return n


def new_pool(num_blocks: int, num_kv_heads: int, head_dim: int, *, num_layers: int | None = None,
             device="cuda") -> torch.Tensor:
    """A zeroed pool (of one layer, or [num_layers, ...])."""
    shape = (num_blocks, num_kv_heads, tile_bytes(head_dim))
    return torch.zeros(shape if num_layers is None else (num_layers, *shape), dtype=torch.uint8,
                       device=device)


def append(pool: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor, *,
           weights: torch.Tensor | None = None) -> None:
    """Quantise K and V [T, KVH, D] (bf16 or fp16, any token and head strides that are multiples
    of 8 elements) into slots ``slot_mapping`` [T] int64 = block * 16 + offset.  A negative slot
    skips its token; a slot outside the pool is not written and raises TI_DEVERR_BAD_INPUT; the
    slots of a call are distinct.  With ``weights`` (float32 [num_blocks, KVH, 16]) the new tokens'
    attention-weight totals become zero.  A group of 16 dims with a NaN or an infinity becomes NaN;
    magnitudes above 61440 saturate."""
    _cuda(pool=pool, k=k, v=v, slot_mapping=slot_mapping, weights=weights)
    _check(k.dim() == 3 and v.shape == k.shape and k.dtype == v.dtype and
           k.dtype in (torch.bfloat16, torch.float16),
           "k and v must be [tokens, num_kv_heads, head_dim] of the same 16-bit dtype")
    nb, kvh, d = _pool_shape(pool, k.shape[2])
    _check(k.shape[1] == kvh, "k and v do not have the pool's kv heads")
    _check(slot_mapping.dtype == torch.int64 and slot_mapping.is_contiguous() and
           slot_mapping.numel() == k.shape[0], "slot_mapping must be contiguous int64 [tokens]")
    _weights("weights", weights, nb, kvh)
    if k.shape[0] == 0:
        return
    _check(k.stride(2) == 1 and v.stride(2) == 1, "k and v must have contiguous head_dim")
    with _on(pool):
        N.check(N.lib().ti_kv4_append(
            pool.data_ptr(), _ptr(weights), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
            v.stride(0), v.stride(1), slot_mapping.data_ptr(), k.shape[0], nb, kvh, d, BLOCK,
            N.dtype_code(k.dtype), N.stream_of(pool)))


def _weights(name: str, w: torch.Tensor | None, nb: int, kvh: int) -> None:
    if w is not None:
        _check(w.dtype == torch.float32 and w.is_contiguous() and
               tuple(w.shape) == (nb, kvh, BLOCK),
               f"{name} must be contiguous float32 [num_blocks, num_kv_heads, 16]")


def dequantize(pool: torch.Tensor, block_tables: torch.Tensor, lens: torch.Tensor,
               out_tables: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor, *,
               row_index: torch.Tensor | None = None) -> None:
    """Read the first ``lens[r]`` tokens of each table row back into 16-bit pools ``k_out`` /
    ``v_out`` [out_blocks, KVH, 16, D]: block j of row r goes to block ``out_tables[r, j]`` (a
    negative entry skips it), zeros behind the row's length and where the source entry holds no
    block.  ``row_index`` selects the rows of ``block_tables``.  The target blocks are distinct."""
    _cuda(pool=pool, block_tables=block_tables, lens=lens, out_tables=out_tables, k_out=k_out,
          v_out=v_out, row_index=row_index)
    nb, kvh, d = _pool_shape(pool)
    _check(k_out.dim() == 4 and k_out.shape == v_out.shape and k_out.dtype == v_out.dtype and
           k_out.dtype in (torch.bfloat16, torch.float16) and k_out.is_contiguous() and
           v_out.is_contiguous() and tuple(k_out.shape[1:]) == (kvh, BLOCK, d),
           "k_out and v_out must be contiguous 16-bit [out_blocks, num_kv_heads, 16, head_dim]")
    rows = lens.numel()
    _index("lens", lens)
    _index("row_index", row_index, rows)
    _table("out_tables", out_tables, rows)
    _table("block_tables", block_tables, rows if row_index is None else None)
    _check(block_tables.shape[1] >= out_tables.shape[1], "block_tables is narrower than out_tables")
    if rows == 0 or k_out.shape[0] == 0:
        return
    with _on(pool):
        N.check(N.lib().ti_kv4_dequantize(
            k_out.data_ptr(), v_out.data_ptr(), k_out.shape[0], pool.data_ptr(), nb,
            block_tables.data_ptr(), block_tables.stride(0), _ptr(row_index), lens.data_ptr(),
            out_tables.data_ptr(), out_tables.stride(0), rows, out_tables.shape[1], kvh, d, BLOCK,
            N.dtype_code(k_out.dtype), N.stream_of(pool)))


def _workspace(device: torch.device, nbytes: int, stream: int) -> torch.Tensor:
    """Zeroed scratch, one per (device, stream); inside a stream capture one of the graph's own
    (so graphs that replay at the same time do not share it), zeroed by the graph itself."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)
    return _ws.get(device, nbytes, stream)


def _batch(q, pool, block_tables, context_lens, row_index):
    _rows("q", q)
    nb, kvh, d = _pool_shape(pool, q.shape[2])
    B, NH, _ = q.shape
    _check(NH > 0 and NH % kvh == 0 and NH // kvh <= 16,
           "query heads must be a multiple of the kv heads, at most 16 per kv head")
    _index("context_lens", context_lens, B)
    _index("row_index", row_index, B)
    _table("block_tables", block_tables, B if row_index is None else None)
    return B, NH, nb, kvh, d


def decode_attention(out: torch.Tensor, q: torch.Tensor, pool: torch.Tensor,
                     block_tables: torch.Tensor, context_lens: torch.Tensor, *,
                     row_index: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None) -> None:
    """Single-query attention, scale 1/sqrt(head_dim): out[b] = softmax(q[b] K^T) V over the first
    ``context_lens[b]`` cached tokens of row ``row_index[b]`` (default b) of ``block_tables``.

    q, out: [B, NH, D] bf16 or fp16, at most 16 query heads per kv head, B at most 4096.  ``lse``
    (float32 [B, NH]) receives the natural log of each row's sum of exp(scores).  A sequence of
    length 0 leaves its rows of ``out`` and ``lse`` as they were; one whose table holds no block
    gets NaN, and -inf in ``lse``.  One launch; results do not depend on the batch's other rows'
    contents and are the same on every run."""
    _cuda(out=out, q=q, pool=pool, block_tables=block_tables, context_lens=context_lens,
          row_index=row_index, lse=lse)
    B, NH, nb, kvh, d = _batch(q, pool, block_tables, context_lens, row_index)
    _rows("out", out)
    _check(out.shape == q.shape and out.dtype == q.dtype, "out must have q's shape and dtype")
    if lse is not None:
        _check(lse.dtype == torch.float32 and lse.is_contiguous() and lse.numel() == B * NH,
               "lse must be contiguous float32 [batch, heads]")
    if B == 0:
        return
    lib = N.lib()
    with _on(pool):
        stream = N.stream_of(pool)
        need = lib.ti_kv4_attention_workspace_bytes(B, NH, kvh, d, block_tables.shape[1])
        ws = _workspace(pool.device, need, stream)
        N.check(lib.ti_kv4_attention_decode(
            out.data_ptr(), out.stride(0), _ptr(lse), q.data_ptr(), q.stride(0), pool.data_ptr(),
            nb, block_tables.data_ptr(), block_tables.stride(0), _ptr(row_index),
            context_lens.data_ptr(), B, NH, kvh, d, BLOCK, block_tables.shape[1],
            N.dtype_code(q.dtype), ws.data_ptr(), ws.numel(), stream))


def accumulate_weights(weights: torch.Tensor, q: torch.Tensor, lse: torch.Tensor,
                       pool: torch.Tensor, block_tables: torch.Tensor,
                       context_lens: torch.Tensor, *, row_index: torch.Tensor | None = None,
                       out: torch.Tensor | None = None) -> None:
    """Add to each cached token's total the attention weight that ``q`` gives it, summed over the
    query heads of its kv head: out = weights + sum_h exp(q_h . k / sqrt(D) - lse_h).

    ``lse`` float32 [B, NH] as ``decode_attention`` gives it for the same arguments; weights and
    out (default: weights itself) float32 [num_blocks, KVH, 16], of which only the sequences' own
    tokens are read and written.  The sequences of a call share no block."""
    _cuda(weights=weights, q=q, lse=lse, pool=pool, block_tables=block_tables,
          context_lens=context_lens, row_index=row_index, out=out)
    out = weights if out is None else out
    B, NH, nb, kvh, d = _batch(q, pool, block_tables, context_lens, row_index)
    _weights("weights", weights, nb, kvh)
    _weights("out", out, nb, kvh)
    _check(lse.dtype == torch.float32 and lse.is_contiguous() and lse.numel() == B * NH,
           "lse must be contiguous float32 [batch, heads]")
    if B == 0:
        return
    with _on(pool):
        N.check(N.lib().ti_kv4_accumulate_weights(
            out.data_ptr(), weights.data_ptr(), q.data_ptr(), q.stride(0), lse.data_ptr(),
            pool.data_ptr(), nb, block_tables.data_ptr(), block_tables.stride(0), _ptr(row_index),
            context_lens.data_ptr(), B, NH, kvh, d, BLOCK, block_tables.shape[1],
            N.dtype_code(q.dtype), N.stream_of(pool)))


class PrefillPlan:
    """Layout of a packed prefill: chunk i holds ``counts[i]`` query tokens at positions
    ``starts[i]`` and on, whose K and V are already in the cache.  Built once per batch, used by
    every layer; it holds the query tiles (16 tokens, longest prefix first) and where the cached
    tokens are read back to."""

    def __init__(self, starts, counts, device="cuda") -> None:
        starts, counts = np.asarray(starts, np.int64), np.asarray(counts, np.int64)
        _check(starts.ndim == 1 and starts.shape == counts.shape, "starts and counts must match")
        _check(bool((starts >= 0).all() and (counts >= 0).all()), "starts and counts must be >= 0")
        lens = np.where(counts > 0, starts + counts, 0)
        blocks = -(-lens // BLOCK)
        _check(int(lens.max(initial=0)) < 2 ** 31 and int(blocks.sum()) < 2 ** 31,
               "prefill too long")
        self.num_seqs, self.num_tokens = len(starts), int(counts.sum())
        self.max_blocks = int(blocks.max(initial=0))
        self.scratch_blocks = int(blocks.sum())
        seq, q0, work = [], [], []
        for i, (s, n) in enumerate(zip(starts.tolist(), counts.tolist())):
            for t in range(0, n, 16):
                seq.append(i)
                q0.append(t)
                work.append(s + min(t + 16, n))
        order = np.argsort(-np.asarray(work, np.int64), kind="stable")
        self.num_tiles = len(seq)
        at = np.concatenate([[0], np.cumsum(blocks)[:-1]]) if len(starts) else blocks
        col = np.arange(max(self.max_blocks, 1))
        tables = np.where(col < blocks[:, None], at[:, None] + col, -1)

        def dev(a):
            return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)

        self.start_pos, self.lens = dev(starts), dev(lens)
        self.rows = dev(np.arange(self.num_seqs))
        self.cu_seqlens = dev(np.concatenate([[0], np.cumsum(counts)]))
        self.tile_seq, self.tile_q0 = dev(np.asarray(seq)[order]), dev(np.asarray(q0)[order])
        self.tables = dev(tables.reshape(self.num_seqs, max(self.max_blocks, 1)))


def prefill_attention(out: torch.Tensor, q: torch.Tensor, pool: torch.Tensor,
                      block_tables: torch.Tensor, plan: PrefillPlan, *,
                      row_index: torch.Tensor | None = None) -> None:
    """Causal attention of the plan's query tokens (q, out [tokens, NH, D]) over their sequences'
    cached tokens, positions 0 .. their own, scale 1/sqrt(D).

    The cached values are exact in 16 bits, so they are read back once (``dequantize``, 2 *
    scratch_blocks * KVH * 16 * D values of scratch) and the 16-bit pool's tensor-core prefill
    kernel runs on them; the read-back is a few per cent of a chunk's attention."""
    _cuda(out=out, q=q, pool=pool, block_tables=block_tables, start_pos=plan.start_pos,
          row_index=row_index)
    _rows("q", q)
    _rows("out", out)
    nb, kvh, d = _pool_shape(pool, q.shape[2])
    T, NH, _ = q.shape
    _check(out.shape == q.shape and out.dtype == q.dtype, "out must have q's shape and dtype")
    _check(NH > 0 and NH % kvh == 0 and NH // kvh <= 16,
           "query heads must be a multiple of the kv heads, at most 16 per kv head")
    _check(T == plan.num_tokens, "q does not have the plan's tokens")
    _index("row_index", row_index, plan.num_seqs)
    _table("block_tables", block_tables, plan.num_seqs if row_index is None else None)
    _check(block_tables.shape[1] >= plan.max_blocks, "block_tables is too narrow for the plan")
    if plan.num_tiles == 0:
        return
    shape = (plan.scratch_blocks, kvh, BLOCK, d)
    with _on(pool):
        k = torch.empty(shape, dtype=q.dtype, device=pool.device)
        v = torch.empty(shape, dtype=q.dtype, device=pool.device)
        dequantize(pool, block_tables, plan.lens, plan.tables, k, v, row_index=row_index)
        N.check(N.lib().ti_paged_prefill_attention(
            out.data_ptr(), out.stride(0), q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(),
            plan.scratch_blocks, plan.tables.data_ptr(), plan.tables.stride(0),
            plan.rows.data_ptr(), plan.start_pos.data_ptr(), plan.cu_seqlens.data_ptr(), plan.tile_seq.data_ptr(),
            plan.tile_q0.data_ptr(), plan.num_tiles, NH, kvh, d, BLOCK, N.dtype_code(q.dtype),
            N.stream_of(pool)))


def evict(pool: torch.Tensor, weights: torch.Tensor, block_tables: torch.Tensor,
          context_lens: torch.Tensor, keep: int, recent: int, *,
          row_index: torch.Tensor | None = None, out_block_tables: torch.Tensor | None = None,
          kept: torch.Tensor | None = None) -> None:
    """Bring every sequence longer than ``keep`` tokens down to ``keep``, for every layer and kv
    head on its own: the last ``recent`` tokens stay and the heaviest ``keep - recent`` of the
    older ones by ``weights`` (equal weights: the earlier token; NaN counts as the heaviest), in
    their order, moved with their totals to positions 0 .. keep-1.

    pool [num_blocks, KVH, 18 D] or [layers, num_blocks, KVH, 18 D], weights the same with 16 in
    place of 18 D, float32.  The survivors go to the blocks of ``out_block_tables`` (rows as
    ``block_tables``'; default: the same blocks, in place; otherwise blocks that hold none of the
    call's tokens).  ``kept`` (int32 [layers, B, KVH, >= keep]) receives their old positions.  The
    caller shortens the lengths to min(context_lens, keep) and frees the blocks behind.  A sequence
    with a needed table entry outside the pool is left as it is and raises TI_DEVERR_BAD_INPUT.
    The sequences of a call share no block."""
    _cuda(pool=pool, weights=weights, block_tables=block_tables, context_lens=context_lens,
          row_index=row_index, out_block_tables=out_block_tables, kept=kept)
    _check(pool.dim() in (3, 4), "pool must be [num_blocks, KVH, 18 D] or [layers, ...]")
    layers = pool.shape[0] if pool.dim() == 4 else 1
    if layers == 0:
        return
    _check(pool.is_contiguous(), "pool must be contiguous")
    nb, kvh, d = _pool_shape(pool[0] if pool.dim() == 4 else pool)
    _check(weights.dtype == torch.float32 and weights.is_contiguous() and
           tuple(weights.shape) == (*pool.shape[:-1], BLOCK),
           "weights must be contiguous float32, the pool's shape with 16 in the last place")
    keep, recent = int(keep), int(recent)
    _check(keep >= 1 and 0 <= recent <= keep, "needs keep >= 1 and 0 <= recent <= keep")
    B = context_lens.numel()
    _index("context_lens", context_lens)
    _index("row_index", row_index, B)
    _table("block_tables", block_tables, B if row_index is None else None)
    to = block_tables if out_block_tables is None else out_block_tables
    _table("out_block_tables", to, B if row_index is None else block_tables.shape[0])
    if kept is not None:
        _check(kept.dtype == torch.int32 and kept.is_contiguous() and kept.dim() == 4 and
               tuple(kept.shape[:3]) == (layers, B, kvh) and kept.shape[3] >= keep,
               "kept must be contiguous int32 [layers, batch, num_kv_heads, >= keep]")
    if B == 0:
        return
    with _on(pool):
        N.check(N.lib().ti_kv4_evict(
            pool.data_ptr(), weights.data_ptr(), layers, nb, block_tables.data_ptr(),
            block_tables.stride(0), to.data_ptr(), to.stride(0), _ptr(row_index),
            context_lens.data_ptr(), B, block_tables.shape[1], to.shape[1], keep, recent,
            _ptr(kept), kept.shape[3] if kept is not None else 0, kvh, d, BLOCK,
            N.stream_of(pool)))
