"""Block tables and slots of the paged cache built on the device, from lengths that are there.

The host allocator (``cache_manager.BlockAllocator``) needs every length on the host; these calls keep a
step whose lengths the GPU itself decides (accepted drafts, say) free of a round trip.  They hand out
the blocks that the host allocator would: from the front of a FIFO list, a sequence's in ascending order,
sequence by sequence; freed ones go to its end.

The free list is an int32 tensor ``[2 + n]``: the place of its first entry, how many it has, and a ring of
n block ids (``new_free_list``, ``free_list``; ``free_ids`` reads it back).

* ``reserve``  blocks, slots and positions of new tokens; for drafted trees their masks too
* ``release``  give the blocks behind each row's kept tokens back

Every call runs on the current CUDA stream of its tensors' device; argument errors raise
``RuntimeError`` before anything is launched.
"""
from __future__ import annotations

import torch

from . import _native as N
from .kv4 import _device, _fail, _index, _on, _ptr, _stream, _table

_MOST_SEQS, _MOST_ROWS = 4096, 32768


def free_list(ids, capacity: int | None = None, device="cuda") -> torch.Tensor:
    """The free list that holds these block ids, first one first, with room for ``capacity`` in all
    (default: as many as there are)."""
    ids = [int(i) for i in ids]
    capacity = len(ids) if capacity is None else int(capacity)
    if capacity < max(1, len(ids)):
        _fail("the free list needs room for its entries, and for one at least")
    if any(not 0 <= i < 2 ** 31 for i in ids):
        _fail("block ids must be >= 0")
    ring = torch.zeros(2 + capacity, dtype=torch.int32)
    ring[1] = len(ids)
    if ids:
        ring[2:2 + len(ids)] = torch.tensor(ids, dtype=torch.int32)
    return ring.to(device)


def new_free_list(num_blocks: int, device="cuda") -> torch.Tensor:
    """The free list of a pool whose blocks are all free."""
    return free_list(range(int(num_blocks)), device=device)


def free_ids(ring: torch.Tensor) -> list[int]:
    """The free block ids in the order in which they will be handed out (waits for the device)."""
    r = ring.cpu().tolist()
    head, have, ids = r[0], r[1], r[2:]
    return [ids[(head + i) % len(ids)] for i in range(have)]


def _ring(ring: torch.Tensor) -> int:
    if ring.dtype != torch.int32 or ring.dim() != 1 or not ring.is_contiguous() or ring.numel() < 3:
        _fail("the free list must be contiguous int32 [2 + entries]")
    return ring.numel() - 2


def _rows(block_tables, row_index, seqs: int) -> tuple[int, int]:
    """(row stride, columns) of the block tables of ``seqs`` sequences."""
    stride, cols = _table("block_tables", block_tables, seqs if row_index is None else None)
    rows = block_tables.shape[0]
    if rows > 1 and stride < cols:
        _fail("block_tables' rows overlap")
    if seqs > _MOST_SEQS:
        _fail(f"at most {_MOST_SEQS} sequences a call")
    if row_index is not None:
        if rows > _MOST_ROWS:
            _fail(f"at most {_MOST_ROWS} table rows with row_index")
        _index("row_index", row_index, seqs)
    return stride, cols


def reserve(block_tables: torch.Tensor, seq_lens: torch.Tensor, counts: torch.Tensor,
            ring: torch.Tensor, slot_mapping: torch.Tensor, positions: torch.Tensor,
            cu_seqlens: torch.Tensor, *, block_size: int = 16, row_index: torch.Tensor | None = None,
            granted: torch.Tensor | None = None, pos_offset: torch.Tensor | None = None,
            parents: torch.Tensor | None = None, masks: torch.Tensor | None = None) -> None:
    """Room for ``counts[i]`` new tokens of sequence i behind the ``seq_lens[row]`` cached ones of its
    table row (``row_index[i]``, default i; a negative row is padding).

    Unassigned (negative) entries of ``block_tables`` that the new tokens fall in take blocks from the
    front of ``ring``, sequence by sequence.  The first sequence that needs more than what is left gets
    none, nor does any later one that needs a block; ``granted`` [B] receives each one's tokens, its
    count or 0.  What the step computes for tokens that were not granted means nothing (they have no K
    and V): their rows are to be left out, as ``tree.accept`` does where it keeps the lengths.  A sequence that would pass its row's end, and one whose row an earlier sequence has, get
    none and raise TI_DEVERR_BAD_INPUT.

    ``cu_seqlens`` [B + 1] receives the counts' running sum, granted or not.  ``slot_mapping`` int64 and
    ``positions`` int32, of one length, receive the packed tokens' pool slots (block * block_size +
    offset; -1: not granted) and positions: length + index within the sequence (+ ``pos_offset[row]``).
    Places behind the last token get slot -1, position 0.

    Drafted trees: ``parents`` int32, as long as ``slot_mapping``, holds each token's parent as an index
    within its tree (negative: a root), an earlier one.  A token's position then goes by its depth, and
    row t of ``masks`` (int32 [tokens, words], bit b of word w: node 32 w + b) receives its ancestors
    and itself, as ``tree.attention`` takes them.  A tree with more nodes than bits raises
    TI_DEVERR_BAD_INPUT and loses the bits.  Each token walks up to its root, a dependent load per ancestor,
    again for every four words of ``masks``: trees of up to some hundred levels are what this is for.

    ``seq_lens`` is not advanced; blocks reserved once stay in the row.  At most 4096 sequences, 32768 table
    rows with ``row_index``.  Calls that share a ring or a table follow one another."""
    dev = _device(block_tables, seq_lens, counts, ring, slot_mapping, positions, cu_seqlens, row_index,
                  granted, pos_offset, parents, masks)
    B = counts.numel()
    size = _ring(ring)
    bt_stride, cols = _rows(block_tables, row_index, B)
    rows = block_tables.shape[0]
    _index("counts", counts)
    _index("cu_seqlens", cu_seqlens, B + 1)
    _index("granted", granted, B)
    for name, t in (("seq_lens", seq_lens), ("pos_offset", pos_offset)):
        _index(name, t)
        if t is not None and t.numel() < (B if row_index is None else rows):
            _fail(f"{name} has fewer entries than the batch or the table")
    cap = slot_mapping.numel()
    if slot_mapping.dtype != torch.int64 or not slot_mapping.is_contiguous():
        _fail("slot_mapping must be contiguous int64")
    _index("positions", positions, cap)
    _index("parents", parents, cap)
    if block_size < 1:
        _fail("block_size must be positive")
    words = 0
    if masks is not None:
        if parents is None:
            _fail("masks go with parents")
        if masks.dtype != torch.int32 or masks.dim() != 2 or not masks.is_contiguous() or \
                masks.shape[0] != cap or masks.shape[1] < 1:
            _fail("masks must be contiguous int32 [tokens, words]")
        words = masks.shape[1]
    if B == 0 and cap == 0:
        return
    with _on(dev):
        if granted is None:
            granted = torch.empty_like(counts)
        N.check(N.lib().ti_reserve_slots(
            block_tables.data_ptr(), bt_stride, rows, cols, block_size, _ptr(row_index),
            seq_lens.data_ptr(), _ptr(pos_offset), counts.data_ptr(), B, ring.data_ptr(), size,
            slot_mapping.data_ptr(), positions.data_ptr(), cap, cu_seqlens.data_ptr(),
            granted.data_ptr(), _ptr(parents), _ptr(masks), words, _stream(dev)))


def release(block_tables: torch.Tensor, keep_lens: torch.Tensor, ring: torch.Tensor, *,
            block_size: int = 16, row_index: torch.Tensor | None = None) -> None:
    """Give back the blocks that sequence i does not need for its first ``keep_lens[i]`` tokens (0: all
    of them): the entries behind become -1, the blocks go to the end of ``ring``, row by row, in
    ascending order within a row.  Rows as in ``reserve``; a row named twice is released once.  Blocks
    beyond the ring's room leave everything as it was and raise TI_DEVERR_BAD_INPUT."""
    dev = _device(block_tables, keep_lens, ring, row_index)
    B = keep_lens.numel()
    size = _ring(ring)
    bt_stride, cols = _rows(block_tables, row_index, B)
    _index("keep_lens", keep_lens)
    if block_size < 1:
        _fail("block_size must be positive")
    if B == 0:
        return
    with _on(dev):
        N.check(N.lib().ti_release_blocks(
            block_tables.data_ptr(), bt_stride, block_tables.shape[0], cols, block_size,
            _ptr(row_index), keep_lens.data_ptr(), B, ring.data_ptr(), size, _stream(dev)))
