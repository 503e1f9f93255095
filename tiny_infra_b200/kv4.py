"""Operators on a paged KV cache held in 4 bits, and its eviction by attention weight.

The pool is ``[num_blocks, num_kv_heads, 18 * head_dim]`` uint8 (``new_pool``), blocks of 16
tokens, the same block tables and slots as the 16-bit pool: 9/32 of its bytes.  One (block, kv
head) tile holds K codes, V codes, K scales, V scales; a value is an e2m1 code times the scale of
its 16 dims (an unsigned 8-bit float), exact in bf16 and fp16.  ``head_dim`` is 64 or 128.

* ``append``              quantise new tokens' K and V into their slots
* ``rope_append``         the same from the fused projection's rows, rotating q and k first
* ``dequantize``          read cached tokens back as 16-bit values
* ``decode_attention``    one query token per sequence (out, and log-sum-exp on request)
* ``prefill_attention``   ragged causal chunks (``PrefillPlan`` holds their layout)
* ``accumulate_weights``  add each cached token's attention weight to its running total
* ``evict``               keep the recent tokens and the heaviest older ones, moved to the front

A block-table entry that is negative or outside the pool holds no tokens; entries of ``row_index``
are rows of the block table.  Every call runs on the
current CUDA stream of its tensors' device; argument errors raise ``RuntimeError`` before anything
is launched.
"""
from __future__ import annotations

import contextlib
import functools

import numpy as np
import torch

from . import _native as N

BLOCK = 16
_MOST = 2 ** 31 - 1
_HALF = (torch.bfloat16, torch.float16)
_CODE = {t: N.dtype_code(t) for t in _HALF}
_ws = N.Workspace()


# The checks below run on every call, in front of kernels of a few microseconds: plain conditions
# on cheap attributes, messages built only when they fail.
def _fail(msg: str) -> None:
    raise RuntimeError(msg)


def _device(*tensors) -> int:
    """The CUDA device index that all the tensors (None: absent) are on."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _fail(f"all tensors must be on one CUDA device, not {t.device} and {tensors[0].device}")
    if dev < 0:
        _fail("pool and the other arguments must be CUDA tensors")
    return dev


def _on(dev: int):
    """Launches go to the current device: make it the tensors' one."""
    return _HERE if dev == torch._C._cuda_getDevice() else torch.cuda.device(dev)


_HERE = contextlib.nullcontext()
_stream = torch._C._cuda_getCurrentRawStream


def _pool_shape(pool: torch.Tensor, layered: bool = False):
    shape = pool.shape
    if pool.dtype != torch.uint8 or not pool.is_contiguous() or \
            not (len(shape) == 3 or layered and len(shape) == 4):
        _fail("pool must be a contiguous uint8 [num_blocks, num_kv_heads, 18 * head_dim] tensor"
              + (" or [layers, ...]" if layered else ""))
    nb, kvh, tile = shape if len(shape) == 3 else shape[1:]
    if tile != 1152 and tile != 2304:
        _fail("pool tiles must be 18 * head_dim bytes, head_dim 64 or 128")
    if nb <= 0 or kvh <= 0:
        _fail("the pool is empty")
    return nb, kvh, tile // 18


def _index(name: str, t: torch.Tensor | None, numel: int | None = None) -> None:
    if t is None:
        return
    if t.dtype != torch.int32 or not t.is_contiguous():
        _fail(f"{name} must be contiguous int32")
    if numel is not None and t.numel() != numel:
        _fail(f"{name} must have {numel} entries")


def _table(name: str, t: torch.Tensor, rows: int | None):
    """(row stride, columns) of a block table."""
    shape = t.shape
    if t.dtype != torch.int32 or len(shape) != 2:
        _fail(f"{name} must be int32 [rows, max_blocks]")
    n, cols = shape
    if cols <= 0:
        _fail(f"{name} has no columns")
    stride, inner = t.stride()
    if inner != 1 and cols > 1:
        _fail(f"{name} must have contiguous rows")
    if rows is not None and n < rows:
        _fail(f"{name} has fewer rows than the batch")
    return stride, cols


def _rows(name: str, t: torch.Tensor):
    """Shape and token stride of a [T, heads, D] tensor of a 16-bit type whose tokens' heads are
    contiguous."""
    shape = t.shape
    if len(shape) != 3 or t.dtype not in _HALF:
        _fail(f"{name} must be bf16 or fp16 [tokens, heads, head_dim]")
    T, heads, d = shape
    tok, head, inner = t.stride()
    if (inner != 1 or (head != d and heads > 1)) and T * heads * d:
        _fail(f"{name} must have contiguous [heads, head_dim] rows")
    return T, heads, d, tok


def _out_rows(out: torch.Tensor, q: torch.Tensor) -> int:
    """Token stride of an output of q's shape whose rows do not overlap."""
    if out.shape != q.shape or out.dtype != q.dtype:
        _fail("out must have q's shape and dtype")
    T, heads, d = q.shape
    tok, head, inner = out.stride()
    if (inner != 1 or (head != d and heads > 1)) and T * heads * d:
        _fail("out must have contiguous [heads, head_dim] rows")
    if T > 1 and tok < heads * d:
        _fail("out's rows overlap")
    return tok


def _attention(q, pool, block_tables, context_lens, row_index):
    """Checks shared by the calls that take one query token per sequence."""
    nb, kvh, d = _pool_shape(pool)
    B, NH, dq, q_stride = _rows("q", q)
    if dq != d:
        _fail("head_dim does not match the pool's tiles")
    if NH <= 0 or NH % kvh or NH > 16 * kvh:
        _fail("query heads must be a multiple of the kv heads, at most 16 per kv head")
    _index("context_lens", context_lens, B)
    _index("row_index", row_index, B)
    bt_stride, cols = _table("block_tables", block_tables, B if row_index is None else None)
    return B, NH, nb, kvh, d, q_stride, bt_stride, cols


def _head_sums(name: str, t: torch.Tensor, B: int, NH: int) -> None:
    if t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != B * NH:
        _fail(f"{name} must be contiguous float32 [batch, heads]")


def _totals(name: str, w: torch.Tensor | None, nb: int, kvh: int) -> None:
    if w is not None and (w.dtype != torch.float32 or not w.is_contiguous() or
                          w.shape != (nb, kvh, BLOCK)):
        _fail(f"{name} must be contiguous float32 [num_blocks, num_kv_heads, 16]")


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def tile_bytes(head_dim: int) -> int:
    """Bytes of one (block, kv head): 16 tokens' K and V codes and scales."""
    n = int(N.lib().ti_kv4_tile_bytes(int(head_dim)))
    if n <= 0:
        _fail("head_dim must be 64 or 128")
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
    dev = _device(pool, k, v, slot_mapping, weights)
    nb, kvh, d = _pool_shape(pool)
    if k.dim() != 3 or v.shape != k.shape or k.dtype != v.dtype or k.dtype not in _HALF:
        _fail("k and v must be [tokens, num_kv_heads, head_dim] of the same 16-bit dtype")
    T, heads, dk = k.shape
    if heads != kvh or dk != d:
        _fail("k and v do not have the pool's kv heads and head_dim")
    if slot_mapping.dtype != torch.int64 or not slot_mapping.is_contiguous() or \
            slot_mapping.numel() != T:
        _fail("slot_mapping must be contiguous int64 [tokens]")
    _totals("weights", weights, nb, kvh)
    if T == 0:
        return
    k_tok, k_head, k_in = k.stride()
    v_tok, v_head, v_in = v.stride()
    if k_in != 1 or v_in != 1:
        _fail("k and v must have contiguous head_dim")
    with _on(dev):
        N.check(N.lib().ti_kv4_append(
            pool.data_ptr(), _ptr(weights), k.data_ptr(), k_tok, k_head, v.data_ptr(), v_tok,
            v_head, slot_mapping.data_ptr(), T, nb, kvh, d, BLOCK, _CODE[k.dtype],
            _stream(dev)))


def rope_append(pool: torch.Tensor, qkv: torch.Tensor, num_heads: int,
                slot_mapping: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                positions: torch.Tensor, *, weights: torch.Tensor | None = None) -> None:
    """Rows [q | k | v] of the fused projection, ``qkv`` [T, (num_heads + 2 KVH) * D]: rotate q and k
    in place (rotate-half, tables ``cos`` / ``sin`` float32 [*, D/2], ``positions`` int32 [T]) and
    ``append`` the rotated k and v.  A token whose position is not in the tables is left alone and
    raises TI_DEVERR_BAD_INPUT."""
    dev = _device(pool, qkv, slot_mapping, cos, sin, positions, weights)
    nb, kvh, d = _pool_shape(pool)
    if qkv.dim() != 2 or qkv.dtype not in _HALF or num_heads <= 0 or \
            qkv.shape[1] != (num_heads + 2 * kvh) * d or (qkv.numel() and qkv.stride(1) != 1):
        _fail("qkv must be 16-bit [tokens, (num_heads + 2 * kv heads) * head_dim] rows")
    T = qkv.shape[0]
    if T > 1 and qkv.stride(0) < qkv.shape[1]:
        _fail("qkv's rows overlap")
    if slot_mapping.dtype != torch.int64 or not slot_mapping.is_contiguous() or \
            slot_mapping.numel() != T:
        _fail("slot_mapping must be contiguous int64 [tokens]")
    _index("positions", positions, T)
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != d // 2 or \
                not t.is_contiguous():
            _fail(f"{name} must be contiguous float32 [positions, head_dim / 2]")
    _totals("weights", weights, nb, kvh)
    if T == 0:
        return
    with _on(dev):
        N.check(N.lib().ti_rope_kv4_append(
            qkv.data_ptr(), qkv.stride(0), pool.data_ptr(), _ptr(weights), slot_mapping.data_ptr(),
            cos.data_ptr(), sin.data_ptr(), min(len(cos), len(sin)), positions.data_ptr(), T, nb,
            num_heads, kvh, d, BLOCK, _CODE[qkv.dtype], _stream(dev)))


def dequantize(pool: torch.Tensor, block_tables: torch.Tensor, lens: torch.Tensor,
               out_tables: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor, *,
               row_index: torch.Tensor | None = None) -> None:
    """Read the first ``lens[r]`` tokens of each table row back into 16-bit pools ``k_out`` /
    ``v_out`` [out_blocks, KVH, 16, D]: block j of row r goes to block ``out_tables[r, j]`` (a
    negative entry skips it), with zeros behind the row's length in its last block and where the
    source entry holds no block.  Blocks that lie wholly behind the length are not written, and their
    entries not looked at.  ``row_index`` selects the rows of ``block_tables``.  The target blocks
    are distinct.

    A pool of all layers [layers, num_blocks, KVH, 18 D], as ``evict`` takes it, is read as one of
    layers * num_blocks blocks: block b of layer l is entry l * num_blocks + b."""
    dev = _device(pool, block_tables, lens, out_tables, k_out, v_out, row_index)
    nb, kvh, d = _pool_shape(pool, layered=True)
    if pool.dim() == 4:
        nb *= pool.shape[0]
    if k_out.dim() != 4 or k_out.shape != v_out.shape or k_out.dtype != v_out.dtype or \
            k_out.dtype not in _HALF or not k_out.is_contiguous() or \
            not v_out.is_contiguous() or k_out.shape[1:] != (kvh, BLOCK, d):
        _fail("k_out and v_out must be contiguous 16-bit [out_blocks, num_kv_heads, 16, head_dim]")
    rows = lens.numel()
    _index("lens", lens)
    _index("row_index", row_index, rows)
    ot_stride, cols = _table("out_tables", out_tables, rows)
    bt_stride, width = _table("block_tables", block_tables, rows if row_index is None else None)
    if width < cols:
        _fail("block_tables is narrower than out_tables")
    if rows == 0 or k_out.shape[0] == 0:
        return
    with _on(dev):
        N.check(N.lib().ti_kv4_dequantize(
            k_out.data_ptr(), v_out.data_ptr(), k_out.shape[0], pool.data_ptr(), nb,
            block_tables.data_ptr(), bt_stride, _ptr(row_index), lens.data_ptr(),
            out_tables.data_ptr(), ot_stride, rows, cols, kvh, d, BLOCK,
            _CODE[k_out.dtype], _stream(dev)))


def _workspace(dev: int, nbytes: int, stream: int) -> torch.Tensor:
    """Zeroed scratch, one per (device, stream); inside a stream capture one of the graph's own
    (so graphs that replay at the same time do not share it), zeroed by the graph itself."""
    if torch._C._cuda_isCurrentStreamCapturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=_cuda(dev))
    return _ws.get(_cuda(dev), nbytes, stream)


_cuda = functools.lru_cache(maxsize=None)(functools.partial(torch.device, "cuda"))


@functools.lru_cache(maxsize=4096)
def _decode_bytes(dev: int, *sizes: int) -> int:
    """Workspace of a decode call on ``dev`` (the current device), asked once per sizes."""
    return int(N.lib().ti_kv4_attention_workspace_bytes(*sizes))


def decode_attention(out: torch.Tensor, q: torch.Tensor, pool: torch.Tensor,
                     block_tables: torch.Tensor, context_lens: torch.Tensor, *,
                     row_index: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None) -> None:
    """Single-query attention, scale 1/sqrt(head_dim): out[b] = softmax(q[b] K^T) V over the first
    ``context_lens[b]`` cached tokens of row ``row_index[b]`` (default b) of ``block_tables``.

    q, out: [B, NH, D] bf16 or fp16, at most 16 query heads per kv head, B at most 4096, B * table
    columns * kv heads (twice beyond 8 query heads per kv head) below 2^29.  ``lse``
    (float32 [B, NH]) receives the natural log of each row's sum of exp(scores).  A sequence of
    length 0 leaves its rows of ``out`` and ``lse`` as they were; one whose table holds no block
    gets NaN, and -inf in ``lse``.  One launch; results do not depend on the batch's other rows'
    contents and are the same on every run."""
    dev = _device(pool, out, q, block_tables, context_lens, row_index, lse)
    B, NH, nb, kvh, d, q_stride, bt_stride, cols = _attention(q, pool, block_tables, context_lens,
                                                              row_index)
    out_stride = _out_rows(out, q)
    if lse is not None:
        _head_sums("lse", lse, B, NH)
    if B == 0:
        return
    lib = N.lib()
    with _on(dev):
        stream = _stream(dev)
        ws = _workspace(dev, _decode_bytes(dev, B, NH, kvh, d, cols), stream)
        N.check(lib.ti_kv4_attention_decode(
            out.data_ptr(), out_stride, _ptr(lse), q.data_ptr(), q_stride, pool.data_ptr(), nb,
            block_tables.data_ptr(), bt_stride, _ptr(row_index), context_lens.data_ptr(), B, NH,
            kvh, d, BLOCK, cols, _CODE[q.dtype], ws.data_ptr(), ws.numel(), stream))


def accumulate_weights(weights: torch.Tensor, q: torch.Tensor, lse: torch.Tensor,
                       pool: torch.Tensor, block_tables: torch.Tensor,
                       context_lens: torch.Tensor, *, row_index: torch.Tensor | None = None,
                       out: torch.Tensor | None = None) -> None:
    """Add to each cached token's total the attention weight that ``q`` gives it, summed over the
    query heads of its kv head: out = weights + sum_h exp(q_h . k / sqrt(D) - lse_h).

    ``lse`` float32 [B, NH] as ``decode_attention`` gives it for the same arguments; weights and
    out (default: weights itself) float32 [num_blocks, KVH, 16], of which only the sequences' own
    tokens are written.  The sequences of a call share no block.  Sizes as ``decode_attention``'s."""
    out = weights if out is None else out
    dev = _device(pool, weights, q, lse, block_tables, context_lens, row_index, out)
    B, NH, nb, kvh, d, q_stride, bt_stride, cols = _attention(q, pool, block_tables, context_lens,
                                                              row_index)
    _totals("weights", weights, nb, kvh)
    _totals("out", out, nb, kvh)
    _head_sums("lse", lse, B, NH)
    if B == 0:
        return
    with _on(dev):
        N.check(N.lib().ti_kv4_accumulate_weights(
            out.data_ptr(), weights.data_ptr(), q.data_ptr(), q_stride, lse.data_ptr(),
            pool.data_ptr(), nb, block_tables.data_ptr(), bt_stride, _ptr(row_index),
            context_lens.data_ptr(), B, NH, kvh, d, BLOCK, cols, _CODE[q.dtype],
            _stream(dev)))


class PrefillPlan:
    """Layout of a packed prefill: chunk i holds ``counts[i]`` query tokens at positions
    ``starts[i]`` and on, whose K and V are already in the cache.  Built once per batch, used by
    every layer, on any stream; the work items of a head layout are laid out at its first use and
    kept.  A graph that captured a call reads the plan's memory: lay the plan out before the capture
    and keep it as long as the graph."""

    def __init__(self, starts, counts, device="cuda") -> None:
        starts, counts = np.asarray(starts, np.int64), np.asarray(counts, np.int64)
        if starts.ndim != 1 or starts.shape != counts.shape:
            _fail("starts and counts must be lists of the same length")
        if not ((starts >= 0).all() and (counts >= 0).all()):
            _fail("starts and counts must be >= 0")
        lens = np.where(counts > 0, starts + counts, 0)
        if int(lens.max(initial=0)) >= 2 ** 31 or int(counts.sum()) >= 2 ** 31:
            _fail("prefill too long")
        self.starts, self.counts, self.device = starts, counts, device
        self.num_seqs, self.num_tokens = len(starts), int(counts.sum())
        self.max_blocks = int((-(-lens // BLOCK)).max(initial=0))
        self._dev = torch.from_numpy(np.concatenate([starts, [0], np.cumsum(counts)])
                                     .astype(np.int32)).to(device)
        self.start_pos, self.cu_seqlens = self._dev[:self.num_seqs], self._dev[self.num_seqs:]
        self._layouts: dict = {}
        self._tensors, self._held = [(self._dev, self._home())], {}

    def _home(self) -> int | None:
        """The stream that a device tensor made now belongs to."""
        dev = self._dev.get_device()
        return _stream(dev) if dev >= 0 else None

    def hold(self, dev: int, stream: int) -> None:
        """Calls on ``stream``, the current one of ``dev``, read the plan's tensors: the memory of
        those that belong to another stream is not handed out again before these calls are done.
        (Inside a capture nothing is noted: its graph needs the plan itself.)"""
        if self._held.get(stream, 0) == len(self._tensors) or \
                torch._C._cuda_isCurrentStreamCapturing():
            return
        for t, home in self._tensors[self._held.get(stream, 0):]:
            if home != stream:
                t.record_stream(torch.cuda.current_stream(dev))
        self._held[stream] = len(self._tensors)

    def work(self, group: int, kv_heads: int, head_dim: int = 64):
        """Items and merges (``ti_kv4_prefill_attention``) as host arrays, and the number of parts.

        An item is up to three tiles (head_dim 128: two) of 128 / slots tokens, which share their
        keys' way through the chip: as many as leave an item for each of 148 SMs, ranges of 1024
        keys counted as items.  Items with more keys than a third of what each SM would get on
        average (at least 1024: a range costs a few microseconds of its own) are cut: their keys,
        one item behind the other, at every multiple of that size, so that all pieces but the
        ends are of one size and a few long prefixes still fill the GPU.  Longest first."""
        slots = 1 << (group - 1).bit_length()
        for tiles in (3, 2, 1) if head_dim == 64 else (2, 1):
            step = tiles * (128 // slots)
            seq = np.repeat(np.arange(self.num_seqs), -(-self.counts // step))
            per = np.concatenate([np.arange(0, c, step) for c in self.counts.tolist()] or
                                 [np.zeros(0, np.int64)]).astype(np.int64)
            keys = self.starts[seq] + np.minimum(per + step, self.counts[seq])
            if int((-(-keys // 1024)).sum()) * kv_heads >= 148:
                break
        steps = -(-keys // 64)                                  # a range is whole 64-key steps
        unit = max(16, -(-int(steps.sum()) * kv_heads // (3 * 148)))
        cut = steps > unit
        begin = np.cumsum(np.where(cut, steps, 0)) - steps      # of a cut item among them
        end = begin + steps
        # cuts first .. last, in units; none within an eighth of a unit of either end
        first, last = begin // unit + 1, (end - 1) // unit
        first = first + (first * unit - begin < unit // 8)
        last = last - (end - last * unit < unit // 8)
        n = np.where(cut, last - first + 2, 1)
        first_part = np.cumsum(np.where(n > 1, n, 0)) - np.where(n > 1, n, 0)
        at = np.repeat(np.arange(len(seq)), n)                  # the item of each piece
        k = np.arange(len(at)) - np.repeat(np.cumsum(n) - n, n)  # its place within the item
        at_cut = (first[at] + k) * unit - begin[at]             # where piece k of a cut item ends
        lo = np.where(k > 0, at_cut - unit, 0) * 64
        hi = np.where(k < n[at] - 1, at_cut * 64, keys[at])
        part = np.where(n[at] > 1, first_part[at] + k, -1)
        items = np.stack([seq[at], per[at], lo, hi, part, np.full_like(lo, tiles)], 1)
        items = items[np.argsort(lo - hi, kind="stable")].astype(np.int32)
        cut = n > 1
        merges = np.stack([seq[cut], per[cut], first_part[cut], n[cut],
                           np.full_like(n[cut], tiles)], 1).astype(np.int32)
        return items, merges, int(n[cut].sum())

    def layout(self, group: int, kv_heads: int, head_dim: int):
        """``work`` on the device: pointers and counts, for calls of this head layout."""
        key = (group, kv_heads, head_dim)
        if key not in self._layouts:
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                _fail("this head layout of the plan is new: run it once, or call layout(), "
                      "before the capture")
            items, merges, parts = self.work(group, kv_heads, head_dim)
            dev = torch.from_numpy(np.concatenate([items.reshape(-1), merges.reshape(-1)])
                                   ).to(self.device)
            base = dev.data_ptr()
            self._tensors.append((dev, self._home()))
            self._layouts[key] = (dev, base, len(items), base + 4 * items.size, len(merges), parts)
        return self._layouts[key][1:]


def prefill_attention(out: torch.Tensor, q: torch.Tensor, pool: torch.Tensor,
                      block_tables: torch.Tensor, plan: PrefillPlan, *,
                      row_index: torch.Tensor | None = None) -> None:
    """Causal attention of the plan's query tokens (q, out [tokens, NH, D]) over their sequences'
    cached tokens, positions 0 .. their own, scale 1/sqrt(D), on the tensor cores straight from the
    codes.  At most 16 query heads per kv head.  Tokens whose table entry holds no block are left
    out.  Chunks with long prefixes are cut along the keys and joined by a second launch."""
    dev = _device(pool, out, q, block_tables, plan.start_pos, row_index)
    nb, kvh, d = _pool_shape(pool)
    T, NH, dq, q_stride = _rows("q", q)
    out_stride = _out_rows(out, q)
    if dq != d:
        _fail("head_dim does not match the pool's tiles")
    if NH <= 0 or NH % kvh or NH > 16 * kvh:
        _fail("query heads must be a multiple of the kv heads, at most 16 per kv head")
    if T != plan.num_tokens:
        _fail("q does not have the plan's tokens")
    _index("row_index", row_index, plan.num_seqs)
    bt_stride, cols = _table("block_tables", block_tables,
                             plan.num_seqs if row_index is None else None)
    if cols < plan.max_blocks:
        _fail("block_tables is too narrow for the plan")
    if T == 0:
        return
    lib = N.lib()
    with _on(dev):
        items, num_items, merges, num_merges, parts = plan.layout(NH // kvh, kvh, d)
        stream = _stream(dev)
        plan.hold(dev, stream)
        ws = None
        if parts:
            ws = torch.empty(lib.ti_kv4_prefill_workspace_bytes(parts, kvh, d), dtype=torch.uint8,
                             device=pool.device)
        N.check(lib.ti_kv4_prefill_attention(
            out.data_ptr(), out_stride, q.data_ptr(), q_stride, pool.data_ptr(), nb,
            block_tables.data_ptr(), bt_stride, cols, _ptr(row_index), plan.start_pos.data_ptr(),
            plan.cu_seqlens.data_ptr(), items, num_items, merges, num_merges, parts, NH, kvh, d,
            BLOCK, _CODE[q.dtype], _ptr(ws), 0 if ws is None else ws.numel(), stream))


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
    caller shortens the lengths to min(context_lens, keep) and frees the blocks behind.  Pass the
    columns of ``block_tables`` that are in use: what a call costs goes by the table's width, not by
    the lengths, which are on the device.  A sequence
    with a needed table entry outside the pool is left as it is and raises TI_DEVERR_BAD_INPUT.
    The sequences of a call share no block."""
    dev = _device(pool, weights, block_tables, context_lens, row_index, out_block_tables, kept)
    nb, kvh, d = _pool_shape(pool, layered=True)
    layers = pool.shape[0] if pool.dim() == 4 else 1
    if weights.dtype != torch.float32 or not weights.is_contiguous() or \
            weights.shape != (*pool.shape[:-1], BLOCK):
        _fail("weights must be contiguous float32, the pool's shape with 16 in the last place")
    keep, recent = int(keep), int(recent)
    if keep < 1 or not 0 <= recent <= keep:
        _fail("needs keep >= 1 and 0 <= recent <= keep")
    B = context_lens.numel()
    _index("context_lens", context_lens)
    _index("row_index", row_index, B)
    rows = B if row_index is None else None
    bt_stride, cols = _table("block_tables", block_tables, rows)
    to = block_tables if out_block_tables is None else out_block_tables
    to_stride, to_cols = _table("out_block_tables", to, rows if rows is not None
                                else block_tables.shape[0])
    if kept is not None and (kept.dtype != torch.int32 or not kept.is_contiguous() or
                             kept.dim() != 4 or kept.shape[:3] != (layers, B, kvh) or
                             kept.shape[3] < keep):
        _fail("kept must be contiguous int32 [layers, batch, num_kv_heads, >= keep]")
    if B == 0 or layers == 0:
        return
    # (lengths are 32-bit: beyond them any keep evicts nothing)
    keep, recent = min(keep, _MOST), min(recent, _MOST)
    with _on(dev):
        N.check(N.lib().ti_kv4_evict(
            pool.data_ptr(), weights.data_ptr(), layers, nb, block_tables.data_ptr(), bt_stride,
            to.data_ptr(), to_stride, _ptr(row_index), context_lens.data_ptr(), B, cols, to_cols,
            keep, recent, _ptr(kept), kept.shape[3] if kept is not None else 0, kvh, d, BLOCK,
            _stream(dev)))
