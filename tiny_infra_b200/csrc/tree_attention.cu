// Attention of drafted trees over the paged 16-bit pool, tcgen05.
//
// out = softmax(q K^T / sqrt(D)) V.  Sequence i's nodes are query rows cu[i] .. cu[i+1]-1; their K and V
// are in the pool at positions ctx[i] .. of the sequence's table row, behind its ctx[i] cached tokens.  A
// node attends to every cached token and to the nodes whose bits its mask row has (no masks: to the
// nodes up to itself).
//
// A tile is 128 rows, (node, query head of one kv head) in order.  A CTA takes up to three tiles of a tree
// (two for D = 128: what tensor memory holds), which share each 64-key chunk that TMA brings from the
// pool.  Per chunk and tile:
//   S = Q K^T   M 128, N 64, into TMEM; freed as soon as the softmax warps have it in registers;
//   softmax     one row per thread, a running max that is kept until a row's grows by more than 2^8
//               (then O is rescaled in TMEM), P = 2^(s - m) back into TMEM as the sum of two values of the
//               pool's type, P and what its rounding left (17 bits in all for bf16, 22 for fp16; the
//               prefill attention over the same pool does so too, and for bf16 the decode attention); the
//               sum is taken before that rounding;
//   O += P V    twice, A from TMEM, V in place as an MN-major operand; fp32 O in TMEM.
// O and both parts of P fill 384 of the 512 columns for three tiles of 64 dims (and for two of 128); the
// scores have two buffers of 64, which the CTA's jobs (a tile's chunk each) take in turn: a buffer is free
// once its scores are in registers.
// Trees of one tile (up to 18 nodes of 7 heads) would leave two thirds of the softmax warps without work:
// there the slots take the chunks in turn, each with an O of its own, joined at the end in TMEM.
//
// Work: the lengths are on the device, so one warp of every CTA sums up the batch's work and finds the CTA's
// share of it (tree_schedule.cuh).  Units that are cut over CTAs leave un-normalised parts, joined in
// pairs by whichever CTA of a pair comes second: no CTA waits for another, the joins of a long sequence
// go on side by side, and their order does not depend on who comes when.
//
// Bound: 32 trees of 64 nodes behind 2048 to 8192 tokens (14 heads over 2, D = 64) take 111 us as calls in a
// row.  Their exponentials alone would take 37 (8 clocks a warp instruction), the MMAs 42; a chunk of three
// tiles takes 2820 clocks, of which the exponential unit is busy for 1536 (two tiles: 2330 and 1024, one: 1040;
// four tiles as two and two instead of three and one take 120 us): the softmax warps of a scheduler do not
// hide each other's trips to tensor memory and barriers.  8 trees of up to 16 nodes behind 16384 to 32768
// tokens (32 heads over 8, D = 128): 156 us in a row, 190 to 196 between other work, 0.79 and 0.63 of
// measured copy; a chunk there takes 1320 clocks.  Weights in one part took 100 and 139 us in a row, at 1.3
// times the error against 64 bits; in two parts the error is the output's own rounding alone.
// Measured on the way, with weights in one part: one warp for all MMAs, which then wait for each other's
// operands, 313 us instead of 194 in the latter case; one warp for all TMA boxes 155 instead of 136.  Small
// batches are a chain of dependent trips: 11.8 us in a graph for 4 trees of up to 8 nodes, with the memset
// of the counters.
//
// Values that a node does not see: scores are replaced, so keys may hold anything.  V is multiplied by a
// weight of 0, which a NaN or infinity would survive: in chunks that reach past the cached tokens or hold
// an absent block the first slot's threads zero V's rows behind the end and those blocks, and any
// non-finite elements of drafts; rows that do see such a draft add its values at the end (rare, from the
// pool).  An infinite value of a cached token, which every node sees, makes that dim NaN or infinite (the
// second part of a weight may be 0), as in the prefill attention.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "capi_internal.h"
#include "common.cuh"
#include "softmax_tile.cuh"
#include "tcgen05.cuh"
#include "tree_schedule.cuh"

namespace ti {
namespace tree {

constexpr int kBlock = 16;
constexpr int kMaxGroup = 16;
constexpr int kMaxSeqs = 4096;
constexpr int kRing = 16;                // items on their way: more than chunks on theirs
constexpr int kCtas = 148;               // most CTAs of a launch (one per SM)
// One word per CTA and slot.  It holds the number of the call whose first half of a join is in memory; the second
// half's CTA sets it back to 0.  A call that ends early (a wait gave up) leaves words of its own number
// behind, which mean nothing to the calls that follow.
constexpr size_t kCounterBytes = 4096;

struct Params {
  void* out;
  const void *q, *v;
  float* lse;
  int64_t out_stride, q_stride, num_blocks, bt_stride;
  const int32_t *tables, *row_index, *ctx, *cu, *masks;
  float* parts;
  unsigned* counters;
  int seqs, tokens, rows, cols, NH, KVH, group, mask_words;
  float scale_log2;
  unsigned call;                         // not 0; another one for each call
};

template <int HD>
struct Cfg {
  static constexpr int kSub = HD / 64;                    // 64-dim sub-tiles of a row
  static constexpr int kTiles = HD == 64 ? 3 : 2;
  static constexpr int kSoftWarps = 4 * kTiles;
  static constexpr int kLoadWarp = kSoftWarps, kScoreWarp = kSoftWarps + 1, kValueWarp = kSoftWarps + 2;
  static constexpr int kLoadVWarp = kSoftWarps + 3;
  static constexpr int kThreads = (kSoftWarps + 4) * 32;
  static constexpr int kQTile = kSub * 16384, kKvTile = kSub * 8192, kStage = 2 * kKvTile;
  static constexpr int kStages = HD == 64 ? 8 : 4;
  static constexpr int kKv = kTiles * kQTile;
  static constexpr int kMl = kKv + kStages * kStage;      // [kTiles][128] float2
  static constexpr int kOk = kMl + kTiles * 1024;         // [kStages] ints: blocks there, masked
  static constexpr int kDirty = kOk + 64;                 // [2] ints, by item
  static constexpr int kFlag = kDirty + 64;               // [kTiles] broadcast words
  static constexpr int kBars = kFlag + 64;
  static constexpr int kItems = kBars + 512;              // [kRing] items
  static constexpr int kMask = kItems + kRing * 64;       // [kTiles][128] first two mask words
  static constexpr int kSched = kMask + kTiles * 1024;    // [seqs + 1] ints
  static int smem(int seqs) { return kSched + (seqs + 1) * 4 + 1024; }
  // TMEM columns: two buffers of scores; weights (two 16-bit values a column, 32 columns of first parts and
  // 32 of second ones) and O of every slot
  static __device__ __forceinline__ uint32_t s_col(uint32_t buffer) { return 64 * buffer; }
  static __device__ __forceinline__ uint32_t p_col(int x) { return 128 + 64 * x; }
  static __device__ __forceinline__ uint32_t o_col(int x) { return 128 + 64 * kTiles + HD * x; }
  static_assert(128 + (64 + HD) * kTiles <= 512, "tensor memory");
  static constexpr int64_t kPart = 128 * (HD + 2);        // floats of a part of one tile: O, then (m, l)
};

// A unit's piece in this CTA.  The load warp finds them and passes them on; tiles 0: there are no more.
struct Item {
  int tiles, kvh, nodes, ctx, row0, tile0, c0, c1, keys, first, parts;   // first: CTA of part 0
  const int32_t* table;                  // null: the row does not exist
};
static_assert(sizeof(Item) <= 64, "ring entries");

// A sequence as the load warp sees it; start: the place of its first unit on the line of work.
struct Seq {
  SeqWork w;
  int ctx, row0, nodes, row;
  unsigned start;
};

template <int TILES>
__device__ __forceinline__ Seq sequence(const Params& p, int i) {
  Seq s;
  s.row0 = max(p.cu[i], 0);
  s.nodes = max(min(p.cu[i + 1], p.tokens) - s.row0, 0);
  s.ctx = max(p.ctx[i], 0);
  s.row = p.row_index ? p.row_index[i] : i;
  if (s.row >= p.rows) s.row = -1;
  s.w = seq_work(s.ctx, s.nodes, s.row >= 0, p.group, p.KVH, p.cols * kBlock, TILES);
  return s;
}

// This CTA's items, found by one warp.  Up to 32 sequences a lane holds one of them, so that none is looked
// up twice: at these sizes the way to the first load is a good part of a call.
template <int TILES>
struct Walk {
  Plan plan;
  unsigned begin, end;
  Seq mine, cur;
  int seq;
  Units at;                              // of the current sequence: its full ones, or what is left
  int unit, k;                           // the next one, and its pieces
  unsigned start, len;                   // where they begin on the line of work, and a unit's length there
  bool rest;
  unsigned* starts;

  __device__ __forceinline__ Walk(const Params& p, unsigned* starts_) : starts(starts_) {
    const int lane = threadIdx.x & 31, each = (p.seqs + 31) / 32;
    const int i0 = min(p.seqs, lane * each), i1 = min(p.seqs, i0 + each);
    unsigned jobs = 0, units = 0;
    mine.w = SeqWork{0, 0, 0, {0, 0, 0, 0}, {0, 0, 0, 0}};
    for (int i = i0; i < i1; ++i) {
      mine = sequence<TILES>(p, i);
      jobs += seq_jobs(mine.w);
      units += (unsigned)(mine.w.full.count + mine.w.rest.count);
    }
    plan = Plan{dense_share(__reduce_add_sync(0xffffffffu, jobs), kCtas), 0u};
    if (__reduce_add_sync(0xffffffffu, units) <= (unsigned)kCtas) {
      auto fits = [&](unsigned per) {
        unsigned n = 0;
        for (int i = i0; i < i1; ++i) {
          if (each > 1) mine = sequence<TILES>(p, i);
          n += seq_pieces(mine.w, per);
        }
        return __reduce_add_sync(0xffffffffu, n) <= (unsigned)kCtas;
      };
      // (the smallest share that fits, if the largest one that is tried does)
      if (fits(tried_share(plan.per, 0))) {
        plan.aligned = 1;
      } else if (fits(tried_share(plan.per, kTries - 1))) {
        int k = 1;
        while (!fits(tried_share(plan.per, k))) ++k;
        plan = Plan{tried_share(plan.per, k), 1u};
      }
    }
    unsigned own = 0;
    for (int i = i0; i < i1; ++i) {
      if (each > 1) mine = sequence<TILES>(p, i);
      if (each > 1) starts[i] = own;
      own += seq_length(mine.w, plan);
    }
    unsigned v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    const unsigned total = __shfl_sync(0xffffffffu, v, 31);
    begin = min(total, blockIdx.x * plan.per);
    end = min(total, begin + plan.per);
    if (each <= 1) {
      mine.start = v - own;
      if (i0 >= i1) mine.w.full.count = mine.w.rest.count = 0;
      const unsigned here = __ballot_sync(0xffffffffu, begin >= mine.start && begin < v);
      seq = here ? __ffs(here) - 1 : 0;
    } else {
      for (int i = i0; i < i1; ++i) starts[i] += v - own;
      __syncwarp();
      int lo = 0, hi = p.seqs - 1;
      while (lo < hi) {                            // the last sequence that starts at or before `begin`
        const int mid = (lo + hi + 1) >> 1;
        if (starts[mid] <= begin) lo = mid; else hi = mid - 1;
      }
      seq = lo;
    }
    load(p);
    if (begin > cur.start && begin < end) {
      unit = (int)((begin - cur.start) / len);
      if (unit >= cur.w.full.count && cur.w.rest.count) {
        second();
        unit = (int)((begin - start) / len);
      }
    }
  }
  // from the sequence's full units to those of what is left
  __device__ __forceinline__ void second() {
    start += (unsigned)at.count * len;
    at = cur.w.rest;
    k = pieces(at, plan);
    len = length(at, plan, k);
    unit = 0;
    rest = true;
  }
  __device__ __forceinline__ void load(const Params& p) {
    if (p.seqs > 32) {
      cur = sequence<TILES>(p, seq);
      cur.start = starts[seq];
    } else {
      int* to = reinterpret_cast<int*>(&cur);
      const int* from = reinterpret_cast<const int*>(&mine);
#pragma unroll
      for (int i = 0; i < (int)(sizeof(Seq) / 4); ++i) to[i] = __shfl_sync(0xffffffffu, from[i], seq);
    }
    at = cur.w.full;
    k = pieces(at, plan);
    len = length(at, plan, k);
    start = cur.start;
    unit = 0;
    rest = false;
  }
  __device__ __forceinline__ bool next(const Params& p, Item& it) {
    while (begin < end) {
      while (unit >= at.count) {
        if (!rest && cur.w.rest.count) {
          second();
        } else {
          if (++seq >= p.seqs) return false;
          load(p);
        }
      }
      const unsigned place = start + (unsigned)unit * len;
      if (place >= end) return false;
      const int u = unit++;
      it.c0 = chunk_at(begin, place, at, plan, k);
      it.c1 = chunk_at(end, place, at, plan, k);
      if (it.c0 >= it.c1) continue;
      it.kvh = rest || cur.w.groups == 1 ? u : u / cur.w.groups;
      it.nodes = cur.nodes;
      it.ctx = cur.ctx;
      it.row0 = cur.row0;
      it.keys = cur.w.keys;
      it.table = cur.row >= 0 ? p.tables + (int64_t)cur.row * p.bt_stride : nullptr;
      it.tile0 = (rest ? cur.w.groups : u - it.kvh * cur.w.groups) * cur.w.full.width;
      it.tiles = at.width;
      it.first = blockIdx.x;
      it.parts = 1;
      if (it.c0 > 0 || it.c1 < at.chunks) {
        it.first = first_cta(place, at, plan, k);
        it.parts = last_cta(place, at, plan, k) - it.first + 1;
      }
      return true;
    }
    return false;
  }
};

__device__ __forceinline__ bool bar_or(int id, int threads, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %3, 0;\n\t"
      "barrier.cta.red.or.pred p, %1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((uint32_t)v)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Bits of the keys k0 .. k0 + 63 that node `node` (row t) sees; have: the blocks that exist; first: the
// row's first two mask words.
__device__ __forceinline__ uint64_t seen(const Params& p, const Item& it, int64_t t, int node, int k0, int have,
                                         uint2 first) {
  const int b0 = k0 - it.ctx;                     // the first key as a node's number
  uint64_t see;
  if (!p.masks) {
    const long long n = (long long)node - b0 + 1;
    see = n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
  } else {
    const uint32_t* m = reinterpret_cast<const uint32_t*>(p.masks) + t * p.mask_words;
    auto word = [&](int w) -> uint64_t { return w == 0 ? first.x : w == 1 ? first.y : w < p.mask_words ? (uint64_t)m[w] : 0ull; };
    if (b0 >= 0) {
      const int w = b0 >> 5, sh = b0 & 31;
      see = (word(w) | word(w + 1) << 32) >> sh;
      if (sh) see |= word(w + 2) << (64 - sh);
    } else if (b0 > -64) {
      see = ((uint64_t)first.x | (uint64_t)first.y << 32) << -b0 | ((1ull << -b0) - 1);
    } else {
      see = ~0ull;
    }
  }
  const int left = it.keys - k0;
  if (left < 64) see &= left > 0 ? (1ull << left) - 1 : 0ull;
#pragma unroll
  for (int b = 0; b < 4; ++b)
    if (!((have >> b) & 1)) see &= ~(0xFFFFull << (16 * b));
  return see;
}

template <typename T, int HD>
__global__ void __launch_bounds__(Cfg<HD>::kThreads, 1)
attention_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                 const __grid_constant__ Params p) {
  using C = Cfg<HD>;
  constexpr int kTiles = C::kTiles, kStages = C::kStages;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  // fp16 weights are held times 2^7 (at most 2^15, steps of 2^-31 at the small end); bf16 has the range
  constexpr float kPScale = kBf16 ? 0.f : 7.f;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sb = smem_u32(smem);
  // per stage: chunk there, chunk done with; per slot, a phase per job: scores written, weights written, P V
  // done; per buffer of scores, a phase for every second job: read; per item: Q there, the item itself there
  const uint32_t kv_full = sb + C::kBars, kv_empty = kv_full + 8 * kStages, s_full = kv_empty + 8 * kStages;
  const uint32_t s_read = s_full + 8 * kTiles, p_ready = s_read + 16, pv_done = p_ready + 8 * kTiles;
  const uint32_t q_full = pv_done + 8 * kTiles, item_full = q_full + 8;   // (item_full: one per ring entry)
  uint32_t* tslot = reinterpret_cast<uint32_t*>(smem + C::kBars + 496);
  volatile int* s_ok = reinterpret_cast<volatile int*>(smem + C::kOk);
  volatile int* s_flag = reinterpret_cast<volatile int*>(smem + C::kFlag);
  uint2* s_mask = reinterpret_cast<uint2*>(smem + C::kMask);
  float2* s_ml = reinterpret_cast<float2*>(smem + C::kMl);
  Item* s_item = reinterpret_cast<Item*>(smem + C::kItems);
  unsigned* s_start = reinterpret_cast<unsigned*>(smem + C::kSched);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (warp == C::kScoreWarp) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        mbar_init(kv_full + 8 * i, 2);            // (the K and the V warp)
        mbar_init(kv_empty + 8 * i, 1);
      }
      for (int i = 0; i < kTiles; ++i) {
        mbar_init(s_full + 8 * i, 1);
        mbar_init(p_ready + 8 * i, 4);
        mbar_init(pv_done + 8 * i, 1);
      }
      for (int i = 0; i < 2; ++i) mbar_init(s_read + 8 * i, 4);
      mbar_init(q_full, C::kSoftWarps);
      for (int i = 0; i < kRing; ++i) mbar_init(item_full + 8 * i, 1);
      fence_mbar_init();
      prefetch_tensormap(&kmap);
      prefetch_tensormap(&vmap);
    }
    __syncwarp();
    tmem_alloc(smem_u32(tslot), 512);
  }
  pdl_wait();

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  pdl_launch_dependents();

  if (warp == C::kLoadWarp || warp == C::kLoadVWarp) {
    // ---- TMA, one warp for K and one for V (a chunk is 4 or 8 small boxes each, and issuing them is what
    // a tree of one tile would wait for: one warp for both took 1100 clocks a chunk of 64 dims); the K warp
    // also finds the items
    const bool keys = warp == C::kLoadWarp, leader = elect_one();
    const CUtensorMap* map = keys ? &kmap : &vmap;
    auto load = [&](const Item& it, int& g) {
      auto ids_from = [&](int c) {                 // the ids of eight chunks, one per lane
        const int blk = c * 4 + lane;
        return it.table && c < it.c1 && (int64_t)blk * kBlock < it.keys ? it.table[blk] : -1;
      };
      int ids = ids_from(it.c0), after = ids_from(it.c0 + 8);
      const int c0 = it.c0, c1 = it.c1, kvh = it.kvh, ctx = it.ctx;
      for (int c = c0; c < c1; ++c, ++g) {
        const int k = (c - c0) & 7, st = g % kStages;
        if (k == 0 && c > c0) {
          ids = after;
          after = ids_from(c + 8);
        }
        int y[4], have = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int id = __shfl_sync(0xffffffffu, ids, k * 4 + b);
          have |= (unsigned)id < (unsigned)p.num_blocks ? 1 << b : 0;
          y[b] = (id * p.KVH + kvh) * kBlock;
        }
        if (g >= kStages &&
            !__all_sync(0xffffffffu, mbar_wait(kv_empty + 8 * st, ((g / kStages) - 1) & 1, TI_DEVERR_PREFILL_WAIT)))
          return false;
        if (leader) {
          const uint32_t bar = kv_full + 8 * st, dst = sb + C::kKv + st * C::kStage + (keys ? 0 : C::kKvTile);
          if (keys) s_ok[st] = have | (have != 15 || (c + 1) * kChunk > ctx ? 16 : 0);
          mbar_arrive_expect_tx(bar, (uint32_t)__popc(have) * (C::kSub * 2048));
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if ((have >> b) & 1)
#pragma unroll
              for (int sub = 0; sub < C::kSub; ++sub)
                tma_load_2d(dst + sub * 8192 + b * 2048, map, bar, sub * 64, y[b]);
        }
        __syncwarp();
      }
      return true;
    };
    int g = 0;                                     // chunks so far
    bool ok = true;
    if (keys) {
      Walk<kTiles> walk(p, s_start);
      Item it;
      for (int items = 0;; ++items) {
        // (at most kStages items are ahead of the softmax, each has a chunk: the entry is free)
        if (!ok || !walk.next(p, it)) it.tiles = 0;
        if (lane == 0) {
          s_item[items % kRing] = it;
          mbar_arrive(item_full + 8 * (items % kRing));
        }
        if (it.tiles == 0) break;
        // Q's rows on their way into L2, ahead of the chunks in the queue to memory
        const int n0 = it.tile0 * 128 / p.group;
        const int n1 = min(it.nodes, ((it.tile0 + it.tiles) * 128 + p.group - 1) / p.group);
        const int lines = (p.group * HD * 2 + 127) / 128;
        for (int i = lane; i < (n1 - n0) * lines; i += 32) {
          const char* row = reinterpret_cast<const char*>((const T*)p.q + (int64_t)(it.row0 + n0 + i / lines) * p.q_stride +
                                                          (int64_t)it.kvh * p.group * HD);
          asm volatile("prefetch.global.L2 [%0];" ::"l"(row + (i % lines) * 128));
        }
        ok = load(it, g);
      }
    } else {
      for (int items = 0; ok; ++items) {
        ok = __all_sync(0xffffffffu, mbar_wait(item_full + 8 * (items % kRing), (items / kRing) & 1, TI_DEVERR_PREFILL_WAIT));
        if (!ok || s_item[items % kRing].tiles == 0) break;
        ok = load(s_item[items % kRing], g);
      }
    }
  } else if (warp == C::kScoreWarp || warp == C::kValueWarp) {
    // ---- MMA issue: one warp for the scores, one for the values, so that neither waits for what the
    // other needs; the whole warp walks the loop, one elected lane issues
    constexpr uint32_t id_s = idesc_f16(128, kChunk, kBf16, false, false);
    constexpr uint32_t id_pv = idesc_f16(128, 64, kBf16, false, true);
    const bool leader = elect_one();
    int g = 0, items = 0;
    uint32_t done[kTiles] = {};                    // jobs of each slot so far
    uint32_t job = 0;                              // jobs whose scores have been issued
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, TI_DEVERR_PREFILL_WAIT));
      return ok;
    };
    while (ok) {
      if (!wait(item_full + 8 * (items % kRing), (items / kRing) & 1)) break;
      const Item& it = s_item[items % kRing];
      // (a shuffle tells the compiler that a value is the same in all lanes: descriptors then stay in
      // uniform registers)
      const int tiles = __shfl_sync(0xffffffffu, it.tiles, 0);
      const int n = __shfl_sync(0xffffffffu, it.c1 - it.c0, 0);
      if (tiles == 0) break;
      const bool turns = tiles == 1;               // the slots take the chunks in turn
      const int rounds = turns ? (n + kTiles - 1) / kTiles : n;
      if (warp == C::kScoreWarp) {
        const uint64_t qd = smem_desc_sw128(sb, false), kd = smem_desc_sw128(sb + C::kKv, false);
        if (!wait(q_full, items & 1)) break;
        for (int q = 0; q < rounds && ok; ++q) {
#pragma unroll
          for (int x = 0; x < kTiles; ++x) {
            if (turns ? q * kTiles + x >= n : x >= tiles) continue;
            const int c = g + (turns ? q * kTiles + x : q), st = c % kStages;
            if ((x == 0 || turns) && !wait(kv_full + 8 * st, (c / kStages) & 1)) break;
            const uint32_t buffer = job & 1;
            if (job >= 2 && !wait(s_read + 8 * buffer, ((job >> 1) - 1) & 1)) break;
            ++job;
            tc_fence_after();
            if (leader) {
              const uint32_t at = (uint32_t)st * (C::kStage >> 4), qt = turns ? 0u : (uint32_t)x * (C::kQTile >> 4);
#pragma unroll
              for (int k = 0; k < HD / 16; ++k)
                tc_mma(tmem + C::s_col(buffer), qd + qt + (((k / 4) * 16384 + 32 * (k % 4)) >> 4),
                       kd + at + (((k / 4) * 8192 + 32 * (k % 4)) >> 4), id_s, k > 0 ? 1u : 0u);
              tc_commit(s_full + 8 * x);
            }
            __syncwarp();
          }
        }
      } else {
        const uint64_t vd = smem_desc_sw128(sb + C::kKv + C::kKvTile, true);
        for (int q = 0; q < rounds && ok; ++q) {
#pragma unroll
          for (int x = 0; x < kTiles; ++x) {
            if (turns ? q * kTiles + x >= n : x >= tiles) continue;
            const int c = g + (turns ? q * kTiles + x : q), st = c % kStages;
            if (!wait(p_ready + 8 * x, (done[x] + q) & 1)) break;
            tc_fence_after();
            if (leader) {
              const uint32_t at = (uint32_t)st * (C::kStage >> 4);
#pragma unroll
              for (int u = 0; u < C::kSub; ++u)
#pragma unroll
                for (int k = 0; k < 8; ++k)         // (keys 16 k .. of the first parts, then of the second)
                  tc_mma_tmem_a(tmem + C::o_col(x) + 64 * u, tmem + C::p_col(x) + 8 * k,
                                vd + at + ((u * 8192 + 2048 * (k & 3)) >> 4), id_pv, (q > 0 || k > 0) ? 1u : 0u);
              tc_commit(pv_done + 8 * x);
              if (turns || x == tiles - 1) tc_commit(kv_empty + 8 * st);
            }
            __syncwarp();
          }
        }
      }
      ++items;
#pragma unroll
      for (int x = 0; x < kTiles; ++x)
        done[x] += turns ? (uint32_t)((n + kTiles - 1 - x) / kTiles) : x < tiles ? (uint32_t)n : 0u;
      g += n;
    }
  } else if (warp < C::kSoftWarps) {
    // ---- softmax and epilogue: thread <-> row (TMEM lane) r of slot x
    const int x = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t t_o = trow + C::o_col(x);
    const float sc = p.scale_log2;
    int g = 0, items = 0;
    uint32_t done = 0, before = 0;                 // jobs of this slot so far; of all slots
    bool ok = true;
    auto wait_all = [&](uint32_t bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, TI_DEVERR_PREFILL_WAIT));
    };
    while (true) {
      // (a wait that gave up here ends all softmax warps at the barrier below, with no chunks in between)
      if (!wait_all(item_full + 8 * (items % kRing), (items / kRing) & 1)) ok = false;
      const Item& it = s_item[items % kRing];
      if (ok && it.tiles == 0) break;
      const bool turns = it.tiles == 1;
      const int n = ok ? it.c1 - it.c0 : 0;
      // this thread's row: node, its query row, head within the group, and whether there is one
      struct Row { int64_t t; int node, h; bool mine; };
      auto row = [&]() {
        const int R = (it.tile0 + (turns ? 0 : x)) * 128 + r, node = R / p.group;
        return Row{(int64_t)it.row0 + node, node, R - node * p.group, node < it.nodes && (turns || x < it.tiles)};
      };
      // Q: this thread's row of the tile (zeros where there is none), swizzled, K-major; the first mask words
      // wait in shared memory for the chunks that need them.  One trip to memory for both
      if (ok) {
        const Row w = row();
        const bool fill = turns ? x == 0 : x < it.tiles;
        uint2 first = make_uint2(0u, 0u);
        uint4 v[HD / 8];
        if (w.mine && p.masks) {
          const uint32_t* src = reinterpret_cast<const uint32_t*>(p.masks) + w.t * p.mask_words;
          first.x = src[0];
          if (p.mask_words > 1) first.y = src[1];
        }
        const uint4* src = reinterpret_cast<const uint4*>((const T*)p.q + w.t * p.q_stride +
                                                          (int64_t)(it.kvh * p.group + w.h) * HD);
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) v[c] = w.mine && fill ? src[c] : make_uint4(0u, 0u, 0u, 0u);
        s_mask[x * 128 + r] = first;               // (read by this thread only)
        if (fill) {
#pragma unroll
          for (int c = 0; c < HD / 8; ++c)
            *reinterpret_cast<uint4*>(smem + (turns ? 0 : x) * C::kQTile + (c >> 3) * 16384 + r * 128 +
                                      (((c & 7) ^ (r & 7)) << 4)) = v[c];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      // V of a chunk that some rows do not see all of, by the slot's 128 threads: nothing behind the end
      // or of absent blocks, no non-finite elements of drafts (true: there were some)
      auto mend_values = [&](int st, int k0, int flags) {
        bool found = false;
        for (int i = r; i < C::kSub * kChunk * 8; i += 128) {
          const int row = (i >> 3) & (kChunk - 1), key = k0 + row;
          uint4* at = reinterpret_cast<uint4*>(smem + C::kKv + st * C::kStage + C::kKvTile + i * 16);
          if (key >= it.keys || !((flags >> (row / kBlock)) & 1)) {
            *at = make_uint4(0u, 0u, 0u, 0u);
          } else if (key >= it.ctx) {
            constexpr uint32_t kInf = kBf16 ? 0x7F80u : 0x7C00u;
            uint4 v = *at;
            uint32_t e[4] = {v.x, v.y, v.z, v.w};
            bool bad = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const bool lo = (e[k] & kInf) == kInf, hi = (e[k] >> 16 & kInf) == kInf;
              e[k] &= (lo ? 0u : 0x0000FFFFu) | (hi ? 0u : 0xFFFF0000u);
              bad |= lo | hi;
            }
            if (bad) *at = make_uint4(e[0], e[1], e[2], e[3]);
            found |= bad;
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        return found;
      };
      const int step = turns ? kTiles : 1;
      const int jobs = !ok ? 0 : turns ? (n + kTiles - 1 - x) / kTiles : x < it.tiles ? n : 0;
      const bool idle = !__any_sync(0xffffffffu, row().mine);   // a warp without rows only keeps step
      float m = -INFINITY, l = 0.f;
      bool dirty = false;
      for (int k = 0, c = turns ? x : 0; k < jobs && ok; ++k, c += step) {
        const int st = (g + c) % kStages;
        const uint32_t par = (done + k) & 1;
        const uint32_t buffer = (before + (uint32_t)(turns ? c : c * it.tiles + x)) & 1;
        // (the chunk has been there since before its scores: no wait, but the loader's word)
        const bool there = mbar_try_wait(s_full + 8 * x, par) & mbar_try_wait(kv_full + 8 * st, ((g + c) / kStages) & 1);
        if (!__all_sync(0xffffffffu, there) &&
            !(wait_all(s_full + 8 * x, par) && wait_all(kv_full + 8 * st, ((g + c) / kStages) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (idle) {
          const int flags = s_ok[st];
          if ((flags & 16) && (x == 0 || turns)) dirty |= mend_values(st, (it.c0 + c) * kChunk, flags);
          __syncwarp();
          if (lane == 0) mbar_arrive(s_read + 8 * buffer);
          // (behind the last job's product: this job's phase of p_ready must not begin earlier)
          if (k >= 1 && !wait_all(pv_done + 8 * x, (done + k - 1) & 1)) { ok = false; break; }
          if (lane == 0) mbar_arrive(p_ready + 8 * x);
          continue;
        }
        float sv[kChunk];
        uint32_t sr[kChunk];
        tmem_ld64_start(trow + C::s_col(buffer), sr);
        const int flags = s_ok[st];
        tmem_ld64_end(sr, sv);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_read + 8 * buffer);
        if (flags & 16) {
          const Row w = row();
          if (x == 0 || turns) dirty |= mend_values(st, (it.c0 + c) * kChunk, flags);
          const uint64_t see = w.mine ? seen(p, it, w.t, w.node, (it.c0 + c) * kChunk, flags & 15, s_mask[x * 128 + r]) : 0ull;
          const uint32_t lo = (uint32_t)see, hi = (uint32_t)(see >> 32);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            sv[i] = (lo >> i) & 1 ? sv[i] : -INFINITY;
            sv[32 + i] = (hi >> i) & 1 ? sv[32 + i] : -INFINITY;
          }
        }
        float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kChunk; i += 2) mxs[i / 2 % 4] = max3(mxs[i / 2 % 4], sv[i], sv[i + 1]);
        const float mx = max3(fmaxf(mxs[0], mxs[1]), mxs[2], mxs[3]) * sc;
        const bool outgrown = __any_sync(0xffffffffu, mx > m + 8.f);
        float alpha = 1.f;
        if (outgrown && mx > m + 8.f) {            // (from no key at all: alpha 0 of zeros)
          alpha = m == -INFINITY ? 0.f : fast_exp2(m - mx);
          m = mx;
        }
        if (outgrown && k >= 1) {                  // O at rest, for a rescale (here, while the weights need no registers)
          if (!wait_all(pv_done + 8 * x, (done + k - 1) & 1)) { ok = false; break; }
          tc_fence_after();
          float ov[32];
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            tmem_ld32(t_o + d, ov);
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] *= alpha;
            tmem_st32(t_o + d, ov);
          }
        }
        const float off = kPScale - (m == -INFINITY ? 0.f : m);
        const uint64_t sc2 = pair(sc, sc), off2 = pair(off, off);
        // the chunk's sum first, in four chains of pairs: a long row's total stays exact enough
        uint64_t sums[4] = {0, 0, 0, 0};
        uint32_t pk[kChunk];                       // first parts, then what their rounding left
#pragma unroll
        for (int i = 0; i < kChunk; i += 2) {
          const float2 e = unpair(fma2(pair(sv[i], sv[i + 1]), sc2, off2));
          const float p0 = fast_exp2(e.x), p1 = fast_exp2(e.y);
          sums[i / 2 % 4] = add2(sums[i / 2 % 4], pair(p0, p1));
          pk[i / 2] = Elem<T>::pack2(p0, p1);
          const float2 h = Elem<T>::unpack2(pk[i / 2]);
          const float2 rest = unpair(fma2(pair(h.x, h.y), pair(-1.f, -1.f), pair(p0, p1)));
          pk[kChunk / 2 + i / 2] = Elem<T>::pack2(rest.x, rest.y);
        }
        const float2 t2 = unpair(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])));
        l = l * alpha + (t2.x + t2.y);
        // P V of the slot's last job has long been done: P's place is free
        if (k >= 1 && !wait_all(pv_done + 8 * x, (done + k - 1) & 1)) { ok = false; break; }
        tmem_st32_u(trow + C::p_col(x), pk);
        tmem_st32_u(trow + C::p_col(x) + 32, pk + 32);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + 8 * x);
      }
      if (ok && jobs > 0 && !wait_all(pv_done + 8 * x, (done + jobs - 1) & 1)) ok = false;
      tc_fence_before();
      // (slots with a job only, which are those that slot 0 reads: a slot without one waits for nothing that
      // this item's slot 0 does last, and may be here while it still reads the last item's entries)
      if (turns && jobs > 0) s_ml[x * 128 + r] = make_float2(m, l);
      if (bar_or(1, C::kSoftWarps * 32, !ok)) break;       // (a wait gave up: everyone leaves)
      dirty = bar_or(1, C::kSoftWarps * 32, dirty);
      tc_fence_after();
      done += (uint32_t)jobs;
      before += (uint32_t)(turns ? n : n * it.tiles);
      ++items;
      // ---- a tile's result: (m, l) here, O in tensor memory
      if (turns ? x == 0 : x < it.tiles) {
        const Row me = row();
        const bool mine = me.mine;
        const int64_t t = me.t;
        const int node = me.node, h = me.h;
        const int slots = turns ? min(kTiles, n) : 1;
        if (slots > 1) {
          float ms[kTiles], f[kTiles], M = m;
#pragma unroll
          for (int y = 1; y < kTiles; ++y) {
            const float2 o = y < slots ? s_ml[y * 128 + r] : make_float2(-INFINITY, 0.f);
            ms[y] = o.x;
            f[y] = o.y;
            M = fmaxf(M, o.x);
          }
          // (a part without a finite score holds zeros, or NaN)
          const float f0 = m == -INFINITY ? 1.f : fast_exp2(m - M);
          l *= f0;
#pragma unroll
          for (int y = 1; y < kTiles; ++y) {
            const float w = ms[y] == -INFINITY ? 1.f : fast_exp2(ms[y] - M);
            l += w * f[y];
            f[y] = w;
          }
          m = M;
          if (!idle) {
#pragma unroll 1
            for (int d = 0; d < HD; d += 32) {
              float a[32], b[32];
              tmem_ld32(t_o + d, a);
#pragma unroll
              for (int i = 0; i < 32; ++i) a[i] *= f0;
#pragma unroll
              for (int y = 1; y < kTiles; ++y)
                if (y < slots) {
                  tmem_ld32(trow + C::o_col(y) + d, b);
#pragma unroll
                  for (int i = 0; i < 32; ++i) a[i] = fmaf(f[y], b[i], a[i]);
                }
              tmem_st32(t_o + d, a);
            }
          }
        }
        if (dirty && !idle) {
          // non-finite values of drafts were left out of the products: the rows that see them get them
          for (int d = 0; d < HD; d += 32) {
            float ov[32];
            tmem_ld32(t_o + d, ov);
            for (int c = max(it.c0, it.ctx / kChunk); c < it.c1; ++c) {
              int have = 0;
              for (int b = 0; b < 4; ++b) {
                const int64_t blk = (int64_t)c * 4 + b;
                if (it.table && blk * kBlock < it.keys && it.table[blk] >= 0 && it.table[blk] < p.num_blocks) have |= 1 << b;
              }
              const uint64_t see = mine ? seen(p, it, t, node, c * kChunk, have, s_mask[x * 128 + r]) : 0ull;
              for (int i = 0; i < kChunk; ++i) {
                const int key = c * kChunk + i;
                if (!((see >> i) & 1) || key < it.ctx) continue;
                const T* v = (const T*)p.v + (((int64_t)it.table[key / kBlock] * p.KVH + it.kvh) * kBlock + key % kBlock) * HD + d;
                for (int e = 0; e < 32; ++e) {
                  const float val = Elem<T>::to_f(v[e]);
                  if (!(fabsf(val) < INFINITY)) {
#pragma unroll
                    for (int q = 0; q < 32; ++q) ov[q] += q == e ? val : 0.f;
                  }
                }
              }
            }
            __syncwarp();
            tmem_st32(t_o + d, ov);
          }
        }
        // ---- parts of a unit that other CTAs hold: joined in pairs, first index by first index
        bool last = true;
        if (it.parts > 1) {
          int i = blockIdx.x - it.first;
          auto part_of = [&](int j) {              // a unit's first part and the others: a CTA may have one of each
            return p.parts + (((int64_t)(it.first + j) * 2 + (j > 0)) * kTiles + x) * C::kPart;
          };
          for (int stride = 1; stride < it.parts; stride <<= 1) {
            const int left = i & ~(2 * stride - 1), right = left + stride;
            if (right >= it.parts) { i = left; continue; }
            const bool is_right = i != left;
            unsigned* counter = p.counters + (it.first + right) * kTiles + x;
            // the other half is there: nothing has to be written; else this half goes to memory, and the
            // word says whether the other one has come meanwhile
            bar_sync(2 + x, 128);                  // (the word below has been read by all)
            if (quad == 0 && lane == 0) {
              unsigned there;
              asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(there) : "l"(counter) : "memory");
              s_flag[x] = there == p.call;
            }
            bar_sync(2 + x, 128);
            bool second = s_flag[x] != 0;
            if (!second) {
              float* own = part_of(i);
              if (!idle) {
#pragma unroll 1
                for (int d = 0; d < HD; d += 32) {
                  float ov[32];
                  tmem_ld32(t_o + d, ov);
                  if (mine) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                      __stcg(reinterpret_cast<float4*>(own) + ((d + e) / 4) * 128 + r,
                             make_float4(ov[e], ov[e + 1], ov[e + 2], ov[e + 3]));
                  }
                  __syncwarp();
                }
                if (mine) __stcg(reinterpret_cast<float2*>(own + 128 * HD) + r, make_float2(m, l));
              }
              bar_sync(2 + x, 128);
              if (quad == 0 && lane == 0) {
                unsigned old;
                asm volatile("atom.exch.acq_rel.gpu.global.b32 %0, [%1], %2;" : "=r"(old) : "l"(counter), "r"(p.call) : "memory");
                s_flag[x] = old == p.call;
              }
              bar_sync(2 + x, 128);
              second = s_flag[x] != 0;
            }
            if (!second) { last = false; break; }
            if (quad == 0 && lane == 0) *counter = 0u;
            const float* other = part_of(is_right ? left : right);
            if (!idle) {
              float2 o = make_float2(-INFINITY, 0.f);
              if (mine) o = __ldcg(reinterpret_cast<const float2*>(other + 128 * HD) + r);
              const float M = fmaxf(m, o.x);
              const float fa = m == -INFINITY ? 1.f : fast_exp2(m - M), fb = o.x == -INFINITY ? 1.f : fast_exp2(o.x - M);
              // left half first, whoever joins
              l = is_right ? fmaf(fb, o.y, fa * l) : fmaf(fa, l, fb * o.y);
              m = M;
#pragma unroll 1
              for (int d = 0; d < HD; d += 32) {
                float4 b[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  b[e] = mine ? __ldcg(reinterpret_cast<const float4*>(other) + (d / 4 + e) * 128 + r) : make_float4(0.f, 0.f, 0.f, 0.f);
                float a[32];
                tmem_ld32(t_o + d, a);
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float4& q = b[e / 4];
                  const float y = e % 4 == 0 ? q.x : e % 4 == 1 ? q.y : e % 4 == 2 ? q.z : q.w;
                  a[e] = is_right ? fmaf(fb, y, fa * a[e]) : fmaf(fa, a[e], fb * y);
                }
                __syncwarp();
                tmem_st32(t_o + d, a);
              }
            }
            i = left;
          }
        }
        if (last && !idle) {
          const bool none = m == -INFINITY && l == 0.f;
          const float inv = none ? 0.f : 1.f / l;
          T* dst = (T*)p.out + t * p.out_stride + (int64_t)(it.kvh * p.group + h) * HD;
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            float ov[32];
            tmem_ld32(t_o + d, ov);
            if (mine) {
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                uint4 u;
                u.x = Elem<T>::pack2(ov[e] * inv, ov[e + 1] * inv);
                u.y = Elem<T>::pack2(ov[e + 2] * inv, ov[e + 3] * inv);
                u.z = Elem<T>::pack2(ov[e + 4] * inv, ov[e + 5] * inv);
                u.w = Elem<T>::pack2(ov[e + 6] * inv, ov[e + 7] * inv);
                *reinterpret_cast<uint4*>(dst + d + e) = none ? make_uint4(0u, 0u, 0u, 0u) : u;
              }
            }
            __syncwarp();
          }
          if (mine && p.lse)
            p.lse[t * p.NH + it.kvh * p.group + h] =
                none ? -INFINITY : (m == -INFINITY ? l : (m + log2f(l) - kPScale) * 0.6931471805599453f);
        }
        tc_fence_before();
      }
      g += n;
      // (the next item's products wait for q_full, to which every softmax warp arrives: O of the other
      // slots, Q's tiles and the sums of slots that have a product to wait for are free by then)
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kScoreWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int HD>
static int launch(const Params& p, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};          // devices whose limit has been raised
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(attention_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               Cfg<HD>::smem(kMaxSeqs));
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return set_cuda_error(e, "cudaFuncSetAttribute(tree attention)");
    }
    ready.fetch_or(bit, std::memory_order_release);
  }
  return launch_kernel("tree attention launch", attention_kernel<T, HD>, dim3(kCtas), dim3(Cfg<HD>::kThreads),
                       Cfg<HD>::smem(p.seqs), s, 1, km, vm, p);
}

}  // namespace tree
}  // namespace ti

using namespace ti;

extern "C" size_t ti_tree_attention_workspace_bytes(int num_heads, int num_kv_heads, int head_dim) {
  if (num_heads <= 0 || num_kv_heads <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  // counters, then two parts a CTA and slot
  const size_t part = head_dim == 64 ? tree::Cfg<64>::kTiles * tree::Cfg<64>::kPart
                                     : tree::Cfg<128>::kTiles * tree::Cfg<128>::kPart;
  return tree::kCounterBytes + (size_t)tree::kCtas * 2 * part * 4;
}

extern "C" int ti_tree_attention(void* out, int64_t out_tok_stride, float* lse, const void* q,
                                 int64_t q_tok_stride, const void* k_cache, const void* v_cache,
                                 int64_t num_blocks, const int32_t* block_tables, int64_t bt_stride,
                                 int num_rows, int max_blocks_per_seq, const int32_t* row_index,
                                 const int32_t* context_lens, const int32_t* cu_seqlens, int num_seqs,
                                 int num_tokens, const int32_t* masks, int mask_words, int num_heads,
                                 int num_kv_heads, int head_dim, int block_size, int dtype,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (num_seqs == 0 || num_tokens == 0) return TI_OK;
  if (!out || !q || !k_cache || !v_cache || !block_tables || !context_lens || !cu_seqlens || !workspace ||
      num_seqs < 0 || num_tokens < 0 || mask_words < 0 || (mask_words > 0 && !masks))
    return set_error(TI_ERR_INVALID_ARGUMENT, "tree attention: null pointer or negative size");
  if (num_blocks <= 0 || max_blocks_per_seq <= 0 || num_rows <= 0 || num_kv_heads <= 0 || num_heads <= 0 ||
      num_heads % num_kv_heads || (!row_index && num_rows < num_seqs))
    return set_error(TI_ERR_INVALID_ARGUMENT,
                     "tree attention: bad table, pool size or head counts (num_heads must be a multiple of num_kv_heads)");
  if (num_heads / num_kv_heads > tree::kMaxGroup)
    return set_error(TI_ERR_UNSUPPORTED, "tree attention: at most 16 query heads per kv head");
  if ((head_dim != 64 && head_dim != 128) || block_size != tree::kBlock)
    return set_error(TI_ERR_UNSUPPORTED, "tree attention: head_dim must be 64 or 128, block_size 16");
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_FP16)
    return set_error(TI_ERR_UNSUPPORTED, "tree attention: dtype must be bf16 or fp16");
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) |
        reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
        reinterpret_cast<uintptr_t>(workspace)) & 15) || (out_tok_stride % 8) || (q_tok_stride % 8))
    return set_error(TI_ERR_INVALID_ARGUMENT, "tree attention: tensors must be 16-byte aligned");
  if (workspace_bytes < ti_tree_attention_workspace_bytes(num_heads, num_kv_heads, head_dim))
    return set_error(TI_ERR_WORKSPACE, "tree attention: workspace too small");
  const int group = num_heads / num_kv_heads;
  const int64_t most_jobs = ((int64_t)num_tokens * group / 128 + num_seqs) * num_kv_heads *
                            (2 * ((int64_t)max_blocks_per_seq / 4 + 1) + tree::kUnitJobs);
  if (num_seqs > tree::kMaxSeqs || most_jobs >= (int64_t)1 << 31 ||
      (int64_t)max_blocks_per_seq * block_size >= (int64_t)1 << 31 ||
      (int64_t)num_tokens * num_heads >= (int64_t)1 << 31 ||
      num_blocks * num_kv_heads * block_size >= (int64_t)1 << 31)
    return set_error(TI_ERR_UNSUPPORTED, "tree attention: at most 4096 sequences, and sizes within 31 bits");
  tree::Params p{out, q, v_cache, lse, out_tok_stride, q_tok_stride, num_blocks, bt_stride, block_tables, row_index,
                 context_lens, cu_seqlens, mask_words ? masks : nullptr,
                 reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + tree::kCounterBytes),
                 static_cast<unsigned*>(workspace), num_seqs, num_tokens, num_rows, max_blocks_per_seq, num_heads,
                 num_kv_heads, group, mask_words, 1.4426950408889634f / sqrtf((float)head_dim), 0};
  static std::atomic<unsigned> calls{0};
  do p.call = calls.fetch_add(1, std::memory_order_relaxed) + 1;
  while (p.call == 0);
  CUtensorMap km, vm;
  const cuuint64_t dims[2] = {(cuuint64_t)head_dim, (cuuint64_t)(num_blocks * num_kv_heads * block_size)};
  const cuuint64_t strides[1] = {(cuuint64_t)head_dim * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)tree::kBlock}, es[2] = {1, 1};
  const CUtensorMapDataType type =
      dtype == TI_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (int rc = encode_tensor_map_2d(&km, type, const_cast<void*>(k_cache), dims, strides, box, es,
                                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
    return rc;
  if (int rc = encode_tensor_map_2d(&vm, type, const_cast<void*>(v_cache), dims, strides, box, es,
                                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
    return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == TI_DTYPE_BF16)
    return head_dim == 64 ? tree::launch<__nv_bfloat16, 64>(p, km, vm, s) : tree::launch<__nv_bfloat16, 128>(p, km, vm, s);
  return head_dim == 64 ? tree::launch<__half, 64>(p, km, vm, s) : tree::launch<__half, 128>(p, km, vm, s);
}
