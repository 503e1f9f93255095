// Ragged causal prefill attention over the 4-bit paged KV cache, tcgen05.  Format: kv4.cuh.
//
// out = softmax(q K^T / sqrt(D), keys 0 .. own position) V for chunks of query tokens whose K and V are
// already in the cache.
//
// A tile is 128 rows: the query heads of one kv head (a power of two of slots, at most 16) times 128 /
// slots tokens.  One CTA takes up to three tiles of neighbouring tokens (two for D = 128: what tensor
// memory holds) and a range of keys; they share each 64-key chunk, which three warps read as codes
// (asynchronous copies, three chunks ahead) and write to shared memory as half precision -- exact, 2.25
// times less to read than 16-bit keys and no scratch copy of the cache.  Per chunk and tile:
//   S = Q K^T   M 128, N 64, into TMEM; the softmax warps free it once it is in registers, and S of the
//               next chunk is computed under their arithmetic;
//   softmax     one row per thread: causal mask, a running max that is kept until a row's grows by more
//               than 2^8 (then O is rescaled in TMEM), P = 2^(s - m) as half precision back into TMEM,
//               the A operand of the next product;
//   O += P V    A from TMEM, V read in place as an MN-major operand; fp32 O in TMEM.
// bf16 queries are scaled by a power of two per row as in the decode kernel; P is held times 2^7 (at
// most 2^15; steps of 2^-31), its sum taken before rounding.
//
// Bound: four chunks of 1024 tokens behind prefixes up to 32767 (14 heads over 2, D = 64) take 414 us.
// The exponentials alone would take 230 (one warp instruction in 8 clocks of a scheduler: 512 clocks a
// tile and chunk), the MMAs 146 at their full rate.  The three warps of a scheduler that have them to
// do mostly run in step, so for half of a chunk's clocks the exponential unit is busy, and half it
// waits for their other work: waits, tensor memory, the max.  What was measured on the way: two tiles a
// CTA with double-buffered scores 473 us; two threads a row 534; three tiles with a fourth loader warp,
// 17 warps of 96 registers instead of 16 of 128, 436; the max taken beside the exponentials, which then
// may have to be taken again, 444.  An order of the warps by flags in shared memory cost registers and
// more time than it gave (524 to 765 against 436).
//
// Work: the host cuts the keys of long sequences into ranges of the same size, longest first, so that a
// few long prefixes fill the GPU; tiles cut into several ranges leave un-normalised partials that
// merge_kernel joins in order.
//
// A key that is masked in some row of a tile and is NaN costs that row nothing: its score is replaced.
// A masked value that is NaN would (0 * NaN): NaN groups of V go into the product as zeros, and the
// first position of one is kept per 16 dims; rows at or behind it get NaN there.
#include <algorithm>
#include <atomic>

#include "capi_internal.h"
#include "common.cuh"
#include "kv4.cuh"
#include "softmax_tile.cuh"
#include "tcgen05.cuh"

namespace ti {
namespace kv4 {
namespace pre {

constexpr int kChunk = 64;                       // keys per step
constexpr int kStages = 3;                       // chunks of K and V in half precision
constexpr int kRaw = 4;                          // chunks of codes
constexpr int kLoadWarps = 3;
constexpr int kLoaders = kLoadWarps * 32;
constexpr float kPScale = 7.f;
constexpr int kStagger = 500, kStaggerFrom = 16; // clocks, chunks
constexpr int kItemInts = 6;                     // sequence, first token, key range, part or -1, tiles
constexpr int kMergeInts = 5;                    // sequence, first token, first part, parts, tiles

struct Params {
  void* out;
  const void* q;
  const uint8_t* pool;
  int64_t out_stride, q_stride, num_blocks, bt_stride;
  const int32_t *tables, *row_index, *start_pos, *cu_seqlens, *items;
  float* parts;
  int NH, KVH, group, slots_log2, max_blocks;
  float scale_log2;
};

template <int HD>
struct Smem {
  static constexpr int kSub = HD / 64;           // 64-dim sub-tiles of a row
  static constexpr int kQTile = kSub * 16384;
  static constexpr int kKvTile = kSub * 8192;    // K or V of a chunk
  static constexpr int kRawChunk = 4 * Tile<HD>::kBytes;
  static constexpr int kTiles = HD == 64 ? 3 : 2;                // query tiles of a CTA
  static constexpr int kSoftWarps = 4 * kTiles;
  static constexpr int kThreads = (kSoftWarps + kLoadWarps + 1) * 32;
  static constexpr int kQ = 0, kKv = kTiles * kQTile, kRawAt = kKv + kStages * 2 * kKvTile;
  // TMEM columns: scores, weights (half precision, two a column) and O of every tile
  static __device__ __forceinline__ uint32_t s_col(int x) { return 64 * x; }
  static __device__ __forceinline__ uint32_t p_col(int x) { return 64 * kTiles + 32 * x; }
  static __device__ __forceinline__ uint32_t o_col(int x) { return 96 * kTiles + HD * x; }
  static_assert((96 + HD) * kTiles <= 512, "tensor memory");
  static constexpr int kInv = kRawAt + kRaw * kRawChunk;         // [kTiles][128] floats
  static constexpr int kNan = kInv + kTiles * 512;                       // [HD/16] ints
  static constexpr int kOk = kNan + 64;                          // [8] ints
  static constexpr int kIds = kOk + 64;                          // [8][4] ints
  static constexpr int kBars = kIds + 128;
  static constexpr int kTotal = kBars + 192 + 1024;              // and alignment slack
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

template <typename T, int HD>
__global__ void __launch_bounds__(Smem<HD>::kThreads, 1) prefill_kernel(const __grid_constant__ Params p) {
  using S = Smem<HD>;
  constexpr int kThreads = S::kThreads, kSoftWarps = S::kSoftWarps;
  using L = Tile<HD>;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const uint32_t sb = smem_u32(smem);
  const uint32_t kv_full = sb + S::kBars, kv_empty = kv_full + 8 * kStages;
  // per tile, a phase per chunk: scores written, scores read, weights written, P V done
  const uint32_t s_full = kv_empty + 8 * kStages, s_read = s_full + 8 * S::kTiles;
  const uint32_t p_ready = s_read + 8 * S::kTiles, pv_done = p_ready + 8 * S::kTiles;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(smem + S::kBars + 160);
  float* s_inv = reinterpret_cast<float*>(smem + S::kInv);
  int* s_nan = reinterpret_cast<int*>(smem + S::kNan);
  int* s_ids = reinterpret_cast<int*>(smem + S::kIds);
  volatile int* s_ok = reinterpret_cast<int*>(smem + S::kOk);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  constexpr int kMmaWarp = kSoftWarps + kLoadWarps;

  if (warp == kMmaWarp) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        mbar_init(kv_full + 8 * i, kLoaders);
        mbar_init(kv_empty + 8 * i, 1);
      }
      for (int i = 0; i < S::kTiles; ++i) {
        mbar_init(s_full + 8 * i, 1);
        mbar_init(s_read + 8 * i, 4);
        mbar_init(p_ready + 8 * i, 4);
        mbar_init(pv_done + 8 * i, 1);
      }
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(smem_u32(tslot), 512);
  }
  if (tid < HD / 16) s_nan[tid] = 0x7FFFFFFF;
  pdl_wait();

  const int kvh = blockIdx.x % p.KVH;
  const int32_t* item = p.items + (int64_t)(blockIdx.x / p.KVH) * kItemInts;
  const int seq = item[0], q0 = item[1], kb = item[2], ke = item[3], part = item[4];
  const int tile_tokens = 128 >> p.slots_log2;
  const int row0 = p.cu_seqlens[seq], count = p.cu_seqlens[seq + 1] - row0;
  const int start = p.start_pos[seq], cached = start + count;
  const int ntiles = min(min(item[5], S::kTiles), (count - q0 + tile_tokens - 1) / tile_tokens);
  const int n = (ke - kb + kChunk - 1) / kChunk;
  const int32_t* table = p.tables + (int64_t)(p.row_index ? p.row_index[seq] : seq) * p.bt_stride;

  // Q: row r of a tile = head slot r % slots of token r / slots (zeros beyond the group or the chunk)
  for (int i = tid; i < ntiles * 128 * (HD / 8); i += kThreads) {
    const int c = i % (HD / 8), r = (i / (HD / 8)) & 127, x = i / (128 * (HD / 8));
    const int h = r & ((1 << p.slots_log2) - 1), t = q0 + x * tile_tokens + (r >> p.slots_log2);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (h < p.group && t < count)
      v = *reinterpret_cast<const uint4*>((const T*)p.q + (int64_t)(row0 + t) * p.q_stride +
                                          (int64_t)(kvh * p.group + h) * HD + c * 8);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      // (the HD/8 threads of a row are neighbouring lanes of one warp: kThreads and the loop's bound
      // are multiples of 32)
      uint32_t w[4] = {v.x, v.y, v.z, v.w}, top = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7FFFu, (w[k] >> 16) & 0x7FFFu));
#pragma unroll
      for (int d = HD / 16; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
      const int e = min(max((int)(top >> 7), 15), 254);
      const float mul = __uint_as_float((uint32_t)(254 + 14 - e) << 23);       // 2^(14 - (e - 127))
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = Elem<T>::unpack2(w[k]);
        w[k] = Elem<__half>::pack2(f.x * mul, f.y * mul);
      }
      v = make_uint4(w[0], w[1], w[2], w[3]);
      if (c == 0) s_inv[x * 128 + r] = __uint_as_float((uint32_t)(e - 14) << 23);
    } else if (c == 0) {
      s_inv[x * 128 + r] = 1.f;
    }
    *reinterpret_cast<uint4*>(smem + S::kQ + x * S::kQTile + (c >> 3) * 16384 + r * 128 +
                              (((c & 7) ^ (r & 7)) << 4)) = v;
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  pdl_launch_dependents();
  if (warp >= kSoftWarps && warp < kMmaWarp) {
    // ---- loaders: codes -> half precision
    const int lt = tid - kSoftWarps * 32;
    constexpr int kUnits = S::kRawChunk / 16, kTileUnits = L::kBytes / 16;
    // Block ids come through a ring of eight chunks in shared memory, copied there seven chunks ahead
    // and looked at where they are used.  (A table read per copy put its latency into every chunk: 796
    // us instead of 770 at four chunks of 1024; ids that pass through a register are waited for
    // where they are loaded, which kept the softmax waiting for the loaders: 536 instead of 502.)
    auto want_id = [&](int c, int b) {              // of block b of chunk c
      const int blk = kb / kBlock + c * 4 + b, at = (c & 7) * 4 + b;
      if (c < n && blk < p.max_blocks && (int64_t)blk * kBlock < cached)
        cp_async4(sb + S::kIds + at * 4, table + blk);
      else
        s_ids[at] = -1;
    };
    const uint32_t num_blocks = (uint32_t)min(p.num_blocks, (int64_t)0x7FFFFFFF);
    auto valid = [&](int id) { return (uint32_t)id < num_blocks; };
    if (lt < 28) want_id(lt / 4, lt % 4);
    asm volatile("cp.async.wait_all;" ::: "memory");
    asm volatile("bar.sync 1, 96;" ::: "memory");
    auto issue = [&](int c) {
      const uint32_t raw = sb + S::kRawAt + (c % kRaw) * S::kRawChunk;
      constexpr int kEach = kUnits / kLoaders;
      static_assert(kUnits % kLoaders == 0, "whole rounds of copies");
      int id[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        id[i] = s_ids[(c & 7) * 4 + (lt + i * kLoaders) / kTileUnits];
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int u = lt + i * kLoaders;
        if (valid(id[i]))
          cp_async16(raw + u * 16, p.pool + ((int64_t)id[i] * p.KVH + kvh) * L::kBytes + (u % kTileUnits) * 16);
      }
    };
    for (int c = 0; c < kRaw - 1; ++c) {
      issue(c);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // a piece is 32 dims, two scale groups, of a token's K or V; whole warps take whole runs of them
    constexpr int kPieces = kChunk * 2 * (HD / 32), kRounds = (kPieces + kLoaders - 1) / kLoaders;
    // after a wait that gave up the loop goes on without waiting: all the threads keep meeting at the
    // barrier, and the results are void anyway
    bool ok = true;
    for (int c = 0; c < n; ++c) {
      const int st = c % kStages;
      asm volatile("cp.async.wait_group %0;" ::"n"(kRaw - 2) : "memory");
      asm volatile("bar.sync 1, 96;" ::: "memory");   // everyone's copies; chunk c-1 was read
      issue(c + kRaw - 1);
      if (warp == kMmaWarp - 1) {                // (the warp with the fewest pieces)
        if (lane < 4) want_id(c + 7, lane);      // in chunk c-1's place: every thread is past it
        const uint32_t have = __ballot_sync(0xffffffffu, lane < 4 && valid(s_ids[(c & 7) * 4 + (lane & 3)]));
        if (lane == 0) s_ok[c & 7] = (int)(have & 15u);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      const uint8_t* raw = smem + S::kRawAt + (c % kRaw) * S::kRawChunk;
      const uint32_t dst = sb + S::kKv + st * 2 * S::kKvTile;
      // (all reads before the first write: the compiler keeps their order)
      uint4 w[kRounds];
      uint32_t by[kRounds][2];
#pragma unroll
      for (int i = 0; i < kRounds; ++i) {
        const int e = lt + i * kLoaders, tok = e / (HD / 32) % kChunk, d0 = e % (HD / 32) * 32;
        const bool v = e / (HD / 32) >= kChunk;
        const uint8_t* tile = raw + (tok / kBlock) * L::kBytes;
        w[i] = make_uint4(0u, 0u, 0u, 0u);
        by[i][0] = by[i][1] = 0;
        if (e < kPieces && kb + c * kChunk + tok < cached && valid(s_ids[(c & 7) * 4 + tok / kBlock])) {
          w[i] = *reinterpret_cast<const uint4*>(tile + (v ? L::kV : L::kK) + tok % kBlock * L::kRow + d0 / 2);
#pragma unroll
          for (int g = 0; g < 2; ++g)
            by[i][g] = tile[(v ? L::kVs : L::kKs) + (d0 / 16 + g) * kBlock + tok % kBlock];
        }
      }
      if (ok && c >= kStages && !mbar_wait(kv_empty + 8 * st, ((c / kStages) - 1) & 1, TI_DEVERR_PREFILL_WAIT)) ok = false;
#pragma unroll
      for (int i = 0; i < kRounds; ++i) {
        const int e = lt + i * kLoaders, tok = e / (HD / 32) % kChunk, d0 = e % (HD / 32) * 32;
        const bool v = e / (HD / 32) >= kChunk;
        if (e >= kPieces) break;
        if (v) {
#pragma unroll
          for (int g = 0; g < 2; ++g)
            if (by[i][g] >= 0xF8u) { atomicMin(&s_nan[d0 / 16 + g], kb + c * kChunk + tok); by[i][g] = 0; }
        }
        const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        const uint32_t row = dst + (v ? S::kKvTile : 0) + (d0 / 64) * 8192 + tok * 128;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t h[4];
          codes_to_half2(ws[k], h);
          const uint32_t s2 = by[i][k / 2] * 0x00800080u;
          const int ch = (d0 % 64) / 8 + k;
          st_shared_v4(row + ((ch ^ (tok & 7)) << 4), hmul2(h[0], s2), hmul2(h[1], s2),
                       hmul2(h[2], s2), hmul2(h[3], s2));
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(kv_full + 8 * st);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (warp == kMmaWarp) {
    // ---- MMA issue: the whole warp walks the loop and one elected lane issues, so that descriptors
    // stay in uniform registers (one lane alone took 100 clocks per MMA: 3000 a chunk)
    constexpr uint32_t id_s = idesc_f16(128, kChunk, false, false, false);
    constexpr uint32_t id_pv = idesc_f16(128, 64, false, false, true);
    const uint64_t qd = smem_desc_sw128(sb + S::kQ, false), kd = smem_desc_sw128(sb + S::kKv, false);
    const uint64_t vd = smem_desc_sw128(sb + S::kKv + S::kKvTile, true);
    const bool leader = elect_one();
    auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity, TI_DEVERR_PREFILL_WAIT); };
    auto scores = [&](int x, uint32_t stage) {
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          tc_mma(tmem + S::s_col(x), qd + ((x * S::kQTile + (k / 4) * 16384 + 32 * (k % 4)) >> 4),
                 kd + stage + (((k / 4) * 8192 + 32 * (k % 4)) >> 4), id_s, k > 0 ? 1u : 0u);
        tc_commit(s_full + 8 * x);
      }
      __syncwarp();
    };
    auto values = [&](int x, uint32_t stage, bool begin, uint32_t empty) {   // O += P V
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int u = 0; u < S::kSub; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc_mma_tmem_a(tmem + S::o_col(x) + 64 * u, tmem + S::p_col(x) + 8 * k,
                          vd + stage + ((u * 8192 + 2048 * k) >> 4), id_pv, (!begin || k > 0) ? 1u : 0u);
        tc_commit(pv_done + 8 * x);
        if (empty) tc_commit(empty);
      }
      __syncwarp();
    };
    auto full = [&](int c) { return wait(kv_full + 8 * (c % kStages), (c / kStages) & 1); };
    auto stage = [&](int c) { return (uint32_t)((c % kStages) * 2 * S::kKvTile) >> 4; };
    bool ok = full(0);
    for (int x = 0; x < ntiles; ++x) scores(x, stage(0));
    // P V of chunk c-1 and S of chunk c+1, tile by tile: a tile's weights of c-1 and its having read
    // the scores of c come one soon after the other.
    for (int c = 0; c <= n && __all_sync(0xffffffffu, ok); ++c) {   // (a wait that gave up: the error bit is set)
      for (int x = 0; x < ntiles; ++x) {
        if (c >= 1) {
          ok &= wait(p_ready + 8 * x, (c - 1) & 1);
          values(x, stage(c - 1), c == 1, x == ntiles - 1 ? kv_empty + 8 * ((c - 1) % kStages) : 0u);
        }
        if (c + 1 < n) {
          if (x == 0) ok &= full(c + 1);
          ok &= wait(s_read + 8 * x, c & 1);
          scores(x, stage(c + 1));
        }
      }
    }
  } else if (warp / 4 < ntiles) {
    // ---- softmax and epilogue of tile x: thread <-> row (TMEM lane) r
    const int x = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const int h = r & ((1 << p.slots_log2) - 1), t = q0 + x * tile_tokens + (r >> p.slots_log2);
    const bool mine = h < p.group && t < count;
    const int qp = start + t;                     // (rows that do not exist: finite nonsense)
    const int first = start + q0 + x * tile_tokens;
    const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t t_s = trow + S::s_col(x), t_o = trow + S::o_col(x);
    const float sc = s_inv[x * 128 + r] * p.scale_log2;
    auto wait_all = [&](uint32_t bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, TI_DEVERR_PREFILL_WAIT));
    };
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int c = 0, st = 0, ph = 0; c < n; ++c) {
      const int k0 = kb + c * kChunk;
      // (kv_full of this chunk has completed when its scores have: no wait, but the loaders' flags;
      // both are asked at once, they are mostly there)
      const uint32_t sbar = s_full + 8 * x, kbar = kv_full + 8 * st;
      const bool there = mbar_try_wait(sbar, c & 1) & mbar_try_wait(kbar, ph);
      if (!__all_sync(0xffffffffu, there)) {
        const bool got = mbar_wait(sbar, c & 1, TI_DEVERR_PREFILL_WAIT) &&
                         mbar_wait(kbar, ph, TI_DEVERR_PREFILL_WAIT);
        if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
      }
      if (++st == kStages) {
        st = 0;
        ph ^= 1;
      }
      // The tiles of long items start some clocks apart: 414 us instead of 424 at four chunks of 1024
      // (1000 clocks: 424; they drift back into step); at 4 x 512 behind 1024 tokens 43.0 instead of
      // 43.7.  Short ones end later by as much: 8 x 256 behind 512 27.7 instead of 27.4.
      if (c == 0 && x > 0 && n >= kStaggerFrom) {
        const long long t0 = clock64();
        while (clock64() - t0 < kStagger * x) {}
      }
      tc_fence_after();
      float sv[kChunk];
      uint32_t sr[kChunk];
      tmem_ld64_start(t_s, sr);
      const int have = s_ok[c & 7];
      tmem_ld64_end(sr, sv);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read + 8 * x);
      if (have != 15 || k0 + kChunk - 1 > first) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
          sv[i] = (k0 + i <= qp && ((have >> (i / kBlock)) & 1)) ? sv[i] : -INFINITY;
      }
      float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < kChunk; i += 2) mxs[i / 2 % 4] = max3(mxs[i / 2 % 4], sv[i], sv[i + 1]);
      const float mx = max3(fmaxf(mxs[0], mxs[1]), mxs[2], mxs[3]) * sc;
      const bool outgrown = __any_sync(0xffffffffu, mx > m + 8.f);
      float alpha = 1.f;
      if (outgrown && mx > m + 8.f) {             // (from no key at all: alpha 0 of zeros)
        alpha = m == -INFINITY ? 0.f : fast_exp2(m - mx);
        m = mx;
      }
      const float off = kPScale - (m == -INFINITY ? 0.f : m);
      const uint64_t sc2 = pair(sc, sc), off2 = pair(off, off);
      // the chunk's sum first, in four chains of pairs: a long row's total stays exact enough
      uint64_t sums[4] = {0, 0, 0, 0};
      uint32_t pk[kChunk / 2];
#pragma unroll
      for (int i = 0; i < kChunk; i += 2) {
        const float2 e = unpair(fma2(pair(sv[i], sv[i + 1]), sc2, off2));
        const float p0 = fast_exp2(e.x), p1 = fast_exp2(e.y);
        sums[i / 2 % 4] = add2(sums[i / 2 % 4], pair(p0, p1));
        pk[i / 2] = Elem<__half>::pack2(p0, p1);
      }
      const float2 t2 = unpair(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])));
      l = l * alpha + (t2.x + t2.y);
      // P V of chunk c-1 has long been done: P's place is free, and O is at rest for a rescale
      if (c >= 1 && !wait_all(pv_done + 8 * x, (c - 1) & 1)) { ok = false; break; }
      if (outgrown && c >= 1) {
        tc_fence_after();
        float ov[32];
#pragma unroll
        for (int d = 0; d < HD; d += 32) {
          tmem_ld32(t_o + d, ov);
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] *= alpha;
          tmem_st32(t_o + d, ov);
        }
      }
      tmem_st32_u(trow + S::p_col(x), pk);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready + 8 * x);
    }
    if (ok && wait_all(pv_done + 8 * x, (n - 1) & 1)) {
      tc_fence_after();
      const float inv = 1.f / l;
      T* dst = (T*)p.out + (int64_t)(row0 + t) * p.out_stride + (int64_t)(kvh * p.group + h) * HD;
      float* po = p.parts + (((int64_t)part * p.KVH + kvh) * S::kTiles + x) * (128 * (HD + 2));
#pragma unroll
      for (int d = 0; d < HD; d += 32) {
        float ov[32];
        tmem_ld32(t_o + d, ov);
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (qp >= s_nan[d / 16 + g]) {
#pragma unroll
            for (int i = 0; i < 16; ++i) ov[g * 16 + i] = __int_as_float(0x7FC00000);
          }
        if (part >= 0) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(po + r * HD + d + i) = make_float4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
        } else if (mine) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 u;
            u.x = Elem<T>::pack2(ov[i] * inv, ov[i + 1] * inv);
            u.y = Elem<T>::pack2(ov[i + 2] * inv, ov[i + 3] * inv);
            u.z = Elem<T>::pack2(ov[i + 4] * inv, ov[i + 5] * inv);
            u.w = Elem<T>::pack2(ov[i + 6] * inv, ov[i + 7] * inv);
            *reinterpret_cast<uint4*>(dst + d + i) = u;
          }
        }
      }
      if (part >= 0) {
        po[128 * HD + r] = m;
        po[128 * HD + 128 + r] = l;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Join the key ranges of one tile of an item and kv head: 16 rows a CTA, in the ranges' order.
constexpr int kMergeRows = 16;

template <typename T, int HD>
__global__ void __launch_bounds__(kMergeRows * HD / 4) merge_kernel(const __grid_constant__ Params p,
                                                                  const int32_t* merges) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int kTiles = Smem<HD>::kTiles;
  const int kvh = blockIdx.x % p.KVH, x = blockIdx.y % kTiles;
  const int32_t* e = merges + (int64_t)(blockIdx.x / p.KVH) * kMergeInts;
  const int seq = e[0], q0 = e[1], slot = e[2], n = e[3];
  if (x >= e[4]) return;
  const int r = (blockIdx.y / kTiles) * kMergeRows + threadIdx.x / (HD / 4), d = threadIdx.x % (HD / 4) * 4;
  const int row0 = p.cu_seqlens[seq], count = p.cu_seqlens[seq + 1] - row0;
  const int h = r & ((1 << p.slots_log2) - 1);
  const int t = q0 + x * (128 >> p.slots_log2) + (r >> p.slots_log2);
  if (h >= p.group || t >= count) return;         // (rows of an item's absent last tiles end here too)
  auto part = [&](int i) { return p.parts + (((int64_t)(slot + i) * p.KVH + kvh) * kTiles + x) * (128 * (HD + 2)); };
  float m = -INFINITY, l = 0.f;
  for (int i = 0; i < n; ++i) m = fmaxf(m, part(i)[128 * HD + r]);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float* b = part(i);
    const float mi = b[128 * HD + r];
    const float c = mi == -INFINITY ? 1.f : fast_exp2(mi - m);   // (no finite score: zeros, or NaN)
    const float4 v = *reinterpret_cast<const float4*>(b + r * HD + d);
    l += c * b[128 * HD + 128 + r];
    o.x += c * v.x;
    o.y += c * v.y;
    o.z += c * v.z;
    o.w += c * v.w;
  }
  const float inv = 1.f / l;
  T* dst = (T*)p.out + (int64_t)(row0 + t) * p.out_stride + (int64_t)(kvh * p.group + h) * HD + d;
  *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<T>::pack2(o.x * inv, o.y * inv),
                                              Elem<T>::pack2(o.z * inv, o.w * inv));
}

template <typename T, int HD>
static int launch(const Params& p, int num_items, const int32_t* merges, int num_merges, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};          // devices whose limit has been raised
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(prefill_kernel<T, HD>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD>::kTotal);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return set_cuda_error(e, "cudaFuncSetAttribute(kv4 prefill)");
    }
    ready.fetch_or(bit, std::memory_order_release);
  }
  if (int rc = launch_kernel("kv4 prefill launch", prefill_kernel<T, HD>,
                             dim3((unsigned)num_items * p.KVH), dim3(Smem<HD>::kThreads), Smem<HD>::kTotal, s, 1, p))
    return rc;
  if (num_merges == 0) return TI_OK;
  return launch_kernel("kv4 prefill merge launch", merge_kernel<T, HD>,
                       dim3((unsigned)num_merges * p.KVH, Smem<HD>::kTiles * 128 / kMergeRows),
                       dim3(kMergeRows * HD / 4), 0, s, 1, p, merges);
}

}  // namespace pre
}  // namespace kv4
}  // namespace ti

using namespace ti;

extern "C" size_t ti_kv4_prefill_workspace_bytes(int num_parts, int num_kv_heads, int head_dim) {
  if (num_parts <= 0 || num_kv_heads <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  return (size_t)num_parts * num_kv_heads * (head_dim == 64 ? 3 : 2) * 128 * (head_dim + 2) * 4;
}

extern "C" int ti_kv4_prefill_attention(void* out, int64_t out_tok_stride, const void* q,
                                        int64_t q_tok_stride, const void* pool, int64_t num_blocks,
                                        const int32_t* block_tables, int64_t bt_stride,
                                        int max_blocks_per_seq, const int32_t* row_index,
                                        const int32_t* start_pos, const int32_t* cu_seqlens,
                                        const int32_t* items, int num_items, const int32_t* merges,
                                        int num_merges, int num_parts, int num_heads,
                                        int num_kv_heads, int head_dim, int block_size, int dtype,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (num_items == 0) return TI_OK;
  if (!out || !q || !pool || !block_tables || !start_pos || !cu_seqlens || !items || num_items < 0 ||
      num_merges < 0 || num_parts < 0 || (num_merges > 0 && !merges) || (num_parts > 0 && !workspace))
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4 prefill: null pointer or negative size");
  if (num_blocks <= 0 || max_blocks_per_seq <= 0 || num_kv_heads <= 0 || num_heads <= 0 ||
      num_heads % num_kv_heads)
    return set_error(TI_ERR_INVALID_ARGUMENT,
                     "kv4 prefill: bad table width, pool size or head counts (num_heads must be a multiple of num_kv_heads)");
  if (num_heads / num_kv_heads > 16)
    return set_error(TI_ERR_UNSUPPORTED, "kv4 prefill: at most 16 query heads per kv head");
  if ((head_dim != 64 && head_dim != 128) || block_size != kv4::kBlock)
    return set_error(TI_ERR_UNSUPPORTED, "kv4 prefill: head_dim must be 64 or 128, block_size 16");
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_FP16)
    return set_error(TI_ERR_UNSUPPORTED, "kv4 prefill: dtype must be bf16 or fp16");
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) |
        reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (out_tok_stride % 8) || (q_tok_stride % 8))
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4 prefill: tensors must be 16-byte aligned");
  if ((int64_t)num_items * num_kv_heads >= (int64_t)1 << 31 ||
      (int64_t)num_merges * num_kv_heads >= (int64_t)1 << 31)
    return set_error(TI_ERR_UNSUPPORTED, "kv4 prefill: too many work items");
  if (workspace_bytes < ti_kv4_prefill_workspace_bytes(num_parts, num_kv_heads, head_dim))
    return set_error(TI_ERR_WORKSPACE, "kv4 prefill: workspace too small");
  const int group = num_heads / num_kv_heads;
  int slots_log2 = 0;
  while ((1 << slots_log2) < group) ++slots_log2;
  kv4::pre::Params p{out, q, (const uint8_t*)pool, out_tok_stride, q_tok_stride, num_blocks,
                     bt_stride, block_tables, row_index, start_pos, cu_seqlens, items,
                     (float*)workspace, num_heads, num_kv_heads, group, slots_log2,
                     max_blocks_per_seq, 1.4426950408889634f / sqrtf((float)head_dim)};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == TI_DTYPE_BF16)
    return head_dim == 64 ? kv4::pre::launch<__nv_bfloat16, 64>(p, num_items, merges, num_merges, s)
                          : kv4::pre::launch<__nv_bfloat16, 128>(p, num_items, merges, num_merges, s);
  return head_dim == 64 ? kv4::pre::launch<__half, 64>(p, num_items, merges, num_merges, s)
                        : kv4::pre::launch<__half, 128>(p, num_items, merges, num_merges, s);
}
