// The 4-bit KV cache's writes and moves: quantise-and-append (with or without RoPE), read back as
// 16-bit values, and eviction by accumulated attention weight.  Format: kv4.cuh.
#include <algorithm>
#include <atomic>

#include "capi_internal.h"
#include "common.cuh"
#include "kv4.cuh"
#include "rmsnorm_row.cuh"

namespace ti {
namespace kv4 {

using ew::load8f;
using ew::rotate8;
using ew::Vec8;

// One quantised group of token `off` of a tile, from 16 elements of a 16-bit type.
template <typename T, int HD>
__device__ __forceinline__ void store_group(uint8_t* tile, bool is_v, int off, int g,
                                            const uint4 lo, const uint4 hi) {
  using L = Tile<HD>;
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  float f[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = Elem<T>::unpack2(w[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
  uint32_t sb;
  const uint2 c = quantize16(f, largest16<T>(w), sb);
  *reinterpret_cast<uint2*>(tile + (is_v ? L::kV : L::kK) + off * L::kRow + g * 8) = c;
  tile[(is_v ? L::kVs : L::kKs) + g * kBlock + off] = (uint8_t)sb;
}

// ---- append -------------------------------------------------------------------------------------
// One thread per (token, group of 16 dims), grid.y over K and V of the heads: 32 bytes in, 9 bytes
// out.  The groups of a token run over neighbouring lanes and then the tokens, so a warp reads whole
// lines and writes whole 32-byte rows of codes and runs of scale bytes.  Bound: HBM, then the
// conversions' instructions: 16384 tokens of 8 kv heads of 128 dims, 86 MB, 20 us from cold caches (4.3
// TB/s, 77 % of the issue slots); 256 tokens of 2 heads of 64, 1.6 us, one chain of latencies.
struct AppendParams {
  uint8_t* pool;
  float* weights;                    // attention-weight totals to clear for the new tokens, or null
  const void *k, *v;
  int64_t k_tok, k_head, v_tok, v_head;
  const int64_t* slots;
  int64_t pool_slots;
  int tokens, KVH;
};

template <typename T, int HD>
__global__ void append_kernel(AppendParams p) {
  pdl_wait();
  pdl_launch_dependents();
  using L = Tile<HD>;
  const int h = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  const T* base = is_v ? (const T*)p.v + h * p.v_head : (const T*)p.k + h * p.k_head;
  const int64_t stride = is_v ? p.v_tok : p.k_tok;
  const int64_t total = (int64_t)p.tokens * L::kGroups;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int t = (int)(i / L::kGroups), g = (int)(i % L::kGroups);
    const int64_t slot = p.slots[t];
    const uint4* src = reinterpret_cast<const uint4*>(base + t * stride + g * kGroup);
    const uint4 lo = src[0], hi = src[1];
    if (slot < 0) continue;
    if (slot >= p.pool_slots) {
      if (blockIdx.y == 0 && g == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
      continue;
    }
    const int64_t tile = (int64_t)((uint64_t)slot / kBlock) * p.KVH + h;
    const int off = (int)slot & (kBlock - 1);
    store_group<T, HD>(p.pool + tile * L::kBytes, is_v, off, g, lo, hi);
    if (p.weights && !is_v && g == 0) p.weights[tile * kBlock + off] = 0.f;
  }
}

// ---- RoPE and append ---------------------------------------------------------------------------------
// The decode and prefill layers' form, on rows [q | k | v] of the fused projection: q and k are rotated
// in place and rounded to the type, as ti_rope_inplace does, then k and v are quantised from those
// values.  One thread per 16 dims and their 16 partners of a q or k head, or per 16 dims of v.
// Measured, 14 query heads over 2 of 64 dims: 256 tokens 2.9 us, 16384 tokens 20.3 us (76 MB at 3.7
// TB/s); 32 over 8 of 128, 16384 tokens: 94 us (407 MB at 4.3 TB/s, 0.66 of measured copy).
struct RopeAppendParams {
  void* qkv;
  int64_t stride;
  uint8_t* pool;
  float* weights;
  const int64_t* slots;
  int64_t pool_slots;
  const float *cos, *sin;
  const int32_t* pos;
  int positions, tokens, NH, KVH;
};

template <typename T, int HD>
__global__ void __launch_bounds__(128) rope_append_kernel(RopeAppendParams p) {
  using L = Tile<HD>;
  constexpr int kHalf = HD / 2, kPieces = kHalf / kGroup;        // pieces of a rotated head
  pdl_wait();
  pdl_launch_dependents();
  const int turns = (p.NH + p.KVH) * kPieces, per_tok = turns + p.KVH * L::kGroups;
  const int64_t total = (int64_t)p.tokens * per_tok;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int t = (int)(i / per_tok), r = (int)(i - (int64_t)t * per_tok);
    T* row = (T*)p.qkv + t * p.stride;
    const int64_t slot = p.slots[t];
    const int pos = p.pos[t];
    const bool write = slot >= 0 && slot < p.pool_slots, turn = (uint32_t)pos < (uint32_t)p.positions;
    if ((slot >= p.pool_slots || !turn) && r == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
    if (!turn) continue;
    const int off = (int)slot & (kBlock - 1);
    uint8_t* tiles = p.pool + (int64_t)((uint64_t)(write ? slot : 0) / kBlock) * p.KVH * L::kBytes;
    if (r < turns) {
      const int h = r / kPieces, piece = r % kPieces, d0 = piece * kGroup;
      T* base = row + (int64_t)h * HD;             // q heads, then k heads
      const int64_t tab = (int64_t)pos * kHalf + d0;
      uint4 x[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        Vec8<T> a, b;
        float c[8], s[8], x1[8], x2[8];
        load8f(p.cos + tab + 8 * u, c);
        load8f(p.sin + tab + 8 * u, s);
        a.load(base + d0 + 8 * u);
        b.load(base + kHalf + d0 + 8 * u);
        a.to_float(x1);
        b.to_float(x2);
        rotate8(x1, x2, c, s);
        a.from_float(x1);
        b.from_float(x2);
        a.store(base + d0 + 8 * u);
        b.store(base + kHalf + d0 + 8 * u);
        x[0][u] = a.raw;
        x[1][u] = b.raw;
      }
      if (h >= p.NH && write) {
        uint8_t* tile = tiles + (int64_t)(h - p.NH) * L::kBytes;
        store_group<T, HD>(tile, false, off, piece, x[0][0], x[0][1]);
        store_group<T, HD>(tile, false, off, piece + kPieces, x[1][0], x[1][1]);
        if (p.weights && piece == 0)
          p.weights[((int64_t)((uint64_t)slot / kBlock) * p.KVH + h - p.NH) * kBlock + off] = 0.f;
      }
    } else if (write) {
      const int h = (r - turns) / L::kGroups, g = (r - turns) % L::kGroups;
      const uint4* src = reinterpret_cast<const uint4*>(row + (int64_t)(p.NH + p.KVH + h) * HD + g * kGroup);
      store_group<T, HD>(tiles + (int64_t)h * L::kBytes, true, off, g, src[0], src[1]);
    }
  }
}

// ---- read back ------------------------------------------------------------------------------------
// One thread per (table entry, head, token, 8 dims), K and V both: 8 bytes of codes and 2 scales in,
// 32 bytes out, the lanes of a warp on neighbouring 16 bytes (with 16 dims per thread the 16-byte
// stores took half a sector each: 122 us instead of 105 for 393 MB); zeros behind the row's length in
// its last block, and nothing for the blocks behind that.
// grid = (runs of a row's blocks, head, row).
struct DequantParams {
  void *k_out, *v_out;
  int64_t out_blocks;
  const uint8_t* pool;
  int64_t num_blocks;
  const int32_t* tables;
  int64_t bt_stride;
  const int32_t* row_index;
  const int32_t* lens;
  const int32_t* out_tables;
  int64_t ot_stride;
  int rows, max_blocks, KVH;
};

// (Append and read-back of 16384 tokens of 8 kv heads of 128 dims, one behind the other, the codes
// then in L2: 36 us for 172 MB, 4.8 TB/s, 0.73 of measured copy.)
constexpr int kDequantThreads = 256;
constexpr int kDequantUnroll = 2;                // tiles per thread

// 8 values in a 16-bit type.
template <typename T>
__device__ __forceinline__ uint4 values8(uint32_t codes, uint32_t scale_byte) {
  uint32_t h[4], w[4];
  codes_to_half2(codes, h);
  if constexpr (std::is_same<T, __half>::value) {
    // (exact in half precision; 16384 tokens of 8 heads of 128 read back in 15.4 us instead of 17.5)
    const __half2 s = __half2half2(__ushort_as_half((unsigned short)(scale_byte << 7)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), s);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  } else {
    const float s = scale_value(scale_byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = Elem<__half>::unpack2(h[i]);
      w[i] = Elem<T>::pack2(v.x * s, v.y * s);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kDequantThreads) dequantize_kernel(DequantParams p) {
  using L = Tile<HD>;
  constexpr int kPer = HD / 8, kPerTile = kBlock * kPer, kTiles = kDequantThreads / kPerTile;
  const int w = threadIdx.x % kPerTile, off = w / kPer, c = w % kPer, h = blockIdx.y;
  const int code = off * L::kRow + c * 4, scale = (c / 2) * kBlock + off;
  const int64_t j0 = (int64_t)blockIdx.x * (kTiles * kDequantUnroll) + threadIdx.x / kPerTile;
  pdl_wait();
  pdl_launch_dependents();
  for (int r = blockIdx.z; r < p.rows; r += gridDim.z) {
    const int64_t len = p.lens[r];
    const int32_t* srcs = p.tables + (p.row_index ? p.row_index[r] : r) * p.bt_stride;
    const int32_t* dsts = p.out_tables + r * p.ot_stride;
    uint32_t kc[kDequantUnroll], vc[kDequantUnroll], ks[kDequantUnroll], vs[kDequantUnroll];
    int32_t dst[kDequantUnroll];
#pragma unroll
    for (int u = 0; u < kDequantUnroll; ++u) {
      const int64_t j = j0 + u * kTiles, left = len - j * kBlock;   // the row's tokens from block j on
      kc[u] = vc[u] = ks[u] = vs[u] = 0u;
      dst[u] = -1;
      if (j >= p.max_blocks || left <= 0) continue;
      dst[u] = dsts[j];
      const int32_t src = srcs[j];
      if (src < 0 || src >= p.num_blocks || off >= left) continue;
      const uint8_t* tile = p.pool + ((int64_t)src * p.KVH + h) * L::kBytes;
      kc[u] = *reinterpret_cast<const uint32_t*>(tile + L::kK + code);
      vc[u] = *reinterpret_cast<const uint32_t*>(tile + L::kV + code);
      ks[u] = tile[L::kKs + scale];
      vs[u] = tile[L::kVs + scale];
    }
#pragma unroll
    for (int u = 0; u < kDequantUnroll; ++u) {
      if (dst[u] < 0) continue;
      if (dst[u] >= p.out_blocks) {
        if (w == 0 && h == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
        continue;
      }
      const int64_t at = (((int64_t)dst[u] * p.KVH + h) * kBlock + off) * HD + c * 8;
      *reinterpret_cast<uint4*>((T*)p.k_out + at) = values8<T>(kc[u], ks[u]);
      *reinterpret_cast<uint4*>((T*)p.v_out + at) = values8<T>(vc[u], vs[u]);
    }
  }
}

// ---- eviction -------------------------------------------------------------------------------------
// One CTA per (layer, sequence, kv head).  With n cached tokens and n > keep it keeps the last
// `recent` and the keep - recent heaviest of the older ones (ties: the earlier token), in order.
//
// evict_kernel: the weights become order-preserving 32-bit keys in shared memory, read once.  The
// lightest kept key is found two bits at a time from the top (how many keys are at least each of the
// three trial values?), leaving out the bits that all keys share and stopping as soon as a count is
// exact, which for distinct weights is after about log2(n) bits below the exponent.  Ranks come from
// one scan of (heavier, equal) counts; the survivors' slots replace the keys in shared memory (a rank
// is never behind its token), then a warp per block of 16 survivors moves their codes, scales and
// weights.  A survivor's place is never behind its old one and a round reads all of its tokens before
// it writes any, so the move may be in place.  Bound: HBM for a large batch (24 layers x 32 sequences of
// U[600, 4096] to 1000: 100 us, 353 MB, 3.5 TB/s; the survivors' codes are gathered 32 bytes at a time),
// the chain of barriers for one sequence (24 layers x 2048 to 1024: 9 us).  The keys' place goes by the
// table's width, so a caller passes the columns in use, as the cache manager does: 24 layers x 2048 to
// 1024 take 16 us (events around a call) through 128 columns and 37 through 8192.
//
// evict_long_kernel: the same for sequences whose keys exceed shared memory, or fill so much of it that
// few CTAs fit (see the launch), the weights read again in each pass.
struct EvictParams {
  uint8_t* pool;
  float* weights;
  int64_t num_blocks;
  const int32_t* tables;
  int64_t bt_stride;
  const int32_t* out_tables;
  int64_t ot_stride;
  const int32_t* row_index;
  const int32_t* ctx;
  int32_t* kept;
  int64_t kept_stride;
  int batch, KVH, max_blocks, out_max_blocks, keep, recent;
};

constexpr int kEvictMaxTokens = 48 * 1024;       // keys of the longest sequence: 192 KB
constexpr int kEvictLongThreads = 256;

// Larger weight, larger key; NaN counts as the largest, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(w + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Is any block that the sequence's n tokens or its m survivors need outside the pool or the tables?
// Thread `tid` of `threads` looks at its share of the entries.
__device__ __forceinline__ bool bad_entries(const EvictParams& p, const int32_t* src, const int32_t* dst,
                                            int n, int m, int tid, int threads) {
  const int nb = (n - 1) / kBlock + 1, mb = (m - 1) / kBlock + 1;
  bool bad = nb > p.max_blocks || mb > p.out_max_blocks;
  if (!bad)
    for (int j = tid; j < nb; j += threads) {
      bad |= (uint32_t)src[j] >= (uint64_t)p.num_blocks;
      if (j < mb) bad |= (uint32_t)dst[j] >= (uint64_t)p.num_blocks;
    }
  return bad;
}

template <int HD, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) evict_kernel(EvictParams p) {
  using L = Tile<HD>;
  constexpr int kEvictWarps = kThreads / 32;
  extern __shared__ __align__(16) uint32_t keys[];             // then the survivors' slots
  __shared__ uint2 s_trial[2][kEvictWarps];
  __shared__ uint32_t s_count[2][kEvictWarps];
  __shared__ uint32_t s_and, s_or;
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) { s_and = 0xFFFFFFFFu; s_or = 0; }
  pdl_wait();
  pdl_launch_dependents();
  const int n = p.ctx[b];
  if (n <= 0) return;
  const int row = p.row_index ? p.row_index[b] : b;
  const int32_t* src_row = p.tables + (int64_t)row * p.bt_stride;
  const int32_t* dst_row = p.out_tables + (int64_t)row * p.ot_stride;
  int32_t* kept = p.kept ? p.kept + ((int64_t)(layer * p.batch + b) * p.KVH + h) * p.kept_stride
                         : nullptr;
  uint8_t* pool = p.pool + (int64_t)layer * p.num_blocks * p.KVH * L::kBytes;
  float* weights = p.weights + (int64_t)layer * p.num_blocks * p.KVH * kBlock;
  const int m = min(n, p.keep);
  const int old = n - p.recent;                   // candidates: positions 0 .. old-1
  const int want = p.keep - p.recent;             // how many of them stay (when n > keep)
  const bool all = n <= p.keep, pick = !all && want > 0;
  uint32_t bound = 0xFFFFFFFFu, ties = 0;         // keys above bound stay, and `ties` of those at it
  __syncthreads();
  // the keys' loads and the check of the table entries overlap: a bad entry's weights are not read
  uint32_t both = 0xFFFFFFFFu, any = 0;
  if (pick && n <= p.max_blocks * (int64_t)kBlock) {
    for (int i = tid * 4; i < old; i += kThreads * 4) {         // four tokens of one block
      const uint32_t id = (uint32_t)src_row[i / kBlock];
      float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
      if (id < (uint64_t)p.num_blocks)
        w = *reinterpret_cast<const float4*>(weights + ((int64_t)id * p.KVH + h) * kBlock + i % kBlock);
      const float f[4] = {w.x, w.y, w.z, w.w};
      uint32_t k[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        k[u] = weight_key(f[u]);
        if (i + u < old) {
          both &= k[u];
          any |= k[u];
        } else {
          k[u] = 0;                               // below every trial value
        }
      }
      *reinterpret_cast<uint4*>(keys + i) = make_uint4(k[0], k[1], k[2], k[3]);
    }
    both = __reduce_and_sync(0xffffffffu, both);
    any = __reduce_or_sync(0xffffffffu, any);
    if (lane == 0) {
      atomicAnd(&s_and, both);
      atomicOr(&s_or, any);
    }
  }
  if (__syncthreads_or(bad_entries(p, src_row, dst_row, n, m, tid, kThreads))) {
    if (tid == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
    return;
  }
  if (pick) {
    const uint32_t differ = s_and ^ s_or;
    const int top = differ ? (31 - __clz(differ)) | 1 : -1;      // odd: pairs of bits from here down
    uint32_t low = s_and;                         // at least `want` keys are >= low
    if (top >= 0) low &= ~((2u << top) - 1u);
    bool exact = false;
    int pass = 0;
    for (int sh = top - 1; sh >= 0 && !exact; sh -= 2, pass ^= 1) {
      const uint32_t t1 = low | (1u << sh), t2 = low | (2u << sh), t3 = low | (3u << sh);
      uint32_t c12 = 0, c3 = 0;                   // counts of two trials in 16 bits each
      for (int i = tid * 4; i < old; i += kThreads * 4) {
        const uint4 k = *reinterpret_cast<const uint4*>(keys + i);
        const uint32_t v[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          c12 += (v[u] >= t1) + ((uint32_t)(v[u] >= t2) << 16);
          c3 += v[u] >= t3;
        }
      }
      c12 = __reduce_add_sync(0xffffffffu, c12);
      c3 = __reduce_add_sync(0xffffffffu, c3);
      if (lane == 0) s_trial[pass][warp] = make_uint2(c12, c3);
      __syncthreads();
      const uint2 part = lane < kEvictWarps ? s_trial[pass][lane] : make_uint2(0u, 0u);
      c12 = __reduce_add_sync(0xffffffffu, part.x);
      c3 = __reduce_add_sync(0xffffffffu, part.y);
      const uint32_t goal = (uint32_t)want, c1 = c12 & 0xFFFFu, c2 = c12 >> 16;
      const uint32_t c = c3 >= goal ? c3 : c2 >= goal ? c2 : c1;
      if (c3 >= goal) low = t3;
      else if (c2 >= goal) low = t2;
      else if (c1 >= goal) low = t1;
      exact = c == goal;
    }
    if (exact) {
      bound = low - 1u;                           // keys >= low are exactly the wanted ones
    } else {
      // low is the key of the lightest kept token; the earliest ones of that key fill up
      uint32_t c = 0;
      for (int i = tid * 4; i < old; i += kThreads * 4) {
        const uint4 k = *reinterpret_cast<const uint4*>(keys + i);
        c += (k.x > low) + (k.y > low) + (k.z > low) + (k.w > low);
      }
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0) s_count[0][warp] = c;
      __syncthreads();
      c = __reduce_add_sync(0xffffffffu, lane < kEvictWarps ? s_count[0][lane] : 0u);
      bound = low;
      ties = (uint32_t)want - c;
      __syncthreads();                            // s_count is used again below
    }
  }
  // ranks: tokens above the bound and tokens at it before each token (16 bits each in a round)
  uint32_t above = 0, at = 0;
  for (int i0 = 0, pass = 0; i0 < n; i0 += kThreads * 4, pass ^= 1) {
    const int i = i0 + tid * 4;
    uint32_t gt = 0, eq = 0;                      // bits of this thread's four tokens
    if (i < n) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (i + u >= n) break;
        if (all || i + u >= old) {
          gt |= 1u << u;
        } else if (want > 0) {
          const uint32_t k = keys[i + u];
          if (k > bound) gt |= 1u << u;
          else if (k == bound) eq |= 1u << u;
        }
      }
    }
    const uint32_t mine = (uint32_t)__popc(gt) | ((uint32_t)__popc(eq) << 16);
    uint32_t x = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) s_count[pass][warp] = x;
    __syncthreads();                              // (also: the round's keys have been read)
    const uint32_t other = lane < kEvictWarps ? s_count[pass][lane] : 0u;
    const uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? other : 0u) + x - mine;
    uint32_t r_gt = above + (before & 0xFFFFu), r_eq = at + (before >> 16);
    const uint32_t round = __reduce_add_sync(0xffffffffu, other);
    above += round & 0xFFFFu;
    at += round >> 16;
    if (gt | eq) {
      const uint32_t slot = (uint32_t)src_row[i / kBlock] * kBlock + i % kBlock;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool is_eq = (eq >> u) & 1u, stay = ((gt >> u) & 1u) || (is_eq && r_eq < ties);
        if (stay) {
          const uint32_t rank = r_gt + min(r_eq, ties);
          keys[rank] = slot + u;
          if (kept) kept[rank] = i + u;
        }
        r_gt += (gt >> u) & 1u;
        r_eq += is_eq;
      }
    }
  }
  __syncthreads();
  // move: HD/16 lanes a token, each 16 bytes of its K or V codes and two of their scales, so a warp
  // reads and writes whole rows; kAtOnce groups of tokens of a warp in flight
  constexpr int kLanes = HD / 16, kTok = 32 / kLanes, kAtOnce = 4;
  const int part = (lane % kLanes) / (kLanes / 2), chunk = lane % (kLanes / 2);
  const int code = (part ? L::kV : L::kK) + chunk * 16;
  const int scale = (part ? L::kVs : L::kKs) + 2 * chunk * kBlock;
  const bool has_weight = lane % kLanes == 0;
  for (int j0 = 0; j0 < m; j0 += kEvictWarps * kAtOnce * kTok) {
    uint4 c[kAtOnce];
    uint32_t sc[kAtOnce];
    float w[kAtOnce];
#pragma unroll
    for (int a = 0; a < kAtOnce; ++a) {
      const int to = j0 + (a * kEvictWarps + warp) * kTok + lane / kLanes;
      if (to >= m) continue;
      const uint32_t slot = keys[to];
      const int64_t tile = (int64_t)(slot / kBlock) * p.KVH + h;
      const int off = (int)(slot % kBlock);
      const uint8_t* src = pool + tile * L::kBytes;
      c[a] = *reinterpret_cast<const uint4*>(src + code + off * L::kRow);
      sc[a] = src[scale + off] | ((uint32_t)src[scale + kBlock + off] << 8);
      if (has_weight) w[a] = weights[tile * kBlock + off];
    }
    __syncthreads();                              // the round's tokens have been read
#pragma unroll
    for (int a = 0; a < kAtOnce; ++a) {
      const int to = j0 + (a * kEvictWarps + warp) * kTok + lane / kLanes;
      if (to >= m) continue;
      const int64_t tile = (int64_t)dst_row[to / kBlock] * p.KVH + h;
      const int off = to % kBlock;
      uint8_t* dst = pool + tile * L::kBytes;
      *reinterpret_cast<uint4*>(dst + code + off * L::kRow) = c[a];
      dst[scale + off] = (uint8_t)sc[a];
      dst[scale + kBlock + off] = (uint8_t)(sc[a] >> 8);
      if (has_weight) weights[tile * kBlock + off] = w[a];
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(kEvictLongThreads) evict_long_kernel(EvictParams p) {
  pdl_wait();
  pdl_launch_dependents();
  using L = Tile<HD>;
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ uint32_t hist[256];
  __shared__ uint32_t s_prefix, s_left;
  __shared__ int s_warp[kEvictLongThreads / 32];
  const int row = p.row_index ? p.row_index[b] : b;
  const int n = p.ctx[b];
  if (n <= 0) return;
  int32_t* kept = p.kept ? p.kept + ((int64_t)(layer * p.batch + b) * p.KVH + h) * p.kept_stride
                         : nullptr;
  const int32_t* src_row = p.tables + (int64_t)row * p.bt_stride;
  const int32_t* dst_row = p.out_tables + (int64_t)row * p.ot_stride;
  if (__syncthreads_or(bad_entries(p, src_row, dst_row, n, min(n, p.keep), tid, kEvictLongThreads))) {
    if (tid == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
    return;
  }
  uint8_t* pool = p.pool + (int64_t)layer * p.num_blocks * p.KVH * L::kBytes;
  float* weights = p.weights + (int64_t)layer * p.num_blocks * p.KVH * kBlock;
  auto tile_of = [&](const int32_t* r, int i) { return (int64_t)r[i / kBlock] * p.KVH + h; };
  const int old = n - p.recent;                 // candidates: positions 0 .. old-1
  const int want = p.keep - p.recent;           // how many of them stay (when n > keep)
  uint32_t bound = 0, ties = 0;
  if (n > p.keep && want > 0) {
    if (tid == 0) { s_prefix = 0; s_left = want; }
    for (int shift = 24; shift >= 0; shift -= 8) {
      hist[tid] = 0;
      __syncthreads();
      const uint32_t prefix = s_prefix;
      for (int i = tid; i < old; i += kEvictLongThreads) {
        const uint32_t key = weight_key(weights[tile_of(src_row, i) * kBlock + i % kBlock]);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t left = s_left;
        int d = 255;
        for (; d > 0 && hist[d] < left; --d) left -= hist[d];
        s_left = left;
        s_prefix = prefix | ((uint32_t)d << shift);
      }
      __syncthreads();
    }
    bound = s_prefix;                           // key of the lightest kept token
    ties = s_left;                              // how many of the tokens with that key stay
  }
  int placed = 0;
  uint32_t tied = 0;
  for (int i0 = 0; i0 < n; i0 += kEvictLongThreads) {
    const int i = i0 + tid;
    uint32_t key = 0;
    bool in = i < n, gt = false, eq = false;
    int64_t st = 0;
    float w = 0.f;
    if (in) {
      st = tile_of(src_row, i);
      w = weights[st * kBlock + i % kBlock];
      if (n <= p.keep || i >= old) {
        gt = true;
      } else if (want > 0) {
        key = weight_key(w);
        gt = key > bound;
        eq = key == bound;
      }
    }
    // ranks in order: first among the tied tokens, then among the kept ones
    auto scan = [&](bool f, int& total) {
      const uint32_t bal = __ballot_sync(0xffffffffu, f);
      if (lane == 0) s_warp[warp] = __popc(bal);
      __syncthreads();
      int before = 0;
      total = 0;
      for (int k = 0; k < kEvictLongThreads / 32; ++k) {
        if (k < warp) before += s_warp[k];
        total += s_warp[k];
      }
      __syncthreads();
      return before + __popc(bal & ((1u << lane) - 1u));
    };
    int n_eq, n_keep;
    const int r_eq = scan(eq, n_eq);
    const bool stay = gt || (eq && tied + r_eq < ties);
    tied += n_eq;
    const int to = placed + scan(stay, n_keep);
    placed += n_keep;
    uint4 c[HD / 16];
    uint8_t sc[HD / 8];
    if (stay) {
      const uint8_t* tile = pool + st * L::kBytes;
      const int off = i % kBlock;
#pragma unroll
      for (int u = 0; u < HD / 32; ++u) {
        c[u] = *reinterpret_cast<const uint4*>(tile + L::kK + off * L::kRow + u * 16);
        c[HD / 32 + u] = *reinterpret_cast<const uint4*>(tile + L::kV + off * L::kRow + u * 16);
      }
#pragma unroll
      for (int u = 0; u < HD / 8; ++u) sc[u] = tile[L::kKs + u * kBlock + off];
    }
    __syncthreads();
    if (stay) {
      const int64_t dt = tile_of(dst_row, to);
      uint8_t* tile = pool + dt * L::kBytes;
      const int off = to % kBlock;
#pragma unroll
      for (int u = 0; u < HD / 32; ++u) {
        *reinterpret_cast<uint4*>(tile + L::kK + off * L::kRow + u * 16) = c[u];
        *reinterpret_cast<uint4*>(tile + L::kV + off * L::kRow + u * 16) = c[HD / 32 + u];
      }
#pragma unroll
      for (int u = 0; u < HD / 8; ++u) tile[L::kKs + u * kBlock + off] = sc[u];
      weights[dt * kBlock + off] = w;
      if (kept) kept[to] = i;
    }
    __syncthreads();
  }
}

static int sm_count() {
  static int sms = 0;
  if (!sms) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (sms <= 0) sms = 148;
  }
  return sms;
}
static int grid_for(int64_t work, int threads) {
  return (int)std::max<int64_t>(1, std::min<int64_t>((work + threads - 1) / threads,
                                                     (int64_t)sm_count() * 16));
}

}  // namespace kv4
}  // namespace ti

using namespace ti;

extern "C" size_t ti_kv4_tile_bytes(int head_dim) {
  return (head_dim == 64 || head_dim == 128) ? (size_t)18 * head_dim : 0;
}

extern "C" int ti_kv4_append(void* pool, float* weights, const void* k, int64_t k_tok_stride,
                             int64_t k_head_stride, const void* v, int64_t v_tok_stride,
                             int64_t v_head_stride, const int64_t* slot_mapping, int num_tokens,
                             int64_t num_blocks, int num_kv_heads, int head_dim, int block_size,
                             int dtype, void* stream) {
  clear_error();
  if (num_tokens == 0) return TI_OK;
  if (!pool || !k || !v || !slot_mapping || num_tokens < 0 || num_blocks <= 0 || num_kv_heads <= 0)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4_append: null pointer, negative size or empty pool");
  if ((head_dim != 64 && head_dim != 128) || block_size != kv4::kBlock)
    return set_error(TI_ERR_UNSUPPORTED, "kv4_append: head_dim must be 64 or 128, block_size 16");
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_FP16)
    return set_error(TI_ERR_UNSUPPORTED, "kv4_append: dtype must be bf16 or fp16");
  if (((k_tok_stride | k_head_stride | v_tok_stride | v_head_stride) % 8) ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
        reinterpret_cast<uintptr_t>(pool)) & 15))
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4_append: rows must be 16-byte aligned");
  kv4::AppendParams p{(uint8_t*)pool, weights, k, v, k_tok_stride, k_head_stride, v_tok_stride,
                      v_head_stride, slot_mapping, num_blocks * kv4::kBlock, num_tokens,
                      num_kv_heads};
  if (num_kv_heads > 32767)
    return set_error(TI_ERR_UNSUPPORTED, "kv4_append: at most 32767 kv heads");
  // (64 threads for few tokens: 1.59 us against 1.67 at 1024 tokens of 2 kv heads of 64 dims, 1.64 against
  // 1.54 at 64; of 8 heads of 128 2.57 against 2.37 at 1024, 1.74 against 1.65 at 256)
  constexpr int threads = 256;
  const dim3 grid(kv4::grid_for((int64_t)num_tokens * (head_dim / 16), threads), 2 * num_kv_heads);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) { return launch_kernel("kv4_append launch", kern, grid, dim3(threads), 0, s, 1, p); };
  if (dtype == TI_DTYPE_BF16)
    return head_dim == 64 ? go(kv4::append_kernel<__nv_bfloat16, 64>)
                          : go(kv4::append_kernel<__nv_bfloat16, 128>);
  return head_dim == 64 ? go(kv4::append_kernel<__half, 64>) : go(kv4::append_kernel<__half, 128>);
}

extern "C" int ti_rope_kv4_append(void* qkv, int64_t qkv_stride, void* pool, float* weights,
                                  const int64_t* slot_mapping, const float* cos, const float* sin,
                                  int num_positions, const int32_t* pos, int num_tokens,
                                  int64_t num_blocks, int num_heads, int num_kv_heads,
                                  int head_dim, int block_size, int dtype, void* stream) {
  clear_error();
  if (num_tokens == 0) return TI_OK;
  if (!qkv || !pool || !slot_mapping || !cos || !sin || !pos || num_tokens < 0 ||
      num_positions < 0 || num_blocks <= 0 || num_heads <= 0 || num_kv_heads <= 0)
    return set_error(TI_ERR_INVALID_ARGUMENT, "rope_kv4_append: null pointer, negative size or empty pool");
  if ((head_dim != 64 && head_dim != 128) || block_size != kv4::kBlock)
    return set_error(TI_ERR_UNSUPPORTED, "rope_kv4_append: head_dim must be 64 or 128, block_size 16");
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_FP16)
    return set_error(TI_ERR_UNSUPPORTED, "rope_kv4_append: dtype must be bf16 or fp16");
  if ((qkv_stride % 8) ||
      ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(pool) |
        reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15))
    return set_error(TI_ERR_INVALID_ARGUMENT, "rope_kv4_append: tensors must be 16-byte aligned");
  kv4::RopeAppendParams p{qkv, qkv_stride, (uint8_t*)pool, weights, slot_mapping,
                          num_blocks * kv4::kBlock, cos, sin, pos, num_positions, num_tokens, num_heads,
                          num_kv_heads};
  const int64_t work = (int64_t)num_tokens * ((num_heads + num_kv_heads) * (head_dim / 32) +
                                              num_kv_heads * (head_dim / 16));
  const dim3 grid(kv4::grid_for(work, 128));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) { return launch_kernel("rope_kv4_append launch", kern, grid, dim3(128), 0, s, 1, p); };
  if (dtype == TI_DTYPE_BF16)
    return head_dim == 64 ? go(kv4::rope_append_kernel<__nv_bfloat16, 64>)
                          : go(kv4::rope_append_kernel<__nv_bfloat16, 128>);
  return head_dim == 64 ? go(kv4::rope_append_kernel<__half, 64>)
                        : go(kv4::rope_append_kernel<__half, 128>);
}

extern "C" int ti_kv4_dequantize(void* k_out, void* v_out, int64_t out_blocks, const void* pool,
                                 int64_t num_blocks, const int32_t* block_tables,
                                 int64_t bt_stride, const int32_t* row_index, const int32_t* lens,
                                 const int32_t* out_tables, int64_t ot_stride, int rows,
                                 int max_blocks, int num_kv_heads, int head_dim, int block_size,
                                 int dtype, void* stream) {
  clear_error();
  if (rows == 0 || max_blocks == 0) return TI_OK;
  if (!k_out || !v_out || !pool || !block_tables || !lens || !out_tables || rows < 0 ||
      max_blocks < 0 || num_blocks <= 0 || out_blocks <= 0 || num_kv_heads <= 0)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4_dequantize: null pointer, negative size or empty pool");
  if ((head_dim != 64 && head_dim != 128) || block_size != kv4::kBlock)
    return set_error(TI_ERR_UNSUPPORTED, "kv4_dequantize: head_dim must be 64 or 128, block_size 16");
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_FP16)
    return set_error(TI_ERR_UNSUPPORTED, "kv4_dequantize: dtype must be bf16 or fp16");
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out) |
       reinterpret_cast<uintptr_t>(pool)) & 15)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4_dequantize: tensors must be 16-byte aligned");
  kv4::DequantParams p{k_out, v_out, out_blocks, (const uint8_t*)pool, num_blocks, block_tables,
                       bt_stride, row_index, lens, out_tables, ot_stride, rows, max_blocks,
                       num_kv_heads};
  if (num_kv_heads > 65535)
    return set_error(TI_ERR_UNSUPPORTED, "kv4_dequantize: at most 65535 kv heads");
  const int per_cta = kv4::kDequantThreads / (2 * head_dim) * kv4::kDequantUnroll;   // tiles
  const dim3 grid((unsigned)(((int64_t)max_blocks + per_cta - 1) / per_cta), num_kv_heads,
                  std::min(rows, 65535));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) { return launch_kernel("kv4_dequantize launch", kern, grid, dim3(kv4::kDequantThreads), 0, s, 1, p); };
  if (dtype == TI_DTYPE_BF16)
    return head_dim == 64 ? go(kv4::dequantize_kernel<__nv_bfloat16, 64>)
                          : go(kv4::dequantize_kernel<__nv_bfloat16, 128>);
  return head_dim == 64 ? go(kv4::dequantize_kernel<__half, 64>)
                        : go(kv4::dequantize_kernel<__half, 128>);
}

extern "C" int ti_kv4_evict(void* pool, float* weights, int num_layers, int64_t num_blocks,
                            const int32_t* block_tables, int64_t bt_stride,
                            const int32_t* out_tables, int64_t ot_stride,
                            const int32_t* row_index, const int32_t* context_lens, int batch,
                            int max_blocks_per_seq, int out_max_blocks, int keep, int recent,
                            int32_t* kept, int64_t kept_stride, int num_kv_heads, int head_dim,
                            int block_size, void* stream) {
  clear_error();
  if (batch == 0 || num_layers == 0) return TI_OK;
  if (!pool || !weights || !block_tables || !out_tables || !context_lens || batch < 0 ||
      num_layers < 0 || num_blocks <= 0 || num_kv_heads <= 0 || max_blocks_per_seq <= 0 ||
      out_max_blocks <= 0)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4_evict: null pointer, negative size or empty pool");
  if ((head_dim != 64 && head_dim != 128) || block_size != kv4::kBlock)
    return set_error(TI_ERR_UNSUPPORTED, "kv4_evict: head_dim must be 64 or 128, block_size 16");
  if (keep < 1 || recent < 0 || recent > keep)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4_evict: needs 1 <= keep and 0 <= recent <= keep");
  if (kept && kept_stride < keep)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4_evict: kept rows are shorter than keep");
  if ((reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(weights)) & 15)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4_evict: pool and weights must be 16-byte aligned");
  if (batch > 65535 || num_layers > 65535)
    return set_error(TI_ERR_UNSUPPORTED, "kv4_evict: at most 65535 sequences and layers");
  kv4::EvictParams p{(uint8_t*)pool, weights, num_blocks, block_tables, bt_stride, out_tables,
                     ot_stride, row_index, context_lens, kept, kept_stride, batch, num_kv_heads,
                     max_blocks_per_seq, out_max_blocks, keep, recent};
  const dim3 grid(num_kv_heads, batch, num_layers);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // the widest table bounds the sequences' lengths; slots are 32 bits in shared memory
  const int64_t tokens = (int64_t)max_blocks_per_seq * kv4::kBlock;
  // With fewer than three CTAs to an SM (tables above some 18000 tokens) a second wave of them costs more
  // than reading the weights again: 24 layers, half of the tokens kept, us here / in the long kernel:
  // 96 units (2 heads, 2 sequences) of 32768 tokens 197 / 321; 192 units of 24576 186 / 285, of 32768
  // 385 / 373; 384 units of 16384 204 / 236, of 24576 482 / 346, of 32768 863 / 453; 768 units of 16384
  // 390 / 458, of 24576 743 / 679.
  const int64_t units = (int64_t)num_kv_heads * batch * num_layers;
  const int64_t per_sm = 227 * 1024 / (tokens * 4 + 2048);
  const bool waves = per_sm < 3 && units > per_sm * kv4::sm_count();
  if (tokens > kv4::kEvictMaxTokens || num_blocks > (int64_t)1 << 28 || waves)
    return launch_kernel("kv4_evict launch", head_dim == 64 ? kv4::evict_long_kernel<64> : kv4::evict_long_kernel<128>,
                         grid, dim3(kv4::kEvictLongThreads), 0, s, 1, p);
  // Many (layer, sequence, head) units: small CTAs, several per SM (while the table is narrow: see
  // above); few: wide ones, the chain of one unit counts.  24 layers x 2 heads, one sequence of 2048:
  // 17 us with 512 threads, 23 with 256; 32 sequences of up to 4096: 111 and 99 (cold caches).
  auto go = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    static std::atomic<uint64_t> ready[2];
    const bool small = units > 2 * kv4::sm_count();
    auto kern = small ? kv4::evict_kernel<HD, 256> : kv4::evict_kernel<HD, 512>;
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(ready[small].load(std::memory_order_acquire) & bit)) {
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           kv4::kEvictMaxTokens * 4);
      if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return set_cuda_error(e, "cudaFuncSetAttribute(kv4_evict)");
      }
      ready[small].fetch_or(bit, std::memory_order_release);
    }
    return launch_kernel("kv4_evict launch", kern, grid, dim3(small ? 256 : 512), (size_t)tokens * 4,
                         s, 1, p);
  };
  return head_dim == 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}
