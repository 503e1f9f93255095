// Decode attention over the 4-bit paged KV cache, and the attention-weight totals that eviction
// ranks tokens by.  Format: kv4.cuh.
#include <algorithm>
#include <atomic>

#include "capi_internal.h"
#include "common.cuh"
#include "kv4.cuh"

namespace ti {
namespace kv4 {

// ---- decode attention ------------------------------------------------------------------------------
// out = softmax(q K^T / sqrt(D)) V for one query token of each sequence, from the codes: per
// (block, kv head) tile 18 * D bytes are read once for all query heads of the kv head, so the floor is
// those bytes at HBM speed, 23 bytes per clock and SM.
//
// Work split.  A unit is (sequence, kv head, group of at most 8 query heads); all units' tiles form
// one stream (units in order, a unit's tiles in order) that is cut evenly over the CTAs and, inside a
// CTA, over its 16 warps, so ragged lengths balance.  A warp keeps the running max and sum of its
// current unit in registers; units cut by a warp boundary are joined in shared memory by the CTA,
// those cut by a CTA boundary through the workspace by the CTA that arrives last (pieces in order:
// the same bits on every run).  One launch.
//
// A warp's step is 64 tokens (D = 64; 32 for D = 128): its 4608 bytes come through a private ring of
// two stages by 16-byte asynchronous copies, 9 per lane, issued a step ahead.
//
// Mathematics of a step, tokens as the matrix instruction's M dimension, heads as N:
//   S^T = K q^T   A = K: lane (g, t) holds tokens g and g+8 and one or two whole scale groups of
//                 each (dims D/4 * t ...), so it needs one scale per 16 dims; the order of the dims
//                 in the sum is free, q is laid out to match.
//   O^T += V^T P^T  A = V^T: lane (g, t) holds dims D/8 * g ... of tokens 2t, 2t+1, 2t+8, 2t+9; the
//                 codes of two tokens are interleaved as half-bytes, so one conversion gives the
//                 pair; P^T comes from S^T by an 8x8 transpose between lanes.
// Codes become half precision by the hardware conversion and are multiplied by their scale: exact, so
// both types run on half-precision operands.  bf16 queries are scaled by a power of two that brings
// the row's largest magnitude to 2^14 (elements below 2^-28 of it lose bits: 2^-39 of the largest);
// the scores' factor takes it back.  Weights are held as 2^14 p in half precision: 2^-11 relative
// (the 16-bit outputs round by as much) down to p = 2^-28; their sum is taken before that rounding.
//
// Measured, 14 query heads over 2 of 64 dims: 256 x U[8192, 32768] tokens 152 us over 24 pools in turn, as
// a model's layers are (0.76 GB at 5.1 TB/s, 0.77 of measured copy), 135 us with one pool read again and
// again (5.6 TB/s, 0.85; 70 % of the issue slots); 256 x U[128, 2048] 18.6 us, where a warp has four
// steps and the length scan, three dependent loads before the first step and the joins are as long as
// the stream; 8 x U[1, 512] 7.7 us, latency.  32 heads over 8 of 128, 32 x U[1024, 8192]: 45 us, 3.8 TB/s
// (a scale serves twice the dims a lane, but a step is 32 tokens: its fixed work weighs double).
struct DecodeParams {
  void* out;
  float* lse;                        // [batch, NH] or null
  const void* q;
  const uint8_t* pool;
  int64_t out_stride, q_stride, num_blocks, bt_stride;
  const int32_t *tables, *row_index, *ctx;
  int batch, NH, KVH, group, max_blocks;
  int subs;                          // groups of at most 8 query heads per kv head
  float scale_log2;
  uint32_t* counters;                // [gridDim.x], zero between calls
  float* parts;                      // [gridDim.x][2] pieces
};

constexpr int kMaxBatch = 4096;
constexpr int kWarps = 16;
constexpr int kStages = 2;                       // (the code below counts on two)
constexpr int kStepBytes = 4608;                 // 64 (D = 64) or 32 tokens of one kv head
constexpr float kPScale = 14.f;                  // weights are held as 2^14 p

// What the warps of a CTA tell one another.
struct Shared {
  uint32_t scan[kWarps];
  int start[kWarps + 1];             // first grain of every warp, counted from the CTA's
  // cut units by where their first piece in this CTA is: tail of warp i, or (16) head of warp 0;
  // x = first grain counted from the CTA's, y = grains (0: none), z = sequence, w = unit of it
  int4 cut[kWarps + 1];
  int2 last[2];                      // first and last CTA of a unit that this CTA joins
};

template <int HD>
struct Shape {
  static constexpr int kTiles = kStepBytes / Tile<HD>::kBytes;   // tiles of a step
  static constexpr int kLanes = 32 / kTiles;                     // lanes that copy one tile
  static constexpr uint32_t kFirsts = kTiles == 4 ? 0x01010101u : 0x00010001u;
  static constexpr int kPiece = 8 * HD + 16;                     // floats: O, m[8], l[8]
  static constexpr int kRing = kWarps * kStages * kStepBytes;
  static constexpr int kPark = kWarps * kPiece * 4;
  // All of it dynamic, so that the rings begin on a 128-byte line: copies of 8 lanes' 16-byte chunks
  // that straddle lines cost 165 -> 228 us at 256 x U[8192, 32768].
  static size_t smem(int batch) { return kRing + kPark + sizeof(Shared) + ((size_t)batch + 1) * 4; }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void lds64(uint32_t a, uint32_t& x, uint32_t& y) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(a));
}
__device__ __forceinline__ void lds128(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(a));
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Where a warp stands in the stream.  The stream is cut at grains: whole steps (the last one of a unit
// may be short), or tiles where a CTA has one unit.  A warp is at grain `at` of unit hv of sequence b,
// whose units have n grains, the last one of `tail` tiles; `left` more grains are its own.
struct Cursor {
  int b, hv, at, n, tail, left;
  __device__ __forceinline__ int piece() const { return min(n - at, left); }
  __device__ __forceinline__ int piece_tiles(int grain) const {
    const int k = piece();
    return at + k == n ? (k - 1) * grain + tail : k * grain;
  }
  // Grains of a unit of sequence b; pref[b] = those of the sequences before b, times 8, plus tail - 1.
  __device__ __forceinline__ void look_up(const uint32_t* pref) {
    n = (int)((pref[b + 1] >> 3) - (pref[b] >> 3));
    tail = (int)(pref[b] & 7u) + 1;
  }
  __device__ __forceinline__ void next_unit(int units, const uint32_t* pref, int batch) {
    left -= piece();
    if (left == 0) return;
    at = 0;
    if (++hv < units) return;
    hv = 0;
    do {
      ++b;
      look_up(pref);
    } while (n == 0 && b < batch - 1);
  }
};

// An even cut of `total` grains over `n` warps: the first `rem` warps take one more.
struct Cut {
  uint32_t quot, rem;
  __device__ __forceinline__ Cut(uint32_t total, uint32_t n) : quot(total / n), rem(total - quot * n) {}
  __device__ __forceinline__ uint32_t start(uint32_t w) const { return w * quot + min(w, rem); }
  __device__ __forceinline__ uint32_t owner(uint32_t pos) const {
    const uint32_t big = rem * (quot + 1);
    return pos < big ? pos / (quot + 1) : rem + (pos - big) / quot;
  }
};

// The batch's stream in grains of KT tiles, cut evenly over the warps of (at most) gridDim.x CTAs: at
// least one grain per warp, so little work takes fewer CTAs.  All threads call it; pref [batch + 1]
// and scan [kWarps] are shared memory.  With total == 0 or a CTA index >= ctas there is no work here.
struct Place {
  uint32_t total;
  int ctas;
};
template <int KT>
__device__ __forceinline__ Place scan_batch(const int32_t* ctx, int batch, int cap, int units,
                                            uint32_t* pref, uint32_t* scan) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t carry = 0;
  for (int b0 = 0; b0 < batch; b0 += kWarps * 32) {
    const int b = b0 + tid;
    const int len = b < batch ? min(ctx[b], cap) : 0;
    const int tiles = len > 0 ? (len - 1) / kBlock + 1 : 0;
    const uint32_t n = (tiles + KT - 1) / KT;
    uint32_t x = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    uint32_t before = carry, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      all += scan[w];
    }
    if (b < batch) pref[b] = (before + x - n) * 8u + (uint32_t)(tiles + KT - 1) % KT;
    carry += all;
    if (tid == 0) pref[batch] = carry * 8u;
    __syncthreads();
  }
  const uint32_t total = carry * (uint32_t)units;
  return {total, min((int)gridDim.x, (int)((total + kWarps - 1) / kWarps))};
}
// Where grain `pos` of the stream is; all lanes of a warp call it.
__device__ __forceinline__ void find_place(uint32_t pos, int batch, int units, const uint32_t* pref,
                                           int lane, Cursor& cur) {
  // last b with (grains before b) * units <= pos: 32 probes at a time
  int lo = 0, len = batch;                         // the answer is in [lo, lo + len)
  while (len > 1) {
    const int step = (len + 31) / 32, probe = lo + lane * step;
    const uint32_t ok = __ballot_sync(0xffffffffu, lane * step < len &&
                                      (pref[min(probe, batch)] >> 3) * (uint32_t)units <= pos);
    const int k = 31 - __clz(ok);
    lo += k * step;
    len = min(step, len - k * step);
  }
  cur.b = lo;
  cur.look_up(pref);
  const uint32_t r = pos - (pref[lo] >> 3) * (uint32_t)units, n = max(cur.n, 1);
  cur.hv = (int)(r / n);
  cur.at = (int)(r - cur.hv * n);
}

// Query rows of a unit: lane (g, t) holds dims D/4 * t ... of head g (zeros beyond the unit's heads).
template <typename T, int HD>
__device__ __forceinline__ void load_query(const T* q, int heads, int g, int t, uint4 (&raw)[HD / 32]) {
  constexpr int N = HD / 4;                      // dims of a lane
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    raw[i] = make_uint4(0u, 0u, 0u, 0u);
    if (g < heads) raw[i] = *reinterpret_cast<const uint4*>(q + (int64_t)g * HD + t * N + i * 8);
  }
}
// ... as the B operand: f[s][0..1] hold dims D/4 * t + 4 s + {0,1,2,3} of head g.  Returns the factor
// that the rows of heads 2t and 2t+1 were multiplied by, inverted.
template <typename T, int HD>
__device__ __forceinline__ float2 convert_query(const uint4 (&raw4)[HD / 32], int t, uint32_t (&f)[HD / 16][2]) {
  constexpr int N = HD / 4;
  uint32_t raw[N / 2];
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    raw[4 * i] = raw4[i].x;
    raw[4 * i + 1] = raw4[i].y;
    raw[4 * i + 2] = raw4[i].z;
    raw[4 * i + 3] = raw4[i].w;
  }
  if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) f[i / 2][i % 2] = raw[i];
    return make_float2(1.f, 1.f);
  }
  uint32_t top = 0;                              // largest magnitude's bits (as bf16)
#pragma unroll
  for (int i = 0; i < N / 2; ++i) top = max(top, max(raw[i] & 0x7FFFu, (raw[i] >> 16) & 0x7FFFu));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  // exponent field of the largest, between what keeps both factors normal numbers
  const int e = min(max((int)(top >> 7), 15), 254);
  const float mul = __uint_as_float((uint32_t)(254 + 14 - e) << 23);   // 2^(14 - (e - 127))
  const float inv = __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 v = Elem<T>::unpack2(raw[i]);
    f[i / 2][i % 2] = Elem<__half>::pack2(v.x * mul, v.y * mul);
  }
  return make_float2(__shfl_sync(0xffffffffu, inv, 8 * t), __shfl_sync(0xffffffffu, inv, 8 * t + 4));
}

// The scores of one tile's 16 tokens: c[0], c[1] = token g, heads 2t, 2t+1; c[2], c[3] = token g+8.
template <int HD>
__device__ __forceinline__ void tile_scores(uint32_t codes, uint32_t scales, int g, int t,
                                            const uint32_t (&q)[HD / 16][2], float (&c)[4]) {
  constexpr int W = HD / 32;                     // words of a lane's dims
  uint32_t w[2][W];
  uint32_t sc[2][HD / 64];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint32_t a = codes + (g + 8 * r) * (HD / 2) + t * (HD / 8);
    if constexpr (HD == 64) lds64(a, w[r][0], w[r][1]);
    else lds128(a, w[r]);
#pragma unroll
    for (int u = 0; u < HD / 64; ++u)
      sc[r][u] = lds8(scales + (t * (HD / 64) + u) * kBlock + g + 8 * r) * 0x00800080u;
  }
  c[0] = c[1] = c[2] = c[3] = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    uint32_t a[2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      codes_to_half2(w[r][i], a[r]);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[r][j] = hmul2(a[r][j], sc[r][i / 2]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t frag[4] = {a[0][2 * j], a[1][2 * j], a[0][2 * j + 1], a[1][2 * j + 1]};
      Mma<__half>::run(c, frag, q[2 * i + j][0], q[2 * i + j][1]);
    }
  }
}

// Row of a V code row in shared memory: tokens 0, 2, 4, 6 (and 1, 3, 5, 7) in rows that differ modulo
// 4, so the lanes of one load cover all banks.
__device__ __forceinline__ int v_row(int tok) {
  return (tok & 8) | ((tok & 1) << 2) | ((tok >> 1) & 3);
}

// O^T += V^T P^T for one tile: o[m][0..1] = dim D/8 * g + 2m, heads 2t, 2t+1; o[m][2..3] = the dim
// after it.  `live`: tokens of the tile that exist (the others' scales count as zero).
template <int HD, bool FULL>
__device__ __forceinline__ void tile_values(uint32_t codes, uint32_t scales, int g, int t, int live,
                                            const uint32_t (&p)[2], float (&o)[HD / 16][4]) {
  constexpr int W = HD / 64;                     // words of a lane's dims, per token
  {
    uint32_t w[4][W], sc[2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int tok = 2 * t + (k & 1) + 8 * (k >> 1), row = v_row(tok);
      if constexpr (HD == 64) {
        w[k][0] = lds32(codes + row * 32 + g * 4);
      } else {
        // 64-byte rows: the halves of rows 2 and 3 (modulo 4) change places, see copy_tile
        lds64(codes + row * 64 + ((g * 8) ^ ((row & 2) << 4)), w[k][0], w[k][1]);
      }
    }
    const int grp = HD == 64 ? g >> 1 : g;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t b2 = lds16(scales + grp * kBlock + 2 * t + 8 * k);
      if constexpr (!FULL) {
        const int n = live - (2 * t + 8 * k);
        if (n < 2) b2 = n == 1 ? (b2 & 0xFFu) : 0u;
      }
      sc[k] = __byte_perm(b2, 0, 0x1404) >> 1;   // bytes to the halves' tops, then << 7 in all
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      uint32_t ev[2][4], od[2][4];               // dims 2m and 2m+1, token pairs
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t x = w[2 * k][i], y = w[2 * k + 1][i];
        codes_to_half2((x & 0x0F0F0F0Fu) | ((y << 4) & 0xF0F0F0F0u), ev[k]);
        codes_to_half2(((x >> 4) & 0x0F0F0F0Fu) | (y & 0xF0F0F0F0u), od[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ev[k][j] = hmul2(ev[k][j], sc[k]);
          od[k][j] = hmul2(od[k][j], sc[k]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t frag[4] = {ev[0][j], od[0][j], ev[1][j], od[1][j]};
        Mma<__half>::run(o[4 * i + j], frag, p[0], p[1]);
      }
    }
  }
}

// This lane's 9 copies of a step: the lanes of one tile take neighbouring 16-byte chunks, the V code
// rows land permuted (v_row, and for 64-byte rows with the halves of rows 2 and 3 exchanged).  A
// lane's chunk l + kLanes * i lies in row 4 i + (l / chunks of a row), whose place is a constant of i
// plus one of the lane: `even` and `odd` are the lane's parts for even and odd i.
template <int HD>
struct CopyLane {
  uint32_t k, even, odd;
  __device__ __forceinline__ explicit CopyLane(int l) {
    constexpr int kPer = HD / 32;                // chunks of a row of codes
    const int r = l / kPer, c = l % kPer;
    const uint32_t row = ((r & 1) * 4 + (r >> 1)) * kPer * 16;
    k = l * 16;
    even = Tile<HD>::kV + row + c * 16;
    odd = Tile<HD>::kV + row + (HD == 64 ? c : c ^ 2) * 16;
  }
  __device__ __forceinline__ void copy(uint32_t dst, const uint8_t* src) const {
    constexpr int kStep = Shape<HD>::kLanes * 16, kRowBytes = Tile<HD>::kRow;
    const uint8_t* p = src + k;
#pragma unroll
    for (int i = 0; i < 4; ++i) cp_async16(dst + k + i * kStep, p + i * kStep);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      cp_async16(dst + ((i & 1) ? odd : even) + ((i >> 1) * 8 + (i & 1) * 2) * kRowBytes,
                 p + Tile<HD>::kV + i * kStep);
    cp_async16(dst + k + Tile<HD>::kKs, p + Tile<HD>::kKs);
  }
};

// ln of the sum: m in units of the exponent, l times 2^14 (lg2.approx: off by 2^-22).
__device__ __forceinline__ float row_lse(float m, float l) {
  float g;
  asm("lg2.approx.f32 %0, %1;" : "=f"(g) : "f"(l));
  return ((m == -INFINITY ? 0.f : m - kPScale) + g) * 0.6931471805599453f;
}

// Write a unit's finished rows: heads 2t and 2t+1, this lane's D/8 dims.
template <typename T, int HD>
__device__ __forceinline__ void store_rows(const DecodeParams& p, int b, int h0, int heads, int g,
                                           int t, const float (&o)[HD / 16][4], const float (&m)[2],
                                           const float (&l)[2]) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int h = 2 * t + x;
    if (h >= heads) continue;
    const float r = 1.f / l[x];
    T* out = (T*)p.out + b * p.out_stride + (int64_t)(h0 + h) * HD + g * (HD / 8);
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
      uint4 u;
      u.x = Elem<T>::pack2(o[4 * i][x] * r, o[4 * i][2 + x] * r);
      u.y = Elem<T>::pack2(o[4 * i + 1][x] * r, o[4 * i + 1][2 + x] * r);
      u.z = Elem<T>::pack2(o[4 * i + 2][x] * r, o[4 * i + 2][2 + x] * r);
      u.w = Elem<T>::pack2(o[4 * i + 3][x] * r, o[4 * i + 3][2 + x] * r);
      *reinterpret_cast<uint4*>(out + i * 8) = u;
    }
    if (p.lse && g == 0)
      p.lse[(int64_t)b * p.NH + h0 + h] = row_lse(m[x], l[x]);
  }
}

// A piece of a unit: O [8][HD], m[8], l[8] (m in the exponent's units, l and O times 2^14).
template <int HD>
__device__ __forceinline__ void store_piece(float* dst, int g, int t, const float (&o)[HD / 16][4],
                                            const float (&m)[2], const float (&l)[2]) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    float* row = dst + (2 * t + x) * HD + g * (HD / 8);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
      *reinterpret_cast<float4*>(row + 4 * i) =
          make_float4(o[2 * i][x], o[2 * i][2 + x], o[2 * i + 1][x], o[2 * i + 1][2 + x]);
    if (g == 0) {
      dst[8 * HD + 2 * t + x] = m[x];
      dst[8 * HD + 8 + 2 * t + x] = l[x];
    }
  }
}

// Joining pieces takes HD/4 lanes a row, 4 dims each: half a warp or a warp per (unit, head).
template <int HD>
struct Row {
  static constexpr int kLanes = HD / 4, kWarpsPerUnit = 8 * kLanes / 32;
  int h, j, at;                      // head of the unit, lane of the row, its place in a piece
  __device__ __forceinline__ Row(int warp, int lane)
      : h((warp % kWarpsPerUnit) * (32 / kLanes) + lane / kLanes), j(lane % kLanes), at(h * HD + j * 4) {}
};
__device__ __forceinline__ void fma4(float4& acc, float c, const float4 v) {
  acc.x += c * v.x;
  acc.y += c * v.y;
  acc.z += c * v.z;
  acc.w += c * v.w;
}
template <typename T, int HD>
__device__ __forceinline__ void store_joined(const DecodeParams& p, int b, int h, int j,
                                             const float4 o, float m, float l) {
  const float r = 1.f / l;
  *reinterpret_cast<uint2*>((T*)p.out + b * p.out_stride + (int64_t)h * HD + j * 4) =
      make_uint2(Elem<T>::pack2(o.x * r, o.y * r), Elem<T>::pack2(o.z * r, o.w * r));
  if (p.lse && j == 0) p.lse[(int64_t)b * p.NH + h] = row_lse(m, l);
}

// Add to a counter, after this thread's (and, behind a barrier, its CTA's) writes, before its reads.
__device__ __forceinline__ uint32_t arrive(uint32_t* counter) {
  uint32_t old;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
  return old;
}

// Units cut between the warps of this CTA.  Returns the bits of the entries of sh.cut that other CTAs
// share.
template <typename T, int HD>
__device__ __forceinline__ uint32_t join_warps(const DecodeParams& p, Shared& sh, const float* park,
                                            const float* tails, int cta) {
  using S = Shape<HD>;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // Lane i (modulo 16) stands for warp i's piece of a unit: parked when the unit began before the
  // warp's range, else left in the ring.  Positions count from the CTA's first tile; a unit that began
  // before it has a negative one.
  static_assert(kWarps == 16, "a piece per lane of half a warp");
  const Row<HD> row(warp, lane);
  const int hl = lane & 15, c_len = sh.start[kWarps];
  const int my_start = sh.start[hl], my_end = sh.start[hl + 1];
  const int4 entry = lane <= kWarps ? sh.cut[lane] : make_int4(0, 0, 0, 0);
  uint32_t cuts = __ballot_sync(0xffffffffu, entry.y > 0);
  const uint32_t cross = __ballot_sync(0xffffffffu, entry.y > 0 && (entry.x < 0 || entry.x + entry.y > c_len));
  constexpr int kAtOnce = kWarps / Row<HD>::kWarpsPerUnit;
  for (int i = 0; cuts; ++i, cuts &= cuts - 1) {
    if (i % kAtOnce != warp / Row<HD>::kWarpsPerUnit) continue;
    const int4 u = sh.cut[__ffs(cuts) - 1];
    const int sub = p.subs == 1 ? 0 : u.w % p.subs, kvh = p.subs == 1 ? u.w : u.w / p.subs;
    const int h0 = kvh * p.group + sub * 8, us = u.x, e = u.x + u.y;
    const bool has = my_start < my_end && my_start < e && my_end > us;
    const uint32_t pieces = __ballot_sync(0xffffffffu, has) & 0xFFFFu;
    const int wa = __ffs(pieces) - 1, wb = 31 - __clz(pieces);
    // only its first piece can be a tail: the unit reaches into every later warp from the left
    const float* first = (us < sh.start[wa] ? park : tails) + wa * S::kPiece;
    const float* src = hl == wa ? first : park + hl * S::kPiece;
    const float mi = has ? src[8 * HD + row.h] : -INFINITY;
    const float li = has ? src[8 * HD + 8 + row.h] : 0.f;
    float mm = mi;
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
    // (a piece without a finite score keeps its sum: zero, or NaN)
    const float c = mi == -INFINITY ? 1.f : fast_exp2(mi - mm);
    float ll = c * li;
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, d);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int w = wa; w <= wb; ++w) {
      const float cw = __shfl_sync(0xffffffffu, c, w, 16);
      if ((pieces >> w) & 1u)                      // (else an empty range)
        fma4(acc, cw, *reinterpret_cast<const float4*>((w == wa ? first : park + w * S::kPiece) + row.at));
    }
    if (row.h >= p.group - sub * 8) continue;
    if (us >= 0 && e <= c_len) {
      store_joined<T, HD>(p, u.z, h0 + row.h, row.j, acc, mm, ll);
    } else {
      float* ws = p.parts + ((int64_t)cta * 2 + (us < 0 ? 0 : 1)) * S::kPiece;
      *reinterpret_cast<float4*>(ws + row.at) = acc;
      if (row.j == 0) {
        ws[8 * HD + row.h] = mm;
        ws[8 * HD + 8 + row.h] = ll;
      }
    }
  }
  return cross;
}

// Units that other CTAs share: announce this CTA's pieces; the CTA that is the last of a unit joins
// them, in order.  cross: bits of the entries of sh.cut concerned (one or two).
template <typename T, int HD>
__device__ __forceinline__ void join_ctas(const DecodeParams& p, Shared& sh, uint32_t cross,
                                       uint32_t c_begin, Cut cut_of) {
  using S = Shape<HD>;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hl = lane & 15;
  __syncthreads();
  const int x0 = __ffs(cross) - 1, x1 = 31 - __clz(cross), n_cross = __popc(cross);
  if (tid < n_cross) {
    const int4 u = sh.cut[tid ? x1 : x0];
    const uint32_t s = c_begin + u.x;
    const int fst = cut_of.owner(s) / kWarps, lst = cut_of.owner(s + u.y - 1) / kWarps;
    const bool last = arrive(p.counters + fst) == (uint32_t)(lst - fst);
    if (last) p.counters[fst] = 0;                 // zero again for the next call
    sh.last[tid] = last ? make_int2(fst, lst) : make_int2(-1, -1);
  }
  __syncthreads();
  // the pieces of a unit from all its CTAs, in order
  const Row<HD> row(warp, lane);
  const int x = warp / Row<HD>::kWarpsPerUnit;
  if (x >= n_cross || sh.last[x].x < 0) return;
  const int4 u = sh.cut[x ? x1 : x0];
  const int fst = sh.last[x].x, n = sh.last[x].y - fst + 1;
  const int sub = u.w % p.subs, h0 = (u.w / p.subs) * p.group + sub * 8;
  // (rows of heads beyond the group were not written: their values are loaded, not used)
  auto part = [&](int c) { return p.parts + ((int64_t)(fst + c) * 2 + (c == 0 ? 1 : 0)) * S::kPiece; };
  auto value = [&](int c) { return __ldcg(reinterpret_cast<const float4*>(part(c) + row.at)); };
  float mm = -INFINITY, ll = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c0 = 0; c0 < n; c0 += 16) {             // rounds of 16 pieces, rescaled between them
    const bool in = c0 + hl < n;
    const float mi = in ? __ldcg(part(c0 + hl) + 8 * HD + row.h) : -INFINITY;
    const float li = in ? __ldcg(part(c0 + hl) + 8 * HD + 8 + row.h) : 0.f;
    const int k_n = min(16, n - c0);
    constexpr int kAhead = 4;                      // pieces whose values load beside the sums
    float4 v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) v[k] = k < k_n ? value(c0 + k) : make_float4(0.f, 0.f, 0.f, 0.f);
    float m2 = mi;
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) m2 = fmaxf(m2, __shfl_xor_sync(0xffffffffu, m2, d));
    m2 = fmaxf(mm, m2);
    const float a = mm == -INFINITY ? 1.f : fast_exp2(mm - m2);
    const float f = mi == -INFINITY ? 1.f : fast_exp2(mi - m2);
    float sum = f * li;
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    mm = m2;
    ll = ll * a + sum;
    acc = make_float4(acc.x * a, acc.y * a, acc.z * a, acc.w * a);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fma4(acc, __shfl_sync(0xffffffffu, f, k, 16), v[k]);
#pragma unroll 4
    for (int k = kAhead; k < k_n; ++k) fma4(acc, __shfl_sync(0xffffffffu, f, k, 16), value(c0 + k));
  }
  if (row.h < p.group - sub * 8) store_joined<T, HD>(p, u.z, h0 + row.h, row.j, acc, mm, ll);
}

// UNIT: one CTA per unit instead of the even cut.
template <typename T, int HD, bool UNIT>
__global__ void __launch_bounds__(kWarps * 32, 1) decode_kernel(const __grid_constant__ DecodeParams p) {
  using S = Shape<HD>;
  using L = Tile<HD>;
  extern __shared__ __align__(128) uint8_t smem[];
  float* park = reinterpret_cast<float*>(smem + S::kRing);
  Shared& sh = *reinterpret_cast<Shared*>(smem + S::kRing + S::kPark);
  uint32_t* pref = reinterpret_cast<uint32_t*>(&sh + 1);                      // [batch + 1]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int units = p.KVH * p.subs;
  pdl_wait();
  pdl_launch_dependents();

  // the grains of the batch (in unit mode: of this CTA's sequence)
  const int cap = (int)min((int64_t)p.max_blocks * kBlock, (int64_t)0x7FFFFFFF);
  constexpr int grain = UNIT ? 1 : S::kTiles;      // tiles
  uint32_t total;
  int ctas;
  if constexpr (UNIT) {
    const int len = min(p.ctx[blockIdx.x / units], cap);
    ctas = 1;
    total = len > 0 ? (len - 1) / kBlock + 1 : 0;
  } else {
    const Place pl = scan_batch<S::kTiles>(p.ctx, p.batch, cap, units, pref, sh.scan);
    total = pl.total;
    ctas = pl.ctas;
  }
  const int cta = UNIT ? 0 : blockIdx.x;
  if (total == 0 || cta >= ctas) return;
  const Cut cut_of(total, (uint32_t)ctas * kWarps);
  const uint32_t c_begin = cut_of.start(cta * kWarps);
  const uint32_t w_begin = cut_of.start(cta * kWarps + warp);

  Cursor cur;
  cur.left = (int)(cut_of.start(cta * kWarps + warp + 1) - w_begin);
  if constexpr (UNIT) {
    cur.b = blockIdx.x / units;
    cur.hv = blockIdx.x % units;
    cur.n = (int)total;
    cur.tail = 1;
    cur.at = (int)w_begin;
  } else {
    find_place(w_begin, p.batch, units, pref, lane, cur);
  }
  if (lane == 0) {
    sh.start[warp] = (int)(w_begin - c_begin);
    if (warp == kWarps - 1) sh.start[kWarps] = (int)(w_begin - c_begin) + cur.left;
    sh.cut[warp] = make_int4(0, 0, 0, 0);
    if (warp == 0) sh.cut[kWarps] = make_int4(0, 0, 0, 0);
  }

  float o[HD / 16][4], m[2], l[2];
  bool tail = false;                               // a piece is left in registers after the loop
  const bool head_cut = cur.at > 0;               // the first unit began before this warp
  if (cur.left > 0) {
    const uint32_t ring = smem_u32(smem) + warp * (kStages * kStepBytes);
    // copies run one step ahead of the arithmetic, the block ids one step ahead of the copies
    const int j = lane / S::kLanes;
    const CopyLane<HD> mine(lane % S::kLanes);
    const uint32_t my_tile = ring + j * L::kBytes;
    const uint32_t num_blocks = (uint32_t)min(p.num_blocks, (int64_t)0x7FFFFFFF);
    const int64_t block_bytes = (int64_t)p.KVH * L::kBytes;
    Cursor ld = cur;
    int ld_left = 0, ld_stage = 0, id = -1;
    const int32_t* ids = nullptr;
    const uint8_t* pool_h = nullptr;
    auto open_loads = [&]() {
      const int row = p.row_index ? p.row_index[ld.b] : ld.b;
      ids = p.tables + (int64_t)row * p.bt_stride + (int64_t)ld.at * grain + j;
      pool_h = p.pool + (int64_t)(p.subs == 1 ? ld.hv : ld.hv / p.subs) * L::kBytes;
      ld_left = ld.piece_tiles(grain);
    };
    open_loads();
    id = j < ld_left ? *ids : -1;
    // start the next step's copies; returns which of its tiles exist (bits of S::kFirsts)
    auto issue = [&]() -> uint32_t {
      const bool ok = (uint32_t)id < num_blocks;
      if (ok) mine.copy(my_tile + ld_stage, pool_h + id * block_bytes);
      cp_commit();
      ld_stage = kStepBytes - ld_stage;
      ids += S::kTiles;
      ld_left -= S::kTiles;
      if (!UNIT && ld_left <= 0 && ld.left > 0) {
        ld.next_unit(units, pref, p.batch);
        if (ld.left > 0) open_loads();
      }
      id = j < ld_left ? *ids : -1;
      return __ballot_sync(0xffffffffu, ok) & S::kFirsts;
    };
    uint32_t qf[HD / 16][2];
    float2 sc = make_float2(0.f, 0.f);
    int ctx = 0, heads = 0, h0 = 0;
    uint4 raw[HD / 32];
    auto load_unit = [&]() {
      const int kvh = cur.hv / p.subs, sub = cur.hv % p.subs;
      h0 = kvh * p.group + sub * 8;
      heads = min(8, p.group - sub * 8);
      ctx = min(p.ctx[cur.b], cap);
      load_query<T, HD>((const T*)p.q + cur.b * p.q_stride + (int64_t)h0 * HD, heads, g, t, raw);
    };
    auto open_unit = [&]() {
      const float2 inv = convert_query<T, HD>(raw, t, qf);
      sc = make_float2(inv.x * p.scale_log2, inv.y * p.scale_log2);
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
    };
    load_unit();                                   // (in flight beside the first block ids)
    uint32_t ok_next = issue();
    open_unit();
    const int total_left = cur.left;
    bool first = true;
    // one step: full = all tiles exist and all their tokens are within the length
    auto run_step = [&](auto full_t, uint32_t st, uint32_t ok, int live) {
      constexpr bool FULL = decltype(full_t)::value;
      float s[S::kTiles][4];
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int x = 0; x < S::kTiles; ++x) {
        if (FULL || ((ok >> (x * S::kLanes)) & 1u)) {
          tile_scores<HD>(st + x * L::kBytes + L::kK, st + x * L::kBytes + L::kKs, g, t, qf, s[x]);
          if constexpr (!FULL) {
            const int n = live - x * kBlock;
            if (g >= n) s[x][0] = s[x][1] = -INFINITY;
            if (g + 8 >= n) s[x][2] = s[x][3] = -INFINITY;
          }
        } else {
          s[x][0] = s[x][1] = s[x][2] = s[x][3] = -INFINITY;
        }
        mx0 = fmaxf(mx0, fmaxf(s[x][0], s[x][2]));
        mx1 = fmaxf(mx1, fmaxf(s[x][1], s[x][3]));
      }
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, d));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, d));
      }
      const float n0 = fmaxf(m[0], mx0 * sc.x), n1 = fmaxf(m[1], mx1 * sc.y);
      if (__any_sync(0xffffffffu, n0 != m[0] || n1 != m[1])) {
        // (a row that had no token yet: its sums are zero, and stay so)
        const float a0 = m[0] == -INFINITY ? 0.f : fast_exp2(m[0] - n0);
        const float a1 = m[1] == -INFINITY ? 0.f : fast_exp2(m[1] - n1);
        l[0] *= a0;
        l[1] *= a1;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          o[i][0] *= a0;
          o[i][1] *= a1;
          o[i][2] *= a0;
          o[i][3] *= a1;
        }
        m[0] = n0;
        m[1] = n1;
      }
      const float f0 = kPScale - (n0 == -INFINITY ? 0.f : n0), f1 = kPScale - (n1 == -INFINITY ? 0.f : n1);
#pragma unroll
      for (int x = 0; x < S::kTiles; ++x) {
        if (!FULL && !((ok >> (x * S::kLanes)) & 1u)) continue;
        const float e0 = fast_exp2(fmaf(s[x][0], sc.x, f0)), e1 = fast_exp2(fmaf(s[x][1], sc.y, f1));
        const float e2 = fast_exp2(fmaf(s[x][2], sc.x, f0)), e3 = fast_exp2(fmaf(s[x][3], sc.y, f1));
        l[0] += e0 + e2;
        l[1] += e1 + e3;
        const uint32_t pt[2] = {transpose8x8(Elem<__half>::pack2(e0, e1)),
                                transpose8x8(Elem<__half>::pack2(e2, e3))};
        tile_values<HD, FULL>(st + x * L::kBytes + L::kV, st + x * L::kBytes + L::kVs, g, t,
                              live - x * kBlock, pt, o);
      }
    };
    for (uint32_t st = ring;;) {                   // one unit's tiles
      int live = ctx - cur.at * grain * kBlock;    // its tokens from the step's first on
      for (int rem = cur.piece_tiles(grain); rem > 0; rem -= S::kTiles, live -= S::kTiles * kBlock) {
        const uint32_t ok = ok_next;
        ok_next = issue();                         // (an empty group when nothing is left)
        cp_wait<1>();
        __syncwarp();
        if (ok == S::kFirsts && live >= S::kTiles * kBlock) run_step(std::true_type{}, st, ok, live);
        else run_step(std::false_type{}, st, ok, live);
        __syncwarp();                              // the stage is free for the copies after next
        st = 2 * ring + kStepBytes - st;
      }
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[0] += __shfl_xor_sync(0xffffffffu, l[0], d);
        l[1] += __shfl_xor_sync(0xffffffffu, l[1], d);
      }
      const bool cut = first && head_cut;
      if (cur.n - cur.at <= cur.left && !cut) {   // the unit whole
        store_rows<T, HD>(p, cur.b, h0, heads, g, t, o, m, l);
      } else {
        if (cut) store_piece<HD>(park + warp * S::kPiece, g, t, o, m, l);
        else tail = true;
        if (lane == 0 && (!cut || warp == 0))
          sh.cut[cut ? kWarps : warp] = make_int4(
              (int)(w_begin - c_begin) + total_left - cur.left - cur.at, cur.n, cur.b, cur.hv);
      }
      first = false;
      if constexpr (UNIT) break;
      cur.next_unit(units, pref, p.batch);
      if (cur.left == 0) break;
      load_unit();
      open_unit();
    }
    cp_wait<0>();
  }
  __syncthreads();
  // the rings are free: pieces that are still in registers go there
  float* tails = reinterpret_cast<float*>(smem);
  if (tail) store_piece<HD>(tails + warp * S::kPiece, g, t, o, m, l);
  __syncthreads();

  const uint32_t cross = join_warps<T, HD>(p, sh, park, tails, cta);
  if constexpr (!UNIT)
    if (cross) join_ctas<T, HD>(p, sh, cross, c_begin, cut_of);
}

// ---- attention-weight totals ------------------------------------------------------------------------
// weights += sum over the kv head's query heads of exp(q.k / sqrt(D) - lse), a read of the K half of the
// cache (9/16 D bytes a token and kv head) and 8 bytes of totals.  The same stream, cut, scores and
// two-stage ring as the decode kernel, without anything to join: a token belongs to one warp.  A step
// is 8 tiles (D = 64; 4 for D = 128).  Heads are the columns of the scores, so a token's total is the sum
// of two columns over four lanes; a step's totals are brought together by a reduce-scatter (12
// shuffles for 8 tiles instead of 32) and go through shared memory to the lanes that hold the old
// totals, four tokens each, loaded a step ahead.  Measured: 32 x U[8192, 32768] 15.6 us (3.7 TB/s, 0.57
// of measured copy), 256 x U[128, 2048] 8.8 us: the decode kernel's fixed costs on half its bytes.
struct WeightParams {
  float* out;
  const float* in;
  const void* q;
  const float* lse;
  const uint8_t* pool;
  int64_t q_stride, num_blocks, bt_stride;
  const int32_t *tables, *row_index, *ctx;
  int batch, NH, KVH, group, max_blocks;
  float scale_log2;
};

template <int HD>
struct WShape {
  static constexpr int kTileBytes = 9 * HD;                      // K codes, K scales
  static constexpr int kTiles = kStepBytes / kTileBytes;
  static constexpr int kLanes = 32 / kTiles;
  static constexpr int kRing = kWarps * 2 * kStepBytes;
  static constexpr int kSums = kWarps * kTiles * kBlock * 4;
  static size_t smem(int batch) { return kRing + kSums + kWarps * 4 + ((size_t)batch + 1) * 4; }
};

// NS: groups of at most 8 query heads per kv head.
template <typename T, int HD, int NS>
__global__ void __launch_bounds__(kWarps * 32, 1) weights_kernel(const __grid_constant__ WeightParams p) {
  using S = WShape<HD>;
  using L = Tile<HD>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  float* sums = reinterpret_cast<float*>(smem + S::kRing) + warp * S::kTiles * kBlock;
  uint32_t* scan = reinterpret_cast<uint32_t*>(smem + S::kRing + S::kSums);
  uint32_t* pref = scan + kWarps;
  pdl_wait();
  pdl_launch_dependents();
  const int cap = (int)min((int64_t)p.max_blocks * kBlock, (int64_t)0x7FFFFFFF);
  const Place pl = scan_batch<S::kTiles>(p.ctx, p.batch, cap, p.KVH, pref, scan);
  if (pl.total == 0 || (int)blockIdx.x >= pl.ctas) return;
  const Cut cut_of(pl.total, (uint32_t)pl.ctas * kWarps);
  const uint32_t w_begin = cut_of.start(blockIdx.x * kWarps + warp);
  Cursor cur;
  cur.left = (int)(cut_of.start(blockIdx.x * kWarps + warp + 1) - w_begin);
  if (cur.left == 0) return;
  find_place(w_begin, p.batch, p.KVH, pref, lane, cur);

  const uint32_t ring = smem_u32(smem) + warp * (2 * kStepBytes);
  const int j = lane / S::kLanes, cl = lane % S::kLanes;
  const uint32_t my_tile = ring + j * S::kTileBytes + cl * 16;
  const uint32_t num_blocks = (uint32_t)min(p.num_blocks, (int64_t)0x7FFFFFFF);
  Cursor ld = cur;
  int ld_left = 0, ld_stage = 0, id = -1;
  const int32_t* ids = nullptr;
  auto open_loads = [&]() {
    const int row = p.row_index ? p.row_index[ld.b] : ld.b;
    ids = p.tables + (int64_t)row * p.bt_stride + (int64_t)ld.at * S::kTiles + j;
    ld_left = ld.piece_tiles(S::kTiles);
  };
  open_loads();
  id = j < ld_left ? *ids : -1;
  // old totals of the next step: lane (tile j, quarter cl) holds tokens 4 cl .. 4 cl + 3
  float4 w_next = make_float4(0.f, 0.f, 0.f, 0.f);
  int64_t at_next = -1;
  auto issue = [&]() {
    const bool ok = (uint32_t)id < num_blocks;
    at_next = -1;
    if (ok) {
      const int64_t tile = (int64_t)id * p.KVH + ld.hv;
      const uint8_t* src = p.pool + tile * L::kBytes + cl * 16;
#pragma unroll
      for (int i = 0; i < 8; ++i) cp_async16(my_tile + ld_stage + i * S::kLanes * 16, src + i * S::kLanes * 16);
      cp_async16(my_tile + ld_stage + 8 * HD, src + L::kKs);
      if (cl < 4) {
        at_next = tile * kBlock + cl * 4;
        w_next = *reinterpret_cast<const float4*>(p.in + at_next);
      }
    }
    cp_commit();
    ld_stage = kStepBytes - ld_stage;
    ids += S::kTiles;
    ld_left -= S::kTiles;
    if (ld_left <= 0 && ld.left > 0) {
      ld.next_unit(p.KVH, pref, p.batch);
      if (ld.left > 0) open_loads();
    }
    id = j < ld_left ? *ids : -1;
  };

  uint32_t qf[NS][HD / 16][2];
  float2 sc[NS], off[NS];
  int ctx = 0;
  auto open_unit = [&](bool start) {
    uint4 raw[NS][HD / 32];
#pragma unroll
    for (int u = 0; u < NS; ++u)
      load_query<T, HD>((const T*)p.q + cur.b * p.q_stride + ((int64_t)cur.hv * p.group + u * 8) * HD,
                        min(8, p.group - u * 8), g, t, raw[u]);
    ctx = min(p.ctx[cur.b], cap);
    const float* lse = p.lse + (int64_t)cur.b * p.NH + cur.hv * p.group;
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      // heads beyond the group weigh nothing: 2^(0 - inf)
      const int h = u * 8 + 2 * t;
      off[u].x = h < p.group ? -1.4426950408889634f * lse[h] : -INFINITY;
      off[u].y = h + 1 < p.group ? -1.4426950408889634f * lse[h + 1] : -INFINITY;
    }
    if (start) issue();
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const float2 inv = convert_query<T, HD>(raw[u], t, qf[u]);
      sc[u] = make_float2(inv.x * p.scale_log2, inv.y * p.scale_log2);
    }
  };
  open_unit(true);
  for (uint32_t st = ring;;) {
    int live = ctx - cur.at * (S::kTiles * kBlock);
    for (int rem = cur.piece_tiles(S::kTiles); rem > 0; rem -= S::kTiles, live -= S::kTiles * kBlock) {
      const float4 w = w_next;
      const int64_t at = at_next;
      issue();                                     // (an empty group when nothing is left)
      cp_wait<1>();
      __syncwarp();
      float v[S::kTiles * 2];                      // [tile][token g, token g + 8], two heads summed
#pragma unroll
      for (int x = 0; x < S::kTiles; ++x) {
        v[2 * x] = v[2 * x + 1] = 0.f;
        if (x >= rem) continue;
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          float c[4];
          tile_scores<HD>(st + x * S::kTileBytes, st + x * S::kTileBytes + 8 * HD, g, t, qf[u], c);
          v[2 * x] += fast_exp2(fmaf(c[0], sc[u].x, off[u].x)) + fast_exp2(fmaf(c[1], sc[u].y, off[u].y));
          v[2 * x + 1] += fast_exp2(fmaf(c[2], sc[u].x, off[u].x)) + fast_exp2(fmaf(c[3], sc[u].y, off[u].y));
        }
      }
      // sum over the four lanes of a token; lane t keeps tiles t and t + 4
      float h1[S::kTiles], h2[S::kTiles / 2];
#pragma unroll
      for (int k = 0; k < S::kTiles; ++k) {        // k = 2 * (tile / 2) + row: tiles of this lane's parity
        const float even = v[4 * (k / 2) + k % 2], odd = v[4 * (k / 2) + 2 + k % 2];
        h1[k] = ((t & 1) ? odd : even) + __shfl_xor_sync(0xffffffffu, (t & 1) ? even : odd, 1);
      }
#pragma unroll
      for (int k = 0; k < S::kTiles / 2; ++k) {
        const float lo = h1[4 * (k / 2) + k % 2], hi = h1[4 * (k / 2) + 2 + k % 2];
        h2[k] = ((t & 2) ? hi : lo) + __shfl_xor_sync(0xffffffffu, (t & 2) ? lo : hi, 2);
      }
#pragma unroll
      for (int k = 0; k < S::kTiles / 2; ++k)
        sums[(4 * (k / 2) + t) * kBlock + g + 8 * (k % 2)] = h2[k];
      __syncwarp();
      if (at >= 0) {
        const float4 n = *reinterpret_cast<const float4*>(sums + j * kBlock + cl * 4);
        const int left = live - j * kBlock - cl * 4;
        float* out = p.out + at;
        if (left >= 4) {
          *reinterpret_cast<float4*>(out) = make_float4(w.x + n.x, w.y + n.y, w.z + n.z, w.w + n.w);
        } else {
          if (left > 0) out[0] = w.x + n.x;
          if (left > 1) out[1] = w.y + n.y;
          if (left > 2) out[2] = w.z + n.z;
        }
      }
      __syncwarp();                                // the stage and the sums are free again
      st = 2 * ring + kStepBytes - st;
    }
    cur.next_unit(p.KVH, pref, p.batch);
    if (cur.left == 0) break;
    open_unit(false);
  }
  cp_wait<0>();
}

constexpr int kMaxCtas = 256;
constexpr size_t kCounterBytes = kMaxCtas * 4;
// Widest table that runs one CTA per unit (the lengths are on the device: a short context behind a wider
// table takes the even cut).  8 sequences, 14 heads of 64 dims over 2: 512 tokens 7.7 us
// against 8.6 for the even cut, 1536 tokens 9.9 against 10.8, 2048 tokens 10.7 against 11.0, 4096 tokens
// 14.9 against 11.2; 32 heads of 128 over 8: 1536 tokens 13.2 against 14.2, 2048 tokens 14.9 against 14.4.
constexpr int kUnitBlocks = 96;

// One CTA per SM of the current device (its ring fills the shared memory).
static int decode_ctas() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
    (void)cudaGetLastError();
    sms = 148;
  }
  return std::min(sms, kMaxCtas);
}

// Raise a kernel's shared-memory limit, once per device (bits of `ready`).
template <typename K>
static int allow_smem(K kern, size_t bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (ready.load(std::memory_order_acquire) & bit) return TI_OK;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return set_cuda_error(e, "cudaFuncSetAttribute(kv4)");
  }
  ready.fetch_or(bit, std::memory_order_release);
  return TI_OK;
}

template <typename T, int HD, int NS>
static int launch_weights(const WeightParams& p, dim3 grid, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  if (int rc = allow_smem(weights_kernel<T, HD, NS>, WShape<HD>::smem(kMaxBatch), ready)) return rc;
  return launch_kernel("kv4 weights launch", weights_kernel<T, HD, NS>, grid, dim3(kWarps * 32),
                       WShape<HD>::smem(p.batch), s, 1, p);
}

template <typename T, int HD, bool UNIT>
static int launch_decode(const DecodeParams& p, dim3 grid, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  if (int rc = allow_smem(decode_kernel<T, HD, UNIT>, Shape<HD>::smem(kMaxBatch), ready)) return rc;
  return launch_kernel("kv4 attention launch", decode_kernel<T, HD, UNIT>, grid, dim3(kWarps * 32),
                       Shape<HD>::smem(UNIT ? 0 : p.batch), s, 1, p);
}

static int check_shape(int batch, int NH, int KVH, int HD, int block_size,
                       int max_blocks, int64_t num_blocks, int dtype) {
  if (batch < 0 || max_blocks <= 0 || num_blocks <= 0 || KVH <= 0 || NH <= 0 || NH % KVH)
    return set_error(TI_ERR_INVALID_ARGUMENT,
                     "kv4: bad batch, table width, pool size or head counts (num_heads must be a multiple of num_kv_heads)");
  if (HD != 64 && HD != 128) return set_error(TI_ERR_UNSUPPORTED, "kv4: head_dim must be 64 or 128");
  if (block_size != kBlock) return set_error(TI_ERR_UNSUPPORTED, "kv4: block_size must be 16");
  if (NH / KVH > 16) return set_error(TI_ERR_UNSUPPORTED, "kv4: at most 16 query heads per kv head");
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_FP16)
    return set_error(TI_ERR_UNSUPPORTED, "kv4: dtype must be bf16 or fp16");
  if (batch > kMaxBatch) return set_error(TI_ERR_UNSUPPORTED, "kv4: at most 4096 sequences per call");
  if ((int64_t)batch * max_blocks * KVH * ((NH / KVH + 7) / 8) >= (int64_t)1 << 29)
    return set_error(TI_ERR_UNSUPPORTED,
                     "kv4: batch * table width * kv heads (twice beyond 8 query heads each) must be below 2^29");
  return TI_OK;
}

}  // namespace kv4
}  // namespace ti

using namespace ti;

extern "C" size_t ti_kv4_attention_workspace_bytes(int batch, int num_heads, int num_kv_heads,
                                                   int head_dim, int max_blocks_per_seq) {
  (void)batch; (void)num_heads; (void)num_kv_heads; (void)max_blocks_per_seq;
  return kv4::kCounterBytes + (size_t)kv4::decode_ctas() * 2 * (8 * (size_t)head_dim + 16) * 4;
}

extern "C" int ti_kv4_attention_decode(void* out, int64_t out_seq_stride, float* lse,
                                       const void* q, int64_t q_seq_stride, const void* pool,
                                       int64_t num_blocks, const int32_t* block_tables,
                                       int64_t bt_stride, const int32_t* row_index,
                                       const int32_t* context_lens, int batch, int num_heads,
                                       int num_kv_heads, int head_dim, int block_size,
                                       int max_blocks_per_seq, int dtype, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  clear_error();
  if (batch == 0) return TI_OK;
  if (!out || !q || !pool || !block_tables || !context_lens || !workspace)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4 attention: null pointer");
  if (int rc = kv4::check_shape(batch, num_heads, num_kv_heads, head_dim, block_size,
                                max_blocks_per_seq, num_blocks, dtype))
    return rc;
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) |
        reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      (out_seq_stride % 8) || (q_seq_stride % 8))
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4 attention: tensors must be 16-byte aligned");
  if (workspace_bytes < ti_kv4_attention_workspace_bytes(batch, num_heads, num_kv_heads, head_dim,
                                                         max_blocks_per_seq))
    return set_error(TI_ERR_WORKSPACE, "kv4 attention: workspace too small");
  const int group = num_heads / num_kv_heads, subs = (group + 7) / 8;
  const int ctas = kv4::decode_ctas();
  const int64_t units = (int64_t)batch * num_kv_heads * subs;
  const bool unit_mode = units <= ctas && max_blocks_per_seq <= kv4::kUnitBlocks;
  kv4::DecodeParams p{out, lse, q, (const uint8_t*)pool, out_seq_stride, q_seq_stride, num_blocks,
                      bt_stride, block_tables, row_index, context_lens, batch, num_heads,
                      num_kv_heads, group, max_blocks_per_seq, subs,
                      1.4426950408889634f / sqrtf((float)head_dim), (uint32_t*)workspace,
                      (float*)((uint8_t*)workspace + kv4::kCounterBytes)};
  const dim3 grid(unit_mode ? (unsigned)units : (unsigned)ctas);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    return unit_mode ? kv4::launch_decode<T, HD, true>(p, grid, s)
                     : kv4::launch_decode<T, HD, false>(p, grid, s);
  };
  auto go_dim = [&](auto t) {
    return head_dim == 64 ? go(t, std::integral_constant<int, 64>{})
                          : go(t, std::integral_constant<int, 128>{});
  };
  return dtype == TI_DTYPE_BF16 ? go_dim(__nv_bfloat16{}) : go_dim(__half{});
}

extern "C" int ti_kv4_accumulate_weights(float* weights_out, const float* weights, const void* q,
                                         int64_t q_seq_stride, const float* lse, const void* pool,
                                         int64_t num_blocks, const int32_t* block_tables,
                                         int64_t bt_stride, const int32_t* row_index,
                                         const int32_t* context_lens, int batch, int num_heads,
                                         int num_kv_heads, int head_dim, int block_size,
                                         int max_blocks_per_seq, int dtype, void* stream) {
  clear_error();
  if (batch == 0) return TI_OK;
  if (!weights_out || !weights || !q || !lse || !pool || !block_tables || !context_lens)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4 weights: null pointer");
  if (int rc = kv4::check_shape(batch, num_heads, num_kv_heads, head_dim,
                                block_size, max_blocks_per_seq, num_blocks, dtype))
    return rc;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pool) |
        reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(weights_out)) & 15) ||
      (q_seq_stride % 8))
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4 weights: tensors must be 16-byte aligned");
  kv4::WeightParams p{weights_out, weights, q, lse, (const uint8_t*)pool, q_seq_stride, num_blocks,
                      bt_stride, block_tables, row_index, context_lens, batch, num_heads,
                      num_kv_heads, num_heads / num_kv_heads, max_blocks_per_seq,
                      1.4426950408889634f / sqrtf((float)head_dim)};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(kv4::decode_ctas());
  auto go = [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    return p.group <= 8 ? kv4::launch_weights<T, HD, 1>(p, grid, s) : kv4::launch_weights<T, HD, 2>(p, grid, s);
  };
  auto go_dim = [&](auto t) {
    return head_dim == 64 ? go(t, std::integral_constant<int, 64>{})
                          : go(t, std::integral_constant<int, 128>{});
  };
  return dtype == TI_DTYPE_BF16 ? go_dim(__nv_bfloat16{}) : go_dim(__half{});
}
