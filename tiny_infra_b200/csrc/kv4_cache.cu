// The 4-bit KV cache's writes and moves: quantise-and-append (with or without RoPE), read back as
// 16-bit values, and eviction by accumulated attention weight.  Format: kv4.cuh.
#include <algorithm>

#include "capi_internal.h"
#include "common.cuh"
#include "kv4.cuh"
#include "rmsnorm_row.cuh"

namespace ti {
namespace kv4 {

using ew::Vec8;

// 16 consecutive elements of a 16-bit type as floats (two 16-byte loads).
template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&f)[16]) {
  Vec8<T> a, b;
  a.load(p);
  b.load(p + 8);
  a.to_float(f);
  b.to_float(f + 8);
}

// Store one quantised group of token `off` of a tile.
template <int HD>
__device__ __forceinline__ void store_group(uint8_t* tile, bool is_v, int off, int g,
                                            const float (&f)[16]) {
  using L = Tile<HD>;
  uint32_t sb;
  const uint2 c = quantize16(f, sb);
  *reinterpret_cast<uint2*>(tile + (is_v ? L::kV : L::kK) + off * L::kRow + g * 8) = c;
  tile[(is_v ? L::kVs : L::kKs) + g * kBlock + off] = (uint8_t)sb;
}

// ---- append -------------------------------------------------------------------------------------
// One thread per (token, K or V of a head, group of 16 dims): 32 bytes in, 9 bytes out.  The
// groups of a token run over neighbouring lanes and then the tokens, so a warp writes whole
// 32-byte rows of codes and runs of scale bytes.
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
  const int64_t per = (int64_t)p.tokens * L::kGroups, total = per * 2 * p.KVH;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int hv = (int)(i / per), h = hv >> 1, g = (int)(i % L::kGroups);
    const int t = (int)((i % per) / L::kGroups);
    const bool is_v = hv & 1;
    const int64_t slot = p.slots[t];
    if (slot < 0) continue;
    if (slot >= p.pool_slots) {
      if (hv == 0 && g == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
      continue;
    }
    const T* src = is_v ? (const T*)p.v + t * p.v_tok + h * p.v_head
                        : (const T*)p.k + t * p.k_tok + h * p.k_head;
    float f[16];
    load16(src + g * kGroup, f);
    const int64_t tile = (slot / kBlock) * p.KVH + h;
    const int off = (int)(slot % kBlock);
    store_group<HD>(p.pool + tile * L::kBytes, is_v, off, g, f);
    if (p.weights && !is_v && g == 0) p.weights[tile * kBlock + off] = 0.f;
  }
}

// ---- read back ------------------------------------------------------------------------------------
// One thread per (table entry, head, K or V, token, group): 9 bytes in, 32 bytes out; zeros behind
// the row's length.
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

template <typename T, int HD>
__global__ void dequantize_kernel(DequantParams p) {
  pdl_wait();
  pdl_launch_dependents();
  using L = Tile<HD>;
  constexpr int kPerTile = 2 * kBlock * L::kGroups;
  const int64_t entries = (int64_t)p.rows * p.max_blocks;
  const int64_t total = entries * p.KVH * kPerTile;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int w = (int)(i % kPerTile);
    const int64_t eh = i / kPerTile;
    const int h = (int)(eh % p.KVH);
    const int64_t entry = eh / p.KVH;
    const int r = (int)(entry / p.max_blocks), j = (int)(entry % p.max_blocks);
    const int len = p.lens[r];
    if ((int64_t)j * kBlock >= len) continue;
    const int32_t dst = p.out_tables[r * p.ot_stride + j];
    if (dst < 0) continue;
    if (dst >= p.out_blocks) {
      if (w == 0 && h == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
      continue;
    }
    const int32_t src = p.tables[(p.row_index ? p.row_index[r] : r) * p.bt_stride + j];
    const bool is_v = w >= kPerTile / 2;
    const int off = (w / L::kGroups) % kBlock, g = w % L::kGroups;
    Vec8<T> lo, hi;
    lo.raw = hi.raw = make_uint4(0u, 0u, 0u, 0u);
    if (src >= 0 && src < p.num_blocks && j * kBlock + off < len) {
      const uint8_t* tile = p.pool + ((int64_t)src * p.KVH + h) * L::kBytes;
      const uint2 c = *reinterpret_cast<const uint2*>(tile + (is_v ? L::kV : L::kK) +
                                                      off * L::kRow + g * 8);
      const float s = scale_value(tile[(is_v ? L::kVs : L::kKs) + g * kBlock + off]);
      uint32_t h4[4];
      float f[16];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        codes_to_half2(u ? c.y : c.x, h4);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 v = Elem<__half>::unpack2(h4[q]);
          f[u * 8 + 2 * q] = v.x * s;
          f[u * 8 + 2 * q + 1] = v.y * s;
        }
      }
      lo.from_float(f);
      hi.from_float(f + 8);
    }
    T* out = (T*)(is_v ? p.v_out : p.k_out) +
             (((int64_t)dst * p.KVH + h) * kBlock + off) * HD + g * kGroup;
    lo.store(out);
    hi.store(out + 8);
  }
}

// ---- eviction -------------------------------------------------------------------------------------
// One CTA per (layer, sequence, kv head).  With n cached tokens and n > keep it keeps the last
// `recent` and the keep - recent heaviest of the older ones (ties: the earlier token), in order.
// The weight of the lightest kept token is found by a radix select over order-preserving 32-bit
// keys (4 passes of 8 bits); then the tokens are scanned in order and each kept one's codes, scales
// and weight move to the next place in front.  A place is never behind its token, and a round
// reads all of its tokens before it writes any, so the move may be in place.
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

constexpr int kEvictThreads = 256;

// Larger weight, larger key; NaN counts as the largest, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(w + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <int HD>
__global__ void __launch_bounds__(kEvictThreads) evict_kernel(EvictParams p) {
  pdl_wait();
  pdl_launch_dependents();
  using L = Tile<HD>;
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ uint32_t hist[256];
  __shared__ uint32_t s_prefix, s_left;
  __shared__ int s_bad, s_warp[kEvictThreads / 32];
  const int row = p.row_index ? p.row_index[b] : b;
  const int n = p.ctx[b];
  if (n <= 0) return;
  int32_t* kept = p.kept ? p.kept + ((int64_t)(layer * p.batch + b) * p.KVH + h) * p.kept_stride
                         : nullptr;
  const int32_t* src_row = p.tables + (int64_t)row * p.bt_stride;
  const int32_t* dst_row = p.out_tables + (int64_t)row * p.ot_stride;
  const int m = min(n, p.keep);
  // every block of the sequence, and every block that the survivors go to, has to be in the pool
  const int nb = (n - 1) / kBlock + 1, mb = (m - 1) / kBlock + 1;
  if (tid == 0) s_bad = (nb > p.max_blocks || mb > p.out_max_blocks);
  __syncthreads();
  if (!s_bad) {
    bool bad = false;
    for (int j = tid; j < nb; j += kEvictThreads) {
      bad |= (uint32_t)src_row[j] >= (uint64_t)p.num_blocks;
      if (j < mb) bad |= (uint32_t)dst_row[j] >= (uint64_t)p.num_blocks;
    }
    if (bad) s_bad = 1;
  }
  __syncthreads();
  if (s_bad) {
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
      for (int i = tid; i < old; i += kEvictThreads) {
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
  for (int i0 = 0; i0 < n; i0 += kEvictThreads) {
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
      for (int k = 0; k < kEvictThreads / 32; ++k) {
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
  const dim3 grid(kv4::grid_for((int64_t)num_tokens * num_kv_heads * (head_dim / 8), 256));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) { return launch_kernel("kv4_append launch", kern, grid, dim3(256), 0, s, 1, p); };
  if (dtype == TI_DTYPE_BF16)
    return head_dim == 64 ? go(kv4::append_kernel<__nv_bfloat16, 64>)
                          : go(kv4::append_kernel<__nv_bfloat16, 128>);
  return head_dim == 64 ? go(kv4::append_kernel<__half, 64>) : go(kv4::append_kernel<__half, 128>);
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
  const dim3 grid(kv4::grid_for((int64_t)rows * max_blocks * num_kv_heads * 2 * head_dim, 256));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) { return launch_kernel("kv4_dequantize launch", kern, grid, dim3(256), 0, s, 1, p); };
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
  if (reinterpret_cast<uintptr_t>(pool) & 15)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4_evict: the pool must be 16-byte aligned");
  if (batch > 65535 || num_layers > 65535)
    return set_error(TI_ERR_UNSUPPORTED, "kv4_evict: at most 65535 sequences and layers");
  kv4::EvictParams p{(uint8_t*)pool, weights, num_blocks, block_tables, bt_stride, out_tables,
                     ot_stride, row_index, context_lens, kept, kept_stride, batch, num_kv_heads,
                     max_blocks_per_seq, out_max_blocks, keep, recent};
  const dim3 grid(num_kv_heads, batch, num_layers);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return launch_kernel("kv4_evict launch", head_dim == 64 ? kv4::evict_kernel<64> : kv4::evict_kernel<128>,
                       grid, dim3(kv4::kEvictThreads), 0, s, 1, p);
}
