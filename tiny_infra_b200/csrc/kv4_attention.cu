// Decode attention over the 4-bit paged KV cache, and the attention-weight totals that eviction
// ranks tokens by.  Format: kv4.cuh.
#include <algorithm>

#include "capi_internal.h"
#include "common.cuh"
#include "kv4.cuh"

namespace ti {
namespace kv4 {

struct DecodeParams {
  void* out;
  float* lse;                        // [batch, NH] or null
  const void* q;
  const uint8_t* pool;
  int64_t out_stride, q_stride, num_blocks, bt_stride;
  const int32_t *tables, *row_index, *ctx;
  int batch, NH, KVH, group, max_blocks;
  float scale;
};

// The HD/32 dims lane `lane` holds of one token's codes (a 32-bit word serves 256 / HD lanes).
template <int HD>
__device__ __forceinline__ void lane_values(const uint8_t* row, int lane, float s,
                                            float (&f)[HD / 32]) {
  constexpr int PL = HD / 64;                      // bytes (dim pairs) of a lane
  uint32_t h[4];
  codes_to_half2(*reinterpret_cast<const uint32_t*>(row + ((lane * PL) & ~3)), h);
#pragma unroll
  for (int u = 0; u < PL; ++u) {
    const int j = (lane * PL + u) & 3;
    const float2 v = Elem<__half>::unpack2(j == 0 ? h[0] : j == 1 ? h[1] : j == 2 ? h[2] : h[3]);
    f[2 * u] = v.x * s;
    f[2 * u + 1] = v.y * s;
  }
}

// One CTA per (sequence, query head); warps take every 4th token, lanes HD/32 dims each.
template <typename T, int HD>
__global__ void __launch_bounds__(128) decode_kernel(DecodeParams p) {
  pdl_wait();
  pdl_launch_dependents();
  using L = Tile<HD>;
  constexpr int PL = HD / 64;                      // bytes (dim pairs) of a lane
  const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = p.ctx[b];
  if (n <= 0) return;
  const int32_t* table = p.tables + (int64_t)(p.row_index ? p.row_index[b] : b) * p.bt_stride;
  const int kvh = h / p.group;
  const T* q = (const T*)p.q + b * p.q_stride + (int64_t)h * HD;
  float qf[2 * PL], o[2 * PL];
  for (int u = 0; u < 2 * PL; ++u) {
    qf[u] = Elem<T>::to_f(q[lane * 2 * PL + u]) * p.scale;
    o[u] = 0.f;
  }
  float m = -INFINITY;
  double l = 0.;                   // a long flat tail is many small terms beside a large one
  const int n_max = min((int64_t)n, (int64_t)p.max_blocks * kBlock);
  for (int i = warp; i < n_max; i += 4) {
    const int32_t blk = table[i / kBlock];
    if (blk < 0 || blk >= p.num_blocks) continue;
    const uint8_t* tile = p.pool + ((int64_t)blk * p.KVH + kvh) * L::kBytes;
    const int off = i % kBlock, g = lane * 2 * PL / kGroup;
    const float ks = scale_value(tile[L::kKs + g * kBlock + off]);
    const float vs = scale_value(tile[L::kVs + g * kBlock + off]);
    float s = 0.f, k[2 * PL], v[2 * PL];
    lane_values<HD>(tile + L::kK + off * L::kRow, lane, ks, k);
    lane_values<HD>(tile + L::kV + off * L::kRow, lane, vs, v);
    for (int u = 0; u < 2 * PL; ++u) s += qf[u] * k[u];
    s = warp_sum(s);
    const float m2 = fmaxf(m, s), ref = m2 == -INFINITY ? 0.f : m2;
    const float c = expf(m - ref), e = expf(s - ref);
    l = l * c + e;
    for (int u = 0; u < 2 * PL; ++u) o[u] = o[u] * c + e * v[u];
    m = m2;
  }
  __shared__ float sm[4], so[4][HD];
  __shared__ double sl[4];
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
  for (int u = 0; u < 2 * PL; ++u) so[warp][lane * 2 * PL + u] = o[u];
  __syncthreads();
  if (threadIdx.x >= HD) return;
  float mm = -INFINITY, oo = 0.f;
  double ll = 0.;
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm[w]);
  const float ref = mm == -INFINITY ? 0.f : mm;
  for (int w = 0; w < 4; ++w) {
    const float c = expf(sm[w] - ref);
    ll += sl[w] * c;
    oo += so[w][threadIdx.x] * c;
  }
  ((T*)p.out)[b * p.out_stride + (int64_t)h * HD + threadIdx.x] = Elem<T>::from_f(oo / (float)ll);
  if (p.lse && threadIdx.x == 0) p.lse[(int64_t)b * p.NH + h] = ref + logf((float)ll);
}

struct WeightParams {
  float* out;
  const float* in;
  const void* q;
  const float* lse;
  const uint8_t* pool;
  int64_t q_stride, num_blocks, bt_stride;
  const int32_t *tables, *row_index, *ctx;
  int batch, NH, KVH, group, max_blocks;
  float scale;
};

// One warp per (sequence, kv head, token): the weights of the group's heads, summed in head order.
template <typename T, int HD>
__global__ void __launch_bounds__(256) weights_kernel(WeightParams p) {
  pdl_wait();
  pdl_launch_dependents();
  using L = Tile<HD>;
  constexpr int PL = HD / 64;
  const int kvh = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
  const int n = (int)min((int64_t)p.ctx[b], (int64_t)p.max_blocks * kBlock);
  const int32_t* table = p.tables + (int64_t)(p.row_index ? p.row_index[b] : b) * p.bt_stride;
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += gridDim.x * 8) {
    const int32_t blk = table[i / kBlock];
    if (blk < 0 || blk >= p.num_blocks) continue;
    const int64_t tile_i = (int64_t)blk * p.KVH + kvh;
    const uint8_t* tile = p.pool + tile_i * L::kBytes;
    const int off = i % kBlock, g = lane * 2 * PL / kGroup;
    const float ks = scale_value(tile[L::kKs + g * kBlock + off]);
    float k[2 * PL];
    lane_values<HD>(tile + L::kK + off * L::kRow, lane, ks, k);
    float w = 0.f;
    for (int hg = 0; hg < p.group; ++hg) {
      const int h = kvh * p.group + hg;
      const T* q = (const T*)p.q + b * p.q_stride + (int64_t)h * HD + lane * 2 * PL;
      float s = 0.f;
      for (int u = 0; u < 2 * PL; ++u) s += Elem<T>::to_f(q[u]) * k[u];
      w += expf(warp_sum(s) * p.scale - p.lse[(int64_t)b * p.NH + h]);
    }
    if (lane == 0) p.out[tile_i * kBlock + off] = p.in[tile_i * kBlock + off] + w;
  }
}

static int check_shape(const char* what, int batch, int NH, int KVH, int HD, int block_size,
                       int max_blocks, int64_t num_blocks, int dtype) {
  (void)what;
  if (batch < 0 || max_blocks <= 0 || num_blocks <= 0 || KVH <= 0 || NH <= 0 || NH % KVH)
    return set_error(TI_ERR_INVALID_ARGUMENT,
                     "kv4: bad batch, table width, pool size or head counts (num_heads must be a multiple of num_kv_heads)");
  if (HD != 64 && HD != 128) return set_error(TI_ERR_UNSUPPORTED, "kv4: head_dim must be 64 or 128");
  if (block_size != kBlock) return set_error(TI_ERR_UNSUPPORTED, "kv4: block_size must be 16");
  if (NH / KVH > 16) return set_error(TI_ERR_UNSUPPORTED, "kv4: at most 16 query heads per kv head");
  if (dtype != TI_DTYPE_BF16 && dtype != TI_DTYPE_FP16)
    return set_error(TI_ERR_UNSUPPORTED, "kv4: dtype must be bf16 or fp16");
  if (batch > 4096) return set_error(TI_ERR_UNSUPPORTED, "kv4: at most 4096 sequences per call");
  return TI_OK;
}

}  // namespace kv4
}  // namespace ti

using namespace ti;

extern "C" size_t ti_kv4_attention_workspace_bytes(int batch, int num_heads, int num_kv_heads,
                                                   int head_dim, int max_blocks_per_seq) {
  (void)batch; (void)num_heads; (void)num_kv_heads; (void)head_dim; (void)max_blocks_per_seq;
  return 16;
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
  if (!out || !q || !pool || !block_tables || !context_lens)
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4 attention: null pointer");
  if (int rc = kv4::check_shape("kv4 attention", batch, num_heads, num_kv_heads, head_dim,
                                block_size, max_blocks_per_seq, num_blocks, dtype))
    return rc;
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) |
        reinterpret_cast<uintptr_t>(pool)) & 15) || (out_seq_stride % 8) || (q_seq_stride % 8))
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4 attention: tensors must be 16-byte aligned");
  (void)workspace; (void)workspace_bytes;
  kv4::DecodeParams p{out, lse, q, (const uint8_t*)pool, out_seq_stride, q_seq_stride, num_blocks,
                      bt_stride, block_tables, row_index, context_lens, batch, num_heads,
                      num_kv_heads, num_heads / num_kv_heads, max_blocks_per_seq,
                      1.0f / sqrtf((float)head_dim)};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) {
    return launch_kernel("kv4 attention launch", kern, dim3(num_heads, batch), dim3(128), 0, s, 1, p);
  };
  if (dtype == TI_DTYPE_BF16)
    return head_dim == 64 ? go(kv4::decode_kernel<__nv_bfloat16, 64>)
                          : go(kv4::decode_kernel<__nv_bfloat16, 128>);
  return head_dim == 64 ? go(kv4::decode_kernel<__half, 64>) : go(kv4::decode_kernel<__half, 128>);
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
  if (int rc = kv4::check_shape("kv4 weights", batch, num_heads, num_kv_heads, head_dim,
                                block_size, max_blocks_per_seq, num_blocks, dtype))
    return rc;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pool)) & 15) ||
      (q_seq_stride % 8))
    return set_error(TI_ERR_INVALID_ARGUMENT, "kv4 weights: tensors must be 16-byte aligned");
  kv4::WeightParams p{weights_out, weights, q, lse, (const uint8_t*)pool, q_seq_stride, num_blocks,
                      bt_stride, block_tables, row_index, context_lens, batch, num_heads,
                      num_kv_heads, num_heads / num_kv_heads, max_blocks_per_seq,
                      1.0f / sqrtf((float)head_dim)};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(std::min(max_blocks_per_seq, 64), num_kv_heads, batch);
  auto go = [&](auto kern) {
    return launch_kernel("kv4 weights launch", kern, grid, dim3(256), 0, s, 1, p);
  };
  if (dtype == TI_DTYPE_BF16)
    return head_dim == 64 ? go(kv4::weights_kernel<__nv_bfloat16, 64>)
                          : go(kv4::weights_kernel<__nv_bfloat16, 128>);
  return head_dim == 64 ? go(kv4::weights_kernel<__half, 64>)
                        : go(kv4::weights_kernel<__half, 128>);
}
