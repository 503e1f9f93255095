// Attention of drafted trees over the paged 16-bit pool.
//
// Sequence i's nodes are query rows cu[i] .. cu[i+1]-1; their K and V are in the pool at positions
// ctx[i] .. of the sequence's table row, behind its ctx[i] cached tokens.  A node attends to every cached
// token and to the nodes whose bits its mask row has (no masks: to the nodes up to itself).
//
// First form: one warp per (node, query head), a lane per key for the scores, a lane per D / 32 dims for
// the values.
#include <algorithm>

#include "capi_internal.h"
#include "common.cuh"

namespace ti {
namespace tree {

constexpr int kBlock = 16;
constexpr int kMaxGroup = 16;

struct Params {
  void* out;
  const void *q, *k, *v;
  float* lse;
  int64_t out_stride, q_stride, num_blocks, bt_stride;
  const int32_t *tables, *row_index, *ctx, *cu, *masks;
  int seqs, tokens, rows, cols, NH, KVH, group, mask_words;
  float scale_log2;
};

template <typename T, int HD>
__global__ void simple_kernel(const __grid_constant__ Params p) {
  __shared__ float s_q[kMaxGroup][HD];
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (t >= p.cu[p.seqs] || t < p.cu[0]) return;
  int lo = 0, hi = p.seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  const int i = lo, node = t - p.cu[i], nodes = p.cu[i + 1] - p.cu[i], ctx = max(p.ctx[i], 0);
  const int row = p.row_index ? p.row_index[i] : i, h = kvh * p.group + warp;
  const bool known = row >= 0 && row < p.rows;
  const T* q = (const T*)p.q + (int64_t)t * p.q_stride + (int64_t)h * HD;
  for (int d = lane; d < HD; d += 32) s_q[warp][d] = Elem<T>::to_f(q[d]);
  __syncwarp();
  constexpr int kD = HD / 32;
  float m = -INFINITY, l = 0.f, o[kD];
#pragma unroll
  for (int d = 0; d < kD; ++d) o[d] = 0.f;
  const int n = known ? (int)min((int64_t)ctx + nodes, (int64_t)p.cols * kBlock) : 0;
  for (int k0 = 0; k0 < n; k0 += 32) {
    const int key = k0 + lane;
    int64_t at = -1;
    if (key < n) {
      const int b = p.tables[(int64_t)row * p.bt_stride + key / kBlock], x = key - ctx;
      bool see = b >= 0 && b < p.num_blocks;
      if (x >= 0) {
        if (p.masks) see = see && x < 32 * p.mask_words &&
                           ((p.masks[(int64_t)t * p.mask_words + x / 32] >> (x & 31)) & 1);
        else see = see && x <= node;
      }
      if (see) at = (((int64_t)b * p.KVH + kvh) * kBlock + key % kBlock) * HD;
    }
    float s = -INFINITY;
    if (at >= 0) {
      s = 0.f;
      const T* k = (const T*)p.k + at;
      for (int d = 0; d < HD; ++d) s += s_q[warp][d] * Elem<T>::to_f(k[d]);
      s *= p.scale_log2;
    }
    const float mn = fmaxf(m, warp_max(s));
    const bool any_nan = __any_sync(0xffffffffu, s != s);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = m == -INFINITY ? 0.f : exp2f(m - base), w = any_nan && s != s ? s : exp2f(s - base);
    m = mn;
    l = l * f + w;
#pragma unroll
    for (int d = 0; d < kD; ++d) o[d] *= f;
    for (int e = 0; e < 32; ++e) {
      const int64_t a = __shfl_sync(0xffffffffu, at, e);
      const float pe = __shfl_sync(0xffffffffu, w, e);
      if (a < 0) continue;
#pragma unroll
      for (int d = 0; d < kD; ++d) o[d] += pe * Elem<T>::to_f(((const T*)p.v)[a + lane + 32 * d]);
    }
  }
  l = warp_sum(l);
  T* dst = (T*)p.out + (int64_t)t * p.out_stride + (int64_t)h * HD;
  const bool none = m == -INFINITY && !(l != l);
#pragma unroll
  for (int d = 0; d < kD; ++d) dst[lane + 32 * d] = Elem<T>::from_f(none ? 0.f : o[d] / l);
  if (p.lse && lane == 0) p.lse[(int64_t)t * p.NH + h] = none ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace tree
}  // namespace ti

using namespace ti;

extern "C" size_t ti_tree_attention_workspace_bytes(int num_heads, int num_kv_heads, int head_dim) {
  (void)num_heads;
  (void)num_kv_heads;
  (void)head_dim;
  return 16;
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
  tree::Params p{out, q, k_cache, v_cache, lse, out_tok_stride, q_tok_stride, num_blocks, bt_stride,
                 block_tables, row_index, context_lens, cu_seqlens, mask_words ? masks : nullptr, num_seqs,
                 num_tokens, num_rows, max_blocks_per_seq, num_heads, num_kv_heads, group, mask_words,
                 1.4426950408889634f / sqrtf((float)head_dim)};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)num_tokens, (unsigned)num_kv_heads), block(32 * group);
#define TREE_GO(T, D) launch_kernel("tree attention launch", tree::simple_kernel<T, D>, grid, block, 0, s, 1, p)
  if (dtype == TI_DTYPE_BF16) return head_dim == 64 ? TREE_GO(__nv_bfloat16, 64) : TREE_GO(__nv_bfloat16, 128);
  return head_dim == 64 ? TREE_GO(__half, 64) : TREE_GO(__half, 128);
#undef TREE_GO
}
