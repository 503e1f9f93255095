// Acceptance of drafted tokens.  Node 0 of a tree is the sequence's last token, every other node a guess
// for the token behind its parent; targets[c] is the token drawn at node c.  The walk starts at node 0
// and goes to the first child (the lowest index) that holds the token drawn at the current node, until
// there is none: the nodes passed are the sequence's next cached tokens, the draws at them the tokens it
// emits.  K and V of the path's j-th node move to the slot of place j, in every layer.
//
// One launch: each CTA of a sequence walks its tree (a warp looks at 32 nodes at once; a few hundred
// nanoseconds in shared memory) and moves its share of layers and heads.  A thread moves 16 bytes of
// one (layer, K or V, head) for all places of the path, in ascending order, four loads ahead of their
// stores.  In place this is safe: path[j] >= j, so the slot of place j, which is node j's, is read for no
// place behind j.
//
// Bound: HBM, each kept byte read and written once.  256 trees of up to 64 nodes (24 layers, 8 heads of 128, 4.0
// nodes kept on average: 202 MB) take 41 us, 4.9 TB/s or 0.75 of measured copy: the rows are 256 bytes long and
// lie 4 KB apart.  Four loads ahead in 32 registers, so that 8 CTAs fit an SM, and three rounds of them:
// 47 us with eight loads, 5 CTAs an SM and one and a half rounds.  8 trees of 8 nodes take 4.3 us in a graph and 16 as
// a call: the host.
#include <algorithm>

#include "capi_internal.h"
#include "common.cuh"

namespace ti {
namespace accept {

constexpr int kThreads = 256;
constexpr int kStage = 512;              // nodes of a tree held in shared memory; more are read in place
constexpr int kAhead = 4;

struct Params {
  uint4 *kc, *vc;
  const int32_t *tokens, *parents, *targets, *cu;
  const int64_t *slots, *out_slots;
  int32_t *num, *path, *out_tokens, *seq_lens;
  const int32_t* row_index;
  int64_t num_slots, layer_units;              // pool slots, 16-byte units of a layer
  unsigned per_layer, items;                   // units of a token's K in a layer, of its K and V in all
  int deep, rows, block, kvh, units, layers, total;
};

__global__ void __launch_bounds__(kThreads, 8) accept_kernel(const __grid_constant__ Params p) {
  extern __shared__ int64_t s_move[];            // source and target unit of each place
  __shared__ int s_parent[kStage], s_token[kStage], s_target[kStage];
  __shared__ int s_num;
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int first = max(p.cu[seq], 0), n = min(p.cu[seq + 1], p.total) - first;
  const bool staged = n <= kStage;
  if (staged)
    for (int i = tid; i < n; i += kThreads) {
      s_parent[i] = p.parents[first + i];
      s_token[i] = p.tokens[first + i];
      s_target[i] = p.targets[first + i];
    }
  __syncthreads();
  int32_t* s_path = reinterpret_cast<int32_t*>(s_move + 2 * p.deep);
  if (tid < 32) {
    int count = 0;
    // lengths count cached tokens: where they are kept here, a tree whose first node or place has no slot was
    // not run (a sequence's new tokens have slots all or none), so it emits nothing
    const bool run = n > 0 && !(p.seq_lens && (p.slots[first] < 0 || p.out_slots[first] < 0));
    if (run) {
      const int32_t* parent = staged ? s_parent : p.parents + first;
      const int32_t* token = staged ? s_token : p.tokens + first;
      const int32_t* target = staged ? s_target : p.targets + first;
      int cur = 0;
      while (count < p.deep) {
        const int drawn = target[cur];
        if (lane == 0) {
          s_path[count] = cur;
          if (blockIdx.y == 0) p.out_tokens[(int64_t)seq * p.deep + count] = drawn;
        }
        ++count;
        int next = -1;
        for (int c0 = cur + 1; c0 < n && next < 0; c0 += 32) {
          const int c = c0 + lane;
          const uint32_t hit = __ballot_sync(0xffffffffu, c < n && parent[c] == cur && token[c] == drawn);
          if (hit) next = c0 + __ffs(hit) - 1;
        }
        if (next < 0) break;
        cur = next;
      }
    }
    if (lane == 0) {
      s_num = count;
      if (blockIdx.y == 0) {
        p.num[seq] = count;
        const int row = p.row_index ? p.row_index[seq] : seq;
        if (p.seq_lens && row >= 0 && row < p.rows && count) atomicAdd(p.seq_lens + row, count);
      }
    }
  }
  __syncthreads();
  const int count = s_num;
  if (blockIdx.y == 0)
    for (int j = tid; j < p.deep; j += kThreads) {
      p.path[(int64_t)seq * p.deep + j] = j < count ? s_path[j] : -1;
      if (j >= count) p.out_tokens[(int64_t)seq * p.deep + j] = -1;
    }
  bool bad = false;
  for (int j = tid; j < count; j += kThreads) {
    const int64_t from = p.slots[first + s_path[j]], to = p.out_slots[first + j];
    bad |= from >= p.num_slots || to >= p.num_slots;
    const bool ok = from >= 0 && from < p.num_slots && to >= 0 && to < p.num_slots && from != to;
    auto unit = [&](int64_t s) { return (s / p.block * p.kvh * p.block + s % p.block) * (int64_t)p.units; };
    s_move[2 * j] = ok ? unit(from) : -1;
    s_move[2 * j + 1] = ok ? unit(to) : -1;
  }
  if (bad) raise_device_error(TI_DEVERR_BAD_INPUT);
  __syncthreads();
  // an item: 16 bytes of K or V of one head of one layer
  const unsigned units = (unsigned)p.units;
  for (unsigned e = blockIdx.y * kThreads + tid; e < p.items; e += gridDim.y * kThreads) {
    const unsigned lkv = e / p.per_layer, in = e - lkv * p.per_layer, head = in / units;
    uint4* base = ((lkv & 1) ? p.vc : p.kc) + (int64_t)(lkv >> 1) * p.layer_units +
                  (int64_t)head * (p.block * units) + (in - head * units);
    for (int j0 = 0; j0 < count; j0 += kAhead) {
      uint4 v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (j0 + k < count && s_move[2 * (j0 + k)] >= 0) v[k] = base[s_move[2 * (j0 + k)]];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (j0 + k < count && s_move[2 * (j0 + k)] >= 0) base[s_move[2 * (j0 + k) + 1]] = v[k];
    }
  }
}

}  // namespace accept
}  // namespace ti

using namespace ti;

extern "C" int ti_tree_accept(void* key_cache, void* value_cache, int num_layers, int64_t num_blocks,
                              int num_kv_heads, int head_dim, int block_size, int elem_bytes,
                              const int32_t* tokens, const int32_t* parents, const int32_t* targets,
                              const int32_t* cu_seqlens, int num_seqs, int num_tokens,
                              const int64_t* slot_mapping, const int64_t* out_slots, int32_t* num,
                              int32_t* path, int32_t* out_tokens, int max_path, int32_t* seq_lens,
                              const int32_t* row_index, int num_rows, void* stream) {
  clear_error();
  if (num_seqs == 0) return TI_OK;
  if (!key_cache || !value_cache || !cu_seqlens || !num || !path || !out_tokens || num_seqs < 0 ||
      num_tokens < 0 || (num_tokens > 0 && (!tokens || !parents || !targets || !slot_mapping || !out_slots)))
    return set_error(TI_ERR_INVALID_ARGUMENT, "tree accept: null pointer or bad size");
  if (num_layers <= 0 || num_blocks <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
      elem_bytes <= 0 || max_path <= 0 || (seq_lens && num_rows <= 0))
    return set_error(TI_ERR_INVALID_ARGUMENT, "tree accept: bad size");
  if (((int64_t)head_dim * elem_bytes) % 16 ||
      ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache)) & 15))
    return set_error(TI_ERR_INVALID_ARGUMENT, "tree accept: cache rows must be 16-byte aligned");
  if (max_path > 1024) return set_error(TI_ERR_UNSUPPORTED, "tree accept: at most 1024 places in a path");
  accept::Params p{};
  p.kc = (uint4*)key_cache;
  p.vc = (uint4*)value_cache;
  p.tokens = tokens;
  p.parents = parents;
  p.targets = targets;
  p.cu = cu_seqlens;
  p.slots = slot_mapping;
  p.out_slots = out_slots;
  p.num = num;
  p.path = path;
  p.out_tokens = out_tokens;
  p.seq_lens = seq_lens;
  p.row_index = row_index;
  p.units = (int)((int64_t)head_dim * elem_bytes / 16);
  p.num_slots = num_blocks * block_size;
  // (32 bits: 64-bit divisions, two an item, took 48.6 us where these take 47.3)
  const double row = (double)head_dim * elem_bytes / 16;
  if (2.0 * num_layers * num_kv_heads * row > 0x3fffffff || block_size * row > 0x3fffffff)
    return set_error(TI_ERR_UNSUPPORTED, "tree accept: a token's K and V have more than 2^30 16-byte units");
  p.per_layer = (unsigned)num_kv_heads * (unsigned)p.units;
  const int64_t items = (int64_t)num_layers * 2 * p.per_layer;
  p.items = (unsigned)items;
  p.layer_units = num_blocks * block_size * (int64_t)p.per_layer;
  p.deep = max_path;
  p.rows = num_rows;
  p.block = block_size;
  p.kvh = num_kv_heads;
  p.layers = num_layers;
  p.total = num_tokens;
  // a CTA walks its tree again: as few as still fill the GPU
  const int64_t want = std::max<int64_t>(1, (148 * 24 + num_seqs - 1) / num_seqs);
  const unsigned y = (unsigned)std::min<int64_t>(std::min<int64_t>((items + accept::kThreads - 1) / accept::kThreads, want), 65535);
  return launch_kernel_cl("tree accept launch", accept::accept_kernel, dim3((unsigned)num_seqs, y),
                          dim3(accept::kThreads), (size_t)max_path * 20, reinterpret_cast<cudaStream_t>(stream),
                          dim3(1), p);
}
