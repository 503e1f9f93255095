// Block tables and slots built on the device.  The free list is a ring: ring[0] the place of its first
// entry, ring[1] how many it has, ring[2 ..] the block ids.  Blocks leave at the front and come back at
// the end, in the order in which the host's allocator would hand them out.
//
// reserve: sequence i gets counts[i] new tokens behind its lens[row] cached ones.  It needs a block for
// every table entry of their range that is unassigned; with c_i the sum of the needs up to and including
// i, it is served when it needs none or c_i <= ring[1] (the first one that does not fit ends the list).
// release: the blocks behind ceil(keep / block) of each row go to the ring's end, row by row.
//
// One cluster does either: a warp counts a sequence's entries, the counts go to every CTA's shared
// memory, each CTA sums them up itself, and the warp that counted a row writes it, so rows wait for one
// barrier only.  Tokens follow in the same launch, or, above kFusedTokens, in a second one over the
// whole GPU (one cluster alone writes too slowly: 64 prompts of up to 16384 tokens took 44 us).
//
// Bound: latency, dependent trips to memory.  One token for each of 256 sequences takes 7.3 us on the device,
// trees of up to 64 nodes for 64 sequences 10.0; as calls 17 and 18, of which the host is 10.  The 64 prompts
// (655000 tokens, 8 MB of slots and positions) take 24.5 us as a call: two launches, the second
// bound by its writes and by one division or shift and one table load a token.
#include <algorithm>
#include <atomic>

#include "capi_internal.h"
#include "common.cuh"

namespace ti {
namespace paging {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kCluster = 8;
constexpr int kMaxSeqs = 4096;
constexpr int kMaxRows = 32768;          // with row_index: a word of shared memory each
constexpr int64_t kFusedTokens = 65536;
constexpr int kExpand = 256;             // threads of the second launch
constexpr int kAhead = 8;                // table columns (times 32) that a warp has in flight
constexpr int kTokens = 4;               // neighbouring tokens of a thread, in the second launch

struct Params {
  int32_t *tables, *ring;
  int64_t bt_stride;
  const int32_t *row_index, *lens, *counts, *pos_offset, *parents;
  int64_t* slots;
  int32_t *positions, *cu, *granted, *masks;
  int64_t capacity, ring_size;
  int seqs, rows, cols, block, shift, mask_words, fused;   // shift: log2 of the block size, or -1
};

__device__ __forceinline__ int64_t block_of(const Params& p, int64_t pos) {
  return p.shift >= 0 ? pos >> p.shift : pos / p.block;
}

// Dynamic shared memory: needs [seqs], their sums [seqs], token offsets [seqs + 1], owners [rows] (with
// row_index).
static size_t smem_bytes(int seqs, int rows, bool indexed) {
  return ((size_t)3 * seqs + 1 + (indexed ? rows : 0)) * 4;
}

__device__ __forceinline__ void st_peer_i32(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}

// Exclusive sums of v[0 .. n), in place, held at 2^31 - 1 where they would pass it (every thread of the
// block calls it); returns the total, held likewise.
__device__ int exclusive_sums(int* v, int n, long long* warp_sums) {
  constexpr long long kMost = 0x7FFFFFFF;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long base = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + threadIdx.x, own = i < n ? v[i] : 0;
    long long s = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    long long w = warp_sums[lane];                // (32 warps: every warp sums them up)
    const long long mine = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    const long long before = __shfl_sync(0xffffffffu, w - mine, warp);
    const long long total = __shfl_sync(0xffffffffu, w, 31);
    if (i < n) v[i] = (int)min(base + before + s - own, kMost);
    base += total;
    __syncthreads();
  }
  return (int)min(base, kMost);
}

// One place of the token buffers: its sequence by binary search in the offsets, its block's entry, and,
// for a tree, the way up to its root.
__device__ __forceinline__ void expand(const Params& p, const int* s_cu, int64_t t) {
  int64_t slot = -1, pos = 0;
  int first = 0, j = -1;
  if (t < s_cu[p.seqs]) {
    int lo = 0, hi = p.seqs - 1;                  // the last i with cu[i] <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_cu[mid] <= t) lo = mid; else hi = mid - 1;
    }
    first = s_cu[lo];
    j = (int)(t - first);
    const int row = p.row_index ? p.row_index[lo] : lo;
    pos = j;                                      // (a row that does not exist: length 0)
    if (row >= 0 && row < p.rows) {
      const int len = p.lens[row];
      pos = (int64_t)len + (p.pos_offset ? p.pos_offset[row] : 0) + j;
      if (__ldcg(p.granted + lo) > 0) {
        const int at = len + j, col = (int)block_of(p, at);      // (granted: within the row)
        const int b = __ldcg(p.tables + (int64_t)row * p.bt_stride + col);
        if (b >= 0) slot = (int64_t)b * p.block + (at - col * p.block);
      }
    }
  }
  if (p.parents) {
    // parents come before their children; one that does not ends the way up
    int depth = 0;
    bool bad = false;
    for (int w0 = 0; w0 == 0 || w0 < p.mask_words; w0 += 4) {
      uint32_t m[4] = {0, 0, 0, 0};
      depth = 0;
      for (int a = j; a >= 0;) {
        ++depth;
        const int w = (a >> 5) - w0;
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] |= w == k ? 1u << (a & 31) : 0u;
        bad |= p.mask_words > 0 && a >= 32 * p.mask_words;
        const int up = p.parents[first + a];
        bad |= up >= a;
        a = up >= a ? -1 : up;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (w0 + k < p.mask_words) p.masks[t * p.mask_words + w0 + k] = (int32_t)m[k];
    }
    if (j >= 0) pos += depth - 1 - j;
    if (bad) raise_device_error(TI_DEVERR_BAD_INPUT);
  }
  p.slots[t] = slot;
  p.positions[t] = (int32_t)pos;
}

__global__ void __launch_bounds__(kThreads, 1) reserve_kernel(const __grid_constant__ Params p) {
  extern __shared__ int s_dyn[];
  __shared__ long long warp_sums[32];
  __shared__ int s_stop;
  int* s_raw = s_dyn;                             // blocks each sequence needs (negative: not to be served)
  int* s_need = s_raw + p.seqs;                   // the sums before it
  int* s_cu = s_need + p.seqs;
  int* s_owner = s_cu + p.seqs + 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ctas = cluster_size(), rank = ctas > 1 ? cluster_rank() : 0;
  if (ctas > 1) cluster_arrive_relaxed();         // (waited for before a peer's memory is written)
  pdl_wait();
  pdl_launch_dependents();
  if (tid == 0) s_stop = p.seqs;
  // a row that several sequences name belongs to the first of them
  if (p.row_index) {
    for (int r = tid; r < p.rows; r += kThreads) s_owner[r] = 0x7FFFFFFF;
    __syncthreads();
    for (int i = tid; i < p.seqs; i += kThreads) {
      const int row = p.row_index[i];
      if (row >= 0 && row < p.rows) atomicMin(&s_owner[row], i);
    }
  }
  bool negative = false;
  for (int i = tid; i < p.seqs; i += kThreads) {
    const int n = p.counts[i];
    negative |= n < 0;
    s_cu[i] = max(n, 0);
  }
  __syncthreads();

  // ---- needs: a warp per sequence
  auto whole_row = [&](int i, int& row, int& n, int& len) {
    row = p.row_index ? p.row_index[i] : i;
    n = s_cu[i];
    if (row < 0 || row >= p.rows) return false;
    len = p.lens[row];
    return (!p.row_index || s_owner[row] == i) && len >= 0 && n >= 0 &&
           (int64_t)len + n <= (int64_t)p.cols * p.block;
  };
  bool bad = negative;
  if (ctas > 1) cluster_wait_acquire();
  for (int i = warp * (int)ctas + (int)rank; i < p.seqs; i += kWarps * (int)ctas) {
    int row, n, len = 0, need = 0;
    const bool ok = whole_row(i, row, n, len);
    if (ok && n > 0) {
      const int32_t* t = p.tables + (int64_t)row * p.bt_stride;
      const int last = (int)block_of(p, len + n - 1);
      for (int c0 = (int)block_of(p, len); c0 <= last; c0 += 32 * kAhead) {
        int id[kAhead];                            // (kAhead loads in flight)
#pragma unroll
        for (int a = 0; a < kAhead; ++a) id[a] = c0 + 32 * a + lane <= last ? __ldcg(t + c0 + 32 * a + lane) : 0;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) need += __popc(__ballot_sync(0xffffffffu, id[a] < 0));
      }
    }
    bad |= !ok && row >= 0 && n > 0;              // (a negative row is padding)
    // (the top bit: not to be served; it stays out of the sums)
    const int word = ok ? need : (int)0x80000000;
    for (uint32_t c = lane; c < ctas; c += 32)
      st_peer_i32(map_peer(smem_u32(s_raw + i), c), word);
  }
  if (bad && lane == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
  int head = p.ring[0], have = p.ring[1];
  const bool ring_ok = head >= 0 && head < p.ring_size && have >= 0 && have <= p.ring_size;
  if (!ring_ok) {
    head = have = 0;
    if (tid == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
  }
  if (ctas > 1) cluster_sync(); else __syncthreads();

  // ---- sums, by every CTA for itself
  for (int i = tid; i < p.seqs; i += kThreads) s_need[i] = max(s_raw[i], 0);
  __syncthreads();
  const int total = exclusive_sums(s_need, p.seqs, warp_sums);
  const int tokens = exclusive_sums(s_cu, p.seqs, warp_sums);
  if (tid == 0) s_cu[p.seqs] = tokens;
  for (int i = tid; i < p.seqs; i += kThreads)
    if (s_raw[i] > 0 && (long long)s_need[i] + s_raw[i] > have) atomicMin(&s_stop, i);
  __syncthreads();
  const int stop = s_stop;                        // the first sequence that does not fit
  if (rank == 0)
    for (int i = tid; i < p.seqs; i += kThreads) {
      const bool served = s_raw[i] == 0 || (s_raw[i] > 0 && i < stop);
      p.granted[i] = served ? s_cu[i + 1] - s_cu[i] : 0;
      p.cu[i] = s_cu[i];
    }
  // ---- the rows that are served
  for (int i = warp * (int)ctas + (int)rank; i < stop; i += kWarps * (int)ctas) {
    if (s_raw[i] <= 0) continue;
    const int base = s_need[i], next = base + s_raw[i];
    const int row = p.row_index ? p.row_index[i] : i, len = p.lens[row];
    const int n = s_cu[i + 1] - s_cu[i], last = (int)block_of(p, len + n - 1);
    int32_t* t = p.tables + (int64_t)row * p.bt_stride;
    int taken = base;
    for (int c0 = (int)block_of(p, len); c0 <= last && taken < next; c0 += 32 * kAhead) {
      int id[kAhead], from[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) id[a] = c0 + 32 * a + lane <= last ? __ldcg(t + c0 + 32 * a + lane) : 0;
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const uint32_t all = __ballot_sync(0xffffffffu, id[a] < 0);
        int64_t at = (int64_t)head + taken + __popc(all & ((1u << lane) - 1));
        if (at >= p.ring_size) at -= p.ring_size;
        from[a] = id[a] < 0 ? (int)at : -1;
        taken += __popc(all);
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) id[a] = from[a] >= 0 ? p.ring[2 + from[a]] : 0;
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        if (from[a] >= 0) __stcg(t + c0 + 32 * a + lane, id[a]);
    }
  }
  if (rank == 0 && tid == 0) {
    p.cu[p.seqs] = tokens;
    if (tokens > p.capacity) raise_device_error(TI_DEVERR_BAD_INPUT);
  }
  // every CTA has read the ring's state, and the rows are written
  __threadfence();
  if (ctas > 1) cluster_sync(); else __syncthreads();
  if (rank == 0 && tid == 0 && ring_ok) {
    const int used = stop < p.seqs ? s_need[stop] : total;
    const int64_t at = (int64_t)head + used;
    p.ring[0] = (int32_t)(at >= p.ring_size ? at - p.ring_size : at);
    p.ring[1] = have - used;
  }
  if (!p.fused) return;
  for (int64_t t = (int64_t)rank * kThreads + tid; t < p.capacity; t += (int64_t)ctas * kThreads)
    expand(p, s_cu, t);
}

// Four neighbouring tokens of one sequence, whose entry is looked up where the block changes; anything else
// (the end of a sequence among them, trees) token by token.
__device__ __forceinline__ void expand_run(const Params& p, const int* s_cu, int64_t t) {
  int lo = 0, hi = p.seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_cu[mid] <= t) lo = mid; else hi = mid - 1;
  }
  const int row = p.seqs == 0 ? -1 : p.row_index ? p.row_index[lo] : lo;
  if (p.parents || t + kTokens > p.capacity || row < 0 || row >= p.rows || t + kTokens > s_cu[lo + 1] ||
      __ldcg(p.granted + lo) == 0) {
    for (int64_t i = t; i < min(t + kTokens, p.capacity); ++i) expand(p, s_cu, i);
    return;
  }
  const int at = p.lens[row] + (int)(t - s_cu[lo]), pos = at + (p.pos_offset ? p.pos_offset[row] : 0);
  const int32_t* table = p.tables + (int64_t)row * p.bt_stride;
  int col = (int)block_of(p, at), off = at - col * p.block, b = __ldcg(table + col);
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    if (off == p.block) {
      off = 0;
      b = __ldcg(table + ++col);
    }
    p.slots[t + i] = b >= 0 ? (int64_t)b * p.block + off : -1;
    p.positions[t + i] = pos + i;
    ++off;
  }
}

__global__ void __launch_bounds__(kExpand) expand_kernel(const __grid_constant__ Params p) {
  extern __shared__ int s_cu_dyn[];
  pdl_wait();
  pdl_launch_dependents();
  for (int i = threadIdx.x; i <= p.seqs; i += kExpand) s_cu_dyn[i] = p.cu[i];
  __syncthreads();
  for (int64_t t = ((int64_t)blockIdx.x * kExpand + threadIdx.x) * kTokens; t < p.capacity;
       t += (int64_t)gridDim.x * kExpand * kTokens)
    expand_run(p, s_cu_dyn, t);
}

// p.counts: the tokens that each row keeps.
__global__ void __launch_bounds__(kThreads, 1) release_kernel(const __grid_constant__ Params p) {
  extern __shared__ int s_dyn[];
  __shared__ long long warp_sums[32];
  int* s_free = s_dyn;
  int* s_owner = s_dyn + p.seqs;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ctas = cluster_size(), rank = ctas > 1 ? cluster_rank() : 0;
  if (ctas > 1) cluster_arrive_relaxed();         // (waited for before a peer's memory is written)
  pdl_wait();
  pdl_launch_dependents();
  if (p.row_index) {
    for (int r = tid; r < p.rows; r += kThreads) s_owner[r] = 0x7FFFFFFF;
    __syncthreads();
    for (int i = tid; i < p.seqs; i += kThreads) {
      const int row = p.row_index[i];
      if (row >= 0 && row < p.rows) atomicMin(&s_owner[row], i);
    }
    __syncthreads();
  }
  bool bad = false;
  if (ctas > 1) cluster_wait_acquire();
  for (int i = warp * (int)ctas + (int)rank; i < p.seqs; i += kWarps * (int)ctas) {
    const int row = p.row_index ? p.row_index[i] : i;
    const bool ok = row >= 0 && row < p.rows && (!p.row_index || s_owner[row] == i) && p.counts[i] >= 0;
    int n = 0;
    if (ok) {
      const int32_t* t = p.tables + (int64_t)row * p.bt_stride;
      for (int64_t c0 = block_of(p, (int64_t)p.counts[i] + p.block - 1); c0 < p.cols; c0 += 32 * kAhead) {
        int id[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) id[a] = c0 + 32 * a + lane < p.cols ? __ldcg(t + c0 + 32 * a + lane) : -1;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) n += __popc(__ballot_sync(0xffffffffu, id[a] >= 0));
      }
    }
    bad |= !ok && row >= 0;
    for (uint32_t c = lane; c < ctas; c += 32) st_peer_i32(map_peer(smem_u32(s_free + i), c), n);
  }
  if (bad && lane == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
  const int head = p.ring[0], have = p.ring[1];
  const bool ring_ok = head >= 0 && head < p.ring_size && have >= 0 && have <= p.ring_size;
  if (ctas > 1) cluster_sync(); else __syncthreads();
  const int total = exclusive_sums(s_free, p.seqs, warp_sums);
  // blocks that the ring has no room for are not its own: nothing is changed then
  const bool fits = ring_ok && total <= p.ring_size - have;
  if (!fits && rank == 0 && tid == 0) raise_device_error(TI_DEVERR_BAD_INPUT);
  for (int i = warp * (int)ctas + (int)rank; fits && i < p.seqs; i += kWarps * (int)ctas) {
    const int base = s_free[i], next = i + 1 < p.seqs ? s_free[i + 1] : total;
    if (next == base) continue;
    const int row = p.row_index ? p.row_index[i] : i;
    int32_t* t = p.tables + (int64_t)row * p.bt_stride;
    int done = base;
    for (int64_t c0 = block_of(p, (int64_t)p.counts[i] + p.block - 1); c0 < p.cols && done < next; c0 += 32 * kAhead) {
      int id[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) id[a] = c0 + 32 * a + lane < p.cols ? __ldcg(t + c0 + 32 * a + lane) : -1;
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const uint32_t all = __ballot_sync(0xffffffffu, id[a] >= 0);
        if (id[a] >= 0) {
          int64_t at = (int64_t)head + have + done + __popc(all & ((1u << lane) - 1));
          while (at >= p.ring_size) at -= p.ring_size;
          p.ring[2 + at] = id[a];
          __stcg(t + c0 + 32 * a + lane, -1);
        }
        done += __popc(all);
      }
    }
  }
  if (ctas > 1) cluster_sync(); else __syncthreads();    // every CTA has read the ring's state
  if (fits && rank == 0 && tid == 0) p.ring[1] = have + total;
}

// The kernels' dynamic shared memory limit, raised once per device.
template <typename K>
static int raise_limit(K kern, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (ready.load(std::memory_order_acquire) & bit) return TI_OK;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)smem_bytes(kMaxSeqs, kMaxRows, true));
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return set_cuda_error(e, "cudaFuncSetAttribute(paging)");
  }
  ready.fetch_or(bit, std::memory_order_release);
  return TI_OK;
}

static int shift_of(int block) {
  if (block <= 0 || (block & (block - 1))) return -1;
  int s = 0;
  while ((1 << s) < block) ++s;
  return s;
}

static int check_sizes(const Params& p) {
  if (p.seqs < 0 || p.rows < 0 || p.cols <= 0 || p.block <= 0 || p.ring_size <= 0 || p.capacity < 0)
    return set_error(TI_ERR_INVALID_ARGUMENT, "paging: bad size");
  if (p.seqs > kMaxSeqs) return set_error(TI_ERR_UNSUPPORTED, "paging: at most 4096 sequences");
  if (p.row_index && p.rows > kMaxRows)
    return set_error(TI_ERR_UNSUPPORTED, "paging: at most 32768 table rows with row_index");
  if (!p.row_index && p.rows < p.seqs)
    return set_error(TI_ERR_INVALID_ARGUMENT, "paging: fewer table rows than sequences");
  if ((int64_t)p.cols * p.block >= (int64_t)1 << 31 || p.ring_size >= (int64_t)1 << 31 ||
      p.capacity >= (int64_t)1 << 31)
    return set_error(TI_ERR_UNSUPPORTED, "paging: sizes beyond 31 bits");
  return TI_OK;
}

}  // namespace paging
}  // namespace ti

using namespace ti;

extern "C" int ti_reserve_slots(int32_t* block_tables, int64_t bt_stride, int num_rows,
                                int max_blocks_per_seq, int block_size, const int32_t* row_index,
                                const int32_t* lens, const int32_t* pos_offset, const int32_t* counts,
                                int num_seqs, int32_t* ring, int64_t ring_size, int64_t* slot_mapping,
                                int32_t* positions, int64_t capacity, int32_t* cu_seqlens,
                                int32_t* granted, const int32_t* parents, int32_t* masks,
                                int mask_words, void* stream) {
  clear_error();
  if (num_seqs == 0 && capacity == 0) return TI_OK;
  if (!block_tables || !ring || !cu_seqlens || (num_seqs > 0 && (!lens || !counts || !granted)) ||
      (capacity > 0 && (!slot_mapping || !positions)) || mask_words < 0 ||
      (mask_words > 0 && (!parents || !masks)))
    return set_error(TI_ERR_INVALID_ARGUMENT, "reserve slots: null pointer or bad size");
  paging::Params p{block_tables, ring, bt_stride, row_index, lens, counts, pos_offset, parents,
                   slot_mapping, positions, cu_seqlens, granted, masks, capacity, ring_size,
                   num_seqs, num_rows, max_blocks_per_seq, block_size, paging::shift_of(block_size), mask_words,
                   capacity <= paging::kFusedTokens};
  if (int rc = paging::check_sizes(p)) return rc;
  static std::atomic<uint64_t> ready{0};
  if (int rc = paging::raise_limit(paging::reserve_kernel, ready)) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned ctas = num_seqs > 32 || capacity > 1024 ? paging::kCluster : 1;
  if (int rc = launch_kernel_cl("reserve launch", paging::reserve_kernel, dim3(ctas), dim3(paging::kThreads),
                                paging::smem_bytes(num_seqs, num_rows, row_index), s, dim3(ctas), p))
    return rc;
  if (p.fused) return TI_OK;
  const unsigned grid = (unsigned)std::min<int64_t>((capacity + paging::kExpand * paging::kTokens - 1) / (paging::kExpand * paging::kTokens), 148 * 8);
  return launch_kernel("reserve tokens launch", paging::expand_kernel, dim3(grid), dim3(paging::kExpand),
                       (size_t)(num_seqs + 1) * 4, s, 1, p);
}

extern "C" int ti_release_blocks(int32_t* block_tables, int64_t bt_stride, int num_rows,
                                 int max_blocks_per_seq, int block_size, const int32_t* row_index,
                                 const int32_t* keep_lens, int num_seqs, int32_t* ring,
                                 int64_t ring_size, void* stream) {
  clear_error();
  if (num_seqs == 0) return TI_OK;
  if (!block_tables || !ring || !keep_lens)
    return set_error(TI_ERR_INVALID_ARGUMENT, "release blocks: null pointer");
  paging::Params p{};
  p.tables = block_tables;
  p.ring = ring;
  p.bt_stride = bt_stride;
  p.row_index = row_index;
  p.counts = keep_lens;
  p.ring_size = ring_size;
  p.seqs = num_seqs;
  p.rows = num_rows;
  p.cols = max_blocks_per_seq;
  p.block = block_size;
  p.shift = paging::shift_of(block_size);
  if (int rc = paging::check_sizes(p)) return rc;
  static std::atomic<uint64_t> ready{0};
  if (int rc = paging::raise_limit(paging::release_kernel, ready)) return rc;
  const unsigned ctas = num_seqs > 32 ? paging::kCluster : 1;
  return launch_kernel_cl("release launch", paging::release_kernel, dim3(ctas), dim3(paging::kThreads),
                          paging::smem_bytes(num_seqs, num_rows, row_index), reinterpret_cast<cudaStream_t>(stream), dim3(ctas), p);
}
