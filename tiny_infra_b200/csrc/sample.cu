// A token per row of logits: temperature, top-k, top-p, min-p and the draw, in 64 bits.
//
// z = x / t; weights w = exp(z - max z).  In the order of descending values (equal ones by index) the
// kept tokens are a prefix: top-k ends it behind the last value that equals the k-th, top-p behind the
// first place where the sum of weights exceeds p of top-k's, min-p before the first weight below m.  The
// token is the first place whose sum exceeds u of the kept sum.
//
// Weights are 64-bit fixed point (units of 2^-44 up to 2^18 tokens): their sums do not depend on an
// order, and a draw next to the border of two tokens falls on the right side.  First form: one CTA per
// row; every place is found by a radix select over order-preserving 32-bit keys.
#include <algorithm>
#include <type_traits>

#include "capi_internal.h"
#include "common.cuh"

namespace ti {
namespace sample {

typedef unsigned long long u64;
constexpr int kThreads = 512, kWarps = kThreads / 32;

struct Params {
  const void* logits;
  int64_t ld;
  const float *temps, *top_ps, *min_ps, *uniforms;
  const int32_t* top_ks;
  int32_t* tokens;
  float* logprobs;
  int vocab;
  double unit;                           // fixed-point units of a weight of 1
};

__device__ __forceinline__ uint32_t key_of(float x) {   // larger value, larger key; NaN as -inf; -0 as 0
  if (x != x) x = -INFINITY;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

template <typename T> __device__ __forceinline__ float load(const T* p, int j) {
  if constexpr (std::is_same<T, float>::value) return p[j]; else return Elem<T>::to_f(p[j]);
}

struct Weights {
  float top;
  double inv, unit;
  __device__ __forceinline__ double real(float x) const {
    return x == top ? 1.0 : exp(((double)x - (double)top) * inv);
  }
  __device__ __forceinline__ u64 fixed(float x) const { return (u64)__double2ll_rn(real(x) * unit); }
};

struct Shared {
  u64 hist[256];
  u64 part[kWarps];
  float val[kWarps];
  int idx[kWarps];
  uint32_t key;
  int found, index;
  u64 acc, cum;
};

// The first place of the order whose sum of weights (COUNT: of ones) exceeds `target`, among keys >= low.
template <typename T, bool COUNT>
__device__ void find(Shared& sh, const T* row, int V, uint32_t low, const Weights& w, u64 target) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t prefix = 0, mask = 0;
  u64 acc = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int b = tid; b < 256; b += kThreads) sh.hist[b] = 0;
    if (tid == 0) sh.found = 0;
    __syncthreads();
    for (int j = tid; j < V; j += kThreads) {
      const float x = load(row, j);
      const uint32_t k = key_of(x);
      if (k >= low && (k & mask) == prefix) atomicAdd(&sh.hist[(k >> shift) & 255], COUNT ? 1ull : w.fixed(value_of(k)));
    }
    __syncthreads();
    if (tid == 0) {
      u64 run = acc;
      for (int b = 255; b >= 0; --b) {
        if (run + sh.hist[b] > target) { sh.found = 1; sh.key = b; sh.acc = run; break; }
        run += sh.hist[b];
      }
    }
    __syncthreads();
    if (!sh.found) return;
    prefix |= sh.key << shift;
    mask |= 255u << shift;
    acc = sh.acc;
    __syncthreads();
  }
  // equal values, by index
  const u64 one = COUNT ? 1 : w.fixed(value_of(prefix));
  if (tid == 0) { sh.key = prefix; sh.index = -1; }
  const int chunk = (V + kThreads - 1) / kThreads, j0 = min(V, tid * chunk), j1 = min(V, j0 + chunk);
  u64 mine = 0;
  for (int j = j0; j < j1; ++j) mine += key_of(load(row, j)) == prefix;
  u64 incl = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const u64 v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.part[warp] = incl;
  __syncthreads();
  for (int i = 0; i < warp; ++i) incl += sh.part[i];
  u64 run = acc + (incl - mine) * one;
  if (run <= target && run + mine * one > target)
    for (int j = j0; j < j1; ++j) {
      if (key_of(load(row, j)) != prefix) continue;
      run += one;
      if (run > target) { sh.index = j; sh.cum = run; break; }
    }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) row_kernel(const __grid_constant__ Params p) {
  __shared__ Shared sh;
  pdl_wait();
  pdl_launch_dependents();
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = p.vocab;
  const T* row = (const T*)p.logits + (int64_t)r * p.ld;
  float best = -INFINITY;
  int at = 0x7fffffff;
  for (int j = tid; j < V; j += kThreads) {
    const float x = load(row, j);
    if (x > best) { best = x; at = j; }
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, o);
    const int i = __shfl_xor_sync(0xffffffffu, at, o);
    if (v > best || (v == best && i < at)) { best = v; at = i; }
  }
  if (lane == 0) { sh.val[warp] = best; sh.idx[warp] = at; }
  __syncthreads();
  for (int i = 0; i < kWarps; ++i)
    if (sh.val[i] > best || (sh.val[i] == best && sh.idx[i] < at)) { best = sh.val[i]; at = sh.idx[i]; }
  const float temp = p.temps[r];
  int token = best > -INFINITY ? at : -1;
  float logprob = best > -INFINITY ? 0.f : -INFINITY;
  if (token >= 0 && temp > 0.f) {
    const Weights w{best, 1.0 / (double)temp, p.unit};
    const int k = p.top_ks ? p.top_ks[r] : 0;
    uint32_t low = key_of(-INFINITY);
    if (k > 0 && k < V) {
      find<T, true>(sh, row, V, 0, w, (u64)(k - 1));
      low = sh.key;
      __syncthreads();
    }
    const double least = p.min_ps ? fmin((double)p.min_ps[r], 1.0) : 0.0;
    u64 z = 0, zm = 0;
    for (int j = tid; j < V; j += kThreads) {
      const float x = load(row, j);
      const uint32_t key = key_of(x);
      if (key < low) continue;
      const float v = value_of(key);
      const u64 f = w.fixed(v);
      z += f;
      if (w.real(v) >= least) zm += f;
    }
    u64 sum[2] = {z, zm};
    for (int q = 0; q < 2; ++q) {
      for (int o = 16; o > 0; o >>= 1) sum[q] += __shfl_xor_sync(0xffffffffu, sum[q], o);
      __syncthreads();
      if (lane == 0) sh.part[warp] = sum[q];
      __syncthreads();
      sum[q] = 0;
      for (int i = 0; i < kWarps; ++i) sum[q] += sh.part[i];
    }
    u64 kept = sum[0];
    const float top_p = p.top_ps ? p.top_ps[r] : 1.f;
    if (top_p < 1.f) {
      __syncthreads();
      find<T, false>(sh, row, V, low, w, (u64)fmax(0.0, (double)top_p * (double)kept));
      if (sh.found && sh.index >= 0) kept = sh.cum;
      __syncthreads();
    }
    if (least > 0.0) kept = min(kept, sum[1]);
    const double u = fmin(fmax((double)p.uniforms[r], 0.0), 1.0 - 1.0 / 16777216.0);
    find<T, false>(sh, row, V, low, w, (u64)(u * (double)kept));
    if (sh.found && sh.index >= 0) {
      token = sh.index;
      logprob = (float)log(w.real(value_of(sh.key)) * p.unit / (double)kept);
    }
  }
  if (tid == 0) {
    p.tokens[r] = token;
    if (p.logprobs) p.logprobs[r] = logprob;
  }
}

}  // namespace sample
}  // namespace ti

using namespace ti;

extern "C" int ti_sample_ex(const void* logits, int64_t ld, int dtype, int rows, int vocab,
                            const float* temperatures, const int32_t* top_ks, const float* top_ps,
                            const float* min_ps, const float* uniforms, int32_t* out_tokens,
                            float* logprobs, void* stream) {
  clear_error();
  if (rows == 0) return TI_OK;
  if (!logits || !temperatures || !uniforms || !out_tokens || rows < 0 || vocab <= 0 || (rows > 1 && ld < vocab))
    return set_error(TI_ERR_INVALID_ARGUMENT, "sample: null pointer or bad size");
  if (vocab > 1 << 24) return set_error(TI_ERR_UNSUPPORTED, "sample: at most 2^24 tokens");
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  const sample::Params p{logits, ld, temperatures, top_ps, min_ps, uniforms, top_ks, out_tokens, logprobs, vocab,
                         (double)(1ull << std::min(44, 62 - bits))};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)rows), block(sample::kThreads);
  if (dtype == TI_DTYPE_BF16) return launch_kernel("sample launch", sample::row_kernel<__nv_bfloat16>, grid, block, 0, s, 1, p);
  if (dtype == TI_DTYPE_FP16) return launch_kernel("sample launch", sample::row_kernel<__half>, grid, block, 0, s, 1, p);
  if (dtype == TI_DTYPE_FP32) return launch_kernel("sample launch", sample::row_kernel<float>, grid, block, 0, s, 1, p);
  return set_error(TI_ERR_UNSUPPORTED, "sample: dtype must be bf16, fp16 or fp32");
}
