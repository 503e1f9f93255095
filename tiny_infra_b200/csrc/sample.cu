// A token per row of logits: temperature, top-k, top-p, min-p and the draw, in 64 bits.
//
// z = x / t; weights w = exp(z - max z).  In the order of descending values (equal ones by index) the
// kept tokens are a prefix: top-k ends it behind the last value that equals the k-th, top-p behind the
// first place where the sum of weights exceeds p of top-k's, min-p before the first weight below m.  The
// token is the first place whose sum exceeds u of the kept sum.  A sum of many weights has to be right to
// far less than one weight, or draws next to the border of two tokens would go astray: sums are in 64 bits,
// weights exp2 of a rounded exponent times a polynomial of degree 8 on [-1/2, 1/2] (interpolated at the
// Chebyshev nodes; relative error 1.1e-12).
//
// A cluster of up to 8 CTAs shares a row (as many as let the rows fill the GPU).  One pass finds the maximum.
// Then one of three ways, by what the row asks for:
//   few tokens   the k-th largest of a CTA's 128 (or 512) group maxima is a lower bound of the row's k-th
//                largest value, and m times the largest weight is one for min-p: one more pass collects
//                what reaches the bound; rank 0 sorts that, and reads everything off its prefix sums;
//   all tokens   a histogram of weights (4096 bins of equal width in x, a bin's sum in units of 2^-14 of its
//                middle weight; counts too, if top-k has to be placed) bounds the sum down to any bin
//                from both sides, to a few parts in 2^14; so it names the few bins in which top-k's,
//                top-p's and the draw's place can lie.  The next pass adds up the weights above each of
//                these intervals, in 64 bits, and collects what is in them;
//   many ties    when either collection overflows (thousands of equal values): radix selects over 32-bit
//                keys, on fixed-point weights, by rank 0 alone.
// All sums have a fixed order: the same token on every run.
//
// Bound, 151936 tokens: 256 rows of everything the whole vocabulary can ask (fp32, 156 MB) take 206 us.  Of
// the same on bf16 logits with top-p alone (192 us) the maximum's pass is 17 us, the histogram's 53 (shared-memory
// atomics, 4.6 clocks a warp instruction), the weights' 70 to 87 (17 double-precision operations an element
// at 16 a clock and scheduler are 37 of them: each adds 2.2; the rest is issue slots), and barriers, places and
// the draw 25 a CTA, of which an SM has three or four, two at a time.  256 rows of temperature 0.7, top-k 20,
// top-p 0.9 (bf16, 78 MB) take 53 (39 with one CTA a row): a pass from HBM, one from L2, 7 us to the token.
// One such row takes 13.5 as a call: a chain of passes, cluster barriers and code that is run for the first
// time.  Measured on the way, one row: exponentials and scans inlined for each use 26 us, every CTA
// collecting into rank 0's list 22 us; 256 rows: radix selects 5200 us, branches for the sums above the
// intervals 880 us (fp32) instead of masks; loads four steps at a time instead of always two in flight 225
// instead of 206; collecting by the first eighth's bound in the first pass 86 us instead of 62 (top-k 20).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "capi_internal.h"
#include "common.cuh"

namespace ti {
namespace sample {

typedef unsigned long long u64;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kCluster = 8;              // most CTAs of a row
constexpr int kSlice = 8192;             // least elements of a CTA's share
constexpr int kLongSlice = 65536;
constexpr int kFew = 256;                // collected tokens that are ranked rather than sorted
constexpr int kList = 4096;              // collected tokens (a power of two)
constexpr int kGroups = 128;             // of 4 threads
constexpr int kBins = 4096;
constexpr double kOctaves = 40.0;        // range of the histogram below the maximum; what is below it is in the last
                                         // bin, whose tokens are collected (or, if too many, placed by the
                                         // radix selects) when a place can lie there

struct Params {
  const void* logits;
  int64_t ld;
  const float *temps, *top_ps, *min_ps, *uniforms;
  const int32_t* top_ks;
  int32_t* tokens;
  float* logprobs;
  int vocab;
  float quanta;                          // units of a bin's largest weight in its sum (a row's fit 32 bits)
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

// f(x, j) for every 8 elements j .. j + 7 of the row's share j0 .. j1 - 1 (j0 a multiple of 8), by all
// threads, a thread's in ascending order; -inf behind the end.  The loads of U steps are in flight; f's
// code is there once (code that is run for the first time costs more here than the work: it comes from L2).
template <int U, typename T, typename F>
__device__ __forceinline__ void scan8(const T* row, int j0, int j1, F&& f) {
  constexpr int kRaw = (int)sizeof(T) / 2;         // 16-byte words of 8 elements
  const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
  const int full = aligned ? (j1 - j0) / 8 : 0, steps = (j1 - j0 + 7) / 8;
  const uint4* pv = reinterpret_cast<const uint4*>(row + j0);
  uint4 raw[U][kRaw];
  auto fetch = [&](uint4 (&to)[kRaw], int v) {
    if (v < full)
#pragma unroll
      for (int i = 0; i < kRaw; ++i) to[i] = __ldg(pv + v * kRaw + i);
  };
#pragma unroll
  for (int u = 0; u < U; ++u) fetch(raw[u], (int)threadIdx.x + u * kThreads);
#pragma unroll 1
  for (int v = threadIdx.x; v < steps; v += kThreads) {
    uint4 cur[kRaw];
#pragma unroll
    for (int i = 0; i < kRaw; ++i) {
      cur[i] = raw[0][i];
#pragma unroll
      for (int u = 0; u + 1 < U; ++u) raw[u][i] = raw[u + 1][i];
    }
    fetch(raw[U - 1], v + U * kThreads);
    const int j = j0 + v * 8;
    float x[8];
    if (v < full) {
      const T* e = reinterpret_cast<const T*>(cur);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = load(e, i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = j + i < j1 ? load(row, j + i) : -INFINITY;
    }
    f(x, j);
  }
}

// f(x, j) for each element, in no particular order (ties only).
template <typename T, typename F>
__device__ __forceinline__ void scan(const T* row, int j0, int j1, F&& f) {
#pragma unroll 1
  for (int j = j0 + (int)threadIdx.x; j < j1; j += kThreads) f(load(row, j), j);
}

// (one copy of its code in the kernel)
__device__ __noinline__ double exp_once(double x) { return exp(x); }

struct Weights {
  float top;
  double inv, inv2;                      // 1 / t, log2(e) / t
  unsigned low_word;                     // high word of -1000 / inv2
  // exp((x - top) / t) to the last bits; x finite or -inf, or top itself
  __device__ __forceinline__ double exact(float x) const { return x == top ? 1.0 : exp_once(((double)x - (double)top) * inv); }
  // the same for sums (see above); next to nothing for -inf and NaN
  __device__ __forceinline__ double fast(float x) const {
    const double d = (double)x - (double)top;
    // (no double-precision instruction: d is not positive, and its high word grows with its size)
    const double c = __hiloint2double((int)min((unsigned)__double2hiint(d) | 0x80000000u, low_word), __double2loint(d));
    const double t = fma(c, inv2, 6755399441055744.0);   // 1.5 * 2^52: the nearest integer in the low word
    const double r = fma(c, inv2, -(t - 6755399441055744.0));
    double q = 1.3255224878668817e-06;
    q = fma(q, r, 1.5310079402249296e-05);
    q = fma(q, r, 0.00015403455852453838);
    q = fma(q, r, 0.0013333450568000645);
    q = fma(q, r, 0.009618129159402558);
    q = fma(q, r, 0.05550410941205933);
    q = fma(q, r, 0.2402265069581299);
    q = fma(q, r, 0.6931471805459335);
    q = fma(q, r, 1.0);
    return __hiloint2double(__double2hiint(q) + (__double2loint(t) << 20), __double2loint(q));
  }
  __device__ __forceinline__ u64 fixed(float x, double unit) const { return (u64)__double2ll_rn(exact(x) * unit); }
};

// An interval of bins whose tokens are collected: the values from high down to low.
struct Interval {
  int first, last;                       // bins
  float high, low;
};

struct Shared {
  union {
    u64 list[kList];                     // (key << 32) | ~index; group maxima before
    unsigned hist_n[kBins];              // counts
    double prefix[kBins];                // sums of the histogram down to each bin
  };
  union {
    unsigned hist[kBins];
    u64 joined[kList];                   // rank 0: what all CTAs have collected
    double cum[kList];                   // sums down to each of the list's tokens
  };
  // what the CTAs of a cluster tell each other
  float best[kCluster], least[kCluster], bound[kCluster], bound2[kCluster];
  int at[kCluster];
  double sums[kCluster][5];              // weights above intervals 0, 1, 2, all, at least min-p
  int count, at_0, total;                // collected; where they go in rank 0's joined list; rank 0: in all
  Interval iv[3];
  double above[3];                       // sums of the weights before the intervals
  int intervals, mode;
  unsigned long long k_above;            // tokens before the bin of top-k's place, whose largest value is
  float k_high;
  int iv_k, iv_p, iv_u;                  // intervals of the three places
  // scratch
  double part[kWarps][5], scan_d[kWarps];
  u64 part64[kWarps];
  unsigned part_n[kWarps];
  float fpart[kWarps], fpart2[kWarps], kth, kth2;
  int ipart[kWarps], k_bin, edge[4];
  uint32_t key;
  int found, index;
  u64 acc, upto;
};

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void st_peer(uint32_t a, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory"); }
__device__ __forceinline__ void st_peer(uint32_t a, int v) { asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void st_peer(uint32_t a, unsigned v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void st_peer(uint32_t a, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(a), "d"(v) : "memory"); }
__device__ __forceinline__ void st_peer(uint32_t a, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }
__device__ __forceinline__ int ld_peer(uint32_t a) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ int add_peer(uint32_t a, int v) {
  int r;
  asm volatile("atom.shared::cluster.add.s32 %0, [%1], %2;" : "=r"(r) : "r"(a), "r"(v) : "memory");
  return r;
}

// Bitonic sort of list[0 .. n2) in descending order (n2 a power of two); all threads of the CTA.
__device__ void sort_desc(u64* list, int n2) {
  for (int size = 2; size <= n2; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      for (int i = threadIdx.x; i < n2 / 2; i += kThreads) {
        const int a = 2 * i - (i & (stride - 1)), b = a + stride;
        const u64 x = list[a], y = list[b];
        if ((x < y) == ((a & size) == 0)) { list[a] = y; list[b] = x; }
      }
      __syncthreads();
    }
}

// from[0 .. n) to `list` in descending order (n <= kList; they may be the same).  Few tokens: each thread
// finds one's place by comparing it with all others, two barriers instead of one per step.
__device__ __forceinline__ void sort_list(u64* list, const u64* from, int n) {
  const int tid = threadIdx.x;
  if (n > kFew) {
    int n2 = 1;
    while (n2 < n) n2 <<= 1;
    for (int i = tid; i < n2; i += kThreads) list[i] = i < n ? from[i] : 0;     // (0 sorts last)
    __syncthreads();
    sort_desc(list, n2);
    return;
  }
  const u64 mine = tid < n ? from[tid] : 0;
  int place = 0;
  if (tid < ((n + 31) & ~31))
#pragma unroll 8
    for (int i = 0; i < n; ++i) place += from[i] > mine;           // (all entries are different)
  __syncthreads();
  if (tid < n) list[place] = mine;
  __syncthreads();
}

// Inclusive sum over the block, in thread order.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* parts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) parts[warp] = v;
  __syncthreads();
  V before = 0;
  for (int w = 0; w < warp; ++w) before += parts[w];
  return before + v;
}

// ---- many ties: radix selects over the whole row by one CTA -------------------------------------------
// The first place of the order whose sum of weights (COUNT: of ones) exceeds `target`, among keys >= low.
template <typename T, bool COUNT>
__device__ void find(Shared& sh, const T* row, int V, uint32_t low, const Weights& w, double unit, u64 target) {
  const int tid = threadIdx.x;
  u64* hist = sh.list;                             // (256 words; the list is not in use)
  uint32_t prefix = 0, mask = 0;
  u64 acc = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int b = tid; b < 256; b += kThreads) hist[b] = 0;
    if (tid == 0) sh.found = 0;
    __syncthreads();
    // (runs of equal values in registers: they are why this way is taken)
    uint32_t last = 0;
    u64 weight = 0, sum = 0;
    scan(row, 0, V, [&](float x, int) {
      const uint32_t k = key_of(x);
      if (k < low || (k & mask) != prefix) return;
      if (k != last) {
        if (sum) atomicAdd(&hist[(last >> shift) & 255], sum);
        last = k;
        weight = COUNT ? 1ull : w.fixed(value_of(k), unit);
        sum = 0;
      }
      sum += weight;
    });
    if (sum) atomicAdd(&hist[(last >> shift) & 255], sum);
    __syncthreads();
    u64 run = tid < 256 ? hist[255 - tid] : 0ull;
    const u64 own = run;
    run = block_scan(run, sh.part64) + acc;
    if (tid < 256 && run > target && run - own <= target) {
      sh.found = 1;
      sh.key = 255 - tid;
      sh.acc = run - own;
    }
    __syncthreads();
    if (!sh.found) return;
    prefix |= sh.key << shift;
    mask |= 255u << shift;
    acc = sh.acc;
  }
  // equal values, by index
  const u64 one = COUNT ? 1 : w.fixed(value_of(prefix), unit);
  __syncthreads();
  if (tid == 0) { sh.key = prefix; sh.index = -1; }
  const int chunk = (V + kThreads - 1) / kThreads, j0 = min(V, tid * chunk), j1 = min(V, j0 + chunk);
  u64 mine = 0;
  for (int j = j0; j < j1; ++j) mine += key_of(load(row, j)) == prefix;
  const u64 incl = block_scan(mine, sh.part64);
  u64 run = acc + (incl - mine) * one;
  if (run <= target && run + mine * one > target)
    for (int j = j0; j < j1; ++j) {
      if (key_of(load(row, j)) != prefix) continue;
      run += one;
      if (run > target) { sh.index = j; sh.upto = run; break; }
    }
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ void draw_by_radix(Shared& sh, const T* row, int V, const Weights& w, int k,
                                           float top_p, double least, double u, int& token, double& logp) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t low = key_of(-INFINITY);
  if (k > 0 && k < V) {
    find<T, true>(sh, row, V, 0, w, 0.0, (u64)(k - 1));
    low = sh.key;
    __syncthreads();
  }
  // fixed-point units of a weight of 1: as many as keep the whole sum between 2^61 and 2^62, so that the
  // roundings of 2^24 weights move it by 2^-38 at most, whether it is the many tokens or the likely one
  double about = 0;
  {
    uint32_t last = 0;
    double weight = 0;
    scan(row, 0, V, [&](float x, int) {
      const uint32_t key = key_of(x);
      if (key < low) return;
      if (key != last) {
        last = key;
        weight = w.exact(value_of(key));
      }
      about += weight;
    });
    for (int o = 16; o > 0; o >>= 1) about += __shfl_xor_sync(0xffffffffu, about, o);
    __syncthreads();
    if (lane == 0) sh.scan_d[warp] = about;
    __syncthreads();
    about = 0;
    for (int i = 0; i < kWarps; ++i) about += sh.scan_d[i];
  }
  const double unit = scalbn(1.0, 61 - ilogb(about));
  u64 sum[2] = {0, 0}, weight = 0;
  uint32_t last = 0;
  bool heavy = false;
  scan(row, 0, V, [&](float x, int) {
    const uint32_t key = key_of(x);
    if (key < low) return;
    if (key != last) {
      last = key;
      weight = w.fixed(value_of(key), unit);
      heavy = w.exact(value_of(key)) >= least;
    }
    sum[0] += weight;
    if (heavy) sum[1] += weight;
  });
  for (int q = 0; q < 2; ++q) {
    for (int o = 16; o > 0; o >>= 1) sum[q] += __shfl_xor_sync(0xffffffffu, sum[q], o);
    __syncthreads();
    if (lane == 0) sh.part64[warp] = sum[q];
    __syncthreads();
    sum[q] = 0;
    for (int i = 0; i < kWarps; ++i) sum[q] += sh.part64[i];
  }
  u64 kept = sum[0];
  if (top_p < 1.f) {
    find<T, false>(sh, row, V, low, w, unit, (u64)fmax(0.0, (double)top_p * (double)kept));
    if (sh.found && sh.index >= 0) kept = sh.upto;
    __syncthreads();
  }
  if (least > 0.0) kept = min(kept, sum[1]);
  find<T, false>(sh, row, V, low, w, unit, (u64)(u * (double)kept));
  if (sh.found && sh.index >= 0) {
    token = sh.index;
    logp = log(w.exact(value_of(sh.key)) * unit / (double)kept);
  }
}

// ---- rank 0: the three places from the collected tokens and the sums above them ----------------------
// The list's tokens lie in sh.intervals intervals; all: the sum of top-k's weights (k = 0), at_least: of the
// weights >= least; below 0: those sums are the list's own, taken here in its order (the tokens were collected
// in any order, and a sum in that order would have other last bits on every run).
__device__ __forceinline__ void finish(Shared& sh, const u64* collected, int n, const Weights& w, int k, float top_p, double least, double u,
                                       double all, double at_least, bool want_logp, int& token, double& logp) {
  const int tid = threadIdx.x;
  sort_list(sh.list, collected, n);
  auto value = [&](int i) { return value_of((uint32_t)(sh.list[i] >> 32)); };
  double base = 0;
  int heavy = 0;                                   // the list's tokens of weight >= least
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + tid;
    const double e = i < n ? w.exact(value(i)) : 0.0, c = block_scan(e, sh.scan_d);
    if (i < n) sh.cum[i] = base + c;
    heavy += __syncthreads_count(i < n && e >= least);
    base = sh.cum[min(n, i0 + kThreads) - 1];
  }
  if (at_least < 0.0) at_least = heavy > 0 ? sh.cum[heavy - 1] : 0.0;
  if (all < 0.0) all = at_least;
  // from here on every thread finds the same, by binary searches
  auto first = [&](int lo, int hi, auto&& test) {    // the first of [lo, hi) that passes, else hi
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (test(mid)) hi = mid; else lo = mid + 1;
    }
    return lo;
  };
  // an interval's tokens [b, e), and what turns their sums in the list into places in the order
  auto span = [&](int q, int& b, int& e) {
    b = 0;
    e = n;
    if (sh.intervals > 1) {
      b = first(0, n, [&](int i) { return value(i) <= sh.iv[q].high; });
      e = first(b, n, [&](int i) { return value(i) < sh.iv[q].low; });
    }
    return sh.above[q] - (b > 0 ? sh.cum[b - 1] : 0.0);
  };
  int end = n;                                     // top-k's last token is before
  if (k > 0 && n > 0) {
    int b, e;
    const double off = span(sh.iv_k, b, e);
    const long long at = (long long)first(b, e, [&](int i) { return value(i) <= sh.k_high; }) + (k - 1) - (long long)sh.k_above;
    const uint32_t cut = (uint32_t)(sh.list[min((long long)n - 1, at)] >> 32);
    end = first(0, n, [&](int i) { return (uint32_t)(sh.list[i] >> 32) < cut; });
    all = end > b ? sh.cum[end - 1] + off : sh.above[sh.iv_k];
  }
  double kept = all;
  // the first token of an interval whose place's sum exceeds the target (the last one if none does: a sum
  // that ends a rounding short)
  auto place = [&](int q, double target, double& sum) {
    int b, e;
    const double off = span(q, b, e);
    e = min(e, end);
    const int at = min(first(b, e, [&](int i) { return sh.cum[i] + off > target; }), e - 1);
    if (at >= b) sum = sh.cum[at] + off;
    return at >= b ? at : -1;
  };
  if (top_p < 1.f) place(sh.iv_p, fmax(0.0, (double)top_p * all), kept);
  if (least > 0.0) kept = fmin(kept, at_least);
  double sum = 0;
  const int at = place(sh.iv_u, u * kept, sum);
  if (at >= 0) {
    token = (int)~(uint32_t)sh.list[at];
    if (want_logp) logp = (value(at) == w.top ? 0.0 : ((double)value(at) - (double)w.top) * w.inv) - log(kept);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
  const uint32_t ctas = cluster_size(), rank = ctas > 1 ? cluster_rank() : 0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = p.vocab;
  const int64_t r = blockIdx.x / ctas;
  if (tid == 0) sh.count = sh.total = 0;
  auto meet = [&]() { if (ctas > 1) cluster_sync(); else __syncthreads(); };
  if (ctas > 1) cluster_arrive_release();          // (waited for before a peer's memory is touched)
  pdl_wait();
  pdl_launch_dependents();
  const T* row = (const T*)p.logits + r * p.ld;
  const float temp = p.temps[r];
  const bool greedy = !(temp > 0.f);
  int k = p.top_ks ? p.top_ks[r] : 0;
  if (k <= 0 || k >= V) k = 0;
  const float top_p = p.top_ps ? p.top_ps[r] : 1.f;
  const float min_p = p.min_ps ? p.min_ps[r] : 0.f;
  const double least = min_p > 0.f && temp < INFINITY ? fmin((double)min_p, 1.0) : 0.0;   // (at inf all are as likely)
  const double u = fmin(fmax((double)p.uniforms[r], 0.0), 1.0 - 1.0 / 16777216.0);
  const int share = (int)((((int64_t)(V + 7) / 8 + ctas - 1) / ctas) * 8);
  const int j0 = (int)min((int64_t)V, (int64_t)rank * share), j1 = min(V, j0 + share);

  // ---- the largest value and its first place, the smallest finite one, thread maxima
  float best = -INFINITY, smallest = INFINITY;
  int at = 0x7fffffff;
  scan8<2>(row, j0, j1, [&](const float (&x)[8], int j) {
    // (a thread sees its places in ascending order)
    const float a = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    if (a > best) {
      best = a;
#pragma unroll
      for (int i = 7; i >= 0; --i)
        if (x[i] == a) at = j + i;
    }
    // (infinities and NaN among the eight are rare)
    const float b = fminf(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), fminf(fminf(x[4], x[5]), fminf(x[6], x[7])));
    if (b > -INFINITY) {
      smallest = fminf(smallest, b);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) smallest = fminf(smallest, x[i] > -INFINITY ? x[i] : INFINITY);
    }
  });
  const bool by_rank = !greedy && k > 0 && k <= kThreads;
  // (and each of q CTAs' ceil(k / q)-th largest: the least of them has k values above it too)
  const int part_k = (k + (int)ctas - 1) / (int)ctas;
  float bound = -INFINITY, bound2 = -INFINITY;
  if (by_rank && k <= kGroups / 2) {
    // the k-th largest of 128 group maxima: four threads compare one with a quarter of the others each
    float g = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
    g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
    float* groups = reinterpret_cast<float*>(sh.list);
    if ((tid & 3) == 0) groups[tid >> 2] = g;
    __syncthreads();
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < kGroups / 4; ++i) {
      const int o = i * 4 + (tid & 3);
      above += groups[o] > g || (groups[o] == g && o < tid >> 2);
    }
    above += __shfl_xor_sync(0xffffffffu, above, 1);
    above += __shfl_xor_sync(0xffffffffu, above, 2);
    if ((tid & 3) == 0 && above == k - 1) sh.kth = g;
    if ((tid & 3) == 0 && above == part_k - 1) sh.kth2 = g;
    __syncthreads();
    bound = sh.kth;
    bound2 = sh.kth2;
  } else if (by_rank) {
    sh.list[tid] = ((u64)key_of(best) << 32) | (uint32_t)tid;
    __syncthreads();
    sort_desc(sh.list, kThreads);
    bound = value_of((uint32_t)(sh.list[k - 1] >> 32));
    bound2 = value_of((uint32_t)(sh.list[part_k - 1] >> 32));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, o);
    const int i = __shfl_xor_sync(0xffffffffu, at, o);
    if (v > best || (v == best && i < at)) { best = v; at = i; }
    smallest = fminf(smallest, __shfl_xor_sync(0xffffffffu, smallest, o));
  }
  if (lane == 0) { sh.fpart[warp] = best; sh.ipart[warp] = at; sh.fpart2[warp] = smallest; }
  __syncthreads();
  best = sh.fpart[lane & (kWarps - 1)];
  at = sh.ipart[lane & (kWarps - 1)];
  smallest = sh.fpart2[lane & (kWarps - 1)];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, o);
    const int i = __shfl_xor_sync(0xffffffffu, at, o);
    if (v > best || (v == best && i < at)) { best = v; at = i; }
    smallest = fminf(smallest, __shfl_xor_sync(0xffffffffu, smallest, o));
  }
  if (ctas > 1) {
    cluster_wait_acquire();
    if (tid < (int)ctas) {
      st_peer(map_peer(smem_u32(&sh.best[rank]), tid), best);
      st_peer(map_peer(smem_u32(&sh.at[rank]), tid), at);
      st_peer(map_peer(smem_u32(&sh.least[rank]), tid), smallest);
      st_peer(map_peer(smem_u32(&sh.bound[rank]), tid), bound);
      st_peer(map_peer(smem_u32(&sh.bound2[rank]), tid), bound2);
    }
    cluster_sync();
    for (int i = 0; i < (int)ctas; ++i) {
      if (sh.best[i] > best || (sh.best[i] == best && sh.at[i] < at)) { best = sh.best[i]; at = sh.at[i]; }
      smallest = fminf(smallest, sh.least[i]);
      bound = fmaxf(bound, sh.bound[i]);           // (each is a bound by itself)
      bound2 = fminf(bound2, sh.bound2[i]);
    }
    bound = fmaxf(bound, bound2);
  }
  int token = best > -INFINITY ? at : -1;
  double logp = best > -INFINITY ? 0.0 : -INFINITY;
  const bool writer = rank == 0 && tid == 0;
  if (greedy || token < 0) {
    if (writer) {
      p.tokens[r] = token;
      if (p.logprobs) p.logprobs[r] = (float)logp;
    }
    return;
  }
  // (an infinite one as 1e250: every finite value then weighs 1, and -inf still nothing rather than NaN)
  const double t = fmin((double)temp, 1e250);
  const Weights w{best, 1.0 / t, 1.4426950408889634 / t, (unsigned)__double2hiint(-1000.0 / 1.4426950408889634 * t)};
  auto collect = [&](float x, int j) {
    const int slot = atomicAdd(&sh.count, 1);
    if (slot < kList) sh.list[slot] = ((u64)key_of(x) << 32) | (uint32_t)~(uint32_t)j;
  };
  // what the CTAs have collected -> rank 0's `joined`
  auto hand_over = [&]() {
    if (ctas == 1) return;
    __syncthreads();
    const int n = sh.count;
    if (tid == 0 && n > 0) sh.at_0 = add_peer(map_peer(smem_u32(&sh.total), 0), n);
    __syncthreads();
    const uint32_t to = map_peer(smem_u32(sh.joined), 0);
    for (int i = tid; i < min(n, kList); i += kThreads)
      if (sh.at_0 + i < kList) st_peer(to + (sh.at_0 + i) * 8, sh.list[i]);
  };
  // five sums of every thread -> rank 0's sh.sums
  auto send_sums = [&](double (&s)[5]) {
#pragma unroll
    for (int q = 0; q < 5; ++q) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s[q] += __shfl_xor_sync(0xffffffffu, s[q], o);
      if (lane == 0) sh.part[warp][q] = s[q];
    }
    __syncthreads();
    if (tid < 5) {
      double t = 0;
      for (int i = 0; i < kWarps; ++i) t += sh.part[i][tid];
      if (ctas > 1) st_peer(map_peer(smem_u32(&sh.sums[rank][tid]), 0), t); else sh.sums[0][tid] = t;
    }
  };
  auto total = [&](int q) {
    double t = 0;
    for (int i = 0; i < (int)ctas; ++i) t += sh.sums[i][q];
    return t;
  };

  // ---- few tokens
  bool done = false;
  // (min-p's bound leaves out tokens of top-k that top-p's sum needs)
  const bool by_weight = least > 0.0 && (k == 0 || top_p >= 1.f);
  if (by_rank || by_weight) {
    __syncthreads();                               // (the list held the thread maxima)
    if (ctas > 1) cluster_sync();
    float low = bound;
    if (by_weight) {
      // a little below the value whose weight is m; the weights themselves decide later
      const double v = (double)best + log(least) * t;
      const float f = (float)(v - 1e-6 * (fabs(v) + fabs((double)best)));
      low = fmaxf(low, f);
    }
    if (best == INFINITY) low = INFINITY;
    double s[5] = {0, 0, 0, 0, 0};
    const bool sum_all = k == 0 && top_p < 1.f;
    auto reach = [&](const float (&x)[8], int j) {
      const float a = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      if (a >= low) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (x[i] >= low && j + i < j1) {
            collect(x[i], j + i);
            s[3] += best == INFINITY ? 1.0 : 0.0;
          }
      }
    };
    if (sum_all && best < INFINITY)
      scan8<2>(row, j0, j1, [&](const float (&x)[8], int j) {
        reach(x, j);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[3] += w.fast(x[i]);
      });
    else
      scan8<2>(row, j0, j1, reach);
    hand_over();
    send_sums(s);
    meet();
    const int n = ctas > 1 ? ld_peer(map_peer(smem_u32(&sh.total), 0)) : sh.count;
    if (n <= kList) {
      if (ctas > 1) cluster_arrive_release();      // (rank 0 stays until its peers have read the count)
      if (rank != 0) { cluster_wait_acquire(); return; }
      const double all = total(3);
      const u64* collected = ctas > 1 ? sh.joined : sh.list;
      if (tid == 0) {
        sh.intervals = 1;
        sh.above[0] = 0.0;
        sh.iv_k = sh.iv_p = sh.iv_u = 0;
        sh.k_above = 0;
        sh.k_high = INFINITY;
      }
      __syncthreads();
      finish(sh, collected, n, w, k, top_p, least, u, sum_all ? all : -1.0, -1.0, p.logprobs != nullptr, token, logp);
      done = true;
      if (ctas > 1) cluster_wait_acquire();
    } else {
      meet();                                      // (everyone has read the count)
    }
  }

  // ---- all tokens
  // bins of equal width from the maximum down to the smallest value, or 40 octaves
  const double octaves = fmin(((double)best - (double)smallest) * w.inv2, kOctaves);
  const double bins = (double)(kBins - 1) * w.inv2 / octaves;        // a unit of x
  if (!done && best < INFINITY && octaves > 0.0 && bins < 1e38) {    // (temperatures from 1e-36 on)
    // (bin b: the values whose distance from the maximum rounds to b; halves to even, monotonic all the same)
    const float per = (float)bins;
    const double width = w.inv2 / (double)per;                       // octaves of a bin (at most 40 / 4095)
    constexpr float kRound = 12582912.f;                             // 1.5 * 2^23: the nearest integer in the low bits
    auto rounded = [&](float x) { return fminf(fmaf(best - x, per, kRound), kRound + (float)(kBins - 1)); };
    auto bin = [&](float x) { return __float_as_int(rounded(x)) - __float_as_int(kRound); };
    for (int b = tid; b < kBins; b += kThreads) {
      sh.hist[b] = 0;
      if (k > 0) sh.hist_n[b] = 0;
    }
    if (tid == 0) sh.count = sh.total = 0;
    __syncthreads();
    // a weight in units of its bin's middle: 2^(-width f), f from -1/2 to 1/2, as a polynomial; the sum with 2^23
    // leaves its nearest integer in the low bits
    const float drop = (float)(-0.6931471805599453 * width);
    const float c2 = p.quanta * 0.5f * drop * drop, c1 = p.quanta * drop, c0 = p.quanta + 8388608.f;
    auto weigh = [&](float x) {
      const float t = rounded(x);
      const int b = __float_as_int(t) - __float_as_int(kRound);
      const float f = fminf(fmaf(best - x, per, kRound - t), 0.5f);  // (the last bin: not below its own end)
      atomicAdd(&sh.hist[b], __float_as_uint(fmaf(f, fmaf(f, c2, c1), c0)) & 0x7fffffu);
      return b;
    };
    scan8<2>(row, j0, j1, [&](const float (&x)[8], int) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (x[i] > -INFINITY) {
          const int b = weigh(x[i]);
          if (k > 0) atomicAdd(&sh.hist_n[b], 1u);
        }
    });
    meet();
    if (ctas > 1) {
      // each CTA sums its part of the bins over the cluster into rank 0's histograms
      const int part = kBins / (int)ctas;
      for (int which = 0; which < (k > 0 ? 2 : 1); ++which) {
        unsigned* h = which ? sh.hist_n : sh.hist;
        unsigned sum[kBins / 2 / kThreads];
#pragma unroll
        for (int i = 0; i < kBins / 2 / kThreads; ++i) {
          const int b = i * kThreads + tid;
          sum[i] = 0;
          if (b < part)
            for (int c = 0; c < (int)ctas; ++c)
              sum[i] += (unsigned)ld_peer(map_peer(smem_u32(h + (int)rank * part + b), c));
        }
        cluster_sync();
#pragma unroll
        for (int i = 0; i < kBins / 2 / kThreads; ++i) {
          const int b = i * kThreads + tid;
          if (b < part) st_peer(map_peer(smem_u32(h + (int)rank * part + b), 0), sum[i]);
        }
      }
      cluster_sync();
    }
    if (rank == 0) {
      constexpr int E = kBins / kThreads;          // a thread has 8 neighbouring bins
      if (k > 0) {
        // the bin of the k-th largest value, and the tokens before it (the last bin, if there are fewer)
        unsigned cnt[E], own_n = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) own_n += cnt[e] = sh.hist_n[tid * E + e];
        unsigned run = block_scan(own_n, sh.part_n) - own_n;
        if (tid == kThreads - 1) { sh.k_bin = kBins - 1; sh.k_above = run + own_n - cnt[E - 1]; }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (run < (unsigned)k && run + cnt[e] >= (unsigned)k) { sh.k_bin = tid * E + e; sh.k_above = run; }
          run += cnt[e];
        }
        __syncthreads();
      }
      // sums down to each bin.  A weight was rounded to a unit, and the distance from the maximum to 24 bits,
      // which moves it by 0.03 units at most; a token has at least 0.99 of the units of its bin's middle, less
      // one.  So each bin's true sum is between (1 - d) and (1 + d) times what is held, and so are sums over
      // bins; the last bin has the tokens below the range too, its sum may be next to nothing.
      const double d = 0.6 / ((double)p.quanta * 0.99 - 1.0);
      double sum[E];                               // down to each of this thread's bins
      {
        double own = 0, most = exp2(-(double)(tid * E) * width) / (double)p.quanta;
        const double ratio = exp2(-width);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          sum[e] = own += (double)sh.hist[tid * E + e] * most;
          most *= ratio;
        }
        const double before = block_scan(own, sh.scan_d) - own;
#pragma unroll
        for (int e = 0; e < E; ++e) sh.prefix[tid * E + e] = sum[e] += before;
        if (tid < 4) sh.edge[tid] = kBins - 1;
      }
      __syncthreads();
      auto upto = [&](int b) { return b < 0 ? 0.0 : sh.prefix[b]; };
      // Bins in which the sum can first exceed q of the kept one, when what is kept ends in bins keep_a + 1 ..
      // keep_b: s(b) > q s(end) is (1 - q) s(b) > q (s(end) - s(b)), the difference a sum of bins too, so
      // that a place near the end is known as well as one near the beginning.
      int keep_a = kBins - 1, keep_b = kBins - 1;
      const double last = sh.prefix[kBins - 1] - sh.prefix[kBins - 2];
      auto bracket = [&](double q, int slot) {
        // (the last bin may hold nothing: it does not count towards a sum that is to be small)
        const double end_a = upto(keep_a) - (keep_a == kBins - 1 ? last : 0.0), end_b = upto(keep_b);
        const double up = 1.0 + d, down = 1.0 - d;
        unsigned f = kBins - 1, l = kBins - 1;
#pragma unroll
        for (int e = E - 1; e >= 0; --e) {
          if ((1.0 - q) * sum[e] * up > q * (end_a - sum[e]) * down) f = tid * E + e;
          if ((1.0 - q) * sum[e] * down > q * (end_b - sum[e]) * up) l = tid * E + e;
        }
        f = __reduce_min_sync(0xffffffffu, f);
        l = __reduce_min_sync(0xffffffffu, l);
        if (lane == 0 && f < kBins - 1) atomicMin(&sh.edge[slot], (int)f);
        if (lane == 0 && l < kBins - 1) atomicMin(&sh.edge[slot + 1], (int)l);
        __syncthreads();
        Interval iv;
        iv.first = sh.edge[slot];
        iv.last = max(sh.edge[slot + 1], iv.first);
        return iv;
      };
      Interval ik, ip;
      ik.first = ip.first = -1;
      if (k > 0) {
        ik.first = ik.last = sh.k_bin;
        keep_a = ik.first - 1;
        keep_b = ik.first;
      }
      if (top_p < 1.f) {
        ip = bracket(fmax(0.0, (double)top_p), 0);
        keep_a = min(keep_a, ip.first - 1);
        keep_b = min(keep_b, ip.last);
      }
      if (least > 0.0) {
        // (the bins around the value of weight m)
        const int b = (int)fmin(fmax(-log2(least) / width, 0.0), (double)(kBins - 1));
        keep_a = min(keep_a, max(b - 3, -1));
        keep_b = min(keep_b, min(b + 3, kBins - 1));
      }
      const Interval iu = bracket(u, 2);
      __syncthreads();
      if (tid == 0) {
        // the union of the intervals, in order
        int first[3] = {}, end[3] = {}, m = 0;
        auto add = [&](const Interval& i) {
          int a = m++;
          for (; a > 0 && first[a - 1] > i.first; --a) { first[a] = first[a - 1]; end[a] = end[a - 1]; }
          first[a] = i.first;
          end[a] = i.last;
        };
        if (ik.first >= 0) add(ik);
        if (ip.first >= 0) add(ip);
        add(iu);
        int out = 0;
        for (int a = 1; a < m; ++a) {
          if (first[a] <= end[out] + 1) end[out] = max(end[out], end[a]);
          else { ++out; first[out] = first[a]; end[out] = end[a]; }
        }
        sh.intervals = out + 1;
        auto in = [&](const Interval& i) { return out > 1 && i.first >= first[2] ? 2 : out > 0 && i.first >= first[1] ? 1 : 0; };
        sh.iv_k = ik.first >= 0 ? in(ik) : 0;
        sh.iv_p = ip.first >= 0 ? in(ip) : 0;
        sh.iv_u = in(iu);
        for (int a = 0; a <= out; ++a) { sh.iv[a].first = first[a]; sh.iv[a].last = end[a]; }
      }
      __syncthreads();
      // an interval's values (warp 2 a: the largest, warp 2 a + 1: the smallest of its bins; warp 6: the
      // largest of top-k's bin), and whether the tokens fit the list (warp 7)
      const int m = sh.intervals;
      if (warp < 2 * m || (warp == 6 && k > 0)) {
        // keys lo < hi of neighbouring values whose bins are on either side of the edge before bin e, found in
        // steps of 32 places at once; they are near best - e / per: two bins on either side, if that is right
        const int e = warp == 6 ? ik.first : warp & 1 ? sh.iv[warp >> 1].last + 1 : sh.iv[warp >> 1].first;
        uint32_t lo = key_of(best - (float)(e + 2) / per), hi = key_of(fminf(best, best - (float)(e - 2) / per));
        if (!(bin(value_of(lo)) >= e)) lo = key_of(-INFINITY);
        if (bin(value_of(hi)) >= e) hi = key_of(best);
#pragma unroll 1
        while (hi - lo > 1) {
          const uint32_t step = (hi - lo + 32) / 33, mid = min(lo + step * (uint32_t)(lane + 1), hi);
          const uint32_t in = __ballot_sync(0xffffffffu, mid < hi && bin(value_of(mid)) >= e);
          const int n = __popc(in);                // (they are the first n places)
          const uint32_t next = lo + step * (uint32_t)(n + 1);
          lo += step * (uint32_t)n;
          hi = min(hi, next);
        }
        if (lane == 0) {
          const float above = e == 0 ? best : value_of(lo), below = e == kBins ? -3.402823466e38f : value_of(hi);
          if (warp == 6) sh.k_high = above;
          else if (warp & 1) sh.iv[warp >> 1].low = below;
          else sh.iv[warp >> 1].high = above;
        }
      } else if (warp == 7) {
        float n = 0;
        for (int a = 0; a < m; ++a)
          for (int b = sh.iv[a].first + lane; b <= sh.iv[a].last; b += 32)
            n += ceilf((float)sh.hist[b] / (p.quanta * 0.98f - 1.f));
        const unsigned most_n = __reduce_add_sync(0xffffffffu, (unsigned)fminf(n, (float)(kList + 1)));
        if (lane == 0) sh.mode = most_n <= (unsigned)kList;
      }
      __syncthreads();
      if (ctas > 1 && tid < (int)ctas && tid > 0) {
        for (int a = 0; a < 3; ++a) {
          st_peer(map_peer(smem_u32(&sh.iv[a].high), tid), sh.iv[a].high);
          st_peer(map_peer(smem_u32(&sh.iv[a].low), tid), sh.iv[a].low);
        }
        st_peer(map_peer(smem_u32(&sh.intervals), tid), sh.intervals);
        st_peer(map_peer(smem_u32(&sh.mode), tid), sh.mode);
      }
    }
    meet();
    if (sh.mode) {                                 // (the intervals' tokens fit the list)
      const int m = sh.intervals;
      float high[3], low[3];
#pragma unroll
      for (int a = 0; a < 3; ++a) {
        high[a] = a < m ? sh.iv[a].high : -INFINITY;
        low[a] = a < m ? sh.iv[a].low : INFINITY;
      }
      double s[5] = {0, 0, 0, 0, 0};
      // e or next to nothing: without its high word it is below 2^-1000
      auto masked = [](bool yes, double e) { return __hiloint2double(yes ? __double2hiint(e) : 0, __double2loint(e)); };
      scan8<1>(row, j0, j1, [&](const float (&x)[8], int j) {
        unsigned in = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double e = w.fast(x[i]);
          s[3] += e;
          s[0] += masked(x[i] > high[0], e);
          in |= x[i] <= high[0] && x[i] >= low[0] ? 1u << i : 0u;
          if (m > 1) {
            s[1] += masked(x[i] > high[1], e);
            in |= x[i] <= high[1] && x[i] >= low[1] ? 1u << i : 0u;
          }
          if (m > 2) {
            s[2] += masked(x[i] > high[2], e);
            in |= x[i] <= high[2] && x[i] >= low[2] ? 1u << i : 0u;
          }
          if (least > 0.0) s[4] += masked(e >= least, e);
        }
#pragma unroll 1
        for (; in; in &= in - 1) {                 // (one or two of a warp's 256: read again rather than selected)
          const int i = j + __ffs(in) - 1;
          collect(load(row, i), i);
        }
      });
      hand_over();
      send_sums(s);
      meet();
      if (rank == 0) {
        if (tid < 3) sh.above[tid] = total(tid);
        const double all = total(3), m = total(4);
        const int n = ctas > 1 ? sh.total : sh.count;
        __syncthreads();
        finish(sh, ctas > 1 ? sh.joined : sh.list, n, w, k, top_p, least, u, all, m, p.logprobs != nullptr, token, logp);
      }
      done = true;
    }
  }
  if (!done && rank == 0) {
    __syncthreads();
    draw_by_radix(sh, row, V, w, k, top_p, least, u, token, logp);
  }
  if (writer) {
    p.tokens[r] = token;
    if (p.logprobs) p.logprobs[r] = (float)logp;
  }
}

template <typename T>
static int launch(const Params& p, int rows, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};          // devices whose limit has been raised
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared));
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return set_cuda_error(e, "cudaFuncSetAttribute(sample)");
    }
    ready.fetch_or(bit, std::memory_order_release);
  }
  // CTAs of a row: while all of them fit the GPU (two an SM) and each has a share worth a barrier, or up to
  // twice as many while the shares are long, since one row that asks for the whole vocabulary is then the
  // end of the launch (256 rows of 151936, two CTAs each instead of one: mixed 126 us instead of 172, all
  // open 206 instead of 214, all top-k 20 53 instead of 39; with four, mixed 140, open 252; 256 rows of 32000
  // gain nothing).  Pairs of which one CTA leaves where a row does not need it are no way out: the GPU keeps
  // its place until the pair ends (open 347, all top-k 20 71).  Measured at these two sizes only: where between
  // them the border lies is a guess, and rows that all ask for few tokens would be better off without it
  unsigned ctas = 1;
  while (ctas < (unsigned)kCluster) {
    const int64_t next = (int64_t)rows * ctas * 2;
    const int share = p.vocab / (int)(ctas * 2);
    if (!(next <= 296 && share >= kSlice) && !(next <= 592 && share >= kLongSlice)) break;
    ctas *= 2;
  }
  return launch_kernel_cl("sample launch", sample_kernel<T>, dim3((unsigned)rows * ctas), dim3(kThreads), sizeof(Shared), s,
                          dim3(ctas), p);
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
  if (vocab > 1 << 24 || rows > 1 << 24)
    return set_error(TI_ERR_UNSUPPORTED, "sample: at most 2^24 tokens and rows");
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  const sample::Params p{logits, ld, temperatures, top_ps, min_ps, uniforms, top_ks, out_tokens, logprobs, vocab,
                         (float)(1 << std::min(14, 31 - bits))};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == TI_DTYPE_BF16) return sample::launch<__nv_bfloat16>(p, rows, s);
  if (dtype == TI_DTYPE_FP16) return sample::launch<__half>(p, rows, s);
  if (dtype == TI_DTYPE_FP32) return sample::launch<float>(p, rows, s);
  return set_error(TI_ERR_UNSUPPORTED, "sample: dtype must be bf16, fp16 or fp32");
}
