// The 4-bit KV cache's format (shared by its kernels).
//
// A pool is [num_blocks, num_kv_heads, 18 * D] bytes, blocks of 16 tokens.  One tile (block, kv
// head) holds, in this order:
//   K codes  [16 tokens][D/2]     two e2m1 codes per byte, the lower dim in the low half
//   V codes  [16 tokens][D/2]
//   K scales [D/16][16 tokens]    one unsigned 8-bit float (5 exponent, 3 mantissa bits) per 16
//   V scales [D/16][16 tokens]    dims of a token: the half-precision number with bits b << 7
// so a value is code * scale: code in {0, .5, 1, 1.5, 2, 3, 4, 6} with a sign has 2 significant
// bits, scale 4, the product at most 6, and it is exact in bf16 and in fp16.  Both e2m1 and 16-dim
// groups keep the error of a group near 1/12 of its largest magnitude whatever the other groups
// of the head hold (keys have a few dims far larger than the rest).  The scales of a group are
// contiguous over the tokens, so a tile's 16 tokens take one or two bytes per lane.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

namespace ti {
namespace kv4 {

constexpr int kBlock = 16;                       // tokens per block
constexpr int kGroup = 16;                       // dims per scale
constexpr float kMaxScale = 10240.f;             // 6 * 10240 = 61440: finite in fp16
constexpr uint32_t kNanScale = 0xFFu;            // 0xFF << 7 = 0x7F80: a half-precision NaN

template <int HD>
struct Tile {
  static constexpr int kRow = HD / 2;            // bytes of one token's codes
  static constexpr int kCodes = kBlock * kRow;
  static constexpr int kGroups = HD / kGroup;
  static constexpr int kK = 0, kV = kCodes;
  static constexpr int kKs = 2 * kCodes, kVs = 2 * kCodes + kGroups * kBlock;
  static constexpr int kBytes = 18 * HD;
};

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __half2float(__ushort_as_half((unsigned short)(byte << 7)));
}

// Eight e2m1 codes (low half of each byte first) as four half2: exact.
__device__ __forceinline__ void codes_to_half2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// Four pairs (lo, hi) to four bytes of e2m1 codes, round to nearest even, saturating at 6.
__device__ __forceinline__ uint32_t floats_to_codes(const float* f) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return w;
}

// Quantise one group of 16 values (of a 16-bit type, held in fp32; `top` = the fp32 bits of their
// largest magnitude): 8 bytes of codes and the scale byte.  scale = amax / 6 rounded to 4 significant
// bits (ties to even, steps of 2^-17 below 2^-14), at most 10240; code = x / scale rounded to e2m1
// (ties to even), saturating.  A group with a NaN or an infinity becomes NaN as a whole (scale 0xFF);
// a group whose scale rounds to zero (amax at most 6 * 2^-18) becomes zero.
//
// Both quotients are products with an approximate reciprocal, off by less than 2^-19 where they are
// rounded, and are first rounded to a multiple of 2^-15 (the sum with 384): x and amax have at most 11
// significant bits and a midpoint of two codes times the scale, or of two scales times 6, at most 7,
// so a quotient that is not a midpoint is at least 2^-13 away from one (2^-8 for the scale's 8 .. 16),
// and one that is lands on it exactly.  The results are therefore those of the exact quotients.
__device__ __forceinline__ uint2 quantize16(const float (&f)[16], uint32_t top, uint32_t& scale_byte) {
  const float a = __uint_as_float(top) * (1.0f / 6.0f);
  const int e = max((int)(__float_as_uint(a) >> 23) - 127, -14);
  const float inv_step = __uint_as_float((uint32_t)(127 + 3 - e) << 23);
  const float step = __uint_as_float((uint32_t)(127 - 3 + e) << 23);
  const float s = fminf(rintf(__fsub_rn(__fmaf_rn(a, inv_step, 384.f), 384.f)) * step, kMaxScale);
  scale_byte = (uint32_t)__half_as_ushort(__float2half_rn(s)) >> 7;
  if (top >= 0x7F800000u) {
    scale_byte = kNanScale;
    return make_uint2(0u, 0u);
  }
  if (s == 0.f) return make_uint2(0u, 0u);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  float y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = __fsub_rn(__fmaf_rn(f[i], r, 384.f), 384.f);
  return make_uint2(floats_to_codes(y), floats_to_codes(y + 8));
}

// fp32 bits of the largest magnitude of 16 values of a 16-bit type, two at a time (a NaN among them
// comes through as one: at least the bits of infinity).
template <typename T>
__device__ __forceinline__ uint32_t largest16(const uint32_t (&w)[8]) {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  T2 top;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = w[i] & 0x7FFF7FFFu;
    const T2 v = *reinterpret_cast<const T2*>(&u);
    top = i == 0 ? v : __hmax2_nan(top, v);
  }
  const float a = Elem<T>::to_f(top.x), b = Elem<T>::to_f(top.y);
  return max(__float_as_uint(a), __float_as_uint(b));             // (both are >= 0, or NaN)
}

}  // namespace kv4
}  // namespace ti
