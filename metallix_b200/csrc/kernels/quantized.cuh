// Rows of a cache held in 8 bits: head_dim codes and one float32 scale per
// (page, plane, key/value head, row of the page).
//
//     scale = max |x| / limit      rounded to float32
//     code  = the code nearest to the exact quotient x / scale, of two equally near the even one
//     value = code * scale         in float32
//
// with e4m3 codes (limit 448) or whole numbers -127..127 (limit 127). A row of
// zeros has scale 0; a row with an infinity or a NaN has scale NaN and reads
// back as NaN throughout, so that it shows where it is used.
//
// Layout of one layer: codes [pages, 2 (K, V), kv_heads, page_tokens, head_dim],
// scales [pages, 2, kv_heads, page_tokens].
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace mxb {

// What the codes are, in the C interface.
enum CodeKind : int { kCodesE4M3 = 0, kCodesInt8 = 1 };

template <int KIND> struct CodeLimit { static constexpr float value = KIND == kCodesE4M3 ? 448.0f : 127.0f; };

template <int KIND> __device__ __forceinline__ float code_value(uint32_t byte) {
  if (KIND == kCodesInt8) return static_cast<float>(static_cast<int8_t>(byte));
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}

// The four codes of a word as two pairs of halves. Whole numbers: with its sign
// bit turned a code is an unsigned u = code + 128, and the half with the bits
// 0x6400 + u is 1024 + u.
template <int KIND> __device__ __forceinline__ void code_halves(uint32_t word, uint32_t& lower, uint32_t& upper) {
  if (KIND == kCodesE4M3) {
    asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\ncvt.rn.f16x2.e4m3x2 %0, lo;\ncvt.rn.f16x2.e4m3x2 %1, hi;\n}\n"
        : "=r"(lower), "=r"(upper) : "r"(word));
  } else {
    const uint32_t turned = word ^ 0x80808080u, off = 0xe480e480u;   // -1152
    const __half2 less = *reinterpret_cast<const __half2*>(&off);
    const uint32_t lo = __byte_perm(turned, 0x64646464u, 0x4140), hi = __byte_perm(turned, 0x64646464u, 0x4342);
    const __half2 a = __hadd2(*reinterpret_cast<const __half2*>(&lo), less), b = __hadd2(*reinterpret_cast<const __half2*>(&hi), less);
    lower = *reinterpret_cast<const uint32_t*>(&a);
    upper = *reinterpret_cast<const uint32_t*>(&b);
  }
}

// What a row's codes are made with. `largest` holds the bits of max |x|: as
// whole numbers they order like the magnitudes, and a NaN's lie above all.
struct RowScale {
  float scale;            // stored
  float divisor, inverse; // the scale, and 1 over it, times `shift`
  float shift;            // a power of two that keeps the quotient's steps away from the ends of float32
};
template <int KIND> __device__ __forceinline__ RowScale row_scale(uint32_t largest) {
  RowScale r;
  if (largest >= 0x7f800000u) {   // not finite: no code has a meaning
    r.scale = __uint_as_float(0x7fc00000u);
    r.divisor = r.inverse = r.shift = 0.0f;
    return r;
  }
  r.scale = __fdiv_rn(__uint_as_float(largest), CodeLimit<KIND>::value);
  r.shift = r.scale < 0x1p-60f ? 0x1p80f : (r.scale > 0x1p60f ? 0x1p-80f : 1.0f);
  r.divisor = r.scale * r.shift;   // exact
  r.inverse = r.divisor > 0.0f ? __frcp_rn(r.divisor) : 0.0f;
  return r;
}

// The quotient x / scale rounded to odd: of the two float32 numbers around an
// inexact quotient the one whose last bit is set, so that rounding it again to
// a code's few bits gives what rounding the exact quotient would. One step of
// Newton's method from x times the reciprocal is within an ulp of the
// quotient; the sign of what is left over (exact, by a fused multiply-add)
// says on which side.
__device__ __forceinline__ float odd_quotient(float x, const RowScale& r) {
  const float xs = x * r.shift;
  float y = xs * r.inverse;
  y = fmaf(fmaf(-y, r.divisor, xs), r.inverse, y);
  const float rest = fmaf(-y, r.divisor, xs);
  if (rest != 0.0f) {
    uint32_t bits = __float_as_uint(y);
    const bool beyond = (rest > 0.0f) == (x > 0.0f);   // the quotient is larger than y in magnitude
    if (!beyond && (bits & 0x7fffffffu) != 0) bits -= 1;
    y = __uint_as_float(bits | 1u);
  }
  return y;
}

// Four quotients' codes as the bytes of a word.
template <int KIND> __device__ __forceinline__ uint32_t round_to_codes(const float* y) {
  if (KIND == kCodesE4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  // to the nearest even by the sum's own rounding: |y| is below 127.5, and the low byte is the code's
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) c[j] = __float_as_uint(__fadd_rn(y[j], 12582912.0f));   // 1.5 x 2^23
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}

// Four values' codes as the bytes of a word. The product by the reciprocal is within 2^-23 of the quotient, so if both ends
// of the numbers within 2^-21 of it have one code that is the quotient's; else (of e4m3 codes one value in 10^5, of whole
// numbers |code| x 2^-20, 12 in 10^5 at most; more where the scale is a power of two; and rows whose scale lies beyond
// 2^-60 ... 2^60) the quotient is rounded to odd first. Five instructions a value instead of fourteen.
template <int KIND> __device__ __forceinline__ uint32_t four_codes(const float* x, const RowScale& r) {
  if (r.inverse == 0.0f) return 0u;   // a row of zeros, or one that is not finite
  float below[4], beyond[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float y = x[j] * r.inverse;
    below[j] = y * (1.0f - 0x1p-21f);
    beyond[j] = y * (1.0f + 0x1p-21f);
  }
  const uint32_t codes = round_to_codes<KIND>(below);
  if (codes == round_to_codes<KIND>(beyond) && r.shift == 1.0f) return codes;
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[j] = odd_quotient(x[j], r);
    // scales among the smallest numbers are coarse: their quotients may lie beyond 127.5
    if (KIND == kCodesInt8) y[j] = fminf(fmaxf(y[j], -127.0f), 127.0f);
  }
  return round_to_codes<KIND>(y);
}

template <int KIND> __device__ __forceinline__ uint32_t code_of(float x, const RowScale& r) {
  if (r.inverse == 0.0f) return 0u;   // a row of zeros, or one that is not finite
  const float y = odd_quotient(x, r);
  if (KIND == kCodesInt8) return static_cast<uint32_t>(max(-127, min(127, __float2int_rn(y)))) & 0xffu;
  return static_cast<uint32_t>(__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3));
}

__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// The larger magnitude, or NaN where either is one.
__device__ __forceinline__ float larger_magnitude(float x, float y) {
  float z;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(z) : "f"(fabsf(x)), "f"(fabsf(y)));
  return z;
}

// Which row of the pool position `key` of a request lies in, counted over
// [pages, page_tokens] of one plane and head: (page * 2 * kv_heads + kv) *
// page_tokens + row is its row number for keys, kv_heads * page_tokens further
// its row number for values. Negative, with a status bit, where the block
// table has no such page. Row numbers of a pool stay below 2^31 (the entries check it).
__device__ __forceinline__ int quantized_row(const int* __restrict__ table, int max_pages, int num_pages, int kv_heads, int kv,
                                             int page_tokens, int key, int* status) {
  const int slot = key / page_tokens;
  const int page = slot < max_pages ? table[slot] : -1;
  if (page < 0 || page >= num_pages) {
    atomicOr(status, kStatusBadPage);
    return -1;
  }
  return (page * 2 * kv_heads + kv) * page_tokens + (key - slot * page_tokens);
}

}  // namespace mxb
