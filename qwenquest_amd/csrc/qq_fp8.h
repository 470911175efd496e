// The 8-bit K/V cache: its layout, and what its kernels share.
//
// A cache holds blocks of 64 tokens.  Of one layer, block b and KV head h has 64 * D bytes of
// e4m3 codes for K and for V, and one float scale each, a power of two; a value is code * scale.
// The codes lie in the order in which the matrix instructions take them, so that a wave's
// 16-byte loads of a block are 1 KiB runs and nothing is transposed on the way:
//   K: token t = 16 T + m, channel d:  ((T * D / 16 + d / 16) * 16 + m) * 16 + d % 16
//      (16 channels of a token are 16 bytes; 16 tokens' pieces of the same channels follow
//      one another: operand A of K Q^T, lane m + 16 g holding piece g of token m)
//   V: token t = 16 T + 4 g + u, channel d:  ((d / 16 * 4 + g) * 16 + d % 16) * 16 + 4 T + u
//      (16 tokens of a channel are 16 bytes: operand A of V^T P^T, lane m + 16 g holding
//      those tokens of channel m whose weights the same lanes get from K Q^T)
// Codes are never NaN, whatever was written: what is not finite makes the scale NaN, so that
// a masked token's stale codes times a weight of 0 are 0.
#pragma once

#include "qq_common.h"

namespace qq {

constexpr int kMaxPoolBlocks = 1 << 24;  // rows fit req_to_token's int32
constexpr int kCacheTokens = 64;         // tokens of a block
constexpr int kScaleMin = -110;          // least exponent of a scale: code * scale is a normal bf16 or 0

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

struct Fp8Cache {  // one layer, or the first of several
  uint8_t* kc;     // [blocks, KV, 64 * D]
  uint8_t* vc;
  float* ks;       // [blocks, KV]
  float* vs;
  int blocks, KV, D;
};

inline bool fp8_dim_ok(int D) { return D == 64 || D == 128; }

__host__ __device__ inline float pow2f(int e) {  // -126 .. 127
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}
__host__ __device__ inline int exponent_of(float x) { return (int)((__builtin_bit_cast(uint32_t, x) >> 23) & 255u) - 127; }

// The least e >= kScaleMin with amax <= 448 * 2^e (448 = 1.75 * 2^8, the largest code).
__host__ __device__ inline int scale_exponent(float amax) {
  const uint32_t u = __builtin_bit_cast(uint32_t, amax);
  const int e = (int)(u >> 23) - 127 - ((u & 0x7FFFFFu) <= 0x600000u ? 8 : 7);
  return e > kScaleMin ? e : kScaleMin;
}

// e4m3 codes of four floats of magnitude <= 448 (round to nearest even), and back.
__device__ inline uint32_t encode4(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
__device__ inline float4 decode4(uint32_t w) {
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return make_float4(lo.x, lo.y, hi.x, hi.y);
}
__device__ inline uint32_t rescale4(uint32_t w, float f) {
  const float4 x = decode4(w);
  return encode4(x.x * f, x.y * f, x.z * f, x.w * f);
}

// Byte offset of (token t, channel d) in a head's codes.
__device__ inline int k_offset(int D, int t, int d) { return (((t >> 4) * (D >> 4) + (d >> 4)) * 16 + (t & 15)) * 16 + (d & 15); }
__device__ inline int v_offset(int t, int d) {
  return (((d >> 4) * 4 + ((t >> 2) & 3)) * 16 + (d & 15)) * 16 + (t >> 4) * 4 + (t & 3);
}

// Block of a pool row, or 0 (padding, nothing is kept there) for one outside the cache.
__device__ inline int block_of(int64_t row, int blocks) {
  const int64_t b = row >> 6;
  return b > 0 && b < blocks ? (int)b : 0;
}

int check_cache(const Fp8Cache& c, const char* what);

}  // namespace qq
