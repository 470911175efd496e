// The 4-bit K/V cache: its layout, and what its kernels share.
//
// A cache holds blocks of 64 tokens.  Of one layer, block b and KV head h has 32 * D bytes of
// e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign) for K and for V.  A value is code * 2^(scale - 127);
// a scale is one byte, the exponent's: of K one for each token and 32 channels, of V one for each
// token.  Keys have channels that stand out, so their scales follow the channels, and fit the operands of
// K Q^T, whose lanes hold 32 channels of a token; a token's V scale rides on its softmax weight.
// Every token has its own scales and its own bytes: rows are written in any order and over and over,
// and no write touches another token's values.
//
// The codes lie in the order in which the matrix instructions take them, so that a wave's
// 16-byte loads of a block are 1 KiB runs and nothing is transposed on the way (even channels in the
// low half of K's bytes):
//   K: token t = 16 T + m, channel d = 32 c + j:  ((T * D / 32 + c) * 16 + m) * 16 + j / 2
//      (32 channels of a token are 16 bytes: a lane's operands A of K Q^T, four steps of 8)
//   V: token t = 16 T + 4 g + u, channel d = 64 c + 32 x + 16 y + m, half x of byte
//      (((c * 2 + y) * 4 + g) * 16 + m) * 16 + 4 T + u
//      (16 tokens of two channels are 16 bytes; a byte is one token's, so that a token's write is
//      whole bytes.  Words T and T' = T + 1 hold 4 tokens each; (T & 0F0F0F0F) | (T' & 0F0F0F0F) << 4 are the
//      8 tokens of the lower channel, as pairs (T, T') that a conversion takes together)
//   K's scales: (c * 16 + m) * 4 + T: a lane's four tokens in a word
//   V's scales: g * 16 + 4 T + u:     a lane's sixteen tokens in 16 bytes
// Codes are never NaN: a token and head with a value that is not finite, or one of V above 7 * 2^59, has the scale 255 in K and in V,
// which the conversions of K read as NaN whatever the code, and zeros for codes.
#pragma once

#include "qq_fp8.h"

namespace qq {

constexpr int kFp4Group = 32;               // channels of K that share a scale
constexpr int kFp4Lo = -96, kFp4Hi = 125;   // exponents of K's scales: 6 * 2^125 is finite, 2^-97 a normal bf16
constexpr int kFp4VLo = -50, kFp4VHi = 59;  // of V's: within 2^109, so that weights times scales fit one range (fp4_extend.hip)
constexpr uint32_t kFp4Lost = 255;          // the scale of what was not finite

struct Fp4Cache {  // one layer, or the first of several
  uint8_t* kc;     // [blocks, KV, 32 * D]
  uint8_t* vc;
  uint8_t* ks;     // [blocks, KV, 2 * D]
  uint8_t* vs;     // [blocks, KV, 64]
  int blocks, KV, D;
};

// The least exponent with amax <= 7 * 2^e: values between 6 and 7 round to 6, the largest code.
__host__ __device__ inline int fp4_exponent(float amax) {
  const uint32_t u = __builtin_bit_cast(uint32_t, amax);
  return (int)(u >> 23) - 127 - ((u & 0x7FFFFFu) <= 0x600000u ? 2 : 1);  // 7 = 1.75 * 2^2
}
// The scale bytes of K's 32 channels (the largest finite values stand at 6 * 2^125) and of a token's V.
__host__ __device__ inline uint32_t fp4_k_scale(float amax) {
  const int e = fp4_exponent(amax);
  return (uint32_t)(127 + (e < kFp4Lo ? kFp4Lo : e > kFp4Hi ? kFp4Hi : e));
}
__host__ __device__ inline uint32_t fp4_v_scale(float amax) {
  const int e = fp4_exponent(amax);
  return (uint32_t)(127 + (e < kFp4VLo ? kFp4VLo : e > kFp4VHi ? kFp4VHi : e));
}
constexpr float kFp4VMax = 7.0f * 576460752303423488.0f;  // 7 * 2^59: V beyond is lost

// 2^(byte - 127) of byte i of a word; 255 gives infinity's bits.
__device__ inline float fp4_factor(uint32_t w, int i) {
  return __uint_as_float((i == 3 ? w >> 1 : w << (23 - 8 * i)) & 0x7F800000u);
}

// Byte offsets in a head's codes and scales.
__device__ inline int fp4_k_offset(int D, int t, int d) {
  return (((t >> 4) * (D >> 5) + (d >> 5)) * 16 + (t & 15)) * 16 + (d & 31) / 2;
}
__device__ inline int fp4_v_offset(int t, int d) {  // half (d >> 5) & 1 of it
  return ((((d >> 6) * 2 + ((d >> 4) & 1)) * 4 + ((t >> 2) & 3)) * 16 + (d & 15)) * 16 + (t >> 4) * 4 + (t & 3);
}
__device__ inline int fp4_ks_offset(int t, int d) { return ((d >> 5) * 16 + (t & 15)) * 4 + (t >> 4); }
__device__ inline int fp4_vs_offset(int t) { return ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3); }

// Codes of eight finite floats, s a power of two: to nearest even, 6 at most.
__device__ inline uint32_t fp4_encode8(const float (&x)[8], float s) {
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
}

// Codes 2 i and 2 i + 1 of a word times s, as bf16 (exact); NaN, whatever the code, for the s of a lost
// token, whose exponent bits are all set.
__device__ inline bf16x2_t fp4_pair(uint32_t w, float s, int i) {
  switch (i) {
    case 0: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0);
    case 1: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
    case 2: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2);
    default: return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
  }
}

// The 8 tokens of the lower (x = 0) or upper channel of two words of V, token pairs side by side.
__device__ inline uint32_t fp4_lower(uint32_t a, uint32_t b) { return (a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u); }
__device__ inline uint32_t fp4_upper(uint32_t a, uint32_t b) { return ((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u); }

int check_cache(const Fp4Cache& c, const char* what);

}  // namespace qq
