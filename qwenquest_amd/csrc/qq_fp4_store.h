// Writing into the 4-bit K/V cache (layout: qq_fp4.h).  A token's K has for each 32 channels, its V as a
// whole
//   e = least with max |x| <= 7 * 2^e, of K's -96 .. 125, of V's -50 .. 59,  code = e2m1(x / 2^e),
// to nearest even, 6 at most.  Of a row listed twice in a run of one block the last entry counts.
#pragma once

#include "qq_fp4.h"
#include "qq_fp8_store.h"

namespace qq {
namespace {

constexpr float kFinite = 3.4028234663852886e38f;  // the largest finite float

struct Fp4StoreArgs {
  Fp4Cache c;
  const void* k;  // [n, KV, D] bf16 or fp32
  const void* v;
  int dtype;
  const int64_t* loc;
  int64_t n;
  int seg;
};

// Whether an entry after i in its run of one block has the same row: that one counts.
__device__ inline bool written_again(const Fp4StoreArgs& a, int64_t i, int64_t row) {
  for (int64_t j = i + 1; j < a.n; ++j) {
    const int64_t other = a.loc[j];
    if (other == row) return true;
    if (other >> 6 != row >> 6) return false;
  }
  return false;
}

// Single entries, each of one head by a group of D / 4 lanes, K in the group's first half and V in the
// second, 8 channels a lane.  `i` is the group's entry, if `on`.  The writes are under way when
// it returns.
template <int D, typename SRC>
__device__ inline void fp4_store_group(const Fp4StoreArgs& a, int64_t i, bool on, int h) {
  constexpr int DG = D / 8;
  const int lane = threadIdx.x & 63, dg = lane % DG;
  const bool isv = lane / DG & 1;
  if (!on) i = 0;
  const int64_t row = a.loc[i];
  Values8<SRC> in;
  in.load(isv ? a.v : a.k, (i * a.c.KV + h) * D + dg * 8);
  const int block = on ? block_of(row, a.c.blocks) : 0, t = (int)(row & 63);
  const bool mine = block > 0 && !written_again(a, i, row);
  float x[8], m = 0.0f;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = in[j];
    bad |= !(fabsf(x[j]) <= (isv ? kFp4VMax : kFinite));
    m = fmaxf(m, fabsf(x[j]));
  }
  const uint64_t lost = __ballot(bad);
  bad = lost >> (lane / (2 * DG) * (2 * DG)) & (2 * DG == 64 ? ~0ull : (1ull << (2 * DG % 64)) - 1ull);
  m = fmaxf(m, __shfl_xor(m, 1, 64));
  m = fmaxf(m, __shfl_xor(m, 2, 64));  // of 32 channels
  float all = m;
#pragma unroll
  for (int d = 4; d < DG; d <<= 1) all = fmaxf(all, __shfl_xor(all, d, 64));
  const uint32_t e = isv ? fp4_v_scale(all) : fp4_k_scale(m);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = bad ? 0.0f : x[j];
  const uint32_t code = fp4_encode8(x, __uint_as_float(e << 23));
  const uint32_t other = __shfl_xor(code, 4, 64);  // the channels 32 further on (or back)
  if (!mine) return;
  const int64_t at = (int64_t)block * a.c.KV + h;
  const uint8_t scale = (uint8_t)(bad ? kFp4Lost : e);
  if (!isv) {
    *reinterpret_cast<uint32_t*>(a.c.kc + at * (32 * D) + fp4_k_offset(D, t, dg * 8)) = code;
    if (dg % 4 == 0) a.c.ks[at * (2 * D) + fp4_ks_offset(t, dg * 8)] = scale;
    return;
  }
  if (dg == 0) a.c.vs[at * 64 + fp4_vs_offset(t)] = scale;
  // the lane of the lower 32 channels writes its channels 0 .. 3, the other one 4 .. 7, of both
  const bool up = dg & 4;
  uint8_t* codes = a.c.vc + at * (32 * D) + fp4_v_offset(t, (dg & ~4) * 8);
  const uint32_t lo = up ? other >> 16 : code, hi = up ? code >> 16 : other;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    codes[((up ? 4 : 0) + j) * 16] = (uint8_t)(((lo >> (4 * j)) & 15u) | (((hi >> (4 * j)) & 15u) << 4));
}

template <int D>
__device__ inline void fp4_store_tokens(const Fp4StoreArgs& a, int64_t i, bool on, int h) {
  if (a.dtype == QQ_DTYPE_BF16) fp4_store_group<D, uint16_t>(a, i, on, h);
  else fp4_store_group<D, float>(a, i, on, h);
}

}  // namespace
}  // namespace qq
