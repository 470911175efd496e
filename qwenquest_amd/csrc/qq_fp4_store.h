// Writing into the 4-bit K/V cache (layout: qq_fp4.h).  A token's K has for each 32 channels, its V as a
// whole
//   e = least with max |x| <= 7 * 2^e, of K's -96 .. 125, of V's -50 .. 59,  code = e2m1(x / 2^e),
// to nearest even, 6 at most.  Of a row listed twice in a run of one block the last entry counts.
//
// A token's V is half bytes of D / 2 places (its byte at each holds two channels), a token's K 16 bytes at D / 32 places: a
// token alone writes them so (fp4_store_group), the tokens of a run turn theirs between the lanes until 16 tokens of
// two channels are a lane's 16 bytes (fp4_store_block; times: fp4_cache.hip).
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

// Whether an entry after i in its run of one block has the same row, which is the one that counts then; by the
// W lanes of i's group, as many entries at a time.  `next`: the row of this lane's first, i + 1 + its place in the group.
template <int W>
__device__ inline bool written_again(const Fp4StoreArgs& a, int64_t i, int64_t row, int64_t next, bool on) {
  const int lane = threadIdx.x & 63, first = lane / W * W;
  constexpr uint64_t kGroup = (1ull << W) - 1ull;
  bool again = false;
  for (int64_t j = i + 1 + lane - first; __any(on); j += W) {
    const int64_t other = on && j < a.n ? (j < i + 1 + W ? next : a.loc[j]) : (int64_t)-1;
    const uint64_t ends = __ballot(other >> 6 != row >> 6) >> first & kGroup;
    const uint64_t same = __ballot(other == row) >> first & kGroup;
    again |= on && (ends ? same & ((ends & -ends) - 1) : same) != 0;
    on = on && ends == 0;
  }
  return again;
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
  const int64_t row = a.loc[i], next = a.loc[min(i + 1 + lane % (2 * DG), a.n - 1)];  // (in one round trip)
  Values8<SRC> in;
  in.load(isv ? a.v : a.k, (i * a.c.KV + h) * D + dg * 8);
  const int block = on ? block_of(row, a.c.blocks) : 0, t = (int)(row & 63);
  const bool again = written_again<2 * DG>(a, i, row, next, block > 0), mine = block > 0 && !again;
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

// Nibbles of a half word, each in a byte, and back.
__device__ inline uint32_t spread_nibbles(uint32_t x) {
  x = (x | (x << 8)) & 0x00FF00FFu;
  return (x | (x << 4)) & 0x0F0F0F0Fu;
}
__device__ inline uint32_t gather_nibbles(uint32_t x) {
  x &= 0x0F0F0F0Fu;
  x = (x | (x >> 4)) & 0x00FF00FFu;
  return (x | (x >> 8)) & 0xFFFFu;
}

// Of four lanes u, DG apart, their words' bytes turned: byte k of lane u becomes byte u of lane k.
template <int DG>
__device__ inline uint32_t turn_bytes(uint32_t w, int u) {
  uint32_t b = __shfl_xor(w, DG, 64);
  w = u & 1 ? __builtin_amdgcn_perm(b, w, 0x03070105u) : __builtin_amdgcn_perm(b, w, 0x06020400u);
  b = __shfl_xor(w, 2 * DG, 64);
  return u & 2 ? __builtin_amdgcn_perm(b, w, 0x03020706u) : __builtin_amdgcn_perm(b, w, 0x05040100u);
}

// K and V of one (block, head) of a run of entries, by the first 2 D of the thread block's threads: thread (4 g + u,
// dg) has tokens 16 T + 4 g + u, T = 0 .. 3, channels 8 dg .. + 7, of both.
template <int D, typename SRC>
__device__ inline void fp4_store_block(const Fp4StoreArgs& a, const int (&from)[64], int block, int h) {
  constexpr int DG = D / 8;
  if (threadIdx.x >= 2 * D) return;  // whole waves
  const int lane = threadIdx.x & 63, tt = threadIdx.x / DG, dg = lane % DG, g = tt >> 2, u = tt & 3;
  const int64_t at = (int64_t)block * a.c.KV + h;
  uint8_t *kc = a.c.kc + at * (32 * D), *vc = a.c.vc + at * (32 * D), *ks = a.c.ks + at * (2 * D), *vs = a.c.vs + at * 64;
  int f[4];
  Values8<SRC> in[2][4];
#pragma unroll
  for (int T = 0; T < 4; ++T) {
    f[T] = from[16 * T + tt];
    // a token that the call does not write reads the run's values and counts for nothing
    const int64_t row = ((int64_t)max(f[T], 0) * a.c.KV + h) * D + dg * 8;
    in[0][T].load(a.k, row);
    in[1][T].load(a.v, row);
  }
  uint32_t scales = 0, v[4], here = 0;  // here: bit 4 T + u of the tokens that are written
#pragma unroll
  for (int T = 0; T < 4; ++T) {
    float x[2][8], m[2] = {0.0f, 0.0f};
    bool bad = false;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[w][j] = in[w][T][j];
        bad |= !(fabsf(x[w][j]) <= (w ? kFp4VMax : kFinite));
        m[w] = fmaxf(m[w], fabsf(x[w][j]));
      }
    const uint64_t lost = __ballot(bad), on = __ballot(f[T] >= 0);
    bad = lost >> (lane / DG * DG) & ((1ull << DG) - 1ull);
#pragma unroll
    for (int d = 1; d < DG; d <<= 1) {
      if (d < 4) m[0] = fmaxf(m[0], __shfl_xor(m[0], d, 64));
      m[1] = fmaxf(m[1], __shfl_xor(m[1], d, 64));
    }
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[w][j] = bad ? 0.0f : x[w][j];
    const uint32_t e = fp4_k_scale(m[0]), ev = fp4_v_scale(m[1]);
    const uint32_t code = fp4_encode8(x[0], __uint_as_float(e << 23)), vcode = fp4_encode8(x[1], __uint_as_float(ev << 23));
    scales |= (bad ? kFp4Lost : e) << (8 * T);
    if (f[T] >= 0) {
      *reinterpret_cast<uint32_t*>(kc + fp4_k_offset(D, 16 * T + tt, dg * 8)) = code;
      if (dg == 0) vs[fp4_vs_offset(16 * T + tt)] = (uint8_t)(bad ? kFp4Lost : ev);
    }
    // V's channels 0 .. 3 of this lane's and of the one 32 channels on, or 4 .. 7, a byte for each two
    const uint32_t other = __shfl_xor(vcode, 4, 64);
    const uint32_t w = dg & 4 ? spread_nibbles(other >> 16) | (spread_nibbles(vcode >> 16) << 4)
                              : spread_nibbles(vcode & 0xFFFFu) | (spread_nibbles(other & 0xFFFFu) << 4);
    // and of the four lanes u the tokens of one channel pair, the u-th
    v[T] = turn_bytes<DG>(w, u);
#pragma unroll
    for (int y = 0; y < 4; ++y) here |= (uint32_t)(on >> (lane / (4 * DG) * (4 * DG) + y * DG) & 1) << (4 * T + y);
  }
  uint8_t* sp = ks + fp4_ks_offset(tt, dg * 8);
  uint8_t* vp = vc + fp4_v_offset(4 * g, (dg & ~4) * 8 + (dg & 4) + u);
  if (here == 0xFFFFu) {  // the same in the lanes of one g
    if (dg % 4 == 0) *reinterpret_cast<uint32_t*>(sp) = scales;
    *reinterpret_cast<uint4*>(vp) = make_uint4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int T = 0; T < 4; ++T) {
    if (dg % 4 == 0 && f[T] >= 0) sp[T] = (uint8_t)(scales >> (8 * T));
    const uint32_t mine = here >> (4 * T) & 15u;
    if (mine == 15u) {
      *reinterpret_cast<uint32_t*>(vp + 4 * T) = v[T];
      continue;
    }
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (mine >> y & 1u) vp[4 * T + y] = (uint8_t)(v[T] >> (8 * y));
  }
}

template <int D>
__device__ inline void fp4_store_tokens(const Fp4StoreArgs& a, int64_t i, bool on, int h) {
  if (a.dtype == QQ_DTYPE_BF16) fp4_store_group<D, uint16_t>(a, i, on, h);
  else fp4_store_group<D, float>(a, i, on, h);
}

}  // namespace
}  // namespace qq
