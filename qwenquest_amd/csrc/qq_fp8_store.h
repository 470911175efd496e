// Writing into the 8-bit K/V cache (layout: qq_fp8.h).  Of the values x that a call puts into a
// (block, head), K and V apart,
//   e = max(e_before, least e >= -110 with max |x| <= 448 * 2^e),  code = e4m3(x / 2^e)
// with e_before = -110 when the call writes the block's first row (that begins the block: its
// earlier contents are void), and when e grows the codes already there are re-rounded at the new
// scale (exact but for the least bits of subnormal codes, the scale being a power of two).  A
// value that is not finite makes the scale NaN until the block is begun again.
//
// One thread block per (run of entries of one cache block, head, K or V).  Bound at prompts: HBM;
// at decode steps the chain entries -> values -> write, three round trips.  Measured, 4 heads of
// 128 from bf16: 131071 tokens 83 us (4.9 TB/s; 454 when one block did K and V and wrote the codes
// as it had them instead of composing whole blocks in the LDS), 32 decode tokens 4.9 us.
#pragma once

#include "qq_fp8.h"

namespace qq {
namespace {

struct StoreArgs {
  Fp8Cache c;
  const void* k;  // [n, KV, D] bf16 or fp32
  const void* v;
  int dtype;
  const int64_t* loc;
  int64_t n;
  int seg;  // entries of loc whose runs one thread block looks after, at most 64
};

// Eight consecutive values, as they are stored and as floats.
template <typename SRC>
struct Values8;
template <>
struct Values8<uint16_t> {
  uint4 w;
  __device__ inline void load(const void* base, int64_t at) { w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at); }
  __device__ inline float operator[](int i) const {
    const uint32_t u = i < 2 ? w.x : i < 4 ? w.y : i < 6 ? w.z : w.w;
    return __uint_as_float(i & 1 ? u & 0xFFFF0000u : u << 16);
  }
};
template <>
struct Values8<float> {
  float4 a, b;
  __device__ inline void load(const void* base, int64_t at) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    a = p[0];
    b = p[1];
  }
  __device__ inline float operator[](int i) const {
    const float4& v = i < 4 ? a : b;
    return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
  }
};

__device__ inline bool is_finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

template <int D>
struct StoreSmem {
  static constexpr int kRows = 64 * D / 256;
  int from[64];  // entry that writes each token of the block, or -1
  float amax[4];
  int bad;
  // whole blocks are composed here: 256-byte rows of 16-byte pieces, 16 bytes apart so that
  // the rows' equal columns lie in different banks
  __align__(16) uint8_t codes[kRows * 272];
};

// K (V = false) or V of one (block, head) of a run of entries, by the first 2 D of the thread
// block's threads.  Thread (quad, dg): tokens 4 quad .. + 3, channels 8 dg .. + 7, which are 8-byte
// pieces of K and 4-byte pieces of V.
template <int D, typename SRC, bool V>
__device__ inline void store_block(const StoreArgs& a, StoreSmem<D>& sm, int block, int h) {
  constexpr int NT = 2 * D, DG = D / 8, kWaves = NT / 64;
  const bool mine = threadIdx.x < NT;  // whole waves
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int quad = (tid / DG) & 15, dg = tid % DG;
  const int64_t at = (int64_t)block * a.c.KV + h;
  uint8_t* codes = (V ? a.c.vc : a.c.kc) + at * (64 * D);
  float* scale = (V ? a.c.vs : a.c.ks) + at;
  const float before = *scale;
  const bool begun = sm.from[0] >= 0;
  int from[4];
  Values8<SRC> x[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    from[u] = mine ? sm.from[4 * quad + u] : -1;
    // a token that the call does not write reads the run's values and counts for nothing
    const int64_t row = ((int64_t)max(from[u], 0) * a.c.KV + h) * D + dg * 8;
    x[u].load(V ? a.v : a.k, row);
  }
  float m = 0.0f;
  bool bad = false;
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = x[u][j];
      const bool ok = is_finite(y);
      bad |= !ok && from[u] >= 0;
      m = fmaxf(m, ok && from[u] >= 0 ? fabsf(y) : 0.0f);
    }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  if (lane == 0 && mine) sm.amax[wave] = m;
  if (bad) sm.bad = 1;
  __syncthreads();
  m = sm.amax[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, sm.amax[w]);
  const bool lost = !begun && before != before;
  const int e_old = begun || lost ? kScaleMin : exponent_of(before);
  const int e = max(e_old, scale_exponent(m));
  const float inv = pow2f(-e);
  if (tid == 0) *scale = sm.bad || lost ? __builtin_nanf("") : pow2f(e);
  uint32_t code[4][2];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = from[u] >= 0 && is_finite(x[u][j]) ? x[u][j] * inv : 0.0f;
    code[u][0] = encode4(y[0], y[1], y[2], y[3]);
    code[u][1] = encode4(y[4], y[5], y[6], y[7]);
  }
  if (V) {  // 4 tokens of a channel are neighbours: transposed to words of 4 tokens
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo01 = __builtin_amdgcn_perm(code[1][i], code[0][i], 0x05010400u), hi01 = __builtin_amdgcn_perm(code[1][i], code[0][i], 0x07030602u);
      const uint32_t lo23 = __builtin_amdgcn_perm(code[3][i], code[2][i], 0x05010400u), hi23 = __builtin_amdgcn_perm(code[3][i], code[2][i], 0x07030602u);
      w[4 * i] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
      w[4 * i + 1] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
      w[4 * i + 2] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
      w[4 * i + 3] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) code[j >> 1][j & 1] = w[j];
  }
  if (begun) {
    if (mine) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (!V) {
          const int t = 4 * quad + u, row = (t >> 4) * (D / 16) + dg / 2;
          *reinterpret_cast<uint2*>(&sm.codes[row * 272 + (t & 15) * 16 + (dg & 1) * 8]) = make_uint2(code[u][0], code[u][1]);
        } else {
          const int row = (dg / 2) * 4 + (quad & 3);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint32_t*>(&sm.codes[row * 272 + ((dg & 1) * 8 + 2 * u + i) * 16 + (quad >> 2) * 4]) = code[u][i];
        }
      }
    }
    __syncthreads();
    if (mine) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int q = tid + i * NT;
        *reinterpret_cast<uint4*>(codes + q * 16) = *reinterpret_cast<const uint4*>(&sm.codes[(q >> 4) * 272 + (q & 15) * 16]);
      }
    }
    return;
  }
  if (!mine) return;
  // a block begun before: the tokens written now, and all of them when the scale has grown
  const bool grown = e > e_old;
  const float f = pow2f(max(e_old - e, -126));
  if (!V) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint2* p = reinterpret_cast<uint2*>(codes + k_offset(D, 4 * quad + u, dg * 8));
      if (from[u] >= 0) {
        *p = make_uint2(code[u][0], code[u][1]);
      } else if (grown) {
        const uint2 old = *p;
        *p = make_uint2(rescale4(old.x, f), rescale4(old.y, f));
      }
    }
    return;
  }
  uint32_t mask = 0;  // bytes written now
#pragma unroll
  for (int u = 0; u < 4; ++u) mask |= from[u] >= 0 ? 255u << (8 * u) : 0u;
  if (!mask && !grown) return;
  uint32_t old[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) old[j] = *reinterpret_cast<const uint32_t*>(codes + v_offset(4 * quad, dg * 8 + j));
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t o = grown ? rescale4(old[j], f) : old[j];
    *reinterpret_cast<uint32_t*>(codes + v_offset(4 * quad, dg * 8 + j)) = (code[j >> 1][j & 1] & mask) | (o & ~mask);
  }
}

// K or V of the runs of loc that begin in segment `segment`, head h.  Entries of one block stand next
// to each other in loc; the thread block in whose segment such a run begins writes its (block,
// head) alone, so nothing is shared between thread blocks and the result does not depend on
// their order.  Of a row listed twice in a run the last entry counts.
template <int D, typename SRC, bool V>
__device__ inline void store_segment(const StoreArgs& a, StoreSmem<D>& sm, int64_t segment, int h) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t e0 = segment * a.seg;
  // every wave for itself: the rows of the segment's entries and of as many after them, and
  // where its runs begin
  auto row_at = [&](int64_t i) { return i >= 0 && i < a.n ? a.loc[i] : (int64_t)-1; };
  const int64_t row0 = row_at(e0 + lane), row1 = row_at(e0 + 64 + lane), row_before = row_at(e0 - 1);
  const int b0 = block_of(row0, a.c.blocks), b1 = block_of(row1, a.c.blocks);
  int prev = __shfl_up(b0, 1, 64);
  if (lane == 0) prev = block_of(row_before, a.c.blocks);
  uint64_t starts = __ballot(lane < a.seg && b0 > 0 && b0 != prev);
  while (starts) {
    const int at = __builtin_ctzll(starts);
    starts &= starts - 1;
    const int block = __builtin_amdgcn_readlane(b0, at);
    __syncthreads();  // the run before is done with sm
    if (tid < 64) {
      sm.from[lane] = -1;
      if (lane == 0) sm.bad = 0;
      // (one wave's LDS operations stay in order)
      const uint64_t other = __ballot(b0 != block && lane >= at);
      const int end0 = other ? __builtin_ctzll(other) : 64;
      if (lane >= at && lane < end0) atomicMax(&sm.from[row0 & 63], (int)(e0 + lane));
      if (end0 == 64) {
        const uint64_t other1 = __ballot(b1 != block);
        const int end1 = other1 ? __builtin_ctzll(other1) : 64;
        if (lane < end1) atomicMax(&sm.from[row1 & 63], (int)(e0 + 64 + lane));
        for (int64_t i0 = e0 + 128; end1 == 64; i0 += 64) {  // rows listed twice
          const int64_t row = row_at(i0 + lane);
          const uint64_t more = __ballot(block_of(row, a.c.blocks) != block);
          const int len = more ? __builtin_ctzll(more) : 64;
          if (lane < len) atomicMax(&sm.from[row & 63], (int)(i0 + lane));
          if (len < 64) break;
        }
      }
    }
    __syncthreads();
    store_block<D, SRC, V>(a, sm, block, h);
  }
}

// Single entries by one wave, each by a group of D / 4 lanes, K in the group's first half and V in the
// second: what store_segment does for runs of one entry.  `i` is the group's entry, if `on`; no two
// in one block.  The writes are under way when it returns.  Three round trips, for the entries of a
// wave together (1024 requests of 100 tokens, 4 heads of 64: 23.7 us a layer, with one entry after
// the other 24.4).
template <int D>
__device__ inline void store_tokens(const StoreArgs& a, int64_t i, bool on, int h) {
  constexpr int DG = D / 8;
  const int lane = threadIdx.x & 63, dg = lane % DG;
  const bool isv = lane / DG & 1;
  if (!on) i = 0;
  const int64_t row = a.loc[i];
  const int block = on ? block_of(row, a.c.blocks) : 0, t = (int)(row & 63);
  const bool mine = block > 0;
  if (!__any(mine)) return;
  const int64_t at = (int64_t)block * a.c.KV + h, from = (i * a.c.KV + h) * D + dg * 8;
  uint8_t* codes = (isv ? a.c.vc : a.c.kc) + at * (64 * D);
  float* scale = (isv ? a.c.vs : a.c.ks) + at;
  const float before = *scale;
  float x[8];
  if (a.dtype == QQ_DTYPE_BF16) {
    Values8<uint16_t> v;
    v.load(isv ? a.v : a.k, from);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = v[j];
  } else {
    Values8<float> v;
    v.load(isv ? a.v : a.k, from);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = v[j];
  }
  const bool begun = t == 0;
  float m = 0.0f;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool ok = is_finite(x[j]);
    bad |= !ok;
    x[j] = ok ? x[j] : 0.0f;
    m = fmaxf(m, fabsf(x[j]));
  }
#pragma unroll
  for (int d = DG / 2; d >= 1; d >>= 1) {
    m = fmaxf(m, __shfl_xor(m, d, 64));
    bad |= (bool)__shfl_xor((int)bad, d, 64);
  }
  const bool lost = !begun && before != before;
  const int e_old = begun || lost ? kScaleMin : exponent_of(before);
  const int e = max(e_old, scale_exponent(m));
  const float inv = pow2f(-e);
  const uint32_t lo = encode4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  const uint32_t hi = encode4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
  // a block's other codes: void, or rounded again; by the whole wave
  const float f = begun ? 0.0f : e > e_old ? pow2f(max(e_old - e, -126)) : 1.0f;
  uint64_t blocks = __ballot(mine && dg == 0 && f != 1.0f);
  const bool any = blocks != 0;
  for (; blocks; blocks &= blocks - 1) {
    const int from_lane = __builtin_ctzll(blocks);
    const float fc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), from_lane));
    uint8_t* all = (from_lane / DG & 1 ? a.c.vc : a.c.kc) +
                   ((int64_t)__builtin_amdgcn_readlane(block, from_lane) * a.c.KV + h) * (64 * D);
    for (int q = lane; q < 4 * D; q += 64) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (fc != 0.0f) {
        w = *reinterpret_cast<const uint4*>(all + q * 16);
        w = make_uint4(rescale4(w.x, fc), rescale4(w.y, fc), rescale4(w.z, fc), rescale4(w.w, fc));
      }
      *reinterpret_cast<uint4*>(all + q * 16) = w;
    }
  }
  if (any) __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the entries' own codes come after them
  if (!mine) return;
  if (dg == 0) *scale = bad || lost ? __builtin_nanf("") : pow2f(e);
  if (!isv) {
    *reinterpret_cast<uint2*>(codes + k_offset(D, t, dg * 8)) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) codes[v_offset(t, dg * 8 + j)] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
  }
}

}  // namespace
}  // namespace qq
