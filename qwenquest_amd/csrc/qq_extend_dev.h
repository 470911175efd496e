// What the prefill kernels share: their tiles of query rows, and K/V tiles that go from memory to
// the LDS directly.  (Reference src/qwenquest/attention/base.py:65-93.)
#pragma once

#include "qq_quest_dev.h"
#include "qq_rules.h"

namespace qq {
namespace {

typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr int kExtWaves = 4;
using rules::extend_request_tiles;
using rules::extend_splits;
using rules::extend_tiles;
using rules::kExtMaxSplits;
using rules::kExtRows;
using rules::kExtTile;
using rules::split_chunk;
static_assert(kExtRows == 32 * kExtWaves && kExtMaxSplits <= 32, "a wave's rows; the merge's lanes");

// What a block works on: request, first query row of its tile, the request's rows.
struct ExtendTile {
  int b;         // request, or -1: a tile past the requests' rows
  int tile;      // tile of the request
  int q0;        // the request's first row in q (tokens); b == -1: first token past every request
  int n;         // the request's new tokens
  int past;      // b == -1: tiles past the last request's
  int req;       // table row, or -1: outside the table
  int kv_len;    // context, cut to the table's width
  int prefix;
};

// Tiles are numbered request after request, as many as each request's rows need.
// Every wave finds the tile's request by itself: 64 requests at a time, a prefix
// sum over the lanes.
template <typename Args>
__device__ inline ExtendTile find_tile(const Args& a, int t) {
  const int lane = threadIdx.x & 63;
  int tok = 0, tile = 0;  // tokens and tiles of the requests before this group of 64
  for (int b0 = 0; b0 < a.bs; b0 += 64) {
    const int b = b0 + lane;
    // the request's four words go out together
    const int64_t len = b < a.bs ? a.ext[b] : 0;
    const int64_t req = b < a.bs ? a.rpi[b] : 0;
    const int64_t seq = b < a.bs ? a.seq[b] : 0;
    const int64_t prefix = b < a.bs ? a.prefix[b] : 0;
    int n = (int)min(max(len, (int64_t)0), (int64_t)a.n);
    int nt = 0, sn = n;  // inclusive sums over the lanes
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(sn, d, 64);
      if (lane >= d) sn = min(sn + u, a.n);
    }
    // q holds a.n rows: a request past them has what is left
    const int before = __shfl_up(sn, 1, 64);
    const int first = min(tok + (lane > 0 ? before : 0), a.n);
    n = min(n, a.n - first);
    const int mine = extend_request_tiles(n, a.G);
    nt = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(nt, d, 64);
      if (lane >= d) nt += u;
    }
    const uint64_t hit = __ballot(b < a.bs && t < tile + nt);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      ExtendTile r;
      r.b = b0 + src;
      r.tile = t - (tile + __shfl(nt, src, 64) - __shfl(mine, src, 64));
      r.q0 = __shfl(first, src, 64);
      r.n = __shfl(n, src, 64);
      r.past = 0;
      const int64_t row = req < 0 ? req + a.r2t_rows : req;  // a negative index counts from the table's end
      r.req = __shfl(row >= 0 && row < a.r2t_rows ? (int)row : -1, src, 64);
      const int kv = (int)min(max(seq, (int64_t)0), a.r2t_stride);
      r.kv_len = r.req >= 0 ? __shfl(kv, src, 64) : 0;  // wave-uniform branch
      r.prefix = __shfl((int)min(max(prefix, -(int64_t)(1 << 30)), (int64_t)(1 << 30)), src, 64);
      return r;
    }
    tok = min(tok + __shfl(sn, 63, 64), a.n);
    tile += __shfl(nt, 63, 64);
  }
  return {-1, 0, tok, 0, t - tile, -1, 0, 0};
}

// 64 lanes x 16 bytes from per-lane global addresses to LDS byte address `lds` + 16 *
// lane.  In inline asm (it writes no register; tile_barrier waits for it), since the
// compiler would wait for the builtin's pending LDS write before the other buffer's
// reads, that is for the next tile before this one's products.  (M0 has no other use
// in these kernels.)
__device__ inline void load_lds16(const void* g, uint32_t lds) {
  __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(g) : "memory");
}

// This wave's tile loads have landed, then every wave's: one block barrier per tile.
// (The builtin wait also tells the compiler that its own loads have landed.)
__device__ inline void wait_vm() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt(0)
__device__ inline void tile_barrier() {
  wait_vm();
  __asm__ volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A sum of weights relative to 2^from, brought to the maximum `to` of what the output sums, w = 2^(from - to): where V's
// scales are in those maxima, tokens may count in the weights' sum that far below it.
__device__ inline float scaled_sum(float sum, float from, float to, float w) {
  if (w > 0.0f || from == -INFINITY) return w * sum;
  const float half = __builtin_amdgcn_exp2f(0.5f * (from - to));
  return half * (half * sum);
}

// Adds up a tile's splits: one block per (tile, KV head, 8 rows), 32 threads a row (of 64
// channels the upper 16 write nothing).
template <int D, typename Args>
__global__ __launch_bounds__(256) void extend_merge_kernel(Args a) {
  const int h = blockIdx.y, t_lin = blockIdx.x;
  const ExtendTile et = find_tile(a, t_lin);
  if (et.b < 0) return;
  const int kv_len = et.kv_len, prefix = et.prefix;
  const int rows_n = et.n * a.G, r0 = et.tile * kExtRows;
  const int tok_last = (min(r0 + kExtRows, rows_n) - 1) / a.G;
  const int lim_blk = min(kv_len, prefix + tok_last + 1);
  const int nt_all = lim_blk > 0 ? (lim_blk + kExtTile - 1) / kExtTile : 0;
  const int chunk = split_chunk(nt_all, a.splits);
  if (nt_all <= chunk) return;
  const int parts = (nt_all + chunk - 1) / chunk;
  const int i = blockIdx.z * 8 + (threadIdx.x >> 5), d4 = min((threadIdx.x & 31) * 4, D - 4);
  const int r = r0 + i;
  if (r >= rows_n) return;  // all 32 lanes of the row
  const int64_t step = (int64_t)a.KV * a.tiles * kExtRows;
  const int64_t pr = ((int64_t)h * a.tiles + t_lin) * kExtRows + i;
  // lane p of the row's 32 holds part p's (m, l): parts <= kExtMaxSplits
  const int p = threadIdx.x & 31;
  const float2 ml = p < parts ? *reinterpret_cast<const float2*>(a.part_ml + (pr + p * step) * 2)
                              : make_float2(-INFINITY, 0.0f);
  float Mx = ml.x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) Mx = fmaxf(Mx, __shfl_xor(Mx, d, 32));
  const float w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - Mx);
  float Ls = scaled_sum(ml.y, ml.x, Mx, w);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) Ls += __shfl_xor(Ls, d, 32);
  float4 Os = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < parts; p0 += 8) {
    float4 ov[8];  // a group's loads go out together; past the last part they re-read it
#pragma unroll
    for (int u = 0; u < 8; ++u)
      ov[u] = *reinterpret_cast<const float4*>(a.part_o + (pr + min(p0 + u, parts - 1) * step) * D + d4);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float wu = __shfl(w, p0 + u, 32);  // p0 + u < 32
      if (p0 + u >= parts) break;  // block-uniform; a weight of 0 would make NaN of an infinite sum
      Os.x += wu * ov[u].x;
      Os.y += wu * ov[u].y;
      Os.z += wu * ov[u].z;
      Os.w += wu * ov[u].w;
    }
  }
  if ((threadIdx.x & 31) * 4 >= D) return;
  const float inv = 1.0f / Ls;
  const int tok = r / a.G;
  uint16_t* op = a.out + ((int64_t)(et.q0 + tok) * a.H + h * a.G + r - tok * a.G) * D + d4;
  *reinterpret_cast<uint2*>(op) = make_uint2((uint32_t)f2bf(Os.x * inv) | ((uint32_t)f2bf(Os.y * inv) << 16),
                                             (uint32_t)f2bf(Os.z * inv) | ((uint32_t)f2bf(Os.w * inv) << 16));
}

}  // namespace
}  // namespace qq
