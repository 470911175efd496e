// The division of a decode batch over the 8-bit cache (fp8_decode.hip): what it takes from the
// batch's lengths, what it leaves for the attention, and where that lies in the workspace.
#pragma once

#include "qq_fp8.h"
#include "qq_rules.h"

namespace qq {
namespace {

constexpr int kTile = 16;  // query heads of a tile

struct DecPlan {
  int32_t total, len, slices;  // units of the batch, units of a slice, slices
  int32_t bs, top_k;           // what it is of
};
struct DecItem {  // a slice's first request: its units are [c0, c1) of the batch's
  int32_t b, c0, c1, seq;
  int32_t req, pad[3];  // its table row, or -1: outside the table
};


struct PlanArgs {
  const int64_t* rpi;
  const int64_t* seq;
  int bs, table_rows, table_cols;
  int top_k;              // tokens that a longer context selects, or 0: none does
  int max_slices, heads;  // heads: KV * tiles
  DecPlan* plan;
  int32_t* cu;     // [bs + 1] units before each request
  DecItem* items;  // [max_slices]
  uint32_t* done;  // [max_slices, heads] parts finished of the request that goes on behind a slice; left 0
};

__device__ inline int context_of(const PlanArgs& a, int b) {
  return (int)min(max(a.seq[b], (int64_t)0), (int64_t)a.table_cols * kCacheTokens);
}
__device__ inline int table_row(const PlanArgs& a, int b) {
  const int64_t req = a.rpi[b];
  return req >= 0 && req < a.table_rows ? (int)req : -1;
}
__device__ inline bool is_sparse(const PlanArgs& a, int s) { return a.top_k > 0 && s > a.top_k; }
__device__ inline int units_of(const PlanArgs& a, int s) {
  if (is_sparse(a, s)) return a.top_k / 64;
  return max((s + 63) / 64, 1);  // an empty context: one unit without tokens, which writes its zeros
}

// Cuts the batch's units into slices; 256 threads.
__device__ inline void plan_slices(const PlanArgs& a) {
  __shared__ int s_sum[4], s_long[4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  for (int i = tid; i < a.max_slices * a.heads; i += 256) a.done[i] = 0u;
  int base = 0, longest = 0;
  for (int b0 = 0; b0 < a.bs; b0 += 256) {
    const int b = b0 + tid;
    const int u = b < a.bs ? units_of(a, context_of(a, b)) : 0;
    int x = u;
    longest = max(longest, u);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(x, d, 64);
      if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) s_sum[wave] = x;
    __syncthreads();
    int before = base;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += s_sum[w];
      base += s_sum[w];
    }
    if (b < a.bs) a.cu[b] = before + x - u;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) longest = max(longest, __shfl_xor(longest, d, 64));
  if (lane == 0) s_long[wave] = longest;
  if (tid == 0) a.cu[a.bs] = base;
  __syncthreads();
  longest = max(max(s_long[0], s_long[1]), max(s_long[2], s_long[3]));
  const int len = rules::fp8_slice_len(base, longest, a.max_slices);
  const int slices = (base + len - 1) / len;
  if (tid == 0) *a.plan = {base, len, slices, a.bs, a.top_k};
  for (int i = tid; i < slices; i += 256) {
    const int at = i * len;
    int lo = 0, hi = a.bs;  // the last request that begins at or before this unit
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid] <= at) lo = mid;
      else hi = mid;
    }
    a.items[i] = {lo, a.cu[lo], a.cu[lo + 1], context_of(a, lo), table_row(a, lo), {0, 0, 0}};
  }
}

// The workspace's parts, in order; offsets are multiples of 256 bytes.
struct DecSpace {
  int64_t cu, items, done, part_o, part_ml, bytes;
  int max_slices;
};
inline DecSpace decode_space(int bs, int H, int KV, int D) {
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  const int tiles = (H / KV + kTile - 1) / kTile, heads = KV * tiles;
  DecSpace s;
  s.max_slices = rules::fp8_max_slices(heads);
  s.cu = up(sizeof(DecPlan));
  s.items = s.cu + up((int64_t)(bs + 1) * 4);
  s.done = s.items + up((int64_t)s.max_slices * sizeof(DecItem));
  s.part_o = s.done + up((int64_t)s.max_slices * heads * 4);
  s.part_ml = s.part_o + (int64_t)s.max_slices * 2 * heads * kTile * D * 4;
  s.bytes = s.part_ml + (int64_t)s.max_slices * 2 * heads * kTile * 2 * 4;
  return s;
}

// The plan's part of the arguments; `ws` holds s.bytes.
inline void set_plan(PlanArgs& a, const DecSpace& s, void* ws, const int64_t* rpi, const int64_t* seq, int bs, int table_rows,
                     int table_cols, int top_k, int heads) {
  char* p = static_cast<char*>(ws);
  a.rpi = rpi;
  a.seq = seq;
  a.bs = bs;
  a.table_rows = table_rows;
  a.table_cols = table_cols;
  a.top_k = top_k;
  a.max_slices = s.max_slices;
  a.heads = heads;
  a.plan = reinterpret_cast<DecPlan*>(p);
  a.cu = reinterpret_cast<int32_t*>(p + s.cu);
  a.items = reinterpret_cast<DecItem*>(p + s.items);
  a.done = reinterpret_cast<uint32_t*>(p + s.done);
}

}  // namespace
}  // namespace qq
