// Decode attention over the 8-bit K/V cache (layout: qq_fp8.h), dense or over the pages that
// Quest selected (reference src/qwenquest/attention/dense.py:26-42, quest_only.py:132-159,
// ops.py:48-66 over that cache).  With ks, vs the scales of token j's block and kc, vc its codes
//   t_j = scale * log2(e) * ks * (q . kc_j),  p_j = 2^(t_j - max t),  out = sum p_j vs vc_j / sum p_j.
//
// The work comes in units, a (partial) block of the cache: of a dense request its blocks in
// order, of one with selected pages those and its recent window (the last 64 tokens, which lie at
// 64 different places of two blocks: a place comes from one or the other).  All
// requests' units in a row are cut into equal slices, one to a thread block per (KV head, tile
// of 16 query heads), so that any mix of lengths fills the chip evenly in one round; a
// request that lies in one slice is finished there, the others' (m, l, o) parts are merged by
// the block that completes them.
//
// Launches: fp8_begin_kernel cuts the slices, stores the new tokens and selects pages,
// fp8_attend_kernel does the rest.  The slices depend on the lengths alone: cut once for a step
// (fp8_plan_kernel, or beside the page bounds), a dense layer is one launch, in which the wave that
// has a request's last block stores the request's new token into it first; a layer of Quest stores
// beside the page scores (a selected page may be the one that is written) and selects here, at
// shapes where that costs less than a launch (selects_itself).
//
// Of its block's slice a wave takes an eighth, units in a row, and goes through their requests on
// its own; what a request's end finds in one wave is written by that wave, the rest meets in the
// LDS.  A slice of many short requests thus has eight of them in work at once, their blocks
// looked up together, and a request's first unit is loaded under the one before it.  A wave
// takes a unit at a time: K and V codes straight from memory to registers in the
// operands' order (1 KiB runs), converted to bf16 (exact), S^T = K Q^T, the softmax in
// registers, O^T += V^T P^T, with P's values scaled by vs as three bf16 pieces, which hold all 24
// significand bits (in two pieces, 16 bits, bf16 outputs were off by a step in a few of a thousand places,
// for 2 us less of 145 in 12 layers of one request of 2000 tokens).  fp32 queries go in as three bf16
// pieces, too.
// Bound: HBM, the codes once, when they are many: 16 requests of 131072 tokens, 4 heads of 128,
// 379 us (5.7 TB/s; matrix pipes 18 % busy, vector units 44 %).  A small batch is bound by its chain
// of memory round trips (slice, table words, scales and codes, partials, count, merge, ~1 us each):
// one request of 2000 tokens 11.4 us a layer, of which its waves wait 80 %; 15.8 in two launches; the
// plan 4.6 us a step.  16 requests' 31 pages and window of 131072 tokens 18.1 us with the selection
// (waiting 54 %), 16.1 behind a begin launch of 5.4.
#include "qq_fp8_plan.h"
#include "qq_fp8_store.h"
#include "qq_quest_dev.h"
#include "qq_rules.h"

namespace qq {
namespace {

constexpr int kDecWaves = 8;
constexpr int kDecParts = rules::kFp8Parts;  // slices of a request, at most: the merge's table of weights

struct DecArgs : PlanArgs {
  const void* q;  // [bs, H, D]
  int64_t q_bstride;
  int H, G, tiles;  // query heads, of a KV head, tiles of those
  Fp8Cache c;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* positions;  // nullptr: dense, or the attention selects
  int64_t pos_stride;
  float sl2;  // scale * log2(e)
  void* out;  // [bs, H, D]
  float* part_o;   // [max_slices, 2, heads, 16, D]
  float* part_ml;  // [max_slices, 2, heads, 16, 2]
};

__global__ __launch_bounds__(256) void fp8_plan_kernel(DecArgs a) { plan_slices(a); }

// Block 0: the slices; then a block per request that selects its pages (KPT > 0: scores per
// thread), and a block per new token, head, and K or V.
template <int D, typename SRC, int KPT>
__global__ __launch_bounds__(256) void fp8_begin_kernel(DecArgs a, StoreArgs st, SelectArgs sel) {
  __shared__ union Smem {
    StoreSmem<D> st;
    SelectSmem<(KPT > 0 ? KPT : 1)> sel;
    __device__ Smem() {}
  } sm;
  if (blockIdx.x == 0) {
    plan_slices(a);
    return;
  }
  int i = blockIdx.x - 1;
  if constexpr (KPT > 0) {
    if (i < a.bs) {
      select_filter_block<KPT>(sel, i, sm.sel);
      return;
    }
    i -= a.bs;
  }
  const int tok = i / (2 * a.c.KV), rest = i - tok * 2 * a.c.KV;
  if (rest & 1) store_segment<D, SRC, true>(st, sm.st, tok, rest >> 1);
  else store_segment<D, SRC, false>(st, sm.st, tok, rest >> 1);
}

__device__ inline float trunc_bf16(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }
__device__ inline uint32_t pack_trunc(float even, float odd) {
  return __builtin_amdgcn_perm(__float_as_uint(odd), __float_as_uint(even), 0x07060302u);
}

// Eight codes as bf16.
__device__ inline bf16x8_t codes8(uint32_t a, uint32_t b) {
  u32x4_t w;
  w.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
  w.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
  w.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
  w.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
  return __builtin_bit_cast(bf16x8_t, w);
}

__device__ inline void store4(uint16_t* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2((uint32_t)f2bf(a) | ((uint32_t)f2bf(b) << 16),
                                            (uint32_t)f2bf(c) | ((uint32_t)f2bf(d) << 16));
}
__device__ inline void store4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}

// Channels d0 .. d0 + 7 of a query row as P bf16 pieces.
template <int P>
__device__ inline void load_query(const void* q, int64_t at, bool in, bf16x8_t (&f)[P]) {
  if constexpr (P == 1) {
    u32x4_t w = {0, 0, 0, 0};
    if (in) w = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(q) + at);
    f[0] = __builtin_bit_cast(bf16x8_t, w);
  } else {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = in ? static_cast<const float*>(q)[at + i] : 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      u32x4_t w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = pack_trunc(x[2 * i], x[2 * i + 1]);
        // what is left of an infinity is nothing (not NaN): its first piece says it all
        const float a = x[2 * i] - trunc_bf16(x[2 * i]), b = x[2 * i + 1] - trunc_bf16(x[2 * i + 1]);
        x[2 * i] = fabsf(x[2 * i]) == INFINITY ? 0.0f : a;
        x[2 * i + 1] = fabsf(x[2 * i + 1]) == INFINITY ? 0.0f : b;
      }
      f[p] = __builtin_bit_cast(bf16x8_t, w);
    }
  }
}

// What waves leave for the block to add up: slot 2 w of wave w for the request that goes on in its
// units, 2 w + 1 for the one that goes on behind them.
constexpr int kSlots = 2 * kDecWaves;
struct DecSmem {
  union {
    struct {
      float m[kSlots][kTile], l[kSlots][kTile];
      int32_t b[kSlots];      // request, or -1: nothing there
      int32_t c0[kSlots], c1[kSlots];
      int32_t ended[kSlots];  // its last unit is among them
    };
    struct {
      float w[kTile][kDecParts], sum[kTile];
      float4 red[64 * kDecWaves];
    } merge;
  };
  uint32_t last;
  float4 o[1];  // [kSlots][rows][D + 4] floats
};
constexpr int dec_row_floats(int D) { return D + 4; }
inline size_t dec_smem_bytes(int rows, int D) { return sizeof(DecSmem) + (size_t)kSlots * rows * dec_row_floats(D) * 4; }

// The parts of a request's tile added up, by the block that finished the last of them: a wave
// per query head and a lane per part for the weights, then a thread per 4 channels of a head,
// and where those are few, of every ng-th part.
template <int D, typename T>
__device__ inline void merge_parts(const DecArgs& a, DecSmem& sm, int head, int first, int parts, int rows, T* out) {
  constexpr int NT = 64 * kDecWaves;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  // row r of part i: of slice first + i, the part that begins its request there, or goes on in it
  auto row_of = [&](int i) { return ((first + i) * 2 + (i == 0 ? 1 : 0)) * a.heads + head; };
  const uint64_t* ml = reinterpret_cast<const uint64_t*>(a.part_ml);
  const int items = rows * (D / 4), ng = max(NT / items, 1);
  const int grp = items <= NT ? tid / items : 0;
  const int it0 = tid - grp * items;
  const __amdgpu_buffer_rsrc_t ro =
      agent_rsrc(a.part_o, (uint32_t)((int64_t)a.max_slices * 2 * a.heads * kTile * D * (int)sizeof(float)));
  // a batch of an item's parts; past the last part they re-read it.  The first go out before the
  // weights are known.  (Batches of 16 or 32: one request of 2000 tokens 15.5 -> 16.5, 17.3 us.)
  constexpr int kBatch = 8;
  float4 x[kBatch];
  auto load_parts = [&](int it, int i0) {
    const int r = it / (D / 4), d = (it - r * (D / 4)) * 4;
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      x[u] = ld_agent_x4(ro, (uint32_t)(((row_of(min(i0 + u * ng, parts - 1)) * kTile + r) * D + d) * (int)sizeof(float)));
  };
  load_parts(min(it0, items - 1), grp);
  for (int r = wave; r < rows; r += kDecWaves) {
    constexpr int kPer = (kDecParts + 63) / 64;
    float m[kPer], l[kPer], Mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = lane + 64 * i;
      const uint64_t e = p < parts ? ld_agent(ml + (int64_t)row_of(p) * kTile + r) : (uint64_t)0xFF800000u;  // (-inf, 0)
      m[i] = __uint_as_float((uint32_t)e);
      l[i] = __uint_as_float((uint32_t)(e >> 32));
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) Mx = fmaxf(Mx, m[i]);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) Mx = fmaxf(Mx, __shfl_xor(Mx, d, 64));
    float Ls = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float w = m[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[i] - Mx);
      Ls += l[i] != l[i] ? l[i] : w * l[i];
      sm.merge.w[r][lane + 64 * i] = w;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) Ls += __shfl_xor(Ls, d, 64);
    if (lane == 0) sm.merge.sum[r] = Ls;
  }
  lds_barrier();
  if (ng == 1 && grp > 0) return;  // threads past the items
  for (int it = it0; it < items; it += NT) {  // once where ng > 1
    const int r = it / (D / 4), d = (it - r * (D / 4)) * 4;
    float4 Os = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp < ng) {
      for (int i0 = grp; i0 < parts; i0 += kBatch * ng) {
        if (it != it0 || i0 != grp) load_parts(it, i0);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (i0 + u * ng >= parts) break;
          const float w = sm.merge.w[r][i0 + u * ng];
          Os.x += w * x[u].x;
          Os.y += w * x[u].y;
          Os.z += w * x[u].z;
          Os.w += w * x[u].w;
        }
      }
    }
    if (ng > 1) {  // block-uniform
      sm.merge.red[tid] = Os;
      __syncthreads();
      if (grp != 0) return;
      for (int g = 1; g < ng; ++g) {
        const float4 y = sm.merge.red[tid + g * items];
        Os.x += y.x;
        Os.y += y.y;
        Os.z += y.z;
        Os.w += y.w;
      }
    }
    const float Ls = sm.merge.sum[r];
    const float inv = Ls <= 0.0f ? 0.0f : 1.0f / Ls;
    store4(out + (int64_t)r * D + d, Os.x * inv, Os.y * inv, Os.z * inv, Os.w * inv);
  }
}

// The pages that request b attends, by a whole block of 64 * kDecWaves threads: in the scores' order
// into pages[0 .. k_sel).
template <int KPT>
__device__ inline void select_pages(const SelectArgs& sel, int b, RankSelectSmem<KPT, 64 * kDecWaves>& sm, int32_t* pages) {
  constexpr int NT = 64 * kDecWaves;
  const float* sc = sel.scores + (int64_t)b * sel.MP;
  float sv[KPT];
#pragma unroll
  for (int i = 0; i < KPT; ++i) sv[i] = sc[min((int)threadIdx.x + NT * i, sel.MP - 1)];
  const int64_t req = sel.rpi[b];
  const int lim = req >= 0 && req < sel.R ? min(sel.limit[b], sel.MP) : 0;
  int rank = -1, page = -1, row0 = -1;
  select_ranked<KPT, NT>(sv, lim, max(lim, sel.k_sel), sel.k_sel, sm, nullptr, sel.MP, rank, page, row0);
  if (threadIdx.x < 64 && rank >= 0 && rank < sel.k_sel) pages[rank] = page;
  lds_barrier();
}

// KPT > 0: the requests' pages are selected here, KPT scores a thread.
template <int D, typename T, int KPT>
__global__ __launch_bounds__(64 * kDecWaves, 2) void fp8_attend_kernel(DecArgs a, StoreArgs st, SelectArgs sel) {
  constexpr int QP = sizeof(T) == 2 ? 1 : 3, PP = 3;  // pieces of q and of the weights
  constexpr int KL = D / 64, VL = D / 16;  // 16-byte loads a lane: per 16 tokens of K, per block of V
  constexpr int RF = dec_row_floats(D);
  extern __shared__ __align__(16) unsigned char smem_raw[];
  DecSmem& sm = *reinterpret_cast<DecSmem*>(smem_raw);
  float* sm_o = reinterpret_cast<float*>(sm.o);
  const int head = blockIdx.x % a.heads, slice = blockIdx.x / a.heads;
  const DecPlan plan = *a.plan;
  const DecItem item = a.items[slice];  // both in one round trip; stale past the last slice
  const int h = head / a.tiles, tile = head - h * a.tiles;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int m16 = lane & 15, g = lane >> 4;
  const int rows = min(a.G - tile * kTile, kTile);  // query heads of this tile
  const int q_head = h * a.G + tile * kTile;
  if (plan.bs != a.bs || plan.top_k != a.top_k) {  // another batch's plan: no answer to any request
    const float nan = __builtin_nanf("");
    for (int b = slice; b < a.bs; b += a.max_slices)
      for (int i = tid; i < rows * (D / 4); i += 64 * kDecWaves)
        store4(static_cast<T*>(a.out) + ((int64_t)b * a.H + q_head) * D + i * 4, nan, nan, nan, nan);
    return;
  }
  if (slice >= plan.slices) return;
  const int at = slice * plan.len, end = min(at + plan.len, plan.total);
  // this wave's units
  const int s0 = at + (int)((int64_t)(end - at) * wave / kDecWaves), s1 = at + (int)((int64_t)(end - at) * (wave + 1) / kDecWaves);
  const int picked = a.top_k / 64 - 1;  // selected pages; the unit after them is the window
  if (lane < 2) sm.b[2 * wave + lane] = -1;
  // lengths or requests that have changed since the plan: no answer (0.25 us a layer)
  const bool stale = context_of(a, item.b) != item.seq || table_row(a, item.b) != item.req;

  // The selections of this slice's requests: a slice is no longer than one of them, so there are two
  // at most.
  __shared__ int32_t s_pages[KPT > 0 ? 2 : 1][64];
  int sel_first = -1;  // the first of the two
  // f(request lane, its units' begin, its context) of 64 requests from r0 on that begin in or before the slice
  auto each_64 = [&](auto f) {
    bool more = true;
    for (int r0 = item.b; more; r0 += 64) {
      const int r = r0 + lane;
      int c0 = 0x7FFFFFFF, seq = 0;
      if (r == item.b) {
        c0 = item.c0;
        seq = item.seq;
      } else if (end > item.c1 && r < a.bs) {
        c0 = a.cu[r];
        seq = context_of(a, r);
      }
      f(r0, c0, seq);
      more = __builtin_amdgcn_readlane(c0, 63) < end;
    }
  };
  if constexpr (KPT > 0) {
    auto& sm_sel = *reinterpret_cast<RankSelectSmem<KPT, 64 * kDecWaves>*>(sm.o);
    each_64([&](int r0, int c0, int seq) {
      for (uint64_t hits = __ballot(c0 < end && is_sparse(a, seq)); hits; hits &= hits - 1) {
        const int b = r0 + __builtin_ctzll(hits);
        select_pages<KPT>(sel, b, sm_sel, s_pages[sel_first >= 0 ? 1 : 0]);
        if (sel_first < 0) sel_first = b;
      }
    });
  }

  // New tokens of the requests that end among this wave's units, each in its request's last block,
  // which no other wave of this head reads.
  if (st.k && s1 >= item.c1) {
    bool more = true;
    for (int r0 = item.b; more; r0 += 64) {
      const int r = r0 + lane;
      int c1 = 0x7FFFFFFF;
      if (r == item.b) c1 = item.c1;
      else if (s1 > item.c1 && r < a.bs) c1 = a.cu[r + 1];
      for (uint64_t tails = __ballot(c1 > s0 && c1 <= s1); tails;) {
        int mine = -1;  // of the requests at hand, this lane group's
#pragma unroll
        for (int i = 0; i < 256 / D; ++i) {
          if (lane / (D / 4) == i && tails) mine = __builtin_ctzll(tails);
          tails &= tails - 1;  // (0 stays 0)
        }
        store_tokens<D>(st, r0 + mine, mine >= 0, h);
      }
      more = __builtin_amdgcn_readlane(c1, 63) < s1;
    }
    wait_memory();
  }

  // Of unit u0 + lane: its request, place in it, block and scales; a window has two blocks.  64 units
  // belong to 64 requests at most, from request rb on.
  int rb = item.b;
  int u_b = 0, u_c0 = 0, u_c1 = 0, u_seq = 0, blk = 0, blk2 = 0;
  bool u_bad = false;
  float ks = 0.0f, vs = 0.0f, ks2 = 0.0f, vs2 = 0.0f;
  auto resolve = [&](int u0) {
    const int u = u0 + lane, u_end = min(u0 + 64, s1);
    int row = item.req;
    if (rb == item.b && u_end <= item.c1) {  // all of them the slice's first request's
      u_b = rb;
      u_c0 = item.c0;
      u_c1 = item.c1;
      u_seq = item.seq;
    } else {
      int begins, ends;  // units of request rb + lane
      for (;;) {
        const int r = rb + lane;
        begins = r <= a.bs ? a.cu[r] : 0x7FFFFFFF;
        ends = r < a.bs ? a.cu[r + 1] : 0x7FFFFFFF;
        const int skip = __popcll(__ballot(begins <= u0)) - 1;  // those that begin before: a run of lanes from 0
        if (skip == 0) break;
        rb += skip;
      }
      const int r = rb + lane;
      const int my_seq = r < a.bs ? context_of(a, r) : 0, my_row = r < a.bs ? table_row(a, r) : -1;
      int i = 0;  // of the window's requests
      for (int x = 1; x < 64; ++x) {
        const int c = __builtin_amdgcn_readlane(begins, x);
        if (c >= u_end) break;
        i += u >= c ? 1 : 0;
      }
      u_b = rb + i;
      u_c0 = __shfl(begins, i, 64);
      u_seq = __shfl(my_seq, i, 64);
      row = __shfl(my_row, i, 64);
      u_c1 = __shfl(ends, i, 64);
    }
    blk = blk2 = 0;
    u_bad = row < 0 || (u_b == item.b ? stale : units_of(a, u_seq) != u_c1 - u_c0);
    const int32_t* tr = a.table + (int64_t)max(row, 0) * a.table_stride;
    auto block_at = [&](int page) {
      const int x = page >= 0 && page < a.table_cols ? tr[page] : 0;
      if (x > 0 && x < a.c.blocks) return x;
      u_bad = true;  // no block there: no answer
      return 0;
    };
    const bool sparse = is_sparse(a, u_seq), win = sparse && u - u_c0 == picked;
    if (u < u_end && u_seq > 0 && row >= 0) {
      const int place = u - u_c0;
      int page = place;
      if (win) page = (u_seq - 64) >> 6;
      else if (sparse) page = KPT > 0 ? s_pages[u_b == sel_first ? 0 : 1][place] : a.positions[(int64_t)u_b * a.pos_stride + place * 64] >> 6;
      blk = block_at(page);
      blk2 = win && (u_seq & 63) ? block_at(u_seq >> 6) : blk;
    }
    const int64_t e = (int64_t)blk * a.c.KV + h, e2 = (int64_t)blk2 * a.c.KV + h;
    ks = a.c.ks[e];
    vs = a.c.vs[e];
    if (a.top_k) {
      ks2 = a.c.ks[e2];
      vs2 = a.c.vs[e2];
    }
  };
  uint4 kr[4][KL], vr[VL];
  auto head_at = [&](int blocks, int j) {
    return ((int64_t)__builtin_amdgcn_readlane(blocks, j) * a.c.KV + h) * (64 * D) + lane * 16;
  };
  // K of lane j's unit: a window's tokens before place seq % 64 come from its second block
  auto load_k = [&](int j) {
    const uint8_t* p = a.c.kc + head_at(blk, j);
    const uint8_t* p2 = a.c.kc + head_at(blk2, j);
    const int from2 = __builtin_amdgcn_readlane(u_seq, j) & 63;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint8_t* pt = t * 16 + m16 < from2 ? p2 : p;
#pragma unroll
      for (int i = 0; i < KL; ++i) kr[t][i] = *reinterpret_cast<const uint4*>(pt + (t * KL + i) * 1024);
    }
  };
  auto load_v = [&](int blocks, int j, uint4* v) {
    const uint8_t* p = a.c.vc + head_at(blocks, j);
#pragma unroll
    for (int i = 0; i < VL; ++i) v[i] = *reinterpret_cast<const uint4*>(p + i * 1024);
  };
  bf16x8_t qf[2 * KL][QP];
  float4_t o[VL];
  float M = -INFINITY, L = 0.0f;
  bool bad = false;
  int first = s0;  // this request's first unit here
  auto load_q = [&](int b) {
#pragma unroll
    for (int i = 0; i < 2 * KL; ++i) {
      const int d = ((i >> 1) * 4 + g) * 16 + (i & 1) * 8;
      load_query<QP>(a.q, (int64_t)b * a.q_bstride + (int64_t)(q_head + min(m16, rows - 1)) * D + d, m16 < rows, qf[i]);
    }
  };
  // loads come back in order: the queries before the keys, the keys before the values
  if (s0 < s1) {
    resolve(s0);
    load_q(__builtin_amdgcn_readlane(u_b, 0));
    load_k(0);
    load_v(blk, 0, vr);
  }
  for (int u = s0; u < s1; ++u) {
    const int j = (u - s0) & 63;
    const int b = __builtin_amdgcn_readlane(u_b, j), c0 = __builtin_amdgcn_readlane(u_c0, j), c1 = __builtin_amdgcn_readlane(u_c1, j);
    const int seq = __builtin_amdgcn_readlane(u_seq, j);
    if (u == s0 || u == c0) {  // a request begins here
      first = u;
#pragma unroll
      for (int i = 0; i < VL; ++i) o[i] = float4_t{0.f, 0.f, 0.f, 0.f};
      M = -INFINITY;
      L = 0.0f;
      bad = false;
    }
    const bool sparse = is_sparse(a, seq), win = sparse && u - c0 == picked;
    const int hi = sparse ? 64 : min(64, seq - (u - c0) * 64);  // tokens of this unit
    const float kscale = __shfl(ks, j, 64) * a.sl2, vscale = __shfl(vs, j, 64);
    const float kscale2 = win ? __shfl(ks2, j, 64) * a.sl2 : kscale, vscale2 = win ? __shfl(vs2, j, 64) : vscale;
    bad |= (bool)__builtin_amdgcn_readlane((int)u_bad, j);
    const bool last = u + 1 >= s1, next_set = j == 63;
    float4_t s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const bf16x8_t k0 = codes8(kr[t][i].x, kr[t][i].y), k1 = codes8(kr[t][i].z, kr[t][i].w);
#pragma unroll
        for (int p = 0; p < QP; ++p) {
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qf[2 * i][p], s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qf[2 * i + 1][p], s[t], 0, 0, 0);
        }
      }
    }
    if (!last && u + 1 == c1) load_q(b + 1);
    // the next unit's K under this one's softmax and values; a window's second V goes there instead
    if (win) load_v(blk2, j, &kr[0][0]);
    else if (!last && !next_set) load_k(j + 1);
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = t * 16 + g * 4 + i;
        s[t][i] = tok < hi ? s[t][i] * (tok < (seq & 63) ? kscale2 : kscale) : -INFINITY;
        mx = fmaxf(mx, s[t][i]);
      }
    mx = fmaxf(mx, lane_xor16(mx, lane));
    mx = fmaxf(mx, lane_xor32(mx, lane));
    const float Mn = fmaxf(M, mx);
    const float mb = Mn == -INFINITY ? 0.0f : Mn;
    const float alpha = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - mb);
    M = Mn;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(s[t][i] - mb);
        sum += p;
        // a masked token weighs nothing whatever its block's scale is
        s[t][i] = s[t][i] == -INFINITY ? 0.0f : p * (t * 16 + g * 4 + i < (seq & 63) ? vscale2 : vscale);
      }
    if (win) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int from2 = min(max((seq & 63) - t * 16 - g * 4, 0), 4);  // of the word's four tokens
        const uint32_t mask = from2 >= 4 ? 0xFFFFFFFFu : (1u << (8 * from2)) - 1u;
#pragma unroll
        for (int i = 0; i < VL; ++i) {
          uint32_t& w = reinterpret_cast<uint32_t*>(&vr[i])[t];
          w = (reinterpret_cast<const uint32_t*>(&kr[0][0])[i * 4 + t] & mask) | (w & ~mask);
        }
      }
    }
    L = L * alpha + sum;
#pragma unroll
    for (int i = 0; i < VL; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[i][x] *= alpha;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      bf16x8_t pw[PP];
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        u32x4_t w;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float e = s[2 * st + (x >> 1)][(x & 1) * 2], f = s[2 * st + (x >> 1)][(x & 1) * 2 + 1];
          w[x] = pack_trunc(e, f);
          s[2 * st + (x >> 1)][(x & 1) * 2] = e - trunc_bf16(e);
          s[2 * st + (x >> 1)][(x & 1) * 2 + 1] = f - trunc_bf16(f);
        }
        pw[p] = __builtin_bit_cast(bf16x8_t, w);
      }
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const uint32_t x[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
        const bf16x8_t vb = codes8(x[2 * st], x[2 * st + 1]);
#pragma unroll
        for (int p = 0; p < PP; ++p) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb, pw[p], o[i], 0, 0, 0);
      }
    }
    if (!last) {
      if (next_set) resolve(u + 1);
      if (next_set || win) load_k(next_set ? 0 : j + 1);
      load_v(blk, next_set ? 0 : j + 1, vr);
    }
    if (!last && u + 1 < c1) continue;
    // the request's units here are done
    float l = L + lane_xor16(L, lane);
    l += lane_xor32(l, lane);
    if (bad) l = __builtin_nanf("");
    const bool began = first == c0, ended = u + 1 == c1;
    if (began && ended) {
      const float inv = l <= 0.0f ? 0.0f : 1.0f / l;  // nothing attended: zeros
      if (m16 < rows) {
        T* out = static_cast<T*>(a.out) + ((int64_t)b * a.H + q_head + m16) * D + g * 4;
#pragma unroll
        for (int i = 0; i < VL; ++i) store4(out + i * 16, o[i][0] * inv, o[i][1] * inv, o[i][2] * inv, o[i][3] * inv);
      }
      continue;
    }
    const int slot = 2 * wave + (began ? 1 : 0);
    if (lane == 0) {
      sm.b[slot] = b;
      sm.c0[slot] = c0;
      sm.c1[slot] = c1;
      sm.ended[slot] = ended;
    }
    if (g == 0) {
      sm.m[slot][m16] = M;
      sm.l[slot][m16] = l;
    }
    if (m16 < rows) {
#pragma unroll
      for (int i = 0; i < VL; ++i) *reinterpret_cast<float4_t*>(sm_o + (slot * rows + m16) * RF + i * 16 + g * 4) = o[i];
    }
  }
  if constexpr (KPT > 0) {  // the layout of the requests that begin here, for those who read it
    if (head == 0)
      each_64([&](int r0, int c0, int seq) {
        const uint64_t long_ones = __ballot(is_sparse(a, seq));
        for (uint64_t hits = __ballot(c0 >= at && c0 < end); hits; hits &= hits - 1) {
          const int i = __builtin_ctzll(hits), b = r0 + i;
          int32_t* pos = sel.positions + (int64_t)b * sel.top_k;
          if (!(long_ones >> i & 1)) {
            write_dense(pos, a.seq[b], sel.top_k);
            continue;
          }
          const int32_t* pages = s_pages[b == sel_first ? 0 : 1];
          for (int slot = tid; slot < sel.k_sel * 64; slot += 64 * kDecWaves) pos[slot] = pages[slot >> 6] * 64 + (slot & 63);
          write_recent(pos + (int64_t)sel.k_sel * 64, a.seq[b], 64);
        }
      });
  }
  __syncthreads();
  // The requests that more than one wave has, or that go on in another slice: their slots follow one
  // another, from the one where the request begins here to the one where it ends (or the slice).
  const int sl = lane & (kSlots - 1);
  const int sl_b = sm.b[sl], sl_c0 = sm.c0[sl], sl_c1 = sm.c1[sl];
  uint32_t left = (uint32_t)__ballot(sl_b >= 0) & ((1u << kSlots) - 1u);
  const uint32_t ends = (uint32_t)__ballot(sm.ended[sl] != 0) & left;
  bool handed = false;
  int next_b = -1, next_c0 = 0, next_c1 = 0;  // the request that goes on in the next slice
  while (left) {
    const int f = __builtin_ctz(left);
    const uint32_t stop = ends & ~((1u << f) - 1u);
    const bool ended = stop != 0;
    const uint32_t mask = ended ? left & ((2u << __builtin_ctz(stop)) - 1u) : left;
    left &= ~mask;
    const int b = __builtin_amdgcn_readlane(sl_b, f), c0 = __builtin_amdgcn_readlane(sl_c0, f), c1 = __builtin_amdgcn_readlane(sl_c1, f);
    const bool whole = c0 >= at && ended;
    T* out = static_cast<T*>(a.out) + ((int64_t)b * a.H + q_head) * D;
    const int part = ((slice * 2 + (c0 >= at ? 1 : 0)) * a.heads + head) * kTile;
    const __amdgpu_buffer_rsrc_t po = agent_rsrc(a.part_o + (int64_t)part * D, (uint32_t)(kTile * D * sizeof(float)));
    for (int it = tid; it < rows * (D / 4); it += 64 * kDecWaves) {
      const int r = it / (D / 4), d = (it - r * (D / 4)) * 4;
      float Mx = -INFINITY, Ls = 0.0f;
      for (uint32_t left_w = mask; left_w; left_w &= left_w - 1) Mx = fmaxf(Mx, sm.m[__builtin_ctz(left_w)][r]);
      float4 Os = make_float4(0.f, 0.f, 0.f, 0.f);
      for (uint32_t left_w = mask; left_w; left_w &= left_w - 1) {
        const int w = __builtin_ctz(left_w);
        const float wt = sm.m[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm.m[w][r] - Mx);
        const float lw = sm.l[w][r];
        Ls += lw != lw ? lw : wt * lw;
        const float4 x = *reinterpret_cast<const float4*>(sm_o + (w * rows + r) * RF + d);
        Os.x += wt * x.x;
        Os.y += wt * x.y;
        Os.z += wt * x.z;
        Os.w += wt * x.w;
      }
      if (whole) {
        const float inv = Ls <= 0.0f ? 0.0f : 1.0f / Ls;
        store4(out + (int64_t)r * D + d, Os.x * inv, Os.y * inv, Os.z * inv, Os.w * inv);
      } else {
        st_agent_x4(po, (uint32_t)((r * D + d) * sizeof(float)), Os);
        if (d == 0) {
          st_agent(a.part_ml + (int64_t)(part + r) * 2, Mx);
          st_agent(a.part_ml + (int64_t)(part + r) * 2 + 1, Ls);
        }
      }
    }
    handed |= !whole;
    if (c0 >= at && !ended) {
      next_b = b;
      next_c0 = c0;
      next_c1 = c1;
    }
  }
  if (!handed) return;
  // parts handed out: of the request that comes from the slice before, and of the one that goes on in
  // the next; the block that finishes a request's last part adds them up
  wait_memory();
  for (int x = 0; x < 2; ++x) {
    const int b = x ? next_b : item.c0 < at ? item.b : -1;
    if (b < 0) continue;  // block-uniform
    const int c0 = x ? next_c0 : item.c0, c1 = x ? next_c1 : item.c1;
    const int first_slice = c0 / plan.len, parts = (c1 - 1) / plan.len - first_slice + 1;
    __syncthreads();
    if (tid == 0) {
      uint32_t* done = &a.done[first_slice * a.heads + head];
      sm.last = add_agent(done, 1u) == (uint32_t)parts - 1;
      if (sm.last) st_agent(done, 0u);  // for the step's next layer
    }
    __syncthreads();
    if (sm.last)
      merge_parts<D, T>(a, sm, head, first_slice, parts, rows, static_cast<T*>(a.out) + ((int64_t)b * a.H + q_head) * D);
  }
}

template <int D, int KPT>
void begin(const DecArgs& a, const StoreArgs& st, const SelectArgs& sel, hipStream_t s) {
  const unsigned blocks = 1 + (KPT > 0 ? a.bs : 0) + (st.k ? 2u * a.bs * a.c.KV : 0);
  if (st.dtype == QQ_DTYPE_BF16) fp8_begin_kernel<D, uint16_t, KPT><<<blocks, 256, 0, s>>>(a, st, sel);
  else fp8_begin_kernel<D, float, KPT><<<blocks, 256, 0, s>>>(a, st, sel);
}

// LDS past the 64 KiB default (tiles of more than 15 heads of 128, large selections): opted in once
// per device.
template <int D, typename T, int KPT>
void attend(const DecArgs& a, const StoreArgs& st, const SelectArgs& sel, hipStream_t s) {
  size_t bytes = dec_smem_bytes(min(a.G, kTile), D);
  if (KPT > 0) bytes = max(bytes, sizeof(DecSmem) + sizeof(RankSelectSmem<(KPT > 0 ? KPT : 1), 64 * kDecWaves>));
  if (bytes > 60 * 1024) {
    static bool opted[64] = {false};
    int dev = 0;
    if (hipGetDevice(&dev) == hipSuccess && dev >= 0 && dev < 64 && !opted[dev]) {
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&fp8_attend_kernel<D, T, KPT>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)max(dec_smem_bytes(kTile, D), bytes));
      opted[dev] = true;
    }
  }
  fp8_attend_kernel<D, T, KPT><<<a.max_slices * a.heads, 64 * kDecWaves, bytes, s>>>(a, st, sel);
}

constexpr int kBeginPages = 16 * 256;  // pages that a begin launch selects of, at most

// `sel`: with k_sel > 0 the pages are selected first, from scores that are there.  planned: the
// workspace holds the slices, and nothing of another head tile waits for the new tokens.
template <int D>
void launch(const DecArgs& a, const StoreArgs& st, const SelectArgs& sel, bool planned, int q_dtype, hipStream_t s) {
  const int n = max(sel.MP, sel.k_sel);
  StoreArgs in{};  // what is left to store for the attention
  if (planned) in = st;
  else if (!sel.positions) begin<D, 0>(a, st, sel, s);
  else if (sel.k_sel <= 64 && n <= 4 * 256) begin<D, 4>(a, st, sel, s);
  else if (sel.k_sel <= 64 && n <= 9 * 256) begin<D, 9>(a, st, sel, s);
  else if (sel.k_sel <= 64 && n <= kBeginPages) begin<D, 16>(a, st, sel, s);
  else {
    launch_select(sel, a.bs, sel.MP, sel.k_sel, s);
    begin<D, 0>(a, st, sel, s);
  }
  if (q_dtype == QQ_DTYPE_BF16) attend<D, uint16_t, 0>(a, in, sel, s);
  else attend<D, float, 0>(a, in, sel, s);
}

// Whether a planned step of Quest runs as two launches: the scores with the new tokens, and an
// attention that selects by itself.  A slice must not be longer than a request's selection (at
// most as many requests as the grid has slices, and 8 units, fp8_slice_len's least), so that a block
// selects for two requests at most.
//
// Every block of a request repeats its selection, which is dear once more than a wave's 64 pages pass
// its filter (the k-th largest of 64 groups' maxima: 64 ln(64 / (64 - k)) pages, 64 of them from
// k = 40 on), where a launch for it does it once: two launches are taken up to that, and past the 4096
// pages that a begin launch can select of, which takes four.  A layer-step in two launches and in
// three, us, 32 heads on 4, contexts of 32768 tokens unless said: 1 request, 31 pages 16.6, 18.9; 12:
// 26.4, 28.1; 40: 43.3, 45.4; 63: 47.7, 51.4; 12 of 131072: 33.7, 35.5; 40 pages, 1 request 17.1, 19.9; 7:
// 24.9, 26.5; 63: 56.5, 58.9; 42 pages, 7 requests 28.4, 26.6; 63 pages, 1: 24.9, 23.2; 64 pages, 16: 53.9,
// 46.7.  In tables of 4097 pages: 44 pages, 1 of 262144 tokens 22.9, 52.0; 64 pages, 12: 44.1, 52.5; 63:
// 107, 104.
bool selects_itself(const DecArgs& a, const SelectArgs& sel, int q_dtype) {
  const int n = max(sel.MP, sel.k_sel);
  return q_dtype == QQ_DTYPE_BF16 && a.c.D == 128 && a.tiles == 1 && a.bs <= a.max_slices && sel.top_k >= 8 * 64 &&
         sel.k_sel <= (n <= kBeginPages ? 40 : 64) && sel.MP > 0 && n <= 16 * 64 * kDecWaves &&
         (int64_t)a.table_cols * kCacheTokens > sel.top_k;
}

void launch_selecting(DecArgs a, const SelectArgs& sel, hipStream_t s) {
  const int n = max(sel.MP, sel.k_sel);
  constexpr int NT = 64 * kDecWaves;
  a.positions = nullptr;
  const StoreArgs none{};
  if (n <= NT) attend<128, uint16_t, 1>(a, none, sel, s);
  else if (n <= 2 * NT) attend<128, uint16_t, 2>(a, none, sel, s);
  else if (n <= 5 * NT) attend<128, uint16_t, 5>(a, none, sel, s);
  else attend<128, uint16_t, 16>(a, none, sel, s);
}

// Everything of a call but its launches; `what` refuses.
int set_args(DecArgs& a, StoreArgs& st, const char* what, const void* q, int q_dtype, int64_t q_batch_stride,
             int num_q_heads, const void* k_new, const void* v_new, int new_dtype, const int64_t* out_cache_loc,
             const Fp8Cache& c, const int32_t* block_table, int64_t block_table_stride, int block_table_rows,
             int block_table_cols, const int64_t* req_pool_indices, const int64_t* seq_lens, int bs,
             const int32_t* positions, int64_t positions_stride, int top_k, float scale, void* out, void* workspace,
             int64_t workspace_bytes) {
  const int ok = check_cache(c, what);
  if (ok != QQ_OK) return ok;
  QQ_REQUIRE(dtype_ok(q_dtype), "%s: bad dtype", what);
  QQ_REQUIRE(num_q_heads > 0 && num_q_heads % c.KV == 0 && num_q_heads < 65536,
             "%s: q_heads %d not divisible by kv_heads %d", what, num_q_heads, c.KV);
  QQ_REQUIRE(bs >= 0 && block_table_rows > 0 && block_table_cols > 0 && block_table_cols <= kMaxPoolBlocks &&
                 block_table_stride >= block_table_cols,
             "%s: bad sizes", what);
  QQ_REQUIRE(!positions || (top_k > 0 && top_k % 64 == 0 && positions_stride >= top_k),
             "%s: top_k %d is not a multiple of the block of 64", what, top_k);
  QQ_REQUIRE((int64_t)block_table_cols * bs < (int64_t)1 << 30, "%s: too many units of work", what);
  if (bs == 0) return QQ_OK;
  QQ_REQUIRE(q && block_table && req_pool_indices && seq_lens && out, "%s: null pointer", what);
  QQ_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && q_batch_stride % 8 == 0,
             "%s: q and out must be 16-byte aligned", what);
  QQ_REQUIRE(!k_new || (v_new && out_cache_loc), "%s: null pointer", what);
  QQ_REQUIRE(!k_new || dtype_ok(new_dtype), "%s: bad dtype", what);
  QQ_REQUIRE(((uintptr_t)k_new | (uintptr_t)v_new) % 16 == 0, "%s: k_new and v_new must be 16-byte aligned", what);
  QQ_REQUIRE(!k_new || (int64_t)bs * c.KV < (int64_t)1 << 29, "%s: bad sizes", what);
  const DecSpace sp = decode_space(bs, num_q_heads, c.KV, c.D);
  QQ_REQUIRE(workspace && workspace_bytes >= sp.bytes, "%s: workspace %lld bytes < %lld needed", what,
             (long long)workspace_bytes, (long long)sp.bytes);
  char* ws = static_cast<char*>(workspace);
  a.q = q;
  a.q_bstride = q_batch_stride;
  a.H = num_q_heads;
  a.G = num_q_heads / c.KV;
  a.tiles = (a.G + kTile - 1) / kTile;
  a.c = c;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.positions = positions;
  a.pos_stride = positions_stride;
  a.sl2 = scale * kLog2e;
  a.out = out;
  set_plan(a, sp, ws, req_pool_indices, seq_lens, bs, block_table_rows, block_table_cols, positions ? top_k : 0, c.KV * a.tiles);
  a.part_o = reinterpret_cast<float*>(ws + sp.part_o);
  a.part_ml = reinterpret_cast<float*>(ws + sp.part_ml);
  st = StoreArgs{c, k_new, v_new, new_dtype, out_cache_loc, bs, 1};
  return QQ_OK;
}

}  // namespace
}  // namespace qq

using namespace qq;

extern "C" int64_t qq_fp8_decode_workspace_bytes(int bs, int num_q_heads, int kv_heads, int head_dim) {
  if (bs <= 0 || kv_heads <= 0 || num_q_heads < kv_heads || num_q_heads % kv_heads || !fp8_dim_ok(head_dim)) return 0;
  return decode_space(bs, num_q_heads, kv_heads, head_dim).bytes;
}

extern "C" int qq_fp8_decode_attention(const void* q, int q_dtype, int64_t q_batch_stride, int num_q_heads,
                                       const void* k_new, const void* v_new, int new_dtype, const int64_t* out_cache_loc,
                                       uint8_t* k_codes, uint8_t* v_codes, float* k_scale, float* v_scale,
                                       int num_blocks, int kv_heads, int head_dim, const int32_t* block_table,
                                       int64_t block_table_stride, int block_table_rows, int block_table_cols,
                                       const int64_t* req_pool_indices, const int64_t* seq_lens, int bs,
                                       const int32_t* positions, int64_t positions_stride, int top_k, float scale,
                                       void* out, void* workspace, int64_t workspace_bytes, int planned,
                                       void* stream) {
  const char* what = "qq_fp8_decode_attention";
  DecArgs a{};
  StoreArgs st{};
  const int ok = set_args(a, st, what, q, q_dtype, q_batch_stride, num_q_heads, k_new, v_new, new_dtype, out_cache_loc,
                          {k_codes, v_codes, k_scale, v_scale, num_blocks, kv_heads, head_dim}, block_table,
                          block_table_stride, block_table_rows, block_table_cols, req_pool_indices, seq_lens, bs, positions,
                          positions_stride, top_k, scale, out, workspace, workspace_bytes);
  if (ok != QQ_OK || bs == 0) return ok;
  QQ_REQUIRE(!planned || !positions, "%s: a plan is of whole contexts, not of selected pages", what);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool one = planned && a.tiles == 1;
  if (head_dim == 128) launch<128>(a, st, SelectArgs{}, one, q_dtype, s);
  else launch<64>(a, st, SelectArgs{}, one, q_dtype, s);
  return check_launch(what);
}

extern "C" int qq_fp8_decode_plan(int num_blocks, int kv_heads, int head_dim, int block_table_rows, int block_table_cols,
                                  const int64_t* req_pool_indices, const int64_t* seq_lens, int bs, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const char* what = "qq_fp8_decode_plan";
  // what the slices do not depend on stands in for itself
  uint8_t* any = reinterpret_cast<uint8_t*>(workspace);
  float* any_scale = static_cast<float*>(workspace);
  DecArgs a{};
  StoreArgs st{};
  QQ_REQUIRE(bs <= 0 || workspace, "%s: null pointer", what);
  if (bs == 0) return QQ_OK;
  const int ok = set_args(a, st, what, any, QQ_DTYPE_BF16, 0, kv_heads, nullptr, nullptr, QQ_DTYPE_BF16, nullptr,
                          {any, any, any_scale, any_scale, num_blocks, kv_heads, head_dim},
                          static_cast<const int32_t*>(workspace), block_table_cols, block_table_rows, block_table_cols,
                          req_pool_indices, seq_lens, bs, nullptr, 0, 0, 1.0f, workspace, workspace, workspace_bytes);
  if (ok != QQ_OK) return ok;
  fp8_plan_kernel<<<1, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  return check_launch(what);
}

extern "C" int qq_fp8_quest_step(const void* q, int q_dtype, int64_t q_batch_stride, int num_q_heads, const void* k_new,
                                 const void* v_new, int new_dtype, const int64_t* out_cache_loc, uint8_t* k_codes,
                                 uint8_t* v_codes, float* k_scale, float* v_scale, int num_blocks, int kv_heads,
                                 int head_dim, const int32_t* block_table, int64_t block_table_stride,
                                 int block_table_rows, int block_table_cols, const uint16_t* page_k_bounds, int layer,
                                 const int64_t* req_pool_indices, const int64_t* seq_lens, const int32_t* candidate_limit,
                                 int bs, int max_reqs, int max_pages, int top_k, float scale, float* scores_ws,
                                 int32_t* positions, void* out, void* workspace, int64_t workspace_bytes, int phase,
                                 int planned, void* stream) {
  const char* what = "qq_fp8_quest_step";
  QQ_REQUIRE(phase >= 1 && phase <= 3, "%s: phase must be 1, 2 or 3, got %d", what, phase);
  QQ_REQUIRE(bs == 0 || (page_k_bounds && candidate_limit && scores_ws && positions), "%s: null pointer", what);
  QQ_REQUIRE(layer >= 0 && max_reqs > 0 && max_pages >= 0, "%s: bad sizes", what);
  DecArgs a{};
  StoreArgs st{};
  const int ok = set_args(a, st, what, q, q_dtype, q_batch_stride, num_q_heads, k_new, v_new, new_dtype, out_cache_loc,
                          {k_codes, v_codes, k_scale, v_scale, num_blocks, kv_heads, head_dim}, block_table,
                          block_table_stride, block_table_rows, block_table_cols, req_pool_indices, seq_lens, bs, positions,
                          top_k, top_k, scale, out, workspace, workspace_bytes);
  if (ok != QQ_OK || bs == 0) return ok;
  const int C = kv_heads * head_dim, k_sel = top_k / 64 - 1;
  QQ_REQUIRE(C <= kMaxC, "%s: kv_heads*head_dim %d exceeds %d", what, C, kMaxC);
  QQ_REQUIRE(k_sel <= 1024, "%s: %d selected pages exceed 1024", what, k_sel);
  SelectArgs sel{};
  sel.q = q;
  sel.q_dtype = q_dtype;
  sel.q_bstride = q_batch_stride;
  sel.H = num_q_heads;
  sel.bounds_layer = reinterpret_cast<const uint32_t*>(page_k_bounds) + (int64_t)layer * max_reqs * max_pages * C;
  sel.rpi = req_pool_indices;
  sel.seq = seq_lens;
  sel.limit = candidate_limit;
  sel.R = max_reqs;
  sel.MP = max_pages;
  sel.KV = kv_heads;
  sel.D = head_dim;
  sel.C = C;
  sel.m = (C + 63) / 64;
  sel.P = 64;
  sel.top_k = top_k;
  sel.k_sel = k_sel;
  sel.ppb = 32;
  sel.scores = scores_ws;
  sel.positions = positions;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (planned && phase == 3 && selects_itself(a, sel, q_dtype)) {
    const int scored = launch_score_codes(sel, bs, a.c, k_new, v_new, new_dtype, out_cache_loc, s);
    if (scored < 0) return scored;
    if (scored == QQ_OK) {
      launch_selecting(a, sel, s);
      return check_launch(what);
    }
  }
  if (phase == 1) return launch_retrieve(sel, bs, s);
  if (phase == 3) {
    const int scored = launch_score(sel, bs, false, s);
    if (scored != QQ_OK) return scored;
  } else {
    sel = SelectArgs{};  // phase 1 left the positions
  }
  if (head_dim == 128) launch<128>(a, st, sel, false, q_dtype, s);
  else launch<64>(a, st, sel, false, q_dtype, s);
  return check_launch(what);
}
