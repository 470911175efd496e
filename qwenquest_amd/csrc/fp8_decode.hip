// Decode attention over the 8-bit K/V cache (layout: qq_fp8.h), dense or over the pages that
// Quest selected (reference src/qwenquest/attention/dense.py:26-42, quest_only.py:132-159,
// ops.py:48-66 over that cache).  With ks, vs the scales of token j's block and kc, vc its codes
//   t_j = scale * log2(e) * ks * (q . kc_j),  p_j = 2^(t_j - max t),  out = sum p_j vs vc_j / sum p_j.
//
// The division of the work and the kernels' frame are qq_decode_dev.h's; a unit's codes are 1 KiB runs
// a load.  A layer of Quest stores beside the page scores (a selected page may be the one that is
// written) and selects in the attention, at shapes where that costs less than a launch (selects_itself).
//
// P's values scaled by vs go in as three bf16 pieces, which hold all 24
// significand bits (in two pieces, 16 bits, bf16 outputs were off by a step in a few of a thousand places,
// for 2 us less of 145 in 12 layers of one request of 2000 tokens).
// Bound: HBM, the codes once, when they are many: 16 requests of 131072 tokens, 4 heads of 128,
// 379 us (5.7 TB/s; matrix pipes 18 % busy, vector units 44 %).  A small batch is bound by its chain
// of memory round trips (slice, table words, scales and codes, partials, count, merge, ~1 us each):
// one request of 2000 tokens 11.4 us a layer, of which its waves wait 80 %; 15.8 in two launches; the
// plan 4.6 us a step.  16 requests' 31 pages and window of 131072 tokens 18.1 us with the selection
// (waiting 54 %), 16.1 behind a begin launch of 5.4.
#include "qq_decode_dev.h"
#include "qq_fp8_store.h"

namespace qq {
namespace {

// Eight codes as bf16.
__device__ inline bf16x8_t codes8(uint32_t a, uint32_t b) {
  u32x4_t w;
  w.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
  w.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
  w.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
  w.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
  return __builtin_bit_cast(bf16x8_t, w);
}

template <int D>
struct Fp8Unit {
  using Cache = Fp8Cache;
  using Store = StoreArgs;
  using BeginSmem = StoreSmem<D>;
  static constexpr int kDim = D;
  static constexpr bool kOneFactor = false;  // a block's scale is one
  static constexpr bool kStoresSelecting = false;
  static constexpr int KL = D / 64, VL = D / 16;  // 16-byte loads a lane: per 16 tokens of K, per block of V
  float ks = 0.0f, vs = 0.0f, ks2 = 0.0f, vs2 = 0.0f;  // of this lane's unit
  float kscale, vscale, kscale2, vscale2;              // of the unit at hand
  uint4 kr[4][KL], vr[VL];

  static __device__ inline int channel(int i, int g) { return ((i >> 1) * 4 + g) * 16 + (i & 1) * 8; }
  __device__ inline void look_up(const Fp8Cache& c, int h, int blk, int blk2, bool two) {
    const int64_t e = (int64_t)blk * c.KV + h, e2 = (int64_t)blk2 * c.KV + h;
    ks = c.ks[e];
    vs = c.vs[e];
    if (two) {
      ks2 = c.ks[e2];
      vs2 = c.vs[e2];
    }
  }
  static __device__ inline int64_t head_at(const Fp8Cache& c, int h, int lane, int blk) {
    return ((int64_t)blk * c.KV + h) * (64 * D) + lane * 16;
  }
  __device__ inline void load_k(const Fp8Cache& c, int h, int lane, int blk, int blk2, int from2) {
    const uint8_t* p = c.kc + head_at(c, h, lane, blk);
    const uint8_t* p2 = c.kc + head_at(c, h, lane, blk2);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint8_t* pt = t * 16 + (lane & 15) < from2 ? p2 : p;
#pragma unroll
      for (int i = 0; i < KL; ++i) kr[t][i] = *reinterpret_cast<const uint4*>(pt + (t * KL + i) * 1024);
    }
  }
  __device__ inline void load_values(const Fp8Cache& c, int h, int lane, int blk, uint4* v) {
    const uint8_t* p = c.vc + head_at(c, h, lane, blk);
#pragma unroll
    for (int i = 0; i < VL; ++i) v[i] = *reinterpret_cast<const uint4*>(p + i * 1024);
  }
  __device__ inline void load_v(const Fp8Cache& c, int h, int lane, int blk) { load_values(c, h, lane, blk, vr); }
  __device__ inline void load_window_v(const Fp8Cache& c, int h, int lane, int blk2) { load_values(c, h, lane, blk2, &kr[0][0]); }
  __device__ inline void begin(int j, bool win, float sl2) {
    kscale = __shfl(ks, j, 64) * sl2, vscale = __shfl(vs, j, 64);
    kscale2 = win ? __shfl(ks2, j, 64) * sl2 : kscale, vscale2 = win ? __shfl(vs2, j, 64) : vscale;
  }
  __device__ inline void keys(int t, int i, bf16x8_t& k0, bf16x8_t& k1) const {
    k0 = codes8(kr[t][i].x, kr[t][i].y), k1 = codes8(kr[t][i].z, kr[t][i].w);
  }
  __device__ inline float score(int tok, int from2) const { return tok < from2 ? kscale2 : kscale; }
  __device__ inline float weight(int, int, int tok, int from2) const { return tok < from2 ? vscale2 : vscale; }
  __device__ inline void merge_window(int from2, int g) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int in2 = min(max(from2 - t * 16 - g * 4, 0), 4);  // of the word's four tokens
      const uint32_t mask = in2 >= 4 ? 0xFFFFFFFFu : (1u << (8 * in2)) - 1u;
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        uint32_t& w = reinterpret_cast<uint32_t*>(&vr[i])[t];
        w = (reinterpret_cast<const uint32_t*>(&kr[0][0])[i * 4 + t] & mask) | (w & ~mask);
      }
    }
  }
  static constexpr int tile_of(int st, int x, int) { return 2 * st + (x >> 1); }
  static constexpr int place_of(int x, int y) { return (x & 1) * 2 + y; }
  __device__ inline bf16x8_t values(int i, int st) const {
    const uint32_t x[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
    return codes8(x[2 * st], x[2 * st + 1]);
  }

  static __device__ inline void store_tokens(const StoreArgs& st, int64_t i, bool on, int h) { qq::store_tokens<D>(st, i, on, h); }
  // a block per new token, head, and K or V
  static unsigned begin_blocks(const StoreArgs& st) { return 2u * (unsigned)st.n * st.c.KV; }
  template <typename SRC>
  static __device__ inline void begin_store(const StoreArgs& st, BeginSmem& sm, int i) {
    const int tok = i / (2 * st.c.KV), rest = i - tok * 2 * st.c.KV;
    if (rest & 1) store_segment<D, SRC, true>(st, sm, tok, rest >> 1);
    else store_segment<D, SRC, false>(st, sm, tok, rest >> 1);
  }
};

// Where a layer selects in its attention (selects_itself): a layer-step in two launches and in
// three, us, 32 heads on 4, contexts of 32768 tokens unless said: 1 request, 31 pages 16.6, 18.9; 12:
// 26.4, 28.1; 40: 43.3, 45.4; 63: 47.7, 51.4; 12 of 131072: 33.7, 35.5; 40 pages, 1 request 17.1, 19.9; 7:
// 24.9, 26.5; 63: 56.5, 58.9; 42 pages, 7 requests 28.4, 26.6; 63 pages, 1: 24.9, 23.2; 64 pages, 16: 53.9,
// 46.7.  In tables of 4097 pages: 44 pages, 1 of 262144 tokens 22.9, 52.0; 64 pages, 12: 44.1, 52.5; 63:
// 107, 104.
constexpr int kSelfPages = 40;

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
  DecArgs<Fp8Cache> a{};
  StoreArgs st{};
  const int ok = set_args(a, st, what, q, q_dtype, q_batch_stride, num_q_heads, k_new, v_new, new_dtype, out_cache_loc,
                          Fp8Cache{k_codes, v_codes, k_scale, v_scale, num_blocks, kv_heads, head_dim}, block_table,
                          block_table_stride, block_table_rows, block_table_cols, req_pool_indices, seq_lens, bs, positions,
                          positions_stride, top_k, scale, out, workspace, workspace_bytes);
  if (ok != QQ_OK || bs == 0) return ok;
  QQ_REQUIRE(!planned || !positions, "%s: a plan is of whole contexts, not of selected pages", what);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool one = planned && a.tiles == 1;
  QQ_REQUIRE(one || (head_dim == 128 ? begin_fits<Fp8Unit<128>>(a, st) : begin_fits<Fp8Unit<64>>(a, st)), "%s: bad sizes", what);
  if (head_dim == 128) launch_decode<Fp8Unit<128>>(a, st, SelectArgs{}, one, q_dtype, s);
  else launch_decode<Fp8Unit<64>>(a, st, SelectArgs{}, one, q_dtype, s);
  return check_launch(what);
}

extern "C" int qq_fp8_decode_plan(int num_blocks, int kv_heads, int head_dim, int block_table_rows, int block_table_cols,
                                  const int64_t* req_pool_indices, const int64_t* seq_lens, int bs, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const char* what = "qq_fp8_decode_plan";
  // what the slices do not depend on stands in for itself
  uint8_t* any = reinterpret_cast<uint8_t*>(workspace);
  float* any_scale = static_cast<float*>(workspace);
  DecArgs<Fp8Cache> a{};
  StoreArgs st{};
  QQ_REQUIRE(bs <= 0 || workspace, "%s: null pointer", what);
  if (bs == 0) return QQ_OK;
  const int ok = set_args(a, st, what, any, QQ_DTYPE_BF16, 0, kv_heads, nullptr, nullptr, QQ_DTYPE_BF16, nullptr,
                          Fp8Cache{any, any, any_scale, any_scale, num_blocks, kv_heads, head_dim},
                          static_cast<const int32_t*>(workspace), block_table_cols, block_table_rows, block_table_cols,
                          req_pool_indices, seq_lens, bs, nullptr, 0, 0, 1.0f, workspace, workspace, workspace_bytes);
  if (ok != QQ_OK) return ok;
  plan_kernel<<<1, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
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
  DecArgs<Fp8Cache> a{};
  StoreArgs st{};
  const int ok = set_args(a, st, what, q, q_dtype, q_batch_stride, num_q_heads, k_new, v_new, new_dtype, out_cache_loc,
                          Fp8Cache{k_codes, v_codes, k_scale, v_scale, num_blocks, kv_heads, head_dim}, block_table,
                          block_table_stride, block_table_rows, block_table_cols, req_pool_indices, seq_lens, bs, positions,
                          top_k, top_k, scale, out, workspace, workspace_bytes);
  if (ok != QQ_OK || bs == 0) return ok;
  QQ_REQUIRE(phase == 1 || (head_dim == 128 ? begin_fits<Fp8Unit<128>>(a, st) : begin_fits<Fp8Unit<64>>(a, st)), "%s: bad sizes", what);
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
  if (planned && phase == 3 && selects_itself(a, sel, q_dtype, kSelfPages)) {
    const int scored = launch_score_codes(sel, bs, a.c, k_new, v_new, new_dtype, out_cache_loc, s);
    if (scored < 0) return scored;
    if (scored == QQ_OK) {
      launch_selecting<Fp8Unit<128>>(a, StoreArgs{}, sel, s);
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
  if (head_dim == 128) launch_decode<Fp8Unit<128>>(a, st, sel, false, q_dtype, s);
  else launch_decode<Fp8Unit<64>>(a, st, sel, false, q_dtype, s);
  return check_launch(what);
}
