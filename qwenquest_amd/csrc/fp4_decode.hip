// Decode attention over the 4-bit K/V cache (layout: qq_fp4.h), dense or over the pages that
// Quest selected (reference src/qwenquest/attention/dense.py:26-42, quest_only.py:132-159,
// ops.py:48-66 over that cache).  With k_j the values of token j's key, vs its scale and vc its codes
//   t_j = scale * log2(e) * (q . k_j),  p_j = 2^(t_j - max t),  out = sum p_j vs_j vc_j / sum p_j.
//
// The division of the work and the kernels' frame are qq_decode_dev.h's.  K's codes become bf16 with their
// scale in the conversion (exact: a code has 2 significand bits), two at a time, NaN for a lost token; V's
// become bf16 as they are, and a weight takes its token's scale, exact in fp32, before it is cut into three
// bf16 pieces.  Every product takes the same factor (kOneFactor), so that only units at an edge mask, and the maximum may lag.
// Bound: 16 requests of 131072 tokens, 4 heads of 128, 207 to 211 us, 5.4 TB/s of codes and scales, with the vector units 63 % busy
// and waves waiting 40 %; 228 with the masks and rescalings in every unit.  A small batch by the chain of round trips, as
// over the 8-bit cache: one request of 2000 tokens 10.9 us a layer (waiting 79 %), 48 of up to 20000 in fp32 23.1.
// Quest, 16 requests' 31 pages and window of 131072 tokens 16.8 us with the selection.  Not taken: the next two
// units in flight instead of one (226 us where this took 214; fp32 spills), rescaling in every unit without the branch (slower), the sign of a
// negative factor on the queries (3 % at one request: another step before the first product).
#include "qq_decode_dev.h"
#include "qq_fp4_store.h"

namespace qq {
namespace {

// Eight codes times s.
__device__ inline bf16x8_t fp4_operand(uint32_t w, float s) {
  u32x4_t y;
  y.x = __builtin_bit_cast(uint32_t, fp4_pair(w, s, 0));
  y.y = __builtin_bit_cast(uint32_t, fp4_pair(w, s, 1));
  y.z = __builtin_bit_cast(uint32_t, fp4_pair(w, s, 2));
  y.w = __builtin_bit_cast(uint32_t, fp4_pair(w, s, 3));
  return __builtin_bit_cast(bf16x8_t, y);
}

template <int D>
struct Fp4Unit {
  using Cache = Fp4Cache;
  using Store = Fp4StoreArgs;
  struct BeginSmem {};
  static constexpr int kDim = D;
  static constexpr bool kOneFactor = true;
  static constexpr bool kStoresSelecting = true;
  static constexpr int KW = D / 32, VL = D / 32;  // words a lane: of a token of K; 16-byte loads: of a block of V
  typedef uint32_t words_t __attribute__((ext_vector_type(KW)));
  words_t kr[4];
  uint32_t ks;         // scales of this lane's tokens 16 T + m
  u32x4_t vr[VL], vs;  // ... and of 16 T + 4 g + u
  u32x4_t v2[VL], vs2; // of a window's second block

  // lane group g's channels: of 128 a scale's 32, of 64 half of that
  static __device__ inline int channel(int i, int g) { return g * (D / 4) + i * 8; }
  __device__ inline void look_up(const Fp4Cache&, int, int, int, bool) {}
  __device__ inline void load_k(const Fp4Cache& c, int h, int lane, int blk, int blk2, int from2) {
    const int m = lane & 15, g = lane >> 4;
    const int at = D == 128 ? lane * 16 : ((g >> 1) * 16 + m) * 16 + (g & 1) * 8;
    const int64_t e = (int64_t)blk * c.KV + h, e2 = (int64_t)blk2 * c.KV + h;
    const uint8_t *p = c.kc + e * (32 * D) + at, *p2 = c.kc + e2 * (32 * D) + at;
    const int scale_at = D == 128 ? lane * 4 : ((g >> 1) * 16 + m) * 4;
    ks = *reinterpret_cast<const uint32_t*>(c.ks + e * (2 * D) + scale_at);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      kr[t] = *reinterpret_cast<const words_t*>((t * 16 + m < from2 ? p2 : p) + t * 8 * D);
    if (blk2 != blk) {  // wave-uniform
      const uint32_t other = *reinterpret_cast<const uint32_t*>(c.ks + e2 * (2 * D) + scale_at);
      const int in2 = from2 <= m ? 0 : (from2 - m + 15) >> 4;  // of the word's four tokens
      const uint32_t mask = in2 >= 4 ? 0xFFFFFFFFu : (1u << (8 * in2)) - 1u;
      ks = (other & mask) | (ks & ~mask);
    }
  }
  __device__ inline void load_values(const Fp4Cache& c, int h, int lane, int blk, u32x4_t (&v)[VL], u32x4_t& scale) {
    const int64_t e = (int64_t)blk * c.KV + h;
    const uint8_t* p = c.vc + e * (32 * D) + lane * 16;
    scale = *reinterpret_cast<const u32x4_t*>(c.vs + e * 64 + (lane >> 4) * 16);
#pragma unroll
    for (int i = 0; i < VL; ++i) v[i] = *reinterpret_cast<const u32x4_t*>(p + i * 1024);
  }
  __device__ inline void load_v(const Fp4Cache& c, int h, int lane, int blk) { load_values(c, h, lane, blk, vr, vs); }
  __device__ inline void load_window_v(const Fp4Cache& c, int h, int lane, int blk2) { load_values(c, h, lane, blk2, v2, vs2); }
  __device__ inline void begin(int, bool, float) {}
  __device__ inline void keys(int t, int i, bf16x8_t& k0, bf16x8_t& k1) const {
    const float s = fp4_factor(ks, t);
    k0 = fp4_operand(kr[t][2 * i], s);
    k1 = fp4_operand(kr[t][2 * i + 1], s);
  }
  __device__ inline float weight(int t, int i, int, int) const { return fp4_factor(vs[t], i); }
  // bytes of word t whose tokens come from a window's second block
  static __device__ inline uint32_t window_mask(int t, int from2, int g) {
    const int in2 = min(max(from2 - t * 16 - g * 4, 0), 4);
    return in2 >= 4 ? 0xFFFFFFFFu : (1u << (8 * in2)) - 1u;
  }
  __device__ inline void merge_window_scales(int from2, int g) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t mask = window_mask(t, from2, g);
      vs[t] = (vs2[t] & mask) | (vs[t] & ~mask);
    }
  }
  __device__ inline void merge_window(int from2, int g) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t mask = window_mask(t, from2, g);
#pragma unroll
      for (int i = 0; i < VL; ++i) vr[i][t] = (v2[i][t] & mask) | (vr[i][t] & ~mask);
    }
  }
  // elements 2 x and 2 x + 1 are token u = x of 16-token groups 2 st and 2 st + 1
  static constexpr int tile_of(int st, int, int y) { return 2 * st + y; }
  static constexpr int place_of(int x, int) { return x; }
  __device__ inline bf16x8_t values(int i, int st) const {
    const u32x4_t& w = vr[(i >> 2) * 2 + (i & 1)];
    return fp4_operand(i & 2 ? fp4_upper(w[2 * st], w[2 * st + 1]) : fp4_lower(w[2 * st], w[2 * st + 1]), 1.0f);
  }

  static __device__ inline void store_tokens(const Fp4StoreArgs& st, int64_t i, bool on, int h) { fp4_store_tokens<D>(st, i, on, h); }
  // 1024 / D entries (of one head) a block
  static unsigned begin_blocks(const Fp4StoreArgs& st) { return (unsigned)((st.n * st.c.KV * (D / 4) + 255) / 256); }
  template <typename SRC>
  static __device__ inline void begin_store(const Fp4StoreArgs& st, BeginSmem&, int block) {
    const int64_t item = ((int64_t)block * 256 + threadIdx.x) / (D / 4), i = item / st.c.KV;
    fp4_store_group<D, SRC>(st, i, i < st.n, (int)(item - i * st.c.KV));
  }
};

// Where a layer selects in its attention (selects_itself).  Of several requests a slice may select twice, and the reading
// behind a selection is half of the 8-bit cache's: a layer-step in two launches and in three, us, contexts of 32768
// tokens, 32 heads on 4 (64 on 8; 8 on 1): 1 request, 31 pages 17.6, 18.3 (19.5, 20.3; 18.0, 18.7); 40 pages 17.3, 18.9 (19.5,
// 21.0; 17.1, 19.1); 63 pages 26.1, 22.2.  16 requests, 31 pages 26.4, 27.2 (33.4, 34.4; 22.9, 23.0); 36 pages 34.2, 33.2 (39.3,
// 39.3; 27.8, 26.7); 40 pages 37.1, 33.3.  4 and 40 requests: 31 pages 0.4 less to 0.8 more, 40 pages 0.1 to 3.8 more.
inline int self_pages(int bs) { return bs == 1 ? 40 : 32; }

}  // namespace
}  // namespace qq

using namespace qq;

extern "C" int64_t qq_fp4_decode_workspace_bytes(int bs, int num_q_heads, int kv_heads, int head_dim) {
  if (bs <= 0 || kv_heads <= 0 || num_q_heads < kv_heads || num_q_heads % kv_heads || !fp8_dim_ok(head_dim)) return 0;
  return decode_space(bs, num_q_heads, kv_heads, head_dim).bytes;
}

extern "C" int qq_fp4_decode_attention(const void* q, int q_dtype, int64_t q_batch_stride, int num_q_heads,
                                       const void* k_new, const void* v_new, int new_dtype, const int64_t* out_cache_loc,
                                       uint8_t* k_codes, uint8_t* v_codes, uint8_t* k_scale, uint8_t* v_scale,
                                       int num_blocks, int kv_heads, int head_dim, const int32_t* block_table,
                                       int64_t block_table_stride, int block_table_rows, int block_table_cols,
                                       const int64_t* req_pool_indices, const int64_t* seq_lens, int bs,
                                       const int32_t* positions, int64_t positions_stride, int top_k, float scale,
                                       void* out, void* workspace, int64_t workspace_bytes, int planned,
                                       void* stream) {
  const char* what = "qq_fp4_decode_attention";
  DecArgs<Fp4Cache> a{};
  Fp4StoreArgs st{};
  const int ok = set_args(a, st, what, q, q_dtype, q_batch_stride, num_q_heads, k_new, v_new, new_dtype, out_cache_loc,
                          Fp4Cache{k_codes, v_codes, k_scale, v_scale, num_blocks, kv_heads, head_dim}, block_table,
                          block_table_stride, block_table_rows, block_table_cols, req_pool_indices, seq_lens, bs, positions,
                          positions_stride, top_k, scale, out, workspace, workspace_bytes);
  if (ok != QQ_OK || bs == 0) return ok;
  QQ_REQUIRE(!planned || !positions, "%s: a plan is of whole contexts, not of selected pages", what);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool one = planned && a.tiles == 1;
  QQ_REQUIRE(one || (head_dim == 128 ? begin_fits<Fp4Unit<128>>(a, st) : begin_fits<Fp4Unit<64>>(a, st)), "%s: bad sizes", what);
  if (head_dim == 128) launch_decode<Fp4Unit<128>>(a, st, SelectArgs{}, one, q_dtype, s);
  else launch_decode<Fp4Unit<64>>(a, st, SelectArgs{}, one, q_dtype, s);
  return check_launch(what);
}

extern "C" int qq_fp4_decode_plan(int num_blocks, int kv_heads, int head_dim, int block_table_rows, int block_table_cols,
                                  const int64_t* req_pool_indices, const int64_t* seq_lens, int bs, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const char* what = "qq_fp4_decode_plan";
  // what the slices do not depend on stands in for itself
  uint8_t* any = reinterpret_cast<uint8_t*>(workspace);
  DecArgs<Fp4Cache> a{};
  Fp4StoreArgs st{};
  QQ_REQUIRE(bs <= 0 || workspace, "%s: null pointer", what);
  if (bs == 0) return QQ_OK;
  const int ok = set_args(a, st, what, any, QQ_DTYPE_BF16, 0, kv_heads, nullptr, nullptr, QQ_DTYPE_BF16, nullptr,
                          Fp4Cache{any, any, any, any, num_blocks, kv_heads, head_dim},
                          static_cast<const int32_t*>(workspace), block_table_cols, block_table_rows, block_table_cols,
                          req_pool_indices, seq_lens, bs, nullptr, 0, 0, 1.0f, workspace, workspace, workspace_bytes);
  if (ok != QQ_OK) return ok;
  plan_kernel<<<1, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  return check_launch(what);
}

extern "C" int qq_fp4_quest_step(const void* q, int q_dtype, int64_t q_batch_stride, int num_q_heads, const void* k_new,
                                 const void* v_new, int new_dtype, const int64_t* out_cache_loc, uint8_t* k_codes,
                                 uint8_t* v_codes, uint8_t* k_scale, uint8_t* v_scale, int num_blocks, int kv_heads,
                                 int head_dim, const int32_t* block_table, int64_t block_table_stride,
                                 int block_table_rows, int block_table_cols, const uint16_t* page_k_bounds, int layer,
                                 const int64_t* req_pool_indices, const int64_t* seq_lens, const int32_t* candidate_limit,
                                 int bs, int max_reqs, int max_pages, int top_k, float scale, float* scores_ws,
                                 int32_t* positions, void* out, void* workspace, int64_t workspace_bytes, int phase,
                                 int planned, void* stream) {
  const char* what = "qq_fp4_quest_step";
  QQ_REQUIRE(phase >= 1 && phase <= 3, "%s: phase must be 1, 2 or 3, got %d", what, phase);
  QQ_REQUIRE(bs == 0 || (page_k_bounds && candidate_limit && scores_ws && positions), "%s: null pointer", what);
  QQ_REQUIRE(layer >= 0 && max_reqs > 0 && max_pages >= 0, "%s: bad sizes", what);
  DecArgs<Fp4Cache> a{};
  Fp4StoreArgs st{};
  const int ok = set_args(a, st, what, q, q_dtype, q_batch_stride, num_q_heads, k_new, v_new, new_dtype, out_cache_loc,
                          Fp4Cache{k_codes, v_codes, k_scale, v_scale, num_blocks, kv_heads, head_dim}, block_table,
                          block_table_stride, block_table_rows, block_table_cols, req_pool_indices, seq_lens, bs, positions,
                          top_k, top_k, scale, out, workspace, workspace_bytes);
  if (ok != QQ_OK || bs == 0) return ok;
  QQ_REQUIRE(phase == 1 || (head_dim == 128 ? begin_fits<Fp4Unit<128>>(a, st) : begin_fits<Fp4Unit<64>>(a, st)), "%s: bad sizes", what);
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
  // the new tokens may go in with the attention: pages that are selected are complete, a new token's is not
  const bool one = planned && phase != 1 && a.tiles == 1;
  if (one && phase == 3 && selects_itself(a, sel, q_dtype, self_pages(bs))) {
    const int scored = launch_score(sel, bs, false, s);
    if (scored != QQ_OK) return scored;
    launch_selecting<Fp4Unit<128>>(a, st, sel, s);
    return check_launch(what);
  }
  if (phase == 1) return launch_retrieve(sel, bs, s);
  if (phase == 3) {
    const int scored = launch_score(sel, bs, false, s);
    if (scored != QQ_OK) return scored;
  } else {
    sel = SelectArgs{};  // phase 1 left the positions
  }
  if (head_dim == 128) launch_decode<Fp4Unit<128>>(a, st, sel, false, q_dtype, s);
  else launch_decode<Fp4Unit<64>>(a, st, sel, false, q_dtype, s);
  return check_launch(what);
}
