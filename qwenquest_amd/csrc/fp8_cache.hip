// The 8-bit K/V cache's writes and reads (layout: qq_fp8.h): the form of
// MHATokenToKVPool.set_kv_buffer (reference src/qwenquest/memory.py:114-120) for blocks of e4m3
// codes with a scale per block and KV head, the rows back as values, and the page bounds of
// QuestAlgorithm (src/qwenquest/quest.py:231-321) from the codes.
#include "qq_fp8_plan.h"
#include "qq_fp8_store.h"

namespace qq {
namespace {

template <int D, typename SRC>
__global__ __launch_bounds__(2 * D) void fp8_store_kernel(StoreArgs a) {
  __shared__ StoreSmem<D> sm;
  const int h = blockIdx.y >> 1;
  if (blockIdx.y & 1) store_segment<D, SRC, true>(a, sm, blockIdx.x, h);
  else store_segment<D, SRC, false>(a, sm, blockIdx.x, h);
}

// Eight codes times a scale; exact in bf16, a code having 4 significand bits.
__device__ inline void write8(uint16_t* out, uint32_t a, uint32_t b, float s) {
  const float4 x = decode4(a), y = decode4(b);
  *reinterpret_cast<uint4*>(out) = make_uint4((uint32_t)f2bf(x.x * s) | ((uint32_t)f2bf(x.y * s) << 16),
                                              (uint32_t)f2bf(x.z * s) | ((uint32_t)f2bf(x.w * s) << 16),
                                              (uint32_t)f2bf(y.x * s) | ((uint32_t)f2bf(y.y * s) << 16),
                                              (uint32_t)f2bf(y.z * s) | ((uint32_t)f2bf(y.w * s) << 16));
}
__device__ inline void write8(float* out, uint32_t a, uint32_t b, float s) {
  const float4 x = decode4(a), y = decode4(b);
  *reinterpret_cast<float4*>(out) = make_float4(x.x * s, x.y * s, x.z * s, x.w * s);
  *reinterpret_cast<float4*>(out + 4) = make_float4(y.x * s, y.y * s, y.z * s, y.w * s);
}

// Values of listed rows: a thread block takes `per` entries (16 or 64) of one head, a thread 8
// channels of every 16th entry.  K is read in place (8 bytes of a token's 16-byte pieces; the
// entries' neighbours share the lines).  A channel's tokens of V lie together, a token's channels
// 16 bytes apart: a run of entries of one block reads the block through the LDS, a few entries
// their bytes.
// Bound: HBM.  Measured, heads of 128 to bf16: 47921 prompt rows of 8 heads 75 us (3.9 TB/s), the
// 1181 rows in the last blocks of 32 requests, 4 heads, 5.9 us.
template <int D, typename DST>
__global__ __launch_bounds__(2 * D) void fp8_rows_kernel(Fp8Cache c, const int64_t* loc, int64_t n, int per, DST* k,
                                                          DST* v) {
  constexpr int NT = 2 * D, DG = D / 8, kRows = 64 * D / 256;
  __shared__ __align__(16) uint8_t codes[kRows * 272];  // 256-byte rows, 16 bytes apart: see StoreSmem
  const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.y;
  const int dg = tid % DG, sub = tid / DG;
  const int64_t e0 = (int64_t)blockIdx.x * per;
  const int count = (int)min((int64_t)per, n - e0);
  const int64_t row = lane < count ? loc[e0 + lane] : -1;
  const bool in = row >= 0 && (row >> 6) < c.blocks;
  const int blk = in ? (int)(row >> 6) : -1, slot = (int)(row & 63);
  // the lane's entry's scales
  const int64_t at = (int64_t)max(blk, 0) * c.KV + h;
  const float nan = __builtin_nanf("");
  const float ks = in ? c.ks[at] : nan, vs = in ? c.vs[at] : nan;
  for (int i = 0; i * 16 < per; ++i) {
    const int e = sub + 16 * i;
    const int b = max(__shfl(blk, e, 64), 0), t = __shfl(slot, e, 64);
    const float s = __shfl(ks, e, 64);
    if (e >= count) continue;
    const uint2 w = *reinterpret_cast<const uint2*>(c.kc + ((int64_t)b * c.KV + h) * (64 * D) + k_offset(D, t, dg * 8));
    write8(k + ((e0 + e) * c.KV + h) * D + dg * 8, w.x, w.y, s);
  }
  for (int first = 0; first < count;) {  // block-uniform: runs of one block (or of none)
    const int b = __builtin_amdgcn_readlane(blk, first);
    const uint64_t other = __ballot(blk != b && lane >= first && lane < count);
    const int end = other ? __builtin_ctzll(other) : count;
    const uint8_t* vp = c.vc + ((int64_t)max(b, 0) * c.KV + h) * (64 * D);
    const bool staged = end - first >= 8;
    if (staged) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int q = tid + i * NT;
        *reinterpret_cast<uint4*>(&codes[(q >> 4) * 272 + (q & 15) * 16]) = *reinterpret_cast<const uint4*>(vp + q * 16);
      }
      __syncthreads();
    }
    for (int i = 0; i * 16 < per; ++i) {
      const int e = sub + 16 * i;
      const int t = __shfl(slot, e, 64);
      const float s = __shfl(vs, e, 64);
      if (e < first || e >= end) continue;
      uint32_t w[2] = {0, 0};
      const int off = v_offset(t, dg * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int o = off + j * 16;
        w[j >> 2] |= (uint32_t)(staged ? codes[o + (o >> 8) * 16] : vp[o]) << (8 * (j & 3));
      }
      write8(v + ((e0 + e) * c.KV + h) * D + dg * 8, w[0], w[1], s);
    }
    first = end;
  }
}

struct PageArgs {
  const uint8_t* kc;  // first layer
  const float* ks;
  int64_t kc_stride, ks_stride;  // of a layer, elements
  int blocks, KV;
  const int32_t* table;
  int64_t table_stride;
  int table_rows, table_cols;
  const int64_t* rpi;
  const int64_t* seq;
  const int64_t* prefix;  // nullptr: from page 0 (prefill)
  int decode;
  uint32_t* bounds;  // [layers, R, MP, KV * D] (min, max) words
  int R, MP;
  int top_k, avoid;
  int32_t* actual;  // nullptr, or the step's layout: actual_lens, candidate_limit
  int32_t* limit;
  int layers;
  PlanArgs plan;  // cu nullptr, or the step's division of the attention's work, by a block past the layers
};

// Min and max of a page's keys per channel, a wave per (page, head, layer).  A scale is
// positive, so the extremes are those of the codes, which f16 holds exactly; the 16 tokens that
// the lanes of a row hold are folded in halves, each lane keeping half of its channels, until
// lane m has channel m: 15 exchanges for 16 channels instead of 64.
// Bound: HBM, the codes once (64 * D bytes per page and head, read as they lie).  Measured: two
// prompts of 16K tokens, 4 heads of 128, 48 layers 161 us (5.3 TB/s, reads and writes); a
// decode step's page of one request, 8 layers 1.9 us, with the step's slices 3.4.
template <int D>
__global__ __launch_bounds__(256) void fp8_page_bounds_kernel(PageArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int b = blockIdx.y, layer = blockIdx.z;
  if (layer == a.layers) {
    if (b == 0 && blockIdx.x == 0) plan_slices(a.plan);
    return;
  }
  const int64_t req = a.rpi[b], seq = a.seq[b], s = max(seq, (int64_t)0);
  if (a.actual && layer == 0 && blockIdx.x == 0 && threadIdx.x == 0) {
    a.actual[b] = (int32_t)min(seq, (int64_t)a.top_k);  // quest.py:343-352
    // the page that the step's own token completes has no bounds yet, whatever lies in its place
    a.limit[b] = (int32_t)(a.avoid ? max(seq / 64 - 1, (int64_t)0) : max(seq - 1, (int64_t)0) / 64);
  }
  if (req < 0 || req >= a.R || req >= a.table_rows) return;
  int64_t lo, hi;  // pages
  if (a.decode) {  // the page that the token before the newest completes
    hi = s >= 2 && (s - 1) % 64 == 0 ? (s - 1) / 64 : 0;
    lo = max(hi - 1, (int64_t)0);
  } else {
    hi = s / 64;
    lo = a.prefix ? max(a.prefix[b], (int64_t)0) / 64 : 0;
  }
  hi = min(hi, (int64_t)min(a.MP, a.table_cols));
  const int64_t units = (hi - lo) * a.KV;
  for (int64_t u = blockIdx.x * 4 + wave; u < units; u += gridDim.x * 4) {
    const int64_t page = lo + u / a.KV;
    const int h = (int)(u % a.KV);
    const int32_t blk = a.table[req * a.table_stride + page];
    const bool in = blk >= 0 && blk < a.blocks;
    const int64_t at = (int64_t)(in ? blk : 0) * a.KV + h;
    const uint8_t* kp = a.kc + layer * a.kc_stride + at * (64 * D) + lane * 16;
    const float scale = in ? a.ks[layer * a.ks_stride + at] : __builtin_nanf("");
    uint4 w[4][D / 64];
#pragma unroll
    for (int T = 0; T < 4; ++T)
#pragma unroll
      for (int i = 0; i < D / 64; ++i) w[T][i] = *reinterpret_cast<const uint4*>(kp + (T * (D / 64) + i) * 1024);
    uint32_t* out = a.bounds + (((int64_t)layer * a.R + req) * a.MP + page) * (a.KV * D) + h * D;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      f16x2_t mn[8], mx[8];
#pragma unroll
      for (int T = 0; T < 4; ++T) {
        const uint32_t x[4] = {w[T][i].x, w[T][i].y, w[T][i].z, w[T][i].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const f16x2_t y = j & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[j >> 1], 1.0f, true)
                                  : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[j >> 1], 1.0f, false);
          mn[j] = T ? __builtin_elementwise_min(mn[j], y) : y;
          mx[j] = T ? __builtin_elementwise_max(mx[j], y) : y;
        }
      }
#pragma unroll
      for (int half = 4; half >= 1; half >>= 1) {  // partner lane ^ 2 * half
        const bool up = lane & (2 * half);
#pragma unroll
        for (int j = 0; j < half; ++j) {
          const int sn = __builtin_bit_cast(int, up ? mn[j] : mn[j + half]), sx = __builtin_bit_cast(int, up ? mx[j] : mx[j + half]);
          const f16x2_t rn = __builtin_bit_cast(f16x2_t, __shfl_xor(sn, 2 * half, 64));
          const f16x2_t rx = __builtin_bit_cast(f16x2_t, __shfl_xor(sx, 2 * half, 64));
          mn[j] = __builtin_elementwise_min(up ? mn[j + half] : mn[j], rn);
          mx[j] = __builtin_elementwise_max(up ? mx[j + half] : mx[j], rx);
        }
      }
      const f16x2_t on = __builtin_bit_cast(f16x2_t, __shfl_xor(__builtin_bit_cast(int, mn[0]), 1, 64));
      const f16x2_t ox = __builtin_bit_cast(f16x2_t, __shfl_xor(__builtin_bit_cast(int, mx[0]), 1, 64));
      const f16x2_t n = __builtin_elementwise_min(mn[0], on), x = __builtin_elementwise_max(mx[0], ox);
      const float fn = (float)(lane & 1 ? n.y : n.x) * scale, fx = (float)(lane & 1 ? x.y : x.x) * scale;
      out[i * 64 + lane] = (uint32_t)f2bf(fn) | ((uint32_t)f2bf(fx) << 16);
    }
  }
}

}  // namespace

int check_cache(const Fp8Cache& c, const char* what) {
  QQ_REQUIRE(c.kc && c.vc && c.ks && c.vs, "%s: null cache pointer", what);
  QQ_REQUIRE(c.blocks > 0 && c.blocks <= kMaxPoolBlocks, "%s: %d blocks, at most %d", what, c.blocks, kMaxPoolBlocks);
  QQ_REQUIRE(c.KV > 0 && c.KV <= 1024, "%s: %d KV heads", what, c.KV);
  QQ_REQUIRE(fp8_dim_ok(c.D), "%s: head_dim %d is not 64 or 128", what, c.D);
  return QQ_OK;
}

}  // namespace qq

using namespace qq;

constexpr int64_t kStoreBlocks = 2048;  // thread blocks that the chip holds

extern "C" int qq_fp8_store(uint8_t* k_codes, uint8_t* v_codes, float* k_scale, float* v_scale, int num_blocks,
                            int kv_heads, int head_dim, const void* k, const void* v, int src_dtype, const int64_t* loc,
                            int64_t n, void* stream) {
  const char* what = "qq_fp8_store";
  StoreArgs a{{k_codes, v_codes, k_scale, v_scale, num_blocks, kv_heads, head_dim}, k, v, src_dtype, loc, n, 1};
  const int st = check_cache(a.c, what);
  if (st != QQ_OK) return st;
  QQ_REQUIRE(dtype_ok(src_dtype), "%s: bad dtype", what);
  QQ_REQUIRE(n >= 0 && n < (int64_t)1 << 31, "%s: bad sizes", what);
  if (n == 0) return QQ_OK;
  QQ_REQUIRE(k && v && loc, "%s: null pointer", what);
  QQ_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "%s: k and v must be 16-byte aligned", what);
  // an entry per thread block while all of them are resident at once, so that a decode batch's runs
  // of one go side by side; of a prompt's entries one in 64 begins a run, and looking at more at a
  // time leaves fewer blocks without one (3440 entries of 4 heads one at a time 50 us, 16 at a time
  // 7.2; 8192 32 at a time 11.7, 64 at a time 15.7)
  while (a.seg < 64 && n * 2 * kv_heads > a.seg * kStoreBlocks) a.seg *= 2;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)((n + a.seg - 1) / a.seg), 2 * kv_heads);
  const bool bf = src_dtype == QQ_DTYPE_BF16;
  if (head_dim == 128) {
    if (bf) fp8_store_kernel<128, uint16_t><<<grid, 256, 0, s>>>(a);
    else fp8_store_kernel<128, float><<<grid, 256, 0, s>>>(a);
  } else {
    if (bf) fp8_store_kernel<64, uint16_t><<<grid, 128, 0, s>>>(a);
    else fp8_store_kernel<64, float><<<grid, 128, 0, s>>>(a);
  }
  return check_launch(what);
}

extern "C" int qq_fp8_rows(const uint8_t* k_codes, const uint8_t* v_codes, const float* k_scale, const float* v_scale,
                           int num_blocks, int kv_heads, int head_dim, const int64_t* loc, int64_t n, void* k, void* v,
                           int dst_dtype, void* stream) {
  const char* what = "qq_fp8_rows";
  const Fp8Cache c{const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(v_codes), const_cast<float*>(k_scale),
                   const_cast<float*>(v_scale), num_blocks, kv_heads, head_dim};
  const int st = check_cache(c, what);
  if (st != QQ_OK) return st;
  QQ_REQUIRE(dtype_ok(dst_dtype), "%s: bad dtype", what);
  QQ_REQUIRE(n >= 0 && n < (int64_t)1 << 31, "%s: bad sizes", what);
  if (n == 0) return QQ_OK;
  QQ_REQUIRE(loc && k && v, "%s: null pointer", what);
  // a block's run is read by as many thread blocks as its entries are dealt to; few entries give
  // more thread blocks of a run or two each (1181 entries of 32 requests 5.9 us, in 64s 10.5)
  const int per = n * kv_heads <= 16384 ? 16 : 64;
  const dim3 grid((unsigned)((n + per - 1) / per), kv_heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint16_t *kb = static_cast<uint16_t*>(k), *vb = static_cast<uint16_t*>(v);
  float *kf = static_cast<float*>(k), *vf = static_cast<float*>(v);
  const bool bf = dst_dtype == QQ_DTYPE_BF16;
  if (head_dim == 128) {
    if (bf) fp8_rows_kernel<128><<<grid, 256, 0, s>>>(c, loc, n, per, kb, vb);
    else fp8_rows_kernel<128><<<grid, 256, 0, s>>>(c, loc, n, per, kf, vf);
  } else {
    if (bf) fp8_rows_kernel<64><<<grid, 128, 0, s>>>(c, loc, n, per, kb, vb);
    else fp8_rows_kernel<64><<<grid, 128, 0, s>>>(c, loc, n, per, kf, vf);
  }
  return check_launch(what);
}

extern "C" int qq_fp8_page_bounds(const uint8_t* k_codes, int64_t codes_layer_stride, const float* k_scale,
                                  int64_t scale_layer_stride, int num_blocks, int kv_heads, int head_dim,
                                  const int32_t* block_table, int64_t block_table_stride, int block_table_rows,
                                  int block_table_cols, const int64_t* req_pool_indices, const int64_t* seq_lens,
                                  const int64_t* prefix_lens, int bs, int decode, int64_t max_new, int n_layers,
                                  uint16_t* page_k_bounds, int max_reqs, int max_pages, int top_k,
                                  int avoid_recent_overlap, int32_t* actual_lens, int32_t* candidate_limit, void* plan,
                                  int64_t plan_bytes, void* stream) {
  const char* what = "qq_fp8_page_bounds";
  const Fp8Cache c{const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(k_codes), const_cast<float*>(k_scale),
                   const_cast<float*>(k_scale), num_blocks, kv_heads, head_dim};
  const int st = check_cache(c, what);
  if (st != QQ_OK) return st;
  QQ_REQUIRE(bs >= 0 && bs < 65536 && n_layers > 0 && n_layers < 65535 && max_reqs > 0 && max_pages > 0 && max_new >= 0 &&
                 block_table_cols > 0 && block_table_stride >= block_table_cols && block_table_rows > 0,
             "%s: bad sizes", what);
  QQ_REQUIRE(!actual_lens == !candidate_limit, "%s: one of the layout's outputs is missing", what);
  if (bs == 0) return QQ_OK;
  QQ_REQUIRE(block_table && req_pool_indices && seq_lens && page_k_bounds, "%s: null pointer", what);
  PageArgs a{k_codes, k_scale, codes_layer_stride, scale_layer_stride, num_blocks, kv_heads, block_table, block_table_stride,
             block_table_rows, block_table_cols, req_pool_indices, seq_lens, prefix_lens, decode,
             reinterpret_cast<uint32_t*>(page_k_bounds), max_reqs, max_pages, top_k, avoid_recent_overlap, actual_lens,
             candidate_limit, n_layers, {}};
  if (plan) {
    QQ_REQUIRE(decode && top_k > 0 && top_k % 64 == 0, "%s: a plan is of a decode step's selections of whole pages", what);
    QQ_REQUIRE((int64_t)block_table_cols * bs < (int64_t)1 << 30, "%s: too many units of work", what);
    const DecSpace sp = decode_space(bs, kv_heads, kv_heads, head_dim);
    QQ_REQUIRE(plan_bytes >= sp.bytes, "%s: workspace %lld bytes < %lld needed", what, (long long)plan_bytes, (long long)sp.bytes);
    set_plan(a.plan, sp, plan, req_pool_indices, seq_lens, bs, block_table_rows, block_table_cols, top_k, kv_heads);
  }
  // pages of a request, at most: those its new tokens can complete
  const int64_t pages = decode ? 1 : min((int64_t)max_pages, max_new > 0 && prefix_lens ? max_new / 64 + 1 : (int64_t)max_pages);
  const int64_t need = (pages * kv_heads + 3) / 4, fill = max((int64_t)1, (int64_t)16384 / ((int64_t)bs * n_layers));
  const dim3 grid((unsigned)min(need, fill), bs, n_layers + (plan ? 1 : 0));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128) fp8_page_bounds_kernel<128><<<grid, 256, 0, s>>>(a);
  else fp8_page_bounds_kernel<64><<<grid, 256, 0, s>>>(a);
  return check_launch(what);
}
