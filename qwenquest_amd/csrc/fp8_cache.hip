// The 8-bit K/V cache's writes and reads (layout: qq_fp8.h): the form of
// MHATokenToKVPool.set_kv_buffer (reference src/qwenquest/memory.py:114-120) for blocks of e4m3
// codes with a scale per block and KV head, the rows back as values, and the page bounds of
// QuestAlgorithm (src/qwenquest/quest.py:231-321) from the codes.
//
// Write: of the values x that a call puts into a (block, head), K and V apart,
//   e = max(e_before, least e >= -110 with max |x| <= 448 * 2^e),  code = e4m3(x / 2^e)
// with e_before = -110 when the call writes the block's first row (that begins the block:
// its earlier contents are void), and when e grows the codes already there are re-rounded at
// the new scale (exact but for the least bits of subnormal codes, the scale being a power of
// two).  A value that is not finite makes the scale NaN until the block is begun again.
#include "qq_fp8.h"

namespace qq {
namespace {

struct StoreArgs {
  Fp8Cache c;
  const void* k;  // [n, KV, D]
  const void* v;
  const int64_t* loc;
  int64_t n;
  int seg;  // entries of loc whose blocks one thread block looks after
};

__device__ inline float finite_or_zero(float x, bool& bad) {
  const bool ok = (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u;
  bad |= !ok;
  return ok ? x : 0.0f;
}

// Eight consecutive values as floats.
__device__ inline void load8(const uint16_t* p, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
  }
}
__device__ inline void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

template <int D>
struct StoreSmem {
  static constexpr int kRows = 64 * D / 256;
  int from[64];              // entry that writes each token of the block, or -1
  float amax[2][4];
  int bad[2];
  // whole blocks are composed here: 256-byte rows of 16-byte pieces, 16 bytes apart so that
  // the rows' equal columns lie in different banks
  __align__(16) uint8_t codes[2][kRows * 272];
};

// One (block, head) of a run of entries.  Thread (quad, dg): tokens 4 quad .. + 3, channels
// 8 dg .. + 7, which are 8-byte pieces of K and 4-byte pieces of V.
template <int D, typename SRC>
__device__ inline void store_block(const StoreArgs& a, StoreSmem<D>& sm, int block, int h) {
  constexpr int NT = 2 * D, DG = D / 8, kWaves = NT / 64;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int quad = tid / DG, dg = tid % DG;
  const int64_t at = (int64_t)block * a.c.KV + h;
  uint8_t* codes[2] = {a.c.kc + at * (64 * D), a.c.vc + at * (64 * D)};
  float* scales[2] = {a.c.ks + at, a.c.vs + at};
  const float before[2] = {*scales[0], *scales[1]};
  const bool begun = sm.from[0] >= 0;
  int from[4];
  float x[2][4][8];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    from[u] = sm.from[4 * quad + u];
    const int64_t row = ((int64_t)max(from[u], 0) * a.c.KV + h) * D + dg * 8;
    if (from[u] >= 0) {
      load8(static_cast<const SRC*>(a.k) + row, x[0][u]);
      load8(static_cast<const SRC*>(a.v) + row, x[1][u]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[0][u][j] = x[1][u][j] = 0.0f;
    }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float m = 0.0f;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[c][u][j] = finite_or_zero(x[c][u][j], bad);
        m = fmaxf(m, fabsf(x[c][u][j]));
      }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    if (lane == 0) sm.amax[c][wave] = m;
    if (bad) sm.bad[c] = 1;
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float m = sm.amax[c][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, sm.amax[c][w]);
    const bool lost = !begun && before[c] != before[c];
    const bool bad = sm.bad[c] || lost;
    const int e_old = begun || lost ? kScaleMin : exponent_of(before[c]);
    const int e = max(e_old, scale_exponent(m));
    const float inv = pow2f(-e);
    if (tid == 0) *scales[c] = bad ? __builtin_nanf("") : pow2f(e);
    uint32_t code[4][2];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        code[u][i] = encode4(x[c][u][4 * i] * inv, x[c][u][4 * i + 1] * inv, x[c][u][4 * i + 2] * inv,
                             x[c][u][4 * i + 3] * inv);
    if (c == 1) {  // 4 tokens of a channel are neighbours: transposed to words of 4 tokens
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int s = 8 * (j & 3);
        w[j] = ((code[0][j >> 2] >> s) & 255u) | (((code[1][j >> 2] >> s) & 255u) << 8) |
               (((code[2][j >> 2] >> s) & 255u) << 16) | (((code[3][j >> 2] >> s) & 255u) << 24);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) code[j >> 1][j & 1] = w[j];
    }
    if (begun) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (c == 0) {
          const int t = 4 * quad + u, row = (t >> 4) * (D / 16) + dg / 2;
          *reinterpret_cast<uint2*>(&sm.codes[0][row * 272 + (t & 15) * 16 + (dg & 1) * 8]) = make_uint2(code[u][0], code[u][1]);
        } else {
          const int row = (dg / 2) * 4 + (quad & 3);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint32_t*>(&sm.codes[1][row * 272 + ((dg & 1) * 8 + 2 * u + i) * 16 + (quad >> 2) * 4]) = code[u][i];
        }
      }
      continue;
    }
    // a block begun before: the tokens written now, and all of them when the scale has grown
    const bool grown = e > e_old;
    const float f = pow2f(max(e_old - e, -126));
    if (c == 0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint2* p = reinterpret_cast<uint2*>(codes[0] + k_offset(D, 4 * quad + u, dg * 8));
        if (from[u] >= 0) {
          *p = make_uint2(code[u][0], code[u][1]);
        } else if (grown) {
          const uint2 old = *p;
          *p = make_uint2(rescale4(old.x, f), rescale4(old.y, f));
        }
      }
    } else {
      uint32_t mask = 0;  // bytes written now
#pragma unroll
      for (int u = 0; u < 4; ++u) mask |= from[u] >= 0 ? 255u << (8 * u) : 0u;
      if (mask || grown) {
        uint32_t old[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) old[j] = *reinterpret_cast<const uint32_t*>(codes[1] + v_offset(4 * quad, dg * 8 + j));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t o = grown ? rescale4(old[j], f) : old[j];
          *reinterpret_cast<uint32_t*>(codes[1] + v_offset(4 * quad, dg * 8 + j)) = (code[j >> 1][j & 1] & mask) | (o & ~mask);
        }
      }
    }
  }
  if (!begun) return;
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int q = tid + i * NT;
      *reinterpret_cast<uint4*>(codes[c] + q * 16) = *reinterpret_cast<const uint4*>(&sm.codes[c][(q >> 4) * 272 + (q & 15) * 16]);
    }
}

// Entries of one block stand next to each other in loc; the thread block in whose segment
// such a run begins writes its (block, head) alone, so nothing is shared between thread
// blocks and the result does not depend on their order.  Of a row listed twice in a run the
// last entry counts.
template <int D, typename SRC>
__global__ __launch_bounds__(2 * D) void fp8_store_kernel(StoreArgs a) {
  __shared__ StoreSmem<D> sm;
  const int tid = threadIdx.x, lane = tid & 63;
  const int h = blockIdx.y;
  const int64_t e0 = (int64_t)blockIdx.x * a.seg;
  auto block_at = [&](int64_t i) { return i >= 0 && i < a.n ? block_of(a.loc[i], a.c.blocks) : 0; };
  // every wave for itself: where the segment's runs begin
  const int mine = lane < a.seg ? block_at(e0 + lane) : 0;
  uint64_t starts = __ballot(mine > 0 && mine != block_at(e0 + lane - 1));
  while (starts) {
    const int at = __builtin_ctzll(starts);
    starts &= starts - 1;
    const int block = __shfl(mine, at, 64);
    __syncthreads();  // the run before is done with sm
    if (tid < 64) {
      sm.from[tid] = -1;
      if (tid < 2) sm.bad[tid] = 0;
    }
    __syncthreads();
    if (tid < 64) {
      for (int64_t i0 = e0 + at;; i0 += 64) {
        const int64_t i = i0 + lane;
        const uint64_t other = __ballot(block_at(i) != block);
        const int len = other ? __builtin_ctzll(other) : 64;
        if (lane < len) atomicMax(&sm.from[a.loc[i] & 63], (int)i);
        if (len < 64) break;
      }
    }
    __syncthreads();
    store_block<D, SRC>(a, sm, block, h);
  }
}

// Values of listed rows: a thread takes 8 channels of one row and head, K and V.
template <typename DST>
__global__ __launch_bounds__(256) void fp8_rows_kernel(Fp8Cache c, const int64_t* loc, int64_t n, DST* k, DST* v) {
  const int per = c.KV * c.D / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * per) return;
  const int64_t e = i / per;
  const int at = (int)(i - e * per), h = at / (c.D / 8), d = (at - h * (c.D / 8)) * 8;
  const int64_t row = loc[e];
  const int t = (int)(row & 63);
  const bool in = row >= 0 && (row >> 6) < c.blocks;
  const int64_t head = (in ? row >> 6 : 0) * c.KV + h;
  const float nan = __builtin_nanf("");
  const float ks = in ? c.ks[head] : nan, vs = in ? c.vs[head] : nan;
  const uint2 kw = *reinterpret_cast<const uint2*>(c.kc + head * (64 * c.D) + k_offset(c.D, t, d));
  const uint8_t* vp = c.vc + head * (64 * c.D) + v_offset(t, d);
  uint32_t vw[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) vw[j >> 2] |= (uint32_t)vp[j * 16] << (8 * (j & 3));
  const float4 x[4] = {decode4(kw.x), decode4(kw.y), decode4(vw[0]), decode4(vw[1])};
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float s = half ? vs : ks;
    DST* out = (half ? v : k) + i * 8;
    const float y[8] = {x[2 * half].x * s, x[2 * half].y * s, x[2 * half].z * s, x[2 * half].w * s,
                        x[2 * half + 1].x * s, x[2 * half + 1].y * s, x[2 * half + 1].z * s, x[2 * half + 1].w * s};
    if constexpr (sizeof(DST) == 2) {  // exact: a code has 4 significand bits
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (uint32_t)f2bf(y[2 * j]) | ((uint32_t)f2bf(y[2 * j + 1]) << 16);
      *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<float4*>(out) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(out + 4) = make_float4(y[4], y[5], y[6], y[7]);
    }
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
};

// Min and max of a page's keys per channel, a wave per (page, head, layer).  A scale is
// positive, so the extremes are those of the codes, which f16 holds exactly; the 16 tokens that
// the lanes of a row hold are folded in halves, each lane keeping half of its channels, until
// lane m has channel m: 15 exchanges for 16 channels instead of 64.
// Bound: HBM, the codes once (64 * D bytes per page and head, read as they lie).
template <int D>
__global__ __launch_bounds__(256) void fp8_page_bounds_kernel(PageArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int b = blockIdx.y, layer = blockIdx.z;
  const int64_t req = a.rpi[b], s = max(a.seq[b], (int64_t)0);
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

extern "C" int qq_fp8_store(uint8_t* k_codes, uint8_t* v_codes, float* k_scale, float* v_scale, int num_blocks,
                            int kv_heads, int head_dim, const void* k, const void* v, int src_dtype, const int64_t* loc,
                            int64_t n, void* stream) {
  const char* what = "qq_fp8_store";
  StoreArgs a{{k_codes, v_codes, k_scale, v_scale, num_blocks, kv_heads, head_dim}, k, v, loc, n, 1};
  const int st = check_cache(a.c, what);
  if (st != QQ_OK) return st;
  QQ_REQUIRE(dtype_ok(src_dtype), "%s: bad dtype", what);
  QQ_REQUIRE(n >= 0 && n < (int64_t)1 << 31, "%s: bad sizes", what);
  if (n == 0) return QQ_OK;
  QQ_REQUIRE(k && v && loc, "%s: null pointer", what);
  QQ_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "%s: k and v must be 16-byte aligned", what);
  // an entry per thread block, so that a decode batch's runs of one go side by side; of a
  // prompt's entries one in 64 begins a run, and looking at 16 at a time spares the blocks
  // that find none
  a.seg = n <= 4096 ? 1 : 16;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)((n + a.seg - 1) / a.seg), kv_heads);
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
  const int64_t blocks = (n * (kv_heads * head_dim / 8) + 255) / 256;
  QQ_REQUIRE(blocks < (int64_t)1 << 31, "%s: too many rows", what);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dst_dtype == QQ_DTYPE_BF16)
    fp8_rows_kernel<uint16_t><<<(unsigned)blocks, 256, 0, s>>>(c, loc, n, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v));
  else
    fp8_rows_kernel<float><<<(unsigned)blocks, 256, 0, s>>>(c, loc, n, static_cast<float*>(k), static_cast<float*>(v));
  return check_launch(what);
}

extern "C" int qq_fp8_page_bounds(const uint8_t* k_codes, int64_t codes_layer_stride, const float* k_scale,
                                  int64_t scale_layer_stride, int num_blocks, int kv_heads, int head_dim,
                                  const int32_t* block_table, int64_t block_table_stride, int block_table_rows,
                                  int block_table_cols, const int64_t* req_pool_indices, const int64_t* seq_lens,
                                  const int64_t* prefix_lens, int bs, int decode, int64_t max_new, int n_layers,
                                  uint16_t* page_k_bounds, int max_reqs, int max_pages, void* stream) {
  const char* what = "qq_fp8_page_bounds";
  const Fp8Cache c{const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(k_codes), const_cast<float*>(k_scale),
                   const_cast<float*>(k_scale), num_blocks, kv_heads, head_dim};
  const int st = check_cache(c, what);
  if (st != QQ_OK) return st;
  QQ_REQUIRE(bs >= 0 && bs < 65536 && n_layers > 0 && n_layers < 65536 && max_reqs > 0 && max_pages > 0 && max_new >= 0 &&
                 block_table_cols > 0 && block_table_stride >= block_table_cols && block_table_rows > 0,
             "%s: bad sizes", what);
  if (bs == 0) return QQ_OK;
  QQ_REQUIRE(block_table && req_pool_indices && seq_lens && page_k_bounds, "%s: null pointer", what);
  PageArgs a{k_codes, k_scale, codes_layer_stride, scale_layer_stride, num_blocks, kv_heads, block_table, block_table_stride,
             block_table_rows, block_table_cols, req_pool_indices, seq_lens, prefix_lens, decode,
             reinterpret_cast<uint32_t*>(page_k_bounds), max_reqs, max_pages};
  // pages of a request, at most: those its new tokens can complete
  const int64_t pages = decode ? 1 : min((int64_t)max_pages, max_new > 0 && prefix_lens ? max_new / 64 + 1 : (int64_t)max_pages);
  const int64_t need = (pages * kv_heads + 3) / 4, fill = max((int64_t)1, (int64_t)16384 / ((int64_t)bs * n_layers));
  const dim3 grid((unsigned)min(need, fill), bs, n_layers);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128) fp8_page_bounds_kernel<128><<<grid, 256, 0, s>>>(a);
  else fp8_page_bounds_kernel<64><<<grid, 256, 0, s>>>(a);
  return check_launch(what);
}
