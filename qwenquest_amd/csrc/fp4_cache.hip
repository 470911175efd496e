// The 4-bit K/V cache's writes and reads (layout: qq_fp4.h): the form of
// MHATokenToKVPool.set_kv_buffer (reference src/qwenquest/memory.py:114-120) for blocks of e2m1
// codes with scales of their own for every token, the rows back as values, and the page bounds of
// QuestAlgorithm (src/qwenquest/quest.py:231-321) from the codes.
//
// Bound: HBM where entries are many: 47921 tokens, 8 heads of 128 in bf16, stored in 51 to 67 us (196 MB read and 51
// written, of which half is in the caches; 456 entry by entry, whose V writes are single bytes), 47971 rows back in 43 us (248 MB, 5.8 TB/s);
// page bounds of two prompts of 16384 tokens, 4 heads of 128, 48 layers 113 us (4.2 TB/s), where the vector
// units have the rest (343 with 4-byte loads and comparisons in fp32).  Few entries are a chain of two round trips behind a launch: 32 tokens
// stored in 3.7 us, 1181 rows in 4.1.
#include <type_traits>

#include "qq_fp4_store.h"
#include "qq_fp8_plan.h"
#include "qq_quest_dev.h"

namespace qq {
namespace {

template <int D, typename SRC>
__global__ __launch_bounds__(256) void fp4_store_kernel(Fp4StoreArgs a) {
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / (D / 4);
  const int64_t i = item / a.c.KV;
  fp4_store_group<D, SRC>(a, i, i < a.n, (int)(item - i * a.c.KV));
}

// Runs of entries of one block, a segment of 64 entries and a head a thread block.  Runs go one after the other, a round trip
// each; where more than 8 begin in the segment, they go entry by entry, 8 at a time.
template <int D, typename SRC>
__global__ __launch_bounds__(2 * D) void fp4_store_runs_kernel(Fp4StoreArgs a) {
  __shared__ int from[64];
  const int lane = threadIdx.x & 63;
  const int64_t e0 = (int64_t)blockIdx.x * 64;
  auto block_at = [&](int64_t i) { return i >= 0 && i < a.n ? block_of(a.loc[i], a.c.blocks) : 0; };
  const int mine = block_at(e0 + lane), before = block_at(e0 + lane - 1);
  const uint64_t starts = __ballot(mine > 0 && mine != before);
  if (__popcll(starts) > 8) {
    int64_t end = e0 + 64;  // of the last run
    for (const int last = __builtin_amdgcn_readlane(mine, 63); last > 0;) {
      const uint64_t past = __ballot(block_at(end + lane) != last);
      end += past ? __builtin_ctzll(past) : 64;
      if (past) break;
    }
    constexpr int kGroups = 2 * D / (D / 4);
    for (int64_t i0 = e0 + __builtin_ctzll(starts); i0 < end; i0 += kGroups) {
      const int64_t i = i0 + threadIdx.x / (D / 4);
      fp4_store_group<D, SRC>(a, i, i < end && i < a.n, blockIdx.y);
    }
    return;
  }
  each_run(a.loc, a.n, a.c.blocks, 64, blockIdx.x, from, [&](int block, int) {
    if (block) fp4_store_block<D, SRC>(a, from, block, blockIdx.y);
  });
}

__device__ inline void fp4_write8(uint16_t* out, uint32_t w, float s) {
  u32x4_t y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = s != s ? 0x7FC07FC0u : __builtin_bit_cast(uint32_t, fp4_pair(w, s, i));
  *reinterpret_cast<u32x4_t*>(out) = y;
}
__device__ inline void fp4_write8(float* out, uint32_t w, float s) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t p = __builtin_bit_cast(uint32_t, fp4_pair(w, s, i));
    y[2 * i] = s != s ? s : __uint_as_float(p << 16);
    y[2 * i + 1] = s != s ? s : __uint_as_float(p & 0xFFFF0000u);
  }
  *reinterpret_cast<float4*>(out) = make_float4(y[0], y[1], y[2], y[3]);
  *reinterpret_cast<float4*>(out + 4) = make_float4(y[4], y[5], y[6], y[7]);
}

// Values of listed rows: a thread 8 channels of K and of V of one row and head.
template <int D, typename DST>
__global__ __launch_bounds__(256) void fp4_rows_kernel(Fp4Cache c, const int64_t* loc, int64_t n, DST* k, DST* v) {
  constexpr int DG = D / 8;
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / DG;
  const int dg = threadIdx.x % DG;
  const int64_t i = item / c.KV;
  if (i >= n) return;
  const int h = (int)(item - i * c.KV);
  const int64_t row = loc[i];
  const bool in = row >= 0 && (row >> 6) < c.blocks;
  const int64_t at = (in ? row >> 6 : 0) * c.KV + h;
  const int t = (int)(row & 63);
  auto factor = [&](uint32_t e) { return in && e != kFp4Lost ? __uint_as_float(e << 23) : __builtin_nanf(""); };
  const float ks = factor(c.ks[at * (2 * D) + fp4_ks_offset(t, dg * 8)]), vs = factor(c.vs[at * 64 + fp4_vs_offset(t)]);
  fp4_write8(k + item * D + dg * 8, *reinterpret_cast<const uint32_t*>(c.kc + at * (32 * D) + fp4_k_offset(D, t, dg * 8)), ks);
  uint32_t w = 0;
  const uint8_t* codes = c.vc + at * (32 * D) + fp4_v_offset(t, dg * 8);
#pragma unroll
  for (int j = 0; j < 8; ++j) w |= ((codes[j * 16] >> (dg & 4 ? 4 : 0)) & 15u) << (4 * j);
  fp4_write8(v + item * D + dg * 8, w, vs);
}

// The same for many rows: a thread block 64 entries of one head.  A run of one block reads its V as it lies, which
// the threads turn to a token's channels side by side, and goes on through the LDS; where more than 8 runs
// meet, as above.
template <int D, typename DST>
__global__ __launch_bounds__(2 * D) void fp4_rows_runs_kernel(Fp4Cache c, const int64_t* loc, int64_t n, DST* k, DST* v) {
  constexpr int DG = D / 8;
  __shared__ uint32_t codes[64 * DG];  // [token][8 channels]
  const int lane = threadIdx.x & 63, tt = threadIdx.x / DG, dg = lane % DG, g = tt >> 2, u = tt & 3, h = blockIdx.y;
  const int64_t e0 = (int64_t)blockIdx.x * 64;
  const int count = (int)min((int64_t)64, n - e0);
  const int64_t row = lane < count ? loc[e0 + lane] : -1;
  const bool in = row >= 0 && (row >> 6) < c.blocks;
  const int blk = in ? (int)(row >> 6) : -1, slot = (int)(row & 63);
  const int prev = __shfl_up(blk, 1, 64);
  const uint64_t starts = __ballot(lane < count && (lane == 0 || blk != prev));
  const bool apart = __popcll(starts) > 8;
  auto factor = [](uint32_t e, bool ok) { return ok && e != kFp4Lost ? __uint_as_float(e << 23) : __builtin_nanf(""); };
  auto entry = [&](int e, bool staged) {
    const int b = __shfl(blk, e, 64), t = __shfl(slot, e, 64);
    if (e >= count) return;
    const int64_t at = (int64_t)max(b, 0) * c.KV + h, to = ((e0 + e) * c.KV + h) * D + dg * 8;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(c.kc + at * (32 * D) + fp4_k_offset(D, t, dg * 8));
    const float ks = factor(c.ks[at * (2 * D) + fp4_ks_offset(t, dg * 8)], b >= 0), vs = factor(c.vs[at * 64 + fp4_vs_offset(t)], b >= 0);
    uint32_t vw = 0;
    if (staged) {
      vw = codes[t * DG + dg];
    } else {
      const uint8_t* p = c.vc + at * (32 * D) + fp4_v_offset(t, dg * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) vw |= ((p[j * 16] >> (dg & 4 ? 4 : 0)) & 15u) << (4 * j);
    }
    fp4_write8(k + to, kw, ks);
    fp4_write8(v + to, vw, vs);
  };
  if (apart) {
    for (int i = 0; i < 4; ++i) entry(tt + 16 * i, false);
    return;
  }
  for (uint64_t left = starts; left;) {
    const int first = __builtin_ctzll(left);
    left &= left - 1;
    const int end = left ? __builtin_ctzll(left) : count;
    const int64_t at = (int64_t)max(__builtin_amdgcn_readlane(blk, first), 0) * c.KV + h;
    const uint4 w = *reinterpret_cast<const uint4*>(c.vc + at * (32 * D) + fp4_v_offset(4 * g, (dg & ~4) * 8 + (dg & 4) + u));
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    __syncthreads();  // the run before is done with the LDS
#pragma unroll
    for (int T = 0; T < 4; ++T) {
      const uint32_t pairs = turn_bytes<DG>(words[T], u);  // of token 16 T + 4 g + u four channel pairs
      const uint32_t other = __shfl_xor(pairs, 4, 64);
      codes[(16 * T + tt) * DG + dg] = dg & 4 ? gather_nibbles(other >> 4) | (gather_nibbles(pairs >> 4) << 16)
                                              : gather_nibbles(pairs) | (gather_nibbles(other) << 16);
    }
    __syncthreads();
    for (int e0r = first & ~15; e0r < end; e0r += 16) {
      const int e = e0r + tt;
      entry(e >= first && e < end ? e : 64, true);
    }
  }
}

struct Fp4PageArgs {
  const uint8_t* kc;  // first layer
  const uint8_t* ks;
  int64_t kc_stride, ks_stride;  // of a layer, bytes
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

// Pairs of channels as the page bounds compare them: in f16, the values relative to the largest scale (exact where the
// scales lie within 2^22), or in fp32.
__device__ inline f16x2_t fp4_two(uint32_t w, float s, int i, f16x2_t) {
  switch (i) {
    case 0: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0);
    case 1: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1);
    case 2: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2);
    default: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3);
  }
}
__device__ inline f32x2_t fp4_two(uint32_t w, float s, int i, f32x2_t) {
  const uint32_t p = __builtin_bit_cast(uint32_t, fp4_pair(w, s, i));
  return f32x2_t{__uint_as_float(p << 16), __uint_as_float(p & 0xFFFF0000u)};
}
template <int J>
__device__ inline f16x2_t lane_xor_pair(f16x2_t v, int lane) {
  return __builtin_bit_cast(f16x2_t, lane_xor_u32<J>(__builtin_bit_cast(uint32_t, v), lane));
}
template <int J>
__device__ inline f32x2_t lane_xor_pair(f32x2_t v, int lane) {
  return f32x2_t{__uint_as_float(lane_xor_u32<J>(__float_as_uint(v.x), lane)), __uint_as_float(lane_xor_u32<J>(__float_as_uint(v.y), lane))};
}

// Least and largest of 32 channels over the T tokens of each lane and the 16 lanes of a row: lane m ends with pair m.
template <typename V, int T>
__device__ inline void fp4_extremes(const u32x4_t (&w)[T], const float (&s)[T], int lane, V& least, V& largest) {
  V mn[16], mx[16];
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const V x = fp4_two(w[t][j >> 2], s[t], j & 3, V{});
      mn[j] = t ? __builtin_elementwise_min(mn[j], x) : x;
      mx[j] = t ? __builtin_elementwise_max(mx[j], x) : x;
    }
  auto fold = [&](auto step) {  // partner lane ^ J, each lane keeping half of its pairs
    constexpr int J = decltype(step)::value;
    const bool up = lane & J;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const V rn = lane_xor_pair<J>(up ? mn[j] : mn[j + J], lane), rx = lane_xor_pair<J>(up ? mx[j] : mx[j + J], lane);
      mn[j] = __builtin_elementwise_min(up ? mn[j + J] : mn[j], rn);
      mx[j] = __builtin_elementwise_max(up ? mx[j + J] : mx[j], rx);
    }
  };
  fold(std::integral_constant<int, 8>{});
  fold(std::integral_constant<int, 4>{});
  fold(std::integral_constant<int, 2>{});
  fold(std::integral_constant<int, 1>{});
  least = mn[0];
  largest = mx[0];
}

// Min and max of a page's keys per channel, a wave per (page, head, layer).  A lane reads 16 bytes, 32 channels that share
// a scale, of tokens 16 T + m.  Codes times scales are compared two channels at a time in f16, as multiples of
// the page's largest scale, or where scales lie further apart than f16 holds in fp32; the 16 tokens of a row of lanes are
// folded in halves, each lane keeping half of its channels.
template <int D>
__global__ __launch_bounds__(256) void fp4_page_bounds_kernel(Fp4PageArgs a) {
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
  // lane (m, g): of 128 channels group g, of 64 group g % 2 and half of the tokens
  constexpr int T = D / 32;
  const int m = lane & 15, g = lane >> 4, c = g % (D / 32), t0 = D == 128 ? 0 : (g >> 1) * 2;
  for (int64_t u = blockIdx.x * 4 + wave; u < units; u += gridDim.x * 4) {
    const int64_t page = lo + u / a.KV;
    const int h = (int)(u % a.KV);
    const int32_t blk = a.table[req * a.table_stride + page];
    const bool in = blk >= 0 && blk < a.blocks;
    const int64_t at = (int64_t)(in ? blk : 0) * a.KV + h;
    const uint8_t* kp = a.kc + layer * a.kc_stride + at * (32 * D) + ((t0 * (D / 32) + c) * 16 + m) * 16;
    const uint32_t e = *reinterpret_cast<const uint32_t*>(a.ks + layer * a.ks_stride + at * (2 * D) + (c * 16 + m) * 4) >> (8 * t0);
    u32x4_t w[T];
#pragma unroll
    for (int t = 0; t < T; ++t) w[t] = *reinterpret_cast<const u32x4_t*>(kp + t * (D / 32) * 256);
    uint32_t top = 0, low = 255;  // scales of the page's channels here
#pragma unroll
    for (int t = 0; t < T; ++t) {
      top = max(top, e >> (8 * t) & 255u);
      low = min(low, e >> (8 * t) & 255u);
    }
    auto over = [&](auto step) {
      constexpr int J = decltype(step)::value;
      top = max(top, lane_xor_u32<J>(top, lane));
      low = min(low, lane_xor_u32<J>(low, lane));
    };
    over(std::integral_constant<int, 1>{});
    over(std::integral_constant<int, 2>{});
    over(std::integral_constant<int, 4>{});
    over(std::integral_constant<int, 8>{});
    if (D == 64) over(std::integral_constant<int, 32>{});
    float s[T];
    f32x2_t least, largest;
    if (__any(top != kFp4Lost && top - low > 22)) {
#pragma unroll
      for (int t = 0; t < T; ++t) s[t] = fp4_factor(e, t);
      fp4_extremes<f32x2_t, T>(w, s, lane, least, largest);
    } else {
#pragma unroll
      for (int t = 0; t < T; ++t) s[t] = __uint_as_float(((e >> (8 * t) & 255u) + 127u - top) << 23);
      f16x2_t n, x;
      fp4_extremes<f16x2_t, T>(w, s, lane, n, x);
      const float f = __uint_as_float(top << 23);
      least = f32x2_t{(float)n.x * f, (float)n.y * f};
      largest = f32x2_t{(float)x.x * f, (float)x.y * f};
    }
    if (D == 64) {
      least = __builtin_elementwise_min(least, lane_xor_pair<32>(least, lane));
      largest = __builtin_elementwise_max(largest, lane_xor_pair<32>(largest, lane));
      if (lane >= 32) continue;
    }
    const bool lost = !in || top == kFp4Lost;
    const uint2 words = make_uint2((uint32_t)f2bf(least.x) | ((uint32_t)f2bf(largest.x) << 16),
                                   (uint32_t)f2bf(least.y) | ((uint32_t)f2bf(largest.y) << 16));
    *reinterpret_cast<uint2*>(a.bounds + (((int64_t)layer * a.R + req) * a.MP + page) * (a.KV * D) + h * D + c * 32 + m * 2) =
        lost ? make_uint2(0x7FC07FC0u, 0x7FC07FC0u) : words;
  }
}

}  // namespace

int check_cache(const Fp4Cache& c, const char* what) {
  QQ_REQUIRE(c.kc && c.vc && c.ks && c.vs, "%s: null cache pointer", what);
  QQ_REQUIRE(c.blocks > 0 && c.blocks <= kMaxPoolBlocks, "%s: %d blocks, at most %d", what, c.blocks, kMaxPoolBlocks);
  QQ_REQUIRE(c.KV > 0 && c.KV <= 1024, "%s: %d KV heads", what, c.KV);
  QQ_REQUIRE(fp8_dim_ok(c.D), "%s: head_dim %d is not 64 or 128", what, c.D);
  return QQ_OK;
}

}  // namespace qq

using namespace qq;

constexpr int64_t kMaxEntries = ((int64_t)1 << 30) - 64;  // a launch holds fewer than 2^32 threads, 256 for 64 entries
// Values (of K, entries x heads x channels) from which runs of entries are stored, and read, together.  Entries one by one
// and in runs, us, 128 channels, a prompt's run that begins inside a block (six such; a block for every entry): stored,
// 8192 entries and heads 6.9 (6.9; 7.9) and 7.7 (8.1; 14); 13760 9.9 (9.8; 11) and 8.2 (8.6; 18); 131072 59 (57; 25)
// and 22 (23; 31): prompts come in runs, and a decode step's entries go in with its attention.  Of 64 channels, 16384
// 6.9 (7.3) and 7.6 (10.7); 24576 9.1 (8.9) and 8.7 (12.3); 32768 11.1 (11.1) and 9.5 (9.8).  Read, six runs, 32768 8.4
// and 8.4 to 10; 49152 12 and 10; 131072 24 and 18; of 64 channels 65536 8.6 and 9.3, 131072 14.3 and 11.7.
constexpr int64_t kStoreValues = (int64_t)3 << 19, kRowValues = (int64_t)6 << 20;

extern "C" int qq_fp4_store(uint8_t* k_codes, uint8_t* v_codes, uint8_t* k_scale, uint8_t* v_scale, int num_blocks,
                            int kv_heads, int head_dim, const void* k, const void* v, int src_dtype, const int64_t* loc,
                            int64_t n, void* stream) {
  const char* what = "qq_fp4_store";
  const Fp4StoreArgs a{{k_codes, v_codes, k_scale, v_scale, num_blocks, kv_heads, head_dim}, k, v, src_dtype, loc, n, 1};
  const int st = check_cache(a.c, what);
  if (st != QQ_OK) return st;
  QQ_REQUIRE(dtype_ok(src_dtype), "%s: bad dtype", what);
  QQ_REQUIRE(n >= 0 && n <= kMaxEntries, "%s: bad sizes", what);
  if (n == 0) return QQ_OK;
  QQ_REQUIRE(k && v && loc, "%s: null pointer", what);
  QQ_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "%s: k and v must be 16-byte aligned", what);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf = src_dtype == QQ_DTYPE_BF16;
  if (n * kv_heads * head_dim >= kStoreValues) {
    const dim3 grid((unsigned)((n + 63) / 64), kv_heads);
    if (head_dim == 128) {
      if (bf) fp4_store_runs_kernel<128, uint16_t><<<grid, 256, 0, s>>>(a);
      else fp4_store_runs_kernel<128, float><<<grid, 256, 0, s>>>(a);
    } else {
      if (bf) fp4_store_runs_kernel<64, uint16_t><<<grid, 128, 0, s>>>(a);
      else fp4_store_runs_kernel<64, float><<<grid, 128, 0, s>>>(a);
    }
    return check_launch(what);
  }
  const unsigned grid = (unsigned)((n * kv_heads * (head_dim / 4) + 255) / 256);
  if (head_dim == 128) {
    if (bf) fp4_store_kernel<128, uint16_t><<<grid, 256, 0, s>>>(a);
    else fp4_store_kernel<128, float><<<grid, 256, 0, s>>>(a);
  } else {
    if (bf) fp4_store_kernel<64, uint16_t><<<grid, 256, 0, s>>>(a);
    else fp4_store_kernel<64, float><<<grid, 256, 0, s>>>(a);
  }
  return check_launch(what);
}

extern "C" int qq_fp4_rows(const uint8_t* k_codes, const uint8_t* v_codes, const uint8_t* k_scale, const uint8_t* v_scale,
                           int num_blocks, int kv_heads, int head_dim, const int64_t* loc, int64_t n, void* k, void* v,
                           int dst_dtype, void* stream) {
  const char* what = "qq_fp4_rows";
  const Fp4Cache c{const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(v_codes), const_cast<uint8_t*>(k_scale),
                   const_cast<uint8_t*>(v_scale), num_blocks, kv_heads, head_dim};
  const int st = check_cache(c, what);
  if (st != QQ_OK) return st;
  QQ_REQUIRE(dtype_ok(dst_dtype), "%s: bad dtype", what);
  QQ_REQUIRE(n >= 0 && n <= kMaxEntries, "%s: bad sizes", what);
  if (n == 0) return QQ_OK;
  QQ_REQUIRE(loc && k && v, "%s: null pointer", what);
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint16_t *kb = static_cast<uint16_t*>(k), *vb = static_cast<uint16_t*>(v);
  float *kf = static_cast<float*>(k), *vf = static_cast<float*>(v);
  const bool bf = dst_dtype == QQ_DTYPE_BF16;
  if (n * kv_heads * head_dim >= kRowValues) {
    const dim3 grid((unsigned)((n + 63) / 64), kv_heads);
    if (head_dim == 128) {
      if (bf) fp4_rows_runs_kernel<128><<<grid, 256, 0, s>>>(c, loc, n, kb, vb);
      else fp4_rows_runs_kernel<128><<<grid, 256, 0, s>>>(c, loc, n, kf, vf);
    } else {
      if (bf) fp4_rows_runs_kernel<64><<<grid, 128, 0, s>>>(c, loc, n, kb, vb);
      else fp4_rows_runs_kernel<64><<<grid, 128, 0, s>>>(c, loc, n, kf, vf);
    }
    return check_launch(what);
  }
  const unsigned grid = (unsigned)((n * kv_heads * (head_dim / 8) + 255) / 256);
  if (head_dim == 128) {
    if (bf) fp4_rows_kernel<128><<<grid, 256, 0, s>>>(c, loc, n, kb, vb);
    else fp4_rows_kernel<128><<<grid, 256, 0, s>>>(c, loc, n, kf, vf);
  } else {
    if (bf) fp4_rows_kernel<64><<<grid, 256, 0, s>>>(c, loc, n, kb, vb);
    else fp4_rows_kernel<64><<<grid, 256, 0, s>>>(c, loc, n, kf, vf);
  }
  return check_launch(what);
}

extern "C" int qq_fp4_page_bounds(const uint8_t* k_codes, int64_t codes_layer_stride, const uint8_t* k_scale,
                                  int64_t scale_layer_stride, int num_blocks, int kv_heads, int head_dim,
                                  const int32_t* block_table, int64_t block_table_stride, int block_table_rows,
                                  int block_table_cols, const int64_t* req_pool_indices, const int64_t* seq_lens,
                                  const int64_t* prefix_lens, int bs, int decode, int64_t max_new, int n_layers,
                                  uint16_t* page_k_bounds, int max_reqs, int max_pages, int top_k,
                                  int avoid_recent_overlap, int32_t* actual_lens, int32_t* candidate_limit, void* plan,
                                  int64_t plan_bytes, void* stream) {
  const char* what = "qq_fp4_page_bounds";
  uint8_t *codes = const_cast<uint8_t*>(k_codes), *scales = const_cast<uint8_t*>(k_scale);
  const int st = check_cache(Fp4Cache{codes, codes, scales, scales, num_blocks, kv_heads, head_dim}, what);
  if (st != QQ_OK) return st;
  QQ_REQUIRE(bs >= 0 && bs < 65536 && n_layers > 0 && n_layers < 65535 && max_reqs > 0 && max_pages > 0 && max_new >= 0 &&
                 block_table_cols > 0 && block_table_stride >= block_table_cols && block_table_rows > 0,
             "%s: bad sizes", what);
  QQ_REQUIRE(!actual_lens == !candidate_limit, "%s: one of the layout's outputs is missing", what);
  if (bs == 0) return QQ_OK;
  QQ_REQUIRE(block_table && req_pool_indices && seq_lens && page_k_bounds, "%s: null pointer", what);
  Fp4PageArgs a{k_codes, k_scale, codes_layer_stride, scale_layer_stride, num_blocks, kv_heads, block_table, block_table_stride,
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
  if (head_dim == 128) fp4_page_bounds_kernel<128><<<grid, 256, 0, s>>>(a);
  else fp4_page_bounds_kernel<64><<<grid, 256, 0, s>>>(a);
  return check_launch(what);
}
