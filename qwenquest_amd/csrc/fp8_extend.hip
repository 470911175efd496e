// Causal prefill attention of a batch over the 8-bit K/V cache (layout: qq_fp8.h), in one launch
// with no host read of the lengths (reference src/qwenquest/attention/base.py:65-93, ops.py:18-45
// over that cache): request i's n_i new tokens attend positions 0 .. prefix_i + t of its blocks.
//
// The tiles are those of the bf16 prefill: a thread block takes 128 query rows (token, query head
// of one KV head's group), a wave 32 of them, and a K/V tile is a block of the cache, 16 KiB that
// go to the LDS as they lie (two buffers, one barrier a tile; 32 KiB).  The codes are in operand
// order, so a lane's 16-byte LDS reads, one after the other in every quarter wave, are 16 codes of
// its token (K) or channel (V): no bank conflicts and nothing transposed.
//   S^T = K Q^T  v_mfma_f32_32x32x16_bf16, K's codes to bf16 (exact).  (The 8-bit matrix instructions
//   take the codes as they are and a query in two pieces, in the same matrix time: 8192 tokens behind
//   8192 1521 us against 1622.  But they do not add in 32 bits: where one of 64 products carries the sum,
//   it comes out off by 2^-11 of itself, bf16's by 2^-22, and keys have channels like that.)
//   O^T += V^T W^T  v_mfma_f32_32x32x16_f16, V's codes to f16 (exact)
// With t = scale log2(e) ks (q . kc), vs = 2^lv, M a row's running maximum of t that is let lag by 8 (the
// sums are rescaled once it lags more), and R that of t - M + lv, a whole number that likewise lags by
// 8 and falls where M rises, a weight goes into the product as
//   w = 2^(t - M + lv - R + 7),
// so V's scale costs nothing per element, w fills f16's range from the top (7 + 8), and a token is
// lost only where its weight times its block's V scale is under 2^-31 of the row's largest such product
// (larger V scales of tokens that weigh next to nothing take nothing from the others).  w goes to f16's
// 11 bits by truncation (one instruction for two weights) of w (1 + 0.72 * 2^-11): truncation takes
// half a step on average, 2^-10 / 2 over the significand's 1 .. 2, in the mean 0.72 * 2^-11.
// A weight is off by 0.64 * 2^-10 at most, an output by that of sum p |v|, where its own rounding
// is 2^-8 of it; the weights' sum stays in fp32.  (Against 64 bits the output of 8192 tokens behind 8192
// is off by 0.001672 of its size, of which the bf16 rounding alone is 0.001658.  A second f16 piece of
// the weights, 22 bits, leaves that alone, and costs another value product: 1601 -> 2167 us, 3440
// tokens of 6 prompts 182 -> 232.)
//
// Bound: the matrix cores and, beside them, the softmax's vector instructions: by the counters
// the matrix pipes are busy for 49 % of the time and the vector units for 65 % (4 cycles for each of
// their other instructions), waves wait for memory for 14 % of theirs, and no LDS access meets a bank
// conflict.  Measured, 32 query heads on 4 of 128: 8192 tokens behind 8192 1618 us (1.02 PFLOP/s of the
// formula's operations; 1598 to 1635 by box), 3440 tokens of 6 prompts 173 to 187 with their store, where
// the longest tile chain is as long as the rest.
#include "qq_extend_dev.h"
#include "qq_fp8.h"

namespace qq {
namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kLift = 7, kSlack = 8;  // w <= 2^(7 + 8) * kRound < f16's 65504
constexpr float kRound = 1.0003516f, kRoundLog2 = 5.0713e-4f;  // 1 + 0.72 * 2^-11
constexpr float kExpFloor = -60.0f;  // of lv - R: f16 has nothing left of such weights, their fp32 sum has

struct Fp8ExtendArgs {
  const uint16_t* q;  // [n, H, D]
  int H, KV, G;
  Fp8Cache c;
  const int32_t* table;
  int64_t table_stride;
  int64_t r2t_stride, r2t_rows;  // the table's width in tokens, its rows
  const int64_t* rpi;
  const int64_t* seq;
  const int64_t* prefix;
  const int64_t* ext;
  int bs, n;
  int tiles;   // query tiles the grid holds (an upper bound of the requests' tiles), one more at its end
  int splits;  // K/V splits the grid holds
  float sl2;   // scale * log2(e)
  uint16_t* out;
  float* part_o;   // [splits, KV, tiles, 128 rows, D]
  float* part_ml;  // [splits, KV, tiles, 128 rows, 2]
};

// Sixteen codes as the operands of two steps.
__device__ inline void codes16(uint4 w, bf16x8_t& a, bf16x8_t& b) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  u32x4_t y[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i >> 1][(i & 1) * 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], 1.0f, false));
    y[i >> 1][(i & 1) * 2 + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], 1.0f, true));
  }
  a = __builtin_bit_cast(bf16x8_t, y[0]);
  b = __builtin_bit_cast(bf16x8_t, y[1]);
}
__device__ inline f16x8_t codes_f16(uint32_t a, uint32_t b) {
  u32x4_t w;
  w.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false));
  w.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true));
  w.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false));
  w.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true));
  return __builtin_bit_cast(f16x8_t, w);
}

// find_tile's answer is the same in every lane; in scalar registers it makes the K/V loop's control
// and its lookups scalar.
__device__ inline ExtendTile uniform_tile(const ExtendTile& t) {
  auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  return {u(t.b), u(t.tile), u(t.q0), u(t.n), u(t.past), u(t.req), u(t.kv_len), u(t.prefix)};
}

// Words that this launch does not write, through the scalar cache.
typedef const __attribute__((address_space(4))) int32_t* scalar_words_t;
typedef const __attribute__((address_space(4))) float* scalar_floats_t;

template <int D>
__global__ __launch_bounds__(64 * kExtWaves, 2) void fp8_extend_kernel(Fp8ExtendArgs a) {
  constexpr int KI = D / 32, NC = D / 32;  // pairs of 16-channel pieces of K, 32-channel tiles of the output
  constexpr int kHead = 64 * D;            // bytes of a block and head
  extern __shared__ __align__(16) unsigned char sm[];  // [buffer][K, V][kHead]
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)sm;
  // block -> (KV head, tile, split): heads fastest, so that an XCD (blocks round robin) keeps to
  // KV / 8 of the heads and its L2 to their blocks; the last tiles of the requests, which attend
  // the most, first
  const int h = blockIdx.x % a.KV;
  const int rest = blockIdx.x / a.KV;
  const bool tail = rest >= a.tiles * a.splits;  // the grid's last tile, past every request's
  const int t_lin = tail ? a.tiles : a.tiles - 1 - rest % a.tiles;
  const int split = tail ? 0 : rest / a.tiles;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int lo = lane & 31, hf = lane >> 5;
  const ExtendTile et = uniform_tile(find_tile(a, t_lin));
  const int64_t row_out = (int64_t)a.H * D;
  if (et.b < 0) {
    // rows of q past the requests' tokens have no answer: NaN, in 8-byte pieces, shared by the
    // tiles past the requests' - the grid's last one always is
    const int past_tiles = a.tiles + 1 - (t_lin - et.past);
    const int pieces = a.G * D / 4;  // of a row, per KV head
    if (split == 0)
      for (int64_t i = et.past * 64 * kExtWaves + tid; i < (int64_t)(a.n - et.q0) * pieces; i += (int64_t)past_tiles * 64 * kExtWaves)
        *reinterpret_cast<uint2*>(a.out + (et.q0 + i / pieces) * row_out + ((int64_t)h * pieces + i % pieces) * 4) =
            make_uint2(0x7FC07FC0u, 0x7FC07FC0u);
    return;
  }
  const int kv_len = et.kv_len, prefix = et.prefix;
  const int rows_n = et.n * a.G;
  const int r0 = et.tile * kExtRows;
  const int r = min(r0 + wave * 32 + lo, rows_n - 1);  // this lane's query row
  const int tok = r / a.G;
  const uint16_t* qp = a.q + (int64_t)(et.q0 + tok) * row_out + (int64_t)(h * a.G + r - tok * a.G) * D;
  const int lim = min(kv_len, prefix + tok + 1);  // attended positions of this row
  const int tok_first = r0 / a.G, tok_last = (min(r0 + kExtRows, rows_n) - 1) / a.G;
  const int lim_full = min(kv_len, prefix + tok_first + 1);
  const int lim_blk = min(kv_len, prefix + tok_last + 1);
  // K/V tiles of this split
  const int nt_all = lim_blk > 0 ? (lim_blk + kExtTile - 1) / kExtTile : 0;
  const int chunk = split_chunk(nt_all, a.splits);
  const bool whole = nt_all <= chunk;  // one split does it all and writes the output
  const int j_begin = split * chunk, j_end = min(nt_all, j_begin + chunk);
  if (j_begin >= j_end && split != 0) return;

  // channels of step (i, p): (2 i + hf) * 16 + 8 p .. + 7
  bf16x8_t qb[2 * KI];
#pragma unroll
  for (int i = 0; i < 2 * KI; ++i)
    qb[i] = *reinterpret_cast<const bf16x8_t*>(qp + ((i >> 1) * 2 + hf) * 16 + (i & 1) * 8);

  const scalar_words_t bt = (scalar_words_t)(uintptr_t)(a.table + (int64_t)max(et.req, 0) * a.table_stride);
  const scalar_floats_t ksp = (scalar_floats_t)(uintptr_t)(a.c.ks + h), vsp = (scalar_floats_t)(uintptr_t)(a.c.vs + h);
  bool bad = et.req < 0;
  // a tile's block; padding and ids outside the cache are read as padding, and spoil the answer
  auto block_of_word = [&](int word) {
    const bool ok = word > 0 && word < a.c.blocks;
    bad |= !ok;
    return ok ? word : 0;
  };
  auto load_tile = [&](int buf, int blk) {
    const int64_t at = ((int64_t)blk * a.KV + h) * kHead + wave * (kHead / 4) + lane * 16;
    const uint32_t base = lds0 + (uint32_t)(buf * 2 * kHead + wave * (kHead / 4));
#pragma unroll
    for (int i = 0; i < kHead / 4096; ++i) {
      load_lds16(a.c.kc + at + i * 1024, base + i * 1024);
      load_lds16(a.c.vc + at + i * 1024, base + kHead + i * 1024);
    }
  };
  float16_t o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = 0.0f;
  float M = -INFINITY, R = 0.0f, L = 0.0f;
  // LDS addresses of this lane's pieces: K token lo of a half, pieces 2 i + hf; V channel lo of a
  // tile of 32, token groups hf and hf + 2
  const int k_off = (lo >> 4) * 16 * D + (lo & 15) * 16 + hf * 256;
  const int v_off = (lo >> 4) * 1024 + (lo & 15) * 16 + hf * 256;
  int word = 0, buf = 0;  // the table's word of the tile after the one in flight
  float ks = 0.0f, vs = 0.0f, ks_next = 0.0f, vs_next = 0.0f;
  if (j_begin < j_end) {
    const int blk = block_of_word(bt[j_begin]);
    ks_next = ksp[(int64_t)blk * a.KV];
    vs_next = vsp[(int64_t)blk * a.KV];
    load_tile(0, blk);
    word = bt[min(j_begin + 1, j_end - 1)];
  }
  for (int j = j_begin; j < j_end; ++j) {
    ks = ks_next;
    vs = vs_next;
    tile_barrier();
    if (j + 1 < j_end) {
      const int blk = block_of_word(word);
      load_tile(buf ^ 1, blk);
      ks_next = ksp[(int64_t)blk * a.KV];
      vs_next = vsp[(int64_t)blk * a.KV];
      word = bt[min(j + 2, j_end - 1)];
    }
    const unsigned char* sk = sm + buf * 2 * kHead + k_off;
    const unsigned char* sv = sm + buf * 2 * kHead + kHead + v_off;
    buf ^= 1;
    // S^T[token 32 t + 8 (i / 4) + 4 hf + i % 4][row lo] in s[t][i]
    float16_t s[2];
    uint4 kw[2][KI], vw[NC][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < KI; ++i) kw[t][i] = *reinterpret_cast<const uint4*>(sk + t * 32 * D + i * 512);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
    }
    // (independent accumulators one after the other)
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      bf16x8_t k0[2], k1[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) codes16(kw[t][i], k0[t], k1[t]);
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k0[t], qb[2 * i], s[t], 0, 0, 0);
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k1[t], qb[2 * i + 1], s[t], 0, 0, 0);
    }
    // the values' codes arrive under the softmax
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < NC; ++x) {
      vw[x][0] = *reinterpret_cast<const uint4*>(sv + x * 2048);
      vw[x][1] = *reinterpret_cast<const uint4*>(sv + x * 2048 + 512);
    }
    __builtin_amdgcn_sched_barrier(0);
    const bool edge = (j + 1) * kExtTile > lim_full;  // block-uniform: some row's limit is inside this tile
    const int left = lim - j * kExtTile - 4 * hf;
    if (edge) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = (t * 32 + 8 * (i / 4) + i % 4) < left ? s[t][i] : -INFINITY;
    }
    // a positive factor, also where the scale underflows; NaN stays
    float c = ks * a.sl2;
    c = c < 1.2e-38f ? 1.2e-38f : c;
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
    mx = fmaxf(mx, lane_xor32(mx, lane)) * c;
    const float lv = vs != vs ? 0.0f : (float)exponent_of(vs);
    if (__any(mx > M + kSlack || mx + lv > M + R + kSlack)) {
      const float Mn = fmaxf(M, mx);
      const float was = M == -INFINITY ? -INFINITY : R + (M - Mn);
      // (at least kScaleMin, but for scores that are not finite and a row without any so far)
      const float Rn = Mn == -INFINITY ? R : fmaxf(ceilf(fmaxf(lv + (mx - Mn), was)), -126.0f);
      const float am = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - Mn);
      const float ao = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(fmaxf(was - Rn, -126.0f));
      L *= am;
#pragma unroll
      for (int x = 0; x < NC; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[x][i] *= ao;
      M = Mn;
      R = Rn;
    }
    const float lift = fmaxf(lv - R, kExpFloor) + (float)kLift;
    // NaN where the block's V scale is
    float bias = lift + kRoundLog2 + (vs != vs ? vs : 0.0f);
    bias = M == -INFINITY ? bias : bias - M;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], c, bias));
    if (edge) {  // a masked token weighs nothing whatever its block's scales are
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = (t * 32 + 8 * (i / 4) + i % 4) < left ? s[t][i] : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += s[t][i];
    L += __builtin_amdgcn_ldexpf(sum * (1.0f / kRound), -(int)lift);
    // O^T += V^T W^T, 16 tokens at a time
    u32x4_t wv[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        wv[u][x] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(s[u >> 1][(u & 1) * 8 + 2 * x], s[u >> 1][(u & 1) * 8 + 2 * x + 1]));
#pragma unroll
    for (int x = 0; x < NC; ++x) {
      const uint4 va = vw[x][0], vb = vw[x][1];
      const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
      for (int u = 0; u < 4; ++u)
        o[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_f16(wa[u], wb[u]), __builtin_bit_cast(f16x8_t, wv[u]), o[x], 0, 0, 0);
    }
  }
  L += lane_xor32(L, lane);
  if (__syncthreads_or(bad)) L = __builtin_nanf("");  // a block that is not there: no answer
  const bool mine = r0 + wave * 32 + lo < rows_n;
  const float unit = __builtin_amdgcn_exp2f(R - (float)kLift);
  if (whole) {
    if (!mine) return;
    uint16_t* op = a.out + (qp - a.q) + 4 * hf;
    const float inv = unit / L;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t w0 = (uint32_t)f2bf(o[c][4 * g] * inv) | ((uint32_t)f2bf(o[c][4 * g + 1] * inv) << 16);
        const uint32_t w1 = (uint32_t)f2bf(o[c][4 * g + 2] * inv) | ((uint32_t)f2bf(o[c][4 * g + 3] * inv) << 16);
        *reinterpret_cast<uint2*>(op + c * 32 + g * 8) = make_uint2(w0, w1);
      }
    return;
  }
  const int64_t pr = (((int64_t)split * a.KV + h) * a.tiles + t_lin) * kExtRows + wave * 32 + lo;
  float* po = a.part_o + pr * D + 4 * hf;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(po + c * 32 + g * 8) =
          make_float4(o[c][4 * g] * unit, o[c][4 * g + 1] * unit, o[c][4 * g + 2] * unit, o[c][4 * g + 3] * unit);
  if (hf == 0) *reinterpret_cast<float2*>(a.part_ml + pr * 2) = make_float2(M, L);
}

template <int D>
void launch(const Fp8ExtendArgs& a, int64_t grid, hipStream_t s) {
  fp8_extend_kernel<D><<<(int)grid, 64 * kExtWaves, 4 * 64 * D, s>>>(a);
  if (a.splits > 1) extend_merge_kernel<D><<<dim3(a.tiles, a.KV, kExtRows / 8), 256, 0, s>>>(a);
}

}  // namespace
}  // namespace qq

using namespace qq;

extern "C" int64_t qq_fp8_extend_workspace_bytes(int64_t n, int bs, int num_q_heads, int kv_heads, int head_dim,
                                                 int block_table_cols) {
  if (n <= 0 || bs <= 0 || kv_heads <= 0 || num_q_heads < kv_heads || block_table_cols <= 0) return 0;
  const int64_t tiles = extend_tiles(n, bs, num_q_heads / kv_heads);
  const int splits = extend_splits(tiles, kv_heads, (int64_t)block_table_cols * kCacheTokens);
  return splits > 1 ? splits * kv_heads * tiles * kExtRows * (head_dim + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int qq_fp8_extend_attention(const void* q, int num_q_heads, const uint8_t* k_codes, const uint8_t* v_codes,
                                       const float* k_scale, const float* v_scale, int num_blocks, int kv_heads,
                                       int head_dim, const int32_t* block_table, int64_t block_table_stride,
                                       int block_table_rows, int block_table_cols, const int64_t* req_pool_indices,
                                       const int64_t* seq_lens, const int64_t* prefix_lens, const int64_t* extend_lens,
                                       int bs, int64_t n, float scale, void* out, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  const char* what = "qq_fp8_extend_attention";
  const Fp8Cache c{const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(v_codes), const_cast<float*>(k_scale),
                   const_cast<float*>(v_scale), num_blocks, kv_heads, head_dim};
  const int ok = check_cache(c, what);
  if (ok != QQ_OK) return ok;
  QQ_REQUIRE(num_q_heads > 0 && num_q_heads % kv_heads == 0, "%s: q_heads %d not divisible by kv_heads %d", what,
             num_q_heads, kv_heads);
  QQ_REQUIRE(scale > 0.0f && scale < INFINITY, "%s: the scale must be positive", what);
  const int G = num_q_heads / kv_heads;
  QQ_REQUIRE(bs >= 0 && n >= 0 && n * G < (int64_t)1 << 30 && block_table_rows > 0 && block_table_cols > 0 &&
                 block_table_cols <= kMaxPoolBlocks && block_table_stride >= block_table_cols,
             "%s: bad sizes", what);
  if (bs == 0 || n == 0) return QQ_OK;
  QQ_REQUIRE(q && block_table && req_pool_indices && seq_lens && prefix_lens && extend_lens && out, "%s: null pointer", what);
  QQ_REQUIRE(((uintptr_t)q | (uintptr_t)out) % 16 == 0, "%s: q and out must be 16-byte aligned", what);
  const int64_t need = qq_fp8_extend_workspace_bytes(n, bs, num_q_heads, kv_heads, head_dim, block_table_cols);
  QQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace %lld bytes < %lld needed", what,
             (long long)workspace_bytes, (long long)need);
  Fp8ExtendArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.H = num_q_heads;
  a.KV = kv_heads;
  a.G = G;
  a.c = c;
  a.table = block_table;
  a.table_stride = block_table_stride;
  a.r2t_stride = min((int64_t)block_table_cols * kCacheTokens, ((int64_t)1 << 30) - kCacheTokens);
  a.r2t_rows = block_table_rows;
  a.rpi = req_pool_indices;
  a.seq = seq_lens;
  a.prefix = prefix_lens;
  a.ext = extend_lens;
  a.bs = bs;
  a.n = (int)n;
  const int64_t tiles = extend_tiles(n, bs, G);
  a.splits = extend_splits(tiles, kv_heads, (int64_t)block_table_cols * kCacheTokens);
  const int64_t grid = (tiles * a.splits + 1) * kv_heads;
  QQ_REQUIRE(grid < (int64_t)1 << 31, "%s: too many query rows", what);
  a.tiles = (int)tiles;
  a.sl2 = scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o ? a.part_o + a.splits * kv_heads * tiles * kExtRows * head_dim : nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128) launch<128>(a, grid, s);
  else launch<64>(a, grid, s);
  return check_launch(what);
}
