// Causal prefill attention of a batch over the 4-bit K/V cache (layout: qq_fp4.h), in one launch
// with no host read of the lengths (reference src/qwenquest/attention/base.py:65-93, ops.py:18-45
// over that cache): request i's n_i new tokens attend positions 0 .. prefix_i + t of its blocks.
//
// The tiles are those of the other prefills: a thread block takes 128 query rows (token, query head
// of one KV head's group), a wave 32 of them, and a K/V tile is a block of the cache, 8 KiB of codes that
// go to the LDS as they lie (two buffers, one barrier a tile; 16 KiB); a lane's scales come from memory a
// tile ahead.
//   S^T = K Q^T  v_mfma_f32_32x32x16_bf16, K's codes times their scales as bf16 (exact)
//   O^T += V^T W^T  v_mfma_f32_32x32x16_f16, V's codes as f16 (exact)
// With t = scale log2(e) (q . k), 2^E a token's V scale and N a row's
// running maximum of t + E, which is let lag by 8 (the sums are rescaled once it lags more), a weight goes
// into the product as
//   w = 2^(t + E - N + 7),
// which fills f16's range from the top (7 + 8); the weights' sum adds w 2^(1 - E), in fp32.  E and 2^(1 - E) of a lane's 32 tokens
// come by matrix instructions, a step of K Q^T that holds them as channels.  w goes to f16's
// 11 bits by truncation (one instruction for two weights) of w (1 + 0.72 * 2^-11): truncation takes
// half a step on average, 2^-10 / 2 over the significand's 1 .. 2, in the mean 0.72 * 2^-11.
// A weight from 2^-14 on is off by 0.64 * 2^-10 at most, an output by that of sum p |v|, where its own rounding
// is 2^-8 of it; smaller ones are whole steps of 2^-24: each token is off by 2^-31 of the row's largest p 2^E at most, times a code
// of up to 6, which shows in channels where the tokens that weigh most hold 0.  (A second f16 piece of the weights is another value
// product: a third more time over the 8-bit cache, and the same error against 64 bits.)
// The sum has no such end.  V's exponents span 109, so tokens that count in it by their number may lie below 2^-126 in w and in the
// rescaling: that goes in two halves, and a tile with an E below kLowE, values under 2^-27, adds weights of their own, 2^kUp times as
// large (then a token is missing only under 2^-88 of another one; above kLowE under 2^-44).
//
// Bound: the matrix cores, near the clock that they hold: 8192 tokens behind 8192, 32 heads on 4 of 128, 1592 to 1664 us (by
// card): 36 matrix instructions a tile and wave are 1.11 to 1.16 PFLOP/s, where a plain product of 8192^3 reaches 1.225; of the
// formula's 0.99 to 1.04.  (The sum's range, V scale bytes behind a context and scores past 2^22 take 0.2 %; at 64 channels, 1068 us,
// where the vector units are the bound, 2 %.)  E and 2^(1 - E) by lane exchanges instead of matrix instructions 1953; weights and products one
// after the other 1690.  Not taken: the next tile's scores between this one's products (256 registers, 1693), three
// blocks a CU with the queries in the LDS (1635), wave priorities (no change).  A short batch by its longest request's
// tiles: 3440 new of 8330 tokens 174 to 179 us with the store.
#include "qq_extend_dev.h"
#include "qq_fp4.h"

namespace qq {
namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kLift = 7, kSlack = 8, kLowE = -30, kUp = 64;  // w <= 2^(7 + 8) * kRound < f16's 65504
constexpr float kDown = 0x1p-64f;  // 2^-kUp
constexpr float kFar = 0x1p22f;    // from there on t + E - N is off by more than 1/2 where the product is not rounded before: w would pass f16's end
constexpr float kRound = 1.0003516f, kRoundLog2 = 5.0713e-4f;  // 1 + 0.72 * 2^-11

struct Fp4ExtendArgs {
  const uint16_t* q;  // [n, H, D]
  int H, KV, G;
  Fp4Cache c;
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
  float sl2;   // scale * log2(e) / q_factor
  float q_factor;  // a power of two, 1 but for scales far from 1: sl2 within 2^+-100
  uint16_t* out;
  float* part_o;   // [splits, KV, tiles, 128 rows, D]
  float* part_ml;  // [splits, KV, tiles, 128 rows, 2]
};

// Eight codes times s as an operand of K Q^T, and as they are as one of V^T W^T.
__device__ inline bf16x8_t fp4_bf16(uint32_t w, float s) {
  u32x4_t y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_bit_cast(uint32_t, fp4_pair(w, s, i));
  return __builtin_bit_cast(bf16x8_t, y);
}
__device__ inline f16x8_t fp4_f16(uint32_t w) {
  u32x4_t y;
  y.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0));
  y.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1));
  y.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2));
  y.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3));
  return __builtin_bit_cast(f16x8_t, y);
}

__device__ inline float trunc_bf16(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }
__device__ inline uint32_t pack_trunc(float even, float odd) {
  return __builtin_amdgcn_perm(__float_as_uint(odd), __float_as_uint(even), 0x07060302u);
}

// find_tile's answer is the same in every lane; in scalar registers it makes the K/V loop's control
// and its lookups scalar.
__device__ inline ExtendTile uniform_tile(const ExtendTile& t) {
  auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  return {u(t.b), u(t.tile), u(t.q0), u(t.n), u(t.past), u(t.req), u(t.kv_len), u(t.prefix)};
}

// Words that this launch does not write, through the scalar cache.
typedef const __attribute__((address_space(4))) int32_t* scalar_words_t;

template <int D>
__global__ __launch_bounds__(64 * kExtWaves, 2) void fp4_extend_kernel(Fp4ExtendArgs a) {
  constexpr int KI = D / 64, NC = D / 32;  // pairs of 32-channel pieces of K, 32-channel tiles of the output
  constexpr int kHead = 32 * D;            // bytes of a block and head
  __shared__ __align__(16) unsigned char sm[4 * kHead];  // [buffer][K, V][kHead]
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

  // channels of step (i, p): (2 i + hf) * 32 + 8 p .. + 7
  bf16x8_t qb[4 * KI];
#pragma unroll
  for (int i = 0; i < 4 * KI; ++i)
    qb[i] = *reinterpret_cast<const bf16x8_t*>(qp + ((i >> 2) * 2 + hf) * 32 + (i & 3) * 8);
  if (a.q_factor != 1.0f) {
#pragma unroll
    for (int i = 0; i < 4 * KI; ++i)
#pragma unroll
      for (int x = 0; x < 8; ++x) qb[i][x] = (__bf16)((float)qb[i][x] * a.q_factor);
  }
  // A further step over channels of which K's side holds (E, E, E, 2^(1 - E)) of a token: against 1 / sl2 in three bf16
  // pieces it adds E / sl2 to every product; against (0, 0, 0, 1) it spreads 2^(1 - E) as the products lie
  bf16x8_t q_add, q_spread;
  {
    const float r = 1.0f / a.sl2, r1 = r - trunc_bf16(r), r2 = r1 - trunc_bf16(r1);
    u32x4_t w = {0, 0, 0, 0}, v = {0, 0, 0, 0};
    if (hf == 0) {
      w.x = pack_trunc(r, r1);
      w.y = __float_as_uint(r2) >> 16;
      v.y = 0x3F800000u;
    }
    q_add = __builtin_bit_cast(bf16x8_t, w);
    q_spread = __builtin_bit_cast(bf16x8_t, v);
  }

  const scalar_words_t bt = (scalar_words_t)(uintptr_t)(a.table + (int64_t)max(et.req, 0) * a.table_stride);
  // this lane's scales: of K pieces 2 i + hf and of V, of tokens lo of both halves (of K's 16 T + lo % 16, a word)
  const uint8_t* ksp = a.c.ks + (int64_t)h * (2 * D) + (hf * 16 + (lo & 15)) * 4;
  const uint8_t* vsp = a.c.vs + (int64_t)h * 64 + ((lo & 15) >> 2) * 16 + (lo >> 4) * 4 + (lo & 3);
  bool bad = et.req < 0;
  // a tile's block; padding and ids outside the cache are read as padding, and spoil the answer
  auto block_of_word = [&](int word) {
    const bool ok = word > 0 && word < a.c.blocks;
    bad |= !ok;
    return ok ? word : 0;
  };
  // 4 KiB (of 64 channels: 2) of codes each for K and V, a KiB per wave and load
  auto load_tile = [&](int buf, int blk) {
    const int64_t at = ((int64_t)blk * a.KV + h) * kHead + lane * 16;
    const uint32_t base = lds0 + (uint32_t)(buf * 2 * kHead);
    if (D == 128) {
      load_lds16(a.c.kc + at + wave * 1024, base + wave * 1024);
      load_lds16(a.c.vc + at + wave * 1024, base + kHead + wave * 1024);
    } else {
      load_lds16((wave < 2 ? a.c.kc : a.c.vc) + at + (wave & 1) * 1024, base + wave * 1024);
    }
  };
  uint32_t ks[KI], ks_next[KI], vs[2], vs_next[2];
  auto load_scales = [&](int blk) {
    const int64_t at = (int64_t)blk * a.KV;
#pragma unroll
    for (int i = 0; i < KI; ++i) ks_next[i] = *reinterpret_cast<const uint32_t*>(ksp + at * (2 * D) + i * 128);
#pragma unroll
    for (int t = 0; t < 2; ++t) vs_next[t] = vsp[at * 64 + t * 8];
  };
  float16_t o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = 0.0f;
  float N = -INFINITY, L = 0.0f;
  float bias = (float)kLift + kRoundLog2, bar = -INFINITY;  // what goes to every exponent, the score that brings another
  // LDS addresses of this lane's pieces: K token lo of a half, piece 2 i + hf; V channel lo of 64 and the
  // one 32 further on, token groups hf and hf + 2
  const int k_off = (lo >> 4) * 8 * D + (lo & 15) * 16 + hf * 256;
  const int v_off = (lo >> 4) * 1024 + (lo & 15) * 16 + hf * 256;
  int word = 0, buf = 0;  // the table's word of the tile after the one in flight
  if (j_begin < j_end) {
    const int blk = block_of_word(bt[j_begin]);
    load_scales(blk);
    load_tile(0, blk);
    word = bt[min(j_begin + 1, j_end - 1)];
  }
  for (int j = j_begin; j < j_end; ++j) {
    tile_barrier();
#pragma unroll
    for (int i = 0; i < KI; ++i) ks[i] = ks_next[i] >> (8 * (lo >> 4));  // bytes 0 and 2: the lane's tokens of the halves
#pragma unroll
    for (int t = 0; t < 2; ++t) vs[t] = max(vs_next[t], 1u);  // (of a byte 0 2^(1 - E) would be infinite)
    if ((j + 1) * kExtTile > lim_blk) {  // behind what the block attends the bytes may be any, and count for 127
#pragma unroll
      for (int t = 0; t < 2; ++t) vs[t] = j * kExtTile + t * 32 + lo < lim_blk ? vs[t] : 127u;
    }
    if (j + 1 < j_end) {
      const int blk = block_of_word(word);
      load_tile(buf ^ 1, blk);
      load_scales(blk);
      word = bt[min(j + 2, j_end - 1)];
    }
    const unsigned char* sk = sm + buf * 2 * kHead + k_off;
    const unsigned char* sv = sm + buf * 2 * kHead + kHead + v_off;
    buf ^= 1;
    // S^T[token 32 t + 8 (i / 4) + 4 hf + i % 4][row lo] in s[t][i]
    float16_t s[2];
    u32x4_t kw[2][KI], vw[KI][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < KI; ++i) kw[t][i] = *reinterpret_cast<const u32x4_t*>(sk + t * 16 * D + i * 512);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
    }
    // (independent accumulators one after the other)
#pragma unroll
    for (int i = 0; i < KI; ++i)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        bf16x8_t kb[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) kb[t] = fp4_bf16(kw[t][i][p], fp4_factor(ks[i], 2 * t));
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kb[t], qb[4 * i + p], s[t], 0, 0, 0);
      }
    float16_t spread[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t e = __float_as_uint((float)vs[t] - 127.0f);
      const u32x4_t w = {__builtin_amdgcn_perm(e, e, 0x07060706u), (e >> 16) | ((255u - vs[t]) << 23), 0, 0};
      const bf16x8_t ext = __builtin_bit_cast(bf16x8_t, w);
#pragma unroll
      for (int i = 0; i < 16; ++i) spread[t][i] = 0.0f;
      s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ext, q_add, s[t], 0, 0, 0);
      spread[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ext, q_spread, spread[t], 0, 0, 0);
    }
    // the values' codes arrive under the softmax
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < KI; ++x) {
      vw[x][0] = *reinterpret_cast<const u32x4_t*>(sv + x * 2048);
      vw[x][1] = *reinterpret_cast<const u32x4_t*>(sv + x * 2048 + 512);
    }
    __builtin_amdgcn_sched_barrier(0);
    const bool edge = (j + 1) * kExtTile > lim_full;  // block-uniform: some row's limit is inside this tile
    const int left = lim - j * kExtTile - 4 * hf;
    if (edge) {
      int last = left;
      __asm__ volatile("" : "+v"(last));  // a branch, not 64 selects in every tile
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = (t * 32 + 8 * (i / 4) + i % 4) < last ? s[t][i] : -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
    mx = fmaxf(mx, lane_xor32(mx, lane)) * a.sl2;
    const bool small = min(vs[0], vs[1]) < (uint32_t)(127 + kLowE);
    if (__any(mx > bar || small)) {
      // (each row by its own maximum, whatever brought its wave here)
      const float Nn = mx - N > kSlack ? mx : N, am = N == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(N - Nn);
      L = scaled_sum(L, N, Nn, am);
#pragma unroll
      for (int x = 0; x < NC; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[x][i] *= am;
      N = Nn;
      const float base = N == -INFINITY ? 0.0f : N;
      const bool far = fabsf(base) > kFar;
      bar = far ? -INFINITY : N + kSlack;
      bias = (float)kLift + kRoundLog2 - (far ? 0.0f : base);
      if (__any(far)) {  // differences first, of rounded products: 0 where the maximum is
        const float inv = 1.0f / a.sl2;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[t][i] = far ? (s[t][i] * a.sl2 - base) * inv : s[t][i];
      }
      if (__any(small)) {  // the tile's part of the sum here, none below
        float part = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            part = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], a.sl2, bias + kUp)), spread[t][i] * kDown, part);
            spread[t][i] = 0.0f;
          }
        L += part;
      }
    }
    float sum = 0.0f;
    // O^T += V^T W^T, 16 tokens at a time, the products of some under the weights of the next
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float w[8];
      u32x4_t wv;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        float& e = w[x];
        e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u >> 1][(u & 1) * 8 + x], a.sl2, bias));
        sum = __builtin_fmaf(e, spread[u >> 1][(u & 1) * 8 + x], sum);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) wv[x] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(w[x], w[4 + x]));
      const f16x8_t wf = __builtin_bit_cast(f16x8_t, wv);
#pragma unroll
      for (int x = 0; x < KI; ++x) {
        const uint32_t va = vw[x][0][u], vb = vw[x][1][u];
        o[2 * x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp4_f16(fp4_lower(va, vb)), wf, o[2 * x], 0, 0, 0);
        o[2 * x + 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp4_f16(fp4_upper(va, vb)), wf, o[2 * x + 1], 0, 0, 0);
      }
    }
    L += sum;
  }
  L += lane_xor32(L, lane);
  if (__syncthreads_or(bad)) L = __builtin_nanf("");  // a block that is not there: no answer
  const bool mine = r0 + wave * 32 + lo < rows_n;
  constexpr float unit = 2.0f * kRound;  // L counts in 2^-1 of o's unit, and what the truncation takes
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
  if (hf == 0) *reinterpret_cast<float2*>(a.part_ml + pr * 2) = make_float2(N, L);
}

template <int D>
void launch(const Fp4ExtendArgs& a, int64_t grid, hipStream_t s) {
  fp4_extend_kernel<D><<<(int)grid, 64 * kExtWaves, 0, s>>>(a);
  if (a.splits > 1) extend_merge_kernel<D><<<dim3(a.tiles, a.KV, kExtRows / 8), 256, 0, s>>>(a);
}

}  // namespace
}  // namespace qq

using namespace qq;

extern "C" int64_t qq_fp4_extend_workspace_bytes(int64_t n, int bs, int num_q_heads, int kv_heads, int head_dim,
                                                 int block_table_cols) {
  if (n <= 0 || bs <= 0 || kv_heads <= 0 || num_q_heads < kv_heads || block_table_cols <= 0) return 0;
  const int64_t tiles = extend_tiles(n, bs, num_q_heads / kv_heads);
  const int splits = extend_splits(tiles, kv_heads, (int64_t)block_table_cols * kCacheTokens);
  return splits > 1 ? splits * kv_heads * tiles * kExtRows * (head_dim + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int qq_fp4_extend_attention(const void* q, int num_q_heads, const uint8_t* k_codes, const uint8_t* v_codes,
                                       const uint8_t* k_scale, const uint8_t* v_scale, int num_blocks, int kv_heads,
                                       int head_dim, const int32_t* block_table, int64_t block_table_stride,
                                       int block_table_rows, int block_table_cols, const int64_t* req_pool_indices,
                                       const int64_t* seq_lens, const int64_t* prefix_lens, const int64_t* extend_lens,
                                       int bs, int64_t n, float scale, void* out, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  const char* what = "qq_fp4_extend_attention";
  const Fp4Cache c{const_cast<uint8_t*>(k_codes), const_cast<uint8_t*>(v_codes), const_cast<uint8_t*>(k_scale),
                   const_cast<uint8_t*>(v_scale), num_blocks, kv_heads, head_dim};
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
  const int64_t need = qq_fp4_extend_workspace_bytes(n, bs, num_q_heads, kv_heads, head_dim, block_table_cols);
  QQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace %lld bytes < %lld needed", what,
             (long long)workspace_bytes, (long long)need);
  Fp4ExtendArgs a{};
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
  QQ_REQUIRE(grid < (int64_t)1 << 24, "%s: too many query rows", what);  // (a launch holds fewer than 2^32 threads)
  a.tiles = (int)tiles;
  a.q_factor = scale < 0x1p-60f ? 0x1p-64f : scale > 0x1p60f ? 0x1p64f : 1.0f;
  a.sl2 = scale / a.q_factor * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o ? a.part_o + a.splits * kv_heads * tiles * kExtRows * head_dim : nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128) launch<128>(a, grid, s);
  else launch<64>(a, grid, s);
  return check_launch(what);
}
