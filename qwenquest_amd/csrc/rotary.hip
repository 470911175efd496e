// Norms of each query and key head and the rotation by position in one pass, from the QKV product's
// rows to the q, k, v that the attention takes.  Of a head x of D channels, with weights w,
//   y = x / sqrt(mean x^2 + eps) * w,
// then of the pairs (a, b) of the first 2 P channels (b is P further on, or next to a) pair j turns by
// the angle pos[axis_j] * f_j:  (a cos - b sin, b cos + a sin).  fp32, rounded once at the end.
//
// The angle is taken in quarter turns in fp64, a product of all its bits, and its fraction goes to fp32 at 1/2 of a quarter at most:
// sine and cosine are good to fp32's last places but for what the frequency, rounded to fp64, leaves of the angle,
// 2^-53 of it (2^-24 at 2^29 radians, 2^-22 at 2^31).
//
// A wave works on a token: a lane per pair for the angles, which meet the heads in the LDS, then D / 8 lanes
// (to the next power of two) per head, 8 channels a lane, whose cosines and sines stay in registers over the
// token's heads; where tokens are few, more waves share a token's heads.
// Bound: HBM at prompts: 16384 tokens, 32 + 4 + 4 heads of 128 in bf16, 74 us (4.5 TB/s, a copy 4.7; 104 with the heads'
// values asked for one after the other, exchanged through the LDS and rounded by hand). 16 tokens 4.4, a launch and
// two memory round trips; 5001 tokens of 14 + 2 + 2 heads of 64 in fp32, one round of waves, 14.2 (a copy of the same bytes 8.3).  Heads of 80
// channels leave 6 of 16 lanes idle and meet their partners through the LDS: 4096 tokens 19.8 us, of 128 channels 22.0.
#include <type_traits>

#include "qq_quest_dev.h"

namespace qq {
namespace {

constexpr int kMaxPairs = 256;
constexpr int kRotWaves = 4;

struct RotaryArgs {
  const void* q;  // [n, H, D], rows q_stride elements apart
  const void* k;
  const void* v;  // nullptr: none
  int64_t q_stride, k_stride, v_stride;
  int H, KV, D;
  int64_t n;
  const float* wq;  // [D], or nullptr: no norm
  const float* wk;
  float eps;
  const double* quarters;  // [pairs] quarter turns per position
  const int32_t* axis;     // [pairs]
  int pairs, neighbours;
  const int64_t* pos;  // [axes, n]
  int64_t pos_stride;
  int axes;
  void* q_out;  // dense
  void* k_out;
  void* v_out;
  int per, parts;  // heads of a wave, waves of a token
};

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

template <typename T>
struct Row8;  // eight values as they lie
template <>
struct Row8<uint16_t> {
  uint4 w;
  __device__ inline void load(const uint16_t* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ inline void store(uint16_t* p) const { *reinterpret_cast<uint4*>(p) = w; }
  __device__ inline void get(float (&x)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(i & 1 ? u[i / 2] & 0xFFFF0000u : u[i / 2] << 16);
  }
  __device__ inline void set(const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bf16x2_t b = {(__bf16)x[2 * i], (__bf16)x[2 * i + 1]};  // to nearest even
      u[i] = __builtin_bit_cast(uint32_t, b);
    }
    w = make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <>
struct Row8<float> {
  float4 a, b;
  __device__ inline void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ inline void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
  __device__ inline void get(float (&x)[8]) const {
    const float y[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i];
  }
  __device__ inline void set(const float (&x)[8]) {
    a = make_float4(x[0], x[1], x[2], x[3]);
    b = make_float4(x[4], x[5], x[6], x[7]);
  }
};

// The sum over L lanes next to each other, in each of them.
template <int L>
__device__ inline float lanes_sum(float v, int lane) {
  auto add = [&](auto j) { v += __uint_as_float(lane_xor_u32<decltype(j)::value>(__float_as_uint(v), lane)); };
  if constexpr (L >= 2) add(std::integral_constant<int, 1>{});
  if constexpr (L >= 4) add(std::integral_constant<int, 2>{});
  if constexpr (L >= 8) add(std::integral_constant<int, 4>{});
  if constexpr (L >= 16) add(std::integral_constant<int, 8>{});
  if constexpr (L >= 32) add(std::integral_constant<int, 16>{});
  if constexpr (L >= 64) add(std::integral_constant<int, 32>{});
  return v;
}

// Where a channel's partner lies: in the lane itself, L / 2 lanes off (D = 8 L, all of it turning), or elsewhere.
enum Partner { kOwn, kAcross, kAway };

// L lanes a head.
template <typename T, int L, Partner P>
__global__ __launch_bounds__(64 * kRotWaves) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float turned[];  // [waves][cosines, sines][pairs]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t token = (int64_t)blockIdx.x * kRotWaves + wave;
  if (token >= a.n) return;  // (no block barrier below)
  const int sub = lane / L, dl = lane % L;
  const bool in = dl * 8 < a.D;
  const int d = in ? dl * 8 : 0;
  const int heads = a.H + a.KV + (a.v ? a.KV : 0);
  const int h0 = blockIdx.y * a.per, h1 = min(h0 + a.per, heads);
  constexpr int kStep = 64 / L;
  // lanes past the last head do it once more, and write nothing
  auto load = [&](Row8<T>& r, int hb) {
    const int h = min(hb + sub, h1 - 1);
    const T* p = static_cast<const T*>(a.q) + token * a.q_stride + (int64_t)h * a.D;
    if (h >= a.H) p = static_cast<const T*>(a.k) + token * a.k_stride + (int64_t)(h - a.H) * a.D;
    if (h >= a.H + a.KV) p = static_cast<const T*>(a.v) + token * a.v_stride + (int64_t)(h - a.H - a.KV) * a.D;
    r.load(p + d);
  };
  // the heads' values are under way while the angles are taken
  constexpr int kAhead = 3;
  Row8<T> rows[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (h0 + i * kStep < h1) load(rows[i], h0 + i * kStep);
  float *cs = turned + wave * 2 * a.pairs, *sn = cs + a.pairs;
  for (int j = lane; j < a.pairs; j += 64) {
    const int64_t at = a.pos[(a.axes == 1 ? 0 : min(a.axis[j], a.axes - 1)) * a.pos_stride + token];
    const double f = a.quarters[j], t = (double)at * f, whole = rint(t), rest = __builtin_fma((double)at, f, -t);
    const int quarter = (int)(whole - 4.0 * floor(whole * 0.25));  // 0 .. 3
    float s, c;
    sincospif(0.5f * (float)(t - whole + rest), &s, &c);
    if (at >= (int64_t)1 << 31 || at <= -((int64_t)1 << 31)) s = c = __builtin_nanf("");
    cs[j] = quarter & 1 ? (quarter & 2 ? s : -s) : (quarter & 2 ? -c : c);
    sn[j] = quarter & 1 ? (quarter & 2 ? -c : c) : (quarter & 2 ? -s : s);
  }
  __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // a wave's own LDS words
  __builtin_amdgcn_wave_barrier();
  // the lane's pairs: its 8 channels are all first or all second ones, or four whole pairs
  const bool turns = in && d < 2 * a.pairs, second = P != kOwn && d >= a.pairs;
  const int hop = second ? -(a.pairs / 8) : a.pairs / 8;  // lanes to the partner
  float c[8], s[8], wq[8], wk[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int j = P == kOwn ? (d + i) / 2 : d + i - (second ? a.pairs : 0);
    c[i] = turns ? cs[j] : 1.0f;
    s[i] = turns ? sn[j] : 0.0f;
    if (P == kOwn ? !(i & 1) : !second) s[i] = -s[i];
    wq[i] = a.wq ? a.wq[d + i] : 1.0f;
    wk[i] = a.wk ? a.wk[d + i] : 1.0f;
  }
  const float share = 1.0f / (float)a.D;
  auto work = [&](Row8<T> r, int hb) {
    const int h = min(hb + sub, h1 - 1);
    float x[8], y[8];
    r.get(x);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(x[i], x[i], sum);
    sum = lanes_sum<L>(in ? sum : 0.0f, lane);
    const bool key = h >= a.H, normed = key ? a.wk != nullptr : a.wq != nullptr;
    float mean = __builtin_fmaf(sum, share, a.eps);
    // Squares that leave float32's range, or all but do: the row in other units
    const bool large = !(sum <= 0x1p100f), small = mean < 0x1p-100f;
    if (__builtin_expect(__any(normed && (large || small)), 0)) {
      const float unit = !normed ? 1.0f : large ? 0x1p-96f : small ? 0x1p96f : 1.0f;
      sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= unit;
        sum = __builtin_fmaf(x[i], x[i], sum);
      }
      mean = __builtin_fmaf(lanes_sum<L>(in ? sum : 0.0f, lane), share, a.eps * unit * unit);
    }
    float f = __builtin_amdgcn_rsqf(mean);
    // a Newton step: the instruction is off by up to 2^-23
    f = mean < INFINITY && mean > 1e-37f ? f + 0.5f * f * __builtin_fmaf(-mean * f, f, 1.0f) : f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = normed ? x[i] * f * (key ? wk[i] : wq[i]) : x[i];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = P == kOwn      ? x[i ^ 1]
             : P == kAcross ? __uint_as_float(lane_xor_u32<L / 2>(__float_as_uint(x[i]), lane))
                            : __shfl(x[i], lane + hop, 64);
    if (h < a.H + a.KV) {
      if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(y[i], s[i], x[i] * c[i]);
      }
      r.set(x);
    }
    if (!in || hb + sub >= h1) return;
    T* p = static_cast<T*>(a.q_out) + (token * a.H + h) * a.D;
    if (h >= a.H) p = static_cast<T*>(a.k_out) + (token * a.KV + h - a.H) * a.D;
    if (h >= a.H + a.KV) p = static_cast<T*>(a.v_out) + (token * a.KV + h - a.H - a.KV) * a.D;
    r.store(p + d);
  };
  for (int hb = h0; hb < h1; hb += kAhead * kStep) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (hb + i * kStep >= h1) break;  // wave-uniform
      const Row8<T> r = rows[i];
      if (hb + (i + kAhead) * kStep < h1) load(rows[i], hb + (i + kAhead) * kStep);
      work(r, hb + i * kStep);
    }
  }
}

template <typename T, int L>
void launch_lanes(const RotaryArgs& a, dim3 blocks, size_t lds, hipStream_t s) {
  if (a.neighbours) rotary_kernel<T, L, kOwn><<<blocks, 64 * kRotWaves, lds, s>>>(a);
  else if (a.D == 8 * L && 2 * a.pairs == a.D) rotary_kernel<T, L, kAcross><<<blocks, 64 * kRotWaves, lds, s>>>(a);
  else rotary_kernel<T, L, kAway><<<blocks, 64 * kRotWaves, lds, s>>>(a);
}

template <typename T>
void launch(const RotaryArgs& a, hipStream_t s) {
  const dim3 blocks((unsigned)((a.n + kRotWaves - 1) / kRotWaves), a.parts);
  const size_t lds = (size_t)kRotWaves * 2 * a.pairs * sizeof(float);
  if (a.D <= 64) launch_lanes<T, 8>(a, blocks, lds, s);
  else if (a.D <= 128) launch_lanes<T, 16>(a, blocks, lds, s);
  else if (a.D <= 256) launch_lanes<T, 32>(a, blocks, lds, s);
  else launch_lanes<T, 64>(a, blocks, lds, s);
}

}  // namespace
}  // namespace qq

using namespace qq;

extern "C" int qq_qk_norm_rotary(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                 int64_t v_stride, int dtype, int num_q_heads, int kv_heads, int head_dim, int64_t n,
                                 const float* q_weight, const float* k_weight, float eps, const double* quarter_turns,
                                 const int32_t* pair_axis, int pairs, int neighbours, const int64_t* positions,
                                 int64_t positions_stride, int axes, void* q_out, void* k_out, void* v_out, void* stream) {
  const char* what = "qq_qk_norm_rotary";
  QQ_REQUIRE(dtype_ok(dtype), "%s: bad dtype", what);
  QQ_REQUIRE(head_dim > 0 && head_dim <= 2 * kMaxPairs && head_dim % 8 == 0, "%s: head_dim %d is not a multiple of 8 up to %d", what,
             head_dim, 2 * kMaxPairs);
  QQ_REQUIRE(num_q_heads > 0 && kv_heads > 0 && num_q_heads < 65536 && kv_heads < 65536, "%s: %d and %d heads", what, num_q_heads,
             kv_heads);
  QQ_REQUIRE(pairs >= 0 && 2 * pairs <= head_dim && pairs % (neighbours ? 4 : 8) == 0,
             "%s: %d pairs of %d channels, in multiples of %d", what, pairs, head_dim, neighbours ? 4 : 8);
  // (a launch holds fewer than 2^32 threads, 64 a token)
  QQ_REQUIRE(n >= 0 && n < ((int64_t)1 << 26) - kRotWaves && axes > 0, "%s: bad sizes", what);
  if (n == 0) return QQ_OK;
  QQ_REQUIRE(q && k && q_out && k_out && (!v || v_out) && (pairs == 0 || (quarter_turns && pair_axis && positions)),
             "%s: null pointer", what);
  QQ_REQUIRE(axes == 1 || positions_stride >= n, "%s: the axes' positions overlap", what);
  const int64_t row = 16 / dtype_size(dtype);  // elements of an aligned piece
  QQ_REQUIRE(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0 &&
                 q_stride % row == 0 && k_stride % row == 0 && v_stride % row == 0,
             "%s: rows must be 16-byte aligned", what);
  RotaryArgs a{q, k, v, q_stride, k_stride, v_stride, num_q_heads, kv_heads, head_dim, n, q_weight, k_weight, eps, quarter_turns,
               pair_axis, pairs, neighbours, positions, positions_stride, axes, q_out, k_out, v_out, 0, 1};
  const int heads = num_q_heads + (v ? 2 : 1) * kv_heads;
  const int step = 64 / (head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : head_dim <= 256 ? 32 : 64);  // heads a wave has at once
  const int rounds = (heads + step - 1) / step;
  // as many waves as the chip has SIMDs, where there are fewer tokens (512 tokens of 32 + 8 heads in 2 parts 6.9 us, in 1
  // 9.2, in 8 9.1; 128 in 8 parts 5.0, in 2 or 10 6.3)
  a.parts = (int)min((int64_t)rounds, max((int64_t)1, 1024 / n));
  a.per = (rounds + a.parts - 1) / a.parts * step;
  a.parts = (heads + a.per - 1) / a.per;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == QQ_DTYPE_BF16) launch<uint16_t>(a, s);
  else launch<float>(a, s);
  return check_launch(what);
}
