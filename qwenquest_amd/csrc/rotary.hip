// Norms of each query and key head and the rotation by position in one pass, from the QKV product's
// rows to the q, k, v that the attention takes.  Of a head x of D channels, with weights w,
//   y = x / sqrt(mean x^2 + eps) * w,
// then of the pairs (a, b) of the first 2 P channels (b is P further on, or next to a) pair j turns by
// the angle pos[axis_j] * f_j:  (a cos - b sin, b cos + a sin).  fp32, rounded once at the end.
//
// The angle is taken in quarter turns in fp64 (53 bits: at position 2^31 still to 2^-22 of a radian), its
// fraction goes to fp32 at 1/2 of a quarter at most, so that sine and cosine are good to fp32's last
// places at any position.
//
// A wave works on a token: a lane per pair for the angles, which meet the heads in the LDS, then D / 8 lanes
// (to the next power of two) per head, 8 channels a lane, whose cosines and sines stay in registers over the
// token's heads; where tokens are few, more waves share a token's heads.
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
    for (int i = 0; i < 4; ++i) u[i] = (uint32_t)f2bf(x[2 * i]) | ((uint32_t)f2bf(x[2 * i + 1]) << 16);
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

// L lanes a head.
template <typename T, int L>
__global__ __launch_bounds__(64 * kRotWaves) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float turned[];  // [waves][cosines, sines][pairs]
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * kRotWaves + wave;
  const int64_t token = item / a.parts;
  if (token >= a.n) return;  // (no block barrier below)
  float *cs = turned + wave * 2 * a.pairs, *sn = cs + a.pairs;
  for (int j = lane; j < a.pairs; j += 64) {
    const int64_t at = a.pos[min(a.axis[j], a.axes - 1) * a.pos_stride + token];
    const double t = (double)at * a.quarters[j], whole = rint(t);
    const int quarter = (int)(whole - 4.0 * floor(whole * 0.25));  // 0 .. 3
    float s, c;
    sincospif(0.5f * (float)(t - whole), &s, &c);
    if (at >= (int64_t)1 << 31 || at <= -((int64_t)1 << 31)) s = c = __builtin_nanf("");
    cs[j] = quarter & 1 ? (quarter & 2 ? s : -s) : (quarter & 2 ? -c : c);
    sn[j] = quarter & 1 ? (quarter & 2 ? -c : c) : (quarter & 2 ? -s : s);
  }
  __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // a wave's own LDS words
  __builtin_amdgcn_wave_barrier();
  const int sub = lane / L, dl = lane % L;
  const bool in = dl * 8 < a.D;
  const int d = in ? dl * 8 : 0;
  // the lane's pairs: its 8 channels are all first or all second ones, or four whole pairs
  const bool turns = in && d < 2 * a.pairs, second = !a.neighbours && d >= a.pairs;
  const int hop = a.neighbours ? 0 : second ? -(a.pairs / 8) : a.pairs / 8;  // lanes to the partner
  float c[8], s[8], wq[8], wk[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int j = a.neighbours ? (d + i) / 2 : d + i - (second ? a.pairs : 0);
    c[i] = turns ? cs[j] : 1.0f;
    s[i] = turns ? sn[j] : 0.0f;
    if (a.neighbours ? !(i & 1) : !second) s[i] = -s[i];
    wq[i] = a.wq ? a.wq[d + i] : 1.0f;
    wk[i] = a.wk ? a.wk[d + i] : 1.0f;
  }
  const int heads = a.H + a.KV + (a.v ? a.KV : 0);
  const int h0 = (int)(item - token * a.parts) * a.per, h1 = min(h0 + a.per, heads);
  auto from = [&](int h) -> const T* {
    if (h < a.H) return static_cast<const T*>(a.q) + token * a.q_stride + (int64_t)h * a.D;
    if (h < a.H + a.KV) return static_cast<const T*>(a.k) + token * a.k_stride + (int64_t)(h - a.H) * a.D;
    return static_cast<const T*>(a.v) + token * a.v_stride + (int64_t)(h - a.H - a.KV) * a.D;
  };
  auto to = [&](int h) -> T* {
    if (h < a.H) return static_cast<T*>(a.q_out) + (token * a.H + h) * a.D;
    if (h < a.H + a.KV) return static_cast<T*>(a.k_out) + (token * a.KV + h - a.H) * a.D;
    return static_cast<T*>(a.v_out) + (token * a.KV + h - a.H - a.KV) * a.D;
  };
  for (int hb = h0; hb < h1; hb += 64 / L) {
    const int h = min(hb + sub, h1 - 1);  // lanes past the last head do it once more, and write nothing
    Row8<T> r;
    r.load(from(h) + d);
    float x[8], y[8];
    r.get(x);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += in ? x[i] * x[i] : 0.0f;
#pragma unroll
    for (int m = L / 2; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, 64);
    const bool key = h >= a.H;
    const float mean = sum / (float)a.D + a.eps;
    float f = __builtin_amdgcn_rsqf(mean);
    // a Newton step: the instruction is off by up to 2^-23
    f = mean < INFINITY && mean > 1e-37f ? f + 0.5f * f * __builtin_fmaf(-mean * f, f, 1.0f) : f;
    const bool normed = key ? a.wk != nullptr : a.wq != nullptr;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = normed ? x[i] * f * (key ? wk[i] : wq[i]) : x[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = a.neighbours ? x[i ^ 1] : __shfl(x[i], lane + hop, 64);
    if (h < a.H + a.KV) {
      if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(y[i], s[i], x[i] * c[i]);
      }
      r.set(x);
    }
    if (in && hb + sub < h1) r.store(to(h) + d);
  }
}

template <typename T>
void launch(const RotaryArgs& a, hipStream_t s) {
  const unsigned blocks = (unsigned)((a.n * a.parts + kRotWaves - 1) / kRotWaves);
  const size_t lds = (size_t)kRotWaves * 2 * a.pairs * sizeof(float);
  if (a.D <= 64) rotary_kernel<T, 8><<<blocks, 64 * kRotWaves, lds, s>>>(a);
  else if (a.D <= 128) rotary_kernel<T, 16><<<blocks, 64 * kRotWaves, lds, s>>>(a);
  else if (a.D <= 256) rotary_kernel<T, 32><<<blocks, 64 * kRotWaves, lds, s>>>(a);
  else rotary_kernel<T, 64><<<blocks, 64 * kRotWaves, lds, s>>>(a);
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
  QQ_REQUIRE(n >= 0 && n < (int64_t)1 << 28 && axes > 0, "%s: bad sizes", what);
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
  a.parts = (int)min((int64_t)rounds, max((int64_t)1, 4096 / n));
  a.per = (rounds + a.parts - 1) / a.parts * step;
  a.parts = (heads + a.per - 1) / a.per;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == QQ_DTYPE_BF16) launch<uint16_t>(a, s);
  else launch<float>(a, s);
  return check_launch(what);
}
