// Rotary positions with several axes: channel pairs of q and k turned by angles that grow
// with a token's place in time, height and width.
//
//   turns(i) = position[axis(i)] * frequency(i)      in float64, frequency in turns
//   (a, b)  -> (a cos - b sin, b cos + a sin)        fp32, rounded once
//
// pairs are channels (i, i + R) or (2 i, 2 i + 1), i < R; channels from 2 R on are copied.
//
// One read and one write of q and k: bound by HBM.  All heads of a token share its angles:
// a workgroup forms the cosines and sines of its tokens once, in LDS (one float64 product
// and one fp32 sincos a token and pair), and then walks over the tokens' heads.  The whole
// turns are taken off in float64, so far positions keep the angle's 24 bits.  16384 tokens of 32 + 8
// heads of 128, bf16: 61-68 us = 4.9-5.5 TB/s (a large copy 5.2); 4 x 1370 tokens of 16 + 16 heads of
// 64, fp16: 10 us; 8 tokens 3.9 us, the latency of a sincos and two reads.
//
// norm_rotary_kernel norms each head of q and k before that, in the same pass:
//
//   y = x w / sqrt(mean(x^2) + eps)                  fp32, turned before its one rounding
//
// a head's channels in 1 to 64 neighbouring lanes, whose sum of squares goes round by lane-crossing
// moves: the same bound.  16384 tokens of 32 + 8 heads of 128, bf16: 61 us = 5.5 TB/s; 4 x 1370
// tokens of 16 + 16 heads of 64, fp16: 12 us; 8 tokens 5 us.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

#include "common.hpp"
#include "storage.hpp"

namespace musc {
namespace rotary {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;
constexpr int kMaxTokens = 16;  // tokens of a workgroup
constexpr int kTable = 256;     // (token, pair) entries of a workgroup: one sincos per thread, or one token's pairs
static_assert(kTable >= kThreads && kTable >= kMaxPairs, "a workgroup's angles fit the table");

struct Side {
  const void* x;
  void* y;
  long long sb, st, sh, ob, ot, oh;  // strides of x and y, elements
  int heads;
};

struct Args {
  Side q, k;
  const void* positions;
  long long pos_sb;
  const double* frequency;
  const int* axis;
  int batch, t, axes, pairs, dim, int_positions, tokens;
  int items;               // vectors (or pairs and single channels) of a head
  uint32_t by_items, by_heads;  // ceil(2^32 / n): n divides numbers below 2^32 / n exactly
  float sign;
};

__device__ __forceinline__ uint32_t over(uint32_t x, uint32_t reciprocal) { return reciprocal ? __umulhi(x, reciprocal) : x; }

// Cosines and sines of `here` tokens from the workgroup's first on, and where those tokens are.
__device__ __forceinline__ void form_angles(const Args& a, long long first, int here, float2* table, long long* at_b,
                                            int* at_t) {
  const int pairs = a.pairs;
  for (int e = threadIdx.x; e < here * pairs; e += kThreads) {
    const int token = e / pairs, i = e % pairs;
    const long long b = (first + token) / a.t, t = (first + token) % a.t;
    const long long p = b * a.pos_sb + t * a.axes + a.axis[i];
    const double place = a.int_positions ? (double)static_cast<const int*>(a.positions)[p]
                                         : (double)static_cast<const float*>(a.positions)[p];
    const double turns = place * a.frequency[i];
    const float rest = (float)(turns - rint(turns));  // in [-1/2, 1/2]
    float s, c;
    sincospif(2.f * rest, &s, &c);
    table[e] = make_float2(c, a.sign * s);
    if (i == 0) {
      at_b[token] = b;
      at_t[token] = (int)t;
    }
  }
}

// kVec: vectors of 16 bytes; otherwise one pair, or one copied channel, per thread.
template <int kDtype, bool kAdjacent, bool kVec>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const Args a) {
  using S = Storage<kDtype>;
  typedef typename S::T T;
  constexpr int N = S::N;
  __shared__ float2 table[kTable];
  __shared__ long long at_b[kMaxTokens];
  __shared__ int at_t[kMaxTokens];
  const long long first = linear_block() * a.tokens, total = (long long)a.batch * a.t;
  if (first >= total) return;
  const int here = (int)min((long long)a.tokens, total - first);
  const int pairs = a.pairs;
  form_angles(a, first, here, table, at_b, at_t);
  __syncthreads();
  const int heads = a.q.heads + a.k.heads;
  const int all = here * heads * a.items;
  for (int e = threadIdx.x; e < all; e += kThreads) {
    const uint32_t rest = over(e, a.by_items);
    const int item = e - rest * a.items;
    const int token = over(rest, a.by_heads);
    int head = rest - token * heads;
    const bool of_k = head >= a.q.heads;
    const Side& side = of_k ? a.k : a.q;
    if (of_k) head -= a.q.heads;
    const long long b = at_b[token], t = at_t[token];
    const T* x = static_cast<const T*>(side.x) + b * side.sb + t * side.st + head * side.sh;
    T* y = static_cast<T*>(side.y) + b * side.ob + t * side.ot + head * side.oh;
    const float2* cs = table + token * pairs;
    if constexpr (kVec) {
      const int turned = kAdjacent ? 2 * pairs / N : pairs / N;
      if (item >= turned) {
        const int c = 2 * pairs + (item - turned) * N;
        *reinterpret_cast<float4*>(y + c) = *reinterpret_cast<const float4*>(x + c);
      } else if constexpr (kAdjacent) {
        float v[N];
        S::load(x + item * N, v);
#pragma unroll
        for (int j = 0; j < N; j += 2) {
          const float2 w = cs[item * (N / 2) + j / 2];
          const float p = v[j], r = v[j + 1];
          v[j] = p * w.x - r * w.y;
          v[j + 1] = r * w.x + p * w.y;
        }
        S::store(y + item * N, v);
      } else {
        float p[N], r[N];
        S::load(x + item * N, p);
        S::load(x + pairs + item * N, r);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float2 w = cs[item * N + j];
          const float u = p[j];
          p[j] = u * w.x - r[j] * w.y;
          r[j] = r[j] * w.x + u * w.y;
        }
        S::store(y + item * N, p);
        S::store(y + pairs + item * N, r);
      }
    } else {
      if (item >= pairs) {
        y[pairs + item] = x[pairs + item];
      } else {
        const int c0 = kAdjacent ? 2 * item : item, c1 = kAdjacent ? c0 + 1 : pairs + item;
        const float2 w = cs[item];
        const float p = S::one(x[c0]), r = S::one(x[c1]);
        y[c0] = S::round(p * w.x - r * w.y);
        y[c1] = S::round(r * w.x + p * w.y);
      }
    }
  }
}

struct Norm {
  const void* w[2];   // of q and k, or null
  long long w_sh[2];  // elements between the weights of two heads, 0: shared
  int w_dtype[2];
  float eps;
  int lane_bits;      // a head is held by 2^lane_bits neighbouring lanes
};

// Sum over groups of 2^bits neighbouring lanes, by lane-crossing moves up to 16 of them.
__device__ __forceinline__ float group_sum(float v, int bits) {
  const auto with = [&](auto move) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(move)::value, 0xf, 0xf, true));
  };
  if (bits > 0) with(std::integral_constant<int, 0xb1>{});   // lane ^ 1
  if (bits > 1) with(std::integral_constant<int, 0x4e>{});   // lane ^ 2
  if (bits > 2) with(std::integral_constant<int, 0x141>{});  // the other half of 8
  if (bits > 3) with(std::integral_constant<int, 0x140>{});  // the other half of 16
  if (bits > 4) v += __shfl_xor(v, 16, kWave);
  if (bits > 5) v += __shfl_xor(v, 32, kWave);
  return v;
}

// N values of a weight in the storage type or fp32.
template <int kDtype, int N>
__device__ __forceinline__ void load_weight(const void* w, int dtype, long long at, float (&v)[N]) {
  typedef typename Storage<kDtype>::T T;
  if (dtype == kDtype) {
    typedef T Vec __attribute__((ext_vector_type(N)));
    const Vec x = *reinterpret_cast<const Vec*>(static_cast<const T*>(w) + at);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (float)x[j];
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + at + j);
      v[j] = x.x, v[j + 1] = x.y, v[j + 2] = x.z, v[j + 3] = x.w;
    }
  }
}

// Vectors of N elements: a lane holds one of a head's turned items (two vectors of a half each, or
// one of neighbouring pairs) or one vector of the channels that do not turn.  The first heads' loads are
// in flight while the angles are formed; weights that heads share wait in LDS as fp32.  One head a lane at a
// time and waves enough to hide its loads: two or four at a time take 64 and 84 us for the 16384 tokens.
template <int kDtype, bool kAdjacent, int N>
__global__ __launch_bounds__(kThreads) void norm_rotary_kernel(const Args a, const Norm n) {
  typedef typename Storage<kDtype>::T T;
  typedef T Vec __attribute__((ext_vector_type(N)));
  __shared__ float2 table[kTable];
  __shared__ __attribute__((aligned(16))) float weights[2][2 * kMaxPairs];
  const long long first = linear_block() * a.tokens, total = (long long)a.batch * a.t;
  if (first >= total) return;
  const int here = (int)min((long long)a.tokens, total - first);
  const int pairs = a.pairs, tid = threadIdx.x;
  const uint32_t first_b = (uint32_t)first / (uint32_t)a.t, first_t = (uint32_t)first - first_b * (uint32_t)a.t;
  // batch entry and place of the workgroup's token
  const auto place = [&](int token, uint32_t& b, uint32_t& t) {
    b = first_b, t = first_t + token;
    if (t >= (uint32_t)a.t) b += t / (uint32_t)a.t, t %= (uint32_t)a.t;
  };
  // this thread's angle (there are no more of them): asked for before anything else
  static_assert(kTable <= kThreads, "one angle a thread");
  const int angle_token = (int)((uint32_t)tid / (uint32_t)pairs), pair = tid - angle_token * pairs;
  const bool has_angle = angle_token < here;
  int axis = 0;
  double frequency = 0.;
  if (has_angle) axis = a.axis[pair], frequency = a.frequency[pair];
  const void *qw = n.w[0], *kw = n.w[1];
  const bool q_each = qw && n.w_sh[0] != 0, k_each = kw && n.w_sh[1] != 0;  // weights of each head
  const int group = tid >> n.lane_bits, item = tid & ((1 << n.lane_bits) - 1), groups = kThreads >> n.lane_bits;
  const int turned = kAdjacent ? 2 * pairs / N : pairs / N;
  const bool turns = item < turned, two = !kAdjacent && turns;
  const int c0 = turns ? item * N : 2 * pairs + (item - turned) * N, c1 = pairs + item * N;
  const int q_heads = a.q.heads, heads = q_heads + a.k.heads, all = here * heads;
  for (int from = 0; from < all; from += groups) {
    const int h = from + group, token = over(h, a.by_heads), of_both = h - token * heads;
    const bool live = item < a.items && h < all, of_k = of_both >= q_heads, each = of_k ? k_each : q_each;
    const int head = of_k ? of_both - q_heads : of_both;
    const auto of = [&](auto field) { return of_k ? a.k.*field : a.q.*field; };
    uint32_t b, t;
    place(token, b, t);
    Vec x0 = Vec{}, x1 = Vec{};
    float w0[N], w1[N];
#pragma unroll
    for (int j = 0; j < N; ++j) w0[j] = w1[j] = 1.f;
    if (live) {
      const T* x = static_cast<const T*>(of(&Side::x)) + b * of(&Side::sb) + t * of(&Side::st) + head * of(&Side::sh);
      x0 = *reinterpret_cast<const Vec*>(x + c0);
      if (two) x1 = *reinterpret_cast<const Vec*>(x + c1);
      if (each) {
        const int w_dtype = of_k ? n.w_dtype[1] : n.w_dtype[0];
        const long long at = head * (of_k ? n.w_sh[1] : n.w_sh[0]);
        load_weight<kDtype, N>(of_k ? kw : qw, w_dtype, at + c0, w0);
        if (two) load_weight<kDtype, N>(of_k ? kw : qw, w_dtype, at + c1, w1);
      }
    }
    if (from == 0) {
      int raw = 0;  // of the position, float or int
      if (has_angle) {
        uint32_t ab, at;
        place(angle_token, ab, at);
        raw = static_cast<const int*>(a.positions)[ab * a.pos_sb + (long long)at * a.axes + axis];
      }
      // half of the workgroup stages q's weight, the other one k's
      const int which = __builtin_amdgcn_readfirstlane(tid / (kThreads / 2)), c = tid % (kThreads / 2) * 4;
      if (c < a.dim) {
        float w[4] = {1.f, 1.f, 1.f, 1.f};
        if ((which ? kw : qw) && !(which ? k_each : q_each))
          load_weight<kDtype, 4>(which ? kw : qw, which ? n.w_dtype[1] : n.w_dtype[0], c, w);
        *reinterpret_cast<float4*>(&weights[which][c]) = make_float4(w[0], w[1], w[2], w[3]);
      }
      const double all_turns = (a.int_positions ? (double)raw : (double)__int_as_float(raw)) * frequency;
      const float rest = (float)(all_turns - rint(all_turns));  // in [-1/2, 1/2]
      if (has_angle) {
        float s, cos;
        sincospif(2.f * rest, &s, &cos);
        table[tid] = make_float2(cos, a.sign * s);
      }
      __syncthreads();
    }
    float q = 0.f, v0[N], v1[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v0[j] = (float)x0[j], v1[j] = (float)x1[j];
      q = fmaf(v0[j], v0[j], q);
      if (!kAdjacent) q = fmaf(v1[j], v1[j], q);
    }
    const float rstd = 1.f / sqrtf(group_sum(q, n.lane_bits) / (float)a.dim + n.eps);
    if (!live) continue;
    if (!each) {
      const float* w = weights[of_k ? 1 : 0];
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const float4 f = *reinterpret_cast<const float4*>(w + c0 + j), g = *reinterpret_cast<const float4*>(w + (two ? c1 : c0) + j);
        w0[j] = f.x, w0[j + 1] = f.y, w0[j + 2] = f.z, w0[j + 3] = f.w;
        w1[j] = g.x, w1[j + 1] = g.y, w1[j + 2] = g.z, w1[j + 3] = g.w;
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) v0[j] = v0[j] * rstd * w0[j], v1[j] = v1[j] * rstd * w1[j];
    if (turns) {
      const float2* cs = table + token * pairs + (kAdjacent ? item * (N / 2) : item * N);
      if constexpr (kAdjacent) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
          const float2 r = cs[j / 2];
          const float p = v0[j];
          v0[j] = p * r.x - v0[j + 1] * r.y;
          v0[j + 1] = v0[j + 1] * r.x + p * r.y;
        }
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float2 r = cs[j];
          const float p = v0[j];
          v0[j] = p * r.x - v1[j] * r.y;
          v1[j] = v1[j] * r.x + p * r.y;
        }
      }
    }
    Vec y0, y1;
#pragma unroll
    for (int j = 0; j < N; ++j) y0[j] = (T)v0[j], y1[j] = (T)v1[j];
    T* y = static_cast<T*>(of(&Side::y)) + b * of(&Side::ob) + t * of(&Side::ot) + head * of(&Side::oh);
    *reinterpret_cast<Vec*>(y + c0) = y0;
    if (two) *reinterpret_cast<Vec*>(y + c1) = y1;
  }
}

// Any alignment: a wave a head, a pair or a channel that does not turn per lane at a time, in two passes.
template <int kDtype, bool kAdjacent>
__global__ __launch_bounds__(kThreads) void norm_rotary_any_kernel(const Args a, const Norm n) {
  using S = Storage<kDtype>;
  typedef typename S::T T;
  __shared__ float2 table[kTable];
  __shared__ long long at_b[kMaxTokens];
  __shared__ int at_t[kMaxTokens];
  const long long first = linear_block() * a.tokens, total = (long long)a.batch * a.t;
  if (first >= total) return;
  const int here = (int)min((long long)a.tokens, total - first);
  const int pairs = a.pairs, lane = threadIdx.x % kWave;
  form_angles(a, first, here, table, at_b, at_t);
  __syncthreads();
  const int heads = a.q.heads + a.k.heads;
  for (int h = threadIdx.x / kWave; h < here * heads; h += kThreads / kWave) {
    const int token = h / heads, which = h % heads >= a.q.heads;
    const int head = h % heads - (which ? a.q.heads : 0);
    const Side& side = which ? a.k : a.q;
    const T* x = static_cast<const T*>(side.x) + at_b[token] * side.sb + at_t[token] * side.st + head * side.sh;
    T* y = static_cast<T*>(side.y) + at_b[token] * side.ob + at_t[token] * side.ot + head * side.oh;
    float q = 0.f;
    for (int c = lane; c < a.dim; c += kWave) {
      const float v = S::one(x[c]);
      q = fmaf(v, v, q);
    }
    const float rstd = 1.f / sqrtf(group_sum(q, 6) / (float)a.dim + n.eps);
    const auto normed = [&](int c) {
      const long long at = head * n.w_sh[which] + c;
      const float w = !n.w[which]                    ? 1.f
                      : n.w_dtype[which] == kDtype ? S::one(static_cast<const T*>(n.w[which])[at])
                                                   : static_cast<const float*>(n.w[which])[at];
      return S::one(x[c]) * rstd * w;
    };
    for (int i = lane; i < a.items; i += kWave) {
      if (i >= pairs) {
        y[pairs + i] = S::round(normed(pairs + i));
      } else {
        const int c0 = kAdjacent ? 2 * i : i, c1 = kAdjacent ? c0 + 1 : pairs + i;
        const float2 r = table[token * pairs + i];
        const float p = normed(c0), s = normed(c1);
        y[c0] = S::round(p * r.x - s * r.y);
        y[c1] = S::round(s * r.x + p * r.y);
      }
    }
  }
}

template <int kDtype>
void launch(const Args& a, bool adjacent, bool vec, dim3 grid, hipStream_t stream) {
  if (adjacent) {
    if (vec) hipLaunchKernelGGL((rotary_kernel<kDtype, true, true>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((rotary_kernel<kDtype, true, false>), grid, dim3(kThreads), 0, stream, a);
  } else {
    if (vec) hipLaunchKernelGGL((rotary_kernel<kDtype, false, true>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((rotary_kernel<kDtype, false, false>), grid, dim3(kThreads), 0, stream, a);
  }
}

// vec: elements of a vector, 0 for any alignment.
template <int kDtype>
void launch_normed(const Args& a, const Norm& n, bool adjacent, int vec, dim3 grid, hipStream_t stream) {
#define MUSC_NORM_ROTARY(...) hipLaunchKernelGGL((__VA_ARGS__), grid, dim3(kThreads), 0, stream, a, n)
  if (vec == 0) {
    if (adjacent) MUSC_NORM_ROTARY(norm_rotary_any_kernel<kDtype, true>);
    else MUSC_NORM_ROTARY(norm_rotary_any_kernel<kDtype, false>);
    return;
  }
  if constexpr (kDtype != MUSC_DTYPE_F32) {
    if (vec == 8) {
      if (adjacent) MUSC_NORM_ROTARY(norm_rotary_kernel<kDtype, true, 8>);
      else MUSC_NORM_ROTARY(norm_rotary_kernel<kDtype, false, 8>);
      return;
    }
  }
  if (adjacent) MUSC_NORM_ROTARY(norm_rotary_kernel<kDtype, true, 4>);
  else MUSC_NORM_ROTARY(norm_rotary_kernel<kDtype, false, 4>);
#undef MUSC_NORM_ROTARY
}

inline uint32_t reciprocal(long long n) { return n > 1 ? (uint32_t)((0x100000000ULL + n - 1) / n) : 0; }

// Checks a call and fills in what both kernels' arguments share.
int arguments(const musc_rotary_call* call, Args& a) {
  if (!call) return MUSC_ERR_INVALID_ARG;
  const auto& [q, q_sb, q_st, q_sh, q_out, qo_sb, qo_st, qo_sh, k, k_sb, k_st, k_sh, k_out, ko_sb, ko_st, ko_sh, positions,
               pos_sb, frequency, axis, q_heads, k_heads, dtype, batch, t, d, int_positions, axes, pairs, adjacent,
               inverse] = *call;
  if (!q || !q_out || !positions || !frequency || !axis || batch < 0 || t < 0 || q_heads < 1 || k_heads < 0 ||
      axes < 1 || pairs < 1 || d < 2 * pairs || pos_sb < 0)
    return MUSC_ERR_INVALID_ARG;
  if (k_heads && (!k || !k_out)) return MUSC_ERR_INVALID_ARG;
  if (dtype != MUSC_DTYPE_F32 && dtype != MUSC_DTYPE_F16 && dtype != MUSC_DTYPE_BF16) return MUSC_ERR_INVALID_ARG;
  if ((q_sb | q_st | q_sh | qo_sb | qo_st | qo_sh) < 0 || (k_heads && (k_sb | k_st | k_sh | ko_sb | ko_st | ko_sh) < 0))
    return MUSC_ERR_INVALID_ARG;
  const long long heads = (long long)q_heads + k_heads;
  if (pairs > kMaxPairs || d > 512 || heads > 1024) return MUSC_ERR_UNSUPPORTED;
  const long long total = (long long)batch * t;
  if (total > 0x7fffffffLL) return MUSC_ERR_UNSUPPORTED;
  const uintptr_t data = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) |
                         (k_heads ? reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out) : 0);
  if (data & (dtype == MUSC_DTYPE_F32 ? 3 : 1)) return MUSC_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(positions) & 3) || (reinterpret_cast<uintptr_t>(frequency) & 7) ||
      (reinterpret_cast<uintptr_t>(axis) & 3))
    return MUSC_ERR_INVALID_ARG;
  a.q = Side{q, q_out, q_sb, q_st, q_sh, qo_sb, qo_st, qo_sh, q_heads};
  a.k = Side{k, k_out, k_sb, k_st, k_sh, ko_sb, ko_st, ko_sh, k_heads};
  a.positions = positions;
  a.pos_sb = pos_sb;
  a.frequency = frequency;
  a.axis = axis;
  a.batch = batch, a.t = t, a.axes = axes, a.pairs = pairs, a.dim = d, a.int_positions = int_positions;
  a.sign = inverse ? -1.f : 1.f;
  // tokens of a workgroup: one sincos per thread, while there are workgroups for every CU
  a.tokens = kThreads / pairs > 1 ? kThreads / pairs : 1;
  if (a.tokens > kMaxTokens) a.tokens = kMaxTokens;
  while (a.tokens > 1 && total / a.tokens < 512) --a.tokens;
  return MUSC_OK;
}

// Whether every vector of n elements starts on its own size.
bool vectors(const musc_rotary_call& c, int n) {
  const uintptr_t data = reinterpret_cast<uintptr_t>(c.q) | reinterpret_cast<uintptr_t>(c.q_out) |
                         (c.k_heads ? reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.k_out) : 0);
  const long long strides = c.q_sb | c.q_st | c.q_sh | c.q_ob | c.q_ot | c.q_oh |
                            (c.k_heads ? c.k_sb | c.k_st | c.k_sh | c.k_ob | c.k_ot | c.k_oh : 0);
  return data % (n * (c.dtype == MUSC_DTYPE_F32 ? 4 : 2)) == 0 && strides % n == 0 && c.d % n == 0 &&
         (c.adjacent ? 2 * c.pairs : c.pairs) % n == 0;
}
int items_of(const musc_rotary_call& c, int n) {
  return n ? (c.adjacent ? 2 * c.pairs / n : c.pairs / n) + (c.d - 2 * c.pairs) / n : c.pairs + (c.d - 2 * c.pairs);
}

}  // namespace rotary
}  // namespace musc

using namespace musc;

extern "C" int musc_rotary(const musc_rotary_call* call, hipStream_t stream) {
  using namespace rotary;
  Args a{};
  if (const int rc = arguments(call, a)) return rc;
  const long long total = (long long)a.batch * a.t, heads = (long long)a.q.heads + a.k.heads;
  if (total == 0) return MUSC_OK;
  const int n = call->dtype == MUSC_DTYPE_F32 ? 4 : 8;
  const bool vec = vectors(*call, n), adjacent = call->adjacent;
  a.items = items_of(*call, vec ? n : 0);
  a.by_items = reciprocal(a.items);
  a.by_heads = reciprocal(heads);
  // the reciprocals divide exactly below 2^32 / divisor (one token: 2^19 * 2^10 at most)
  const long long per_token = heads * a.items, divisor = heads > a.items ? heads : a.items;
  while (a.tokens > 1 && a.tokens * per_token * divisor > 0xffffffffLL) --a.tokens;
  const dim3 grid = linear_grid((total + a.tokens - 1) / a.tokens);
  if (call->dtype == MUSC_DTYPE_F32) launch<MUSC_DTYPE_F32>(a, adjacent, vec, grid, stream);
  else if (call->dtype == MUSC_DTYPE_F16) launch<MUSC_DTYPE_F16>(a, adjacent, vec, grid, stream);
  else launch<MUSC_DTYPE_BF16>(a, adjacent, vec, grid, stream);
  return check_launch();
}

extern "C" int musc_norm_rotary(const musc_rotary_call* call, const void* q_weight, long long q_weight_sh,
                                int q_weight_dtype, const void* k_weight, long long k_weight_sh, int k_weight_dtype,
                                float eps, hipStream_t stream) {
  using namespace rotary;
  Args a{};
  if (const int rc = arguments(call, a)) return rc;
  Norm n{{q_weight, a.k.heads ? k_weight : nullptr}, {q_weight_sh, k_weight_sh}, {q_weight_dtype, k_weight_dtype}};
  const int dtype = call->dtype;
  if (!(eps >= 0.f)) return MUSC_ERR_INVALID_ARG;
  // largest vectors (of up to 64 lanes a head) that start on their own size, weights on 16 bytes at most
  int vec = dtype == MUSC_DTYPE_F32 ? 4 : 8;
  while (vec >= 4 && (!vectors(*call, vec) || items_of(*call, vec) > kWave)) vec /= 2;
  for (int i = 0; i < 2; ++i) {
    if (!n.w[i]) continue;
    const int size = n.w_dtype[i] == MUSC_DTYPE_F32 ? 4 : 2;
    if (n.w_dtype[i] != dtype && n.w_dtype[i] != MUSC_DTYPE_F32) return MUSC_ERR_INVALID_ARG;
    const uintptr_t at = reinterpret_cast<uintptr_t>(n.w[i]);
    if (at % size || n.w_sh[i] < 0) return MUSC_ERR_INVALID_ARG;
    const int bytes = vec * size < 16 ? vec * size : 16;
    if (vec >= 4 && (at % bytes || n.w_sh[i] * size % bytes)) vec = 0;
  }
  const long long total = (long long)a.batch * a.t;
  if (total == 0) return MUSC_OK;
  if (vec < 4) vec = 0;
  a.items = items_of(*call, vec);
  // 8 workgroups a CU: 4 x 1370 tokens 12.2 us so, 12.6 with two; 3 x 900 of 72 channels in fp32 13.6 and 17.8
  while (a.tokens > 1 && total / a.tokens < 2048) --a.tokens;
  while (vec && a.items > 1 << n.lane_bits) ++n.lane_bits;
  a.by_heads = reciprocal((long long)a.q.heads + a.k.heads);  // exact below 2^32 / heads: 16 tokens of 1024 at most
  n.eps = eps;
  const dim3 grid = linear_grid((total + a.tokens - 1) / a.tokens);
  const bool adjacent = call->adjacent;
  if (dtype == MUSC_DTYPE_F32) launch_normed<MUSC_DTYPE_F32>(a, n, adjacent, vec, grid, stream);
  else if (dtype == MUSC_DTYPE_F16) launch_normed<MUSC_DTYPE_F16>(a, n, adjacent, vec, grid, stream);
  else launch_normed<MUSC_DTYPE_BF16>(a, n, adjacent, vec, grid, stream);
  return check_launch();
}
