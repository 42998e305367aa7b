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
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

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

}  // namespace rotary
}  // namespace musc

using namespace musc;

extern "C" int musc_rotary(const musc_rotary_call* call, hipStream_t stream) {
  using namespace rotary;
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
  if (total == 0) return MUSC_OK;
  const int n = dtype == MUSC_DTYPE_F32 ? 4 : 8;
  const long long strides = q_sb | q_st | q_sh | qo_sb | qo_st | qo_sh |
                            (k_heads ? k_sb | k_st | k_sh | ko_sb | ko_st | ko_sh : 0);
  const bool vec = data % 16 == 0 && strides % n == 0 && d % n == 0 && (adjacent ? 2 * pairs : pairs) % n == 0 &&
                   (2 * pairs) % n == 0;
  Args a{};
  a.q = Side{q, q_out, q_sb, q_st, q_sh, qo_sb, qo_st, qo_sh, q_heads};
  a.k = Side{k, k_out, k_sb, k_st, k_sh, ko_sb, ko_st, ko_sh, k_heads};
  a.positions = positions;
  a.pos_sb = pos_sb;
  a.frequency = frequency;
  a.axis = axis;
  a.batch = batch, a.t = t, a.axes = axes, a.pairs = pairs, a.dim = d, a.int_positions = int_positions;
  a.items = vec ? (adjacent ? 2 * pairs / n : pairs / n) + (d - 2 * pairs) / n : pairs + (d - 2 * pairs);
  a.by_items = a.items > 1 ? (uint32_t)((0x100000000ULL + a.items - 1) / a.items) : 0;
  a.by_heads = heads > 1 ? (uint32_t)((0x100000000ULL + heads - 1) / heads) : 0;
  a.sign = inverse ? -1.f : 1.f;
  // tokens of a workgroup: one sincos per thread, while there are workgroups for every CU
  int tokens = kThreads / pairs > 1 ? kThreads / pairs : 1;
  if (tokens > kMaxTokens) tokens = kMaxTokens;
  while (tokens > 1 && total / tokens < 512) --tokens;
  // the reciprocals divide exactly below 2^32 / divisor (one token: 2^19 * 2^10 at most)
  const long long per_token = heads * a.items, divisor = heads > a.items ? heads : a.items;
  while (tokens > 1 && tokens * per_token * divisor > 0xffffffffLL) --tokens;
  a.tokens = tokens;
  const dim3 grid = linear_grid((total + tokens - 1) / tokens);
  if (dtype == MUSC_DTYPE_F32) launch<MUSC_DTYPE_F32>(a, adjacent, vec, grid, stream);
  else if (dtype == MUSC_DTYPE_F16) launch<MUSC_DTYPE_F16>(a, adjacent, vec, grid, stream);
  else launch<MUSC_DTYPE_BF16>(a, adjacent, vec, grid, stream);
  return check_launch();
}
