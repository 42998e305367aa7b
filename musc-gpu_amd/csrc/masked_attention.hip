// Softmax attention over the keys that a query may see, for packed images, padded batches,
// prefixes and frames, with an optional cap on the scores and an optional bias by distance:
//
//   score(i, j) = c(scale q_i . k_j) - sum_a slope[head, a] |p_a(i) - p_a(j)|
//   c(s)        = cap tanh(s / cap), or s
//   seen(i, j)  = document(i) == document(j) >= 0 and order(j) <= order(i)
//   out_i       = sum_seen e^(score - max) v_j / sum_seen e^(score - max); zeros if none is seen
//
// One pass over the keys with the running maximum and sum of the softmax.  As in the
// unmasked kernels a wave forms S^T = K Q^T, so that a lane owns one query row and its
// maximum, sum and probabilities stay in its registers; O^T += V^T P^T follows with P in
// place.  A row is a (token, head of the group) pair: the heads that share a key head are
// neighbouring rows, so K and V are read once for all of them.
//
// Keys come in tiles of kTile.  A small summary of the keys (per 32 of them the range of
// documents and orders, made once per batch) sorts a tile, for the rows of a wave, into unseen
// (skipped without reading K or V), seen whole (no mask is evaluated) and mixed (each score is
// tested).  64 tiles are sorted at a time, one per lane.
//
// Few rows (a new token, a pooling latent): the keys are split over workgroups of one wave
// that write (maximum, sum, output) parts, and a second kernel joins them in a fixed order.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.hpp"

namespace musc {
namespace mattn {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

constexpr int kBufferFlags = 0x00020000;   // buffer resource word 3 for raw byte-addressed loads
constexpr int kNowhere = 0x7fffff00;       // a byte offset past every extent: such loads give zeros
constexpr float kLazyLog2 = 8.f;           // the running maximum moves once a tile exceeds it by this
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSummaryKeys = 32;
constexpr int kMaxAxes = 3;

template <int kDtype>
struct Type;
template <>
struct Type<MUSC_DTYPE_F32> {
  typedef float T;
  static constexpr int kTile = 32;
  static constexpr float kShift = 0.f;
};
template <>
struct Type<MUSC_DTYPE_F16> {
  typedef _Float16 T;
  typedef half8 Vec;
  static constexpr int kTile = 64;
  // probabilities are formed 2^7 times as large, at most 2^15 with the slack: entries down to
  // 2^-21 of the largest stay normal fp16 numbers
  static constexpr float kShift = 7.f;
  static __device__ __forceinline__ floatx16 mfma(Vec a, Vec b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Type<MUSC_DTYPE_BF16> {
  typedef __bf16 T;
  typedef bf8 Vec;
  static constexpr int kTile = 64;
  static constexpr float kShift = 0.f;
  static __device__ __forceinline__ floatx16 mfma(Vec a, Vec b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

struct Args {
  musc_masked_attention c;
  int group, rows, row_tiles, key_tiles, splits, summaries;
  long long units;
  float* part_ml;  // (units in (b, kv head), rows, split) x (maximum, sum)
  float* part_o;   // the same x d
};

__device__ __forceinline__ float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int wave_min_int(int v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = min(v, __shfl_xor(v, off, kWave));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_int(int v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = max(v, __shfl_xor(v, off, kWave));
  return __builtin_amdgcn_readfirstlane(v);
}

// The documents and orders of a set of rows: what a tile is compared with.
struct Range {
  int dmin, dmax, omin, omax;
};

// Per 32 keys: smallest and largest document (negative ones count as -1), smallest and largest
// order of the keys that have a document.  One wave handles two groups of 32.
__global__ __launch_bounds__(256) void token_summary_kernel(const int* __restrict__ documents,
                                                            const int* __restrict__ order, int batch, int t,
                                                            int groups, int4* __restrict__ summary) {
  const long long g = ((long long)blockIdx.x * 256 + threadIdx.x) / kSummaryKeys;
  if (g >= (long long)batch * groups) return;  // whole halves of a wave; the shuffles stay inside them
  const int b = (int)(g / groups), first = (int)(g % groups) * kSummaryKeys;
  const int key = first + threadIdx.x % kSummaryKeys;
  int doc = -1, ord = 0;
  if (key < t) {
    doc = max(documents[(long long)b * t + key], -1);
    if (order) ord = order[(long long)b * t + key];
  }
  int4 s = make_int4(doc, doc, doc < 0 ? 0x7fffffff : ord, doc < 0 ? (int)0x80000000 : ord);
#pragma unroll
  for (int off = kSummaryKeys / 2; off >= 1; off >>= 1) {
    s.x = min(s.x, __shfl_xor(s.x, off, kSummaryKeys));
    s.y = max(s.y, __shfl_xor(s.y, off, kSummaryKeys));
    s.z = min(s.z, __shfl_xor(s.z, off, kSummaryKeys));
    s.w = max(s.w, __shfl_xor(s.w, off, kSummaryKeys));
  }
  if (threadIdx.x % kSummaryKeys == 0) summary[g] = s;
}

// tanh for 16-bit operands: 1 - 2 / (1 + e^2x), absolute error a few 2^-24
__device__ __forceinline__ float tanh_fast(float x) {
  return fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(2.f * kLog2e * x)), 1.f);
}

// kWaves waves of 32 rows each; kD: head width rounded up to 64, 96 or 128.
template <int kDtype, int kD, int kWaves>
__global__ __launch_bounds__(kWaves * kWave) void masked_attention_kernel(const Args a) {
  using Ty = Type<kDtype>;
  typedef typename Ty::T T;
  constexpr bool k16 = kDtype != MUSC_DTYPE_F32;
  constexpr int kTile = Ty::kTile, kSub = kTile / 32;
  constexpr int kPer = 16 / (int)sizeof(T);            // elements of a 16-byte vector
  constexpr int kPitch = kD + kPer;                    // elements of a staged row
  constexpr int kBuffers = kWaves > 1 ? 2 : 1;         // one wave reads a tile before it stores the next
  constexpr int kThreads = kWaves * kWave;
  constexpr int kChunks = kTile * (kD / kPer) / kThreads;  // vectors of K (and of V) a thread stages
  static_assert(kTile * (kD / kPer) % kThreads == 0, "whole vectors per thread");
  constexpr int kO = kD / 32;
  __shared__ __attribute__((aligned(16))) T Ks[kBuffers][kTile * kPitch];
  __shared__ __attribute__((aligned(16))) T Vs[kBuffers][kTile * kPitch];
  __shared__ __attribute__((aligned(16))) int docs_s[kBuffers][kTile], ords_s[kBuffers][kTile];
  __shared__ Range ranges[kWaves];

  const musc_masked_attention& c = a.c;
  const long long unit = xcd_logical_id(blockIdx.x, gridDim.x);
  if (unit >= a.units) return;
  const int split = (int)(unit % a.splits);
  const int row_tile = (int)(unit / a.splits % a.row_tiles);
  const long long bh = unit / a.splits / a.row_tiles;
  const int b = (int)(bh / c.kv_heads), kvh = (int)(bh % c.kv_heads);
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int lq = lane & 31, lh = lane >> 5;
  const int row = (row_tile * kWaves + wave) * 32 + lq;
  const bool inside = row < a.rows;
  const int token = inside ? row / a.group : 0;
  const int head = kvh * a.group + (inside ? row % a.group : 0);
  const int d = c.d, k_len = c.k_len;

  // this row's document and order; rows outside the tensor and padding have none
  int qdoc = -2, qord = 0;
  if (inside) {
    qdoc = c.q_documents ? c.q_documents[b * c.q_tokens_sb + token] : 0;
    if (qdoc < 0) qdoc = -2;
    if (c.q_order) qord = c.q_order[b * c.q_tokens_sb + token];
  }
  const bool live = qdoc >= 0;
  Range mine, all_rows;
  mine.dmin = wave_min_int(live ? qdoc : 0x7fffffff);
  mine.dmax = wave_max_int(live ? qdoc : -1);
  mine.omin = wave_min_int(live ? qord : 0x7fffffff);
  mine.omax = wave_max_int(live ? qord : (int)0x80000000);
  all_rows = mine;
  if constexpr (kWaves > 1) {
    if (lane == 0) ranges[wave] = mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      all_rows.dmin = min(all_rows.dmin, ranges[w].dmin);
      all_rows.dmax = max(all_rows.dmax, ranges[w].dmax);
      all_rows.omin = min(all_rows.omin, ranges[w].omin);
      all_rows.omax = max(all_rows.omax, ranges[w].omax);
    }
  }

  // Q fragments, zeros past d
  const T* qrow = static_cast<const T*>(c.q) + b * c.q_sb + (long long)token * c.q_st + head * c.q_sh;
  constexpr int kQ = k16 ? kD / 16 : kD / 8;
  typedef T TVec __attribute__((ext_vector_type(kPer)));
  TVec qf[kQ];
#pragma unroll
  for (int m = 0; m < kQ; ++m) {
    const int at = (k16 ? 16 * m + 8 * lh : 8 * m + 4 * lh);
    TVec x = {};
    if (live && at < d) x = *reinterpret_cast<const TVec*>(qrow + at);
    qf[m] = x;
  }
  const int axes = c.axes;
  float qpos[kMaxAxes], slope[kMaxAxes];  // the B operand of the distances: 1 and -position
#pragma unroll
  for (int x = 0; x < kMaxAxes; ++x) {
    qpos[x] = 0.f, slope[x] = 0.f;
    if (x < axes) {
      const float p = c.q_positions[b * c.q_positions_sb + (long long)token * axes + x];
      qpos[x] = lh == 0 ? 1.f : -p;
      slope[x] = c.slopes[head * axes + x] * kLog2e;
    }
  }
  const float scale_log2 = c.scale * kLog2e;
  const float cap_log2 = c.cap * kLog2e, scale_by_cap = c.cap > 0.f ? c.scale / c.cap : 0.f;

  // tiles of this split
  const int lo = (int)((long long)a.key_tiles * split / a.splits);
  const int hi = (int)((long long)a.key_tiles * (split + 1) / a.splits);

  // K and V rows of a tile through buffer resources that end with the last key
  const T* kbase = static_cast<const T*>(c.k) + b * c.k_sb + (long long)kvh * c.k_sh;
  const T* vbase = static_cast<const T*>(c.v) + b * c.v_sb + (long long)kvh * c.v_sh;
  TVec kreg[kChunks], vreg[kChunks];
  int dreg = 0, oreg = 0;
  float kpos[kMaxAxes][kSub], kpos_next[kMaxAxes][kSub];
  auto load_tile = [&](int tile) {
    const int first = tile * kTile, rem = min(k_len - first, kTile);
    const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(kbase + (long long)first * c.k_st), (short)0,
                                                      (int)(((rem - 1) * c.k_st + d) * (int)sizeof(T)), kBufferFlags);
    const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(vbase + (long long)first * c.v_st), (short)0,
                                                      (int)(((rem - 1) * c.v_st + d) * (int)sizeof(T)), kBufferFlags);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int e = i * kThreads + tid, key = e / (kD / kPer), at = e % (kD / kPer) * kPer;
      const int ko = at < d ? (int)((key * c.k_st + at) * (int)sizeof(T)) : kNowhere;
      const int vo = at < d ? (int)((key * c.v_st + at) * (int)sizeof(T)) : kNowhere;
      kreg[i] = __builtin_bit_cast(TVec, __builtin_amdgcn_raw_buffer_load_b128(rk, ko, 0, 0));
      vreg[i] = __builtin_bit_cast(TVec, __builtin_amdgcn_raw_buffer_load_b128(rv, vo, 0, 0));
    }
    if (tid < kTile) {
      const int key = first + tid;
      dreg = key < k_len ? 0 : -1, oreg = 0;
      if (key < k_len && c.k_documents) dreg = max(c.k_documents[b * c.k_tokens_sb + key], -1);
      if (key < k_len && c.k_order) oreg = c.k_order[b * c.k_tokens_sb + key];
    }
#pragma unroll
    for (int x = 0; x < kMaxAxes; ++x)
      if (x < axes)
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          const int key = min(first + 32 * s + lq, k_len - 1);
          kpos_next[x][s] = c.k_positions[b * c.k_positions_sb + (long long)key * axes + x];
        }
  };
  auto store_tile = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int e = i * kThreads + tid, key = e / (kD / kPer), at = e % (kD / kPer) * kPer;
      *reinterpret_cast<TVec*>(&Ks[buf][key * kPitch + at]) = kreg[i];
      *reinterpret_cast<TVec*>(&Vs[buf][key * kPitch + at]) = vreg[i];
    }
    if (tid < kTile) docs_s[buf][tid] = dreg, ords_s[buf][tid] = oreg;
#pragma unroll
    for (int x = 0; x < kMaxAxes; ++x)
#pragma unroll
      for (int s = 0; s < kSub; ++s) kpos[x][s] = kpos_next[x][s];
  };

  floatx16 o[kO];
  float m_run, l_run;
  bool mixed_seen;

  // one staged tile; whole: every row sees every key.  careful: in a mixed tile, products
  // of keys that a row does not see are left out one by one (their V may be infinite or NaN)
  auto attend = [&](int buf, bool whole, bool careful) {
    floatx16 s[kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
#pragma unroll
      for (int v = 0; v < 16; ++v) s[u][v] = 0.f;
      const T* krow = &Ks[buf][(32 * u + lq) * kPitch];
      if constexpr (k16) {
#pragma unroll
        for (int m = 0; m < kQ; ++m)
          s[u] = Ty::mfma(*reinterpret_cast<const TVec*>(krow + 16 * m + 8 * lh), qf[m], s[u]);
      } else {
#pragma unroll
        for (int m = 0; m < kQ; ++m) {
          const TVec x = *reinterpret_cast<const TVec*>(krow + 8 * m + 4 * lh);
#pragma unroll
          for (int j = 0; j < 4; ++j) s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], qf[m][j], s[u], 0, 0, 0);
        }
      }
    }
    // scores in log2 units
    if (cap_log2 > 0.f) {
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const float x = s[u][v] * scale_by_cap;
          s[u][v] = cap_log2 * (k16 ? tanh_fast(x) : tanhf(x));
        }
    } else {
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[u][v] *= scale_log2;
    }
    // distances from the matrix cores: position(j) * 1 + 1 * -position(i), exact in fp32
#pragma unroll
    for (int x = 0; x < kMaxAxes; ++x)
      if (x < axes)
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          floatx16 apart;
#pragma unroll
          for (int v = 0; v < 16; ++v) apart[v] = 0.f;
          apart = __builtin_amdgcn_mfma_f32_32x32x2f32(lh == 0 ? kpos[x][u] : 1.f, qpos[x], apart, 0, 0, 0);
#pragma unroll
          for (int v = 0; v < 16; ++v) s[u][v] = fmaf(-slope[x], fabsf(apart[v]), s[u][v]);
        }
    // register v of block u holds key 32 u + 8 (v / 4) + 4 lh + v % 4
    uint32_t seen = 0xffffffffu;
    if (!whole) {
      mixed_seen = true;
      seen = 0;
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int4 kd = *reinterpret_cast<const int4*>(&docs_s[buf][32 * u + 8 * g + 4 * lh]);
          const int4 ko = *reinterpret_cast<const int4*>(&ords_s[buf][32 * u + 8 * g + 4 * lh]);
          const bool see[4] = {kd.x == qdoc && ko.x <= qord, kd.y == qdoc && ko.y <= qord,
                               kd.z == qdoc && ko.z <= qord, kd.w == qdoc && ko.w <= qord};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!see[i]) s[u][4 * g + i] = -INFINITY;
            if (see[i]) seen |= 1u << (16 * u + 4 * g + i);
          }
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) top = __builtin_elementwise_maximum(top, s[u][v]);
    top = halves_max(top);
    if (!__all(top <= m_run + kLazyLog2)) {
      const float m_new = fmaxf(m_run, top);
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));  // 0 at first
      l_run *= alpha;
#pragma unroll
      for (int x = 0; x < kO; ++x)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[x][v] *= alpha;
      m_run = m_new;
    }
    const float base = (m_run == -INFINITY ? 0.f : m_run) - Ty::kShift;  // nothing seen yet: e^-inf = 0
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        s[u][v] = __builtin_amdgcn_exp2f(s[u][v] - base);
        sum += s[u][v];
      }
    l_run += sum;  // this half's keys
    if (careful && !whole) {
      for (int key = 0; key < kTile; ++key) {
        const int u0 = key >> 5, v0 = ((key & 31) >> 3) * 4 + (key & 3), from = lq + 32 * ((key >> 2) & 1);
        float p = 0.f;
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (u == u0 && v == v0) p = s[u][v];
        p = __shfl(p, from, kWave);
        const bool see = (__shfl(seen, from, kWave) >> (16 * u0 + v0)) & 1;
        const T* vrow = &Vs[buf][key * kPitch];
#pragma unroll
        for (int x = 0; x < kO; ++x)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const float value = (float)vrow[32 * x + 8 * (v >> 2) + 4 * lh + (v & 3)];
            if (see) o[x][v] = fmaf(p, value, o[x][v]);
          }
      }
      return;
    }
    if constexpr (k16) {
      // V^T fragments by transposing LDS reads: within a group of 16 lanes, lane i's element j
      // is element i % 4 of the 8 bytes that lane 4 j + i / 4 addressed, so with V row-major the
      // lane that addresses V[key0 + r / 4][d0 + 4 (r % 4) ..] (r its place in the group) hands
      // element j of lane i the value V[key0 + j][d0 + i]: the A operand's row d0 + i, k = j
      const T* vb = &Vs[buf][(4 * lh + ((lq & 15) >> 2)) * kPitch + 16 * (lq >> 4) + 4 * (lq & 3)];
      auto tr = [&](int off) {
        typedef __attribute__((address_space(3))) short4v lds_short4v;
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v*)(vb + off));
      };
#pragma unroll
      for (int mm = 0; mm < 2 * kSub; ++mm) {
        TVec p;
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = (T)s[mm >> 1][8 * (mm & 1) + j];
#pragma unroll
        for (int x = 0; x < kO; ++x) {
          const short4v f0 = tr(16 * mm * kPitch + 32 * x), f1 = tr((16 * mm + 8) * kPitch + 32 * x);
          typedef short short8v __attribute__((ext_vector_type(8)));
          const short8v f = {f0[0], f0[1], f0[2], f0[3], f1[0], f1[1], f1[2], f1[3]};
          o[x] = Ty::mfma(__builtin_bit_cast(TVec, f), p, o[x]);
        }
      }
    } else {
      // step e takes keys 8 (e / 4) + 4 lh + e % 4: register e of s
#pragma unroll
      for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int x = 0; x < kO; ++x)
          o[x] = __builtin_amdgcn_mfma_f32_32x32x2f32(Vs[buf][(8 * (e >> 2) + 4 * lh + (e & 3)) * kPitch + 32 * x + lq],
                                                      s[0][e], o[x], 0, 0, 0);
    }
  };

  // the tiles of this split that some row of the workgroup may see, 64 sorted at a time
  int chunk = 0;
  unsigned long long todo = 0, any_word = 0, whole_word = 0;
  auto sort_tiles = [&]() {
    const int t = chunk * 64 + lane;
    int4 k = make_int4(0, 0, 0, 0);
    const bool here = t >= lo && t < hi;
    if (here && c.k_summary) {
      const int4* sum = reinterpret_cast<const int4*>(c.k_summary) + b * c.k_summary_sb + (long long)t * kSub;
      k = sum[0];
      if (kSub > 1 && t * kSub + 1 < a.summaries) {
        const int4 n = sum[1];
        k = make_int4(min(k.x, n.x), max(k.y, n.y), min(k.z, n.z), max(k.w, n.w));
      }
    }
    auto may_see = [&](const Range& r) {
      return here && k.y >= 0 && k.x <= r.dmax && k.y >= r.dmin && k.z <= r.omax;
    };
    todo = __ballot(may_see(all_rows));
    any_word = __ballot(may_see(mine));
    whole_word = __ballot(here && k.x == k.y && mine.dmin == mine.dmax && k.x == mine.dmin && k.w <= mine.omin &&
                          (t + 1) * kTile <= k_len);
  };
  struct Next {
    int tile;
    bool any, whole;
  };
  auto next_tile = [&]() -> Next {
    while (todo == 0) {
      ++chunk;
      if ((long long)chunk * 64 >= hi) return Next{-1, false, false};
      sort_tiles();
    }
    const int bit = __builtin_ctzll(todo);
    todo &= todo - 1;
    return Next{chunk * 64 + bit, (bool)((any_word >> bit) & 1), (bool)((whole_word >> bit) & 1)};
  };

  for (int pass = 0;; ++pass) {
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[x][v] = 0.f;
    m_run = -INFINITY, l_run = 0.f, mixed_seen = false;
    chunk = lo / 64 - 1;
    todo = 0;
    Next now = next_tile();
    if (now.tile >= 0) load_tile(now.tile);
    int buf = 0;
    while (now.tile >= 0) {
      store_tile(buf);
      const Next then = next_tile();
      if (then.tile >= 0) load_tile(then.tile);
      __syncthreads();  // a buffer is written again only past the next tile's barrier
      if (now.any) attend(buf, now.whole, pass > 0);
      if constexpr (kBuffers == 1) __syncthreads();
      else buf ^= 1;
      now = then;
    }
    if (pass > 0) break;
    // 0 * V of an unseen key is NaN where V is not finite: then all over again, with care
    bool bad = false;
    if (mixed_seen && live) {
#pragma unroll
      for (int x = 0; x < kO; ++x)
#pragma unroll
        for (int v = 0; v < 16; ++v) bad |= !(fabsf(o[x][v]) < INFINITY);
    }
    if (!__syncthreads_or(bad)) break;
  }

  l_run = halves_sum(l_run);
  if (!inside) return;
  // register v of block x holds channel 32 x + 8 (v / 4) + 4 lh + v % 4
  if (a.splits == 1) {
    const bool empty = !live || l_run == 0.f;
    const float inv = 1.f / l_run;
    T* orow = static_cast<T*>(c.out) + b * c.o_sb + (long long)token * c.o_st + head * c.o_sh;
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = 32 * x + 8 * g + 4 * lh;
        typedef T Four __attribute__((ext_vector_type(4)));
        Four y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = empty ? (T)0.f : (T)(o[x][4 * g + i] * inv);
        if (at < d) *reinterpret_cast<Four*>(orow + at) = y;
      }
  } else {
    const long long part = (bh * a.rows + row) * a.splits + split;
    if (lh == 0) {
      a.part_ml[2 * part] = live ? m_run : -INFINITY;
      a.part_ml[2 * part + 1] = live ? l_run : 0.f;
    }
    float* prow = a.part_o + part * d;
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = 32 * x + 8 * g + 4 * lh;
        const float4 y = make_float4(o[x][4 * g], o[x][4 * g + 1], o[x][4 * g + 2], o[x][4 * g + 3]);
        if (at < d) *reinterpret_cast<float4*>(prow + at) = live ? y : make_float4(0.f, 0.f, 0.f, 0.f);
      }
  }
}

// Joins the splits of a row, in their order: one wave per row, two channels per lane.
template <int kDtype>
__global__ __launch_bounds__(256) void join_kernel(const Args a, long long total_rows) {
  typedef typename Type<kDtype>::T T;
  const musc_masked_attention& c = a.c;
  const long long r = (long long)blockIdx.x * 4 + threadIdx.x / kWave;
  if (r >= total_rows) return;
  const int lane = threadIdx.x % kWave;
  const long long bh = r / a.rows;
  const int row = (int)(r % a.rows), token = row / a.group;
  const int head = (int)(bh % c.kv_heads) * a.group + row % a.group;
  const float* ml = a.part_ml + 2 * r * a.splits;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[2 * s]);
  float sum = 0.f, y0 = 0.f, y1 = 0.f;
  const bool ok = 2 * lane < c.d;
  for (int s = 0; s < a.splits; ++s) {
    const float m = ml[2 * s];
    if (ml[2 * s + 1] == 0.f) continue;  // nothing seen (a part whose scores are NaN has its sum NaN)
    const float w = __builtin_amdgcn_exp2f(m - top);
    sum = fmaf(w, ml[2 * s + 1], sum);
    if (ok) {
      const float2 p = *reinterpret_cast<const float2*>(a.part_o + (r * a.splits + s) * c.d + 2 * lane);
      y0 = fmaf(w, p.x, y0);
      y1 = fmaf(w, p.y, y1);
    }
  }
  if (!ok) return;
  const float inv = 1.f / sum;
  typedef T Two __attribute__((ext_vector_type(2)));
  Two y;
  y[0] = sum == 0.f ? (T)0.f : (T)(y0 * inv);
  y[1] = sum == 0.f ? (T)0.f : (T)(y1 * inv);
  T* orow = static_cast<T*>(c.out) + (bh / c.kv_heads) * c.o_sb + (long long)token * c.o_st + head * c.o_sh;
  *reinterpret_cast<Two*>(orow + 2 * lane) = y;
}

// Shape of the launch: rows per workgroup, tiles and splits.
int plan(const musc_masked_attention& c, Args& a, int& waves) {
  const int tile = c.dtype == MUSC_DTYPE_F32 ? 32 : 64;
  a.c = c;
  a.group = c.heads / c.kv_heads;
  const long long rows = (long long)c.q_len * a.group;
  if (rows > 0x7fffff00LL || c.k_len > 0x7fffff00) return MUSC_ERR_UNSUPPORTED;
  a.rows = (int)rows;
  waves = rows <= 32 ? 1 : 4;
  a.row_tiles = (int)((rows + 32 * waves - 1) / (32 * waves));
  a.key_tiles = (c.k_len + tile - 1) / tile;
  a.summaries = (c.k_len + kSummaryKeys - 1) / kSummaryKeys;
  const long long whole = (long long)c.batch * c.kv_heads * a.row_tiles;
  long long splits = 1;
  const long long want = waves == 1 ? 2048 : 512;
  if (whole < want / 2) splits = (want + whole - 1) / whole;
  if (splits > a.key_tiles) splits = a.key_tiles;
  if (splits > 256) splits = 256;
  a.splits = splits < 1 ? 1 : (int)splits;
  a.units = whole * a.splits;
  if (a.units >= (0x100000000LL >> 8)) return MUSC_ERR_UNSUPPORTED;  // 256 threads each in one grid dimension
  return MUSC_OK;
}

size_t part_bytes(const Args& a) {
  if (a.splits == 1) return 0;
  const size_t parts = (size_t)a.c.batch * a.c.kv_heads * a.rows * a.splits;
  return align_up(parts * 2 * sizeof(float), 256) + parts * a.c.d * sizeof(float);
}

// 16-byte vectors from every row of a tensor
inline bool aligned(const void* p, long long sb, long long st, long long sh, int per) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && sb >= 0 && st >= 0 && sh >= 0 && (sb | st | sh) % per == 0;
}

int check(const musc_masked_attention* c) {
  if (!c || !c->q || !c->k || !c->v || !c->out) return MUSC_ERR_INVALID_ARG;
  if (c->dtype != MUSC_DTYPE_F32 && c->dtype != MUSC_DTYPE_F16 && c->dtype != MUSC_DTYPE_BF16) return MUSC_ERR_INVALID_ARG;
  if (c->batch < 1 || c->q_len < 1 || c->k_len < 1 || c->heads < 1 || c->kv_heads < 1 || c->heads % c->kv_heads)
    return MUSC_ERR_INVALID_ARG;
  if (!(c->cap >= 0.f) || c->cap > 3e38f || !(fabsf(c->scale) <= 3e38f)) return MUSC_ERR_INVALID_ARG;
  const int per = c->dtype == MUSC_DTYPE_F32 ? 4 : 8, size = 16 / per;
  if (c->d < 1 || c->d > 128 || c->d % per) return MUSC_ERR_UNSUPPORTED;
  if (!aligned(c->q, c->q_sb, c->q_st, c->q_sh, per) || !aligned(c->k, c->k_sb, c->k_st, c->k_sh, per) ||
      !aligned(c->v, c->v_sb, c->v_st, c->v_sh, per) || !aligned(c->out, c->o_sb, c->o_st, c->o_sh, per))
    return MUSC_ERR_INVALID_ARG;
  if ((63 * c->k_st + c->d) * size > kNowhere - 16 || (63 * c->v_st + c->d) * size > kNowhere - 16)
    return MUSC_ERR_UNSUPPORTED;
  // documents on both sides and the keys' summary, or none; orders and positions likewise
  if (!c->q_documents != !c->k_documents || !c->k_documents != !c->k_summary) return MUSC_ERR_INVALID_ARG;
  if (!c->q_order != !c->k_order || (c->q_order && !c->q_documents)) return MUSC_ERR_INVALID_ARG;
  if (c->axes < 0 || c->axes > kMaxAxes) return MUSC_ERR_UNSUPPORTED;
  if (c->axes && (!c->q_positions || !c->k_positions || !c->slopes)) return MUSC_ERR_INVALID_ARG;
  const uintptr_t words = reinterpret_cast<uintptr_t>(c->q_documents) | reinterpret_cast<uintptr_t>(c->k_documents) |
                          reinterpret_cast<uintptr_t>(c->q_order) | reinterpret_cast<uintptr_t>(c->k_order) |
                          reinterpret_cast<uintptr_t>(c->q_positions) | reinterpret_cast<uintptr_t>(c->k_positions) |
                          reinterpret_cast<uintptr_t>(c->slopes);
  if ((words & 3) || (reinterpret_cast<uintptr_t>(c->k_summary) & 15)) return MUSC_ERR_INVALID_ARG;
  if ((c->q_tokens_sb | c->k_tokens_sb | c->q_positions_sb | c->k_positions_sb | c->k_summary_sb) < 0)
    return MUSC_ERR_INVALID_ARG;
  return MUSC_OK;
}

template <int kDtype, int kD>
void launch(const Args& a, int waves, hipStream_t stream) {
  const dim3 grid((unsigned)align_up((size_t)a.units, kXcds));
  if (waves == 1)
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, 1>), grid, dim3(kWave), 0, stream, a);
  else
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, 4>), grid, dim3(4 * kWave), 0, stream, a);
}

template <int kDtype>
void launch(const Args& a, int waves, hipStream_t stream) {
  if (a.c.d <= 64) launch<kDtype, 64>(a, waves, stream);
  else if (a.c.d <= 96) launch<kDtype, 96>(a, waves, stream);
  else launch<kDtype, 128>(a, waves, stream);
  if (a.splits > 1) {
    const long long rows = (long long)a.c.batch * a.c.kv_heads * a.rows;
    hipLaunchKernelGGL((join_kernel<kDtype>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a, rows);
  }
}

}  // namespace mattn
}  // namespace musc

using namespace musc;

extern "C" int musc_token_summary(const int* documents, const int* order, int batch, int t, int* summary,
                                  hipStream_t stream) {
  if (!documents || !summary || batch < 0 || t < 0) return MUSC_ERR_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(documents) | reinterpret_cast<uintptr_t>(order)) & 3) ||
      (reinterpret_cast<uintptr_t>(summary) & 15))
    return MUSC_ERR_INVALID_ARG;
  if (batch == 0 || t == 0) return MUSC_OK;
  const int groups = (int)(((long long)t + mattn::kSummaryKeys - 1) / mattn::kSummaryKeys);
  const long long blocks = ((long long)batch * groups * mattn::kSummaryKeys + 255) / 256;
  if (blocks >= (0x100000000LL >> 8)) return MUSC_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(mattn::token_summary_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, documents, order, batch,
                     t, groups, reinterpret_cast<int4*>(summary));
  return check_launch();
}

extern "C" int musc_masked_attention_workspace_bytes(const musc_masked_attention* c, size_t* out) {
  if (!out) return MUSC_ERR_INVALID_ARG;
  if (const int rc = mattn::check(c)) return rc;
  mattn::Args a{};
  int waves;
  if (const int rc = mattn::plan(*c, a, waves)) return rc;
  *out = mattn::part_bytes(a);
  return MUSC_OK;
}

extern "C" int musc_masked_attention_fwd(const musc_masked_attention* c, void* workspace, size_t workspace_bytes,
                                         hipStream_t stream) {
  if (const int rc = mattn::check(c)) return rc;
  mattn::Args a{};
  int waves;
  if (const int rc = mattn::plan(*c, a, waves)) return rc;
  const size_t need = mattn::part_bytes(a);
  if (need) {
    if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16) return MUSC_ERR_WORKSPACE;
    a.part_ml = static_cast<float*>(workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                        align_up((size_t)c->batch * c->kv_heads * a.rows * a.splits * 2 * sizeof(float), 256));
  }
  if (c->dtype == MUSC_DTYPE_F32) mattn::launch<MUSC_DTYPE_F32>(a, waves, stream);
  else if (c->dtype == MUSC_DTYPE_F16) mattn::launch<MUSC_DTYPE_F16>(a, waves, stream);
  else mattn::launch<MUSC_DTYPE_BF16>(a, waves, stream);
  return check_launch();
}
