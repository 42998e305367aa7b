// Root-mean-square norm of rows, with the residual's addition and, on request, an 8-bit
// output with scales (the norm in front of an 8-bit product).
//
//   s = x + r rounded to the storage type (s = x without a residual)
//   y = s * w / sqrt(mean(s^2) + eps)                         fp32, rounded once
//   8 bits: per row, or per group of columns, scale = max|y| / MAX (MAX the type's largest
//   number), q = round(y / scale)
//
// One read of x (and r), one write of s and y: bound by HBM.  A row is held in registers
// by the threads that share it (a wave up to 256 vectors of 16 bytes, then 256 and 1024 threads, at
// most 4 vectors each), from its loads, all asked for at once, to its last store: 16384 x 8192
// bf16 with residual, 8 bits in groups of 128 columns, 169 us = 5.6 TB/s (a large copy 5.2); 5480 x
// 1024 fp16 with residual 8.8 us = 5.1 TB/s; 8 x 4096 4.6 us, its latency.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.hpp"
#include "storage.hpp"

namespace musc {
namespace rms {

constexpr int kMaxChunks = 4;  // vectors of 16 bytes per thread

// N consecutive values from element `at`; those from `limit` on (scalar variant only) are 0.
template <int kDtype, bool kVec>
__device__ __forceinline__ void load_row(const void* base, long long at, int col, int limit,
                                         float (&v)[Storage<kDtype>::N]) {
  using S = Storage<kDtype>;
  if constexpr (kVec) {
    S::load(static_cast<const typename S::T*>(base) + at + col, v);
  } else {
#pragma unroll
    for (int j = 0; j < S::N; ++j)
      v[j] = col + j < limit ? S::one(static_cast<const typename S::T*>(base)[at + col + j]) : 0.f;
  }
}

template <int kDtype, bool kVec>
__device__ __forceinline__ void store_row(void* base, long long at, int col, int limit,
                                          const float (&v)[Storage<kDtype>::N]) {
  using S = Storage<kDtype>;
  if constexpr (kVec) {
    S::store(static_cast<typename S::T*>(base) + at + col, v);
  } else {
#pragma unroll
    for (int j = 0; j < S::N; ++j)
      if (col + j < limit) static_cast<typename S::T*>(base)[at + col + j] = S::round(v[j]);
  }
}

// Sum or NaN-propagating maximum over the kTpr threads of a row.
template <int kTpr, bool kMax>
__device__ __forceinline__ float row_reduce(float v, float* shared) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const float o = __shfl_xor(v, off, kWave);
    v = kMax ? __builtin_elementwise_maximum(v, o) : v + o;
  }
  if constexpr (kTpr > kWave) {
    constexpr int kWaves = kTpr / kWave;
    __syncthreads();  // the words of an earlier reduction have been read
    if (threadIdx.x % kWave == 0) shared[threadIdx.x / kWave] = v;
    __syncthreads();
    v = shared[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) v = kMax ? __builtin_elementwise_maximum(v, shared[i]) : v + shared[i];
  }
  return v;
}

struct Args {
  const void* x;
  const void* r;
  void* s;
  const void* w;
  void* y;
  float* scales;
  long long x_stride, r_stride, s_stride, y_stride;
  int w_dtype, rows, width, group, e5m2;
  float eps;
};

// grid: rows / (threads / kTpr), block: 256 threads, or kTpr where that is more.
// Thread t of a row holds its vectors t, t + kTpr, ..; kC of them.
template <int kDtype, bool kEight, int kTpr, int kC, bool kVec>
__global__ __launch_bounds__(kTpr < 256 ? 256 : kTpr) void rmsnorm_kernel(const Args a) {
  using S = Storage<kDtype>;
  constexpr int N = S::N;
  __shared__ float shared[kTpr / kWave];
  constexpr int kRows = kTpr < 256 ? 256 / kTpr : 1;
  const int t = threadIdx.x % kTpr;
  const long long row = linear_block() * kRows + threadIdx.x / kTpr;
  if (row >= a.rows) return;  // whole waves, and whole workgroups where kTpr > kWave
  const int width = a.width;
  float v[kC][N], w[kC][N];
  int col[kC];
  bool ok[kC];
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    col[c] = (c * kTpr + t) * N;
    ok[c] = col[c] < width;
    const int at = ok[c] ? col[c] : 0;
    load_row<kDtype, kVec>(a.x, row * a.x_stride, at, width, v[c]);
  }
  if (a.r) {
    float r[kC][N];
#pragma unroll
    for (int c = 0; c < kC; ++c) load_row<kDtype, kVec>(a.r, row * a.r_stride, ok[c] ? col[c] : 0, width, r[c]);
#pragma unroll
    for (int c = 0; c < kC; ++c) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[c][j] = S::one(S::round(v[c][j] + r[c][j]));
      if (ok[c]) store_row<kDtype, kVec>(a.s, row * a.s_stride, col[c], width, v[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const int at = ok[c] ? col[c] : 0;
    if (!a.w) {
#pragma unroll
      for (int j = 0; j < N; ++j) w[c][j] = 1.f;
    } else if (a.w_dtype == kDtype) {
      load_row<kDtype, kVec>(a.w, 0, at, width, w[c]);
    } else {  // fp32 weights of 16-bit rows
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if constexpr (kVec) {
          if (j % 4 == 0) {
            const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(a.w) + at + j);
            w[c][j] = f.x, w[c][j + 1] = f.y, w[c][j + 2] = f.z, w[c][j + 3] = f.w;
          }
        } else {
          w[c][j] = at + j < width ? static_cast<const float*>(a.w)[at + j] : 0.f;
        }
      }
    }
  }
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < kC; ++c)
    if (ok[c])
#pragma unroll
      for (int j = 0; j < N; ++j) q = fmaf(v[c][j], v[c][j], q);
  const float rstd = 1.f / sqrtf(row_reduce<kTpr, false>(q, shared) / (float)width + a.eps);
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int j = 0; j < N; ++j) v[c][j] = v[c][j] * rstd * w[c][j];
  if constexpr (!kEight) {
#pragma unroll
    for (int c = 0; c < kC; ++c)
      if (ok[c]) store_row<kDtype, kVec>(a.y, row * a.y_stride, col[c], width, v[c]);
    return;
  }
  const float largest = a.e5m2 ? 57344.f : 448.f;
  const int group = a.group;
  float top[kC];
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    top[c] = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) top[c] = __builtin_elementwise_maximum(top[c], ok[c] ? fabsf(v[c][j]) : 0.f);
  }
  if (group == 0) {
#pragma unroll
    for (int c = 1; c < kC; ++c) top[0] = __builtin_elementwise_maximum(top[0], top[c]);
    top[0] = row_reduce<kTpr, true>(top[0], shared);
#pragma unroll
    for (int c = 1; c < kC; ++c) top[c] = top[0];
  } else {  // group / N neighbouring lanes hold a group
    for (int off = 1; off < group / N; off <<= 1)
#pragma unroll
      for (int c = 0; c < kC; ++c) top[c] = __builtin_elementwise_maximum(top[c], __shfl_xor(top[c], off, kWave));
  }
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    // never below the smallest normal number: a scale that underflows would divide by zero
    const float scale = top[c] == 0.f ? 1.f : __builtin_elementwise_maximum(top[c] / largest, 1.17549435e-38f);
    uint32_t packed[N / 4];
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float f0 = v[c][j] / scale, f1 = v[c][j + 1] / scale, f2 = v[c][j + 2] / scale, f3 = v[c][j + 3] / scale;
      int p = 0;
      if (a.e5m2) {
        p = __builtin_amdgcn_cvt_pk_bf8_f32(f0, f1, p, false);
        p = __builtin_amdgcn_cvt_pk_bf8_f32(f2, f3, p, true);
      } else {
        p = __builtin_amdgcn_cvt_pk_fp8_f32(f0, f1, p, false);
        p = __builtin_amdgcn_cvt_pk_fp8_f32(f2, f3, p, true);
      }
      packed[j / 4] = (uint32_t)p;
    }
    if (!ok[c]) continue;
    uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.y_stride + col[c];
    if constexpr (kVec) {
      if constexpr (N == 8) *reinterpret_cast<uint2*>(y) = make_uint2(packed[0], packed[1]);
      else *reinterpret_cast<uint32_t*>(y) = packed[0];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (col[c] + j < width) y[j] = (uint8_t)(packed[j / 4] >> (8 * (j % 4)));
    }
    if (group == 0) {
      if (c == 0 && t == 0) a.scales[row] = scale;
    } else if (col[c] % group == 0) {
      a.scales[row * (width / group) + col[c] / group] = scale;
    }
  }
}

template <int kDtype, bool kEight>
int launch(const Args& a, bool vec, hipStream_t stream) {
  constexpr int N = Storage<kDtype>::N;
  const int vectors = (a.width + N - 1) / N;
#define MUSC_RMS(TPR, C, VEC)                                                                                       \
  hipLaunchKernelGGL((rmsnorm_kernel<kDtype, kEight, TPR, C, VEC>),                                                 \
                     linear_grid(((long long)a.rows + (TPR < 256 ? 256 / TPR : 1) - 1) / (TPR < 256 ? 256 / TPR : 1)), \
                     dim3(TPR < 256 ? 256 : TPR), 0, stream, a)
#define MUSC_RMS_C(TPR)                                                                                             \
  if (!vec) MUSC_RMS(TPR, 4, false);                                                                                \
  else if (vectors <= TPR) MUSC_RMS(TPR, 1, true);                                                                  \
  else if (vectors <= 2 * TPR) MUSC_RMS(TPR, 2, true);                                                              \
  else MUSC_RMS(TPR, 4, true)
  if (vectors <= 4 * 64) {
    MUSC_RMS_C(64);
  } else if (vectors <= 4 * 256) {
    MUSC_RMS_C(256);
  } else {
    MUSC_RMS_C(1024);
  }
#undef MUSC_RMS_C
#undef MUSC_RMS
  return check_launch();
}

}  // namespace rms
}  // namespace musc

using namespace musc;

namespace {

int rmsnorm(rms::Args a, int dtype, bool eight, hipStream_t stream) {
  if (!a.x || !a.y || a.rows < 0 || a.width < 1 || !(a.eps >= 0.f)) return MUSC_ERR_INVALID_ARG;
  if (dtype != MUSC_DTYPE_F32 && dtype != MUSC_DTYPE_F16 && dtype != MUSC_DTYPE_BF16) return MUSC_ERR_INVALID_ARG;
  if (a.w && a.w_dtype != dtype && a.w_dtype != MUSC_DTYPE_F32) return MUSC_ERR_INVALID_ARG;
  if (a.r && !a.s) return MUSC_ERR_INVALID_ARG;
  if (a.rows > 1 && (a.x_stride < a.width || a.y_stride < a.width ||
                     (a.r && (a.r_stride < a.width || a.s_stride < a.width))))
    return MUSC_ERR_INVALID_ARG;
  const int n = dtype == MUSC_DTYPE_F32 ? 4 : 8;
  if (eight) {
    if (!a.scales) return MUSC_ERR_INVALID_ARG;
    if (a.group < 0) return MUSC_ERR_INVALID_ARG;
    if (a.group && a.group != 32 && a.group != 64 && a.group != 128 && a.group != 256) return MUSC_ERR_UNSUPPORTED;
    if (a.group && a.width % a.group) return MUSC_ERR_INVALID_ARG;
  }
  if (a.width > rms::kMaxChunks * 1024 * n) return MUSC_ERR_UNSUPPORTED;
  if (a.rows == 0) return MUSC_OK;
  const uintptr_t wide = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.r) |
                         reinterpret_cast<uintptr_t>(a.s) | reinterpret_cast<uintptr_t>(a.w) |
                         (eight ? 0 : reinterpret_cast<uintptr_t>(a.y));
  const uintptr_t elem = dtype == MUSC_DTYPE_F32 ? 3 : 1;
  if ((wide & elem) || (a.w && a.w_dtype == MUSC_DTYPE_F32 && (reinterpret_cast<uintptr_t>(a.w) & 3)) ||
      (eight && (reinterpret_cast<uintptr_t>(a.scales) & 3)))
    return MUSC_ERR_INVALID_ARG;
  // 16-byte loads and stores where every row starts on such a boundary
  const long long strides = a.x_stride | a.y_stride | (a.r ? a.r_stride | a.s_stride : 0);
  const bool vec = wide % 16 == 0 && (!eight || reinterpret_cast<uintptr_t>(a.y) % 8 == 0) && a.width % n == 0 &&
                   (a.rows == 1 || strides % n == 0);
  if (dtype == MUSC_DTYPE_F32)
    return eight ? rms::launch<MUSC_DTYPE_F32, true>(a, vec, stream) : rms::launch<MUSC_DTYPE_F32, false>(a, vec, stream);
  if (dtype == MUSC_DTYPE_F16)
    return eight ? rms::launch<MUSC_DTYPE_F16, true>(a, vec, stream) : rms::launch<MUSC_DTYPE_F16, false>(a, vec, stream);
  return eight ? rms::launch<MUSC_DTYPE_BF16, true>(a, vec, stream) : rms::launch<MUSC_DTYPE_BF16, false>(a, vec, stream);
}

}  // namespace

extern "C" int musc_rmsnorm_rows(const void* x, long long x_stride, const void* residual, long long residual_stride,
                                 void* sum_out, const void* weight, int weight_dtype, int dtype, int rows, int width,
                                 float eps, void* y, hipStream_t stream) {
  return rmsnorm(rms::Args{x, residual, sum_out, weight, y, nullptr, x_stride, residual_stride, width, width,
                           weight_dtype, rows, width, 0, 0, eps},
                 dtype, false, stream);
}

extern "C" int musc_rmsnorm_rows_8bit(const void* x, long long x_stride, const void* residual,
                                      long long residual_stride, void* sum_out, const void* weight, int weight_dtype,
                                      int dtype, int rows, int width, float eps, int format, int group, void* y,
                                      float* scales, hipStream_t stream) {
  if (format != MUSC_FP8_E4M3 && format != MUSC_FP8_E5M2) return MUSC_ERR_INVALID_ARG;
  return rmsnorm(rms::Args{x, residual, sum_out, weight, y, scales, x_stride, residual_stride, width, width,
                           weight_dtype, rows, width, group, format == MUSC_FP8_E5M2, eps},
                 dtype, true, stream);
}
