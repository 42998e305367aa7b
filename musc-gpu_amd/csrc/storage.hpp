// 16-byte vectors of the storage types (fp32, fp16, bf16) as fp32 values in registers.
#pragma once

#include "common.hpp"

namespace musc {

template <int kDtype>
struct Storage;

template <>
struct Storage<MUSC_DTYPE_F32> {
  static constexpr int N = 4;
  typedef float T;
  static __device__ __forceinline__ float one(T x) { return x; }
  static __device__ __forceinline__ T round(float x) { return x; }
  static __device__ __forceinline__ void load(const T* p, float (&v)[N]) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  }
  static __device__ __forceinline__ void store(T* p, const float (&v)[N]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};

template <typename Half>
struct Storage16 {
  static constexpr int N = 8;
  typedef Half T;
  typedef Half Vec __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float one(T x) { return (float)x; }
  static __device__ __forceinline__ T round(float x) { return (T)x; }  // to nearest, ties to even
  static __device__ __forceinline__ void load(const T* p, float (&v)[N]) {
    const Vec x = *reinterpret_cast<const Vec*>(p);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (float)x[j];
  }
  static __device__ __forceinline__ void store(T* p, const float (&v)[N]) {
    Vec x;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = (T)v[j];
    *reinterpret_cast<Vec*>(p) = x;
  }
};

template <>
struct Storage<MUSC_DTYPE_F16> : Storage16<_Float16> {};
template <>
struct Storage<MUSC_DTYPE_BF16> : Storage16<__bf16> {};

}  // namespace musc
