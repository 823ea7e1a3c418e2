// device_types.h — element types, row vectors and reductions shared by the
// training-step kernels (gfx950, 64-wide wavefronts).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "train_kernels.h"

namespace baguanet {

using bf16 = __bf16;
using fp16 = _Float16;

constexpr int kWave = 64;
constexpr int kVec = 8;  // elements of a row that one lane moves at a time

// 8 elements as loaded and as computed with.  The memory types carry only
// their element's alignment: gfx950 reads and writes 16 bytes at any
// address, so rows of odd length and sliced tensors take the same wide
// accesses as aligned ones.
template <typename T>
struct RowVec {
  typedef T type __attribute__((ext_vector_type(8)));
  typedef T unaligned __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
typedef float float8 __attribute__((ext_vector_type(8)));

template <typename T>
__device__ inline float8 load8(const T* p) {
  typename RowVec<T>::type v = *(const typename RowVec<T>::unaligned*)p;
  return __builtin_convertvector(v, float8);
}

template <typename T>
__device__ inline void store8(T* p, float8 v) {
  *(typename RowVec<T>::unaligned*)p =
      __builtin_convertvector(v, typename RowVec<T>::type);
}

// The first n (1..8) elements; the rest read as zero.
template <typename T>
__device__ inline float8 load_upto(const T* p, int n) {
  if (n >= kVec) return load8(p);
  float8 v = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; i++)
    if (i < n) v[i] = (float)p[i];
  return v;
}

template <typename T>
__device__ inline void store_upto(T* p, float8 v, int n) {
  if (n >= kVec) {
    store8(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; i++)
    if (i < n) p[i] = (T)v[i];
}

// The same without the conversion, for loads that run ahead of their use.
template <typename T>
__device__ inline typename RowVec<T>::type raw_upto(const T* p, int n) {
  if (n >= kVec) return *(const typename RowVec<T>::unaligned*)p;
  typename RowVec<T>::type v = (T)0.f;
#pragma unroll
  for (int i = 0; i < kVec; i++)
    if (i < n) v[i] = p[i];
  return v;
}

template <typename V>
__device__ inline float8 widen(V v) {
  return __builtin_convertvector(v, float8);
}

// A vector of weights held in fp32 or in T.
template <typename T>
__device__ inline float8 weight_upto(const void* p, bool f32, int64_t i,
                                     int n) {
  return f32 ? load_upto((const float*)p + i, n) : load_upto((const T*)p + i, n);
}

template <typename T>
__device__ inline void put_weight_upto(void* p, bool f32, int64_t i, float8 v,
                                       int n) {
  if (f32)
    store_upto((float*)p + i, v, n);
  else
    store_upto((T*)p + i, v, n);
}

__device__ inline float sum8(float8 v) {
  return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}

// Launches a kernel without dynamic LDS.
template <typename... P>
inline void launch(void (*kernel)(P...), dim3 grid, int block,
                   hipStream_t stream, std::common_type_t<P>... args) {
  hipLaunchKernelGGL(kernel, grid, dim3(block), 0, stream, args...);
}

// Calls f with a null T* of the element type that `t` names.
template <typename F>
inline void with_type(ElemType t, F&& f) {
  if (t == ElemType::kF32)
    f((float*)nullptr);
  else if (t == ElemType::kBF16)
    f((bf16*)nullptr);
  else
    f((fp16*)nullptr);
}

__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int o = kWave / 2; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

}  // namespace baguanet
