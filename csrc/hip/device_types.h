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

__device__ inline float sum8(float8 v) {
  return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}

// The columns of a row that one lane takes: 8 from `col` on.  The lane at the
// row's end moves back so that its 8 lie inside the row, and shares `dup`
// columns with the lane before it: both compute the same there and write the
// same, and only sums over the row leave the shared ones out.  So no access
// needs a count, which would cost registers and branches at each.  A lane
// with dup == 8 has nothing of its own.  kTiny: rows of fewer than 8 columns,
// which one lane takes element by element.
template <bool kTiny>
struct Cols {
  int col, dup, count;
  __device__ inline Cols() {}
  __device__ inline Cols(int at, int dim) {
    count = kTiny ? dim : kVec;
    col = kTiny ? 0 : at + kVec <= dim ? at : dim - kVec;
    dup = kTiny ? (at ? kVec : 0) : at >= dim ? kVec : at - col;
  }
  __device__ inline bool own() const { return dup < kVec; }
  template <typename T>
  __device__ inline typename RowVec<T>::type raw(const T* row) const {
    if constexpr (kTiny) return raw_upto(row, count);
    return *(const typename RowVec<T>::unaligned*)(row + col);
  }
  template <typename T>
  __device__ inline float8 load(const T* row) const {
    return widen(raw(row));
  }
  // A vector of weights held in fp32 or in T, `at` elements into p.
  template <typename T>
  __device__ inline float8 weight(const void* p, bool f32, int64_t at) const {
    return f32 ? load((const float*)p + at) : load((const T*)p + at);
  }
  template <typename T>
  __device__ inline void store(T* row, float8 v) const {
    if constexpr (kTiny)
      store_upto(row, v, count);
    else
      store8(row + col, v);
  }
  template <typename T>
  __device__ inline void put_weight(void* p, bool f32, int64_t at,
                                    float8 v) const {
    if (f32)
      store((float*)p + at, v);
    else
      store((T*)p + at, v);
  }
  // row += v, or row = v, on the lane's own columns.
  __device__ inline void accumulate(float* row, float8 v, bool first) const {
    if (!kTiny && dup == 0) {
      if (!first) v += load8(row + col);
      store8(row + col, v);
      return;
    }
#pragma unroll
    for (int i = 0; i < kVec; i++)
      if (i >= dup && i < count)
        row[col + i] = first ? v[i] : row[col + i] + v[i];
  }
  // The sum of the lane's own columns.
  __device__ inline float sum(float8 v) const {
    if (dup) {
#pragma unroll
      for (int i = 0; i < kVec; i++) v[i] = i < dup ? 0.f : v[i];
    }
    return sum8(v);
  }
};

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
