// act8_wgrad.hip — the weight gradient of a linear layer from its input's
// 8-bit checkpoint (gfx950):
//
//   dW[n, k] = sum over m of dy[m, n] * x'[m, k]      db[n] = sum of dy[m, n]
//
// x' is never written out: codes are widened to bf16 (fp16 for fp16
// gradients), which is exact, on their way into LDS.  Both operands are
// stored with the summed index m as their slow one, so their tiles go to LDS
// as they come and the matrix instructions' fragments are read across them
// with transposing LDS reads.
//
// fp32 gradients are split into three bf16 numbers each (8 bits of the
// significand at a time, exact together), which become three row blocks of
// one product with three times as many rows: the sums stay as good as fp32's
// own products.
#include <hip/hip_runtime.h>

#include "act8_codes.h"

namespace baguanet {
namespace {

typedef float float16v __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v* LdsShort4;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef fp16 fp16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;     // four waves, two by two
constexpr int kTN = 128, kTK = 128;  // of dW for a workgroup
constexpr int kTM = 32;           // rows summed for each tile in LDS

template <typename T>
__device__ inline float16v mfma(short8v a, short8v b, float16v c);
template <>
__device__ inline float16v mfma<bf16>(short8v a, short8v b, float16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
      __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
      0);
}
template <>
__device__ inline float16v mfma<fp16>(short8v a, short8v b, float16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(
      __builtin_bit_cast(fp16x8, a), __builtin_bit_cast(fp16x8, b), c, 0, 0,
      0);
}

// A tile in LDS: kTM rows of `width` 16-bit values.  Four rows that one
// transposing read takes together lie on different banks: the 64-byte
// blocks of a row are exchanged by the row's last two bits.
template <int kWidth>
__device__ inline int lds_at(int row, int col) {
  const int block = (col >> 5) ^ (row & 3);
  return row * kWidth + (block << 5) + (col & 31);
}

// 8 rows of one column for each lane: lanes 0..31 take the columns col0..+31
// of rows row0..+7, the others those of rows row0 + 8..+15.
template <int kWidth>
__device__ inline short8v read_fragment(const short* tile, int row0,
                                        int col0) {
  const int lane = threadIdx.x % kWave;
  const int row = row0 + (lane / 32) * 8 + (lane % 16) / 4;
  const int col = col0 + (lane / 16 % 2) * 16 + (lane % 4) * 4;
  const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (LdsShort4)(tile + lds_at<kWidth>(row, col)));
  const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (LdsShort4)(tile + lds_at<kWidth>(row + 4, col)));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// One product's shape: `planes` row blocks of `m` rows in dy, one in x'.
struct Product {
  const void* dy;
  int64_t dstride, plane;  // elements between rows and between planes
  int planes, slices;
  int64_t slice_rows;      // of the planes * m rows, a multiple of kTM
  float* partial;          // [slices, n, k] where slices > 1
};

// T: bf16 or fp16, the operands' type.  O: the type of dW.
template <typename T, typename O>
__global__ __launch_bounds__(kThreads) void act8_wgrad_kernel(Act8Wgrad a,
                                                              Product p) {
  __shared__ __attribute__((aligned(16))) short sy[kTM * kTN];
  __shared__ __attribute__((aligned(16))) short sx[kTM * kTK];
  const int64_t n0 = (int64_t)blockIdx.x * kTN, k0 = (int64_t)blockIdx.y * kTK;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int wn = (wave / 2) * (kTN / 2), wk = (wave % 2) * (kTK / 2);
  const int64_t total = p.planes * a.m;
  const int64_t begin = blockIdx.z * p.slice_rows;
  const int64_t end =
      begin + p.slice_rows < total ? begin + p.slice_rows : total;

  float16v acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++) acc[i][j] = 0.f;

  for (int64_t m0 = begin; m0 < end; m0 += kTM) {
    // dy: 16 lanes to a row of 128, two rows for each lane
#pragma unroll
    for (int i = 0; i < kTM * kTN / (kThreads * 8); i++) {
      const int at = i * kThreads + threadIdx.x;
      const int r = at / (kTN / 8), c = at % (kTN / 8) * 8;
      typename RowVec<T>::type v = (T)0.f;
      const int64_t row = m0 + r, left = a.n - n0 - c;
      if (row < end && left > 0) {
        const int64_t pl = row / a.m, rr = row % a.m;
        v = raw_upto((const T*)p.dy + pl * p.plane + rr * p.dstride + n0 + c,
                     left < 8 ? (int)left : 8);
      }
      *(typename RowVec<T>::type*)&sy[lds_at<kTN>(r, c)] = v;
    }
    // x': 16 lanes to a row too
#pragma unroll
    for (int i = 0; i < kTM * kTK / (kThreads * 8); i++) {
      const int at = i * kThreads + threadIdx.x;
      const int r = at / (kTK / 8), c = at % (kTK / 8) * 8;
      float8 v = 0.f;
      const int64_t row = m0 + r;
      if (row < end && k0 + c < a.pitch) {
        const int64_t at8 = row % a.m * a.pitch + k0 + c;
        v = decode8(*(const uint2*)(a.codes + at8),
                    a.exps[at8 / kAct8Group] - 127);
      }
      *(typename RowVec<T>::type*)&sx[lds_at<kTK>(r, c)] =
          __builtin_convertvector(v, typename RowVec<T>::type);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kTM; s += 16) {
      short8v fy[2], fx[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        fy[i] = read_fragment<kTN>(sy, s, wn + i * 32);
        fx[i] = read_fragment<kTK>(sx, s, wk + i * 32);
      }
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
          acc[i][j] = mfma<T>(fy[i], fx[j], acc[i][j]);
    }
    __syncthreads();
  }

  // element i of a lane: row 8 * (i / 4) + 4 * (lane / 32) + i % 4 of the
  // 32 by 32 block, column lane % 32
#pragma unroll
  for (int bi = 0; bi < 2; bi++)
#pragma unroll
    for (int bj = 0; bj < 2; bj++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int64_t n = n0 + wn + bi * 32 + 8 * (i / 4) + 4 * (lane / 32) +
                          i % 4;
        const int64_t k = k0 + wk + bj * 32 + lane % 32;
        if (n >= a.n || k >= a.k) continue;
        if (p.slices > 1)
          p.partial[(blockIdx.z * a.n + n) * a.k + k] = acc[bi][bj][i];
        else
          ((O*)a.dw)[n * a.k + k] = (O)acc[bi][bj][i];
      }
}

// dW from the slices' sums, in their order.
template <typename O>
__global__ __launch_bounds__(kThreads) void wgrad_join_kernel(
    const float* partial, int slices, int64_t count, O* dw) {
  for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kVec;
       i < count; i += (int64_t)gridDim.x * kThreads * kVec) {
    const int m = (int)(count - i < kVec ? count - i : kVec);
    float8 v = 0.f;
    for (int s = 0; s < slices; s++)
      v += load_upto(partial + s * count + i, m);
    store_upto(dw + i, v, m);
  }
}

// An fp32 gradient as three bf16 planes of 8 bits of its significand each,
// cut off rather than rounded so that no plane can pass the largest number:
// their sum is the value itself, up to the last bits of numbers near the
// smallest.  A NaN or an infinity is whole in the first plane.
__global__ __launch_bounds__(kThreads) void split_kernel(
    const float* dy, int64_t dstride, int64_t m, int64_t n, bf16* planes,
    int64_t pitch) {
  const int64_t cols = (n + kVec - 1) / kVec;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < m * cols;
       i += (int64_t)gridDim.x * kThreads) {
    const int64_t r = i / cols, c = i % cols * kVec;
    float8 v = load_upto(dy + r * dstride + c, (int)(n - c < kVec ? n - c : kVec));
#pragma unroll
    for (int p = 0; p < 3; p++) {
      float8 h;
#pragma unroll
      for (int j = 0; j < kVec; j++) {
        h[j] = is_finite(v[j])
                   ? __uint_as_float(__float_as_uint(v[j]) & 0xffff0000u)
                   : v[j];
        v[j] = is_finite(v[j]) ? v[j] - h[j] : 0.f;
      }
      store8(planes + (p * m + r) * pitch + c, h);
    }
  }
}

// Column sums of dy: strips of rows first, then the strips in their order.
constexpr int kSumCols = 64, kSumLanes = 16;

template <typename T>
__global__ __launch_bounds__(kSumCols* kSumLanes) void column_strip_kernel(
    const T* dy, int64_t dstride, int64_t m, int64_t n, int64_t strip_rows,
    float* strips) {
  __shared__ float part[kSumLanes][kSumCols];
  const int c = threadIdx.x % kSumCols, s = threadIdx.x / kSumCols;
  const int64_t col = (int64_t)blockIdx.x * kSumCols + c;
  const int64_t begin = blockIdx.y * strip_rows;
  const int64_t end = begin + strip_rows < m ? begin + strip_rows : m;
  float sum = 0.f;
  if (col < n) {
#pragma unroll 8
    for (int64_t r = begin + s; r < end; r += kSumLanes)
      sum += (float)dy[r * dstride + col];
  }
  part[s][c] = sum;
  __syncthreads();
  if (s || col >= n) return;
  for (int i = 1; i < kSumLanes; i++) sum += part[i][c];
  strips[blockIdx.y * n + col] = sum;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void column_join_kernel(
    const float* strips, int count, int64_t n, T* db) {
  const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (col >= n) return;
  float sum = 0.f;
#pragma unroll 8
  for (int i = 0; i < count; i++) sum += strips[i * n + col];
  db[col] = (T)sum;
}

struct Plan {
  int planes, slices;
  int64_t slice_rows, pitch, strip_rows, strips;
  size_t plane_bytes, partial_bytes, strip_bytes;
};

size_t round256(size_t b) { return (b + 255) & ~size_t(255); }

Plan plan_of(const Act8Wgrad& a) {
  Plan p = {};
  p.planes = a.type == ElemType::kF32 ? 3 : 1;
  p.pitch = (a.n + 7) / 8 * 8;
  if (p.planes > 1)
    p.plane_bytes = round256((size_t)3 * a.m * p.pitch * sizeof(bf16));
  // Few tiles leave compute units idle: the rows are then cut in slices.
  const int64_t tiles =
      ((a.n + kTN - 1) / kTN) * ((a.k + kTK - 1) / kTK);
  const int64_t rows = p.planes * a.m;
  int64_t slices = 512 / tiles, most = rows / 256;
  if (slices > most) slices = most;
  if (slices < 1) slices = 1;
  p.slice_rows = ((rows + slices - 1) / slices + kTM - 1) / kTM * kTM;
  p.slices = (int)((rows + p.slice_rows - 1) / p.slice_rows);
  if (p.slices > 1)
    p.partial_bytes = round256((size_t)p.slices * a.n * a.k * sizeof(float));
  if (a.db) {
    p.strip_rows = a.m > 256 * 1024 ? (a.m + 1023) / 1024 : 256;
    p.strips = (a.m + p.strip_rows - 1) / p.strip_rows;
    p.strip_bytes = round256((size_t)p.strips * a.n * sizeof(float));
  }
  return p;
}

}  // namespace

size_t act8_wgrad_workspace(const Act8Wgrad& a) {
  if (a.m == 0 || a.n == 0 || a.k == 0) return 0;
  const Plan p = plan_of(a);
  return p.plane_bytes + p.partial_bytes + p.strip_bytes;
}

hipError_t act8_wgrad(const Act8Wgrad& a, hipStream_t stream) {
  if (a.m == 0 || a.n == 0 || a.k == 0) return hipSuccess;
  const Plan plan = plan_of(a);
  char* ws = (char*)a.workspace;
  float* strips = (float*)(ws + plan.plane_bytes + plan.partial_bytes);
  Product p = {a.dy,        a.dstride,        0,
               plan.planes, plan.slices,      plan.slice_rows,
               (float*)(ws + plan.plane_bytes)};
  const dim3 grid((uint32_t)((a.n + kTN - 1) / kTN),
                  (uint32_t)((a.k + kTK - 1) / kTK), (uint32_t)plan.slices);
  if (grid.y > 65535 || (int64_t)grid.x * grid.y * grid.z >= (1 << 24))
    return hipErrorInvalidValue;
  if (a.type == ElemType::kF32) {
    bf16* planes = (bf16*)ws;
    const int64_t items = a.m * ((a.n + 7) / 8);
    const int64_t want = (items + kThreads - 1) / kThreads;
    launch(split_kernel, (uint32_t)(want < 4096 ? want : 4096), kThreads, stream, (const float*)a.dy, a.dstride, a.m, a.n, planes,
                             plan.pitch);
    p.dy = planes;
    p.dstride = plan.pitch;
    p.plane = a.m * plan.pitch;
    launch(act8_wgrad_kernel<bf16, float>, grid, kThreads, stream, a, p);
  } else if (a.type == ElemType::kBF16) {
    launch(act8_wgrad_kernel<bf16, bf16>, grid, kThreads, stream, a, p);
  } else {
    launch(act8_wgrad_kernel<fp16, fp16>, grid, kThreads, stream, a, p);
  }
  with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (plan.slices > 1) {
      const int64_t count = a.n * a.k;
      const int64_t want = (count + kThreads * kVec - 1) / (kThreads * kVec);
      launch(wgrad_join_kernel<T>, (uint32_t)(want < 4096 ? want : 4096), kThreads, stream, 
              p.partial, plan.slices, count, (T*)a.dw);
    }
    if (a.db) {
      const dim3 sums((uint32_t)((a.n + kSumCols - 1) / kSumCols),
                      (uint32_t)plan.strips);
      launch(column_strip_kernel<T>, sums, kSumCols * kSumLanes, stream, 
          (const T*)a.dy, a.dstride, a.m, a.n, plan.strip_rows,
          strips);
      launch(column_join_kernel<T>, (uint32_t)((a.n + kThreads - 1) / kThreads), kThreads, stream, strips, (int)plan.strips, a.n, (T*)a.db);
    }
  });
  return hipGetLastError();
}

}  // namespace baguanet
