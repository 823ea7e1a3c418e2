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
//
// Bound by the matrix cores, fed from LDS: 16384 x 8192 x 4096 bf16 takes 850
// to 930 us (1.2 to 1.3 PFLOP/s, as the clock allows), where the library's
// product of the uncompressed operands takes 980; 4096^3 takes 110 (1.25
// PFLOP/s; 117).  With few rows a tile's start and its way out weigh most: 256
// x 4096 x 25088 fp32 takes 212 to 222 us for 0.16 TFLOP and 411 MB of dW.
#include <hip/hip_runtime.h>

#include <cmath>

#include "act8_codes.h"

namespace baguanet {
namespace {

typedef float float16v __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v* LdsShort4;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef fp16 fp16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;  // four waves, two by two
constexpr int kTM = 64;         // rows summed for each tile in LDS
constexpr int kSteps = kTM / 16;  // of the matrix instructions for a tile
constexpr int kUnits = 256;       // compute units

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

// Two codes' values, exact in bf16 and fp16.
template <typename T>
__device__ inline uint32_t widen2(uint32_t codes, float scale, bool high);
template <>
__device__ inline uint32_t widen2<bf16>(uint32_t codes, float scale,
                                        bool high) {
  return __builtin_bit_cast(
      uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale,
                                                                 true)
                     : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale,
                                                                 false));
}
template <>
__device__ inline uint32_t widen2<fp16>(uint32_t codes, float scale,
                                        bool high) {
  return __builtin_bit_cast(
      uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale,
                                                                true)
                     : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale,
                                                                false));
}

// A tile in LDS: kTM rows of kWidth 16-bit values.  Four rows that one
// transposing read takes together lie on different banks: the 64-byte
// blocks of a row are exchanged by the row's last two bits.
template <int kWidth>
__device__ inline int lds_at(int row, int col) {
  return row * kWidth + (((col >> 5) ^ (row & 3)) << 5) + (col & 31);
}

// 8 rows of one column for each lane, from `p`, the lane's place for the
// fragment's first row: lanes 0..31 take 32 columns of the rows 0..7, the
// others those of the rows 8..15.
template <int kWidth>
__device__ inline short8v read_fragment(const short* p) {
  const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4)p);
  const short4v hi =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4)(p + 4 * kWidth));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Memory that is read a tile of rows at a time.  Reads behind a tile's bytes
// give zeros (the hardware checks them, with the scalar offset counted in,
// against the descriptor's size, 4 bytes at a time), so the last tile needs no
// conditions; those behind a row's end give the next row's values, which only
// reach columns that are not written.
struct Stream {
  const char* base;
  int64_t tile;    // bytes from one tile to the next
  int full, tail;  // bytes of a tile, and of the last
};

__device__ inline __amdgpu_buffer_rsrc_t descriptor(const char* p, int size) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, size, 0x00027000);
}

// A part of dW: its rows and columns from the first up to the end.
struct Part {
  int64_t n0, n1, k0, k1;
  int ntiles, ktiles;
};

// One product, for a part of dW: dy in tiles of kTM rows, `tiles` in all; x'
// starts again after `xtiles` of them (the planes of an fp32 gradient).
struct Product {
  Stream dy, codes, exps;
  int dpitch, cpitch;      // bytes between rows of dy and of codes
  int tiles, xtiles;
  int slices, slice_tiles;
  Part part;
  int64_t k;            // columns of dW
  void* dw;
  void* db;             // null: not wanted, or not from this part
  float* partial;       // [slices, rows, columns of the part], slices > 1
  float* bias_partial;  // [slices, rows of the part], slices > 1
  // kOdd: dy's very last value where n is odd, its column, and its row of x':
  // reads count whole 4 bytes, so the tiles come without it
  const short* odd;
  int64_t odd_col;
  const uint8_t *odd_codes, *odd_exps;
};

// The workgroup's tile of dW.  Workgroups go to the 8 XCDs in turn; each XCD
// takes a run of tiles, in strips 8 tiles high, so that those at work
// together read the same parts of dy and x' through its L2.
__device__ inline void pick_tile(const Part& p, int& tn, int& tk) {
  const int total = p.ntiles * p.ktiles, id = blockIdx.x;
  const int xcd = id % 8, each = total / 8, more = total % 8;
  const int at = xcd * each + (xcd < more ? xcd : more) + id / 8;
  const int strip = at / (8 * p.ktiles), in = at % (8 * p.ktiles);
  const int high = p.ntiles - strip * 8 < 8 ? p.ntiles - strip * 8 : 8;
  tn = strip * 8 + in % high;
  tk = in / high;
}

// The order of a step's instructions: the next step's fragments are read
// between the first half of the matrix instructions, so that they are there
// when that step begins, and the next tile is written and the one after
// loaded between the others.  Left to itself the compiler gathers the loads
// at the tile's end, next to the waits for them.
template <int FN, int FK>
__device__ inline void order_step(bool staging) {
  constexpr int kMfma = 0x8, kScalar = 0x4, kVmem = 0x20;
  constexpr int kRead = 0x100, kWrite = 0x200;
  constexpr int kCount = FN * FK, kHalf = kCount / 2;
  constexpr int kReads = 2 * (FN + FK) / kHalf;
#pragma unroll
  for (int i = 0; i < kHalf; i++) {
    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, kReads, 0);
  }
#pragma unroll
  for (int i = kHalf; i < kCount; i++) {
    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    if (!staging) {
      __builtin_amdgcn_sched_group_barrier(kScalar, 32 / kHalf, 0);
      continue;
    }
    __builtin_amdgcn_sched_group_barrier(kWrite, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kVmem, 2, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// T: bf16 or fp16, the operands' type.  O: the type of dW.  A wave computes
// FN by FK blocks of 32 by 32.  kOdd: dy is read as it is and n is odd.
//
// Two tiles are in LDS: the matrix instructions of one overlap with the
// writing of the next, whose rows are in registers by then, and with the
// loads of the one after.  A step's fragments are read during the step
// before, across the tiles' border too: the one barrier of a tile stands
// before its last step, when all its fragments have been read and all of the
// next tile is written.
template <typename T, typename O, int FN, int FK, bool kOdd>
__global__ __launch_bounds__(kThreads, FN * FK > 8 ? 1 : 2)
void act8_wgrad_kernel(Product p) {
  constexpr int kTN = 64 * FN, kTK = 64 * FK;
  constexpr int kPassN = kTM * kTN / 8 / kThreads;
  constexpr int kPassK = kTM * kTK / 8 / kThreads;
  constexpr int kRowsN = kTM / kPassN, kRowsK = kTM / kPassK;  // of a pass
  constexpr int kTile = kTM * (kTN + kTK);  // both operands' tiles
  __shared__ __attribute__((aligned(alignof(float8)))) short lds[2 * kTile];
  int tn, tk;
  pick_tile(p.part, tn, tk);
  const int64_t n0 = p.part.n0 + (int64_t)tn * kTN;
  const int64_t k0 = p.part.k0 + (int64_t)tk * kTK;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int wn = (wave / 2) * (kTN / 2), wk = (wave % 2) * (kTK / 2);
  const int t0 = blockIdx.y * p.slice_tiles;
  const int t1 = t0 + p.slice_tiles < p.tiles ? t0 + p.slice_tiles : p.tiles;

  // global: this thread's 8 columns of a row of a pass
  const int ry = threadIdx.x / (kTN / 8), cy = threadIdx.x % (kTN / 8) * 8;
  const int rx = threadIdx.x / (kTK / 8), cx = threadIdx.x % (kTK / 8) * 8;
  const int gy = ry * p.dpitch + (int)(n0 + cy) * 2;
  const int gx = rx * p.cpitch + (int)(k0 + cx);
  // LDS: rows of a pass are kRows apart, a multiple of 4
  const int ly = lds_at<kTN>(ry, cy);
  const int lx = kTM * kTN + lds_at<kTK>(rx, cx);
  // fragments: the lane's place in each, for the tile's first row
  const int fr = (lane / 32) * 8 + (lane % 16) / 4;
  const int fc = (lane / 16 % 2) * 16 + (lane % 4) * 4;
  int fy[FN], fx[FK];
#pragma unroll
  for (int i = 0; i < FN; i++) fy[i] = lds_at<kTN>(fr, wn + i * 32 + fc);
#pragma unroll
  for (int i = 0; i < FK; i++)
    fx[i] = kTM * kTN + lds_at<kTK>(fr, wk + i * 32 + fc);

  typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
  typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
  uint4v hy[kPassN];
  uint2v hx[kPassK];
  uint32_t he[kPassK];
  __amdgpu_buffer_rsrc_t by, bx, be;
  // the descriptors of tile ta, and on to the next; past the end: empty
  int ta = t0, tx = t0 % p.xtiles;
  const char* py = p.dy.base + t0 * p.dy.tile;
  const char* px = p.codes.base + tx * p.codes.tile;
  const char* pe = p.exps.base + tx * p.exps.tile;
  auto aim = [&]() {
    const bool live = ta < t1, last = tx == p.xtiles - 1;
    const int sy = ta == p.tiles - 1 ? p.dy.tail : p.dy.full;
    const int sx = last ? p.codes.tail : p.codes.full;
    const int se = last ? p.exps.tail : p.exps.full;
    by = descriptor(py, live ? sy : 0);
    bx = descriptor(px, live ? sx : 0);
    be = descriptor(pe, live ? se : 0);
    ta++;
    py += p.dy.tile;
    tx = last ? 0 : tx + 1;
    px = last ? p.codes.base : px + p.codes.tile;
    pe = last ? p.exps.base : pe + p.exps.tile;
  };
  auto load_y = [&](int i) {
    hy[i] = __builtin_amdgcn_raw_buffer_load_b128(by, gy,
                                                  i * kRowsN * p.dpitch, 0);
  };
  auto load_x = [&](int i) {
    const int off = i * kRowsK * p.cpitch;
    hx[i] = __builtin_amdgcn_raw_buffer_load_b64(bx, gx, off, 0);
    he[i] = __builtin_amdgcn_raw_buffer_load_b8(be, gx >> 5, off >> 5, 0);
  };
  auto write_y = [&](int buf, int i) {
    *(uint4v*)&lds[buf + ly + i * kRowsN * kTN] = hy[i];
  };
  auto write_x = [&](int buf, int i) {
    const float scale = __uint_as_float(he[i] << 23);
    uint4v v;
    v[0] = widen2<T>(hx[i][0], scale, false);
    v[1] = widen2<T>(hx[i][0], scale, true);
    v[2] = widen2<T>(hx[i][1], scale, false);
    v[3] = widen2<T>(hx[i][1], scale, true);
    *(uint4v*)&lds[buf + lx + i * kRowsK * kTK] = v;
  };

  float16v acc[FN][FK];
#pragma unroll
  for (int i = 0; i < FN; i++)
#pragma unroll
    for (int j = 0; j < FK; j++) acc[i][j] = 0.f;
  short8v ay[2][FN], ax[2][FK];
  auto read_step = [&](int buf, int step, int to) {
#pragma unroll
    for (int i = 0; i < FN; i++)
      ay[to][i] = read_fragment<kTN>(&lds[buf + fy[i] + step * 16 * kTN]);
#pragma unroll
    for (int i = 0; i < FK; i++)
      ax[to][i] = read_fragment<kTK>(&lds[buf + fx[i] + step * 16 * kTK]);
  };

  // A step's share of the rows: those in registers go to `write` (LDS), if
  // that is not negative, and the same of the tile aimed at take their place.
  auto stage = [&](int step, int write, auto&& use_row) {
#pragma unroll
    for (int i = 0; i < kPassN; i++)
      if (i * (kSteps - 1) / kPassN == step) {
        if (write >= 0) {
          write_y(write, i);
          use_row(i);
        }
        load_y(i);
      }
#pragma unroll
    for (int i = 0; i < kPassK; i++)
      if (i * (kSteps - 1) / kPassK == step) {
        if (write >= 0) write_x(write, i);
        load_x(i);
      }
  };

  // The workgroups of the first column of tiles add dy's rows up for db as
  // they pass through their registers: a pass over dy of its own took 52 us
  // where the product takes 920.
  float8 sum = 0.f;
  auto add_row = [&](int i) {
    sum += widen(__builtin_bit_cast(typename RowVec<T>::type, hy[i]));
  };
  aim();
#pragma unroll
  for (int s = 0; s < kSteps - 1; s++) stage(s, -1, add_row);
  aim();
#pragma unroll
  for (int s = 0; s < kSteps - 1; s++) {
    stage(s, 0, add_row);
    __builtin_amdgcn_sched_barrier(0);
  }
  aim();
  __syncthreads();
  read_step(0, 0, 0);

  auto all_tiles = [&](auto with_bias) {
    constexpr bool kBias = decltype(with_bias)::value;
    int cur = 0;  // where in LDS the tile at work begins
    for (int t = t0; t < t1; t++) {
      const int nxt = kTile - cur;
#pragma unroll
      for (int s = 0; s < kSteps; s++) {
        if (s == kSteps - 1) __syncthreads();
        read_step(s == kSteps - 1 ? nxt : cur, (s + 1) % kSteps, (s + 1) % 2);
        // the next tile's rows into LDS, spread over the steps but the last
        if (s < kSteps - 1)
          stage(s, nxt, [&](int i) {
            if (kBias) add_row(i);
          });
        else
          aim();  // the loads of the next tile's steps
#pragma unroll
        for (int i = 0; i < FN; i++)
#pragma unroll
          for (int j = 0; j < FK; j++)
            acc[i][j] = mfma<T>(ay[s % 2][i], ax[s % 2][j], acc[i][j]);
        order_step<FN, FK>(s < kSteps - 1);
      }
      cur = nxt;
    }
  };
  if (p.db && tk == 0)
    all_tiles(std::true_type());
  else
    all_tiles(std::false_type());

  // One more step, with the value that the tiles lack and its row of x' alone.
  const bool odd = kOdd && t1 == p.tiles;
  if (odd && p.odd_col >= n0 && p.odd_col < n0 + kTN) {
    int l = lane;  // opaque, or its comparisons would live through the loop
    asm volatile("" : "+v"(l)::"memory");
    const int row = (int)(p.odd_col - n0) - wn;
    short8v y = 0, x = 0;
#pragma unroll
    for (int j = 0; j < FK; j++) {
      const int64_t c = k0 + wk + j * 32 + l;
      x[0] = 0;
      if (l < 32 && c < p.part.k1)
        x[0] = (short)widen2<T>(
            p.odd_codes[c],
            __uint_as_float((uint32_t)p.odd_exps[c / kAct8Group] << 23), false);
#pragma unroll
      for (int i = 0; i < FN; i++) {
        y[0] = l < 32 && row == i * 32 + l ? *p.odd : (short)0;
        acc[i][j] = mfma<T>(y, x, acc[i][j]);
      }
    }
  }

  // Out through LDS, 32 rows of a wave at a time, so that a lane writes 8
  // neighbours of a row: written straight from where the matrix instructions
  // leave them, a tile of 256 by 256 took about 15 us.  Element i of a lane is
  // that of row 8 * (i / 4) + 4 * (lane / 32) + i % 4 of a 32 by 32 block, and
  // of column lane % 32; the pitch puts rows 4 apart on different banks.
  constexpr int kPitch = FK * 32 + 8;
  static_assert(4 * 32 * kPitch * 2 <= 2 * kTile, "LDS");
  __syncthreads();
  if (p.db && tk == 0) {
    // columns' sums of the threads that had the same ones, in a fixed order
    float* part = (float*)lds;
    *(float8*)&part[ry * kTN + cy] = sum;
    __syncthreads();
    const int64_t n = n0 + threadIdx.x;
    if (threadIdx.x < kTN && n < p.part.n1) {
      float v = 0.f;
      for (int r = 0; r < kThreads * 8 / kTN; r++)
        v += part[r * kTN + threadIdx.x];
      if (odd && n == p.odd_col) v += (float)__builtin_bit_cast(T, *p.odd);
      if (p.slices > 1)
        p.bias_partial[blockIdx.y * (p.part.n1 - p.part.n0) + n - p.part.n0] =
            v;
      else
        ((O*)p.db)[n] = (O)v;
    }
    __syncthreads();
  }
  float* out = (float*)lds + wave * 32 * kPitch;
  const int er = lane / (FK * 4), ec = lane % (FK * 4) * kVec;
  const int64_t ek = k0 + wk + ec;
  const int em = p.part.k1 - ek < kVec ? (int)(p.part.k1 - ek) : kVec;
  // where the results go: dW, or the slice's part of it
  const bool sliced = p.slices > 1;
  const int64_t pitch = sliced ? p.part.k1 - p.part.k0 : p.k;
  const int64_t origin =
      sliced ? (blockIdx.y * (p.part.n1 - p.part.n0) - p.part.n0) * pitch -
                   p.part.k0
             : 0;
#pragma unroll
  for (int bi = 0; bi < FN; bi++) {
#pragma unroll
    for (int bj = 0; bj < FK; bj++)
#pragma unroll
      for (int i = 0; i < 16; i++)
        out[(8 * (i / 4) + 4 * (lane / 32) + i % 4) * kPitch + bj * 32 +
            lane % 32] = acc[bi][bj][i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = er; r < 32; r += 16 / FK) {
      const int64_t n = n0 + wn + bi * 32 + r;
      const float8 v = *(const float8*)&out[r * kPitch + ec];
      if (n >= p.part.n1 || em <= 0) continue;
      const int64_t to = origin + n * pitch + ek;
      if (sliced)
        store_upto(p.partial + to, v, em);
      else
        store_upto((O*)p.dw + to, v, em);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// The part's dW and db from the slices' sums, in their order.
template <typename O>
__global__ __launch_bounds__(kThreads) void wgrad_join_kernel(Product p) {
  const uint32_t step = gridDim.x * kThreads;
  const uint32_t first = blockIdx.x * kThreads + threadIdx.x;
  auto join = [&](const float* parts, int64_t each, int m) {
    float8 v = 0.f;
#pragma unroll 4
    for (int s = 0; s < p.slices; s++) v += load_upto(parts + s * each, m);
    return v;
  };
  const uint32_t rows = (uint32_t)(p.part.n1 - p.part.n0);
  const uint32_t cols = (uint32_t)(p.part.k1 - p.part.k0);
  // whole rows of dW are one long row
  const uint32_t width = cols == p.k ? rows * cols : cols;
  const uint32_t vecs = (width + kVec - 1) / kVec;
  const uint32_t items = cols == p.k ? vecs : rows * vecs;
  for (uint32_t i = first; i < items; i += step) {
    const uint32_t r = i / vecs, c = i % vecs * kVec;
    const int m = width - c < kVec ? (int)(width - c) : kVec;
    store_upto((O*)p.dw + (p.part.n0 + r) * p.k + p.part.k0 + c,
               join(p.partial + (int64_t)r * cols + c, (int64_t)rows * cols, m),
               m);
  }
  if (!p.db) return;
  for (uint32_t i = first * kVec; i < rows; i += step * kVec) {
    const int m = rows - i < kVec ? (int)(rows - i) : kVec;
    store_upto((O*)p.db + p.part.n0 + i, join(p.bias_partial + i, rows, m), m);
  }
}

// Gradients that the product cannot read as they are (fp32, or rows that
// overlap or lie far apart), laid out anew: rows
// `pitch` elements apart (a multiple of 8), zeros in the columns and, for each
// plane, the rows that fill the last tile.
//
// An fp32 gradient becomes three bf16 planes of 8 bits of its significand
// each, cut off rather than rounded so that no plane can pass the largest
// number: their sum is the value itself, up to the last bits of numbers near
// the smallest.  A NaN or an infinity is whole in the first plane.
template <typename T, typename P>
__global__ __launch_bounds__(kThreads) void layout_kernel(
    const T* dy, int64_t dstride, int64_t m, int64_t n, P* out, int64_t rows,
    int64_t pitch) {
  constexpr int kPlanes = std::is_same_v<T, float> ? 3 : 1;
  const int64_t cols = pitch / kVec;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
       i < rows * cols; i += (int64_t)gridDim.x * kThreads) {
    const int64_t r = i / cols, c = i % cols * kVec;
    float8 v = 0.f;
    if (r < m && c < n)
      v = load_upto(dy + r * dstride + c, (int)(n - c < kVec ? n - c : kVec));
    if constexpr (kPlanes == 1) {
      store8(out + r * pitch + c, v);
    } else {
#pragma unroll
      for (int p = 0; p < kPlanes; p++) {
        float8 h;
#pragma unroll
        for (int j = 0; j < kVec; j++) {
          h[j] = is_finite(v[j])
                     ? __uint_as_float(__float_as_uint(v[j]) & 0xffff0000u)
                     : v[j];
          v[j] = is_finite(v[j]) ? v[j] - h[j] : 0.f;
        }
        store8(out + (p * rows + r) * pitch + c, h);
      }
    }
  }
}

// How a part is computed: the tiles' shape, and the number of slices that the
// rows are cut in.
struct Shape {
  Part part;
  bool big;
  int slices, slice_tiles;
  double time;  // us, by the model
};

struct Plan {
  bool laid_out;
  int planes, xtiles, parts;
  Shape shape[2];
  int64_t pitch;
  size_t laid_bytes, partial_bytes, bias_bytes;
};

size_t round256(size_t b) { return (b + 255) & ~size_t(255); }

// A part's shape and slices, by the time that they take, from measurements of
// products with 32 to 16384 rows and 64 to 25088 columns (the model is within
// 15% of them).
//
// Tiles of 256 by 256, one workgroup to a compute unit, need half of the LDS
// reads that tiles of 128 by 128 do for the same work (1.5 us for 64 rows, or
// 0.38 for a quarter of it, against 0.62 alone and 1.05 for two that share a
// compute unit).  But they leave more of a small dW's edge empty, cut it in
// fewer pieces, and nothing runs beside their start and their results' way out
// (9 us, or 14.5 with fp32 results, against 4 and 6.5): 2048 x 2048 x 2048
// takes 27 us with the small ones and 41 with the large, 64 x 4096 x 25088 57
// and 71, 4096 x 4096 x 4096 150 and 113.  Small ones do not wait for each
// other's rounds.  Slices fill compute units that too few tiles leave idle and
// cost a second pass over their sums: 16384 x 256 x 256 takes 160 us in one
// slice and 21 in 16.
double tiles_time(bool big, bool f32, int64_t groups, int tiles) {
  const double rounds = (double)groups / (big ? kUnits : 2 * kUnits);
  const double tile = big ? 1.5 : groups > kUnits ? 1.05 : 0.62;
  const double ends = big ? (f32 ? 14.5 : 9) : (f32 ? 6.5 : 4);
  return (!big && rounds > 4 ? rounds : ceil(rounds)) * (tiles * tile + ends);
}

Shape pick_shape(const Part& part, bool f32, int tiles) {
  const int64_t rows = part.n1 - part.n0, cols = part.k1 - part.k0;
  Shape s = {};
  for (int big = 0; big < 2; big++) {
    const int size = big ? 256 : 128;
    const int64_t nt = (rows + size - 1) / size, kt = (cols + size - 1) / size;
    for (int cut = 1; cut <= 512 && cut <= tiles; cut += 1 + cut / 16) {
      const int each = (tiles + cut - 1) / cut;
      if ((tiles + each - 1) / each != cut) continue;
      if (cut > 1 && nt * kt * cut > 1024) break;
      double t = tiles_time(big, f32, nt * kt * cut, each);
      if (cut > 1) t += 4 + cut * (double)rows * cols * 1e-6;
      if (s.time > 0 && t >= s.time) continue;
      s = {part, (bool)big, cut, each, t};
      s.part.ntiles = (int)nt;
      s.part.ktiles = (int)kt;
    }
  }
  return s;
}

// Large tiles that fill the compute units a whole number of times, and the
// columns or rows of dW behind them as a part of its own, where that is
// quicker: a last round of a few large tiles takes as long as a full one.  bf16
// products of 4096 x 4352 x 4352 took 202 us without parts and take 150, 8192
// x 2048 x 8448 335 and 240, 12000 x 6000 x 6000 848 and 748.
void pick_parts(const Act8Wgrad& a, Plan& p) {
  const int tiles = p.planes * p.xtiles;
  const int64_t nt = (a.n + 255) / 256, kt = (a.k + 255) / 256;
  p.parts = 1;
  const bool f32 = p.planes > 1;
  p.shape[0] = pick_shape({0, a.n, 0, a.k}, f32, tiles);
  double best = p.shape[0].time;
  const int64_t full = nt * kt / kUnits;  // rounds
  if (full < 1 || full > 64 || nt * kt % kUnits == 0) return;
  for (int along_k = 0; along_k < 2; along_k++) {
    const int64_t other = along_k ? nt : kt;
    const int64_t own = full * kUnits / other;  // columns or rows of tiles
    if (own < 1) continue;
    Part first = {0, a.n, 0, a.k, (int)nt, (int)kt}, rest = first;
    if (along_k)
      first.k1 = rest.k0 = own * 256, first.ktiles = (int)own;
    else
      first.n1 = rest.n0 = own * 256, first.ntiles = (int)own;
    const double time =
        tiles_time(true, f32, (int64_t)first.ntiles * first.ktiles, tiles);
    const Shape s = pick_shape(rest, f32, tiles);
    if (time + s.time + 2 >= best) continue;
    best = time + s.time + 2;
    p.parts = 2;
    p.shape[0] = {first, true, 1, tiles, time};
    p.shape[1] = s;
  }
}

Plan plan_of(const Act8Wgrad& a) {
  Plan p = {};
  p.planes = a.type == ElemType::kF32 ? 3 : 1;
  // Rows of any alignment are read as they are: laying out those of an odd
  // length first took 133 us where this takes 68 (13622 x 6809 x 140 fp16), and
  // 35 and 31 at 2048 x 2047 x 2047 bf16.
  p.laid_out = p.planes > 1 || a.dstride < a.n || a.dstride > kAct8MaxCols;
  p.pitch = p.laid_out ? (a.n + 7) / 8 * 8 : a.dstride;
  p.xtiles = (int)((a.m + kTM - 1) / kTM);
  if (p.laid_out)
    p.laid_bytes =
        round256((size_t)p.planes * p.xtiles * kTM * p.pitch * 2);
  pick_parts(a, p);
  const Shape& s = p.shape[p.parts - 1];  // the only one that has slices
  if (s.slices > 1) {
    const size_t rows = (size_t)s.slices * (s.part.n1 - s.part.n0);
    p.partial_bytes =
        round256(rows * (s.part.k1 - s.part.k0) * sizeof(float));
    p.bias_bytes = round256(rows * sizeof(float));
  }
  return p;
}

template <typename T, typename O, bool kOdd>
void launch_product(const Shape& s, const Product& p, hipStream_t stream) {
  const dim3 grid((uint32_t)(s.part.ntiles * s.part.ktiles),
                  (uint32_t)s.slices);
  if (s.big)
    launch(act8_wgrad_kernel<T, O, 4, 4, kOdd>, grid, kThreads, stream, p);
  else
    launch(act8_wgrad_kernel<T, O, 2, 2, kOdd>, grid, kThreads, stream, p);
}

uint32_t flat_grid(int64_t items) {
  const int64_t want = (items + kThreads - 1) / kThreads;
  return (uint32_t)(want < 4096 ? want : 4096);
}

}  // namespace

size_t act8_wgrad_workspace(const Act8Wgrad& a) {
  if (a.m == 0 || a.n == 0 || a.k == 0) return 0;
  const Plan p = plan_of(a);
  return p.laid_bytes + p.partial_bytes + p.bias_bytes;
}

hipError_t act8_wgrad(const Act8Wgrad& a, hipStream_t stream) {
  if (a.m == 0 || a.n == 0 || a.k == 0) return hipSuccess;
  if (a.n > kAct8MaxCols || a.pitch > kAct8MaxCols) return hipErrorInvalidValue;
  const Plan plan = plan_of(a);
  for (int i = 0; i < plan.parts; i++) {
    const Shape& s = plan.shape[i];
    if ((int64_t)s.part.ntiles * s.part.ktiles * s.slices > (1 << 23) ||
        s.slices > 65535)
      return hipErrorInvalidValue;
  }
  char* ws = (char*)a.workspace;
  const int64_t laid_rows = (int64_t)plan.xtiles * kTM;
  Product p = {};
  p.dpitch = (int)(plan.pitch * 2);
  p.cpitch = (int)a.pitch;
  const int64_t last = (int64_t)(plan.xtiles - 1) * kTM;  // its first row
  p.dy.base = plan.laid_out ? ws : (const char*)a.dy;
  p.dy.tile = (int64_t)kTM * plan.pitch * 2;
  // the 2 bytes are the next row's first, for a last value in half of 4 bytes
  const bool odd = !plan.laid_out && a.n % 2;
  p.dy.full = (int)p.dy.tile + (odd ? 2 : 0);
  p.dy.tail = plan.laid_out
                  ? p.dy.full
                  : (int)(((a.m - last - 1) * a.dstride + a.n) * 2);
  p.codes = {(const char*)a.codes, kTM * a.pitch, (int)(kTM * a.pitch),
             (int)((a.m - last) * a.pitch)};
  p.exps = {(const char*)a.exps, kTM * a.pitch / kAct8Group,
            (int)(kTM * a.pitch / kAct8Group),
            (int)((a.m - last) * a.pitch / kAct8Group)};
  p.xtiles = plan.xtiles;
  p.tiles = plan.planes * plan.xtiles;
  p.k = a.k;
  p.dw = a.dw;
  if (odd) {
    p.odd = (const short*)a.dy + (a.m - 1) * a.dstride + a.n - 1;
    p.odd_col = a.n - 1;
    p.odd_codes = a.codes + (a.m - 1) * a.pitch;
    p.odd_exps = a.exps + (a.m - 1) * a.pitch / kAct8Group;
  }
  p.partial = (float*)(ws + plan.laid_bytes);
  p.bias_partial = (float*)(ws + plan.laid_bytes + plan.partial_bytes);
  with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    using P = std::conditional_t<std::is_same_v<T, float>, bf16, T>;
    if (plan.laid_out)
      launch(layout_kernel<T, P>, flat_grid(laid_rows * plan.pitch / kVec),
             kThreads, stream, (const T*)a.dy, a.dstride, a.m, a.n, (P*)ws,
             laid_rows, plan.pitch);
    for (int i = 0; i < plan.parts; i++) {
      const Shape& s = plan.shape[i];
      p.part = s.part;
      p.slices = s.slices;
      p.slice_tiles = s.slice_tiles;
      p.db = s.part.k0 == 0 ? a.db : nullptr;
      if constexpr (std::is_same_v<P, T>) {
        if (odd)
          launch_product<P, T, true>(s, p, stream);
        else
          launch_product<P, T, false>(s, p, stream);
      } else {
        launch_product<P, T, false>(s, p, stream);
      }
      if (s.slices > 1)
        launch(wgrad_join_kernel<T>,
               flat_grid((s.part.n1 - s.part.n0) * (s.part.k1 - s.part.k0) /
                             kVec +
                         1),
               kThreads, stream, p);
    }
  });
  return hipGetLastError();
}

}  // namespace baguanet
