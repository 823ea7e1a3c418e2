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
// to 920 us (1.2 to 1.3 PFLOP/s, as the clock allows), where the library's
// product of the uncompressed operands takes 980; 4096^3 takes 110 (1.25
// PFLOP/s; 117).  With few rows a tile's start and its way out weigh most: 256
// x 4096 x 25088 fp32 takes 219 us for 0.16 TFLOP and 411 MB of dW.
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
// against the descriptor's size), so the last tile needs no conditions; those
// behind a row's end give the next row's values, which only reach columns that
// are not written.
struct Stream {
  const char* base;
  int64_t tile;    // bytes from one tile to the next
  int full, tail;  // bytes of a tile, and of the last
};

__device__ inline __amdgpu_buffer_rsrc_t descriptor(const char* p, int size) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, size, 0x00027000);
}

// One product: dy in tiles of kTM rows, `tiles` in all; x' starts again
// after `xtiles` of them (the planes of an fp32 gradient).
struct Product {
  Stream dy, codes, exps;
  int dpitch, cpitch;      // bytes between rows of dy and of codes
  int tiles, xtiles;
  int slices, slice_tiles;
  int ntiles, ktiles;
  int64_t n, k;
  void* dw;
  void* db;                // null: not wanted
  float* partial;          // [slices, n, k] where slices > 1
  float* bias_partial;     // [slices, n] where slices > 1
};

// The workgroup's tile of dW.  Workgroups go to the 8 XCDs in turn; each XCD
// takes a run of tiles, in strips 8 tiles high, so that those at work
// together read the same parts of dy and x' through its L2.
__device__ inline void pick_tile(const Product& p, int& tn, int& tk) {
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
// FN by FK blocks of 32 by 32.
//
// Two tiles are in LDS: the matrix instructions of one overlap with the
// writing of the next, whose rows are in registers by then, and with the
// loads of the one after.  A step's fragments are read during the step
// before, across the tiles' border too: the one barrier of a tile stands
// before its last step, when all its fragments have been read and all of the
// next tile is written.
template <typename T, typename O, int FN, int FK>
__global__ __launch_bounds__(kThreads, FN * FK > 8 ? 1 : 2)
void act8_wgrad_kernel(Product p) {
  constexpr int kTN = 64 * FN, kTK = 64 * FK;
  constexpr int kPassN = kTM * kTN / 8 / kThreads;
  constexpr int kPassK = kTM * kTK / 8 / kThreads;
  constexpr int kRowsN = kTM / kPassN, kRowsK = kTM / kPassK;  // of a pass
  constexpr int kTile = kTM * (kTN + kTK);  // both operands' tiles
  __shared__ __attribute__((aligned(16))) short lds[2 * kTile];
  int tn, tk;
  pick_tile(p, tn, tk);
  const int64_t n0 = (int64_t)tn * kTN, k0 = (int64_t)tk * kTK;
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
    if (threadIdx.x < kTN && n < p.n) {
      float v = 0.f;
      for (int r = 0; r < kThreads * 8 / kTN; r++)
        v += part[r * kTN + threadIdx.x];
      if (p.slices > 1)
        p.bias_partial[blockIdx.y * p.n + n] = v;
      else
        ((O*)p.db)[n] = (O)v;
    }
    __syncthreads();
  }
  float* out = (float*)lds + wave * 32 * kPitch;
  const int er = lane / (FK * 4), ec = lane % (FK * 4) * kVec;
  const int64_t ek = k0 + wk + ec;
  const int em = p.k - ek < kVec ? (int)(p.k - ek) : kVec;
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
      if (n >= p.n || em <= 0) continue;
      if (p.slices > 1)
        store_upto(p.partial + (blockIdx.y * p.n + n) * p.k + ek, v, em);
      else
        store_upto((O*)p.dw + n * p.k + ek, v, em);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// dW and db from the slices' sums, in their order.
template <typename O>
__global__ __launch_bounds__(kThreads) void wgrad_join_kernel(
    const float* partial, const float* bias, int slices, int64_t count,
    int64_t n, O* dw, O* db) {
  const int64_t step = (int64_t)gridDim.x * kThreads * kVec;
  const int64_t first = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kVec;
  auto join = [&](const float* parts, int64_t i, int64_t count, O* out) {
    const int m = (int)(count - i < kVec ? count - i : kVec);
    float8 v = 0.f;
#pragma unroll 4
    for (int s = 0; s < slices; s++) v += load_upto(parts + s * count + i, m);
    store_upto(out + i, v, m);
  };
  for (int64_t i = first; i < count; i += step) join(partial, i, count, dw);
  if (db)
    for (int64_t i = first; i < n; i += step) join(bias, i, n, db);
}

// Gradients that the product cannot read as they are, laid out anew: rows
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

struct Plan {
  bool big, laid_out;
  int planes, slices, slice_tiles, xtiles, ntiles, ktiles;
  int64_t pitch;
  size_t laid_bytes, partial_bytes, bias_bytes;
};

size_t round256(size_t b) { return (b + 255) & ~size_t(255); }

// The tiles' shape and the number of slices that the rows are cut in, by the
// time that they take, in us, from measurements of bf16 products with 64 to
// 16384 rows and 64 to 8192 columns (the model is within 15% of them).
//
// Tiles of 256 by 256, one workgroup to a compute unit, need half of the LDS
// reads that tiles of 128 by 128 do for the same work (1.45 us for 64 rows, or
// 0.36 for a quarter of it, against 0.62 alone and 1.05 for two that share a
// compute unit), but leave more of a small dW's edge empty and cut it in
// fewer pieces: 2048 x 2048 x 2048 takes 27 us with the small ones and 41 with
// the large, 4096 x 4096 x 4096 150 and 113.  Slices fill compute units that
// too few tiles leave idle and cost a second pass over their sums: 16384 x
// 256 x 256 takes 160 us in one slice and 21 in 16.
void pick_shape(const Act8Wgrad& a, Plan& p) {
  const int64_t tiles = (int64_t)p.planes * p.xtiles;
  double best = 0;
  for (int big = 0; big < 2; big++) {
    const int size = big ? 256 : 128;
    const int64_t nt = (a.n + size - 1) / size, kt = (a.k + size - 1) / size;
    for (int64_t cut = 1; cut <= 512 && cut <= tiles;
         cut += 1 + cut / 16) {
      const int64_t each = (tiles + cut - 1) / cut;
      if ((tiles + each - 1) / each != cut) continue;
      const double groups = (double)nt * kt * cut;
      if (cut > 1 && groups > 1024) break;
      const double rounds = ceil(groups / (big ? 256 : 512));
      const double tile = big ? 1.45 : groups > 256 ? 1.05 : 0.62;
      double t = rounds * (each * tile + (big ? 9 : 5));
      if (cut > 1) t += 4 + cut * (double)a.n * a.k * 1e-6;
      if (best > 0 && t >= best) continue;
      best = t;
      p.big = big;
      p.ntiles = (int)nt;
      p.ktiles = (int)kt;
      p.slices = (int)cut;
      p.slice_tiles = (int)each;
    }
  }
}

Plan plan_of(const Act8Wgrad& a) {
  Plan p = {};
  p.planes = a.type == ElemType::kF32 ? 3 : 1;
  // The product reads rows of dy in aligned 16-byte pieces.
  p.laid_out = p.planes > 1 || a.n % 8 || a.dstride % 8 || a.dstride < a.n ||
               a.dstride > kAct8MaxCols || ((uintptr_t)a.dy & 15);
  p.pitch = p.laid_out ? (a.n + 7) / 8 * 8 : a.dstride;
  p.xtiles = (int)((a.m + kTM - 1) / kTM);
  if (p.laid_out)
    p.laid_bytes =
        round256((size_t)p.planes * p.xtiles * kTM * p.pitch * 2);
  pick_shape(a, p);
  if (p.slices > 1) {
    p.partial_bytes = round256((size_t)p.slices * a.n * a.k * sizeof(float));
    p.bias_bytes = round256((size_t)p.slices * a.n * sizeof(float));
  }
  return p;
}

template <typename T, typename O>
void launch_product(const Plan& plan, const Product& p, hipStream_t stream) {
  const dim3 grid((uint32_t)(plan.ntiles * plan.ktiles),
                  (uint32_t)plan.slices);
  if (plan.big)
    launch(act8_wgrad_kernel<T, O, 4, 4>, grid, kThreads, stream, p);
  else
    launch(act8_wgrad_kernel<T, O, 2, 2>, grid, kThreads, stream, p);
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
  if ((int64_t)plan.ntiles * plan.ktiles * plan.slices > (1 << 23) ||
      plan.slices > 65535)
    return hipErrorInvalidValue;
  char* ws = (char*)a.workspace;
  const int64_t laid_rows = (int64_t)plan.xtiles * kTM;
  Product p = {};
  p.dpitch = (int)(plan.pitch * 2);
  p.cpitch = (int)a.pitch;
  const int64_t last = (int64_t)(plan.xtiles - 1) * kTM;  // its first row
  p.dy.base = plan.laid_out ? ws : (const char*)a.dy;
  p.dy.tile = (int64_t)kTM * plan.pitch * 2;
  p.dy.full = (int)p.dy.tile;
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
  p.slices = plan.slices;
  p.slice_tiles = plan.slice_tiles;
  p.ntiles = plan.ntiles;
  p.ktiles = plan.ktiles;
  p.n = a.n;
  p.k = a.k;
  p.dw = a.dw;
  p.db = a.db;
  p.partial = (float*)(ws + plan.laid_bytes);
  p.bias_partial = (float*)(ws + plan.laid_bytes + plan.partial_bytes);
  with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    using P = std::conditional_t<std::is_same_v<T, float>, bf16, T>;
    if (plan.laid_out)
      launch(layout_kernel<T, P>, flat_grid(laid_rows * plan.pitch / kVec),
             kThreads, stream, (const T*)a.dy, a.dstride, a.m, a.n, (P*)ws,
             laid_rows, plan.pitch);
    launch_product<P, T>(plan, p, stream);
    if (plan.slices > 1)
      launch(wgrad_join_kernel<T>, flat_grid(a.n * a.k / kVec + 1), kThreads,
             stream, (const float*)p.partial, (const float*)p.bias_partial,
             plan.slices, a.n * a.k, a.n, (T*)a.dw, (T*)a.db);
  });
  return hipGetLastError();
}

}  // namespace baguanet
