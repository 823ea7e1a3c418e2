// act8.hip — activation checkpoints in 8 bits (gfx950).
//
// A group of 32 neighbouring values of a row is kept as q[i] * 2^e, q in
// e4m3 (round to nearest even), with the smallest e that brings the largest
// finite value to at most 448 = max(e4m3).  2^e is a power of two so that
// q * 2^e is exact in the activation's own type: e is held to the range
// where that is so, [-117, 120] for bf16 and fp32, [-15, 8] for fp16, and at
// its upper end q stops at 240, the last value whose product stays finite.
// A value is off by at most 1/16 of itself, or by 2^(e-10) below 2^(e-6).
// A NaN or an infinity is kept as NaN and does not enter its group's scale.
//
// These kernels are bound by HBM; four lanes hold a group, 8 values each, and
// find its largest value with two lane exchanges.  16384 rows of 8192 bf16
// pairs: silu forward 213 us (5.1 TB/s), backward 197 (5.5); 16384 rows of 4096
// bf16 are packed in 37 us (5.5) and unpacked in 30 (6.7), into fp32 in 88
// (3.8).  A large copy moves 5.0 TB/s.
#include <hip/hip_runtime.h>

#include "act8_codes.h"

namespace baguanet {
namespace {

constexpr int kBlock = 256;

// A team of `tpr` lanes (a power of two, 4 to kBlock) moves a row, or a piece
// of one where rows are too few to fill the chip: 256 rows of 25088 fp32 are
// packed in 6.9 us in pieces and in 9.9 whole, 1000 rows of 16384 bf16 in 12.8
// and 11.4.
struct Teams {
  int tpr;
  uint32_t pieces, items;  // of a row, and in all
  int64_t span;            // columns of a piece
};

// The item's row, and the lane's columns in it: from c on, up to the end.
__device__ inline int64_t place(const Teams& t, uint32_t item, int lane,
                                int64_t cols, int64_t& c, int64_t& end) {
  c = lane * kVec;
  end = cols;
  if (t.pieces == 1) return item;
  const uint32_t row = item / t.pieces;
  const int64_t first = (item - row * t.pieces) * t.span;
  c += first;
  end = first + t.span < cols ? first + t.span : cols;
  return row;
}

template <typename T>
__global__ __launch_bounds__(kBlock) void act8_pack_kernel(Act8Move a,
                                                           Teams t) {
  const int team = threadIdx.x / t.tpr, lane = threadIdx.x % t.tpr;
  const uint32_t teams = kBlock / t.tpr;
  for (uint32_t i = blockIdx.x * teams + team; i < t.items;
       i += gridDim.x * teams) {
    int64_t c, end;
    const int64_t r = place(t, i, lane, a.pitch, c, end);
    const T* src = (const T*)a.x + r * a.xstride;
    for (; c < end; c += t.tpr * kVec) {
      float8 v = 0.f;
      if (c < a.cols)
        v = load_upto(src + c, (int)(a.cols - c < kVec ? a.cols - c : kVec));
      const int e = group_power<T>(v);
      *(uint2*)(a.codes + r * a.pitch + c) = encode8<T>(v, e);
      if (c % kAct8Group == 0)
        a.exps[(r * a.pitch + c) / kAct8Group] = (uint8_t)(e + 127);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void act8_unpack_kernel(Act8Move a,
                                                             Teams t) {
  const int team = threadIdx.x / t.tpr, lane = threadIdx.x % t.tpr;
  const uint32_t teams = kBlock / t.tpr;
  for (uint32_t i = blockIdx.x * teams + team; i < t.items;
       i += gridDim.x * teams) {
    int64_t c, end;
    const int64_t r = place(t, i, lane, a.cols, c, end);
    T* dst = (T*)a.x + r * a.xstride;
    for (; c < end; c += t.tpr * kVec) {
      const uint2 q = *(const uint2*)(a.codes + r * a.pitch + c);
      const int e = a.exps[(r * a.pitch + c) / kAct8Group] - 127;
      store_upto(dst + c, decode8(q, e),
                 (int)(a.cols - c < kVec ? a.cols - c : kVec));
    }
  }
}

// ---- out = silu(a) * b, its inputs kept in 8 bits --------------------------
// x holds a in its first `cols` columns and b in the others.  With the kept
// values a', b' and s = 1 / (1 + exp(-a')):
//   da = dout * b' * s * (1 + a' * (1 - s))     db = dout * a' * s

// s and 1 - s.  With h = exp(-|a| / 2), s is 1 / (1 + h^2) or h^2 times that,
// and stays in two factors: far below 0 it is less than fp32's smallest normal
// number where its product with a and b is not.
struct Sigmoid {
  float s0, s1, rest;
  __device__ inline explicit Sigmoid(float a) {
    const float h = expf(-0.5f * fabsf(a)), e = h * h;
    const float r = __builtin_amdgcn_rcpf(1.f + e);
    s0 = a < 0.f ? h : r;
    s1 = a < 0.f ? h * r : 1.f;
    rest = a < 0.f ? r : e * r;
  }
};

template <typename T>
__global__ __launch_bounds__(kBlock) void silu_forward_kernel(SiluAct8 p,
                                                              Teams t) {
  const int team = threadIdx.x / t.tpr, lane = threadIdx.x % t.tpr;
  const uint32_t teams = kBlock / t.tpr;
  for (uint32_t i = blockIdx.x * teams + team; i < t.items;
       i += gridDim.x * teams) {
    int64_t c, end;
    const int64_t r = place(t, i, lane, p.pitch, c, end);
    const T* src = (const T*)p.x + r * p.xstride;
    for (; c < end; c += t.tpr * kVec) {
      float8 a = 0.f, b = 0.f, o;
      const int m = c < p.cols ? (int)(p.cols - c < kVec ? p.cols - c : kVec)
                               : 0;
      if (m) {
        a = load_upto(src + c, m);
        b = load_upto(src + p.cols + c, m);
#pragma unroll
        for (int i = 0; i < kVec; i++) {
          const Sigmoid s(a[i]);
          o[i] = a[i] * s.s0 * b[i] * s.s1;
        }
        store_upto((T*)p.out + r * p.cols + c, o, m);
      }
      if (!p.codes) continue;
      const int ea = group_power<T>(a), eb = group_power<T>(b);
      uint8_t* q = p.codes + r * 2 * p.pitch + c;
      *(uint2*)q = encode8<T>(a, ea);
      *(uint2*)(q + p.pitch) = encode8<T>(b, eb);
      if (c % kAct8Group == 0) {
        uint8_t* e = p.exps + (r * 2 * p.pitch + c) / kAct8Group;
        e[0] = (uint8_t)(ea + 127);
        e[p.pitch / kAct8Group] = (uint8_t)(eb + 127);
      }
    }
  }
}

// Whole rows here: cut in pieces the kernel takes fewer registers, and with
// more waves at once 204 us where it takes 199 (16384 rows of 8192 bf16).
template <typename T>
__global__ __launch_bounds__(kBlock) void silu_backward_kernel(SiluAct8 p,
                                                               int tpr) {
  const int team = threadIdx.x / tpr, lane = threadIdx.x % tpr;
  const int64_t teams = kBlock / tpr;
  for (int64_t r = (int64_t)blockIdx.x * teams + team; r < p.rows;
       r += (int64_t)gridDim.x * teams) {
    for (int64_t c = (int64_t)lane * kVec; c < p.cols;
         c += (int64_t)tpr * kVec) {
      const int m = (int)(p.cols - c < kVec ? p.cols - c : kVec);
      const uint8_t* q = p.codes + r * 2 * p.pitch + c;
      const uint8_t* e = p.exps + (r * 2 * p.pitch + c) / kAct8Group;
      const float8 a = decode8(*(const uint2*)q, e[0] - 127);
      const float8 b = decode8(*(const uint2*)(q + p.pitch),
                               e[p.pitch / kAct8Group] - 127);
      const float8 d =
          load_upto((const T*)p.dout + r * p.dstride + c, m);
      float8 da, db;
#pragma unroll
      for (int i = 0; i < kVec; i++) {
        const Sigmoid s(a[i]);
        da[i] = d[i] * b[i] * s.s0 * (1.f + a[i] * s.rest) * s.s1;
        db[i] = d[i] * s.s0 * a[i] * s.s1;
      }
      T* dst = (T*)p.dx + r * 2 * p.cols + c;
      store_upto(dst, da, m);
      store_upto(dst + p.cols, db, m);
    }
  }
}

int team_size(int64_t pitch) {
  int tpr = kAct8Group / kVec;
  while (tpr < kBlock && (int64_t)tpr * kVec < pitch) tpr *= 2;
  return tpr;
}

Teams teams_of(int64_t rows, int64_t pitch) {
  Teams t = {team_size(pitch), 1, (uint32_t)rows, pitch};
  if (t.tpr == kBlock && rows < 512) {
    t.span = kBlock * kVec;
    t.pieces = (uint32_t)((pitch + t.span - 1) / t.span);
    t.items = (uint32_t)(rows * t.pieces);
  }
  return t;
}

// One team for each item, up to enough workgroups to fill the chip.
uint32_t team_grid(int64_t items, int tpr) {
  const int64_t teams = kBlock / tpr, want = (items + teams - 1) / teams;
  return (uint32_t)(want < 8192 ? want : 8192);
}

}  // namespace

hipError_t act8_pack(const Act8Move& a, hipStream_t stream) {
  if (a.rows == 0 || a.cols == 0) return hipSuccess;
  const Teams cut = teams_of(a.rows, a.pitch);
  with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    launch(act8_pack_kernel<T>, team_grid(cut.items, cut.tpr), kBlock, stream,
           a, cut);
  });
  return hipGetLastError();
}

hipError_t act8_unpack(const Act8Move& a, hipStream_t stream) {
  if (a.rows == 0 || a.cols == 0) return hipSuccess;
  const Teams cut = teams_of(a.rows, a.pitch);
  with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    launch(act8_unpack_kernel<T>, team_grid(cut.items, cut.tpr), kBlock, stream,
           a, cut);
  });
  return hipGetLastError();
}

hipError_t silu_act8_forward(const SiluAct8& p, hipStream_t stream) {
  if (p.rows == 0 || p.cols == 0) return hipSuccess;
  const Teams cut = teams_of(p.rows, p.pitch);
  with_type(p.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    launch(silu_forward_kernel<T>, team_grid(cut.items, cut.tpr), kBlock,
           stream, p, cut);
  });
  return hipGetLastError();
}

hipError_t silu_act8_backward(const SiluAct8& p, hipStream_t stream) {
  if (p.rows == 0 || p.cols == 0) return hipSuccess;
  const int tpr = team_size(p.pitch);
  with_type(p.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    launch(silu_backward_kernel<T>, team_grid(p.rows, tpr), kBlock, stream, p,
           tpr);
  });
  return hipGetLastError();
}

}  // namespace baguanet
