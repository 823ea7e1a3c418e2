// train_kernels.h — launchers of the training-step kernels, as the torch
// extension calls them.  Sizes, types and strides are checked there.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace baguanet {

enum class ElemType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// ---- embedding (embedding.hip) --------------------------------------------

struct EmbeddingFwd {
  const void* weight;  // [vocab, dim], rows `wstride` elements apart
  const void* tokens;  // [n] int64 or int32
  void* out;           // [n, dim]
  int64_t vocab, dim, n, wstride;
  float scale;
  bool tok64;
  ElemType wtype, otype;
};
hipError_t embedding_forward(const EmbeddingFwd& a, hipStream_t stream);

struct EmbeddingBwd {
  const void* dout;    // [n, dim], rows `dstride` elements apart
  const void* tokens;  // [n] int64 or int32
  void* dweight;       // [vocab, dim]
  void* workspace;     // embedding_workspace() bytes
  int64_t vocab, dim, n, dstride;
  int64_t padding;     // token without a gradient, or -1
  float scale;
  bool tok64;
  ElemType dtype, wtype;
};
// Elements that a table with a gradient may have, fewer than: the launches that
// clear it are counted in 32 bits.
constexpr int64_t kEmbeddingMaxGrad = int64_t(1) << 35;
size_t embedding_workspace(int64_t vocab, int64_t dim, int64_t n);
hipError_t embedding_backward(const EmbeddingBwd& a, hipStream_t stream);

// ---- gated residual norm (residual_norm.hip) -------------------------------

// How a gate multiplies the branch: one value for each column of a group of
// rows, one for each row, or one for each element.
enum class Gate : int { kNone = 0, kGroup = 1, kRow = 2, kFull = 3 };

// The columns that the kernels hold in registers, at most.
constexpr int64_t kNormMaxDim = 16384;

struct NormFwd {
  const void* x;       // [rows, dim], rows `xstride` elements apart
  const void* branch;  // [rows, dim], rows `bstride` apart; null: y = x
  const void* gate;
  const void* post;    // [dim], or null: the branch is added as it is
  const void* pre;     // [dim], or null: ones
  void* y;             // [rows, dim]; null: not written (y = x)
  void* h;             // [rows, dim]; null: not wanted
  float* rbranch;      // [rows] 1 / rms of the branch, or null
  float* ry;           // [rows] 1 / rms of y, or null
  int64_t rows, dim, xstride, bstride;
  int64_t group_rows;  // rows of a gate's group (kGroup)
  float residual_scale, branch_scale, eps;
  Gate gmode;
  bool gate32, post32, pre32;  // their type: fp32, else that of x
  ElemType type;
};
hipError_t norm_forward(const NormFwd& a, hipStream_t stream);

struct NormBwd {
  const void* x;       // [rows, dim] and branch, as in the forward pass: y is
  const void* branch;  // computed again, for its unrounded value
  const void* gate;
  const void* post;
  const void* pre;
  const void* dy;      // [rows, dim], rows `dystride` apart, or null: zero
  const void* dh;      // [rows, dim], rows `dhstride` apart, or null: zero
  const float* rbranch;
  const float* ry;
  void* dx;            // [rows, dim]
  void* dbranch;       // [rows, dim] (with a branch)
  void* dgate;         // the gate's shape, or null; fp32 if dgate32, else T
  void* dpost;         // [dim], or null
  void* dpre;          // [dim], or null
  void* workspace;     // norm_workspace() bytes
  int64_t rows, dim, xstride, bstride, dystride, dhstride;
  int64_t group_rows;
  float residual_scale, branch_scale;
  Gate gmode;
  bool gate32, post32, pre32, dgate32;
  ElemType type;
};
size_t norm_workspace(const NormBwd& a);
hipError_t norm_backward(const NormBwd& a, hipStream_t stream);

// The gradient of a gate that is repeated: the sum of [outer, rows, inner]
// over its rows.
struct GateSum {
  const float* in;     // [outer, rows, inner]
  void* out;           // [outer, inner]
  float* workspace;    // norm_gate_workspace() bytes
  int64_t outer, rows, inner;
  ElemType type;       // of out
};
size_t norm_gate_workspace(const GateSum& a);
hipError_t norm_gate_sum(const GateSum& a, hipStream_t stream);

// ---- 8-bit activation checkpoints (act8.hip, act8_wgrad.hip) ---------------

// Values of a row are kept in groups of 32 that share a power of two 2^e, as
// e4m3 numbers (one byte each) times that power; e + 127 is a byte of its
// own.  Rows of codes are `pitch` bytes apart, a multiple of 32, and the
// columns past the row's end hold zeros.
constexpr int kAct8Group = 32;

// Columns of a gradient or of codes that one product takes, at most: 64 rows
// of them are addressed in 31 bits.
constexpr int64_t kAct8MaxCols = 1 << 23;

struct Act8Move {
  void* x;             // [rows, cols], rows `xstride` elements apart
  uint8_t* codes;      // [rows, pitch]
  uint8_t* exps;       // [rows, pitch / 32]
  int64_t rows, cols, pitch, xstride;
  ElemType type;
};
hipError_t act8_pack(const Act8Move& a, hipStream_t stream);
hipError_t act8_unpack(const Act8Move& a, hipStream_t stream);

struct SiluAct8 {
  const void* x;       // [rows, 2 * cols] (forward), rows `xstride` apart
  void* out;           // [rows, cols] (forward)
  const void* dout;    // [rows, cols] (backward), rows `dstride` apart
  void* dx;            // [rows, 2 * cols] (backward)
  uint8_t* codes;      // [rows, 2 * pitch]; null: not kept
  uint8_t* exps;       // [rows, 2 * pitch / 32]
  int64_t rows, cols, pitch, xstride, dstride;
  ElemType type;
};
hipError_t silu_act8_forward(const SiluAct8& a, hipStream_t stream);
hipError_t silu_act8_backward(const SiluAct8& a, hipStream_t stream);

struct Act8Wgrad {
  const void* dy;      // [m, n], rows `dstride` elements apart
  const uint8_t* codes;  // [m, pitch]
  const uint8_t* exps;
  void* dw;            // [n, k]
  void* db;            // [n], or null
  void* workspace;     // act8_wgrad_workspace() bytes
  int64_t m, n, k, pitch, dstride;
  ElemType type;
};
size_t act8_wgrad_workspace(const Act8Wgrad& a);
hipError_t act8_wgrad(const Act8Wgrad& a, hipStream_t stream);

}  // namespace baguanet
