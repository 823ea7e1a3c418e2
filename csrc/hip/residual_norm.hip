// residual_norm.hip — the seam between two blocks of a network in one pass
// (gfx950):
//
//   u = N(o) * post        N(v) = v / sqrt(mean(v^2) + eps), over a row
//   y = rs * x + bs * g * u          (the residual stream goes on)
//   h = N(y) * pre                   (the next block's input)
//
// and its gradient.  With t = dh * pre, ny = y * ry, no = o * ro:
//
//   dY = dy + ry * (t - ny * mean(ny * t))      dx = rs * dY
//   do = ro * (c * dY - no * mean(no * c * dY)) c  = bs * g * post
//   dpre = sum dh * ny    dpost = sum bs * g * dY * no
//   dg = sum over the gate's elements of bs * post * dY * no
//
// Both passes are bound by HBM: 4 row reads and writes forward, 6 backward.
// 32768 rows of 8192 bf16: forward 378 us (5.7 TB/s), backward 636 (5.1) and 8
// for the join; backward 3.9 TB/s above 8192 columns.  A large copy moves 5.0.
// Backward of 1024 to 8192 columns without a post weight 4.7 to 5.0 TB/s, with
// only h used 4.6 to 5.0, of rms_norm 3.9 (1024), 4.3 and 4.6 (8192).
// A row stays in its team's registers between the sums over it and their
// use, the next row's loads are issued before them, and the weights are read
// once for all rows of a team.  The sums over rows (dpre, dpost, dg) stay in
// registers too, over a slice of rows for each workgroup, and are joined by a
// second small kernel in a fixed order: no atomics, the same result in every
// run.  All sums and products are in fp32; y and h are rounded once, and h
// is taken from y before its rounding.  The backward pass reads x and o, which
// costs what reading y and o would, and computes y again: from a rounded y
// the weights' fp32 gradients would be no better than the activations' type.
#include <hip/hip_runtime.h>

#include "device_types.h"

namespace baguanet {
namespace {

// Sums of N values over the TPR threads of a row.  `red` must be each of two
// buffers in turn, from call to call, which saves the second barrier: a buffer
// is written again only after the barrier of the other.
template <int TPR, int N>
__device__ inline void row_sums(float (&v)[N], float* red) {
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = wave_sum(v[i]);
  if constexpr (TPR > kWave) {
    constexpr int kWaves = TPR / kWave;
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) {
#pragma unroll
      for (int i = 0; i < N; i++) red[i * kWaves + wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; w++) s += red[i * kWaves + w];
      v[i] = s;
    }
  }
}

template <int TPR>
constexpr int block_of() {
  return TPR <= kWave ? 256 : TPR;
}

// The team of a thread: its wave where that is a team, as a uniform number.
template <int TPR>
__device__ inline int team_of() {
  if constexpr (TPR > kWave) return 0;
  return __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
}

template <typename T, int TPR, int VPT, bool kTiny>
__global__ __launch_bounds__(block_of<TPR>()) void norm_forward_kernel(
    NormFwd a) {
  constexpr int kTeams = block_of<TPR>() / TPR;
  __shared__ float red[2][TPR / kWave];
  const int lane = threadIdx.x % TPR, team = team_of<TPR>();
  const int64_t step = (int64_t)gridDim.x * kTeams;
  const float inv_dim = 1.f / (float)a.dim;
  Cols<kTiny> c[VPT];
  float8 coef[VPT], pre[VPT];  // bs * post, and the group's gate if it is one
  const bool fixed_gate = a.gmode == Gate::kGroup && a.group_rows >= a.rows;
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    c[j] = Cols<kTiny>((j * TPR + lane) * kVec, (int)a.dim);
    coef[j] = a.branch_scale;
    pre[j] = 1.f;
    if (a.post) coef[j] *= c[j].template weight<T>(a.post, a.post32, 0);
    if (a.pre) pre[j] = c[j].template weight<T>(a.pre, a.pre32, 0);
    if (fixed_gate) coef[j] *= c[j].template weight<T>(a.gate, a.gate32, 0);
  }
  typename RowVec<T>::type xn[VPT], on[VPT];
  int64_t row = (int64_t)blockIdx.x * kTeams + team;
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      xn[j] = c[j].raw((const T*)a.x + r * a.xstride);
      if (a.branch) on[j] = c[j].raw((const T*)a.branch + r * a.bstride);
    }
  };
  if (row < a.rows) fetch(row);
  int parity = 0;
  for (; row < a.rows; row += step) {
    float8 y[VPT], o[VPT];
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      y[j] = widen(xn[j]) * a.residual_scale;
      if (a.branch) o[j] = widen(on[j]);
    }
    if (row + step < a.rows) fetch(row + step);
    if (a.branch) {
      float ro = 1.f;
      if (a.post) {
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < VPT; j++) s[0] += c[j].sum(o[j] * o[j]);
        row_sums<TPR>(s, red[parity]);
        parity ^= 1;
        ro = 1.f / sqrtf(s[0] * inv_dim + a.eps);
        if (lane == 0 && a.rbranch) a.rbranch[row] = ro;
      }
      float g = ro;
      if (a.gmode == Gate::kRow)
        g *= a.gate32 ? ((const float*)a.gate)[row]
                      : (float)((const T*)a.gate)[row];
      int64_t at = -1;  // the row's own vector of gates
      if (a.gmode == Gate::kFull) at = row * a.dim;
      if (a.gmode == Gate::kGroup && !fixed_gate)
        at = (int64_t)((uint32_t)row / (uint32_t)a.group_rows) * a.dim;
#pragma unroll
      for (int j = 0; j < VPT; j++) {
        float8 k = coef[j] * g;
        if (at >= 0) k *= c[j].template weight<T>(a.gate, a.gate32, at);
        y[j] += k * o[j];
        if (c[j].own()) c[j].store((T*)a.y + row * a.dim, y[j]);
      }
    }
    if (a.h) {
      float s[1] = {0.f};
#pragma unroll
      for (int j = 0; j < VPT; j++) s[0] += c[j].sum(y[j] * y[j]);
      row_sums<TPR>(s, red[parity]);
      parity ^= 1;
      const float ry = 1.f / sqrtf(s[0] * inv_dim + a.eps);
      if (lane == 0 && a.ry) a.ry[row] = ry;
#pragma unroll
      for (int j = 0; j < VPT; j++)
        if (c[j].own())
          c[j].store((T*)a.h + row * a.dim, y[j] * ry * pre[j]);
    }
  }
}

// How the backward pass cuts the rows: `blocks` workgroups, each with
// `per_block` whole groups of rows, or with one of `slices` parts of one.
struct Cut {
  int64_t groups, group_rows, per_block, slices, slice_rows, blocks;
};

// Parts of the workspace, [blocks, dim] fp32 each: dpre's sums, those of
// dpost (the sum of dY * no where all rows share one gate or have none, else
// gate times that), and a group's sum of dY * no where it has several slices.
struct Parts {
  float *pre, *post, *group;
};

// kWhole: the whole seam (branch with its norm, both gradients, a gate of
// groups or none), as between two blocks of a network that norms both a
// block's input and its result; kRows: the same with a gate for each row.  kAny
// is the rest: rms_norm, networks without the norm of results, the last block,
// whose y nothing follows, a gate for each element.  Left to the arguments,
// these choices cost registers, and with them waves in flight, and tests at
// each use: 30000 rows of 2048 columns with a gate per row took 185 us as kAny
// and take 165 as kRows.
enum class Seam { kAny, kWhole, kRows };

template <typename T, int TPR, int VPT, bool kTiny, Seam kind>
__global__ __launch_bounds__(block_of<TPR>()) void norm_backward_kernel(
    NormBwd a, Cut cut, Parts parts) {
  constexpr int kTeams = block_of<TPR>() / TPR;
  __shared__ float red[2][3 * (TPR / kWave)];
  // the teams' column sums on their way to the first team
  __shared__ __attribute__((aligned(alignof(float8)))) float
      joint[kTeams > 1 ? kTeams - 1 : 1][kTeams > 1 ? TPR * VPT * kVec : 1];
  // wide rows: sums over rows that registers have no room for, for each lane
  constexpr bool kWide = TPR * VPT > 1024;
  __shared__ __attribute__((aligned(alignof(float8)))) float
      held[kWide ? 2 * TPR * VPT * kVec : 1];
  constexpr bool kSeam = kind != Seam::kAny;
  const bool has_branch = kSeam || a.branch, has_post = kSeam || a.post;
  const bool has_dy = kSeam || a.dy, has_dh = kSeam || a.dh;
  const bool full = !kSeam && a.gmode == Gate::kFull;
  const bool per_row =
      kind == Seam::kRows || (!kSeam && a.gmode == Gate::kRow);
  const bool grouped =
      kind != Seam::kRows &&
      (kSeam ? a.gmode != Gate::kNone : a.gmode == Gate::kGroup);
  const bool one_gate = grouped && cut.groups == 1;
  const int lane = threadIdx.x % TPR, team = team_of<TPR>();
  const float inv_dim = 1.f / (float)a.dim;
  Cols<kTiny> c[VPT];
  // pre, and bs * post * gate (without the gate of a row or an element);
  // wide rows read them again at each use
  float8 pre[VPT], coef[VPT], acc_pre[VPT], acc_post[VPT];
  auto held_at = [&](int what, int j) -> float8& {
    return *(float8*)&held[((what * VPT + j) * TPR + lane) * kVec];
  };
  auto add_pre = [&](int j, float8 v) {
    if constexpr (kWide)
      held_at(0, j) += v;
    else
      acc_pre[j] += v;
  };
  auto add_post = [&](int j, float8 v) {
    if constexpr (kWide)
      held_at(1, j) += v;
    else
      acc_post[j] += v;
  };
  auto post_at = [&](int j) {
    return has_post ? c[j].template weight<T>(a.post, a.post32, 0)
                    : (float8)1.f;
  };
  auto pre_at = [&](int j) {
    return a.pre ? c[j].template weight<T>(a.pre, a.pre32, 0) : (float8)1.f;
  };
  auto gate_at = [&](int j, int64_t at) {
    return c[j].template weight<T>(a.gate, a.gate32, at);
  };
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    c[j] = Cols<kTiny>((j * TPR + lane) * kVec, (int)a.dim);
    if constexpr (!kWide) pre[j] = pre_at(j);
    if constexpr (kWide)
      held_at(0, j) = held_at(1, j) = 0.f;
    else
      acc_pre[j] = acc_post[j] = 0.f;
  }
  // Adds the teams' sums up in the first team, in the order of the teams.
  auto join = [&](float8 (&v)[VPT]) {
    if constexpr (kTeams > 1) {
      __syncthreads();
      if (team > 0) {
#pragma unroll
        for (int j = 0; j < VPT; j++)
          *(float8*)&joint[team - 1][(j * TPR + lane) * kVec] = v[j];
      }
      __syncthreads();
      if (team == 0) {
        for (int t = 0; t < kTeams - 1; t++) {
#pragma unroll
          for (int j = 0; j < VPT; j++)
            v[j] += *(const float8*)&joint[t][(j * TPR + lane) * kVec];
        }
      }
    }
  };

  auto take = [&](int what, float8 (&v)[VPT]) {
#pragma unroll
    for (int j = 0; j < VPT; j++)
      if constexpr (kWide) v[j] = held_at(what, j);
  };

  const int64_t slice = blockIdx.x % cut.slices;
  const int64_t g0 = blockIdx.x / cut.slices * cut.per_block;
  const int64_t g1 =
      g0 + cut.per_block < cut.groups ? g0 + cut.per_block : cut.groups;
  int parity = 0;
  for (int64_t grp = g0; grp < g1; grp++) {
    const int64_t first = grp * cut.group_rows + slice * cut.slice_rows;
    int64_t last = first + cut.slice_rows;
    if (last > (grp + 1) * cut.group_rows) last = (grp + 1) * cut.group_rows;
    if (last > a.rows) last = a.rows;
    auto coef_at = [&](int j) {
      float8 v = post_at(j) * a.branch_scale;
      if (grouped) v *= gate_at(j, grp * a.dim);
      return v;
    };
    if constexpr (!kWide) {
#pragma unroll
      for (int j = 0; j < VPT; j++) coef[j] = coef_at(j);
    }
    typename RowVec<T>::type xn[VPT], on[VPT], dyn[VPT], dhn[VPT];
    float ro_n = 1.f, ry_n = 0.f, g_n = 1.f;
    auto fetch = [&](int64_t r) {
#pragma unroll
      for (int j = 0; j < VPT; j++) {
        if (has_dh) {
          xn[j] = c[j].raw((const T*)a.x + r * a.xstride);
          dhn[j] = c[j].raw((const T*)a.dh + r * a.dhstride);
        }
        if (has_dy)
          dyn[j] = c[j].raw((const T*)a.dy + r * a.dystride);
        if (has_branch)
          on[j] = c[j].raw((const T*)a.branch + r * a.bstride);
      }
      if (has_dh) ry_n = a.ry[r];
      if (has_branch && has_post) ro_n = a.rbranch[r];
      if (per_row)
        g_n = a.gate32 ? ((const float*)a.gate)[r]
                       : (float)((const T*)a.gate)[r];
    };
    int64_t row = first + team;
    if (!kWide && row < last) fetch(row);
    for (; row < last; row += kTeams) {
      if (kWide) fetch(row);
      const float ry = ry_n, ro = ro_n, g_row = g_n;
      float8 dY[VPT], no[VPT], ny[VPT];
      // sums: ny * t;  q * (dy + ry * t);  q * ny, with q = coef * no (and an
      // element's gate): the mean that do needs then follows without a second
      // pass over the row.
      float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < VPT; j++) {
        ny[j] = dY[j] = 0.f;
        float8 q;
        if (has_branch) {
          no[j] = widen(on[j]) * ro;
          q = no[j] * (kWide ? coef_at(j) : coef[j]);
          if (full) q *= gate_at(j, row * a.dim);
        }
        if (has_dy) dY[j] = widen(dyn[j]);
        if (has_dh) {
          const float8 dh = widen(dhn[j]);
          float8 y = widen(xn[j]) * a.residual_scale;
          if (has_branch) y += q * g_row;
          ny[j] = y * ry;
          const float8 t = dh * (kWide ? pre_at(j) : pre[j]);
          add_pre(j, dh * ny[j]);
          dY[j] += t * ry;
          s[0] += c[j].sum(ny[j] * t);
        }
        if (has_branch) {
          s[1] += c[j].sum(q * dY[j]);
          s[2] += c[j].sum(q * ny[j]);
        }
      }
      if (!kWide && row + kTeams < last) fetch(row + kTeams);
      row_sums<TPR>(s, red[parity]);
      parity ^= 1;
      const float k0 = ry * s[0] * inv_dim;
      // sum of q * dY, without the row's own gate
      const float sq = s[1] - k0 * s[2];
      const float k1 = sq * g_row * inv_dim;
      if (per_row && a.dgate && lane == 0) {
        if (a.dgate32)
          ((float*)a.dgate)[row] = sq;
        else
          ((T*)a.dgate)[row] = (T)sq;
      }
#pragma unroll
      for (int j = 0; j < VPT; j++) {
        dY[j] -= ny[j] * k0;
        if (c[j].own())
          c[j].store((T*)a.dx + row * a.dim, dY[j] * a.residual_scale);
        if (has_branch) {
          float8 e = dY[j] * no[j];
          const float8 k = kWide ? coef_at(j) : coef[j];
          float8 du = dY[j] * k * g_row;
          if (full) {
            const float8 g = gate_at(j, row * a.dim);
            if (a.dgate && c[j].own())
              c[j].template put_weight<T>(a.dgate, a.dgate32, row * a.dim,
                                          e * k);
            e *= g;
            du *= g;
          }
          add_post(j, e * g_row);
          if (has_post) du = (du - no[j] * k1) * ro;
          if (c[j].own()) c[j].store((T*)a.dbranch + row * a.dim, du);
        }
      }
    }
    if (grouped && !one_gate) {
      take(1, acc_post);
      // the group's sum of dY * no goes out, and on into dpost's
      join(acc_post);
      if (team == 0) {
#pragma unroll
        for (int j = 0; j < VPT; j++) {
          if (!c[j].own()) continue;
          if (a.dgate && cut.slices == 1)
            c[j].template put_weight<T>(
                a.dgate, a.dgate32, grp * a.dim,
                acc_post[j] * post_at(j) * a.branch_scale);
          if (parts.group)
            c[j].store(parts.group + blockIdx.x * a.dim, acc_post[j]);
          if (parts.post)
            c[j].accumulate(parts.post + blockIdx.x * a.dim,
                            acc_post[j] * gate_at(j, grp * a.dim), grp == g0);
        }
      }
#pragma unroll
      for (int j = 0; j < VPT; j++) {
        if constexpr (kWide)
          held_at(1, j) = 0.f;
        else
          acc_post[j] = 0.f;
      }
    }
  }
  auto put = [&](float* part, const float8 (&v)[VPT]) {
    if (team == 0) {
#pragma unroll
      for (int j = 0; j < VPT; j++)
        if (c[j].own()) c[j].store(part + blockIdx.x * a.dim, v[j]);
    }
  };
  if (parts.pre) {
    take(0, acc_pre);
    join(acc_pre);
    put(parts.pre, acc_pre);
  }
  if (parts.post && !(grouped && !one_gate)) {
    take(1, acc_post);
    join(acc_post);
    put(parts.post, acc_post);
  }
}

// Sums of the workspace's parts over the workgroups, in their order by
// strips: blockIdx.y is a group (dgate) or one of the whole sums.
constexpr int kJoinCols = 64, kJoinStrips = 16;

template <typename T>
__global__ __launch_bounds__(kJoinCols* kJoinStrips) void norm_join_kernel(
    NormBwd a, Cut cut, Parts parts) {
  __shared__ float strip[kJoinStrips][kJoinCols];
  const int c = threadIdx.x % kJoinCols, s = threadIdx.x / kJoinCols;
  const int64_t col = (int64_t)blockIdx.x * kJoinCols + c;
  const int64_t what = blockIdx.y;  // 0: dpre, 1: dpost, 2 + g: dgate
  const float* part = what == 0 ? parts.pre : what == 1 ? parts.post
                                                        : parts.group;
  const int64_t n = what < 2 ? cut.blocks : cut.slices;
  const int64_t first = what < 2 ? 0 : (what - 2) * cut.slices;
  const bool live = part && col < a.dim;
  const int64_t each = (n + kJoinStrips - 1) / kJoinStrips;
  float sum = 0.f;
  if (live) {
    const int64_t end = (s + 1) * each < n ? (s + 1) * each : n;
#pragma unroll 8
    for (int64_t i = s * each; i < end; i++)
      sum += part[(first + i) * a.dim + col];
  }
  strip[s][c] = sum;
  __syncthreads();
  if (s || !live) return;
  sum = 0.f;
  for (int i = 0; i < kJoinStrips; i++) sum += strip[i][c];
  auto put = [&](void* p, bool f32, int64_t i, float v) {
    if (f32)
      ((float*)p)[i] = v;
    else
      ((T*)p)[i] = (T)v;
  };
  auto get = [&](const void* p, bool f32) {
    return f32 ? ((const float*)p)[col] : (float)((const T*)p)[col];
  };
  if (what == 0) {
    put(a.dpre, a.pre32, col, sum);
  } else if (what == 1) {
    sum *= a.branch_scale;
    if (a.gmode == Gate::kGroup && cut.groups == 1) {
      if (a.dgate)
        put(a.dgate, a.dgate32, col,
            sum * (a.post ? get(a.post, a.post32) : 1.f));
      sum *= get(a.gate, a.gate32);
    }
    if (a.dpost) put(a.dpost, a.post32, col, sum);
  } else {
    sum *= a.branch_scale * (a.post ? get(a.post, a.post32) : 1.f);
    put(a.dgate, a.dgate32, (what - 2) * a.dim + col, sum);
  }
}

// out[o, i] = the sum of in[o, r, i] over r, in fp32 and in a fixed order.  A
// team of `cols` by `strips` threads (powers of two) takes `cols` neighbours
// of i; its strips take every so many of the rows of blockIdx.y's slice, and
// their sums are added in pairs.  Bound by HBM: each value is read once.  16 x
// 2048 x 1024 terms of a [2048, 1024] gate take 30 us (4.7 TB/s; 44 with teams
// of 64 columns and 4 strips), 32768 of one value 5 and 5 for its slices.
constexpr int kGateBlock = 256;

struct GateCut {
  int cols, strips;
  int64_t tiles, items;  // of i for one o, and in all
  int64_t slices, slice_rows;
};

template <typename O>
__global__ __launch_bounds__(kGateBlock) void norm_gate_kernel(GateSum a,
                                                               GateCut g,
                                                               O* out) {
  __shared__ float sums[kGateBlock];
  const int team = g.cols * g.strips, teams = kGateBlock / team;
  const int in = threadIdx.x % team, strip = in / g.cols;
  const int64_t r0 = blockIdx.y * g.slice_rows;
  const int64_t r1 = r0 + g.slice_rows < a.rows ? r0 + g.slice_rows : a.rows;
  for (int64_t first = (int64_t)blockIdx.x * teams; first < g.items;
       first += (int64_t)gridDim.x * teams) {
    const int64_t item = first + threadIdx.x / team;
    const int64_t o = item / g.tiles;
    const int64_t i = item % g.tiles * g.cols + in % g.cols;
    const bool live = item < g.items && i < a.inner;
    float sum = 0.f;
    if (live) {
      const float* p = a.in + o * a.rows * a.inner + i;
#pragma unroll 8
      for (int64_t r = r0 + strip; r < r1; r += g.strips)
        sum += p[r * a.inner];
    }
    for (int half = g.strips / 2; half; half /= 2) {
      __syncthreads();
      sums[threadIdx.x] = sum;
      __syncthreads();
      if (strip < half) sum += sums[threadIdx.x + half * g.cols];
    }
    if (live && strip == 0)
      out[(o * g.slices + blockIdx.y) * a.inner + i] = (O)sum;
  }
}

// Slices of the rows where one workgroup for each tile would leave compute
// units idle; a second launch adds the slices' sums.
GateCut cut_gate(const GateSum& a) {
  GateCut g = {1, 1, 1, 0, 1, a.rows};
  // with enough neighbours for the chip a thread adds all rows of one
  const int wide = a.outer * a.inner >= 256 * 2048 ? kGateBlock : kWave;
  while (g.cols < wide && g.cols < a.inner) g.cols *= 2;
  while (g.cols * g.strips < kGateBlock && g.strips < a.rows) g.strips *= 2;
  g.tiles = (a.inner + g.cols - 1) / g.cols;
  g.items = a.outer * g.tiles;
  const int64_t teams = kGateBlock / (g.cols * g.strips);
  const int64_t blocks = (g.items + teams - 1) / teams;
  const int64_t most = (a.rows + g.strips * 16 - 1) / (g.strips * 16);
  const int64_t want = 1024 / (blocks < 1024 ? blocks : 1024);
  g.slices = most < want ? most : want;
  g.slice_rows = (a.rows + g.slices - 1) / g.slices;
  g.slices = (a.rows + g.slice_rows - 1) / g.slice_rows;
  return g;
}

template <typename O>
void launch_gate(const GateSum& a, const GateCut& g, O* out,
                 hipStream_t stream) {
  const int64_t teams = kGateBlock / (g.cols * g.strips);
  const int64_t blocks = (g.items + teams - 1) / teams;
  launch(norm_gate_kernel<O>,
         dim3((uint32_t)(blocks < 65536 ? blocks : 65536), (uint32_t)g.slices),
         kGateBlock, stream, a, g, out);
}

Cut cut_rows(const NormBwd& a) {
  Cut c;
  // 2048 waves at work, or more where a row takes more than four
  const bool pairs = a.dim > 512 && a.dim <= 1024 && a.type != ElemType::kF32;
  const int64_t target = pairs ? 1024 : 512;
  const bool grouped = a.gmode == Gate::kGroup && a.branch;
  c.group_rows = grouped ? a.group_rows : a.rows;
  c.groups = a.rows / c.group_rows;
  if (c.groups >= target) {
    c.per_block = (c.groups + target - 1) / target;
    c.slices = 1;
  } else {
    c.per_block = 1;
    c.slices = target / c.groups;
    // at least 8 rows for a workgroup, or its parts cost more than the rows
    const int64_t most = (c.group_rows + 7) / 8;
    if (c.slices > most) c.slices = most;
  }
  c.slice_rows = (c.group_rows + c.slices - 1) / c.slices;
  c.slices = (c.group_rows + c.slice_rows - 1) / c.slice_rows;
  c.blocks = (c.groups + c.per_block - 1) / c.per_block * c.slices;
  return c;
}

bool wants_post(const NormBwd& a, const Cut& c) {
  return a.branch &&
         (a.dpost || (a.dgate && a.gmode == Gate::kGroup && c.groups == 1));
}

bool wants_group(const NormBwd& a, const Cut& c) {
  return a.branch && a.dgate && a.gmode == Gate::kGroup && c.groups > 1 &&
         c.slices > 1;
}

// Calls f with the team size and vectors per lane that hold `dim` columns.
// kPairs: up to 1024 columns two waves share a row rather than one taking two
// vectors a lane.  That is for 2-byte gradients: 60000 rows of 787 bf16 take
// 139 us so and 160 with one wave, of 1000 fp32 307 and 299; the forward pass
// takes 90 and 77.
template <bool kPairs, typename F>
void with_team(int64_t dim, F&& f) {
  if (dim < kVec)
    f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>(),
      std::true_type());
  else if (dim <= 512)
    f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>(),
      std::false_type());
  else if (dim <= 1024)
    f(std::integral_constant<int, kPairs ? 128 : 64>(),
      std::integral_constant<int, kPairs ? 1 : 2>(), std::false_type());
  else if (dim <= 2048)
    f(std::integral_constant<int, 256>(), std::integral_constant<int, 1>(),
      std::false_type());
  else if (dim <= 4096)
    f(std::integral_constant<int, 512>(), std::integral_constant<int, 1>(),
      std::false_type());
  else if (dim <= 8192)
    f(std::integral_constant<int, 512>(), std::integral_constant<int, 2>(),
      std::false_type());
  else
    f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>(),
      std::false_type());
}

}  // namespace

hipError_t norm_forward(const NormFwd& a, hipStream_t stream) {
  if (a.rows == 0 || a.dim == 0) return hipSuccess;
  if (a.dim > kNormMaxDim) return hipErrorInvalidValue;
  with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    with_team<false>(a.dim, [&](auto tpr, auto vpt, auto tiny) {
      constexpr int kTpr = decltype(tpr)::value, kVpt = decltype(vpt)::value;
      constexpr bool kTiny = decltype(tiny)::value;
      constexpr int kBlk = block_of<kTpr>();
      const int64_t teams = kBlk / kTpr;
      const int64_t want = (a.rows + teams - 1) / teams;
      const int64_t most = 256 * 2048 / kBlk;
      launch(norm_forward_kernel<T, kTpr, kVpt, kTiny>,
             (uint32_t)(want < most ? want : most), kBlk, stream, a);
    });
  });
  return hipGetLastError();
}

size_t norm_workspace(const NormBwd& a) {
  if (a.rows == 0 || a.dim == 0) return 0;
  const Cut c = cut_rows(a);
  const size_t part = (size_t)c.blocks * a.dim * sizeof(float);
  return part * ((a.dpre ? 1 : 0) + (wants_post(a, c) ? 1 : 0) +
                 (wants_group(a, c) ? 1 : 0));
}

hipError_t norm_backward(const NormBwd& a, hipStream_t stream) {
  if (a.rows == 0 || a.dim == 0) return hipSuccess;
  if (a.dim > kNormMaxDim) return hipErrorInvalidValue;
  const Cut c = cut_rows(a);
  const size_t part = (size_t)c.blocks * a.dim;
  float* ws = (float*)a.workspace;
  Parts parts = {};
  if (a.dpre) parts.pre = ws, ws += part;
  if (wants_post(a, c)) parts.post = ws, ws += part;
  if (wants_group(a, c)) parts.group = ws, ws += part;
  with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    with_team<sizeof(T) == 2>(a.dim, [&](auto tpr, auto vpt, auto tiny) {
      constexpr int kTpr = decltype(tpr)::value, kVpt = decltype(vpt)::value;
      constexpr bool kTiny = decltype(tiny)::value;
      const bool whole = a.branch && a.post && a.dy && a.dh;
      const auto kernel =
          !whole || a.gmode == Gate::kFull
              ? norm_backward_kernel<T, kTpr, kVpt, kTiny, Seam::kAny>
          : a.gmode == Gate::kRow
              ? norm_backward_kernel<T, kTpr, kVpt, kTiny, Seam::kRows>
              : norm_backward_kernel<T, kTpr, kVpt, kTiny, Seam::kWhole>;
      launch(kernel, (uint32_t)c.blocks, block_of<kTpr>(), stream, a, c, parts);
    });
    if (parts.pre || parts.post || parts.group) {
      const dim3 grid((uint32_t)((a.dim + kJoinCols - 1) / kJoinCols),
                      (uint32_t)(2 + (parts.group ? c.groups : 0)));
      launch(norm_join_kernel<T>, grid, kJoinCols * kJoinStrips, stream, a, c,
             parts);
    }
  });
  return hipGetLastError();
}

size_t norm_gate_workspace(const GateSum& a) {
  if (a.outer == 0 || a.rows == 0 || a.inner == 0) return 0;
  const GateCut g = cut_gate(a);
  return g.slices > 1 ? (size_t)(a.outer * g.slices * a.inner) * sizeof(float)
                      : 0;
}

hipError_t norm_gate_sum(const GateSum& a, hipStream_t stream) {
  if (a.outer == 0 || a.rows == 0 || a.inner == 0) return hipSuccess;
  GateSum last = a;
  GateCut g = cut_gate(a);
  if (g.slices > 1) {
    launch_gate(a, g, a.workspace, stream);
    last.in = a.workspace;
    last.rows = g.slices;
    g = cut_gate(last);
    g.slices = 1;
    g.slice_rows = last.rows;
  }
  with_type(a.type, [&](auto* t) {
    using O = std::remove_pointer_t<decltype(t)>;
    launch_gate(last, g, (O*)a.out, stream);
  });
  return hipGetLastError();
}

}  // namespace baguanet
