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

// Sums of N values over the TPR threads of a row.  `red` is one of two
// buffers used in turn, which saves the second barrier: a buffer is written
// again only after the barrier of the other.
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
  return TPR < 256 ? 256 : TPR;
}

template <typename T, int TPR, int VPT>
__global__ __launch_bounds__(block_of<TPR>()) void norm_forward_kernel(
    NormFwd a) {
  constexpr int kTeams = block_of<TPR>() / TPR;
  __shared__ float red[2][TPR / kWave];
  const int lane = threadIdx.x % TPR, team = threadIdx.x / TPR;
  const int64_t step = (int64_t)gridDim.x * kTeams;
  const float inv_dim = 1.f / (float)a.dim;
  int64_t col[VPT];
  int m[VPT];
  float8 coef[VPT], pre[VPT];  // bs * post, and the group's gate if it is one
  const bool fixed_gate = a.gmode == Gate::kGroup && a.group_rows >= a.rows;
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    col[j] = ((int64_t)j * TPR + lane) * kVec;
    const int64_t left = a.dim - col[j];
    m[j] = left < 0 ? 0 : left < kVec ? (int)left : kVec;
    if (m[j] == 0) col[j] = 0;
    coef[j] = a.branch_scale;
    pre[j] = 1.f;
    if (a.post) coef[j] *= weight_upto<T>(a.post, a.post32, col[j], m[j]);
    if (a.pre) pre[j] = weight_upto<T>(a.pre, a.pre32, col[j], m[j]);
    if (fixed_gate)
      coef[j] *= weight_upto<T>(a.gate, a.gate32, col[j], m[j]);
  }
  typename RowVec<T>::type xn[VPT], on[VPT];
  int64_t row = (int64_t)blockIdx.x * kTeams + team;
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      xn[j] = raw_upto((const T*)a.x + r * a.xstride + col[j], m[j]);
      if (a.branch)
        on[j] = raw_upto((const T*)a.branch + r * a.bstride + col[j], m[j]);
    }
  };
  if (row < a.rows) fetch(row);
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
        for (int j = 0; j < VPT; j++) s[0] += sum8(o[j] * o[j]);
        row_sums<TPR>(s, red[0]);
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
        float8 c = coef[j] * g;
        if (at >= 0) c *= weight_upto<T>(a.gate, a.gate32, at + col[j], m[j]);
        y[j] += c * o[j];
        if (m[j]) store_upto((T*)a.y + row * a.dim + col[j], y[j], m[j]);
      }
    }
    if (a.h) {
      float s[1] = {0.f};
#pragma unroll
      for (int j = 0; j < VPT; j++) s[0] += sum8(y[j] * y[j]);
      row_sums<TPR>(s, red[1]);
      const float ry = 1.f / sqrtf(s[0] * inv_dim + a.eps);
      if (lane == 0 && a.ry) a.ry[row] = ry;
#pragma unroll
      for (int j = 0; j < VPT; j++)
        if (m[j])
          store_upto((T*)a.h + row * a.dim + col[j], y[j] * ry * pre[j], m[j]);
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

template <typename T, int TPR, int VPT>
__global__ __launch_bounds__(block_of<TPR>()) void norm_backward_kernel(
    NormBwd a, Cut cut, Parts parts) {
  constexpr int kTeams = block_of<TPR>() / TPR;
  __shared__ float red[2][3 * (TPR / kWave)];
  // the teams' column sums on their way to the first team
  __shared__ float joint[kTeams > 1 ? kTeams - 1 : 1]
                        [kTeams > 1 ? TPR * VPT * kVec : 1];
  const int lane = threadIdx.x % TPR, team = threadIdx.x / TPR;
  const float inv_dim = 1.f / (float)a.dim;
  const bool grouped = a.gmode == Gate::kGroup;
  const bool one_gate = grouped && cut.groups == 1;
  int64_t col[VPT];
  int m[VPT];
  float8 post[VPT], pre[VPT], gate[VPT];
  float8 acc_pre[VPT], acc_post[VPT], acc_all[VPT];
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    col[j] = ((int64_t)j * TPR + lane) * kVec;
    const int64_t left = a.dim - col[j];
    m[j] = left < 0 ? 0 : left < kVec ? (int)left : kVec;
    if (m[j] == 0) col[j] = 0;
    post[j] = pre[j] = gate[j] = 1.f;
    if (a.post) post[j] = weight_upto<T>(a.post, a.post32, col[j], m[j]);
    if (a.pre) pre[j] = weight_upto<T>(a.pre, a.pre32, col[j], m[j]);
    acc_pre[j] = acc_post[j] = acc_all[j] = 0.f;
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
  auto put = [&](float* part, int64_t at, const float8 (&v)[VPT]) {
    if (team == 0) {
#pragma unroll
      for (int j = 0; j < VPT; j++)
        if (m[j]) store_upto(part + at * a.dim + col[j], v[j], m[j]);
    }
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
    if (grouped) {
#pragma unroll
      for (int j = 0; j < VPT; j++)
        gate[j] = weight_upto<T>(a.gate, a.gate32, grp * a.dim + col[j], m[j]);
    }
    typename RowVec<T>::type xn[VPT], on[VPT], dyn[VPT], dhn[VPT];
    float ro_n = 1.f, ry_n = 0.f, g_n = 1.f;
    auto fetch = [&](int64_t r) {
#pragma unroll
      for (int j = 0; j < VPT; j++) {
        if (a.dh) {
          xn[j] = raw_upto((const T*)a.x + r * a.xstride + col[j], m[j]);
          dhn[j] = raw_upto((const T*)a.dh + r * a.dhstride + col[j], m[j]);
        }
        if (a.dy)
          dyn[j] = raw_upto((const T*)a.dy + r * a.dystride + col[j], m[j]);
        if (a.branch)
          on[j] = raw_upto((const T*)a.branch + r * a.bstride + col[j], m[j]);
      }
      if (a.dh) ry_n = a.ry[r];
      if (a.branch && a.post) ro_n = a.rbranch[r];
      if (a.gmode == Gate::kRow)
        g_n = a.gate32 ? ((const float*)a.gate)[r]
                       : (float)((const T*)a.gate)[r];
    };
    int64_t row = first + team;
    if (row < last) fetch(row);
    for (; row < last; row += kTeams) {
      const float ry = ry_n, ro = ro_n, g_row = g_n;
      float8 dY[VPT], no[VPT], ny[VPT], g[VPT];
      // sums: ny * t;  q * (dy + ry * t);  q * ny, with q = no * post * gate:
      // the mean that do needs then follows without a second pass.
      float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < VPT; j++) {
        ny[j] = dY[j] = 0.f;
        float8 c;
        if (a.branch) {
          no[j] = widen(on[j]) * ro;
          g[j] = gate[j] * g_row;
          if (a.gmode == Gate::kFull)
            g[j] = weight_upto<T>(a.gate, a.gate32, row * a.dim + col[j], m[j]);
          c = no[j] * post[j];
        }
        if (a.dy) dY[j] = widen(dyn[j]);
        if (a.dh) {
          const float8 dh = widen(dhn[j]);
          float8 y = widen(xn[j]) * a.residual_scale;
          if (a.branch) y += c * g[j] * a.branch_scale;
          ny[j] = y * ry;
          const float8 t = dh * pre[j];
          acc_pre[j] += dh * ny[j];
          dY[j] += t * ry;
          s[0] += sum8(ny[j] * t);
        }
        if (a.branch) {
          const float8 q = c * (a.gmode == Gate::kFull ? g[j] : gate[j]);
          s[1] += sum8(q * dY[j]);
          s[2] += sum8(q * ny[j]);
        }
      }
      if (row + kTeams < last) fetch(row + kTeams);
      row_sums<TPR>(s, red[parity]);
      parity ^= 1;
      const float k0 = ry * s[0] * inv_dim;
      // sum of no * post * gate * dY, without the row's own gate
      const float sq = s[1] - k0 * s[2];
      const float k1 = sq * a.branch_scale * g_row * inv_dim;
      if (a.gmode == Gate::kRow && a.dgate && lane == 0) {
        const float dg = sq * a.branch_scale;
        if (a.gate32)
          ((float*)a.dgate)[row] = dg;
        else
          ((T*)a.dgate)[row] = (T)dg;
      }
#pragma unroll
      for (int j = 0; j < VPT; j++) {
        dY[j] -= ny[j] * k0;
        if (m[j])
          store_upto((T*)a.dx + row * a.dim + col[j],
                     dY[j] * a.residual_scale, m[j]);
        if (a.branch) {
          const float8 du = dY[j] * g[j] * a.branch_scale;
          float8 db = du * post[j];
          if (a.post) db = (db - no[j] * k1) * ro;
          if (m[j])
            store_upto((T*)a.dbranch + row * a.dim + col[j], db, m[j]);
          if (a.gmode == Gate::kFull && a.dgate && m[j])
            put_weight_upto<T>(a.dgate, a.gate32, row * a.dim + col[j],
                               dY[j] * no[j] * post[j] * a.branch_scale, m[j]);
          const float8 e = dY[j] * no[j];
          acc_post[j] += grouped ? e : e * g[j];
        }
      }
    }
    if (grouped && !one_gate) {
      // the group's sum goes out, and on into dpost's
      join(acc_post);
      if (team == 0) {
#pragma unroll
        for (int j = 0; j < VPT; j++) {
          if (a.dgate && cut.slices == 1 && m[j])
            put_weight_upto<T>(a.dgate, a.gate32, grp * a.dim + col[j],
                               acc_post[j] * post[j] * a.branch_scale, m[j]);
          acc_all[j] += acc_post[j] * gate[j];
        }
      }
      if (a.dgate && cut.slices > 1) put(parts.group, blockIdx.x, acc_post);
#pragma unroll
      for (int j = 0; j < VPT; j++) acc_post[j] = 0.f;
    }
  }
  if (parts.pre) {
    join(acc_pre);
    put(parts.pre, blockIdx.x, acc_pre);
  }
  if (parts.post) {
    if (grouped && !one_gate) {
      put(parts.post, blockIdx.x, acc_all);
    } else {
      join(acc_post);
      put(parts.post, blockIdx.x, acc_post);
    }
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
        put(a.dgate, a.gate32, col,
            sum * (a.post ? get(a.post, a.post32) : 1.f));
      sum *= get(a.gate, a.gate32);
    }
    if (a.dpost) put(a.dpost, a.post32, col, sum);
  } else {
    sum *= a.branch_scale * (a.post ? get(a.post, a.post32) : 1.f);
    put(a.dgate, a.gate32, (what - 2) * a.dim + col, sum);
  }
}

constexpr int64_t kTargetBlocks = 512;

Cut cut_rows(const NormBwd& a) {
  Cut c;
  const bool grouped = a.gmode == Gate::kGroup && a.branch;
  c.group_rows = grouped ? a.group_rows : a.rows;
  c.groups = a.rows / c.group_rows;
  if (c.groups >= kTargetBlocks) {
    c.per_block = (c.groups + kTargetBlocks - 1) / kTargetBlocks;
    c.slices = 1;
  } else {
    c.per_block = 1;
    c.slices = kTargetBlocks / c.groups;
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
template <typename F>
void with_team(int64_t dim, F&& f) {
  if (dim <= 512)
    f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
  else if (dim <= 1024)
    f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
  else if (dim <= 2048)
    f(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
  else if (dim <= 4096)
    f(std::integral_constant<int, 512>(), std::integral_constant<int, 1>());
  else if (dim <= 8192)
    f(std::integral_constant<int, 1024>(), std::integral_constant<int, 1>());
  else if (dim <= 16384)
    f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
  else
    f(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
}

}  // namespace

hipError_t norm_forward(const NormFwd& a, hipStream_t stream) {
  if (a.rows == 0 || a.dim == 0) return hipSuccess;
  if (a.dim > kNormMaxDim) return hipErrorInvalidValue;
  with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    with_team(a.dim, [&](auto tpr, auto vpt) {
      constexpr int kTpr = decltype(tpr)::value, kVpt = decltype(vpt)::value;
      constexpr int kBlk = block_of<kTpr>();
      const int64_t teams = kBlk / kTpr;
      const int64_t want = (a.rows + teams - 1) / teams;
      const int64_t most = 256 * 2048 / kBlk;
      launch(norm_forward_kernel<T, kTpr, kVpt>, (uint32_t)(want < most ? want : most), kBlk, stream, a);
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
    with_team(a.dim, [&](auto tpr, auto vpt) {
      constexpr int kTpr = decltype(tpr)::value, kVpt = decltype(vpt)::value;
      launch(norm_backward_kernel<T, kTpr, kVpt>, (uint32_t)c.blocks, block_of<kTpr>(), stream, a, c, parts);
    });
    if (parts.pre || parts.post || parts.group) {
      const dim3 grid((uint32_t)((a.dim + kJoinCols - 1) / kJoinCols),
                      (uint32_t)(2 + (parts.group ? c.groups : 0)));
      launch(norm_join_kernel<T>, grid, kJoinCols * kJoinStrips, stream, a, c, parts);
    }
  });
  return hipGetLastError();
}

}  // namespace baguanet
