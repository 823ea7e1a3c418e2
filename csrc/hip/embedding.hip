// embedding.hip — scaled lookup of table rows and the table's gradient
// (gfx950).
//
//   out[i]  = scale * W[tok[i]]
//   dW[v]   = scale * sum over { i : tok[i] = v, v != padding } of dout[i]
//
// Both are bound by HBM: the lookup reads and writes n rows, the gradient
// reads n rows and writes the whole table once.  The gradient's sums run in
// the order of the tokens' positions, so its result is the same in every
// run: positions are first sorted by token (stably), then each row of dW is
// summed in fp32 from its run of the sorted positions and written once;
// rows without a token are written as zeros by other workgroups of the same
// launch.  No atomics touch a gradient.
#include <hip/hip_runtime.h>

#include "device_types.h"

namespace baguanet {
namespace {

constexpr int kBlock = 256;

__device__ inline int64_t read_token(const void* tokens, int64_t i,
                                     bool tok64) {
  return tok64 ? ((const int64_t*)tokens)[i] : ((const int32_t*)tokens)[i];
}

// ---- lookup ---------------------------------------------------------------
// `tpr` lanes (a power of two, at most the block) move one row; a block
// holds kBlock / tpr rows at a time.  A token outside the table reads
// nothing and gives a row of NaN, so that it shows in the loss.

template <typename W, typename O>
__global__ __launch_bounds__(kBlock) void embedding_forward_kernel(
    EmbeddingFwd a, int tpr) {
  const int team = threadIdx.x / tpr, lane = threadIdx.x % tpr;
  const int teams = kBlock / tpr;
  for (int64_t i = (int64_t)blockIdx.x * teams + team; i < a.n;
       i += (int64_t)gridDim.x * teams) {
    const int64_t t = read_token(a.tokens, i, a.tok64);
    const bool ok = t >= 0 && t < a.vocab;
    const W* src = (const W*)a.weight + (ok ? t : 0) * a.wstride;
    O* dst = (O*)a.out + i * a.dim;
    for (int64_t c = (int64_t)lane * kVec; c < a.dim; c += (int64_t)tpr * kVec) {
      const int m = (int)(a.dim - c < kVec ? a.dim - c : kVec);
      float8 v = ok ? load_upto(src + c, m) * a.scale
                    : (float8)__builtin_nanf("");
      store_upto(dst + c, v, m);
    }
  }
}

// ---- sorting positions by token -------------------------------------------
// A token that takes no gradient (padding, or outside the table) sorts last,
// under the key `vocab`.

__device__ inline int32_t sort_key(const EmbeddingBwd& a, int64_t i) {
  const int64_t t = read_token(a.tokens, i, a.tok64);
  return (int32_t)(t >= 0 && t < a.vocab && t != a.padding ? t : a.vocab);
}

struct Sorted {
  int32_t *key, *pos;
};

// Least-significant-digit radix sort: each pass counts the digits of every
// tile of tokens, scans the counts (digit-major) and places the tile's
// elements in order.
constexpr int kSortBlock = 512;
constexpr int kSortWaves = kSortBlock / kWave;
constexpr int kTile = 4096;          // elements of a tile
constexpr int kPerWave = kTile / kSortWaves;
constexpr int kMaxBits = 10;         // of a digit: 1024 counters

__device__ inline int32_t pass_key(const EmbeddingBwd& a, const Sorted& in,
                                   int64_t i) {
  return in.key ? in.key[i] : sort_key(a, i);
}

__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(
    EmbeddingBwd a, Sorted in, int shift, int bits, uint32_t* counts) {
  __shared__ uint32_t hist[1 << kMaxBits];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += kSortBlock) hist[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kTile;
  for (int j = threadIdx.x; j < kTile; j += kSortBlock)
    if (base + j < a.n)
      atomicAdd(&hist[(pass_key(a, in, base + j) >> shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortBlock)
    counts[(int64_t)b * gridDim.x + blockIdx.x] = hist[b];
}

// Exclusive scan of `total` counts by one block.
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t* counts,
                                                         int64_t total) {
  __shared__ uint32_t wave_total[16];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  uint32_t carry = 0;
  for (int64_t base = 0; base < total; base += 4096) {
    const int64_t i = base + (int64_t)threadIdx.x * 4;
    uint32_t v[4], own = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      v[j] = i + j < total ? counts[i + j] : 0;
      own += v[j];
    }
    uint32_t incl = own;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint32_t up = __shfl_up(incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == kWave - 1) wave_total[wave] = incl;
    __syncthreads();
    uint32_t before = carry, all = 0;
    for (int w = 0; w < 16; w++) {
      if (w < wave) before += wave_total[w];
      all += wave_total[w];
    }
    uint32_t run = before + incl - own;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (i + j < total) counts[i + j] = run;
      run += v[j];
    }
    carry += all;
    __syncthreads();
  }
}

__global__ __launch_bounds__(kSortBlock) void sort_place_kernel(
    EmbeddingBwd a, Sorted in, Sorted out, int shift, int bits,
    const uint32_t* counts) {
  // next[w][d]: where wave w places its next element of digit d
  __shared__ uint32_t next[kSortWaves][1 << kMaxBits];
  const int bins = 1 << bits;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (int b = threadIdx.x; b < bins * kSortWaves; b += kSortBlock)
    next[b / bins][b % bins] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kTile + wave * kPerWave;
  for (int j = lane; j < kPerWave; j += kWave)
    if (base + j < a.n)
      atomicAdd(
          &next[wave][(pass_key(a, in, base + j) >> shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortBlock) {
    uint32_t run = counts[(int64_t)b * gridDim.x + blockIdx.x];
    for (int w = 0; w < kSortWaves; w++) {
      const uint32_t c = next[w][b];
      next[w][b] = run;
      run += c;
    }
  }
  __syncthreads();
  // Each wave takes its elements 64 at a time, in order; lanes with the
  // same digit find one another by one ballot for each bit.
  for (int j = 0; j < kPerWave; j += kWave) {
    const int64_t i = base + j + lane;
    const bool live = i < a.n;
    const int32_t key = live ? pass_key(a, in, i) : 0;
    const int digit = (key >> shift) & (bins - 1);
    uint64_t same = __ballot(live);
    for (int b = 0; b < bits; b++) {
      const bool bit = (digit >> b) & 1;
      const uint64_t m = __ballot(bit);
      same &= bit ? m : ~m;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    // a wave's LDS accesses run in program order; the atomics keep the
    // compiler to that order too
    uint32_t at = 0;
    if (live)
      at = __hip_atomic_load(&next[wave][digit], __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_WAVEFRONT);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (live && rank == 0)
      __hip_atomic_store(&next[wave][digit], at + (uint32_t)__popcll(same),
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    at += rank;
    if (live) {
      out.key[at] = key;
      out.pos[at] = in.pos ? in.pos[i] : (int32_t)i;
    }
  }
}

// ---- sums over the sorted positions ---------------------------------------
// The sorted positions are cut into chunks of kChunk, one for each team of
// `tpr` lanes and tile of tpr * 8 columns, so the work is even whatever the
// frequencies.  A run of one token inside a chunk is summed and written as
// its row of dW.  A run that crosses a chunk's border leaves a partial sum
// in the workspace: the part that came from the chunk before in slot 0, one
// that starts here in slot 1; embedding_join_kernel adds these in order.

constexpr int kChunk = 64;
constexpr int kAhead = 8;    // rows in flight for each lane
constexpr int kZeroRows = 64;  // table rows that one zeroing block looks at

template <typename D, typename W>
__global__ __launch_bounds__(kBlock) void embedding_sum_kernel(
    EmbeddingBwd a, Sorted s, float* partial, int tpr, int64_t sum_blocks) {
  if (blockIdx.x >= sum_blocks) {
    // rows without a token: lane r asks for row v0 + r by binary search
    __shared__ uint64_t absent;
    const int64_t v0 = ((int64_t)blockIdx.x - sum_blocks) * kZeroRows;
    if (threadIdx.x < kWave) {
      const int64_t v = v0 + threadIdx.x;
      int64_t lo = 0, hi = a.n;
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (s.key[mid] < v)
          lo = mid + 1;
        else
          hi = mid;
      }
      const bool none = v < a.vocab && (lo == a.n || s.key[lo] != v);
      const uint64_t m = __ballot(none);
      if (threadIdx.x == 0) absent = m;
    }
    __syncthreads();
    const float8 zero = 0.f;
    for (uint64_t m = absent; m; m &= m - 1) {
      W* row = (W*)a.dweight + (v0 + __ffsll((long long)m) - 1) * a.dim;
      for (int64_t c = (int64_t)threadIdx.x * kVec; c < a.dim;
           c += (int64_t)kBlock * kVec)
        store_upto(row + c, zero,
                   (int)(a.dim - c < kVec ? a.dim - c : kVec));
    }
    return;
  }
  const int lane = threadIdx.x % tpr;
  const int64_t width = (int64_t)tpr * kVec;
  const int64_t tiles = (a.dim + width - 1) / width;
  const int64_t chunks = (a.n + kChunk - 1) / kChunk;
  const int64_t item =
      (int64_t)blockIdx.x * (kBlock / tpr) + threadIdx.x / tpr;
  const int64_t chunk = item / tiles;
  const int64_t c = (item % tiles) * width + (int64_t)lane * kVec;
  if (chunk >= chunks || c >= a.dim) return;
  const int m = (int)(a.dim - c < kVec ? a.dim - c : kVec);
  const int64_t p0 = chunk * kChunk;
  const int64_t p1 = p0 + kChunk < a.n ? p0 + kChunk : a.n;
  const int32_t before = p0 ? s.key[p0 - 1] : -1;
  const int32_t after = p1 < a.n ? s.key[p1] : -1;
  const D* dout = (const D*)a.dout + c;

  float8 acc = 0.f;
  int32_t cur = s.key[p0];
  bool head = cur == before;  // the run now summed began in a chunk before
  auto flush = [&](bool tail) {
    if (cur >= a.vocab) return;
    if (head || tail) {
      float* dst = partial + (chunk * 2 + (head ? 0 : 1)) * a.dim + c;
      store_upto(dst, acc, m);
    } else {
      store_upto((W*)a.dweight + (int64_t)cur * a.dim + c, acc * a.scale, m);
    }
  };
  for (int64_t p = p0; p < p1; p += kAhead) {
    float8 row[kAhead];
    int32_t key[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      key[j] = p + j < p1 ? s.key[p + j] : a.vocab;
      row[j] = 0.f;
      if (key[j] < a.vocab)
        row[j] = load_upto(dout + (int64_t)s.pos[p + j] * a.dstride, m);
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (p + j >= p1) break;
      if (key[j] != cur) {
        flush(false);
        cur = key[j];
        head = false;
        acc = row[j];
      } else {
        acc += row[j];
      }
    }
  }
  flush(cur == after);
}

// A run that crosses chunk borders, summed from its parts in their order by
// the team of the chunk where it starts.
template <typename W>
__global__ __launch_bounds__(kBlock) void embedding_join_kernel(
    EmbeddingBwd a, Sorted s, const float* partial, int tpr) {
  const int lane = threadIdx.x % tpr;
  const int64_t width = (int64_t)tpr * kVec;
  const int64_t tiles = (a.dim + width - 1) / width;
  const int64_t chunks = (a.n + kChunk - 1) / kChunk;
  const int64_t item =
      (int64_t)blockIdx.x * (kBlock / tpr) + threadIdx.x / tpr;
  const int64_t chunk = item / tiles;
  const int64_t c = (item % tiles) * width + (int64_t)lane * kVec;
  if (chunk + 1 >= chunks || c >= a.dim) return;
  const int64_t p1 = (chunk + 1) * kChunk;
  const int32_t key = s.key[p1 - 1];
  if (key >= a.vocab || s.key[p1] != key) return;   // nothing crosses here
  const int64_t p0 = p1 - kChunk;
  if (p0 && s.key[p0] == key && s.key[p0 - 1] == key) return;  // not its start
  const int m = (int)(a.dim - c < kVec ? a.dim - c : kVec);
  float8 acc = load_upto(partial + (chunk * 2 + 1) * a.dim + c, m);
  // chunks that begin with the key hold a part in slot 0
  int64_t q = chunk + 1;
  while (true) {
    float8 part[kAhead];
    int count = 0;
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      part[j] = 0.f;
      if (q + j < chunks && s.key[(q + j) * kChunk] == key) {
        part[j] = load_upto(partial + ((q + j) * 2) * a.dim + c, m);
        count++;
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++) acc += part[j];
    if (count < kAhead) break;
    q += kAhead;
  }
  store_upto((W*)a.dweight + (int64_t)key * a.dim + c, acc * a.scale, m);
}

// HIP counts a launch's threads in 32 bits.
constexpr int64_t kMaxBlocks = (int64_t(1) << 32) / kBlock - 1;

int team_size(int64_t dim) {
  int tpr = 1;
  while (tpr < kBlock && (int64_t)tpr * kVec < dim) tpr *= 2;
  return tpr;
}

int key_bits(int64_t vocab) {  // of the largest key, which is `vocab`
  int bits = 1;
  while ((vocab >> bits) != 0) bits++;
  return bits;
}

size_t round256(size_t b) { return (b + 255) & ~size_t(255); }

struct Layout {
  size_t sorted, counts, partial, total;
};

Layout layout(int64_t dim, int64_t n) {
  Layout l;
  l.sorted = round256((size_t)n * 4);
  const size_t tiles = (size_t)((n + kTile - 1) / kTile);
  l.counts = round256((tiles << kMaxBits) * 4);
  const size_t chunks = (size_t)((n + kChunk - 1) / kChunk);
  l.partial = round256(chunks * 2 * (size_t)dim * 4);
  l.total = 4 * l.sorted + l.counts + l.partial;
  return l;
}

}  // namespace

hipError_t embedding_forward(const EmbeddingFwd& a, hipStream_t stream) {
  if (a.n == 0 || a.dim == 0) return hipSuccess;
  const int tpr = team_size(a.dim);
  const int64_t rows = kBlock / tpr;
  const int64_t want = (a.n + rows - 1) / rows;
  const uint32_t grid = (uint32_t)(want < 8192 ? want : 8192);
  with_type(a.wtype, [&](auto* w) {
    using W = std::remove_pointer_t<decltype(w)>;
    with_type(a.otype, [&](auto* o) {
      using O = std::remove_pointer_t<decltype(o)>;
      launch(embedding_forward_kernel<W, O>, grid, kBlock, stream, a, tpr);
    });
  });
  return hipGetLastError();
}

size_t embedding_workspace(int64_t, int64_t dim, int64_t n) {
  return layout(dim, n).total;
}

hipError_t embedding_backward(const EmbeddingBwd& a, hipStream_t stream) {
  if (a.vocab == 0 || a.dim == 0) return hipSuccess;
  const Layout l = layout(a.dim, a.n);
  char* ws = (char*)a.workspace;
  Sorted buf[2];
  buf[0] = {(int32_t*)ws, (int32_t*)(ws + l.sorted)};
  buf[1] = {(int32_t*)(ws + 2 * l.sorted), (int32_t*)(ws + 3 * l.sorted)};
  uint32_t* counts = (uint32_t*)(ws + 4 * l.sorted);
  float* partial = (float*)(ws + 4 * l.sorted + l.counts);

  const int tpr = team_size(a.dim);
  const int64_t width = (int64_t)tpr * kVec;
  const int64_t items =
      ((a.n + kChunk - 1) / kChunk) * ((a.dim + width - 1) / width);
  const int64_t teams = kBlock / tpr;
  const int64_t sum_blocks = (items + teams - 1) / teams;
  const int64_t zero_blocks = (a.vocab + kZeroRows - 1) / kZeroRows;
  if (sum_blocks + zero_blocks > kMaxBlocks) return hipErrorInvalidValue;

  Sorted in = {nullptr, nullptr};
  if (a.n > 0) {
    const int bits = key_bits(a.vocab);
    const int passes = (bits + kMaxBits - 1) / kMaxBits;
    const int digit = (bits + passes - 1) / passes;
    const uint32_t tiles = (uint32_t)((a.n + kTile - 1) / kTile);
    for (int p = 0; p < passes; p++) {
      Sorted out = buf[p & 1];
      launch(sort_count_kernel, tiles, kSortBlock, stream, a, in, p * digit,
                                                          digit, counts);
      launch(sort_scan_kernel, 1, 1024, stream, counts, (int64_t)tiles << digit);
      launch(sort_place_kernel, tiles, kSortBlock, stream, 
          a, in, out, p * digit, digit, counts);
      in = out;
    }
  }

  with_type(a.wtype, [&](auto* w) {
    using W = std::remove_pointer_t<decltype(w)>;
    with_type(a.dtype, [&](auto* d) {
      using D = std::remove_pointer_t<decltype(d)>;
      launch(embedding_sum_kernel<D, W>, (uint32_t)(sum_blocks + zero_blocks), kBlock, stream, 
              a, in, partial, tpr, sum_blocks);
    });
    if (a.n > kChunk)
      launch(embedding_join_kernel<W>, (uint32_t)sum_blocks, kBlock, stream, 
          a, in, partial, tpr);
  });
  return hipGetLastError();
}

}  // namespace baguanet
