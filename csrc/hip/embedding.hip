// embedding.hip — scaled lookup of table rows and the table's gradient
// (gfx950).
//
//   out[i]  = scale * W[tok[i]]
//   dW[v]   = scale * sum over { i : tok[i] = v, v != padding } of dout[i]
//
// Both are bound by HBM: the lookup reads and writes n rows, the gradient
// reads n rows and writes the whole table.  The gradient's sums run in the
// order of the tokens' positions, so its result is the same in every run:
// positions are first sorted by token (stably), then each row of dW that has
// tokens is summed in fp32 from its run of the sorted positions.  No atomics
// touch a gradient.
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
//
// Sorting keeps few compute units busy and is bound by latency, so its
// launches zero the table's gradient beside it: each takes a part of dW with
// workgroups of its own.  Rows that get a sum are written twice that way, which
// costs at most what reading their gradients does; looking up which rows have
// no token instead (a binary search for each, then zeroing row by row) took
// 120 us where this takes 60, at 50000 x 2048 and 16384 tokens.

__device__ inline int32_t sort_key(const EmbeddingBwd& a, int64_t i) {
  const int64_t t = read_token(a.tokens, i, a.tok64);
  return (int32_t)(t >= 0 && t < a.vocab && t != a.padding ? t : a.vocab);
}

struct Sorted {
  int32_t *key, *pos;
};

// A launch's part of the bytes to zero, in 16-byte pieces; the workgroups from
// `first` on do it.  The last part takes the rest of fewer than 16 bytes.
struct Zero {
  void* p;
  int64_t begin, end, rest;
  uint32_t first;
};

template <int kThreads>
__device__ inline bool zero_part(const Zero& z) {
  if (blockIdx.x < z.first) return false;
  const int64_t id = (int64_t)(blockIdx.x - z.first) * kThreads + threadIdx.x;
  const int64_t step = (int64_t)(gridDim.x - z.first) * kThreads;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int64_t i = z.begin + id; i < z.end; i += step) ((uint4*)z.p)[i] = zero;
  if (id < z.rest) ((uint16_t*)z.p)[z.end * 8 + id] = 0;
  return true;
}

// Few tokens: an element's place is the number of those before it in the
// order, and these are counted directly.  64 elements to a workgroup, one to a
// lane; its 16 waves count them against every 16th run of 64 others, which
// pass through the lanes' registers.  n * n / 64 lane operations: 20 us at
// 16384 tokens, where the passes of a radix sort take 28.
constexpr int kRankBlock = 1024;
constexpr int kRankWaves = kRankBlock / kWave;

__global__ __launch_bounds__(kRankBlock) void sort_rank_kernel(EmbeddingBwd a,
                                                               Sorted out,
                                                               Zero z) {
  if (zero_part<kRankBlock>(z)) return;
  __shared__ int counts[kRankWaves][kWave];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int64_t i = (int64_t)blockIdx.x * kWave + lane;
  const int32_t key = i < a.n ? sort_key(a, i) : 0;
  const int runs = (int)((a.n + kWave - 1) / kWave);
  int count = 0;
  for (int r = wave; r < runs; r += kRankWaves) {
    const int64_t j = (int64_t)r * kWave + lane;
    const int32_t other = j < a.n ? sort_key(a, j) : INT32_MAX;
    // equal keys count where they come first
    const int32_t limit = key + (r < (int)blockIdx.x ? 1 : 0);
    if (r == (int)blockIdx.x) {
#pragma unroll 16
      for (int l = 0; l < kWave; l++)
        count += __builtin_amdgcn_readlane(other, l) < key + (l < lane) ? 1 : 0;
    } else {
#pragma unroll 16
      for (int l = 0; l < kWave; l++)
        count += __builtin_amdgcn_readlane(other, l) < limit ? 1 : 0;
    }
  }
  counts[wave][lane] = count;
  __syncthreads();
  if (wave || i >= a.n) return;
  count = 0;
#pragma unroll
  for (int w = 0; w < kRankWaves; w++) count += counts[w][lane];
  out.key[count] = key;
  out.pos[count] = (int32_t)i;
}

// More tokens: least-significant-digit radix sort.  Each pass counts the
// digits of every tile of tokens, scans the counts and places the tile's
// elements in order.  With few tiles each of them scans for itself and the
// scan needs no launch.
constexpr int kSortBlock = 256;
constexpr int kSortWaves = kSortBlock / kWave;
constexpr int kTile = 1024;          // elements of a tile
constexpr int kPerWave = kTile / kSortWaves;
constexpr int kMaxBits = 10;         // of a digit: 1024 counters
constexpr int64_t kOwnScan = 128;    // tiles

__device__ inline int32_t pass_key(const EmbeddingBwd& a, const Sorted& in,
                                   int64_t i) {
  return in.key ? in.key[i] : sort_key(a, i);
}

// counts: [tiles, digits]
__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(
    EmbeddingBwd a, Sorted in, int shift, int bits, uint32_t* counts, Zero z) {
  if (zero_part<kSortBlock>(z)) return;
  __shared__ uint32_t hist[1 << kMaxBits];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += kSortBlock) hist[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kTile;
#pragma unroll
  for (int j = threadIdx.x; j < kTile; j += kSortBlock)
    if (base + j < a.n)
      atomicAdd(&hist[(pass_key(a, in, base + j) >> shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortBlock)
    counts[(int64_t)blockIdx.x * bins + b] = hist[b];
}

// The sum of v over the threads before this one, and over all.
template <int kThreads>
__device__ inline uint32_t block_scan(uint32_t v, uint32_t* wave_total,
                                      uint32_t& all) {
  constexpr int kWaves = kThreads / kWave;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  uint32_t incl = v;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t up = __shfl_up(incl, o);
    if (lane >= o) incl += up;
  }
  __syncthreads();
  if (lane == kWave - 1) wave_total[wave] = incl;
  __syncthreads();
  uint32_t before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    if (w < wave) before += wave_total[w];
    all += wave_total[w];
  }
  return before + incl - v;
}

// Where each tile places its first element of each digit, by one workgroup.
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t* counts,
                                                         int64_t tiles,
                                                         int bins) {
  __shared__ uint32_t wave_total[16];
  const int b = threadIdx.x;
  uint32_t total = 0, all;
  if (b < bins)
    for (int64_t t = 0; t < tiles; t++) total += counts[t * bins + b];
  uint32_t run = block_scan<1024>(total, wave_total, all);
  if (b >= bins) return;
  for (int64_t t = 0; t < tiles; t++) {
    const uint32_t c = counts[t * bins + b];
    counts[t * bins + b] = run;
    run += c;
  }
}

__global__ __launch_bounds__(kSortBlock) void sort_place_kernel(
    EmbeddingBwd a, Sorted in, Sorted out, int shift, int bits, int64_t tiles,
    const uint32_t* counts, bool scanned, Zero z) {
  if (zero_part<kSortBlock>(z)) return;
  // next[w][d]: where wave w places its next element of digit d
  __shared__ uint32_t next[kSortWaves][1 << kMaxBits];
  __shared__ uint32_t wave_total[kSortWaves];
  const int bins = 1 << bits;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (int b = threadIdx.x; b < bins * kSortWaves; b += kSortBlock)
    next[b / bins][b % bins] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kTile + wave * kPerWave;
  int32_t keys[kPerWave / kWave];
#pragma unroll
  for (int j = 0; j < kPerWave / kWave; j++) {
    const int64_t i = base + j * kWave + lane;
    keys[j] = i < a.n ? pass_key(a, in, i) : 0;
    if (i < a.n) atomicAdd(&next[wave][(keys[j] >> shift) & (bins - 1)], 1u);
  }
  // bins come four to a thread at most, in order
  const int per = (bins + kSortBlock - 1) / kSortBlock;
  uint32_t first[4], total = 0, all;
#pragma unroll
  for (int q = 0; q < 4; q++) {
    const int b = threadIdx.x * per + q;
    first[q] = 0;
    if (q >= per || b >= bins) continue;
    if (scanned) {
      first[q] = counts[(int64_t)blockIdx.x * bins + b];
    } else {
      uint32_t mine = 0, whole = 0;
#pragma unroll 8
      for (int64_t t = 0; t < tiles; t++) {
        const uint32_t c = counts[t * bins + b];
        whole += c;
        mine += t < (int64_t)blockIdx.x ? c : 0;
      }
      first[q] = total + mine;
      total += whole;
    }
  }
  const uint32_t before = block_scan<kSortBlock>(total, wave_total, all);
#pragma unroll
  for (int q = 0; q < 4; q++) {
    const int b = threadIdx.x * per + q;
    if (q >= per || b >= bins) continue;
    uint32_t run = first[q] + (scanned ? 0 : before);
#pragma unroll
    for (int w = 0; w < kSortWaves; w++) {
      const uint32_t c = next[w][b];
      next[w][b] = run;
      run += c;
    }
  }
  __syncthreads();
  // Each wave takes its elements 64 at a time, in order; lanes with the
  // same digit find one another by one ballot for each bit.
#pragma unroll
  for (int j = 0; j < kPerWave / kWave; j++) {
    const int64_t i = base + j * kWave + lane;
    const bool live = i < a.n;
    const int32_t key = keys[j];
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
// The sorted positions are cut into chunks, one for each team of `tpr` lanes
// and tile of tpr * 8 columns, so the work is even whatever the frequencies.
// A run of one token inside a chunk is summed and written as its row of dW.
// A run that crosses a chunk's border leaves a partial sum in the workspace:
// the part that came from the chunk before in slot 0, one that starts here in
// slot 1; embedding_join_kernel adds these in order.

constexpr int kAhead = 8;      // rows in flight for each lane
constexpr int kJoinAhead = 16;

struct Chunks {
  int64_t size, count;  // positions of a chunk, and chunks
  int64_t tiles;        // of columns
  int tpr;
};

// The team's chunk and this lane's columns; false for those past the end.
template <bool kTiny>
__device__ inline bool pick_chunk(const EmbeddingBwd& a, const Chunks& ch,
                                  int64_t& chunk, int64_t& at,
                                  Cols<kTiny>& c) {
  const int lane = threadIdx.x % ch.tpr;
  const int64_t item =
      (int64_t)blockIdx.x * (kBlock / ch.tpr) + threadIdx.x / ch.tpr;
  chunk = item / ch.tiles;
  at = ((item % ch.tiles) * ch.tpr + lane) * kVec;
  if (chunk >= ch.count || at >= a.dim) return false;
  // columns as an offset into the row, so that a row may have any length
  const int64_t left = a.dim - at;
  c = Cols<kTiny>(0, (int)(left < kVec ? left : kVec));
  if (!kTiny && left < kVec) at = a.dim - kVec, c = Cols<kTiny>(0, kVec);
  return true;
}

template <typename D, typename W, bool kTiny>
__global__ __launch_bounds__(kBlock) void embedding_sum_kernel(
    EmbeddingBwd a, Sorted s, Chunks ch, float* partial) {
  int64_t chunk, at;
  Cols<kTiny> c;
  if (!pick_chunk(a, ch, chunk, at, c)) return;
  const int64_t p0 = chunk * ch.size;
  const int64_t p1 = p0 + ch.size < a.n ? p0 + ch.size : a.n;
  const int32_t before = p0 ? s.key[p0 - 1] : -1;
  const int32_t after = p1 < a.n ? s.key[p1] : -1;
  const D* dout = (const D*)a.dout + at;

  float8 acc = 0.f;
  int32_t cur = s.key[p0];
  bool head = cur == before;  // the run now summed began in a chunk before
  auto flush = [&](bool tail) {
    if (cur >= a.vocab) return;
    if (head || tail)
      c.store(partial + (chunk * 2 + (head ? 0 : 1)) * a.dim + at, acc);
    else
      c.store((W*)a.dweight + (int64_t)cur * a.dim + at, acc * a.scale);
  };
  for (int64_t p = p0; p < p1; p += kAhead) {
    typename RowVec<D>::type row[kAhead];
    int32_t key[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      key[j] = p + j < p1 ? s.key[p + j] : (int32_t)a.vocab;
      row[j] = (D)0.f;
      if (key[j] < a.vocab)
        row[j] = c.raw(dout + (int64_t)s.pos[p + j] * a.dstride);
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (p + j >= p1) break;
      if (key[j] != cur) {
        flush(false);
        cur = key[j];
        head = false;
        acc = widen(row[j]);
      } else {
        acc += widen(row[j]);
      }
    }
  }
  flush(cur == after);
}

// A run that crosses chunk borders, summed from its parts in their order by
// the team of the chunk where it starts.
template <typename W, bool kTiny>
__global__ __launch_bounds__(kBlock) void embedding_join_kernel(
    EmbeddingBwd a, Sorted s, Chunks ch, const float* partial) {
  int64_t chunk, at;
  Cols<kTiny> c;
  if (!pick_chunk(a, ch, chunk, at, c) || chunk + 1 >= ch.count) return;
  const int64_t p1 = (chunk + 1) * ch.size;
  const int32_t key = s.key[p1 - 1];
  if (key >= a.vocab || s.key[p1] != key) return;   // nothing crosses here
  const int64_t p0 = p1 - ch.size;
  if (p0 && s.key[p0] == key && s.key[p0 - 1] == key) return;  // not its start
  float8 acc = c.load(partial + (chunk * 2 + 1) * a.dim + at);
  // chunks that begin with the key hold a part in slot 0
  for (int64_t q = chunk + 1;; q += kJoinAhead) {
    float8 part[kJoinAhead];
    bool more = true;
#pragma unroll
    for (int j = 0; j < kJoinAhead; j++) {
      more = more && q + j < ch.count && s.key[(q + j) * ch.size] == key;
      part[j] = 0.f;
      if (more) part[j] = c.load(partial + (q + j) * 2 * a.dim + at);
    }
#pragma unroll
    for (int j = 0; j < kJoinAhead; j++) acc += part[j];
    if (!more) break;
  }
  c.store((W*)a.dweight + (int64_t)key * a.dim + at, acc * a.scale);
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
  Chunks chunks;
  size_t sorted, counts, total;
};

Layout layout(int64_t dim, int64_t n) {
  Layout l;
  l.chunks.tpr = team_size(dim);
  const int64_t width = (int64_t)l.chunks.tpr * kVec;
  l.chunks.tiles = (dim + width - 1) / width;
  // Chunks of 64 positions leave little to join; with few tokens they are
  // shorter, for about 1024 teams.
  l.chunks.size = 64;
  while (l.chunks.size > 8 && n * l.chunks.tiles / l.chunks.size < 1024)
    l.chunks.size /= 2;
  l.chunks.count = (n + l.chunks.size - 1) / l.chunks.size;
  l.sorted = round256((size_t)n * 4);
  const size_t tiles = (size_t)((n + kTile - 1) / kTile);
  l.counts = round256((tiles << kMaxBits) * 4);
  l.total = 4 * l.sorted + l.counts +
            round256((size_t)l.chunks.count * 2 * (size_t)dim * 4);
  return l;
}

constexpr int64_t kRankMost = 16384;  // tokens that are sorted by counting

// Cuts the zeroing of dW in equal parts over `launches`.
struct Zeroing {
  void* p;
  int64_t bytes;
  int launches;
  Zero part(int i, int64_t first, int threads, uint32_t& grid) const {
    const int64_t pieces = bytes / 16;
    Zero z = {p, pieces * i / launches, pieces * (i + 1) / launches,
              i + 1 == launches ? bytes % 16 / 2 : 0, (uint32_t)first};
    const int64_t want = (z.end - z.begin + threads * 4 - 1) / (threads * 4);
    const int64_t most = 256 * 2048 / threads;
    grid = (uint32_t)(first + (want < 1 ? 1 : want < most ? want : most));
    return z;
  }
};

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
  const Chunks& ch = l.chunks;
  const int64_t teams = kBlock / ch.tpr;
  const int64_t blocks = (ch.count * ch.tiles + teams - 1) / teams;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  char* ws = (char*)a.workspace;
  Sorted buf[2];
  buf[0] = {(int32_t*)ws, (int32_t*)(ws + l.sorted)};
  buf[1] = {(int32_t*)(ws + 2 * l.sorted), (int32_t*)(ws + 3 * l.sorted)};
  uint32_t* counts = (uint32_t*)(ws + 4 * l.sorted);
  float* partial = (float*)(ws + 4 * l.sorted + l.counts);

  Zeroing zero = {a.dweight,
                  a.vocab * a.dim * (a.wtype == ElemType::kF32 ? 4 : 2), 1};
  uint32_t grid;
  Sorted sorted = {nullptr, nullptr};
  if (a.n <= kRankMost) {
    const int64_t own = (a.n + kWave - 1) / kWave;
    const Zero z = zero.part(0, own, kRankBlock, grid);
    sorted = buf[0];
    launch(sort_rank_kernel, grid, kRankBlock, stream, a, sorted, z);
  } else {
    const int bits = key_bits(a.vocab);
    const int passes = (bits + kMaxBits - 1) / kMaxBits;
    const int digit = (bits + passes - 1) / passes;
    const int64_t tiles = (a.n + kTile - 1) / kTile;
    zero.launches = 2 * passes;
    for (int p = 0; p < passes; p++) {
      const Sorted out = buf[p & 1];
      const Zero zc = zero.part(2 * p, tiles, kSortBlock, grid);
      launch(sort_count_kernel, grid, kSortBlock, stream, a, sorted, p * digit,
             digit, counts, zc);
      if (tiles > kOwnScan)
        launch(sort_scan_kernel, 1, 1024, stream, counts, tiles, 1 << digit);
      const Zero zp = zero.part(2 * p + 1, tiles, kSortBlock, grid);
      launch(sort_place_kernel, grid, kSortBlock, stream, a, sorted, out,
             p * digit, digit, tiles, (const uint32_t*)counts,
             tiles > kOwnScan, zp);
      sorted = out;
    }
  }
  if (a.n == 0) return hipGetLastError();

  with_type(a.wtype, [&](auto* w) {
    using W = std::remove_pointer_t<decltype(w)>;
    auto sums = [&](auto tiny) {
      constexpr bool kTiny = decltype(tiny)::value;
      with_type(a.dtype, [&](auto* d) {
        using D = std::remove_pointer_t<decltype(d)>;
        launch(embedding_sum_kernel<D, W, kTiny>, (uint32_t)blocks, kBlock,
               stream, a, sorted, ch, partial);
      });
      if (ch.count > 1)
        launch(embedding_join_kernel<W, kTiny>, (uint32_t)blocks, kBlock,
               stream, a, sorted, ch, (const float*)partial);
    };
    if (a.dim < kVec)
      sums(std::true_type());
    else
      sums(std::false_type());
  });
  return hipGetLastError();
}

}  // namespace baguanet
