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
//
// 65536 tokens, 18600 of them different and a tenth padding, a table of 131072 x
// 4096 bf16: lookup 150 us (690 MB, each row read once: 4.6 TB/s), gradient 369
// us (1.56 GB, 4.2 TB/s), of which the sort with the zeroing of dW (1.07 GB)
// beside it takes 178, the sums 177 and the join of runs 14.  A large copy moves
// 5.0 TB/s, a fill 6.8.
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
    for (int64_t c = (int64_t)lane * kVec; c < a.dim;
         c += (int64_t)tpr * kVec) {
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
// costs at most what reading their gradients does.  (Looking up which rows have
// no token, by binary search, and zeroing those together with the sums made
// it 195 us for lookup and gradient where this made it 135: a table of 50000 x
// 2048 bf16, 16384 tokens.)

__device__ inline int32_t sort_key(const EmbeddingBwd& a, int64_t i) {
  const int64_t t = read_token(a.tokens, i, a.tok64);
  return (int32_t)(t >= 0 && t < a.vocab && t != a.padding ? t : a.vocab);
}

struct Sorted {
  int32_t *key, *pos;
};

// The chunks where a run starts that crosses chunk borders (see below), in any
// order, and how many there are.  The sort sets the number to 0.
struct Starts {
  int32_t *count, *chunk;
};

// A launch's part of the bytes to zero, in 16-byte pieces; the workgroups from
// `first` on do it.  The last part takes the rest of fewer than 16 bytes.
struct Zero {
  void* p;
  int64_t begin, end, rest;
  uint32_t first;
};

constexpr int kZeroPieces = 4;  // of 16 bytes, for each thread

template <int kThreads>
__device__ inline bool zero_part(const Zero& z) {
  if (blockIdx.x < z.first) return false;
  const int64_t block = blockIdx.x - z.first;
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < kZeroPieces; j++) {
    const int64_t i =
        z.begin + (block * kZeroPieces + j) * kThreads + threadIdx.x;
    if (i < z.end) ((uint4*)z.p)[i] = zero;
  }
  if (block == 0 && threadIdx.x < z.rest)
    ((uint16_t*)z.p)[z.end * 8 + threadIdx.x] = 0;
  return true;
}

// Few tokens: an element's place is the number of those before it in the
// order, and these are counted directly.  64 elements to a workgroup, one to a
// lane; its 16 waves count them against every 16th run of 64 others, which
// pass through the lanes' registers: 8 us for 2048 tokens and 21 for 8192,
// where the four launches of a radix sort take 17 and 19.  The table is zeroed
// beside this one launch, which starts less than four do.  Lookup and gradient
// of 2048 and 8192 tokens in us, counted and by radix: 44, 52 and 68, 79 for
// 50000 x 2048 bf16; 33, 45 and 45, 52 for 131072 x 512; 27, 32 and 51, 48 for
// 20011 x 1001; 19, 20 and 36, 24 for 1000 x 64, which is small enough that
// only the sort counts.
constexpr int kRankBlock = 1024;
constexpr int kRankWaves = kRankBlock / kWave;

__global__ __launch_bounds__(kRankBlock) void sort_rank_kernel(EmbeddingBwd a,
                                                               Sorted out,
                                                               Starts starts,
                                                               Zero z) {
  if (zero_part<kRankBlock>(z)) return;
  if (blockIdx.x == 0 && threadIdx.x == 0) *starts.count = 0;
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
// digits of every tile of tokens and places the tile's elements in order.
// The tiles are cut so that there are at most 64, or 128 from 131072 tokens on
// and 256 from 524288 on: each of them then adds up the counts of all for
// itself, and their scan needs no launch of its own.  (262144 tokens of 50000 x
// 512: gradient 189 us with 64 and 173 with 128; 1000000 of 131072 x 64: 437
// with 64, 354 with 128 and 327 with 256.)
constexpr int kSortBlock = 256;
constexpr int kSortWaves = kSortBlock / kWave;
constexpr int kMaxBits = 10;         // of a digit: 1024 counters
constexpr int64_t kMaxTiles = 256;

struct Tiles {
  int64_t size, count;  // elements of a tile, a multiple of kSortBlock
};

__device__ inline int32_t pass_key(const EmbeddingBwd& a, const Sorted& in,
                                   int64_t i) {
  return in.key ? in.key[i] : sort_key(a, i);
}

// counts: [tiles, digits]
__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(
    EmbeddingBwd a, Sorted in, int shift, int bits, Tiles tiles,
    uint32_t* counts, Zero z) {
  if (zero_part<kSortBlock>(z)) return;
  __shared__ uint32_t hist[1 << kMaxBits];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += kSortBlock) hist[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * tiles.size;
#pragma unroll 4
  for (int64_t j = threadIdx.x; j < tiles.size; j += kSortBlock)
    if (base + j < a.n)
      atomicAdd(&hist[(pass_key(a, in, base + j) >> shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortBlock)
    counts[(int64_t)blockIdx.x * bins + b] = hist[b];
}

// The sum of v over the threads before this one.
template <int kThreads>
__device__ inline uint32_t block_scan(uint32_t v, uint32_t* wave_total) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  uint32_t incl = v;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t up = __shfl_up(incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == kWave - 1) wave_total[wave] = incl;
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / kWave; w++)
    if (w < wave) before += wave_total[w];
  return before + incl - v;
}

__global__ __launch_bounds__(kSortBlock) void sort_place_kernel(
    EmbeddingBwd a, Sorted in, Sorted out, int shift, int bits, Tiles tiles,
    const uint32_t* counts, Starts starts, Zero z) {
  if (zero_part<kSortBlock>(z)) return;
  if (blockIdx.x == 0 && threadIdx.x == 0) *starts.count = 0;
  // next[w][d]: where wave w places its next element of digit d
  __shared__ uint32_t next[kSortWaves][1 << kMaxBits];
  __shared__ uint32_t wave_total[kSortWaves];
  const int bins = 1 << bits;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (int b = threadIdx.x; b < bins * kSortWaves; b += kSortBlock)
    next[b / bins][b % bins] = 0;
  __syncthreads();
  const int64_t own = tiles.size / kSortWaves;
  const int64_t base = (int64_t)blockIdx.x * tiles.size + wave * own;
#pragma unroll 4
  for (int64_t j = lane; j < own; j += kWave)
    if (base + j < a.n)
      atomicAdd(
          &next[wave][(pass_key(a, in, base + j) >> shift) & (bins - 1)], 1u);
  __syncthreads();
  // a thread takes four digits: those of the tiles before, and of all
  const int b = threadIdx.x * 4;
  uint4 mine = make_uint4(0, 0, 0, 0), whole = mine;
  if (b < bins) {
    // 16 loads at a time: one by one they would wait for each other
    constexpr int kLoads = 16;
    const int count = (int)tiles.count;
    for (int t0 = 0; t0 < count; t0 += kLoads) {
      uint4 c[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const int t = t0 + i < count ? t0 + i : count - 1;
        c[i] = *(const uint4*)&counts[t * bins + b];
      }
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const uint32_t in_all = t0 + i < count ? ~0u : 0u;
        const uint32_t in_mine = t0 + i < (int)blockIdx.x ? ~0u : 0u;
        whole.x += c[i].x & in_all, mine.x += c[i].x & in_mine;
        whole.y += c[i].y & in_all, mine.y += c[i].y & in_mine;
        whole.z += c[i].z & in_all, mine.z += c[i].z & in_mine;
        whole.w += c[i].w & in_all, mine.w += c[i].w & in_mine;
      }
    }
  }
  const uint32_t before = block_scan<kSortBlock>(
      whole.x + whole.y + whole.z + whole.w, wave_total);
  if (b < bins) {
    uint32_t run[4] = {before + mine.x, before + whole.x + mine.y,
                       before + whole.x + whole.y + mine.z,
                       before + whole.x + whole.y + whole.z + mine.w};
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
      for (int w = 0; w < kSortWaves; w++) {
        const uint32_t c = next[w][b + q];
        next[w][b + q] = run[q];
        run[q] += c;
      }
  }
  __syncthreads();
  // Each wave takes its elements 64 at a time, in order; lanes with the
  // same digit find one another by one ballot for each bit.
  int32_t ahead = base + lane < a.n ? pass_key(a, in, base + lane) : 0;
  for (int64_t j = lane; j < own; j += kWave) {
    const int64_t i = base + j;
    const bool live = i < a.n;
    const int32_t key = ahead;
    const int32_t pos = in.pos && live ? in.pos[i] : (int32_t)i;
    const int64_t after = i + kWave;
    if (j + kWave < own && after < a.n) ahead = pass_key(a, in, after);
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
      out.pos[at] = pos;
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

struct Chunks {
  int64_t size, count;  // positions of a chunk, and chunks
  int64_t tiles;        // of columns
  int tpr;
};

// The team's chunk, or false past the last, and the lane's columns: from `at`
// on, as an offset of its own, so that a row may have any length.  Lanes at
// and behind the row's end move back into it and write what their neighbours
// write.
template <bool kTiny>
__device__ inline bool pick_chunk(const EmbeddingBwd& a, const Chunks& ch,
                                  int64_t& chunk, int64_t& at,
                                  Cols<kTiny>& c) {
  const int lane = threadIdx.x % ch.tpr;
  const int64_t item =
      (int64_t)blockIdx.x * (kBlock / ch.tpr) + threadIdx.x / ch.tpr;
  chunk = item / ch.tiles;
  at = ((item % ch.tiles) * ch.tpr + lane) * kVec;
  if (kTiny)
    at = 0;
  else if (at + kVec > a.dim)
    at = a.dim - kVec;
  c = Cols<kTiny>(0, kTiny ? (int)a.dim : kVec);
  return chunk < ch.count;
}

template <typename D, typename W, bool kTiny>
__global__ __launch_bounds__(kBlock) void embedding_sum_kernel(
    EmbeddingBwd a, Sorted s, Chunks ch, Starts starts, float* partial) {
  int64_t chunk, at;
  Cols<kTiny> c;
  if (!pick_chunk(a, ch, chunk, at, c)) return;
  const int64_t p0 = chunk * ch.size;
  const int64_t p1 = p0 + ch.size < a.n ? p0 + ch.size : a.n;
  const int32_t before = p0 ? s.key[p0 - 1] : -1;
  const int32_t after = p1 < a.n ? s.key[p1] : -1;
  const D* dout = (const D*)a.dout + at;

  // Four rows in flight for each lane: with 8 or 16 the registers they take
  // leave fewer waves (187, 204 and 456 us at 65536 rows of 4096 bf16).
  constexpr int kAhead = 4;
  float8 acc = 0.f;
  int32_t run = s.key[p0];
  bool head = run == before;  // the run now summed began in a chunk before
  auto flush = [&](bool tail) {
    if (run >= a.vocab) return;
    if (head || tail)
      c.store(partial + (chunk * 2 + (head ? 0 : 1)) * a.dim + at, acc);
    else
      c.store((W*)a.dweight + (int64_t)run * a.dim + at, acc * a.scale);
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
      if (key[j] != run) {
        flush(false);
        run = key[j];
        head = false;
        acc = 0.f;
      }
      acc += widen(row[j]);
    }
  }
  flush(run == after);
  if (run == after && run < a.vocab && !head && at == 0)
    starts.chunk[atomicAdd(starts.count, 1)] = (int32_t)chunk;
}

// The runs that cross chunk borders, for each a tile of columns at a time.  A
// workgroup sums one from its parts: its threads look for the run's end
// together, its teams add up every so many of the parts, and the teams' sums
// are added in their order.  Teams have 128 lanes at most, so that the hundreds
// of parts of the most frequent token are shared by four (18 us with 256
// lanes, 13 with 128: 50000 x 2048 bf16, 16384 tokens).
//
// kMany: for many runs, most of a few parts.  A wave sums one of those alone
// and adds its teams' sums pairwise, and the workgroup follows with the
// others: 140 us without this and 60 with it at 1000000 tokens of 131072 x 64,
// but 10 and 15 at 65536 tokens of 1000 x 64.
constexpr int kJoinBlock = 512, kJoinBlocks = 1024;

template <typename W, bool kTiny, bool kMany>
__global__ __launch_bounds__(kJoinBlock) void embedding_join_kernel(
    EmbeddingBwd a, Sorted s, Chunks ch, Starts starts, const float* partial) {
  constexpr int kWaves = kJoinBlock / kWave, kRuns = kMany ? kWaves : 1;
  constexpr int kLanes = kMany ? kWave : 128;
  __shared__ int wave_end[kWaves], many[kRuns];
  __shared__ __attribute__((aligned(alignof(float8)))) float
      joint[kJoinBlock * kVec];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int tpr = ch.tpr < kLanes ? ch.tpr : kLanes;
  const int team = threadIdx.x / tpr, in = threadIdx.x % tpr;
  const int teams = kJoinBlock / tpr;
  const int64_t tiles = (a.dim + tpr * kVec - 1) / (tpr * kVec);
  const int64_t runs = *starts.count, items = runs * tiles;
  const Cols<kTiny> c(0, kTiny ? (int)a.dim : kVec);
  // every `of`-th of the parts from `first` on
  auto add_parts = [&](int64_t chunk, int64_t parts, int64_t at, int first,
                       int of) {
    constexpr int kAhead = 8;
    float8 acc = 0.f;
    for (int64_t j = first; j < parts; j += of * kAhead) {
      float8 part[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        const int64_t k = j + i * of;  // part 0 is in slot 1
        part[i] = 0.f;
        if (k < parts)
          part[i] =
              c.load(partial + ((chunk + k) * 2 + (k ? 0 : 1)) * a.dim + at);
      }
#pragma unroll
      for (int i = 0; i < kAhead; i++) acc += part[i];
    }
    return acc;
  };
  for (int64_t base = (int64_t)blockIdx.x * kRuns; base < items;
       base += (int64_t)gridDim.x * kRuns) {
    // with kMany a run's tiles are far apart, so that no workgroup has many
    // long ones
    auto find = [&](int64_t item, int64_t& chunk, int32_t& key, int64_t& at) {
      chunk = starts.chunk[kMany ? item % runs : item / tiles];
      key = s.key[(chunk + 1) * ch.size - 1];
      at = ((kMany ? item / runs : item % tiles) * tpr + in) * kVec;
      if (kTiny)
        at = 0;
      else if (at + kVec > a.dim)
        at = a.dim - kVec;
    };
    int64_t chunk, at;
    int32_t key;
    if constexpr (kMany) {
      bool more = false;
      if (base + wave < items) {
        find(base + wave, chunk, key, at);
        const int few = 16 * kWave / tpr < kWave ? 16 * kWave / tpr : kWave;
        // chunks that begin with the key hold a part in slot 0
        const int64_t q = chunk + 1 + lane;
        const uint64_t differ =
            __ballot(q >= ch.count || s.key[q * ch.size] != key);
        const int parts = differ ? __ffsll((long long)differ) : kWave + 1;
        more = parts > few;
        if (!more) {
          float8 acc = add_parts(chunk, parts, at, lane / tpr, kWave / tpr);
          for (int o = tpr; o < kWave; o <<= 1)
#pragma unroll
            for (int i = 0; i < kVec; i++) acc[i] += __shfl_xor(acc[i], o);
          if (lane < tpr)
            c.store((W*)a.dweight + (int64_t)key * a.dim + at, acc * a.scale);
        }
      }
      if (lane == 0) many[wave] = more;
      __syncthreads();
    }
    for (int w = 0; w < kRuns; w++) {
      if (kMany && !many[w]) continue;
      find(base + w, chunk, key, at);
      int64_t parts = 1;
      for (bool on = true; on;) {
        const int64_t q = chunk + parts + threadIdx.x;
        const uint64_t differ =
            __ballot(q >= ch.count || s.key[q * ch.size] != key);
        if (lane == 0)
          wave_end[wave] = differ ? __ffsll((long long)differ) - 1 : kWave;
        __syncthreads();
        for (int v = 0; on && v < kWaves; v++) {
          parts += wave_end[v];
          on = wave_end[v] == kWave;
        }
        __syncthreads();
      }
      float8 acc = add_parts(chunk, parts, at, team, teams);
      *(float8*)&joint[threadIdx.x * kVec] = acc;
      __syncthreads();
      if (team == 0) {
        const int used = parts < teams ? (int)parts : teams;
        for (int t = 1; t < used; t++)
          acc += *(const float8*)&joint[(t * tpr + in) * kVec];
        c.store((W*)a.dweight + (int64_t)key * a.dim + at, acc * a.scale);
      }
      __syncthreads();
    }
    if (kMany) __syncthreads();  // before `many` is written again
  }
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
  size_t sorted, counts, starts, total;
};

Layout layout(int64_t dim, int64_t n) {
  Layout l;
  l.chunks.tpr = team_size(dim);
  const int64_t width = (int64_t)l.chunks.tpr * kVec;
  l.chunks.tiles = (dim + width - 1) / width;
  // Chunks of 64 positions leave little to join; with fewer tokens or columns
  // they are shorter, so that each compute unit has 2048 lanes at work.
  l.chunks.size = 64;
  while (l.chunks.size > 8 &&
         n * l.chunks.tiles * l.chunks.tpr / l.chunks.size < 256 * 2048)
    l.chunks.size /= 2;
  l.chunks.count = (n + l.chunks.size - 1) / l.chunks.size;
  l.sorted = round256((size_t)n * 4);
  l.counts = round256((kMaxTiles << kMaxBits) * 4);
  l.starts = round256((size_t)(l.chunks.count + 1) * 4);
  l.total = 4 * l.sorted + l.counts + l.starts +
            round256((size_t)l.chunks.count * 2 * (size_t)dim * 4);
  return l;
}

constexpr int64_t kRankMost = 8192;  // tokens that are sorted by counting

// Cuts the zeroing of dW in equal parts over `launches`.
struct Zeroing {
  void* p;
  int64_t bytes;
  int launches;
  Zero part(int i, int64_t first, int threads, uint32_t& grid) const {
    const int64_t pieces = bytes / 16;
    Zero z = {p, pieces * i / launches, pieces * (i + 1) / launches,
              i + 1 == launches ? bytes % 16 / 2 : 0, (uint32_t)first};
    const int64_t each = (int64_t)threads * kZeroPieces;
    const int64_t want = (z.end - z.begin + each - 1) / each;
    grid = (uint32_t)(first + (want < 1 ? 1 : want));
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
  // the largest launches: the sums', and one that zeroes a part of dW
  static_assert(kEmbeddingMaxGrad / (kSortBlock * kZeroPieces * 4) <=
                    kMaxBlocks / 2 + 1,
                "launches that zero a part of dW");
  if (blocks > kMaxBlocks || a.vocab > kEmbeddingMaxGrad / a.dim)
    return hipErrorInvalidValue;
  char* ws = (char*)a.workspace;
  Sorted buf[2];
  buf[0] = {(int32_t*)ws, (int32_t*)(ws + l.sorted)};
  buf[1] = {(int32_t*)(ws + 2 * l.sorted), (int32_t*)(ws + 3 * l.sorted)};
  uint32_t* counts = (uint32_t*)(ws + 4 * l.sorted);
  int32_t* first = (int32_t*)(ws + 4 * l.sorted + l.counts);
  const Starts starts = {first, first + 1};
  float* partial = (float*)(ws + 4 * l.sorted + l.counts + l.starts);

  Zeroing zero = {a.dweight,
                  a.vocab * a.dim * (a.wtype == ElemType::kF32 ? 4 : 2), 1};
  uint32_t grid;
  Sorted sorted = {nullptr, nullptr};
  if (a.n <= kRankMost) {
    const int64_t own = (a.n + kWave - 1) / kWave;
    const Zero z = zero.part(0, own, kRankBlock, grid);
    sorted = buf[0];
    launch(sort_rank_kernel, grid, kRankBlock, stream, a, sorted, starts, z);
  } else {
    const int bits = key_bits(a.vocab);
    const int passes = (bits + kMaxBits - 1) / kMaxBits;
    // at least 4 bits: the placing reads the counts of four digits at once
    const int even = (bits + passes - 1) / passes, digit = even < 4 ? 4 : even;
    Tiles tiles;
    const int64_t most = a.n < 131072 ? 64 : a.n < 524288 ? 128 : kMaxTiles;
    tiles.size = (a.n + most - 1) / most;
    tiles.size = (tiles.size + kSortBlock - 1) / kSortBlock * kSortBlock;
    tiles.count = (a.n + tiles.size - 1) / tiles.size;
    zero.launches = 2 * passes;
    for (int p = 0; p < passes; p++) {
      const Sorted out = buf[p & 1];
      const Zero zc = zero.part(2 * p, tiles.count, kSortBlock, grid);
      launch(sort_count_kernel, grid, kSortBlock, stream, a, sorted, p * digit,
             digit, tiles, counts, zc);
      const Zero zp = zero.part(2 * p + 1, tiles.count, kSortBlock, grid);
      launch(sort_place_kernel, grid, kSortBlock, stream, a, sorted, out,
             p * digit, digit, tiles, (const uint32_t*)counts, starts, zp);
      sorted = out;
    }
  }
  if (a.n == 0) return hipGetLastError();

  // at most as many runs cross borders as there are chunks or tokens to tell
  // apart
  const bool many_runs =
      (ch.count < a.vocab ? ch.count : a.vocab) * ch.tiles > 8192;
  with_type(a.wtype, [&](auto* w) {
    using W = std::remove_pointer_t<decltype(w)>;
    auto sums = [&](auto tiny) {
      constexpr bool kTiny = decltype(tiny)::value;
      with_type(a.dtype, [&](auto* d) {
        using D = std::remove_pointer_t<decltype(d)>;
        launch(embedding_sum_kernel<D, W, kTiny>, (uint32_t)blocks, kBlock,
               stream, a, sorted, ch, starts, partial);
      });
      if (ch.count < 2) return;
      const auto join = many_runs ? embedding_join_kernel<W, kTiny, true>
                                  : embedding_join_kernel<W, kTiny, false>;
      launch(join, kJoinBlocks, kJoinBlock, stream, a, sorted, ch, starts,
             (const float*)partial);
    };
    if (a.dim < kVec)
      sums(std::true_type());
    else
      sums(std::false_type());
  });
  return hipGetLastError();
}

}  // namespace baguanet
