// dance_kv_fork, dance_kv_reserve, dance_kv_release and dance_kv_copy
// (include/dance_kv_pages.h): who owns a pool's blocks, and copies of blocks.
//
// The first three are chains of dependent loads over little data (a table, a
// count for each block), so they are bound by latency and by their launches; counts
// change by integer atomics, whose order shows in no result. Measured, kernels alone: fork, reserve and
// release of 32 sequences 3.2, 7.6 and 2.8 us, of 512 of up to 60,000 tokens over 173,005
// blocks 7.1, 11.5 (two launches) and 3.0; a call costs the host 5 to 9 us. Copies run at a large copy's rate: 600 blocks
// of 16 layers (2.6 GB moved) 502 us, 5.1 TB/s; 16 blocks of them 11 us.

#include "../../include/dance_kv_pages.h"
#include "kv_common.h"

namespace dance {
namespace kv {
namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kEntries = 4;  // table entries of a thread
constexpr uint32_t kRun = kThreads * kEntries;

struct Pages {
  int32_t* __restrict__ refs;
  uint32_t blocks, bsh;
};
struct Table {
  int32_t* __restrict__ table;
  int32_t* __restrict__ lengths;
  uint32_t seqs, width;
};

// Sum over the workgroup, in every thread.
__device__ __forceinline__ uint32_t block_sum(uint32_t x, uint32_t* lds) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) x += (uint32_t)__shfl_xor((int)x, i);
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  uint32_t sum = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) sum += lds[w];
  return sum;
}

// ---------------------------------------------------------------- fork

constexpr uint32_t kTogether = 8;  // old rows that a workgroup looks at

// Workgroups of old rows change the counts, by a row's children less one. A thread takes a place of several
// rows: rows that lie together, as beams do, mostly share their first blocks, and what one of them loses there another
// gains (128 users of 4 beams, 500 to 60,000 tokens in blocks of 32: 10.8 us with an atomic for each entry, 7.1
// so). Workgroups of new rows copy them.
__global__ __launch_bounds__(kThreads) void k_fork(Pages p, Table t, const int32_t* __restrict__ parents, uint32_t fresh,
                                                   uint32_t runs, uint32_t parts, uint32_t olds, int32_t* __restrict__ table,
                                                   int32_t* __restrict__ lengths) {
  __shared__ int32_t more[kTogether];
  if (blockIdx.x >= olds) {
    const uint32_t run = (blockIdx.x - olds) % runs, to = (blockIdx.x - olds) / runs, e0 = run * kRun + threadIdx.x;
    const int32_t from = parents[to];
    const bool ok = (uint32_t)from < t.seqs;
    const int32_t* const src = t.table + (size_t)(ok ? from : 0) * t.width;
    int32_t* const dst = table + (size_t)to * t.width;
    int32_t x[kEntries];
#pragma unroll
    for (uint32_t i = 0; i < kEntries; ++i) x[i] = src[min(e0 + i * kThreads, t.width - 1u)];
#pragma unroll
    for (uint32_t i = 0; i < kEntries; ++i)
      if (e0 + i * kThreads < t.width) dst[e0 + i * kThreads] = ok ? x[i] : -1;
    if (run == 0 && threadIdx.x == 0) lengths[to] = ok ? t.lengths[from] : 0;
    return;
  }
  const uint32_t row0 = blockIdx.x / parts * kTogether, place = blockIdx.x % parts * kThreads + threadIdx.x;
  const uint32_t rows = min(kTogether, t.seqs - row0);
  int32_t x[kTogether];
#pragma unroll
  for (uint32_t r = 0; r < kTogether; ++r)
    x[r] = t.table[(size_t)(row0 + min(r, rows - 1u)) * t.width + min(place, t.width - 1u)];
  if (threadIdx.x < kTogether) more[threadIdx.x] = -1;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < fresh; i += kThreads) {
    const uint32_t r = (uint32_t)parents[i] - row0;
    if (r < rows) atomicAdd(more + r, 1);
  }
  __syncthreads();
  if (place >= t.width) return;
  int32_t block = x[0], by = 0;
#pragma unroll
  for (uint32_t r = 0; r < kTogether; ++r) {
    if (r >= rows) break;
    if (x[r] != block) {
      if (by != 0 && (uint32_t)block < p.blocks) atomicAdd(p.refs + block, by);
      block = x[r];
      by = 0;
    }
    by += more[r];
  }
  if (by != 0 && (uint32_t)block < p.blocks) atomicAdd(p.refs + block, by);
}

// ------------------------------------------------------------- reserve

constexpr uint32_t kFree = 1024;  // blocks whose free ones a wave counts
constexpr uint32_t kWords = kFree / 64;
constexpr uint32_t kLast = 1u << 31;  // of a need: the sequence keeps a block as the last of several

struct Needs {
  uint64_t* __restrict__ free;   // a bit for each block
  uint64_t* __restrict__ fresh;  // of each sequence, a bit for each place from the first with new tokens
  uint32_t* __restrict__ count;  // free blocks of each kFree
  uint32_t* __restrict__ need;   // blocks of each sequence
  uint32_t counts, words;        // words: of fresh, for a sequence
};

struct Growth {
  int32_t len, upto;
  bool grows;
  uint32_t first, end;  // places
  bool partly;          // tokens stand in the first already
};
__device__ __forceinline__ Growth growth(const Table& t, const int32_t* __restrict__ upto, uint32_t b, uint32_t bsh) {
  Growth g;
  g.len = t.lengths[b];
  g.upto = upto[b];
  g.grows = g.len >= 0 && g.upto > g.len && (int64_t)g.upto <= ((int64_t)t.width << bsh);
  g.first = (uint32_t)g.len >> bsh;
  g.end = (uint32_t)(((int64_t)g.upto + (1 << bsh) - 1) >> bsh);
  g.partly = (g.len & ((1 << bsh) - 1)) != 0;
  return g;
}

// A wave's kFree blocks from `at` * kFree: a word of free ones in each of its first lanes, and their number.
struct Free {
  uint64_t word;
  uint32_t count;
};
struct Refs {
  int32_t r[kWords];
};
__device__ __forceinline__ Refs refs_of(const Pages& p, uint32_t at, uint32_t lane) {
  Refs x;
#pragma unroll
  for (uint32_t i = 0; i < kWords; ++i) x.r[i] = p.refs[min(at * kFree + lane + i * 64, p.blocks - 1u)];
  return x;
}
__device__ __forceinline__ Free free_of(const Pages& p, const Refs& x, uint32_t at, uint32_t lane) {
  const int32_t* const r = x.r;
  const uint32_t b0 = at * kFree + lane;
  Free f{0, 0};
#pragma unroll
  for (uint32_t i = 0; i < kWords; ++i) {
    const uint64_t mask = __ballot(r[i] == 0 && b0 + i * 64 < p.blocks);
    f.count += (uint32_t)__popcll(mask);
    if (lane == i) f.word = mask;
  }
  return f;
}

// The places j0 .. of a sequence that need a block, as far as 64 of them go; without the partly filled one.
__device__ __forceinline__ uint64_t fresh_of(const Pages& p, const Growth& g, const int32_t* row, uint32_t j0, uint32_t lane) {
  const uint32_t j = j0 + lane;
  const bool asked = j < g.end && !(g.partly && j == g.first);
  const int32_t x = asked ? row[j] : -1;
  const bool valid = (uint32_t)x < p.blocks;
  return __ballot(asked && (!valid || p.refs[valid ? x : 0] > 1));
}

// What there is and what is asked for: a wave looks at kFree blocks, a workgroup at one sequence. Nothing
// that the others read is changed here.
__global__ __launch_bounds__(kThreads) void k_needs(Pages p, Table t, const int32_t* __restrict__ upto, Needs n) {
  __shared__ uint32_t lds[kWaves], most[kWaves];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  if (blockIdx.x >= t.seqs) {
    const uint32_t at = (blockIdx.x - t.seqs) * kWaves + wave;
    if (at >= n.counts) return;
    const Free f = free_of(p, refs_of(p, at, lane), at, lane);
    if (lane < kWords) n.free[(size_t)at * kWords + lane] = f.word;
    if (lane == 0) n.count[at] = f.count;
    return;
  }
  const uint32_t b = blockIdx.x;
  const Growth g = growth(t, upto, b, p.bsh);
  if (!g.grows) {
    if (tid == 0) n.need[b] = 0;
    return;
  }
  const int32_t* const row = t.table + (size_t)b * t.width;
  uint32_t need = 0;
  bool last = false, shared = false;
  if (g.partly) {
    const int32_t block = row[g.first];
    const int32_t refs = (uint32_t)block < p.blocks ? p.refs[block] : 0;
    shared = refs > 1;
    if (shared) {
      // The partly filled block has other owners. If all of them grow in this call, the last one need not copy it.
      uint32_t owners = 0, top = 0;
      for (uint32_t c = tid; c < t.seqs; c += kThreads) {
        const Growth o = growth(t, upto, c, p.bsh);
        if (o.grows && o.partly && t.table[(size_t)c * t.width + o.first] == block) {
          ++owners;
          top = c;
        }
      }
      owners = block_sum(owners, lds);
#pragma unroll
      for (int i = 1; i < 64; i <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, i));
      if (lane == 0) most[wave] = top;
      __syncthreads();
#pragma unroll
      for (uint32_t w = 0; w < kWaves; ++w) top = max(top, most[w]);
      last = top == b && (int32_t)owners == refs;
    }
  }
  for (uint32_t w = wave; g.first + w * 64 < g.end; w += kWaves) {
    uint64_t mask = fresh_of(p, g, row, g.first + w * 64, lane);
    if (w == 0 && shared && !last) mask |= 1ull;
    need += lane == 0 ? (uint32_t)__popcll(mask) : 0u;
    if (lane == 0) n.fresh[(size_t)b * n.words + w] = mask;
  }
  need = block_sum(need, lds);
  if (tid == 0) n.need[b] = need | (last ? kLast : 0u);
}

// The bit of a word with `rank` set ones below it; the word has more than that.
__device__ __forceinline__ uint32_t select_bit(uint64_t w, uint32_t rank) {
  uint32_t at = 0;
#pragma unroll
  for (uint32_t half = 32; half; half >>= 1) {
    const uint32_t below = (uint32_t)__popcll(w & ((1ull << half) - 1ull));
    const bool up = rank >= below;
    rank -= up ? below : 0u;
    at += up ? half : 0u;
    w = up ? w >> half : w;
  }
  return at;
}

// The free block with `rank` others before it in a run of kFree, by its words.
template <typename P>
__device__ __forceinline__ uint32_t block_of(P words, uint32_t rank) {
  uint64_t word[kWords], mine = 0;
#pragma unroll
  for (uint32_t i = 0; i < kWords; ++i) word[i] = words[i];
  uint32_t which = kWords;
#pragma unroll
  for (uint32_t i = 0; i < kWords; ++i) {
    const uint32_t ones = (uint32_t)__popcll(word[i]);
    if (which == kWords) {
      if (rank < ones) {
        which = i;
        mine = word[i];
      } else {
        rank -= ones;
      }
    }
  }
  return which * 64 + select_bit(mine, rank);
}

// Gives a sequence the block for its `rank`-th fresh place.
template <typename P>
__device__ __forceinline__ void give(const Pages& p, int32_t* row, uint32_t first, bool partly, P fresh, uint32_t rank,
                                     uint32_t block, int32_t* src, int32_t* dst) {
  uint32_t w = 0;
  for (uint32_t ones; rank >= (ones = (uint32_t)__popcll(fresh[w])); ++w) rank -= ones;
  const uint32_t j = first + w * 64 + select_bit(fresh[w], rank);
  const int32_t old = row[j];
  row[j] = (int32_t)block;
  p.refs[block] = 1;
  if ((uint32_t)old < p.blocks) atomicAdd(p.refs + old, -1);
  if (partly && j == first) {
    *src = old;
    *dst = (int32_t)block;
  }
}

// A workgroup for each sequence: the needs before it say which free blocks are
// its own, and a thread for each of them finds the block and the place. Only the table's row, the sequence's
// numbers and the counts of blocks that it alone takes or leaves change.
__global__ __launch_bounds__(kThreads) void k_give(Pages p, Table t, const int32_t* __restrict__ upto, Needs n,
                                                   int32_t* __restrict__ now, int32_t* __restrict__ src,
                                                   int32_t* __restrict__ dst) {
  __shared__ uint32_t lds[kWaves], upper[kThreads];
  const uint32_t b = blockIdx.x, tid = threadIdx.x;
  const Growth g = growth(t, upto, b, p.bsh);
  const uint32_t mine = n.need[b], need = mine & ~kLast;
  bool served = g.grows;
  uint32_t before = 0;
  if (mine) {
    uint32_t total = 0;
    for (uint32_t i = tid; i < b; i += kThreads) before += n.need[i] & ~kLast;
    for (uint32_t i = tid; i < n.counts; i += kThreads) total += n.count[i];
    before = block_sum(before, lds);
    total = block_sum(total, lds);
    served = (uint64_t)before + need <= total;
  }
  int32_t* const row = t.table + (size_t)b * t.width;
  const uint64_t* const fresh = n.fresh + (size_t)b * n.words;
  if (tid == 0) {
    now[b] = served ? g.upto : g.upto <= g.len ? g.len : 0;
    if (served) t.lengths[b] = g.upto;
    if (!(served && need && g.partly && (fresh[0] & 1u))) src[b] = dst[b] = -1;
  }
  if (!served || !need) return;
  uint32_t base = 0;  // free blocks before those that the workgroup looks at
  for (uint32_t c0 = 0; base < before + need; c0 += kThreads) {
    const uint32_t have = c0 + tid < n.counts ? n.count[c0 + tid] : 0u;
    uint32_t sum = have;
#pragma unroll
    for (uint32_t i = 1; i < 64; i <<= 1) {
      const uint32_t y = (uint32_t)__shfl_up((int)sum, i);
      sum += (tid & 63u) >= i ? y : 0u;
    }
    __syncthreads();
    if ((tid & 63u) == 63u) lds[tid >> 6] = sum;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kWaves - 1; ++w) sum += w < (tid >> 6) ? lds[w] : 0u;
    upper[tid] = sum;
    __syncthreads();
    const uint32_t all = upper[kThreads - 1];
    const uint32_t from = max(before, base), to = min(before + need, base + all);
    for (uint32_t rank = from + tid; rank < to; rank += kThreads) {
      uint32_t r = rank - base, at = 0;  // the first count whose upper end passes r
#pragma unroll
      for (uint32_t step = kThreads / 2; step; step >>= 1)
        if (upper[at + step - 1] <= r) at += step;
      r -= at ? upper[at - 1] : 0u;
      const uint32_t block = (c0 + at) * kFree + block_of(n.free + (size_t)(c0 + at) * kWords, r);
      give(p, row, g.first, g.partly, fresh, rank - before, block, src + b, dst + b);
    }
    base += all;
    if (c0 + kThreads >= n.counts) break;
  }
}

// Both in one workgroup, for up to kSmall runs of blocks and 64 sequences of up to kSmallWords words: a decoding step's
// batch. Its bits stay in LDS. Measured, in a graph, with this and with two launches: 64 sequences over 3979 blocks 4.7 and 6.9
// us, 32 over 254 that all share a block 6.5 and 8.4; a launch is also 3 us of the host.
constexpr uint32_t kSmall = 16, kSmallWords = 16;
__global__ __launch_bounds__(64 * kSmall) void k_reserve(Pages p, Table t, const int32_t* __restrict__ upto, uint32_t counts,
                                                         int32_t* __restrict__ now, int32_t* __restrict__ src,
                                                         int32_t* __restrict__ dst) {
  __shared__ uint64_t free[kSmall][kWords], fresh[64][kSmallWords];
  __shared__ uint32_t count[kSmall], need[64];
  const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const Refs run = refs_of(p, min(wave, counts - 1u), lane);  // asked for before the way to the sequences' blocks
  // Lane b of every wave knows sequence b.
  Growth g{};
  int32_t block = -1, refs = 0;
  if (lane < t.seqs) {
    g = growth(t, upto, lane, p.bsh);
    if (g.grows && g.partly) block = t.table[(size_t)lane * t.width + g.first];
    if ((uint32_t)block < p.blocks) refs = p.refs[block];
  }
  if (wave < counts) {
    const Free f = free_of(p, run, wave, lane);
    if (lane < kWords) free[wave][lane] = f.word;
    if (lane == 0) count[wave] = f.count;
  } else if (lane == 0) {
    count[wave] = 0;
  }
  // Of the owners of a partly filled block that all grow, the last one need not copy it.
  bool copies = refs > 1, last = false;
  for (uint64_t rest = __ballot(copies); rest;) {
    const int32_t one = __builtin_amdgcn_readlane(block, __builtin_ctzll(rest));
    const uint64_t same = __ballot(block == one);
    if (block == one && (int32_t)__popcll(same) == refs && (same >> lane) == 1ull) {
      last = true;
      copies = false;
    }
    rest &= ~same;
  }
  for (uint32_t b = wave; b < t.seqs; b += kSmall) {
    const Growth o{0, 0, true, (uint32_t)__builtin_amdgcn_readlane((int)g.first, (int)b),
                   (uint32_t)__builtin_amdgcn_readlane((int)(g.grows ? g.end : 0u), (int)b),
                   (bool)__builtin_amdgcn_readlane((int)g.partly, (int)b)};
    const uint64_t tail = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)copies, (int)b);
    uint32_t sum = 0;
    for (uint32_t w = 0; o.first + w * 64 < o.end; ++w) {
      const bool known = o.partly && o.end - o.first == 1;  // a token more in a block that has some
      uint64_t mask = w ? 0ull : tail;
      if (!known) mask |= fresh_of(p, o, t.table + (size_t)b * t.width, o.first + w * 64, lane);
      sum += (uint32_t)__popcll(mask);
      if (lane == 0) fresh[b][w] = mask;
    }
    if (lane == 0) need[b] = sum;
  }
  __syncthreads();
  const uint32_t mine = lane < t.seqs ? need[lane] : 0u, have = lane < kSmall ? count[lane] : 0u;
  uint32_t upper = mine, cum = have;
#pragma unroll
  for (uint32_t i = 1; i < 64; i <<= 1) {
    const uint32_t x = (uint32_t)__shfl_up((int)upper, i), y = (uint32_t)__shfl_up((int)cum, i);
    upper += lane >= i ? x : 0u;
    cum += lane >= i ? y : 0u;
  }
  const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)cum, 63);
  const bool served = g.grows && (upper <= total || !(mine || last));
  if (wave == 0 && lane < t.seqs) {
    now[lane] = served ? g.upto : g.upto <= g.len ? g.len : 0;
    if (served) t.lengths[lane] = g.upto;
    if (!(served && copies)) src[lane] = dst[lane] = -1;
  }
  for (uint32_t b = wave; b < t.seqs; b += kSmall) {
    const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)(served ? mine : 0u), (int)b);
    const uint32_t before = (uint32_t)__builtin_amdgcn_readlane((int)(upper - mine), (int)b);
    const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)g.first, (int)b);
    const bool partly = __builtin_amdgcn_readlane((int)g.partly, (int)b);
    for (uint32_t k0 = 0; k0 < n; k0 += 64) {
      uint32_t rank = before + k0 + lane, run = 0, below = 0;
#pragma unroll
      for (uint32_t i = 0; i < kSmall; ++i) {
        const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)cum, (int)i);
        run += rank >= c ? 1u : 0u;
        below = rank >= c ? c : below;
      }
      if (k0 + lane < n)
        give(p, t.table + (size_t)b * t.width, first, partly, fresh[b], k0 + lane,
             run * kFree + block_of(free[run], rank - below), src + b, dst + b);
    }
  }
}

// ------------------------------------------------------------- release

__global__ __launch_bounds__(kThreads) void k_release(Pages p, Table t, const int32_t* __restrict__ keep,
                                                      const int32_t* __restrict__ start, uint32_t runs) {
  const uint32_t run = blockIdx.x % runs, b = blockIdx.x / runs;
  uint32_t from = 0, to = t.width;
  if (start) from = (uint32_t)max(start[b], 0) >> p.bsh;
  if (keep) {
    const int32_t len = min(t.lengths[b], max(keep[b], 0));  // the same whether or not the row's first workgroup has been here
    to = (uint32_t)(((int64_t)len + (1 << p.bsh) - 1) >> p.bsh);
    if (run == 0 && threadIdx.x == 0) t.lengths[b] = len;
  }
  int32_t* const row = t.table + (size_t)b * t.width;
  int32_t x[kEntries];
  const uint32_t j0 = run * kRun + threadIdx.x;
#pragma unroll
  for (uint32_t i = 0; i < kEntries; ++i) x[i] = row[min(j0 + i * kThreads, t.width - 1u)];
#pragma unroll
  for (uint32_t i = 0; i < kEntries; ++i) {
    const uint32_t j = j0 + i * kThreads;
    if (j >= t.width || (j >= from && j < to) || x[i] == -1) continue;
    row[j] = -1;
    if ((uint32_t)x[i] < p.blocks) atomicAdd(p.refs + x[i], -1);
  }
}

// ---------------------------------------------------------------- copy

constexpr uint32_t kLayers = 32;  // caches of a launch
constexpr uint32_t kPairs = 1024;
constexpr uint32_t kUnroll = 4;
constexpr uint32_t kPiece = kThreads * 16 * kUnroll;  // bytes

struct Arrays {
  const int8_t* k;
  const int8_t* v;
  const float* scale;
  const int8_t* bound;
};
struct Copy {
  Arrays from[kLayers], to[kLayers];
  const int32_t* __restrict__ src;
  const int32_t* __restrict__ dst;
  uint32_t caches, pairs, from_blocks, to_blocks, kvh, codes, dim;  // codes: bytes of a block's keys, and of its values
};

// Workgroups walk the pieces of all pairs that are some: of a step's sequences few copy a block, and a
// grid for all of them would be launched for nothing.
__global__ __launch_bounds__(kThreads) void k_copy(Copy c) {
  __shared__ uint32_t lds[kWaves];
  __shared__ int32_t at[kPairs][2];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t parts = (c.codes + kPiece - 1) / kPiece, pieces = 2 * parts + 1;
  for (uint32_t i0 = 0; i0 < c.pairs; i0 += kPairs) {
    uint32_t have = 0;  // pairs found
    for (uint32_t i1 = 0; i1 < min(kPairs, c.pairs - i0); i1 += kThreads) {
      const uint32_t i = i0 + i1 + tid;
      int32_t s = -1, d = -1;
      if (i < c.pairs) {
        s = c.src[i];
        d = c.dst[i];
      }
      const bool ok = (uint32_t)s < c.from_blocks && (uint32_t)d < c.to_blocks;
      const uint64_t mask = __ballot(ok);
      __syncthreads();
      if (lane == 0) lds[wave] = (uint32_t)__popcll(mask);
      __syncthreads();
      uint32_t mine = have + (uint32_t)__popcll(mask & ((1ull << lane) - 1ull));
#pragma unroll
      for (uint32_t w = 0; w < kWaves; ++w) {
        if (w < wave) mine += lds[w];
        have += lds[w];
      }
      if (ok) {
        at[mine][0] = s;
        at[mine][1] = d;
      }
    }
    __syncthreads();
    const uint64_t all = (uint64_t)have * c.caches * pieces;
    for (uint64_t id = blockIdx.x; id < all; id += gridDim.x) {
      const uint32_t piece = (uint32_t)(id % pieces), rest = (uint32_t)(id / pieces);
      const uint32_t layer = rest % c.caches, pair = rest / c.caches;
      const size_t s = (size_t)at[pair][0], d = (size_t)at[pair][1];
      const Arrays& from = c.from[layer];
      const Arrays& to = c.to[layer];
      if (piece == 2 * parts) {  // bounds, and scales of 8 bytes a head
        const u4_t* const bs = reinterpret_cast<const u4_t*>(from.bound + s * c.kvh * 2 * c.dim);
        u4_t* const bd = reinterpret_cast<u4_t*>(const_cast<int8_t*>(to.bound) + d * c.kvh * 2 * c.dim);
        for (uint32_t x = tid; x < c.kvh * c.dim / 8; x += kThreads) bd[x] = bs[x];
        const u2_t* const ss = reinterpret_cast<const u2_t*>(from.scale + s * c.kvh * 2);
        u2_t* const sd = reinterpret_cast<u2_t*>(const_cast<float*>(to.scale) + d * c.kvh * 2);
        for (uint32_t x = tid; x < c.kvh; x += kThreads) sd[x] = ss[x];
        continue;
      }
      const bool v = piece >= parts;
      const uint32_t off = (v ? piece - parts : piece) * kPiece + tid * 16;
      const int8_t* const a = (v ? from.v : from.k) + s * c.codes + off;
      int8_t* const b = const_cast<int8_t*>(v ? to.v : to.k) + d * c.codes + off;
      u4_t x[kUnroll];
#pragma unroll
      for (uint32_t u = 0; u < kUnroll; ++u)
        if (off + u * kThreads * 16 < c.codes) x[u] = *reinterpret_cast<const u4_t*>(a + u * kThreads * 16);
#pragma unroll
      for (uint32_t u = 0; u < kUnroll; ++u)
        if (off + u * kThreads * 16 < c.codes) *reinterpret_cast<u4_t*>(b + u * kThreads * 16) = x[u];
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- host

const char* check_pages(const DanceKvPages* p, uint32_t seqs, uint32_t width) {
  if (!p || !p->refs) return "null pages";
  if (p->blocks == 0 || p->blocks > 0x7FFFFFFFu) return "blocks must be in [1, 2^31)";
  if (p->block_tokens != 16 && p->block_tokens != 32 && p->block_tokens != 64 && p->block_tokens != 128)
    return "block_tokens must be 16, 32, 64 or 128";
  if (seqs == 0 || width == 0 || seqs > 0x7FFFFFFFu) return "seqs and width must be positive, seqs below 2^31";
  if ((uint64_t)width * p->block_tokens > 0x7FFFFF00ull) return "a table row must hold at most 2^31 - 256 tokens";
  return nullptr;
}
Pages pages_args(const DanceKvPages* p) { return Pages{p->refs, p->blocks, log2_of(p->block_tokens)}; }
uint32_t runs_of(uint32_t width) { return (width + kRun - 1) / kRun; }
bool too_many(uint64_t workgroups) { return workgroups * kThreads > 0xFFFFFFFFull; }

struct Sizes {
  uint64_t counts, words, fresh, need, count, all;  // entries, words of a sequence, byte offsets, bytes
  bool small;                                        // one workgroup's LDS holds them
};
Sizes reserve_sizes(const DanceKvPages* p, uint32_t seqs, uint32_t width) {
  Sizes z;
  z.counts = ((uint64_t)p->blocks + kFree - 1) / kFree;
  z.words = ((uint64_t)width + 63) / 64;
  z.fresh = z.counts * kWords * 8;
  z.need = z.fresh + z.words * seqs * 8;
  z.count = z.need + (uint64_t)seqs * 4;
  z.small = z.counts <= kSmall && seqs <= 64 && z.words <= kSmallWords;
  z.all = z.small ? 0 : z.count + z.counts * 4;
  return z;
}

const char* check_layers(const DanceKvCache* c, uint32_t n) {
  for (uint32_t i = 0; i < n; ++i) {
    const DanceKvBatch one{nullptr, nullptr, nullptr, 1, 0, 1, 1, 0};
    if (const char* why = check_shapes(c + i, &one)) return why;
    if (!c[i].k || !c[i].v || !c[i].scale || !c[i].bound) return "null cache pointer";
    if (!aligned(c[i].k, 16) || !aligned(c[i].v, 16) || !aligned(c[i].scale, 8) || !aligned(c[i].bound, 16))
      return "the caches' arrays must be aligned to 16 bytes, their scales to 8";
    if (c[i].kv_heads != c->kv_heads || c[i].dim != c->dim || c[i].block_tokens != c->block_tokens || c[i].blocks != c->blocks)
      return "the caches must have one kv_heads, dim, block_tokens and number of blocks";
  }
  return nullptr;
}

}  // namespace
}  // namespace kv
}  // namespace dance

using namespace dance::kv;

extern "C" {

int dance_kv_fork(const DanceKvPages* pages, const int32_t* table, const int32_t* lengths, uint32_t seqs, uint32_t width,
                  const int32_t* parents, uint32_t new_seqs, int32_t* new_table, int32_t* new_lengths, void* stream) {
  const char* why = check_pages(pages, seqs, width);
  if (!why && (!table || !lengths || !parents || !new_table || !new_lengths)) why = "null pointer";
  if (!why && (new_seqs == 0 || new_seqs > 0x7FFFFFFFu)) why = "new_seqs must be positive, below 2^31";
  if (!why && (table == new_table || lengths == new_lengths)) why = "the new arrays must not be the old ones";
  if (why) KV_ERR("dance_kv_fork", "%s", why);
  const uint32_t runs = runs_of(width), parts = (width + kThreads - 1) / kThreads;
  const uint64_t olds = ((uint64_t)seqs + kTogether - 1) / kTogether * parts, grid = olds + (uint64_t)new_seqs * runs;
  if (too_many(grid)) KV_ERR("dance_kv_fork", "batch is too large for one launch");
  const Table t{const_cast<int32_t*>(table), const_cast<int32_t*>(lengths), seqs, width};
  hipLaunchKernelGGL(k_fork, dim3((uint32_t)grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream), pages_args(pages), t,
                     parents, new_seqs, runs, parts, (uint32_t)olds, new_table, new_lengths);
  return launched("dance_kv_fork");
}

size_t dance_kv_reserve_work(const DanceKvPages* pages, uint32_t seqs, uint32_t width) {
  return check_pages(pages, seqs, width) ? 0 : reserve_sizes(pages, seqs, width).all;
}

int dance_kv_reserve(const DanceKvPages* pages, int32_t* table, int32_t* lengths, uint32_t seqs, uint32_t width,
                     const int32_t* upto, int32_t* now, int32_t* src, int32_t* dst, void* work, size_t work_bytes,
                     void* stream) {
  const char* why = check_pages(pages, seqs, width);
  if (!why && (!table || !lengths || !upto || !now || !src || !dst)) why = "null pointer";
  if (!why && ((uint64_t)seqs * width > 0x7FFFFFFFull)) why = "a table must have fewer than 2^31 entries";
  if (why) KV_ERR("dance_kv_reserve", "%s", why);
  const Sizes z = reserve_sizes(pages, seqs, width);
  const Table t{table, lengths, seqs, width};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (z.small) {
    hipLaunchKernelGGL(k_reserve, dim3(1), dim3(64 * kSmall), 0, st, pages_args(pages), t, upto, (uint32_t)z.counts, now, src,
                       dst);
    return launched("dance_kv_reserve");
  }
  if (!work || work_bytes < z.all || !aligned(work, 16))
    KV_ERR("dance_kv_reserve", "work must hold %zu bytes, aligned to 16", (size_t)z.all);
  const uint64_t first = seqs + (z.counts + kWaves - 1) / kWaves;
  if (too_many(first) || too_many(seqs)) KV_ERR("dance_kv_reserve", "batch is too large for one launch");
  char* const w = static_cast<char*>(work);
  const Needs n{reinterpret_cast<uint64_t*>(w),           reinterpret_cast<uint64_t*>(w + z.fresh),
                reinterpret_cast<uint32_t*>(w + z.count), reinterpret_cast<uint32_t*>(w + z.need),
                (uint32_t)z.counts,                       (uint32_t)z.words};
  hipLaunchKernelGGL(k_needs, dim3((uint32_t)first), dim3(kThreads), 0, st, pages_args(pages), t, upto, n);
  hipLaunchKernelGGL(k_give, dim3(seqs), dim3(kThreads), 0, st, pages_args(pages), t, upto, n, now, src, dst);
  return launched("dance_kv_reserve");
}

int dance_kv_release(const DanceKvPages* pages, int32_t* table, int32_t* lengths, uint32_t seqs, uint32_t width,
                     const int32_t* keep, const int32_t* start, void* stream) {
  const char* why = check_pages(pages, seqs, width);
  if (!why && (!table || !lengths)) why = "null pointer";
  if (why) KV_ERR("dance_kv_release", "%s", why);
  if (!keep && !start) return 0;
  const uint32_t runs = runs_of(width);
  const uint64_t grid = (uint64_t)seqs * runs;
  if (too_many(grid)) KV_ERR("dance_kv_release", "batch is too large for one launch");
  const Table t{table, lengths, seqs, width};
  hipLaunchKernelGGL(k_release, dim3((uint32_t)grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream), pages_args(pages), t,
                     keep, start, runs);
  return launched("dance_kv_release");
}

int dance_kv_copy(const DanceKvCache* from, const DanceKvCache* to, uint32_t caches, const int32_t* src, const int32_t* dst,
                  uint32_t pairs, void* stream) {
  const char* why = !from || !to || caches == 0 ? "caches must be given" : check_layers(from, caches);
  if (!why) why = check_layers(to, caches);
  if (!why && (from->kv_heads != to->kv_heads || from->dim != to->dim || from->block_tokens != to->block_tokens))
    why = "both sides must have one kv_heads, dim and block_tokens";
  if (!why && pairs && (!src || !dst)) why = "null pointer";
  if (!why && pairs > 0x7FFFFFFFu) why = "pairs must be below 2^31";
  if (why) KV_ERR("dance_kv_copy", "%s", why);
  if (pairs == 0) return 0;
  const uint64_t codes = (uint64_t)from->kv_heads * from->dim * from->block_tokens;
  const uint64_t pieces = 2 * ((codes + kPiece - 1) / kPiece) + 1;
  for (uint32_t c0 = 0; c0 < caches; c0 += kLayers) {
    Copy c{};
    c.caches = caches - c0 < kLayers ? caches - c0 : kLayers;
    for (uint32_t i = 0; i < c.caches; ++i) {
      const DanceKvCache &f = from[c0 + i], &t = to[c0 + i];
      c.from[i] = Arrays{f.k, f.v, f.scale, f.bound};
      c.to[i] = Arrays{t.k, t.v, t.scale, t.bound};
    }
    c.src = src, c.dst = dst, c.pairs = pairs;
    c.from_blocks = from->blocks, c.to_blocks = to->blocks;
    c.kvh = from->kv_heads, c.codes = (uint32_t)codes, c.dim = from->dim;
    const uint64_t all = pieces * c.caches * pairs, most = 2048;  // eight workgroups a CU
    hipLaunchKernelGGL(k_copy, dim3((uint32_t)(all < most ? all : most)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), c);
  }
  return launched("dance_kv_copy");
}

}  // extern "C"
