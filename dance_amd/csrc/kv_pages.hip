// dance_kv_fork, dance_kv_reserve, dance_kv_release and dance_kv_copy
// (include/dance_kv_pages.h): who owns a pool's blocks, and copies of blocks.
//
// The first three are chains of dependent loads over little data (a table, a
// count for each block), so they are bound by latency and by their launches; counts
// change by integer atomics, whose order shows in no result.

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

// Workgroups of old rows change the counts, by a row's children less one: where a
// row goes on as one, in whatever slot, nothing is to be counted. Those of new
// rows copy them.
__global__ __launch_bounds__(kThreads) void k_fork(Pages p, Table t, const int32_t* __restrict__ parents, uint32_t fresh,
                                                   uint32_t runs, int32_t* __restrict__ table, int32_t* __restrict__ lengths) {
  __shared__ uint32_t lds[kWaves];
  const uint32_t run = blockIdx.x % runs, row = blockIdx.x / runs;
  const uint32_t e0 = run * kRun + threadIdx.x;
  if (row < fresh) {
    const int32_t from = parents[row];
    const bool ok = (uint32_t)from < t.seqs;
    const int32_t* const src = t.table + (size_t)(ok ? from : 0) * t.width;
    int32_t* const dst = table + (size_t)row * t.width;
    int32_t x[kEntries];
#pragma unroll
    for (uint32_t i = 0; i < kEntries; ++i) x[i] = ok && e0 + i * kThreads < t.width ? src[e0 + i * kThreads] : -1;
#pragma unroll
    for (uint32_t i = 0; i < kEntries; ++i)
      if (e0 + i * kThreads < t.width) dst[e0 + i * kThreads] = x[i];
    if (run == 0 && threadIdx.x == 0) lengths[row] = ok ? t.lengths[from] : 0;
    return;
  }
  const uint32_t old = row - fresh;
  uint32_t mine = 0;
  for (uint32_t i = threadIdx.x; i < fresh; i += kThreads) mine += (uint32_t)parents[i] == old ? 1u : 0u;
  const int32_t more = (int32_t)block_sum(mine, lds) - 1;
  if (more == 0) return;
  const int32_t* const src = t.table + (size_t)old * t.width;
#pragma unroll
  for (uint32_t i = 0; i < kEntries; ++i) {
    const int32_t x = e0 + i * kThreads < t.width ? src[e0 + i * kThreads] : -1;
    if ((uint32_t)x < p.blocks) atomicAdd(p.refs + x, more);
  }
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

// What there is and what is asked for: a wave looks at kFree blocks, or at one sequence. Nothing
// that the other waves read is changed here.
__global__ __launch_bounds__(kThreads) void k_needs(Pages p, Table t, const int32_t* __restrict__ upto, Needs n) {
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t at = blockIdx.x * kWaves + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  if (at < n.counts) {
    int32_t r[kWords];
    const uint32_t b0 = at * kFree + lane;
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) r[i] = b0 + i * 64 < p.blocks ? p.refs[b0 + i * 64] : 1;
    uint64_t mine = 0;
    uint32_t sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWords; ++i) {
      const uint64_t mask = __ballot(r[i] == 0);
      sum += (uint32_t)__popcll(mask);
      if (lane == i) mine = mask;
    }
    if (lane < kWords) n.free[(size_t)at * kWords + lane] = mine;
    if (lane == 0) n.count[at] = sum;
    return;
  }
  const uint32_t b = at - n.counts;
  if (b >= t.seqs) return;
  const Growth g = growth(t, upto, b, p.bsh);
  uint32_t need = 0;
  if (g.grows) {
    const int32_t* const row = t.table + (size_t)b * t.width;
    for (uint32_t j0 = g.first; j0 < g.end; j0 += 64) {
      const uint32_t j = j0 + lane;
      const int32_t x = j < g.end ? row[j] : -1;
      const bool valid = (uint32_t)x < p.blocks;
      const bool many = valid && p.refs[valid ? x : 0] > 1;
      const bool part = g.partly && j == g.first;
      uint64_t mask = __ballot(j < g.end && (part ? many : many || !valid));
      if (g.partly && j0 == g.first && (mask & 1u)) {
        // The partly filled block has other owners. Those that grow in this call too will not write it.
        const int32_t block = __builtin_amdgcn_readfirstlane(x);
        uint32_t owners = 0, last = 0;
        for (uint32_t c = lane; c < t.seqs; c += 64) {
          const Growth o = growth(t, upto, c, p.bsh);
          if (o.grows && o.partly && t.table[(size_t)c * t.width + o.first] == block) {
            ++owners;
            last = c;
          }
        }
#pragma unroll
        for (int i = 1; i < 64; i <<= 1) {
          owners += (uint32_t)__shfl_xor((int)owners, i);
          last = max(last, (uint32_t)__shfl_xor((int)last, i));
        }
        if (last == b && (int32_t)owners == p.refs[block]) {
          mask &= ~1ull;
          need |= kLast;
        }
      }
      need += (uint32_t)__popcll(mask);
      if (lane == 0) n.fresh[(size_t)b * n.words + (j0 - g.first) / 64] = mask;
    }
  }
  if (lane == 0) n.need[b] = need;
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

// A workgroup for each sequence: the needs before it say which free blocks are
// its own, and a thread for each of them finds the block and the place. Only the table's row, the sequence's
// numbers and the counts of blocks that it alone takes or leaves change.
__global__ __launch_bounds__(kThreads) void k_give(Pages p, Table t, const int32_t* __restrict__ upto, Needs n,
                                                   int32_t* __restrict__ now, int32_t* __restrict__ src, int32_t* __restrict__ dst) {
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
      const uint64_t* const words = n.free + (size_t)(c0 + at) * kWords;
      uint64_t word[kWords], bits = 0;
#pragma unroll
      for (uint32_t i = 0; i < kWords; ++i) word[i] = words[i];
      uint32_t which = kWords;
#pragma unroll
      for (uint32_t i = 0; i < kWords; ++i) {
        const uint32_t ones = (uint32_t)__popcll(word[i]);
        if (which == kWords) {
          if (r < ones) {
            which = i;
            bits = word[i];
          } else {
            r -= ones;
          }
        }
      }
      const uint32_t block = ((c0 + at) * kWords + which) * 64 + select_bit(bits, r);
      uint32_t k = rank - before, w = 0;  // its place
      for (uint32_t ones; k >= (ones = (uint32_t)__popcll(fresh[w])); ++w) k -= ones;
      const uint32_t j = g.first + w * 64 + select_bit(fresh[w], k);
      const int32_t old = row[j];
      row[j] = (int32_t)block;
      p.refs[block] = 1;
      if ((uint32_t)old < p.blocks) atomicAdd(p.refs + old, -1);
      if (g.partly && j == g.first) {
        src[b] = old;
        dst[b] = (int32_t)block;
      }
    }
    base += all;
    if (c0 + kThreads >= n.counts) break;
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
#pragma unroll
  for (uint32_t i = 0; i < kEntries; ++i) {
    const uint32_t j = run * kRun + i * kThreads + threadIdx.x;
    if (j >= t.width || (j >= from && j < to)) continue;
    const int32_t x = row[j];
    if (x != -1) row[j] = -1;
    if ((uint32_t)x < p.blocks) atomicAdd(p.refs + x, -1);
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
};
Sizes reserve_sizes(const DanceKvPages* p, uint32_t seqs, uint32_t width) {
  Sizes z;
  z.counts = ((uint64_t)p->blocks + kFree - 1) / kFree;
  z.words = ((uint64_t)width + 63) / 64;
  z.fresh = z.counts * kWords * 8;
  z.need = z.fresh + z.words * seqs * 8;
  z.count = z.need + (uint64_t)seqs * 4;
  z.all = z.count + z.counts * 4;
  return z;
}

const char* check_layers(const DanceKvCache* c, uint32_t n) {
  for (uint32_t i = 0; i < n; ++i) {
    const DanceKvBatch one{nullptr, nullptr, nullptr, 1, 0, 1, 1, 0};
    if (const char* why = check_shapes(c + i, &one)) return why;
    if (!c[i].k || !c[i].v || !c[i].scale || !c[i].bound) return "null cache pointer";
    if (!aligned(c[i].k, 16) || !aligned(c[i].v, 16) || !aligned(c[i].scale, 16) || !aligned(c[i].bound, 16))
      return "the cache's arrays must be aligned to 16 bytes";
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
  const uint32_t runs = runs_of(width);
  const uint64_t grid = ((uint64_t)seqs + new_seqs) * runs;
  if (too_many(grid)) KV_ERR("dance_kv_fork", "batch is too large for one launch");
  const Table t{const_cast<int32_t*>(table), const_cast<int32_t*>(lengths), seqs, width};
  hipLaunchKernelGGL(k_fork, dim3((uint32_t)grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream), pages_args(pages), t,
                     parents, new_seqs, runs, new_table, new_lengths);
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
  if (!work || work_bytes < z.all || !aligned(work, 16))
    KV_ERR("dance_kv_reserve", "work must hold %zu bytes, aligned to 16", (size_t)z.all);
  const uint64_t first = (z.counts + seqs + kWaves - 1) / kWaves;
  if (too_many(first) || too_many(seqs)) KV_ERR("dance_kv_reserve", "batch is too large for one launch");
  char* const w = static_cast<char*>(work);
  const Needs n{reinterpret_cast<uint64_t*>(w), reinterpret_cast<uint64_t*>(w + z.fresh), reinterpret_cast<uint32_t*>(w + z.count),
                reinterpret_cast<uint32_t*>(w + z.need), (uint32_t)z.counts, (uint32_t)z.words};
  const Table t{table, lengths, seqs, width};
  const hipStream_t st = static_cast<hipStream_t>(stream);
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
