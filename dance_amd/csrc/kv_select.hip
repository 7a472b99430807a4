// dance_kv_select (include/dance_kv.h): the blocks whose keys may have the
// largest products with a query, by a bound.
//
// With hi and lo the largest and least key code of a block's tokens in a
// dimension, c k <= max(c hi, c lo) for the code c of the query and each of the
// block's codes k: c hi where c > 0, c lo where c < 0. The bound of all
// dimensions is thus one product of length 2 D, (c+ | c-) with (hi | lo), the
// latter as they lie in memory. It is done with 16x16x64 i8 MFMAs, 16 query rows
// by 16 blocks, exactly; only the block's scale is rounded in (once). The
// result registers of a lane are four rows of one block: with groups of up to
// four heads the group's largest score needs no other lane.
//
// The scores of a few token rows stay in LDS as whole numbers that order like
// them, and the same workgroup chooses: it counts the keys by 8 bits of their
// distance from the least, which spreads them over the counters whatever
// their exponents are, narrows the range to the counter that holds the
// count-th largest until it is all taken or a single key, and writes what
// is larger, and of what equals it the first ones, in index order.
//
// Measured (8 kv heads of 4, 128 dimensions): 16 rows over 60,000 to 131,072 tokens in blocks of 64, 52 MB, 23 us,
// a workgroup's loads and lane exchange of 2048 blocks, then 6 of choice; 1026 rows of two
// sequences over 20,000 to 40,000 in blocks of 32, 71 us, of which the choice 32, loads and exchange 25,
// products and keys 20 (they overlap), all bound by LDS and vector instructions. 16 waves leave a lane 128
// registers: at 96, 128 and 256 dimensions 1, 3 and 9 values go to scratch.

#include <cmath>
#include <type_traits>

#include "kv_common.h"

namespace dance {
namespace kv {
namespace {

constexpr uint32_t kSelWaves = 16;
constexpr uint32_t kSelThreads = 64 * kSelWaves;

constexpr uint32_t kNoKey = 0x007FFFFFu;   // of -inf: holes
constexpr uint32_t kForced = 0xFFFFFFFFu;  // above all scores
__device__ __forceinline__ uint32_t sort_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SelectArgs {
  Cache c;
  Batch b;
  Rows q;
  uint32_t group, gp;    // heads of a kv head; padded to a power of two where they share a row tile
  uint32_t ntok, tiles, slots;  // token rows of a workgroup, workgroups of a sequence (0: see tile_at), of all
  uint32_t count, sink, recent;
  uint32_t blocks;       // keys of a token row
  uint32_t chunks, per;  // k_score: workgroups that share the blocks, blocks of each
  uint32_t* __restrict__ keys;  // where they do not stay in LDS: [token row][kv head][blocks]
  int32_t* __restrict__ chosen;
};

// The token rows of a workgroup and what they see.
struct Tokens {
  uint32_t sq, row, n;  // sequence, first row, rows
  int64_t first;        // position of the first row
  int64_t len;
  __device__ __forceinline__ uint32_t seen(const SelectArgs& a, uint32_t t) const {
    const int64_t end = first + t + 1 < len ? first + t + 1 : len;
    return end > 0 ? min((uint32_t)((end + (1ll << a.c.bsh) - 1) >> a.c.bsh), a.blocks) : 0u;
  }
};
__device__ __forceinline__ Tokens tokens_of(const SelectArgs& a, uint32_t sq, uint32_t tile) {
  const Seq s = seq_of(a.b, sq, a.c.bsh);
  const uint32_t t0 = tile * a.ntok;
  return Tokens{sq, s.row + t0, min(a.ntok, less(s.n, t0)), s.first + t0, s.len};
}

constexpr int kRowTiles = 4;  // row tiles that a pass over the blocks serves
template <int D>
struct Codes {
  // Row stride: 16 bytes over the codes, so that the 16 rows of an operand lie in
  // different banks.
  static constexpr uint32_t kStride = 2 * D + 16;
  int8_t c[kRowTiles * 16 * kStride];
  __attribute__((aligned(16))) float up[kRowTiles * 16];  // 2^e of a row's codes
  uint32_t seen[kRowTiles * 16];  // blocks that a token row sees
};

// Codes of row tiles [p0, p0 + kRowTiles): a wave's four lane groups of 16 take a row each.
template <int D, bool BF, bool VEC>
__device__ __forceinline__ void code_rows(const SelectArgs& a, const Tokens& tk, uint32_t h, uint32_t p0, uint32_t rows,
                                          Codes<D>& qc) {
  constexpr int V = D / 16;  // values of a lane; 8 at a time where they are 8 or 16
  const uint32_t l = threadIdx.x & 15u;
  const uint32_t end = min((uint32_t)kRowTiles, rows - p0) * 16u;
  for (uint32_t r = threadIdx.x >> 4; r < end; r += kSelThreads / 16) {
    const uint32_t t = a.group > 16u ? 0u : (p0 * 16u + r) / a.gp;
    // rows of no head repeat the group's last, which changes no maximum; those of no token are not used
    const uint32_t f = min(a.group > 16u ? p0 * 16u + r : r % a.gp, a.group - 1u);
    const uint16_t* const src = a.q.data + (int64_t)(tk.row + min(t, tk.n - 1u)) * a.q.token_stride +
                                (int64_t)(h * a.group + f) * a.q.head_stride + l * V;
    float x[V];
    if constexpr (VEC && V % 4 == 0) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const u2_t w = *reinterpret_cast<const u2_t*>(src + 4 * i);
#pragma unroll
        for (int b = 0; b < 4; ++b) x[4 * i + b] = load_val<BF>((uint16_t)(w[b >> 1] >> (16 * (b & 1))));
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = load_val<BF>(src[i]);
    }
    float mag = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) mag = fmaxf(mag, finite_abs(x[i]));
    mag = cols_max(mag);
    const int e = scale_exp(mag);
    const float inv = exp2_int(-e);
    int8_t* const out = qc.c + r * Codes<D>::kStride + l * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int code = code_of(x[i], inv);
      out[i] = (int8_t)max(code, 0);
      out[D + i] = (int8_t)min(code, 0);
    }
    if (l == 0) qc.up[r] = exp2_int(e);
  }
}

// Between the lanes that differ in bit X (1 or 2): the lower one gives its y for the other's x.
template <int X>
__device__ __forceinline__ void swap_pieces(i4_t& x, i4_t& y, bool upper) {
  constexpr int perm = X == 1 ? 0xB1 : 0x4E;  // quad lanes 1 0 3 2, 2 3 0 1
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int got = __builtin_amdgcn_mov_dpp(upper ? x[w] : y[w], perm, 0xF, 0xF, true);
    x[w] = upper ? got : x[w];
    y[w] = upper ? y[w] : got;
  }
}

// Keys of blocks [from, to) for the workgroup's token rows: keys[t * stride + block].
template <int D, bool BF, bool VEC>
__device__ __forceinline__ void score_blocks(const SelectArgs& a, const Tokens& tk, uint32_t h, uint32_t from,
                                             uint32_t to, uint32_t* __restrict__ keys, size_t stride, Codes<D>& qc) {
  constexpr int KS = D / 32;  // inner steps of 64 over 2 D
  const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t n = lane & 15u, g = lane >> 4;
  const int32_t* const table = a.b.table + (size_t)tk.sq * a.b.width;
  const uint32_t per_tile = 16u / a.gp;  // token rows of a row tile
  const uint32_t rows = a.group > 16u ? (a.group + 15u) / 16u : (tk.n + per_tile - 1u) / per_tile;
  for (uint32_t t = threadIdx.x; t < tk.n; t += kSelThreads) qc.seen[t] = tk.seen(a, t);
  // A wave takes adjacent tiles of 16 blocks, four at a time: their places come with one
  // load, their scales with another. The bounds of two tiles (of one, beyond 128 dimensions: registers)
  // are on their way while a third is computed.
  constexpr bool kDeep = D <= 128;
  struct Tile {
    i4_t b[KS];
  };
  const uint32_t all = (to - from + 15u) / 16u, share = (all + kSelWaves - 1) / kSelWaves;
  const uint32_t t_end = min(all, (wave + 1) * share), t_begin = min(t_end, wave * share);
  struct Four {  // lane i: block i of the 64
    int32_t ph;
    float ks;
  };
  auto places = [&](uint32_t tile) {
    const uint32_t blk = from + tile * 16u + lane;
    const int32_t ph = blk < to && tile < t_end ? table[blk] : -1;
    Four f{(uint32_t)ph < a.c.blocks ? ph : -1, 0.f};
    if (f.ph >= 0) f.ks = a.c.scale[((size_t)f.ph * a.c.kvh + h) * 2];
    return f;
  };
  // A load instruction that takes 16 bytes of each of 16 blocks costs the address unit a
  // turn for each of its 64 lanes (37 GB/s a CU). So S neighbouring lanes take S
  // adjacent pieces of one block, S loads the blocks of S lanes, and turned() exchanges
  // them: lane r of the S gets all pieces of block r.
  constexpr int S = KS % 4 == 0 ? 4 : KS % 2 == 0 ? 2 : 1;
  auto load = [&](const Four& f, uint32_t i) {
    Tile t;
#pragma unroll
    for (int c = 0; c < S; ++c) {
      const int32_t ph = __shfl(f.ph, (int)(16u * i + (n & ~(uint32_t)(S - 1)) + c));
      const int8_t* const bp = a.c.bound + ((size_t)max(ph, 0) * a.c.kvh + h) * 2 * D + (g * S + (n & (S - 1))) * 16;
#pragma unroll
      for (int k = 0; k < KS / S; ++k) t.b[k * S + c] = *reinterpret_cast<const i4_t*>(bp + k * S * 64);
    }
    return t;
  };
  auto turned = [&](Tile& t) {
    if constexpr (S > 1) {
#pragma unroll
      for (int k = 0; k < KS; k += S) {
#pragma unroll
        for (int c = 0; c < S; c += 2) swap_pieces<1>(t.b[k + c], t.b[k + c + 1], n & 1u);
        if constexpr (S == 4) {
          swap_pieces<2>(t.b[k], t.b[k + 2], n & 2u);
          swap_pieces<2>(t.b[k + 1], t.b[k + 3], n & 2u);
        }
      }
    }
  };
  // where in a row of 2 D codes the inner step c of this lane group stands
  auto piece = [&](int c) { return (uint32_t)(c / S * S * 64 + c % S * 16) + g * S * 16u; };
  Four four = places(t_begin);
  for (uint32_t p0 = 0; p0 < rows; p0 += kRowTiles) {
    if (p0) __syncthreads();
    code_rows<D, BF, VEC>(a, tk, h, p0, rows, qc);
    __syncthreads();
    const uint32_t here = min((uint32_t)kRowTiles, rows - p0);
    auto put = [&](uint32_t t, uint32_t blk, bool hole, float x, bool add) {
      if (t >= tk.n || blk >= to) return;
      const uint32_t seen = qc.seen[t];
      uint32_t key = sort_key(x + 0.f);
      if (blk < a.sink || blk + a.recent >= seen) key = kForced;
      if (hole) key = kNoKey;
      uint32_t* const at = keys + t * stride + blk;
      *at = add ? max(key, *at) : key;  // more than 16 heads: the same lane's key of those before
    };
    auto score = [&](const Tile& b, float ks, bool hole, uint32_t blk, uint32_t r, const i4_t* qf, f4_t up) {
      i4_t acc = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < KS; ++c) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qf[c], b.b[c], acc, 0, 0, 0);
      float x[4];  // rows 4 g + i of block n
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (float)acc[i] * (ks * up[i]);
      const uint32_t t0 = (p0 + r) * per_tile;
      if (a.group > 16u) {
        const float m = rows_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
        if (g == 0) put(0, blk, hole, m, p0 + r != 0);
      } else if (a.gp == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) put(t0 + 4 * g + i, blk, hole, x[i], false);
      } else if (a.gp == 2) {
        put(t0 + 2 * g, blk, hole, fmaxf(x[0], x[1]), false);
        put(t0 + 2 * g + 1, blk, hole, fmaxf(x[2], x[3]), false);
      } else {
        float m = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        if (a.gp == 4) {
          put(t0 + g, blk, hole, m, false);
        } else if (a.gp == 8) {
          m = pair_max(m);
          if ((g & 1u) == 0) put(t0 + (g >> 1), blk, hole, m, false);
        } else {
          m = rows_max(m);
          if (g == 0) put(t0, blk, hole, m, false);
        }
      }
    };
    if (p0) four = places(t_begin);
    Tile t0 = load(four, 0), t1;
    if constexpr (kDeep) t1 = load(four, 1);
    for (uint32_t tile = t_begin; tile < t_end; tile += 4) {
      const Four next = places(tile + 4);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        if (tile + i >= t_end) break;
        constexpr uint32_t kAhead = kDeep ? 2 : 1;
        Tile t2;
        if (tile + i + kAhead < t_end) t2 = i + kAhead < 4 ? load(four, i + kAhead) : load(next, i + kAhead - 4);
        const bool hole = __shfl(four.ph, (int)(16u * i + n)) < 0;
        const float ks = __shfl(four.ks, (int)(16u * i + n));
        turned(t0);
        for (uint32_t r = 0; r < here; ++r) {
          i4_t qf[KS];
#pragma unroll
          for (int c = 0; c < KS; ++c)
            qf[c] = *reinterpret_cast<const i4_t*>(qc.c + (r * 16u + n) * Codes<D>::kStride + piece(c));
          const f4_t up = *reinterpret_cast<const f4_t*>(&qc.up[r * 16u + 4 * g]);
          score(t0, ks, hole, from + (tile + i) * 16u + n, r, qf, up);
        }
        if constexpr (kDeep) {
          t0 = t1;
          t1 = t2;
        } else {
          t0 = t2;
        }
      }
      four = next;
    }
  }
}

// What a team of W waves shares while it chooses. A team of one wave clears its
// counters itself; a team of several has a cleared set for each of the four
// rounds (clear_teams), and every wave reads them, so that a round takes one barrier.
struct Team {
  uint32_t hist[256];
};
struct Shared {  // W > 1: each wave's
  uint32_t lo[kSelWaves], hi[kSelWaves], some[kSelWaves], forced[kSelWaves], more[kSelWaves], same[kSelWaves];
};
constexpr int kRounds = 4;  // of 8 bits
__device__ __forceinline__ void clear_teams(Team* tm) {
  for (uint32_t i = threadIdx.x; i < kRounds * 256; i += kSelThreads) tm[i >> 8].hist[i & 255u] = 0;
}

// Without LDS: over the 16 lanes that differ in bits 0 to 3, then over all 64.
template <typename Op>
__device__ __forceinline__ uint32_t over16(uint32_t x, Op op) {
  auto with = [&](auto ctrl) {  // as in cols_max
    x = op(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, decltype(ctrl)::value, 0xF, 0xF, true));
  };
  with(Int<0xB1>{});
  with(Int<0x4E>{});
  with(Int<0x141>{});
  with(Int<0x140>{});
  return x;
}
template <typename Op>
__device__ __forceinline__ uint32_t over64(uint32_t x, Op op) {
  x = over16(x, op);
  const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = op(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)op(b[0], b[1]));
}
// Sum over this lane and those after it: within rows of 16 by shifts, then the rows behind.
__device__ __forceinline__ uint32_t sum_from(uint32_t x) {
  auto with = [&](auto ctrl) {  // lane i + 1, 2, 4, 8 of the row; 0 beyond its end
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xF, 0xF, true);
  };
  with(Int<0x101>{});
  with(Int<0x102>{});
  with(Int<0x104>{});
  with(Int<0x108>{});
  const uint32_t r3 = (uint32_t)__builtin_amdgcn_readlane((int)x, 48);
  const uint32_t r2 = r3 + (uint32_t)__builtin_amdgcn_readlane((int)x, 32);
  const uint32_t r1 = r2 + (uint32_t)__builtin_amdgcn_readlane((int)x, 16);
  const uint32_t row = (threadIdx.x & 63u) >> 4;
  return x + (row == 0 ? r1 : row == 1 ? r2 : row == 2 ? r3 : 0u);
}

// The `count` blocks of the n with the largest keys, ties to the lower block, ascending.
template <uint32_t W>
__device__ __forceinline__ void choose(const uint32_t* __restrict__ keys, uint32_t n, uint32_t count,
                                       int32_t* __restrict__ out, Team* tm, Shared& sh) {
  const uint32_t lane = threadIdx.x & 63u, wave = W == 1 ? 0u : threadIdx.x >> 6;
  const uint32_t tid = W == 1 ? lane : threadIdx.x;
  auto sync = [&] {
    if constexpr (W > 1) {
      __syncthreads();
    } else {  // a wave's LDS accesses complete in order; the compiler has to keep it
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  };
  // Four keys at a time, read before the first is looked at; a hole beyond the end.
  constexpr uint32_t kStrip = 4;
  auto strip = [&](uint32_t i, uint32_t step, uint32_t end, uint32_t (&k)[kStrip]) {
#pragma unroll
    for (uint32_t x = 0; x < kStrip; ++x) k[x] = i + x * step < end ? keys[i + x * step] : kNoKey;
  };
  // Range of the keys that compete, how many they are, and how many are forced. Forced
  // keys (the largest number) wrap to 0 before the maximum, holes to the largest before the minimum.
  uint32_t lo = ~0u, hi = 0, some = 0, forced = 0;
  for (uint32_t i0 = 0; i0 < n; i0 += kStrip * 64 * W) {
    uint32_t k[kStrip];
    strip(i0 + tid, 64 * W, n, k);
#pragma unroll
    for (uint32_t x = 0; x < kStrip; ++x) {
      hi = max(hi, k[x] + 1u);
      lo = min(lo, k[x] - (kNoKey + 1u));
      some += (uint32_t)__popcll(__ballot(k[x] > kNoKey));
      forced += (uint32_t)__popcll(__ballot(k[x] == kForced));
    }
  }
  auto least = [](uint32_t a, uint32_t b) { return min(a, b); };
  auto most = [](uint32_t a, uint32_t b) { return max(a, b); };
  auto sum = [](uint32_t a, uint32_t b) { return a + b; };
  auto same_in_all = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
  lo = over64(lo, least);
  hi = over64(hi, most);
  if constexpr (W > 1) {
    static_assert(W == 16, "over16");
    if (lane == 0) sh.lo[wave] = lo, sh.hi[wave] = hi, sh.some[wave] = some, sh.forced[wave] = forced;
    __syncthreads();
    const uint32_t w = lane & (W - 1u);
    lo = same_in_all(over16(sh.lo[w], least));
    hi = same_in_all(over16(sh.hi[w], most));
    some = same_in_all(over16(sh.some[w], sum));
    forced = same_in_all(over16(sh.forced[w], sum));
  }
  lo += kNoKey + 1u;
  hi -= 1u;
  some -= forced;
  // All keys above `limit` are taken, and the first `ties` equal to it.
  uint32_t want = less(count, forced), limit, ties = 0;
  if (some <= want) {
    limit = kNoKey;
  } else if (want == 0) {
    limit = kForced - 1u;
  } else {
    for (int round = 0;; ++round) {  // ends: a round of four at most has shift 0
      const uint32_t bits = 32u - (uint32_t)__clz((int)(hi - lo | 1u));
      const uint32_t shift = less(bits, 8u);
      uint32_t* const hist = tm[W == 1 ? 0 : round].hist;
      if constexpr (W == 1) {
        for (uint32_t i = tid; i < 256; i += 64) hist[i] = 0;
        sync();
      }
      for (uint32_t i0 = 0; i0 < n; i0 += kStrip * 64 * W) {
        uint32_t k[kStrip];
        strip(i0 + tid, 64 * W, n, k);
#pragma unroll
        for (uint32_t x = 0; x < kStrip; ++x)
          if (k[x] - lo <= hi - lo) atomicAdd(&hist[(k[x] - lo) >> shift], 1u);
      }
      sync();
      // lane i has counters 4 i .. 4 i + 3; counted from the largest down
      uint32_t c[4], mine = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) c[x] = hist[4 * lane + x], mine += c[x];
      const uint32_t from = sum_from(mine);
      uint32_t above = from - mine;
      const bool here = above < want && from >= want;
      uint32_t digit = 0, left = 0, full = 0;
#pragma unroll
      for (int x = 3; x >= 0; --x) {
        if (above < want && above + c[x] >= want) digit = 4 * lane + x, left = want - above, full = c[x] == left;
        above += c[x];
      }
      const int src = __ffsll((unsigned long long)__ballot(here)) - 1;
      digit = (uint32_t)__builtin_amdgcn_readlane((int)digit, src);
      want = (uint32_t)__builtin_amdgcn_readlane((int)left, src);
      lo += digit << shift;
      if (__builtin_amdgcn_readlane((int)full, src)) {  // all of this counter's keys
        limit = lo - 1u;
        break;
      }
      if (shift == 0) {
        limit = lo;
        ties = want;
        break;
      }
      hi = lo + min(hi - lo, (1u << shift) - 1u);
      if constexpr (W == 1) sync();
    }
  }
  // Each wave takes its part of the blocks, in order.
  const uint32_t part = ((n + W - 1) / W + 63u) & ~63u;
  const uint32_t b0 = min(n, wave * part), b1 = min(n, b0 + part);
  uint32_t first = 0, rank = 0, total = 0, ranks = 0;  // taken, and equal to the limit, before this part and in all
  if constexpr (W > 1) {
    uint32_t more = 0, same = 0;
    for (uint32_t i0 = b0; i0 < b1; i0 += kStrip * 64) {
      uint32_t k[kStrip];
      strip(i0 + lane, 64, b1, k);
#pragma unroll
      for (uint32_t x = 0; x < kStrip; ++x) {
        more += (uint32_t)__popcll(__ballot(k[x] > limit));
        same += (uint32_t)__popcll(__ballot(k[x] == limit && k[x] != kNoKey));
      }
    }
    if (lane == 0) sh.more[wave] = more, sh.same[wave] = same;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      if (w == wave) first = total, rank = ranks;
      total += sh.more[w] + min(sh.same[w], less(ties, ranks));
      ranks += sh.same[w];
    }
  }
  uint32_t at = first;
  const uint64_t below = (1ull << lane) - 1;
  for (uint32_t i0 = b0; i0 < b1; i0 += kStrip * 64) {
    uint32_t k[kStrip];
    strip(i0 + lane, 64, b1, k);
#pragma unroll
    for (uint32_t x = 0; x < kStrip; ++x) {
      bool take = k[x] > limit;
      if (ties) {
        const bool same = k[x] == limit;
        const uint64_t mask = __ballot(same);
        take |= same && rank + (uint32_t)__popcll(mask & below) < ties;
        rank += (uint32_t)__popcll(mask);
      }
      const uint64_t got = __ballot(take);
      if (got) {
        const uint32_t pos = at + (uint32_t)__popcll(got & below);
        if (take && pos < count) out[pos] = (int32_t)(i0 + lane + 64 * x);
        at += (uint32_t)__popcll(got);
      }
    }
  }
  // -1 behind them
  if constexpr (W == 1) total = at;
  for (uint32_t i = total + tid; i < count; i += 64 * W) out[i] = -1;
  if constexpr (W == 1) sync();
}

// A workgroup's head and its index over the rest: all heads of eight such indexes
// in turn, so that the heads of a block, whose bounds and scales share lines and
// pages, are read by one XCD (workgroups go round the eight).
struct Work {
  uint32_t h, rest;
};
__device__ __forceinline__ Work work_of(uint32_t kvh) {
  const uint32_t id = blockIdx.x;
  return Work{id / 8u % kvh, id / 8u / kvh * 8u + id % 8u};
}

// Scores in LDS, chosen by the workgroup that made them.
template <int D, bool BF, bool VEC>
__global__ __launch_bounds__(kSelThreads) void k_select(SelectArgs a) {
  extern __shared__ uint32_t lds_keys[];
  __shared__ Team teams[kSelWaves];
  __shared__ Shared shared;
  __shared__ __attribute__((aligned(16))) Codes<D> codes;
  const Work wk = work_of(a.c.kvh);
  const uint32_t h = wk.h;
  if (wk.rest >= a.slots) return;
  const TileAt at = tile_at(a.b, wk.rest, 1, a.ntok, a.tiles);
  if (at.sq >= a.b.seqs) return;
  const Tokens tk = tokens_of(a, at.sq, at.tile);
  if (tk.n == 0) return;
  clear_teams(teams);
  score_blocks<D, BF, VEC>(a, tk, h, 0, tk.seen(a, tk.n - 1), lds_keys, a.blocks, codes);
  __syncthreads();
  const size_t out = ((size_t)tk.row * a.c.kvh + h) * a.count;
  if (a.ntok == 1) {
    choose<kSelWaves>(lds_keys, tk.seen(a, 0), a.count, a.chosen + out, teams, shared);
  } else {
    const uint32_t wave = threadIdx.x >> 6;
    for (uint32_t t = wave; t < tk.n; t += kSelWaves)
      choose<1>(lds_keys + (size_t)t * a.blocks, tk.seen(a, t), a.count,
                a.chosen + out + (size_t)t * a.c.kvh * a.count, teams + wave, shared);
  }
}

// Scores to memory, the blocks shared out over workgroups.
template <int D, bool BF, bool VEC>
__global__ __launch_bounds__(kSelThreads) void k_score(SelectArgs a) {
  __shared__ __attribute__((aligned(16))) Codes<D> codes;
  const Work wk = work_of(a.c.kvh);
  const uint32_t h = wk.h, chunk = wk.rest % a.chunks, id = wk.rest / a.chunks;
  if (id >= a.slots) return;
  const TileAt at = tile_at(a.b, id, 1, a.ntok, a.tiles);
  if (at.sq >= a.b.seqs) return;
  const Tokens tk = tokens_of(a, at.sq, at.tile);
  if (tk.n == 0) return;
  const uint32_t from = chunk * a.per, to = min(tk.seen(a, tk.n - 1), from + a.per);
  if (from < to)
    score_blocks<D, BF, VEC>(a, tk, h, from, to, a.keys + ((size_t)tk.row * a.c.kvh + h) * a.blocks,
                             (size_t)a.c.kvh * a.blocks, codes);
}

__global__ __launch_bounds__(kSelThreads) void k_top(SelectArgs a) {
  __shared__ Team teams[kRounds];
  __shared__ Shared shared;
  const uint32_t h = blockIdx.x % a.c.kvh;
  const uint32_t row = blockIdx.x / a.c.kvh;
  const uint32_t sq = seq_at(a.b, row);
  const Seq s = seq_of(a.b, sq, a.c.bsh);
  if (row < s.row || row - s.row >= s.n) return;
  const Tokens tk{sq, row, 1, s.first + (row - s.row), s.len};
  const size_t unit = (size_t)row * a.c.kvh + h;
  clear_teams(teams);
  __syncthreads();
  choose<kSelWaves>(a.keys + unit * a.blocks, tk.seen(a, 0), a.count, a.chosen + unit * a.count, teams, shared);
}

}  // namespace
}  // namespace kv
}  // namespace dance

namespace dance {
namespace kv {
namespace {

// Keys that a workgroup may keep: 96 KB, so that its counters and others' LDS fit beside it.
constexpr uint64_t kLdsKeys = 24576;
// A few long rows: scores by many workgroups, to memory and back. Whole calls, of one
// workgroup a row and so: 8 rows of 512 blocks 12.5 and 14.0 us, of 1024 16.7 and 14.9, of
// 2048 24.1 and 16.0; 64 rows of 1024 17.6 and 16.9, 128 rows of 1024 19.4 and 23.4 us.
constexpr uint64_t kFewUnits = 64, kManyBlocks = 768;

struct SelectPlan {
  bool fused;
  uint32_t gp, ntok, tiles, slots, blocks;
};
SelectPlan select_plan(const DanceKvCache* c, const DanceKvBatch* b, uint32_t heads) {
  SelectPlan p{};
  const uint32_t group = heads / c->kv_heads;
  p.gp = 1;
  while (p.gp < group && p.gp < 16) p.gp *= 2;
  p.blocks = most_blocks(c, b);
  uint64_t ntok = group > 16 ? 1 : (uint64_t)kRowTiles * (16 / p.gp);
  if (ntok > b->max_tokens) ntok = b->max_tokens;
  const uint64_t units = (uint64_t)b->seqs * c->kv_heads;
  p.fused = p.blocks <= kLdsKeys && !(b->max_tokens == 1 && units <= kFewUnits && p.blocks > kManyBlocks);
  if (p.fused && ntok * p.blocks > kLdsKeys) ntok = kLdsKeys / p.blocks;
  p.ntok = (uint32_t)ntok;
  p.tiles = (uint32_t)((b->max_tokens + ntok - 1) / ntok);
  p.slots = (uint32_t)tile_slots(b, 1, ntok, p.tiles);
  return p;
}

}  // namespace
}  // namespace kv
}  // namespace dance

using namespace dance::kv;

extern "C" {

size_t dance_kv_select_work(const DanceKvCache* cache, const DanceKvBatch* batch, uint32_t heads, uint32_t count) {
  if (check_shapes(cache, batch) || heads == 0 || heads % cache->kv_heads || count == 0 || batch->tokens == 0) return 0;
  const SelectPlan p = select_plan(cache, batch, heads);
  return p.fused ? 0 : (size_t)batch->tokens * cache->kv_heads * p.blocks * 4;
}

int dance_kv_select(const DanceKvCache* cache, const DanceKvBatch* batch, const DanceKvRows* queries, uint32_t count,
                    uint32_t sink, uint32_t recent, int32_t* chosen, void* work, size_t work_bytes, void* stream) {
  const char* why = check_common(cache, batch);
  if (!why) why = check_rows(cache, queries, false);
  if (!why && !chosen) why = "null output";
  if (!why && (count == 0 || count > 0x7FFFFFFFu || (uint64_t)sink + recent > count))
    why = "count must be positive and hold sink and recent";
  if (why) KV_ERR("dance_kv_select", "%s", why);
  if (batch->tokens == 0) return 0;
  const SelectPlan p = select_plan(cache, batch, queries->heads);
  const size_t need = dance_kv_select_work(cache, batch, queries->heads, count);
  if (need && (!work || work_bytes < need || !aligned(work, 16)))
    KV_ERR("dance_kv_select", "work must hold %zu bytes, aligned to 16", need);
  const uint32_t per = kSelWaves * 16u;
  const uint32_t chunks = p.fused ? 1u : (p.blocks + per - 1) / per;
  const uint64_t units = (uint64_t)batch->tokens * cache->kv_heads;
  const uint64_t grid = ((uint64_t)p.slots * chunks + 7) / 8 * 8 * cache->kv_heads;
  if (grid * kSelThreads > 0xFFFFFFFFull || (!p.fused && units * kSelThreads > 0xFFFFFFFFull))
    KV_ERR("dance_kv_select", "batch is too large for one launch");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const SelectArgs a{cache_args(cache), batch_args(batch), rows_args(queries), queries->heads / cache->kv_heads, p.gp,
                     p.ntok, p.tiles, p.slots, count, sink, recent, p.blocks, chunks, per, static_cast<uint32_t*>(work), chosen};
  const bool vec = rows_vector(queries);
  const size_t lds = (size_t)p.ntok * p.blocks * 4;
  with_kind(cache->dim, queries->dtype, [&](auto d, auto bf) {
    auto go = [&](auto v) {
      constexpr int D = decltype(d)::value;
      constexpr bool BF = decltype(bf)::value, V = decltype(v)::value;
      if (p.fused)
        hipLaunchKernelGGL((k_select<D, BF, V>), dim3((uint32_t)grid), dim3(kSelThreads), lds, st, a);
      else
        hipLaunchKernelGGL((k_score<D, BF, V>), dim3((uint32_t)grid), dim3(kSelThreads), 0, st, a);
    };
    vec ? go(std::true_type{}) : go(std::false_type{});
  });
  if (!p.fused) hipLaunchKernelGGL(k_top, dim3((uint32_t)units), dim3(kSelThreads), 0, st, a);
  return launched("dance_kv_select");
}

}  // extern "C"
