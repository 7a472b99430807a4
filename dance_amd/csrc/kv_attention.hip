// dance_kv_attention and dance_kv_sparse_attention (include/dance_kv.h), dance_kv_cross_attention
// (include/dance_kv_parts.h).
//
// For a tile of 64 tokens (32 at 256 dimensions) and 16 query rows a wave forms S' = K Q' (tokens x
// rows) and then O' += V' P' (dims x rows) with 16x16x32 f16 MFMAs. Codes are
// whole numbers below 2^11, so they are exact in f16, and the scales stay out
// of the products: a key's scale multiplies its logit, a value's the weight.
//
// Both products may take their inner dimension in any order, as long as both
// operands do. The wave uses that so that nothing is shuffled or staged:
//  - row m of the key operand's subtile s is token 16 (m / 4) + 4 s + m % 4, so that
//    the lane group g = lane / 16 finds in its result registers the logits of the
//    16 adjacent tokens 16 g .. 16 g + 15, which lie in one block (one scale);
//  - those registers are, in their order, the weights' operand of the second
//    product, whose value operand is then 16 adjacent bytes of a dimension's
//    tokens: one load, as values lie dims-major;
//  - of keys and queries lane group g holds every fourth piece of 16 dimensions (8
//    where dim is no multiple of 64): a load then takes 64 adjacent bytes of a token.
// Codes go from memory to the registers that the MFMAs read; every code is
// read once per 16 rows.
//
// Softmax, in log2 units: with s a scaled logit and y its value's scale, the second
// product takes p = 2^(s + log2 y - R), and the row's sum is l = sum p / y; the result is
// the product over l. The logit's scale, log2 y and R make one fma of it. R is a running reference per
// row that stays until s + log2 y exceeds it by kLift + kSlack: p is then at most
// 2^(kLift + kSlack), inside f16, which rounds it to 11 bits (down to 2^-27 of a row's largest; the
// f16 outputs have 11 bits too). l and all sums are float32, l of unrounded
// p. Scales below 2^kLeastExp count as that, so that 1 / y is finite. l is held in units of 1 /
// kSumUnit: where all values are zero or of the least scale a token adds up to 2^(15 + 100) to it, and a
// table row's 2^31 tokens stay below 2^128. A token of such a block beside blocks of larger values counts in
// l where its weight is more than 2^-41 times their scale of theirs (p is then a normal number).
//
// Bound by the codes' bytes: a step reads each once and does 4 operations on it per row. Measured (8 kv
// heads of 4, 128 dimensions): 64 sequences of 500 to 12,000 tokens, 497 MB, 105 us (4.7 TB/s; a stream that only
// reads reaches 6.5, a large copy 4.8); 2 of 400,000 to 600,000, 461 MB, 85 us (5.4 TB/s) and 11 of join; 16 rows over
// 64 listed blocks of 64 tokens each, 135 MB, 28 us (4.7 TB/s). One sequence of 700 tokens takes 9.8 us, a chain of
// dependent loads. Lists of 1026 rows over the same 145 MB are bound by instructions (64 % of the cycles) and by
// what the L2s miss of them (1.4 GB): 312 us.

#include <cfloat>
#include <cmath>
#include <type_traits>

#include "../../include/dance_kv_parts.h"
#include "kv_common.h"

namespace dance {
namespace kv {
namespace {

constexpr uint32_t kStepWaves = 4;
constexpr uint32_t kJoinWaves = 8;       // of k_join
constexpr uint32_t kJoinCrossWaves = 4;  // of k_join_cross
constexpr uint32_t kJoinFew = 16;        // splits that k_join_few takes, of rows that see their own part
// Cross attention joins by rows (k_join, k_join_cross) below this many rows for each split: a workgroup a row costs 5.6 ns
// a row, a lane that walks its splits 0.4 us a split of few rows. Measured, calls of 16 heads of 64 in a graph, by rows and
// with k_join_few: 64 rows of 4 splits 9.3 and 9.6 us, of 16 9.4 and 15.5; 1024 of 4 10.8 and 10.2, of 16 17.2 and 22.7; 8192
// of 8 38.8 and 30.1, of 24 68.3 and 70.0. The limit is a straight line through a curve: 1024 rows of 8 splits (13.3 and
// 14.2) and 8192 of 64 (151 and 166) take k_join_few, which is 7 and 9 % slower there.
constexpr uint64_t kJoinRows = 128;
constexpr uint64_t kJoinCrossRows = 256;  // from here on k_join_cross
constexpr uint32_t kJoinThreads = 256;    // of k_join_few
constexpr uint32_t join_rows(uint32_t dim) { return kJoinThreads / (dim / 4); }
constexpr uint32_t kRowTile = 16;
// Waves of a workgroup that takes all of a row tile's tokens. It needs no join (and
// its launch), but a CU reads 75 GB/s at most: up to one workgroup per CU and
// kWideBytes of codes for each, more where many keep the chip busy anyway. Measured
// with it and with splits, whole calls: of 128 dimensions 8 units of 1024 tokens 11.2 and 11.1 us, of 2048 16.3 and
// 14.2, 256 of 2048 (512 KB) 23.6 and 27.0, 128 of 4096 (1 MB) 29.0 and 27.2; of 64 dimensions 72 units of 3000 (384 KB)
// 14.8 and 13.0, 128 of 3000 15.5 and 16.5, 216 of 3500 (448 KB) 19.7 and 24.1.
constexpr uint32_t kWideWaves = 8;
constexpr uint64_t kWideUnits = 256, kWideBytes = 256 << 10;
// k_chunk for sequences of more than 64 rows (of a kv head, on average; 256 at 192 dimensions, where a
// workgroup of 128 rows that is not full costs more than it gains) where that is expected to be faster. k_step's time goes with its row tiles x (tokens that they see + 128), k_chunk's with the longest
// chain of tiles in a workgroup, which splits keep from growing beyond some 12; both in tiles of 64 tokens, and
// the ratio by measurement. Of 901 shapes (64 to 256 dimensions; 8, 12 and 2 kv heads; 1 to 32 sequences; 40 to 8192 rows; 128
// to 32,768 tokens) calls take 1.2 % more on average than with the faster kernel, 29 % where 64 rows alone decide; of
// 139 ragged batches 3.7 %.
// Measured, whole calls (bf16, 8 kv heads of 4; prompts without and rows behind earlier tokens), k_step and k_chunk:
//   dim  sequences x rows / tokens   us              dim  sequences x rows / tokens   us
//   128  1 x 1024 / 256       9 and 13               64   1 x 256 / 8192      26 and 29
//   128  1 x 4096 / 1024     44 and 34               64   8 x 192 / 2048      32 and 29
//   128  8 x 512 / 128       25 and 11               64   32 x 72 / 8192     134 and 187
//   128  8 x 2048 / 512     118 and 54               64   32 x 256 / 8192    382 and 244
//   128  1 x 96 / 8192       24 and 31               192  1 x 2048 / 512      24 and 31
//   128  1 x 256 / 8192      40 and 35               192  8 x 1024 / 256      64 and 41
//   128  8 x 96 / 600        15 and 25               192  8 x 192 / 8192     178 and 204
//   128  32 x 256 / 8192    726 and 383              192  32 x 256 / 8192    881 and 765
//   256  1 x 96 / 8192       43 and 48               256  32 x 72 / 8192     612 and 476
// The average, because k_step's grid goes by the rows: 63 single tokens beside a prompt's 512, over 8192 each,
// 128 dimensions (36 rows) take 368 and 528 us, beside 2048 (132 rows) 822 and 580. The lengths are not known here
// but for the longest: prompts as ragged as 3 to 1270 tokens (12 heads of 96) take 24 and 34 us.
bool chunk_pays(uint32_t dim, uint64_t heads, uint64_t group, uint64_t tokens, uint64_t seqs, uint64_t longest) {
  const uint64_t rows = group * tokens / seqs, own = tokens / seqs < longest ? tokens / seqs : longest;
  if (rows <= (dim == 192 ? 255 : 64)) return false;
  const uint64_t row_tiles = heads / group * seqs * ((rows + kRowTile - 1) / kRowTile), seen = longest - own / 2;
  const uint64_t chain = (longest + 63) / 64 < 12 ? (longest + 63) / 64 : 12;
  return row_tiles * (128 + seen) / 64 >= (dim <= 192 ? 1280 : 800) * chain;
}
// Its workgroups have eight waves where that gives each CU two of them, else four:
// 521 and 557 us for two chunks of 2048 tokens over 6000 to 10000, 41 and 34 us for
// 1024 over 1024. Below one workgroup per CU the tokens are split, up to kChunkUnits workgroups
// of at least kChunkSplitTiles tiles (64 tokens over 8192: 38 us at 8 tiles, 42 at 16).
constexpr uint64_t kChunkSplitTiles = 8;
constexpr uint64_t kChunkUnits = 512;
constexpr int kChunkWide = 8, kChunkSmall = 4;
constexpr float kLift = 13.f, kSlack = 2.f;
constexpr float kLeastScale = 0x1p-100f;  // 2^kLeastExp
// Least factor of a product: above 0, so that a hidden token's, -infinity, stays that.
constexpr float kLeastFactor = 0x1p-120f;
constexpr float kSumUnit = 0x1p-20f;  // of l, see above
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t kSplitUnits = 1024;  // workgroups that fill the chip several times over
constexpr uint32_t kSplitTiles = 16;    // least tiles of a split: its partial sums are then 2 to 6 % of what it reads

struct StepArgs {
  Cache c;
  Batch b;
  Rows q;
  const int32_t* __restrict__ lists;  // LIST: tokens x kv_heads x count
  uint32_t count;
  float scale2;  // scale * log2(e)
  uint32_t group, tiles, slots, splits, per;  // row tiles of a sequence (0: see tile_at), of all; tiles of a split
  uint16_t* __restrict__ out;
  float* __restrict__ lse;
  float* __restrict__ part;  // splits > 1: [row][split][D] sums, then [row][split][2] (R, l)
  bool full;                 // rows see all tokens, whatever their own place
};

// A sum of many tiles with what its additions rounded off: without it the logarithm of 140,000
// tokens' sum is off by 2e-5 where a wave walks them all.
struct Sum {
  float x = 0.f, low = 0.f;
  __device__ __forceinline__ void add(float y) {
    y -= low;
    const float t = x + y;
    low = (t - x) - y;
    x = t;
  }
  __device__ __forceinline__ void scale(float f) {
    x *= f;
    low *= f;
  }
};

// ln(l 2^R / kSumUnit). R and the exponent of l are of opposite signs and about one size: their sum
// first, or the logarithm's rounding is that of the larger number.
__device__ __forceinline__ float lse_of(float R, float l) {
  if (l == 0.f) return -__builtin_inff();
  const bool small = l < 1.f;  // perhaps subnormal in its unit
  const uint32_t u = __float_as_uint(small ? l * (1.f / kSumUnit) : l);
  const float e = (float)((int)(u >> 23) - (small ? 127 : 107)), m = __uint_as_float((u & 0x7FFFFFu) | 0x3F800000u);
  return l < __builtin_inff() ? ((R + e) + log2f(m)) * kLn2 : l;  // l is finite, infinite or NaN
}
static_assert(kSumUnit == 0x1p-20f, "lse_of's exponents");

// Four of a row's sums over l, as the output's type; zeros where nothing was summed. The
// unit goes to the factor that it leaves normal.
template <bool BF>
__device__ __forceinline__ u2_t quotients(f4_t o, float l) {
  const bool small = l < 1.f;
  const float unit = small ? 1.f : kSumUnit, inv = l > 0.f ? 1.f / (small ? l * (1.f / kSumUnit) : l) : 0.f;
  uint16_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = store_val<BF>(l == 0.f ? 0.f : o[i] * unit * inv);
  return u2_t{y[0] | (uint32_t)y[1] << 16, y[2] | (uint32_t)y[3] << 16};
}

// Tokens of a tile: what leaves the registers room for two waves on a SIMD.
constexpr int step_tile(int d) { return d <= 192 ? 64 : 32; }

template <int D, bool BF, bool LIST, bool VEC, uint32_t W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2))) void k_step(StepArgs a) {
  constexpr int KS = D / 32;  // inner steps of the first product
  constexpr int DT = D / 16;  // row tiles of the second
  constexpr int KW = D / 16;  // words of a key row that a lane holds
  constexpr int ST = step_tile(D) / 16;  // subtiles of 16 tokens
  constexpr uint32_t kTile = 16 * ST, kGroup = 4 * ST;  // tokens of a tile, of a lane group
  constexpr int kPiece = KW % 4 == 0 ? 16 : 8;
  // rows 16 bytes longer than their values: 16 of them lie in different banks
  __shared__ __attribute__((aligned(16))) float sm_o[W][kRowTile][D + 4];
  __shared__ float sm_m[W][kRowTile], sm_l[W][kRowTile];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t n = lane & 15u, g = lane >> 4;
  const uint32_t bsh = a.c.bsh, bs = 1u << bsh;
  uint32_t id = blockIdx.x;
  // Heads fastest and splits slowest: workgroups go round the XCDs, and the first splits, which
  // all sequences have, must not all meet on the same ones (with splits
  // fastest, 8 of them: 215 us for a ragged batch that takes 120 like this).
  const uint32_t h = id % a.c.kvh;
  id /= a.c.kvh;
  const uint32_t split = id / a.slots;
  id %= a.slots;
  TileAt at;
  if constexpr (LIST) {
    at.tile = id % a.tiles;
    id /= a.tiles;  // the token row
    at.sq = seq_at(a.b, id);
  } else {
    at = tile_at(a.b, id, a.group, kRowTile, a.tiles);
    if (at.sq >= a.b.seqs) return;
  }
  const uint32_t sq = at.sq, tile = at.tile;
  const Seq s = seq_of(a.b, sq, bsh);
  // rows of the tile: index r counts (token, head of the group), tokens slowest
  uint32_t r_first, r_end;
  if constexpr (LIST) {
    if (id < s.row || id - s.row >= s.n) return;
    r_first = (id - s.row) * a.group + tile * kRowTile;
    r_end = (id - s.row + 1) * a.group;
  } else {
    r_first = tile * kRowTile;
    r_end = s.n * a.group;
  }
  if (r_first >= r_end) return;
  const uint32_t rows = min(kRowTile, r_end - r_first);
  const uint32_t r = r_first + min(n, rows - 1u);
  const uint32_t tok = r / a.group, head = h * a.group + r % a.group;
  // last position that this lane's row sees, and that any row of the tile does
  const int64_t p_all = s.len - 1, p_row = a.full ? p_all : min(s.first + tok, p_all);
  const int64_t p_top = a.full ? p_all : min(s.first + (r_first + rows - 1) / a.group, p_all);
  const int32_t pos = n < rows && p_row >= 0 ? (int32_t)p_row : -1, top = p_top >= 0 ? (int32_t)p_top : -1;
  const int32_t seen = (int32_t)((uint32_t)(top + 1 + (int32_t)bs - 1) >> bsh);  // blocks
  const int32_t* const list = LIST ? a.lists + ((size_t)id * a.c.kvh + h) * a.count : nullptr;
  uint32_t entries = (uint32_t)seen;
  if constexpr (LIST) {  // up to the last one that the row sees: a selection of few blocks ends in -1
    entries = 0;
    for (uint32_t e0 = 0; e0 < a.count; e0 += 64) {
      const int32_t lg = e0 + lane < a.count ? list[e0 + lane] : -1;
      const uint64_t mask = __ballot(lg >= 0 && lg < seen);
      if (mask) entries = e0 + 64u - (uint32_t)__clzll((long long)mask);
    }
    entries = (uint32_t)__builtin_amdgcn_readfirstlane((int)entries);
  }
  const int32_t* const table = a.b.table + (size_t)sq * a.b.width;

  // this split's tiles of listed tokens
  const uint32_t all = (uint32_t)(((uint64_t)entries * bs + kTile - 1) / kTile);
  const uint32_t t_end = split + 1 < a.splits ? min(all, (split + 1) * a.per) : all;
  float* const part_ml = a.part + (size_t)a.b.tokens * a.q.heads * a.splits * D;  // splits > 1
  auto row_of = [&](uint32_t rr) {
    const uint32_t rw = r_first + rr;
    return (size_t)(s.row + rw / a.group) * a.q.heads + h * a.group + rw % a.group;
  };
  if (a.splits > 1 && split * a.per >= all) {  // beyond the end
    if (threadIdx.x < rows) {
      float* const pm = part_ml + (row_of(threadIdx.x) * a.splits + split) * 2;
      pm[0] = -FLT_MAX;
      pm[1] = 0.f;
    }
    return;
  }

  f4_t acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f4_t{0.f, 0.f, 0.f, 0.f};
  float R = -FLT_MAX;
  Sum l;

  // Loads run ahead in the registers that the products have read: the next
  // tile's keys set out behind the first product, its values behind the second, the
  // place of the tile after that one between them, and what a list says of the tile after
  // that. Nothing that has just been asked for is looked at (loads come back in
  // order: to look at the last is to wait for all).
  // Lane group g has the place of its 16 tokens' block: listed (logical), then in the cache (raw).
  auto listed = [&](uint32_t tt) -> int32_t {
    const uint32_t e = (tt * kTile + g * kGroup) >> bsh;
    return e < entries ? LIST ? list[e] : (int32_t)e : -1;
  };
  struct Place {
    int32_t raw, first;  // first: position of the first of the 16 tokens
  };
  auto place = [&](uint32_t tt, int32_t lg) {
    Place p;
    p.raw = lg >= 0 && lg < seen ? table[lg] : -1;
    p.first = (int32_t)(((uint32_t)lg << bsh) + ((tt * kTile + g * kGroup) & (bs - 1u)));
    return p;
  };
  auto block = [&](const Place& p) -> int32_t { return (uint32_t)p.raw < a.c.blocks ? p.raw : -1; };  // -1: a hole
  uint32_t kw[ST][KW];
  typedef uint32_t codes_t __attribute__((ext_vector_type(ST)));
  codes_t vw[DT];
  float ks, vs;
  auto load_keys = [&](uint32_t tt, const Place& p) {
    const uint32_t slot = (tt * kTile + (n >> 2) * kGroup) & (bs - 1u);
    const size_t cell = (size_t)max(__shfl(block(p), (int)((n >> 2) * 16u)), 0) * a.c.kvh + h;
    const int8_t* const kp = a.c.k + ((cell << bsh) + slot + (n & 3u)) * D + g * kPiece;
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      if constexpr (KW % 4 == 0) {
#pragma unroll
        for (int i = 0; i < KW / 4; ++i) {
          const u4_t w = *reinterpret_cast<const u4_t*>(kp + (size_t)st * 4 * D + i * 64);
          kw[st][4 * i] = w.x, kw[st][4 * i + 1] = w.y, kw[st][4 * i + 2] = w.z, kw[st][4 * i + 3] = w.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < KW / 2; ++i) {
          const u2_t w = *reinterpret_cast<const u2_t*>(kp + (size_t)st * 4 * D + i * 32);
          kw[st][2 * i] = w.x, kw[st][2 * i + 1] = w.y;
        }
      }
    }
  };
  auto load_values = [&](uint32_t tt, const Place& p) {
    const uint32_t slot = (tt * kTile + g * kGroup) & (bs - 1u);
    const size_t cell = (size_t)max(block(p), 0) * a.c.kvh + h;
    const int8_t* const vp = a.c.v + ((cell * D + n) << bsh) + slot;
#pragma unroll
    for (int t = 0; t < DT; ++t) vw[t] = *reinterpret_cast<const codes_t*>(vp + ((size_t)(16 * t) << bsh));
  };
  auto load_scales = [&](const Place& p) {
    const float2 x = *reinterpret_cast<const float2*>(a.c.scale + ((size_t)max(block(p), 0) * a.c.kvh + h) * 2);
    ks = x.x;
    vs = x.y;
  };

  uint32_t tt = split * a.per + wave;
  const bool any = tt < t_end;
  Place here, next;
  int32_t then = -1;
  if (any) {
    const int32_t l0 = listed(tt), l1 = listed(tt + W);
    then = listed(tt + 2 * W);
    here = place(tt, l0);
    next = place(tt + W, l1);
  }
  u4_t raw[KS];
  {
    const uint16_t* src = a.q.data + (int64_t)(s.row + tok) * a.q.token_stride + (int64_t)head * a.q.head_stride + g * kPiece;
#pragma unroll
    for (int c = 0; c < KS; ++c) {
      const uint16_t* const at = src + (kPiece == 16 ? 64 * (c / 2) + 8 * (c % 2) : 32 * c);
      if constexpr (VEC) {
        raw[c] = *reinterpret_cast<const u4_t*>(at);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[c][i] = (uint32_t)at[2 * i] | (uint32_t)at[2 * i + 1] << 16;
      }
    }
  }
  if (any) {
    load_scales(here);
    load_keys(tt, here);
    load_values(tt, here);
  }
  // Queries, as f16 with a power of two taken out so that bf16's range fits. A negative
  // scale turns them over, so that the largest product has the largest logit.
  h8_t qf[KS];
  float qscale = fabsf(a.scale2);
  const uint32_t flip = a.scale2 < 0.f ? 0x80008000u : 0u;
  if constexpr (BF) {
    float mag = 0.f;
#pragma unroll
    for (int c = 0; c < KS; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) mag = fmaxf(mag, finite_abs(load_val<true>((uint16_t)(raw[c][i >> 1] >> (16 * (i & 1))))));
    mag = rows_max(mag);
    int e = (int)(__float_as_uint(mag) >> 23) - 127 - 10;  // the largest becomes 2^10 .. 2^11
    e = e < -120 ? -120 : e;  // so that the scale keeps its bits
    const float inv = exp2_int(-e);
    qscale *= exp2_int(e);
#pragma unroll
    for (int c = 0; c < KS; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        qf[c][i] = (_Float16)(load_val<true>((uint16_t)((raw[c][i >> 1] ^ flip) >> (16 * (i & 1)))) * inv);
  } else {
#pragma unroll
    for (int c = 0; c < KS; ++c) qf[c] = __builtin_bit_cast(h8_t, raw[c] ^ u4_t{flip, flip, flip, flip});
  }

  for (; tt < t_end; tt += W) {
    // tokens of this lane that its row sees: the first `lim` + 1
    const bool hole = block(here) < 0;
    const int32_t lim = !hole && here.first <= pos ? pos - here.first : -1;
    const float y = hole ? 1.f : fmaxf(vs, kLeastScale), iv = 1.f / y;
    const float kq = fmaxf(hole ? 0.f : ks * qscale, kLeastFactor);
    const float lv = __builtin_amdgcn_logf(y);
    const bool more = tt + W < t_end;
    f4_t sc[ST];
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      sc[st] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KS; ++c)
        sc[st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(kw[st][2 * c], kw[st][2 * c + 1]), qf[c], sc[st], 0, 0, 0);
    }
    if (more) {
      load_scales(next);
      load_keys(tt + W, next);
    }
    if (__any(lim < (int)kGroup - 1)) {
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * st + i > lim) sc[st][i] = -__builtin_inff();
    }
    float most = -__builtin_inff();
#pragma unroll
    for (int st = 0; st < ST; ++st)
#pragma unroll
      for (int i = 0; i < 4; ++i) most = fmaxf(most, sc[st][i]);
    const float big = __builtin_fmaf(most, kq, lv);
    if (__any(big > R + (kLift + kSlack))) {
      // each row by its own logits alone: a row's result does not depend on its neighbours
      const float row_big = rows_max(big);
      const float r_new = row_big > R + (kLift + kSlack) ? row_big - kLift : R;
      const float f = exp2f(R - r_new);
      l.scale(f);
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] *= f;
      R = r_new;
    }
    h8_t pf[ST / 2];
    float add = 0.f;
    const float off = lv - R;
#pragma unroll
    for (int u = 0; u < ST / 2; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * u + (i >> 2)][i & 3], kq, off));
        add += p;
        pf[u][i] = (_Float16)p;
      }
    l.add(add * iv * kSumUnit);
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      asm volatile("" : "+v"(vw[t]));  // values are waited for here, not where their conversion could begin
#pragma unroll
      for (int u = 0; u < ST / 2; ++u)
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vw[t][2 * u], vw[t][2 * u + 1]), pf[u], acc[t], 0, 0, 0);
    }
    if (more) {
      here = next;
      next = place(tt + 2 * W, then);
      then = listed(tt + 3 * W);
      load_values(tt + W, here);
    }
  }

  // The waves' sums meet in LDS, in wave order.
  const float sum_l = rows_sum(l.x);
  if (g == 0) {
    sm_m[wave][n] = R;
    sm_l[wave][n] = sum_l;
  }
  if (n < rows)
#pragma unroll
    for (int t = 0; t < DT; ++t) *reinterpret_cast<f4_t*>(&sm_o[wave][n][16 * t + 4 * g]) = acc[t];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < rows * (D / 4); i += 64 * W) {
    const uint32_t rr = i / (D / 4), d = i % (D / 4) * 4;
    float m = sm_m[0][rr];
#pragma unroll
    for (uint32_t w = 1; w < W; ++w) m = fmaxf(m, sm_m[w][rr]);
    float sum = 0.f;
    f4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      const float f = exp2f(sm_m[w][rr] - m);
      sum += f * sm_l[w][rr];
      const f4_t y = *reinterpret_cast<const f4_t*>(&sm_o[w][rr][d]);
#pragma unroll
      for (int x = 0; x < 4; ++x) o[x] += f * y[x];
    }
    const size_t row = row_of(rr);
    if (a.splits > 1) {
      *reinterpret_cast<f4_t*>(a.part + (row * a.splits + split) * D + d) = o;
      if (d == 0) {
        float* const pm = part_ml + (row * a.splits + split) * 2;
        pm[0] = m;
        pm[1] = sum;
      }
    } else {
      *reinterpret_cast<u2_t*>(a.out + row * D + d) = quotients<BF>(o, sum);
      if (a.lse && d == 0) a.lse[row] = lse_of(m, sum);
    }
  }
}

#include "kv_chunk.h"

// Joins a row's few splits. Every lane has four dimensions and reads all
// splits' references itself, so that nothing is exchanged (7 ragged prompts, 12 heads of 96, 2
// splits: 6.4 us, bound by the splits' bytes; a wave a row that exchanged them 9.1).
template <int D, bool BF>
__global__ __launch_bounds__(kJoinThreads) void k_join_few(const float* __restrict__ part, uint32_t splits, uint64_t rows,
                                                           uint16_t* __restrict__ out, float* __restrict__ lse) {
  constexpr uint32_t L = D / 4;  // lanes of a row
  const uint64_t row = (uint64_t)blockIdx.x * join_rows(D) + threadIdx.x / L;
  const uint32_t d = threadIdx.x % L * 4;
  if (threadIdx.x / L >= join_rows(D) || row >= rows) return;
  const float2* const ml = reinterpret_cast<const float2*>(part + rows * splits * D) + row * splits;
  const float* const po = part + row * splits * D + d;
  float m = -FLT_MAX, total = 0.f;
  f4_t o = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t i0 = 0; i0 < splits; i0 += 4)
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) m = fmaxf(m, ml[min(i0 + u, splits - 1u)].x);
  for (uint32_t i0 = 0; i0 < splits; i0 += 4)
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t i = min(i0 + u, splits - 1u);
      const float2 e = ml[i];
      const float f = i0 + u < splits && e.y != 0.f ? exp2f(e.x - m) : 0.f;
      // a split without sums was not written: the first one's line again, which is no traffic
      const f4_t x = *reinterpret_cast<const f4_t*>(po + (size_t)(f != 0.f ? i : 0u) * D);
      total += f != 0.f ? f * e.y : 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] += f != 0.f ? f * x[c] : 0.f;
    }
  *reinterpret_cast<u2_t*>(out + row * D + d) = quotients<BF>(o, total);
  if (lse && d == 0) lse[row] = lse_of(m, total);
}

// Joins a row's many splits, W waves for the row: the weights of up to 64
// splits at a time in the lanes of every wave, the sums of the splits that have
// any shared out over the waves. (One wave per row that walked its splits took
// 155 us for 32 rows of 256 splits; eight so 11.)
template <int D, bool BF, uint32_t W>
__device__ __forceinline__ void join_row(const float* __restrict__ part, uint32_t splits, uint64_t rows, uint64_t row,
                                         uint16_t* __restrict__ out, float* __restrict__ lse) {
  constexpr uint32_t L = D / 4;  // lanes that a row of sums takes
  constexpr uint32_t P = 64 / L > 0 ? 64 / L : 1;
  __shared__ f4_t sums[W][64];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const float* const ml = part + rows * splits * D + row * splits * 2;
  const float* const po = part + row * splits * D;
  float m = -FLT_MAX;
  for (uint32_t i = lane; i < splits; i += 64) m = fmaxf(m, ml[2 * i]);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
  float total = 0.f;
  f4_t o = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t i0 = 0; i0 < splits; i0 += 64) {
    const uint32_t i = i0 + lane;
    const float l = i < splits ? ml[2 * i + 1] : 0.f;
    const float f = l != 0.f ? exp2f(ml[2 * i] - m) : 0.f;
    total += f * l;
    const uint32_t n = min(64u, splits - i0);
#pragma unroll 1
    for (uint32_t k0 = wave * P; k0 < n; k0 += 8 * W * P)
#pragma unroll
      for (uint32_t k = k0; k < k0 + 8 * W * P; k += W * P) {
        if (k >= n) continue;
        const uint32_t at = k + lane / L;
        const float other = __shfl(f, (int)min(at, 63u)), w = at < 64u && lane < P * L ? other : 0.f;
        // without sums: the first split's line again, as above
        const f4_t x = *reinterpret_cast<const f4_t*>(po + (size_t)(w != 0.f ? i0 + at : 0u) * D + lane % L * 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += w != 0.f ? w * x[c] : 0.f;
      }
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) total += __shfl_xor(total, x);
  sums[wave][lane] = o;
  __syncthreads();
  if (wave == 0 && lane < L) {
    f4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t w = 0; w < W; ++w)
#pragma unroll
      for (uint32_t p = 0; p < P; ++p)
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] += sums[w][p * L + lane][c];
    *reinterpret_cast<u2_t*>(out + row * D + lane * 4) = quotients<BF>(y, total);
    if (lse && lane == 0) lse[row] = lse_of(m, total);
  }
}
template <int D, bool BF>
__global__ __launch_bounds__(64 * kJoinWaves) void k_join(const float* __restrict__ part, uint32_t splits, uint64_t rows,
                                                          uint16_t* __restrict__ out, float* __restrict__ lse) {
  join_row<D, BF, kJoinWaves>(part, splits, rows, blockIdx.x, out, lse);
}
// Of cross attention, where there may be many rows too: 2048 rows of 32 splits 74 us in all with eight waves a row, 71 with
// four; 64 rows of 128 splits 32 and 34.
template <int D, bool BF>
__global__ __launch_bounds__(64 * kJoinCrossWaves) void k_join_cross(const float* __restrict__ part, uint32_t splits,
                                                                     uint64_t rows, uint16_t* __restrict__ out,
                                                                     float* __restrict__ lse) {
  join_row<D, BF, kJoinCrossWaves>(part, splits, rows, blockIdx.x, out, lse);
}

struct Plan {
  uint64_t units;  // row tiles of all sequences or token rows, x kv heads
  uint32_t tiles, slots, splits, per;
  bool wide, chunk;
  int waves;  // of a workgroup of k_chunk
  bool join;  // k_join, not k_join_few
  size_t work;
};
// Cross attention's plan: the kernel, the waves of a workgroup and the splits with the least expected time. Its rows see
// all tokens, so that a workgroup's work is known but for the lengths. A workgroup takes `per` tiles of 64 tokens (32
// at 256 dimensions in k_step) for 16 rows in k_step, whose waves share them out, and for 32 rows a wave in k_chunk; the
// fullest CU has `load` of them. Expected, in us: what begins and ends a call; the fourth root of the sum of the fourth
// powers of a wave's chain of tiles, a CU's tiles over its four SIMDs (with `start` more for each wave) and the codes'
// bytes; and the join. Fitted to 5,000 random shapes (64 to 256 dimensions, 1 to 20 kv heads of 1 to 16, 1 to 64 sequences,
// 1 to 1500 rows, 20 to 60,000 tokens) with up to 30 plans each: on 800 others the chosen plans take 2.3 % more than the
// best ones on average, those of the rules for rows that see their own part took 9 % more. 48 sequences of 1500 tokens, one row, 16
// heads of 64: 28 us in one split, 31 in the two of those rules. Known to be too kind to k_step: the bytes count once, whatever
// number of row tiles reads them, so that of the shapes with 17 to 128 rows a kv head one in ten takes k_step where k_chunk is
// better, by 11 % on average and up to 62 (20 sequences of 8 rows, 2 kv heads of 8, 64 dimensions, over 55,000 tokens).
struct Rates {
  double begin;
  double chain[5], tile[2][5];  // of each dimension; tile: of four waves, of eight
  double start[2], mb;          // mb: megabytes in a microsecond
};
constexpr Rates kStepRates{
    5.9, {1.1, 1.2, 1.4, 1.6, 1.2}, {{0.67, 0.93, 1.4, 1.8, 1.8}, {0.61, 0.97, 1.3, 1.6, 1.7}}, {1.3, 1.7}, 6.4};
constexpr Rates kChunkRates{
    8.7, {1.0, 1.4, 1.4, 0.0, 0.0}, {{0.59, 0.92, 1.0, 2.3, 3.1}, {0.52, 0.65, 0.73, 0.0, 0.0}}, {2.0, 3.2}, 120.0};
constexpr double kJoinMb = 2.6, kJoinTime = 2.5, kJoinFewTime = 2.0, kJoinFewSplit = 0.24;  // beside the bytes
constexpr uint32_t kCrossSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128};
constexpr uint64_t kCrossStepRows = 1200, kCrossUnits = 4096;

bool joins_rows(uint64_t rows, uint64_t splits) { return rows < kJoinRows * splits; }

void plan_cross(const DanceKvCache* c, const DanceKvBatch* b, uint32_t heads, Plan& p) {
  const uint64_t group = heads / c->kv_heads, rows = group * b->tokens / b->seqs, out_rows = (uint64_t)b->tokens * heads;
  const uint64_t longest = (uint64_t)most_blocks(c, b) * c->block_tokens;
  const uint32_t dim = c->dim == 64 ? 0 : c->dim == 96 ? 1 : c->dim == 128 ? 2 : c->dim == 192 ? 3 : 4;
  const double bytes = 2e-6 * c->dim * c->kv_heads * (double)b->seqs * (double)longest;
  double least = INFINITY;
  for (int chunk = 0; chunk < 2; ++chunk) {
    if (chunk ? rows <= kRowTile : rows > kCrossStepRows) continue;
    const Rates& r = chunk ? kChunkRates : kStepRates;
    const uint64_t tokens = chunk ? 64 : step_tile(c->dim), all = (longest + tokens - 1) / tokens;
    for (int wide = 0; wide < (chunk && c->dim > 128 ? 1 : 2); ++wide) {
      const int waves = wide ? 8 : 4;
      const uint32_t row_tile = chunk ? 32u * waves : kRowTile;
      uint32_t tiles = (uint32_t)((group * b->max_tokens + row_tile - 1) / row_tile);
      const uint64_t slots = tile_slots(b, group, row_tile, tiles), units = slots * c->kv_heads;
      uint64_t before = 0;  // the splits looked at last
      for (const uint32_t want : kCrossSplits) {
        const uint64_t per = (all + want - 1) / want, splits = (all + per - 1) / per;
        if (want > 1 && (per < (chunk ? 4u : (uint32_t)waves) || units * splits > kCrossUnits)) break;
        if (splits == before) continue;
        before = splits;
        const double load = (double)((units * splits + 255) / 256);
        const double chain = r.chain[dim] * (double)(chunk ? per : (per + waves - 1) / waves);
        const double work = r.tile[wide][dim] * ((double)per * (chunk ? waves : 1) + r.start[wide] * waves) * load / 4;
        const double read = bytes / r.mb, c2 = chain * chain, w2 = work * work, r2 = read * read;
        double time = r.begin + std::sqrt(std::sqrt(c2 * c2 + w2 * w2 + r2 * r2));
        const bool by_row = joins_rows(out_rows, splits);
        if (splits > 1)
          time += (by_row ? kJoinTime : kJoinFewTime + kJoinFewSplit * (double)splits) +
                  4e-6 / kJoinMb * (double)out_rows * (c->dim + 2) * (double)splits;
        if (time < least) {
          least = time;
          p.chunk = chunk;
          p.wide = !chunk && wide;
          p.waves = waves;
          p.tiles = tiles;
          p.slots = (uint32_t)slots;
          p.units = units;
          p.per = (uint32_t)per;
          p.splits = (uint32_t)splits;
          p.join = by_row;
        }
      }
    }
  }
  if (p.splits > 1) p.work = (size_t)out_rows * p.splits * (c->dim + 2) * 4;
}

enum Kind { kCausal, kFull, kList };
Plan plan(const DanceKvCache* c, const DanceKvBatch* b, uint32_t heads, Kind kind, uint32_t count) {
  const bool list = kind == kList;
  Plan p{};
  if (b->tokens == 0) return p;
  if (kind == kFull) {
    plan_cross(c, b, heads, p);
    return p;
  }
  const uint64_t group = heads / c->kv_heads;
  const uint64_t rows = list ? group : group * b->max_tokens;
  p.chunk = !list && chunk_pays(c->dim, heads, group, b->tokens, b->seqs, (uint64_t)most_blocks(c, b) * c->block_tokens);
  // by the rows that there are: sequences may have fewer than max_tokens
  const uint64_t big = 32 * kChunkWide;
  p.waves = c->dim <= 128 && (group * b->tokens + big - 1) / big * c->kv_heads >= kChunkUnits ? kChunkWide : kChunkSmall;
  const uint32_t row_tile = p.chunk ? 32u * p.waves : kRowTile;
  p.tiles = (uint32_t)((rows + row_tile - 1) / row_tile);
  const uint64_t slots = list ? (uint64_t)b->tokens * p.tiles : tile_slots(b, group, row_tile, p.tiles);
  p.slots = (uint32_t)slots;
  p.units = slots * c->kv_heads;
  // A split takes a fixed number of tiles, so that sequences of other lengths take
  // other numbers of workgroups.
  const uint64_t tokens = p.chunk ? 64 : step_tile(c->dim);  // of a tile
  const uint64_t all = ((uint64_t)(list ? count : most_blocks(c, b)) * c->block_tokens + tokens - 1) / tokens;
  p.wide = !p.chunk && p.units <= kWideUnits && all * tokens * 2 * c->dim <= kWideBytes + (p.units << 10);
  if (p.wide) {
    p.per = (uint32_t)all;
    p.splits = 1;
    return p;
  }
  const uint64_t want = p.chunk ? kChunkUnits : kSplitUnits, round = p.chunk ? 1 : kStepWaves;
  uint64_t per = p.chunk && p.units * 2 >= want ? all : (p.units * all + want - 1) / want;
  const uint64_t least = p.chunk ? kChunkSplitTiles : kSplitTiles;
  per = per < least ? least : (per + round - 1) / round * round;
  p.per = (uint32_t)(per < all ? per : all);
  p.splits = (uint32_t)((all + p.per - 1) / p.per);
  p.join = p.splits > kJoinFew;
  if (p.splits > 1) p.work = (size_t)b->tokens * heads * p.splits * (c->dim + 2) * 4;
  return p;
}

bool count_fits(const DanceKvCache* c, uint32_t count) {
  return count != 0 && (uint64_t)count * c->block_tokens <= 0x7FFFFFFFull;
}

int run(const char* who, const DanceKvCache* cache, const DanceKvBatch* batch, const DanceKvRows* q,
        const int32_t* lists, Kind kind, uint32_t count, float scale, void* out, float* lse, void* work,
        size_t work_bytes, void* stream) {
  const bool list = kind == kList;
  const char* why = check_common(cache, batch);
  if (!why) why = check_rows(cache, q, false);
  if (!why && (!out || !aligned(out, 16))) why = "out must be given, aligned to 16 bytes";
  if (!why && list && (!lists || !count_fits(cache, count)))
    why = "lists must be given, with 1 to 2^31 / block_tokens entries";
  if (!why && !(scale == scale && std::fabs(scale) < INFINITY)) why = "scale must be finite";
  if (why) {
    std::fprintf(stderr, "[%s] %s\n", who, why);
    return -1;
  }
  if (batch->tokens == 0) return 0;
  const Plan p = plan(cache, batch, q->heads, kind, count);
  if (p.work && (!work || work_bytes < p.work || !aligned(work, 16))) {
    std::fprintf(stderr, "[%s] work must hold %zu bytes, aligned to 16\n", who, p.work);
    return -1;
  }
  // Rows are counted in 31 bits, a launch's threads in 32; the joins' grids count where there is a join.
  const uint64_t grid = p.units * p.splits, rows = (uint64_t)batch->tokens * q->heads;
  const uint64_t join = p.splits > 1 && p.join ? rows * 64 * kJoinWaves
                        : p.splits > 1         ? (rows / join_rows(cache->dim) + 1) * kJoinThreads
                                            : 0;
  if (grid * 64 * 8 > 0xFFFFFFFFull || rows > 0x7FFFFFFFull || join > 0xFFFFFFFFull) {
    std::fprintf(stderr, "[%s] batch is too large for one launch\n", who);
    return -1;
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  StepArgs a{cache_args(cache), batch_args(batch), rows_args(q), lists, count, scale * kLog2e,
             q->heads / cache->kv_heads, p.tiles, p.slots, p.splits, p.per, static_cast<uint16_t*>(out), lse,
             static_cast<float*>(work), kind == kFull};
  const bool vec = rows_vector(q);
  with_kind(cache->dim, q->dtype, [&](auto d, auto bf) {
    constexpr int D = decltype(d)::value;
    constexpr bool BF = decltype(bf)::value;
    auto go = [&](auto l, auto v) {
      constexpr bool L = decltype(l)::value, V = decltype(v)::value;
      if constexpr (!L) {
        if (p.chunk) {
          if constexpr (D <= 128) {
            if (p.waves == kChunkWide) {
              hipLaunchKernelGGL((k_chunk<D, BF, V, kChunkWide>), dim3((uint32_t)grid), dim3(64 * kChunkWide), 0, st, a);
              return;
            }
          }
          hipLaunchKernelGGL((k_chunk<D, BF, V, kChunkSmall>), dim3((uint32_t)grid), dim3(64 * kChunkSmall), 0, st, a);
          return;
        }
      }
      if (p.wide)
        hipLaunchKernelGGL((k_step<D, BF, L, V, kWideWaves>), dim3((uint32_t)grid), dim3(64 * kWideWaves), 0, st, a);
      else
        hipLaunchKernelGGL((k_step<D, BF, L, V, kStepWaves>), dim3((uint32_t)grid), dim3(64 * kStepWaves), 0, st, a);
    };
    if (list)
      vec ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
    else
      vec ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
    if (p.splits > 1 && p.join && kind == kFull && rows >= kJoinCrossRows)
      hipLaunchKernelGGL((k_join_cross<D, BF>), dim3((uint32_t)rows), dim3(64 * kJoinCrossWaves), 0, st, a.part, p.splits, rows,
                         a.out, lse);
    else if (p.splits > 1 && p.join)
      hipLaunchKernelGGL((k_join<D, BF>), dim3((uint32_t)rows), dim3(64 * kJoinWaves), 0, st, a.part, p.splits, rows,
                         a.out, lse);
    else if (p.splits > 1)
      hipLaunchKernelGGL((k_join_few<D, BF>), dim3((uint32_t)((rows + join_rows(D) - 1) / join_rows(D))),
                         dim3(kJoinThreads), 0, st, a.part, p.splits, rows, a.out, lse);
  });
  return launched(who);
}

}  // namespace
}  // namespace kv
}  // namespace dance

using namespace dance::kv;

extern "C" {

int dance_kv_attention(const DanceKvCache* cache, const DanceKvBatch* batch, const DanceKvRows* queries, float scale,
                       void* out, float* lse, void* work, size_t work_bytes, void* stream) {
  return run("dance_kv_attention", cache, batch, queries, nullptr, kCausal, 0, scale, out, lse, work, work_bytes,
             stream);
}

size_t dance_kv_attention_work(const DanceKvCache* cache, const DanceKvBatch* batch, uint32_t heads) {
  if (check_shapes(cache, batch) || heads == 0 || heads % cache->kv_heads) return 0;
  return plan(cache, batch, heads, kCausal, 0).work;
}

int dance_kv_cross_attention(const DanceKvCache* cache, const DanceKvBatch* batch, const DanceKvRows* queries, float scale,
                             void* out, float* lse, void* work, size_t work_bytes, void* stream) {
  return run("dance_kv_cross_attention", cache, batch, queries, nullptr, kFull, 0, scale, out, lse, work, work_bytes,
             stream);
}

size_t dance_kv_cross_attention_work(const DanceKvCache* cache, const DanceKvBatch* batch, uint32_t heads) {
  if (check_shapes(cache, batch) || heads == 0 || heads % cache->kv_heads) return 0;
  return plan(cache, batch, heads, kFull, 0).work;
}

int dance_kv_sparse_attention(const DanceKvCache* cache, const DanceKvBatch* batch, const DanceKvRows* queries,
                              const int32_t* lists, uint32_t count, float scale, void* out, float* lse, void* work,
                              size_t work_bytes, void* stream) {
  return run("dance_kv_sparse_attention", cache, batch, queries, lists, kList, count, scale, out, lse, work, work_bytes,
             stream);
}

size_t dance_kv_sparse_attention_work(const DanceKvCache* cache, const DanceKvBatch* batch, uint32_t heads,
                                      uint32_t count) {
  if (check_shapes(cache, batch) || heads == 0 || heads % cache->kv_heads || !count_fits(cache, count)) return 0;
  return plan(cache, batch, heads, kList, count).work;
}

}  // extern "C"
