// What the key-value cache kernels share: the arguments every kernel takes, the
// place of a token row in its sequence, codes, and the host's checks.
// Interface and layouts: include/dance_kv.h.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "../../include/dance_kv.h"

namespace dance {
namespace kv {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef int i4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

constexpr int kLeastExp = -100;  // exponent of the least scale: smaller blocks become zeros

struct Cache {
  int8_t* __restrict__ k;
  int8_t* __restrict__ v;
  float* __restrict__ scale;
  int8_t* __restrict__ bound;
  uint32_t blocks, kvh, bsh;  // bsh: log2 of the tokens in a block
};

struct Batch {
  const int32_t* __restrict__ table;
  const int32_t* __restrict__ lengths;
  const int32_t* __restrict__ offsets;
  uint32_t seqs, tokens, width;
};

struct Rows {
  const uint16_t* __restrict__ data;
  int64_t token_stride, head_stride;
  uint32_t heads;
};

// A sequence's rows in this call and the position of the first of them.
// Offsets that do not ascend within [0, tokens] give no rows, not a wrong access.
struct Seq {
  uint32_t row, n;
  int64_t first;  // position of row 0; negative where the sequence is shorter than its rows
  int64_t len;    // tokens that the table has room for
};
__device__ __forceinline__ Seq seq_of(const Batch& b, uint32_t s, uint32_t bsh) {
  Seq r;
  const int32_t len = b.lengths[s];
  if (b.offsets) {
    const int32_t lo = b.offsets[s], hi = b.offsets[s + 1];
    const bool ok = lo >= 0 && hi > lo && (uint32_t)hi <= b.tokens;
    r.row = ok ? (uint32_t)lo : 0u;
    r.n = ok ? (uint32_t)(hi - lo) : 0u;
  } else {
    r.row = s;
    r.n = 1;
  }
  r.first = (int64_t)len - r.n;
  const int64_t room = (int64_t)b.width << bsh;
  r.len = len < 0 ? 0 : len < room ? len : room;
  return r;
}

// The sequence of a token row: the last one that starts at or before it and is not empty.
__device__ __forceinline__ uint32_t seq_at(const Batch& b, uint32_t row) {
  if (!b.offsets) return row;
  uint32_t lo = 0, hi = b.seqs;  // offsets[lo] <= row < offsets[hi], as far as the offsets ascend
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (b.offsets[mid] <= (int32_t)row)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// a - b, or 0 where b is more; both below 2^31. In signed numbers: the compiler
// (ROCm 7.2) turns an unsigned difference that stops at 0 of two scalars into s_sub
// without the stop.
__device__ __forceinline__ uint32_t less(uint32_t a, uint32_t b) {
  const int32_t d = (int32_t)a - (int32_t)b;
  return d > 0 ? (uint32_t)d : 0u;
}

// Tiles of `per` of a sequence's rows x `group`, of all sequences in one index: a
// sequence of n has the indexes from slot(b) = offset * group / per + b up to slot(b +
// 1), at least as many as its tiles. So a grid goes by the rows that there are and not by the
// longest sequence's; where that is no fewer, each sequence has `tiles` (not 0). sq = seqs: no such tile.
struct TileAt {
  uint32_t sq, tile;
};
__device__ __forceinline__ TileAt tile_at(const Batch& b, uint32_t id, uint32_t group, uint32_t per, uint32_t tiles) {
  if (tiles) return TileAt{id / tiles, id % tiles};
  auto slot = [&](uint32_t i) { return (uint32_t)max(b.offsets[i], 0) * group / per + i; };
  uint32_t before = 0;  // sequences whose indexes begin at or before this one
  for (uint32_t i0 = 0; i0 < b.seqs; i0 += 64) {
    const uint32_t i = i0 + (threadIdx.x & 63u);
    const uint64_t mask = __ballot(i < b.seqs && slot(min(i, b.seqs - 1u)) <= id);
    before += (uint32_t)__popcll(mask);
    if (mask != ~0ull) break;
  }
  const uint32_t sq = (uint32_t)__builtin_amdgcn_readfirstlane((int)(before - 1u));
  if (sq >= b.seqs) return TileAt{b.seqs, 0};
  return TileAt{sq, id - slot(sq)};
}
// The indexes of a grid, and 0 for `tiles` where they go by the rows.
inline uint64_t tile_slots(const DanceKvBatch* b, uint64_t group, uint64_t per, uint32_t& tiles) {
  const uint64_t by_rows = b->tokens * group / per + b->seqs, by_longest = (uint64_t)b->seqs * tiles;
  if (!b->offsets || by_longest <= by_rows) return by_longest;
  tiles = 0;
  return by_rows;
}

template <bool BF>
__device__ __forceinline__ float load_val(uint16_t u) {
  if constexpr (BF)
    return __uint_as_float((uint32_t)u << 16);
  else
    return (float)__builtin_bit_cast(_Float16, u);
}

// To the output's type, halves to even: the one rounding of a result.
template <bool BF>
__device__ __forceinline__ uint16_t store_val(float x) {
  if constexpr (BF)
    return __builtin_bit_cast(uint16_t, (__bf16)x);
  else
    return __builtin_bit_cast(uint16_t, (_Float16)x);
}

// Least e >= kLeastExp with a <= 127 * 2^e, for finite a >= 0: 127 * 2^e has
// the significand 1.984375, bits 0x7E0000.
__device__ __forceinline__ int scale_exp(float a) {
  const uint32_t u = __float_as_uint(a);
  const int e = (int)(u >> 23) - 127 - 6 + ((u & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
  return e < kLeastExp ? kLeastExp : e;
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The magnitude that counts for a scale: 0 for infinities and NaN.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.f;
}
// Code of x at scale 1 / inv: exact quotient, halves to even.
__device__ __forceinline__ int code_of(float x, float inv) {
  const float r = __builtin_rintf(x * inv);
  return x == x ? (int)fminf(127.f, fmaxf(-127.f, r)) : 0;
}

// Four codes as f16, exactly: 0x6400 | (c + 128) is 1024 + 128 + c.
__device__ __forceinline__ u2_t codes4(uint32_t c) {
  const h2_t bias = {(_Float16)1152.f, (_Float16)1152.f};
  c ^= 0x80808080u;
  const h2_t lo = __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, c, 0x04010400u)) - bias;
  const h2_t hi = __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, c, 0x04030402u)) - bias;
  return u2_t{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}
__device__ __forceinline__ h8_t codes8(uint32_t a, uint32_t b) {
  const u2_t x = codes4(a), y = codes4(b);
  return __builtin_bit_cast(h8_t, u4_t{x.x, x.y, y.x, y.y});
}

// Over the four lanes that differ in bits 4 and 5 of the lane.
__device__ __forceinline__ float rows_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// Over the 16 lanes that differ in bits 0 to 3.
__device__ __forceinline__ float cols_max(float x) {
  auto with = [&](auto ctrl) {  // quad lanes 1 0 3 2, then 2 3 0 1, half rows mirrored, rows mirrored
    x = fmaxf(x, __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), decltype(ctrl)::value, 0xF, 0xF, true)));
  };
  with(std::integral_constant<int, 0xB1>{});
  with(std::integral_constant<int, 0x4E>{});
  with(std::integral_constant<int, 0x141>{});
  with(std::integral_constant<int, 0x140>{});
  return x;
}
// Over the two lanes that differ in bit 4.
__device__ __forceinline__ float pair_max(float x) {
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
#define KV_ERR(who, ...)                          \
  do {                                            \
    std::fprintf(stderr, "[" who "] " __VA_ARGS__); \
    std::fprintf(stderr, "\n");                   \
    return -1;                                    \
  } while (0)

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

inline uint32_t log2_of(uint32_t x) { return 31u - (uint32_t)__builtin_clz(x); }

// Shapes alone: what the workspace sizes and the launches go by.
inline const char* check_shapes(const DanceKvCache* c, const DanceKvBatch* b) {
  if (!c || !b) return "null cache or batch";
  if (c->dim != 64 && c->dim != 96 && c->dim != 128 && c->dim != 192 && c->dim != 256)
    return "dim must be 64, 96, 128, 192 or 256";
  if (c->block_tokens != 16 && c->block_tokens != 32 && c->block_tokens != 64 && c->block_tokens != 128)
    return "block_tokens must be 16, 32, 64 or 128";
  if (c->kv_heads == 0 || c->kv_heads > 65535u || c->blocks == 0 || c->blocks > 0x7FFFFFFFu)
    return "kv_heads must be in [1, 65535], blocks in [1, 2^31)";
  if (b->seqs == 0 || b->table_width == 0 || b->tokens > 0x7FFFFFFFu || b->seqs > 0x7FFFFFFFu)
    return "seqs and table_width must be positive, tokens below 2^31";
  if ((uint64_t)b->table_width * c->block_tokens > 0x7FFFFF00ull)  // positions and a tile beyond them are int32
    return "a table row must hold at most 2^31 - 256 tokens";
  if (b->tokens && (b->max_tokens == 0 || b->max_tokens > b->tokens)) return "max_tokens must be in [1, tokens]";
  return nullptr;
}
inline const char* check_common(const DanceKvCache* c, const DanceKvBatch* b) {
  if (const char* why = check_shapes(c, b)) return why;
  if (!c->k || !c->v || !c->scale || !c->bound || !b->table || !b->lengths) return "null cache or batch pointer";
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->scale, 16) || !aligned(c->bound, 16))
    return "the cache's arrays must be aligned to 16 bytes";
  if (!b->offsets && b->tokens != b->seqs) return "without offsets there is one token row per sequence";
  return nullptr;
}
inline const char* check_rows(const DanceKvCache* c, const DanceKvRows* r, bool kv) {
  if (!r || !r->data) return "null rows";
  if (r->dtype != DANCE_KV_F16 && r->dtype != DANCE_KV_BF16) return "rows must be float16 or bfloat16";
  if (kv ? r->heads != c->kv_heads : (r->heads == 0 || r->heads % c->kv_heads != 0 || r->heads > 65535u))
    return kv ? "new rows must have kv_heads heads" : "heads must be a multiple of kv_heads, at most 65535";
  if (!aligned(r->data, 2)) return "rows must be aligned to their elements";
  return nullptr;
}

inline Cache cache_args(const DanceKvCache* c) {
  return Cache{c->k, c->v, c->scale, c->bound, c->blocks, c->kv_heads, log2_of(c->block_tokens)};
}
inline Batch batch_args(const DanceKvBatch* b) {
  return Batch{b->table, b->lengths, b->offsets, b->seqs, b->tokens, b->table_width};
}
inline Rows rows_args(const DanceKvRows* r) {
  return Rows{static_cast<const uint16_t*>(r->data), r->token_stride, r->head_stride, r->heads};
}
// Rows that 16-byte loads can read.
inline bool rows_vector(const DanceKvRows* r) {
  return aligned(r->data, 16) && r->token_stride % 8 == 0 && r->head_stride % 8 == 0;
}
// Blocks of a sequence that a call may meet.
inline uint32_t most_blocks(const DanceKvCache* c, const DanceKvBatch* b) {
  const uint64_t n = b->max_length ? (b->max_length - 1) / c->block_tokens + 1 : b->table_width;
  return n < b->table_width ? (uint32_t)n : b->table_width;
}

template <int V>
using Int = std::integral_constant<int, V>;

// fn(dim, bf16) with both as compile-time constants.
template <typename Fn>
inline void with_kind(uint32_t dim, int dtype, Fn&& fn) {
  auto go = [&](auto d) {
    if (dtype == DANCE_KV_BF16)
      fn(d, std::true_type{});
    else
      fn(d, std::false_type{});
  };
  switch (dim) {
    case 64: go(Int<64>{}); break;
    case 96: go(Int<96>{}); break;
    case 128: go(Int<128>{}); break;
    case 192: go(Int<192>{}); break;
    default: go(Int<256>{}); break;
  }
}

inline int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return 0;
  std::fprintf(stderr, "[%s] launch failed: %s\n", who, hipGetErrorString(e));
  return -1;
}

}  // namespace kv
}  // namespace dance
