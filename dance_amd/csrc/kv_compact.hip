// dance_kv_compact (include/dance_kv_pages.h): chosen tokens, densely, in blocks of
// their own scales.
//
// A token's code times its block's scale is exact in float32 where the scale is a power of two, and the new
// scale is one, so a code whose block keeps its scale stays as it is and the one
// rounding is that of a block that mixes scales.
//
// One workgroup per (sequence, new block, head), at most 64 codes of keys and as many of values a lane, which stay in
// registers from their one load to their rounding. Keys and values go together, since the way to a token (list,
// table, scale) is three loads in turn. Keys come 16 bytes of a token at a time. Values lie dims-major, so a token's
// are bytes of different lines: lanes stand for neighbouring tokens, which mostly lie in the same lines, and leave as
// words of four tokens that four lanes exchange by DPP.
//
// Measured: all tokens of 31 sequences of 15,000 to 21,000 (one head of 96 dimensions), 57 us, 3.9 TB/s; 44 us where
// the cache behind the L2s holds them. Half of 16 sequences of 4,000 to 24,000 (8 heads of 128), other tokens for each
// head, 96 us: 290 MB that count, 371 that move, since a line of values comes whole; 3.9 TB/s, and the units that form
// the byte loads' addresses are busy for two thirds of the time. Every fiftieth token of 262,144: 51 us, 202 MB of lines
// (4.0 TB/s). Lines read whole and bytes taken out of LDS: 6 % less for half of the tokens, a third more for all of the
// 31 sequences.
//
// Between powers of two the arithmetic is f16's, two codes an instruction: a code is exact there, and c * ratio +
// 1536 has the unit 1, so that one fma rounds it as the definition does and leaves the code in the low byte.

#include "../../include/dance_kv_pages.h"
#include "kv_common.h"

namespace dance {
namespace kv {
namespace {

struct Compact {
  Cache from, to;
  const int32_t* __restrict__ table;
  const int32_t* __restrict__ lengths;
  const int32_t* __restrict__ keep;
  const int32_t* __restrict__ counts;
  const int32_t* __restrict__ into;
  uint32_t width, keep_heads, keep_width, into_width, places;
};

typedef uint16_t u16_2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ h2_t max2(h2_t a, h2_t b) { return __builtin_elementwise_max(a, b); }
__device__ __forceinline__ h2_t min2(h2_t a, h2_t b) { return __builtin_elementwise_min(a, b); }
__device__ __forceinline__ h2_t pair(uint32_t x) { return __builtin_bit_cast(h2_t, x); }
__device__ __forceinline__ uint32_t bits(h2_t x) { return __builtin_bit_cast(uint32_t, x); }
// Four codes as f16 from bytes in halves, as codes4.
__device__ __forceinline__ u2_t codes2x2(u16_2 a, u16_2 b) {
  const h2_t bias = {(_Float16)1152.f, (_Float16)1152.f};
  auto one = [&](u16_2 c) { return bits(pair((__builtin_bit_cast(uint32_t, c) ^ 0x00800080u) | 0x64006400u) - bias); };
  return u2_t{one(a), one(b)};
}
constexpr uint32_t kLowBytes = 0x06040200u;  // of two words' four halves

template <int CTRL>
__device__ __forceinline__ uint32_t quad(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, true);
}
// Of the words of four neighbouring lanes, the lane's byte of each.
__device__ __forceinline__ uint32_t turn4(uint32_t w, uint32_t lane) {
  const uint32_t a = quad<0x00>(w), b = quad<0x55>(w), c = quad<0xAA>(w), d = quad<0xFF>(w);
  const uint32_t at = lane & 3u, sel = 0x0400u + at * 0x0101u;  // byte `at` of the second operand, then of the first
  const uint32_t lo = __builtin_amdgcn_perm(b, a, sel), hi = __builtin_amdgcn_perm(d, c, sel);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// A power of two whose product with any code is a finite, normal number; or 0, a token that is not there.
__device__ __forceinline__ bool plain_scale(float s) {
  const uint32_t u = __float_as_uint(s);
  return u == 0u || ((u & 0x807FFFFFu) == 0u && u >= 1u << 23 && u <= 0x7B800000u);
}

constexpr uint32_t compact_waves(uint32_t d, uint32_t bs) {
  const uint32_t n = (d * bs + 4095) / 4096, w = n > 4 ? 8 : n > 2 ? 4 : n;
  return w * 64 < bs ? bs / 64 : w;
}

template <int D, int BS>
__global__ __launch_bounds__(64 * compact_waves(D, BS)) void k_compact(Compact a) {
  constexpr uint32_t W = compact_waves(D, BS), T = 64 * W;
  constexpr uint32_t C16 = D / 16, R = T / C16 < BS ? T / C16 : BS;  // keys: pieces of a token, tokens at once
  constexpr uint32_t NP = (BS + R - 1) / R;                         // pieces of a lane
  constexpr uint32_t G = T / BS, NW = D / 4 / G;                    // values: lanes of a token, fours of dimensions of a lane
  static_assert(T % BS == 0 && D / 4 % G == 0, "every lane has a token, and as many dimensions as the others");
  __shared__ uint32_t t_cell[BS], t_slot[BS];
  __shared__ float2 t_scale[BS];
  __shared__ float wave_max[W][2];
  __shared__ uint32_t wave_plain[W];
  __shared__ uint32_t part[R][D];  // each token row's largest codes of two dimensions, then the least
  const uint32_t tid = threadIdx.x;
  uint32_t id = blockIdx.x;
  const uint32_t h = id % a.from.kvh;
  id /= a.from.kvh;
  const uint32_t j = id % a.places, b = id / a.places;
  const uint32_t i0 = j * BS + tid;
  int32_t pos = -1;
  if (tid < BS && i0 < a.keep_width)
    pos = a.keep[((size_t)b * a.keep_heads + (a.keep_heads == 1 ? 0u : h)) * a.keep_width + i0];
  const uint32_t count = min((uint32_t)max(a.counts[b], 0), a.keep_width);
  if (j * BS >= count) return;
  const int32_t dst = a.into[(size_t)b * a.into_width + j];
  if ((uint32_t)dst >= a.to.blocks) return;
  const uint32_t live = min((uint32_t)BS, count - j * BS);
  bool plain = true;
  if (tid < BS) {
    uint32_t at = 0, slot = 0;
    float2 s = {0.f, 0.f};  // no such token: whatever is read for it
    if (tid < live && pos >= 0 && pos < a.lengths[b] && (uint32_t)pos / BS < a.width) {
      const int32_t p = a.table[(size_t)b * a.width + (uint32_t)pos / BS];
      if ((uint32_t)p < a.from.blocks) {
        at = (uint32_t)p * a.from.kvh + h;
        slot = (uint32_t)pos % BS;
        s = *reinterpret_cast<const float2*>(a.from.scale + (size_t)at * 2);
        plain = plain_scale(s.x) && plain_scale(s.y);
      }
    }
    t_cell[tid] = at;
    t_slot[tid] = slot;
    t_scale[tid] = s;
  }
  plain = __all(plain);
  if constexpr (W > 1) {
    if ((tid & 63u) == 0) wave_plain[tid >> 6] = plain;
  }
  __syncthreads();
  if constexpr (W > 1) {
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) plain = plain && wave_plain[w];
  }

  // all codes set out
  const uint32_t c16 = tid % C16, r = tid / C16;  // keys
  const uint32_t t = tid % BS, g = tid / BS;      // values
  u4_t kw[NP];
  float ks[NP];
#pragma unroll
  for (uint32_t i = 0; i < NP; ++i) {
    const uint32_t tk = r + i * R;
    kw[i] = u4_t{0u, 0u, 0u, 0u};
    ks[i] = 0.f;
    if (r < R && tk < live) {
      kw[i] = *reinterpret_cast<const u4_t*>(a.from.k + ((size_t)t_cell[tk] * BS + t_slot[tk]) * D + c16 * 16);
      ks[i] = t_scale[tk].x;
    }
  }
  const float vs = t_scale[t].y;
  u16_2 vw[NW][2];  // pairs of codes, as loads leave them
#pragma unroll
  for (uint32_t i = 0; i < NW; ++i) vw[i][0] = vw[i][1] = u16_2{0, 0};
  if (t < live) {
    const uint8_t* const src = reinterpret_cast<const uint8_t*>(a.from.v) + (size_t)t_cell[t] * D * BS + t_slot[t] + 4 * g * BS;
#pragma unroll
    for (uint32_t i = 0; i < NW; ++i) {
      const uint8_t* const p = src + 4 * G * BS * i;
      vw[i][0] = u16_2{p[0], p[BS]};
      vw[i][1] = u16_2{p[2 * BS], p[3 * BS]};
    }
  }

  // the blocks' new scales
  float most_k = 0.f, most_v = 0.f, top = 0.f;
  auto largest = [](h2_t& m, u2_t x) {
    m = max2(m, max2(pair(x.x), -pair(x.x)));
    m = max2(m, max2(pair(x.y), -pair(x.y)));
  };
#pragma unroll
  for (uint32_t i = 0; i < NP; ++i) {
    h2_t m = {(_Float16)0.f, (_Float16)0.f};
#pragma unroll
    for (int x = 0; x < 4; ++x) largest(m, codes4(kw[i][x]));
    const float x = fabsf(fmaxf((float)m.x, (float)m.y) * ks[i]);
    most_k = fmaxf(most_k, finite_abs(x));
    top = fmaxf(top, x);
  }
  {
    h2_t m = {(_Float16)0.f, (_Float16)0.f};
#pragma unroll
    for (uint32_t i = 0; i < NW; ++i) largest(m, codes2x2(vw[i][0], vw[i][1]));
    const float x = fabsf(fmaxf((float)m.x, (float)m.y) * vs);
    most_v = finite_abs(x);
    top = fmaxf(top, x);
  }
  // Where the largest code's product passes float32's range it does not count, but smaller ones do: then the codes are read
  // again and looked at one by one. (From the registers that hold them, this costs every call up to 64 more of those, and
  // half of a batch's tokens take 104 to 116 us, not 96.)
  if (top == __builtin_inff()) {
    auto product = [](float& m, int8_t c, float s) { m = fmaxf(m, finite_abs((float)c * s)); };
    most_k = most_v = 0.f;
    if (r < R)
#pragma unroll 1
      for (uint32_t tk = r; tk < live; tk += R) {
        const int8_t* const src = a.from.k + ((size_t)t_cell[tk] * BS + t_slot[tk]) * D + c16 * 16;
#pragma unroll 1
        for (uint32_t x = 0; x < 16; ++x) product(most_k, src[x], t_scale[tk].x);
      }
    if (t < live) {
      const int8_t* const src = a.from.v + (size_t)t_cell[t] * D * BS + t_slot[t];
#pragma unroll 1
      for (uint32_t d = 4 * g; d < (uint32_t)D; d += 4 * G)
#pragma unroll 1
        for (uint32_t x = 0; x < 4; ++x) product(most_v, src[(d + x) * BS], vs);
    }
  }
  most_k = rows_max(cols_max(most_k));
  most_v = rows_max(cols_max(most_v));
  if constexpr (W > 1) {
    if ((tid & 63u) == 0) {
      wave_max[tid >> 6][0] = most_k;
      wave_max[tid >> 6][1] = most_v;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      most_k = fmaxf(most_k, wave_max[w][0]);
      most_v = fmaxf(most_v, wave_max[w][1]);
    }
  }
  const size_t cell = (size_t)dst * a.to.kvh + h;
  const int ek = scale_exp(most_k), ev = scale_exp(most_v);
  const float inv_k = exp2_int(-ek), inv_v = exp2_int(-ev);
  if (tid == 0) *reinterpret_cast<float2*>(a.to.scale + cell * 2) = float2{exp2_int(ek), exp2_int(ev)};

  // Four codes of scale s, as halves 1536 + code. A code that is not 0 has a ratio of at most 2^6, since the new scale
  // holds it; and one below 2^-8 rounds it to 0, as f16's least numbers do.
  auto rounded = [&](u2_t c, float s, float inv) {
    const h2_t unit = {(_Float16)1536.f, (_Float16)1536.f};
    h2_t x[2] = {pair(c.x), pair(c.y)};
    if (plain) {
      const _Float16 f = (_Float16)fminf(s * inv, 128.f);
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = __builtin_elementwise_fma(x[i], h2_t{f, f}, unit);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        x[i] = h2_t{(_Float16)(float)code_of((float)x[i].x * s, inv), (_Float16)(float)code_of((float)x[i].y * s, inv)} + unit;
    }
    return u2_t{bits(x[0]), bits(x[1])};
  };
  h2_t mx[8], mn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    mx[i] = h2_t{(_Float16)1408.f, (_Float16)1408.f};  // -128
    mn[i] = h2_t{(_Float16)1663.f, (_Float16)1663.f};  // 127
  }
  int8_t* const k_out = a.to.k + cell * D * BS + c16 * 16;
#pragma unroll
  for (uint32_t i = 0; i < NP; ++i) {
    const uint32_t tk = r + i * R;
    if (r >= R || tk >= BS) continue;
    u4_t y = {0u, 0u, 0u, 0u};
    if (tk < live) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const u2_t q = rounded(codes4(kw[i][x]), ks[i], inv_k);
        mx[2 * x] = max2(mx[2 * x], pair(q.x));
        mn[2 * x] = min2(mn[2 * x], pair(q.x));
        mx[2 * x + 1] = max2(mx[2 * x + 1], pair(q.y));
        mn[2 * x + 1] = min2(mn[2 * x + 1], pair(q.y));
        y[x] = __builtin_amdgcn_perm(q.y, q.x, kLowBytes);
      }
    }
    *reinterpret_cast<u4_t*>(k_out + tk * D) = y;
  }
  if (r < R) {
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      part[r][c16 * 8 + x] = bits(mx[x]);
      part[r][D / 2 + c16 * 8 + x] = bits(mn[x]);
    }
  }
  int8_t* const v_out = a.to.v + cell * D * BS + (t & ~3u);
#pragma unroll
  for (uint32_t i = 0; i < NW; ++i) {
    const u2_t q = rounded(codes2x2(vw[i][0], vw[i][1]), vs, inv_v);
    *reinterpret_cast<uint32_t*>(v_out + (4 * (g + i * G) + (tid & 3u)) * BS) =
        turn4(__builtin_amdgcn_perm(q.y, q.x, kLowBytes), tid);
  }
  __syncthreads();
  const uint32_t rows = min(R, live);
  for (uint32_t i = tid; i < D / 2; i += T) {  // a word of the bounds is four dimensions: two words of pairs
    const uint32_t x = 2 * i;
    h2_t p = pair(part[0][x]), q = pair(part[0][x + 1]);
    for (uint32_t y = 1; y < rows; ++y) {
      const h2_t u = pair(part[y][x]), v = pair(part[y][x + 1]);
      p = i < D / 4 ? max2(p, u) : min2(p, u);
      q = i < D / 4 ? max2(q, v) : min2(q, v);
    }
    reinterpret_cast<uint32_t*>(a.to.bound + cell * 2 * D)[i] = __builtin_amdgcn_perm(bits(q), bits(p), kLowBytes);
  }
}

}  // namespace
}  // namespace kv
}  // namespace dance

extern "C" int dance_kv_compact(const DanceKvCache* from, const DanceKvCache* to, const int32_t* table, const int32_t* lengths,
                                uint32_t seqs, uint32_t width, const int32_t* keep, uint32_t keep_heads, uint32_t keep_width,
                                const int32_t* counts, const int32_t* into_table, uint32_t into_width, void* stream) {
  using namespace dance::kv;
  const DanceKvBatch source{table, lengths, nullptr, seqs, seqs, width, 1, 0};
  const DanceKvBatch target{into_table, counts, nullptr, seqs, seqs, into_width, 1, 0};
  const char* why = check_common(from, &source);
  if (!why) why = check_common(to, &target);
  if (!why && (from->kv_heads != to->kv_heads || from->dim != to->dim || from->block_tokens != to->block_tokens))
    why = "both caches must have one kv_heads, dim and block_tokens";
  if (!why && !keep) why = "null keep";
  if (!why && keep_heads != 1 && keep_heads != from->kv_heads) why = "keep_heads must be 1 or kv_heads";
  if (!why && (uint64_t)from->blocks * from->kv_heads > 0xFFFFFFFFull) why = "a cache must have fewer than 2^32 blocks of heads";
  if (!why && (keep_width == 0 || keep_width > 0x7FFFFFFFu)) why = "keep_width must be in [1, 2^31)";
  if (why) KV_ERR("dance_kv_compact", "%s", why);
  // places that the lists can fill
  const uint32_t most = (keep_width - 1) / from->block_tokens + 1, places = most < into_width ? most : into_width;
  const uint64_t grid = (uint64_t)seqs * places * from->kv_heads;
  if (grid * 64 * compact_waves(from->dim, from->block_tokens) > 0xFFFFFFFFull)
    KV_ERR("dance_kv_compact", "batch is too large for one launch");
  const Compact a{cache_args(from), cache_args(to), table, lengths, keep, counts, into_table,
                  width, keep_heads, keep_width, into_width, places};
  with_kind(from->dim, DANCE_KV_F16, [&](auto d, auto) {
    constexpr uint32_t D = decltype(d)::value;
    auto go = [&](auto n) {
      constexpr uint32_t BS = decltype(n)::value;
      hipLaunchKernelGGL((k_compact<D, BS>), dim3((uint32_t)grid), dim3(64 * compact_waves(D, BS)), 0,
                         static_cast<hipStream_t>(stream), a);
    };
    switch (from->block_tokens) {
      case 16: go(Int<16>{}); break;
      case 32: go(Int<32>{}); break;
      case 64: go(Int<64>{}); break;
      default: go(Int<128>{}); break;
    }
  });
  return launched("dance_kv_compact");
}
