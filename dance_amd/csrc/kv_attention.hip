// dance_kv_attention and dance_kv_sparse_attention (include/dance_kv.h).
//
// For a tile of 64 tokens and 16 query rows a wave forms S' = K Q' (tokens x
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
//  - lane group g holds dimensions g D / 4 .. of keys and queries, adjacent bytes too.
// Codes go from memory to the registers that the MFMAs read; every code is
// read once per 16 rows.
//
// Softmax: running reference M and sum l per row, in log2 units. A row keeps its M until
// a logit exceeds it by 2^kSlack; weights are then at most 2^(kLift + kSlack), inside f16,
// and the least normal weight is 2^-20 of a row's largest. The products take
// weight * (value scale / largest value scale so far), which f16 rounds to 11
// bits; the sum l takes the unrounded weights.

#include <cfloat>
#include <cmath>
#include <type_traits>

#include "kv_common.h"

namespace dance {
namespace kv {
namespace {

constexpr uint32_t kStepWaves = 4;
constexpr uint32_t kRowTile = 16;
constexpr uint32_t kTokTile = 64;
constexpr float kLift = 6.f, kSlack = 8.f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t kSplitUnits = 1024;  // workgroups that fill the chip several times over

struct StepArgs {
  Cache c;
  Batch b;
  Rows q;
  const int32_t* __restrict__ lists;  // LIST: tokens x kv_heads x count
  uint32_t count;
  float scale2;  // scale * log2(e)
  uint32_t group, tiles, splits;
  uint16_t* __restrict__ out;
  float* __restrict__ lse;
  float* __restrict__ part;  // splits > 1: [row][split][D] sums, then [row][split][2] (M, l)
};

// The work of one workgroup: 16 rows of one kv head, a split of the tokens they see.
struct Unit {
  uint32_t sq, h, tile, split;
};

template <int D, bool BF, bool LIST, bool VEC>
__global__ __launch_bounds__(64 * kStepWaves) void k_step(StepArgs a) {
  constexpr int KS = D / 32;  // inner steps of the first product
  constexpr int DT = D / 16;  // row tiles of the second
  constexpr int KW = D / 16;  // words of a key row that a lane holds
  __shared__ float sm_o[kStepWaves][kRowTile][D];
  __shared__ float sm_m[kStepWaves][kRowTile], sm_l[kStepWaves][kRowTile];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t n = lane & 15u, g = lane >> 4;
  const uint32_t bsh = a.c.bsh, bs = 1u << bsh;
  uint32_t id = blockIdx.x;
  const uint32_t split = id % a.splits;
  id /= a.splits;
  const uint32_t h = id % a.c.kvh;
  id /= a.c.kvh;
  const uint32_t tile = id % a.tiles;
  id /= a.tiles;
  // id: the token row (LIST) or the sequence
  const uint32_t sq = LIST ? seq_at(a.b, id) : id;
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
  const int64_t p_row = min(s.first + tok, s.len - 1), p_top = min(s.first + (r_first + rows - 1) / a.group, s.len - 1);
  const int32_t pos = n < rows && p_row >= 0 ? (int32_t)p_row : -1, top = p_top >= 0 ? (int32_t)p_top : -1;
  const int32_t seen = (int32_t)((uint32_t)(top + 1 + (int32_t)bs - 1) >> bsh);  // blocks
  const uint32_t entries = LIST ? a.count : (uint32_t)seen;
  const int32_t* const list = LIST ? a.lists + ((size_t)id * a.c.kvh + h) * a.count : nullptr;
  const int32_t* const table = a.b.table + (size_t)sq * a.b.width;

  // Queries, as f16 with a power of two taken out so that bf16's range fits.
  h8_t qf[KS];
  float qscale = a.scale2;
  {
    const uint16_t* src = a.q.data + (int64_t)(s.row + tok) * a.q.token_stride + (int64_t)head * a.q.head_stride + g * (D / 4);
    u4_t raw[KS];
#pragma unroll
    for (int c = 0; c < KS; ++c) {
      if constexpr (VEC) {
        raw[c] = *reinterpret_cast<const u4_t*>(src + 8 * c);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[c][i] = (uint32_t)src[8 * c + 2 * i] | (uint32_t)src[8 * c + 2 * i + 1] << 16;
      }
    }
    if constexpr (BF) {
      float mag = 0.f;
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) mag = fmaxf(mag, finite_abs(load_val<true>((uint16_t)(raw[c][i >> 1] >> (16 * (i & 1))))));
      mag = rows_max(mag);
      int e = (int)(__float_as_uint(mag) >> 23) - 127 - 10;  // the largest becomes 2^10 .. 2^11
      e = e < -100 ? -100 : e;
      const float inv = exp2_int(-e);
      qscale *= exp2_int(e);
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          qf[c][i] = (_Float16)(load_val<true>((uint16_t)(raw[c][i >> 1] >> (16 * (i & 1)))) * inv);
    } else {
#pragma unroll
      for (int c = 0; c < KS; ++c) qf[c] = __builtin_bit_cast(h8_t, raw[c]);
    }
  }

  f4_t acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f4_t{0.f, 0.f, 0.f, 0.f};
  float M = -FLT_MAX, l = 0.f, vref = 0.f, vinv = 0.f;

  // this split's tiles of 64 listed tokens
  const uint32_t all = (uint32_t)(((uint64_t)entries * bs + kTokTile - 1) / kTokTile);
  const uint32_t per = (all + a.splits - 1) / a.splits;
  const uint32_t t_end = min(all, (split + 1) * per);
  // the block with the 16 tokens of group `grp` of a tile, and its first position; a hole: -1
  auto locate = [&](uint32_t tt, uint32_t grp, int32_t& first) -> int32_t {
    const uint32_t vt = tt * kTokTile + grp * 16u;
    const uint32_t e = vt >> bsh;
    int32_t lg = -1;
    if (e < entries) lg = LIST ? list[e] : (int32_t)e;
    int32_t ph = -1;
    if (lg >= 0 && lg < seen) ph = table[lg];
    if ((uint32_t)ph >= a.c.blocks) ph = -1;
    first = (int32_t)(((uint32_t)lg << bsh) + (vt & (bs - 1u)));
    return ph;
  };
  for (uint32_t tt = split * per + wave; tt < t_end; tt += kStepWaves) {
    int32_t first, other;
    const int32_t pv = locate(tt, g, first), pk = locate(tt, n >> 2, other);
    const uint32_t slot_v = (tt * kTokTile + g * 16u) & (bs - 1u), slot_k = (tt * kTokTile + (n >> 2) * 16u) & (bs - 1u);
    const size_t cell_v = (size_t)max(pv, 0) * a.c.kvh + h, cell_k = (size_t)max(pk, 0) * a.c.kvh + h;
    uint32_t kw[4][KW];
    u4_t vw[DT];
    const int8_t* kp = a.c.k + ((cell_k << bsh) + slot_k + (n & 3u)) * D + g * (D / 4);
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      if constexpr (KW % 4 == 0) {
#pragma unroll
        for (int i = 0; i < KW / 4; ++i) {
          const u4_t w = *reinterpret_cast<const u4_t*>(kp + (size_t)st * 4 * D + i * 16);
          kw[st][4 * i] = w.x, kw[st][4 * i + 1] = w.y, kw[st][4 * i + 2] = w.z, kw[st][4 * i + 3] = w.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < KW / 2; ++i) {
          const u2_t w = *reinterpret_cast<const u2_t*>(kp + (size_t)st * 4 * D + i * 8);
          kw[st][2 * i] = w.x, kw[st][2 * i + 1] = w.y;
        }
      }
    }
    const int8_t* vp = a.c.v + ((cell_v * D + n) << bsh) + slot_v;
#pragma unroll
    for (int t = 0; t < DT; ++t) vw[t] = *reinterpret_cast<const u4_t*>(vp + ((size_t)(16 * t) << bsh));
    const float ks = pv >= 0 ? a.c.scale[cell_v * 2] * qscale : 0.f;
    const float vs = pv >= 0 ? a.c.scale[cell_v * 2 + 1] : 0.f;

    f4_t sc[4];
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      sc[st] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KS; ++c)
        sc[st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(kw[st][2 * c], kw[st][2 * c + 1]), qf[c], sc[st], 0, 0, 0);
    }
    // tokens of this lane that its row sees: the first `lim` + 1 of its 16
    const int32_t lim = pv >= 0 && first <= pos ? pos - first : -1;
    float big = -FLT_MAX;
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = sc[st][i] * ks;
        sc[st][i] = 4 * st + i <= lim ? x : -__builtin_inff();
        big = fmaxf(big, sc[st][i]);
      }
    if (__any(big > M + (kLift + kSlack) || vs > vref)) {
      // each row by its own logits alone: a row's result does not depend on its neighbours
      const float row_big = rows_max(big);
      const float m_new = row_big > M + (kLift + kSlack) ? row_big - kLift : M;
      const float v_new = fmaxf(vref, rows_max(vs));
      const float f = exp2f(M - m_new);
      const float fo = v_new > 0.f ? f * (vref / v_new) : 0.f;
      l *= f;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] *= fo;
      M = m_new;
      vref = v_new;
      vinv = v_new > 0.f ? 1.f / v_new : 0.f;
    }
    const float w = vs * vinv;
    h8_t pf[2];
    float add = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = __builtin_amdgcn_exp2f(sc[2 * u + (i >> 2)][i & 3] - M);
        add += p;
        pf[u][i] = (_Float16)(p * w);
      }
    l += add;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vw[t].x, vw[t].y), pf[0], acc[t], 0, 0, 0);
      acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(vw[t].z, vw[t].w), pf[1], acc[t], 0, 0, 0);
    }
  }

  // The waves' sums meet in LDS, in wave order.
  l = rows_sum(l);
  if (g == 0) {
    sm_m[wave][n] = M;
    sm_l[wave][n] = l;
  }
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) sm_o[wave][n][16 * t + 4 * g + i] = acc[t][i] * vref;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < rows * (D / 4); i += 64 * kStepWaves) {
    const uint32_t rr = i / (D / 4), d = i % (D / 4) * 4;
    float m = sm_m[0][rr];
#pragma unroll
    for (uint32_t w = 1; w < kStepWaves; ++w) m = fmaxf(m, sm_m[w][rr]);
    float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t w = 0; w < kStepWaves; ++w) {
      const float f = exp2f(sm_m[w][rr] - m);
      sum += f * sm_l[w][rr];
#pragma unroll
      for (int x = 0; x < 4; ++x) o[x] += f * sm_o[w][rr][d + x];
    }
    const uint32_t rw = r_first + rr;
    const size_t row = (size_t)(s.row + rw / a.group) * a.q.heads + h * a.group + rw % a.group;
    if (a.splits > 1) {
      float* const po = a.part + (row * a.splits + split) * D + d;
#pragma unroll
      for (int x = 0; x < 4; ++x) po[x] = o[x];
      if (d == 0) {
        float* const pm = a.part + (size_t)a.b.tokens * a.q.heads * a.splits * D + (row * a.splits + split) * 2;
        pm[0] = m;
        pm[1] = sum;
      }
    } else {
      const float inv = sum > 0.f ? 1.f / sum : 0.f;
      uint16_t y[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) y[x] = store_val<BF>(sum == 0.f ? 0.f : o[x] * inv);
      *reinterpret_cast<u2_t*>(a.out + row * D + d) = u2_t{y[0] | (uint32_t)y[1] << 16, y[2] | (uint32_t)y[3] << 16};
      if (a.lse && d == 0) a.lse[row] = sum == 0.f ? -__builtin_inff() : (m + log2f(sum)) * kLn2;
    }
  }
}

// Joins the splits of a row; one wave per row.
template <int D, bool BF>
__global__ __launch_bounds__(64) void k_join(const float* __restrict__ part, uint32_t splits, uint64_t rows,
                                             uint16_t* __restrict__ out, float* __restrict__ lse) {
  const uint64_t row = blockIdx.x;
  const float* const ml = part + rows * splits * D + row * splits * 2;
  float m = -FLT_MAX;
  for (uint32_t i = 0; i < splits; ++i) m = fmaxf(m, ml[2 * i]);
  float sum = 0.f, o[D / 64 + 1];
#pragma unroll
  for (int x = 0; x <= D / 64; ++x) o[x] = 0.f;
  for (uint32_t i = 0; i < splits; ++i) {
    const float f = exp2f(ml[2 * i] - m);
    sum += f * ml[2 * i + 1];
    const float* const po = part + (row * splits + i) * D;
#pragma unroll
    for (uint32_t x = 0; x < D; x += 64)
      if (x + threadIdx.x < D) o[x / 64] += f * po[x + threadIdx.x];
  }
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
  for (uint32_t x = 0; x < D; x += 64)
    if (x + threadIdx.x < D) out[row * D + x + threadIdx.x] = store_val<BF>(sum == 0.f ? 0.f : o[x / 64] * inv);
  if (lse && threadIdx.x == 0) lse[row] = sum == 0.f ? -__builtin_inff() : (m + log2f(sum)) * kLn2;
}

// How many workgroups share a row tile's tokens.
uint32_t split_rule(uint64_t units, uint64_t tokens) {
  const uint64_t most = (tokens + kStepWaves * kTokTile - 1) / (kStepWaves * kTokTile);  // a tile for every wave
  const uint64_t want = (kSplitUnits + units - 1) / (units ? units : 1);
  const uint64_t n = want < most ? want : most;
  return n < 1 ? 1u : n > 256 ? 256u : (uint32_t)n;
}

struct Plan {
  uint64_t units;  // sequences or token rows, x row tiles x kv heads
  uint32_t tiles, splits;
  size_t work;
};
Plan plan(const DanceKvCache* c, const DanceKvBatch* b, uint32_t heads, bool list, uint32_t count) {
  Plan p{};
  if (b->tokens == 0) return p;
  const uint64_t group = heads / c->kv_heads;
  const uint64_t rows = list ? group : group * b->max_tokens;
  p.tiles = (uint32_t)((rows + kRowTile - 1) / kRowTile);
  p.units = (uint64_t)(list ? b->tokens : b->seqs) * p.tiles * c->kv_heads;
  p.splits = split_rule(p.units, (uint64_t)(list ? count : most_blocks(c, b)) * c->block_tokens);
  if (p.splits > 1) p.work = (size_t)b->tokens * heads * p.splits * (c->dim + 2) * 4;
  return p;
}

int run(const char* who, const DanceKvCache* cache, const DanceKvBatch* batch, const DanceKvRows* q,
        const int32_t* lists, bool list, uint32_t count, float scale, void* out, float* lse, void* work,
        size_t work_bytes, void* stream) {
  const char* why = check_common(cache, batch);
  if (!why) why = check_rows(cache, q, false);
  if (!why && (!out || !aligned(out, 16))) why = "out must be given, aligned to 16 bytes";
  if (!why && list && (!lists || count == 0 || (uint64_t)count * cache->block_tokens > 0x7FFFFFFFull))
    why = "lists must be given, with 1 to 2^31 / block_tokens entries";
  if (!why && !(scale == scale && std::fabs(scale) < INFINITY)) why = "scale must be finite";
  if (why) {
    std::fprintf(stderr, "[%s] %s\n", who, why);
    return -1;
  }
  if (batch->tokens == 0) return 0;
  const Plan p = plan(cache, batch, q->heads, list, count);
  if (p.work && (!work || work_bytes < p.work || !aligned(work, 16))) {
    std::fprintf(stderr, "[%s] work must hold %zu bytes, aligned to 16\n", who, p.work);
    return -1;
  }
  const uint64_t grid = p.units * p.splits;
  if (grid * 64 * kStepWaves > 0xFFFFFFFFull || (uint64_t)batch->tokens * q->heads * 64 > 0xFFFFFFFFull) {
    std::fprintf(stderr, "[%s] batch is too large for one launch\n", who);
    return -1;
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  StepArgs a{cache_args(cache), batch_args(batch), rows_args(q), lists, count, scale * kLog2e,
             q->heads / cache->kv_heads, p.tiles, p.splits, static_cast<uint16_t*>(out), lse,
             static_cast<float*>(work)};
  const bool vec = rows_vector(q);
  with_kind(cache->dim, q->dtype, [&](auto d, auto bf) {
    constexpr int D = decltype(d)::value;
    constexpr bool BF = decltype(bf)::value;
    auto go = [&](auto l, auto v) {
      hipLaunchKernelGGL((k_step<D, BF, decltype(l)::value, decltype(v)::value>), dim3((uint32_t)grid),
                         dim3(64 * kStepWaves), 0, st, a);
    };
    if (list)
      vec ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
    else
      vec ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
    if (p.splits > 1)
      hipLaunchKernelGGL((k_join<D, BF>), dim3(batch->tokens * q->heads), dim3(64), 0, st, a.part, p.splits,
                         (uint64_t)batch->tokens * q->heads, a.out, lse);
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
  return run("dance_kv_attention", cache, batch, queries, nullptr, false, 0, scale, out, lse, work, work_bytes, stream);
}

size_t dance_kv_attention_work(const DanceKvCache* cache, const DanceKvBatch* batch, uint32_t heads) {
  if (check_shapes(cache, batch) || heads == 0 || heads % cache->kv_heads) return 0;
  return plan(cache, batch, heads, false, 0).work;
}

int dance_kv_sparse_attention(const DanceKvCache* cache, const DanceKvBatch* batch, const DanceKvRows* queries,
                              const int32_t* lists, uint32_t count, float scale, void* out, float* lse, void* work,
                              size_t work_bytes, void* stream) {
  return run("dance_kv_sparse_attention", cache, batch, queries, lists, true, count, scale, out, lse, work, work_bytes,
             stream);
}

size_t dance_kv_sparse_attention_work(const DanceKvCache* cache, const DanceKvBatch* batch, uint32_t heads,
                                      uint32_t count) {
  if (check_shapes(cache, batch) || heads == 0 || heads % cache->kv_heads) return 0;
  return plan(cache, batch, heads, true, count).work;
}

}  // extern "C"
