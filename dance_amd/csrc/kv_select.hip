// dance_kv_select (include/dance_kv.h): the blocks whose keys may have the
// largest products with a query, by a bound.
//
// With hi and lo the largest and least key code of a block's tokens in a
// dimension, c k <= max(c hi, c lo) for the code c of the query and each of the
// block's codes k: c hi where c > 0, c lo where c < 0. The bound of all
// dimensions is thus one product of length 2 D, (c+ | c-) with (hi | lo), the
// latter as they lie in memory. It is done with 16x16x64 i8 MFMAs, 16 blocks by
// 16 query rows, exactly; only the block's scale is rounded in (once).
//
// Choice: the count-th largest key by its 8-bit digits from the top (counts
// in LDS), then one pass in index order that keeps what is larger, and of what
// equals it the first ones.

#include <cmath>
#include <type_traits>

#include "kv_common.h"

namespace dance {
namespace kv {
namespace {

constexpr uint32_t kScoreWaves = 4;
constexpr uint32_t kTopThreads = 256;

struct SelectArgs {
  Cache c;
  Batch b;
  Rows q;
  uint32_t group, count, sink, recent;
  uint32_t stride;  // scores of a (token row, kv head)
  float* __restrict__ score;
  int32_t* __restrict__ chosen;
};

// Position of a token row and the blocks it sees; none for a row of no sequence.
struct Place {
  uint32_t sq, seen;
};
__device__ __forceinline__ Place place_of(const SelectArgs& a, uint32_t row) {
  Place p;
  p.sq = seq_at(a.b, row);
  const Seq s = seq_of(a.b, p.sq, a.c.bsh);
  p.seen = 0;
  if (row >= s.row && row - s.row < s.n) {
    const int64_t at = s.first + (row - s.row);
    const int64_t end = at + 1 < s.len ? at + 1 : s.len;
    if (end > 0) p.seen = min((uint32_t)((end + (1ll << a.c.bsh) - 1) >> a.c.bsh), a.stride);
  }
  return p;
}

template <int D, bool BF>
__global__ __launch_bounds__(64 * kScoreWaves) void k_score(SelectArgs a, uint32_t chunks, uint32_t per) {
  constexpr int KS = D / 32;  // inner steps of 64 over 2 D
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t n = lane & 15u, g = lane >> 4;
  uint32_t id = blockIdx.x;
  const uint32_t chunk = id % chunks;
  id /= chunks;
  const uint32_t h = id % a.c.kvh, row = id / a.c.kvh;
  const Place p = place_of(a, row);
  const uint32_t first = chunk * per, end = min(first + per, p.seen);
  if (first >= end) return;
  const int32_t* const table = a.b.table + (size_t)p.sq * a.b.width;
  float* const out = a.score + ((size_t)row * a.c.kvh + h) * a.stride;
  const uint32_t forced = p.seen > a.recent ? p.seen - a.recent : 0u;

  for (uint32_t r0 = 0; r0 < a.group; r0 += 16) {
    // This lane's part of its row's codes: positive part in lane groups 0 and 1
    // (against hi), negative part in 2 and 3 (against lo).
    const uint32_t r = r0 + n;
    const bool live = r < a.group;
    const uint16_t* const src = a.q.data + (int64_t)row * a.q.token_stride +
                                (int64_t)(h * a.group + (live ? r : 0u)) * a.q.head_stride + (g & 1u) * (D / 2);
    float mag = 0.f;
    for (int i = 0; i < D / 2; ++i) mag = fmaxf(mag, finite_abs(load_val<BF>(src[i])));
    mag = rows_max(mag);
    const int e = scale_exp(mag);
    const float inv = exp2_int(-e), up = exp2_int(e);
    i4_t qf[KS];
#pragma unroll
    for (int c = 0; c < KS; ++c)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t x = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int code = code_of(load_val<BF>(src[16 * c + 4 * w + b]), inv);
          const int part = g < 2 ? max(code, 0) : min(code, 0);
          x |= (uint32_t)(part & 255) << (8 * b);
        }
        qf[c][w] = (int)x;
      }
    for (uint32_t b0 = first + wave * 16; b0 < end; b0 += kScoreWaves * 16) {
      const uint32_t mine = b0 + n;  // the block that this lane loads for
      int32_t ph = mine < end ? table[mine] : -1;
      if ((uint32_t)ph >= a.c.blocks) ph = -1;
      const size_t cell = (size_t)max(ph, 0) * a.c.kvh + h;
      const int8_t* const bp = a.c.bound + cell * 2 * D + g * (D / 2);
      const float ks = ph >= 0 ? a.c.scale[cell * 2] : 0.f;
      i4_t acc = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < KS; ++c)
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i4_t*>(bp + 16 * c), qf[c], acc, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t m = 4 * g + i;  // block b0 + m, held by lane m
        const float sc = __shfl(ks, (int)m);
        const bool hole = __shfl(ph, (int)m) < 0;
        float x = live ? ((float)acc[i] * sc) * up + 0.f : -__builtin_inff();
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
        const uint32_t blk = b0 + m;
        if (n == 0 && blk < end) {
          if (r0) x = fmaxf(x, out[blk]);
          if (blk < a.sink || blk >= forced) x = __builtin_inff();
          out[blk] = hole ? -__builtin_inff() : x;
        }
      }
    }
  }
}

__device__ __forceinline__ uint32_t sort_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kNoKey = 0x007FFFFFu;  // sort_key(-inf): holes

__global__ __launch_bounds__(kTopThreads) void k_top(SelectArgs a) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t pick[2];
  __shared__ uint32_t wave_more[kTopThreads / 64], wave_same[kTopThreads / 64];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t h = blockIdx.x % a.c.kvh, row = blockIdx.x / a.c.kvh;
  const Place p = place_of(a, row);
  const float* const score = a.score + ((size_t)row * a.c.kvh + h) * a.stride;
  int32_t* const out = a.chosen + ((size_t)row * a.c.kvh + h) * a.count;
  // Digits from the top: `want` of the keys that share the prefix are still to be found.
  uint32_t prefix = 0, want = a.count;
  bool all = p.seen <= a.count;
  for (int shift = 24; shift >= 0 && !all; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
    for (uint32_t i = tid; i < p.seen; i += kTopThreads) {
      const uint32_t k = sort_key(score[i]);
      if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & 255u], 1u);
    }
    __syncthreads();
    if (wave == 0) {
      // lane i sums digits 4 i .. 4 i + 3, then counts from the largest digit down
      const uint32_t c0 = hist[4 * lane], c1 = hist[4 * lane + 1], c2 = hist[4 * lane + 2], c3 = hist[4 * lane + 3];
      const uint32_t mine = c0 + c1 + c2 + c3;
      uint32_t above = mine;  // becomes the sum over this lane and those after it
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_down(above, d);
        if (lane + d < 64) above += o;
      }
      above -= mine;
      if (above < want && above + mine >= want) {
        uint32_t left = want - above, digit = 4 * lane + 3;
        if (left > c3) left -= c3, digit = 4 * lane + 2;
        if (digit == 4 * lane + 2 && left > c2) left -= c2, digit = 4 * lane + 1;
        if (digit == 4 * lane + 1 && left > c1) left -= c1, digit = 4 * lane;
        pick[0] = digit;
        pick[1] = left;
      }
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    want = pick[1];
    __syncthreads();
  }
  // Keys above the limit, and the first `want` that equal it; no hole.
  const uint32_t limit = all ? kNoKey : max(prefix, kNoKey);
  if (limit == kNoKey) want = 0;
  uint32_t done = 0, same_done = 0;
  for (uint32_t i0 = 0; i0 < p.seen; i0 += kTopThreads) {
    const uint32_t i = i0 + tid;
    const uint32_t k = i < p.seen ? sort_key(score[i]) : 0u;
    const bool same = k == limit && i < p.seen;
    const uint64_t same_mask = __ballot(same);
    const uint64_t below = (1ull << lane) - 1;
    if (lane == 0) wave_same[wave] = (uint32_t)__popcll(same_mask);
    __syncthreads();
    uint32_t rank = same_done + (uint32_t)__popcll(same_mask & below);
#pragma unroll
    for (uint32_t w = 0; w < kTopThreads / 64; ++w) {
      if (w < wave) rank += wave_same[w];
      same_done += wave_same[w];
    }
    const bool take = k > limit || (same && rank < want);
    const uint64_t take_mask = __ballot(take);
    if (lane == 0) wave_more[wave] = (uint32_t)__popcll(take_mask);
    __syncthreads();
    uint32_t at = done + (uint32_t)__popcll(take_mask & below);
#pragma unroll
    for (uint32_t w = 0; w < kTopThreads / 64; ++w) {
      if (w < wave) at += wave_more[w];
      done += wave_more[w];
    }
    if (take && at < a.count) out[at] = (int32_t)i;
    __syncthreads();
  }
  for (uint32_t i = done + tid; i < a.count; i += kTopThreads) out[i] = -1;
}

}  // namespace
}  // namespace kv
}  // namespace dance

using namespace dance::kv;

extern "C" {

size_t dance_kv_select_work(const DanceKvCache* cache, const DanceKvBatch* batch, uint32_t heads, uint32_t count) {
  if (check_shapes(cache, batch) || heads == 0 || heads % cache->kv_heads || count == 0) return 0;
  return (size_t)batch->tokens * cache->kv_heads * most_blocks(cache, batch) * 4;
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
  const size_t need = dance_kv_select_work(cache, batch, queries->heads, count);
  if (!work || work_bytes < need || !aligned(work, 16))
    KV_ERR("dance_kv_select", "work must hold %zu bytes, aligned to 16", need);
  const uint32_t blocks = most_blocks(cache, batch);
  const uint64_t units = (uint64_t)batch->tokens * cache->kv_heads;
  const uint32_t per = 16 * kScoreWaves * 2;
  const uint32_t chunks = (blocks + per - 1) / per;
  if (units * chunks * 64 * kScoreWaves > 0xFFFFFFFFull || units * kTopThreads > 0xFFFFFFFFull)
    KV_ERR("dance_kv_select", "batch is too large for one launch");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const SelectArgs a{cache_args(cache), batch_args(batch), rows_args(queries), queries->heads / cache->kv_heads,
                     count, sink, recent, blocks, static_cast<float*>(work), chosen};
  with_kind(cache->dim, queries->dtype, [&](auto d, auto bf) {
    hipLaunchKernelGGL((k_score<decltype(d)::value, decltype(bf)::value>), dim3((uint32_t)(units * chunks)),
                       dim3(64 * kScoreWaves), 0, st, a, chunks, per);
  });
  hipLaunchKernelGGL(k_top, dim3((uint32_t)units), dim3(kTopThreads), 0, st, a);
  return launched("dance_kv_select");
}

}  // extern "C"
