// dance_kv_append (include/dance_kv.h): new keys and values become 8-bit codes
// of their block's scale.
//
// Scales are powers of two, the least that holds the block's largest value. So
// x / s is exact and its rounding the only one; a block that grows at least
// doubles its scale, so that re-rounding its old codes moves a value by less
// than one step of the final scale however often it grows; and any order or
// precision of the arithmetic gives the same codes.
//
// One workgroup per (sequence, touched block, head) and for keys and values
// apart: the scale is a maximum over exactly that, so one launch finds it and
// writes the codes, and the second read of the rows comes from the cache.

#include <cmath>
#include <type_traits>

#include "kv_common.h"

namespace dance {
namespace kv {
namespace {

constexpr uint32_t kAppendThreads = 256;

struct V8 {
  float x[8];
};
template <bool BF, bool VEC>
__device__ __forceinline__ V8 load8(const uint16_t* __restrict__ p) {
  V8 r;
  if constexpr (VEC) {
    const u4_t u = *reinterpret_cast<const u4_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) r.x[i] = load_val<BF>((uint16_t)(u[i >> 1] >> (16 * (i & 1))));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.x[i] = load_val<BF>(p[i]);
  }
  return r;
}

__device__ __forceinline__ int byte_of(uint32_t w, int i) { return (int)(int8_t)(w >> (8 * i)); }
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)(d & 255) << 24;
}
__device__ __forceinline__ int shrink(int c, float ratio) { return (int)__builtin_rintf((float)c * ratio); }

template <int D, bool BF, bool VEC>
__global__ __launch_bounds__(kAppendThreads) void k_append(Cache c, Batch bt, Rows keys, Rows values, uint32_t per) {
  constexpr uint32_t C8 = D / 8;                      // chunks of 8 dimensions in a row
  constexpr uint32_t kRows = kAppendThreads / C8;     // rows that the workgroup walks at once
  __shared__ float wave_max[kAppendThreads / 64];
  __shared__ int top[2 * D];  // the block's new bounds
  uint32_t id = blockIdx.x;
  const bool is_v = id & 1u;
  id >>= 1;
  const uint32_t h = id % c.kvh;
  id /= c.kvh;
  const uint32_t j = id % per, sq = id / per;
  const Seq s = seq_of(bt, sq, c.bsh);
  const int64_t bs = 1ll << c.bsh;
  const int64_t blk = ((s.first > 0 ? s.first : 0) >> c.bsh) + j;
  const int64_t lo = s.first > blk * bs ? s.first : blk * bs;
  const int64_t end = s.first + s.n < s.len ? s.first + s.n : s.len;
  const int64_t hi = end < (blk + 1) * bs ? end : (blk + 1) * bs;
  if (lo >= hi) return;
  const int32_t phys = bt.table[(size_t)sq * bt.width + (size_t)blk];
  if (phys < 0 || (uint32_t)phys >= c.blocks) return;
  const uint32_t old = (uint32_t)(lo - blk * bs), cnt = (uint32_t)(hi - lo);
  const size_t cell = (size_t)phys * c.kvh + h;
  const Rows& rows = is_v ? values : keys;
  const uint16_t* src = rows.data + (int64_t)(s.row + (uint32_t)(lo - s.first)) * rows.token_stride +
                        (int64_t)h * rows.head_stride;
  const uint32_t tid = threadIdx.x, d8 = tid % C8, r0 = tid / C8;

  float a = 0.f;
  if (r0 < kRows)
    for (uint32_t t = r0; t < cnt; t += kRows) {
      const V8 x = load8<BF, VEC>(src + (int64_t)t * rows.token_stride + d8 * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(x.x[i]));
    }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) a = fmaxf(a, __shfl_xor(a, m));
  if ((tid & 63u) == 0) wave_max[tid >> 6] = a;
  if (!is_v)
    for (uint32_t i = tid; i < 2 * D; i += kAppendThreads) top[i] = i < D ? -128 : 127;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < kAppendThreads / 64; ++w) a = fmaxf(a, wave_max[w]);
  float* const scale = c.scale + cell * 2 + (is_v ? 1 : 0);
  const float was = old ? *scale : 0.f;
  const float now = fmaxf(was, exp2_int(scale_exp(a)));
  const bool grow = old && now > was;
  const float ratio = was / now;  // old codes' factor; 1 where the block keeps its scale
  __syncthreads();                // every thread has read the scale
  if (tid == 0) *scale = now;
  // A scale that this call or an earlier one chose is a power of two, whose
  // inverse is exact; others divide.
  const bool pow2 = (__float_as_uint(now) & 0x7FFFFFu) == 0;
  const float inv = 1.f / now;
  auto code = [&](float x) { return pow2 ? code_of(x, inv) : code_of(x / now, 1.f); };

  if (!is_v) {
    int8_t* const out = c.k + (cell << c.bsh) * D;
    int8_t* const bound = c.bound + cell * 2 * D;
    int mx[8], mn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) mx[i] = -128, mn[i] = 127;
    // The bounds come from the block's codes, the old ones included.
    const uint32_t to = old ? old + cnt : (uint32_t)bs;
    if (r0 < kRows)
      for (uint32_t t = r0; t < to; t += kRows) {
        u2_t* const at = reinterpret_cast<u2_t*>(out + (size_t)t * D + d8 * 8);
        int q[8];
        if (t < old) {
          const u2_t o = *at;
#pragma unroll
          for (int i = 0; i < 8; ++i) q[i] = shrink(byte_of(o[i >> 2], i & 3), ratio);
        } else if (t < old + cnt) {
          const V8 x = load8<BF, VEC>(src + (int64_t)(t - old) * rows.token_stride + d8 * 8);
#pragma unroll
          for (int i = 0; i < 8; ++i) q[i] = code(x.x[i]);
        } else {
          *at = u2_t{0u, 0u};
          continue;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          mx[i] = max(mx[i], q[i]);
          mn[i] = min(mn[i], q[i]);
        }
        if (t >= old || grow) *at = u2_t{pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7])};
      }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (mx[i] >= mn[i]) {
        atomicMax(&top[d8 * 8 + i], mx[i]);
        atomicMin(&top[D + d8 * 8 + i], mn[i]);
      }
    }
    __syncthreads();
    for (uint32_t i = tid; i < 2 * D; i += kAppendThreads) bound[i] = (int8_t)top[i];
  } else {
    // Values lie dims-major: a thread turns 4 tokens x 8 dimensions into a word
    // for each dimension; neighbouring threads hold neighbouring words.
    int8_t* const out = c.v + (cell * D << c.bsh);
    const uint32_t from = old && !grow ? old / 4 : 0u, to = old ? (old + cnt + 3) / 4 : (uint32_t)bs / 4;
    const uint32_t quads = to - from;
    for (uint32_t i = tid; i < quads * C8; i += kAppendThreads) {
      const uint32_t q = from + i % quads, e8 = i / quads;
      int got[4][8];
#pragma unroll
      for (uint32_t r = 0; r < 4; ++r) {
        const uint32_t t = 4 * q + r;
        if (t >= old && t < old + cnt) {
          const V8 x = load8<BF, VEC>(src + (int64_t)(t - old) * rows.token_stride + e8 * 8);
#pragma unroll
          for (int d = 0; d < 8; ++d) got[r][d] = code(x.x[d]);
        } else {
#pragma unroll
          for (int d = 0; d < 8; ++d) got[r][d] = 0;
        }
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        uint32_t* const at = reinterpret_cast<uint32_t*>(out + ((size_t)(e8 * 8 + d) << c.bsh)) + q;
        if (4 * q < old) {
          const uint32_t o = *at;
#pragma unroll
          for (uint32_t r = 0; r < 4; ++r)
            if (4 * q + r < old) got[r][d] = shrink(byte_of(o, r), ratio);
        }
        *at = pack4(got[0][d], got[1][d], got[2][d], got[3][d]);
      }
    }
  }
}

}  // namespace
}  // namespace kv
}  // namespace dance

extern "C" int dance_kv_append(const DanceKvCache* cache, const DanceKvBatch* batch, const DanceKvRows* keys,
                               const DanceKvRows* values, void* stream) {
  using namespace dance::kv;
  const char* why = check_common(cache, batch);
  if (!why) why = check_rows(cache, keys, true);
  if (!why) why = check_rows(cache, values, true);
  if (!why && keys->dtype != values->dtype) why = "keys and values must have one type";
  if (why) KV_ERR("dance_kv_append", "%s", why);
  if (batch->tokens == 0) return 0;
  const uint32_t bs = cache->block_tokens;
  const uint32_t per = (batch->max_tokens + bs - 2) / bs + 1;  // blocks that max_tokens adjacent tokens can touch
  const uint64_t grid = (uint64_t)batch->seqs * per * cache->kv_heads * 2;
  if (grid * kAppendThreads > 0xFFFFFFFFull) KV_ERR("dance_kv_append", "batch is too large for one launch");
  const bool vec = rows_vector(keys) && rows_vector(values);
  with_kind(cache->dim, keys->dtype, [&](auto d, auto bf) {
    constexpr int D = decltype(d)::value;
    constexpr bool BF = decltype(bf)::value;
    if (vec)
      hipLaunchKernelGGL((k_append<D, BF, true>), dim3((uint32_t)grid), dim3(kAppendThreads), 0,
                         static_cast<hipStream_t>(stream), cache_args(cache), batch_args(batch), rows_args(keys),
                         rows_args(values), per);
    else
      hipLaunchKernelGGL((k_append<D, BF, false>), dim3((uint32_t)grid), dim3(kAppendThreads), 0,
                         static_cast<hipStream_t>(stream), cache_args(cache), batch_args(batch), rows_args(keys),
                         rows_args(values), per);
  });
  return launched("dance_kv_append");
}
