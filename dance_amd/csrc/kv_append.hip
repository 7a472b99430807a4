// dance_kv_append (include/dance_kv.h): new keys and values become 8-bit codes
// of their block's scale.
//
// Scales are powers of two, the least that holds the block's largest value. So
// x / s is exact and its rounding the only one; a block that grows at least
// doubles its scale, so that re-rounding its old codes moves a value by less
// than one step of the final scale however often it grows; and any order or
// precision of the arithmetic gives the same codes.
// What a block that held tokens before holds behind its last one is not kept: of the 16 values that are
// written together those are zeros.
//
// One workgroup per (sequence, touched block, head) and for keys and values
// apart: the scale is a maximum over exactly that, so one launch finds it and
// writes the codes, and the second read of the rows comes from the cache.
// Measured: 64 sequences of one token, 8 heads of 128, 9.2 us, a chain of dependent loads
// (length, table, rows, scale); 7,105 tokens of 16 prompts 21 us, 2.1 TB/s of
// compulsory bytes, the same chain in eight workgroups a CU.

#include <cmath>
#include <type_traits>

#include "kv_common.h"

namespace dance {
namespace kv {
namespace {

constexpr uint32_t kAppendThreads = 256;
constexpr uint32_t kMostTokens = 128;  // of a block

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
__global__ __launch_bounds__(kAppendThreads) void k_append(Cache c, Batch bt, Rows keys, Rows values) {
  constexpr uint32_t C8 = D / 8;                   // chunks of 8 dimensions in a row
  constexpr uint32_t kRows = kAppendThreads / C8;  // rows that the workgroup walks at once
  constexpr uint32_t C16 = D / 16, kRows16 = kAppendThreads / C16;
  constexpr uint32_t kAhead = 2;  // rows of old key codes that a thread asks for at the start
  __shared__ float wave_max[kAppendThreads / 64];
  // keys: each thread row's largest and least codes; values: codes [dim][4 tokens], rows a word longer than a block
  __shared__ __attribute__((aligned(16))) uint32_t lds[D * (kMostTokens / 4 + 1)];
  uint32_t id = blockIdx.x;
  const bool is_v = id & 1u;
  id >>= 1;
  const uint32_t h = id % c.kvh;
  id /= c.kvh;
  uint32_t sq = id, j = 0;  // the j-th block that the sequence's rows may touch
  if (bt.offsets) {
    // Sequence b has the indexes from slot(b) up to slot(b + 1): n rows touch at most
    // n / tokens + 2 blocks. So the grid goes by the rows that there are, not by the
    // longest sequence's (16 prompts of 1 to 4,000 tokens: 2,288 workgroups, not 16,384; 20.5 and 22.3 us).
    auto slot = [&](uint32_t b) { return ((uint32_t)max(bt.offsets[b], 0) >> c.bsh) + 2u * b; };
    uint32_t before = 0;  // sequences that start at or before this index, by 64
    for (uint32_t b0 = 0; b0 < bt.seqs; b0 += 64) {
      const uint32_t b = b0 + (threadIdx.x & 63u);
      const uint64_t mask = __ballot(b < bt.seqs && slot(b) <= id);
      before += (uint32_t)__popcll(mask);
      if (mask != ~0ull) break;
    }
    sq = (uint32_t)__builtin_amdgcn_readfirstlane((int)(before - 1u));
    if (sq >= bt.seqs) return;
    j = id - slot(sq);
  }
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

  const uint32_t c16 = tid % C16, r16 = tid / C16;
  int8_t* const keys_out = c.k + (cell << c.bsh) * D;
  u4_t was_code[kAhead];
#pragma unroll
  for (uint32_t i = 0; i < kAhead; ++i)
    if (!is_v && r16 < kRows16 && r16 + i * kRows16 < old)
      was_code[i] = *reinterpret_cast<const u4_t*>(keys_out + (size_t)(r16 + i * kRows16) * D + c16 * 16);

  float* const scale = c.scale + cell * 2 + (is_v ? 1 : 0);
  const float was = old ? *scale : 0.f;
  float a = 0.f;
  if (r0 < kRows)
    for (uint32_t t = r0; t < cnt; t += kRows) {
      const V8 x = load8<BF, VEC>(src + (int64_t)t * rows.token_stride + d8 * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(x.x[i]));
    }
  a = rows_max(cols_max(a));
  if ((tid & 63u) == 0) wave_max[tid >> 6] = a;
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < kAppendThreads / 64; ++w) a = fmaxf(a, wave_max[w]);
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
    // The bounds come from the block's codes, the old ones included.
    int mx[16], mn[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) mx[i] = -128, mn[i] = 127;
    const uint32_t to = old ? old + cnt : (uint32_t)bs;
    auto keep = [&](uint32_t t, const int (&q)[16], bool write) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        mx[i] = max(mx[i], q[i]);
        mn[i] = min(mn[i], q[i]);
      }
      if (write)
        *reinterpret_cast<u4_t*>(keys_out + (size_t)t * D + c16 * 16) =
            u4_t{pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]), pack4(q[8], q[9], q[10], q[11]),
                 pack4(q[12], q[13], q[14], q[15])};
    };
    auto one = [&](uint32_t t, u4_t o) {  // o: the old codes, where t has them
      int q[16];
      if (t < old) {
#pragma unroll
        for (int i = 0; i < 16; ++i) q[i] = shrink(byte_of(o[i >> 2], i & 3), ratio);
        keep(t, q, grow);
      } else if (t < old + cnt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const V8 x = load8<BF, VEC>(src + (int64_t)(t - old) * rows.token_stride + c16 * 16 + 8 * e);
#pragma unroll
          for (int i = 0; i < 8; ++i) q[8 * e + i] = code(x.x[i]);
        }
        keep(t, q, true);
      } else {
        *reinterpret_cast<u4_t*>(keys_out + (size_t)t * D + c16 * 16) = u4_t{0u, 0u, 0u, 0u};
      }
    };
    if (r16 < kRows16) {
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i)
        if (r16 + i * kRows16 < to) one(r16 + i * kRows16, was_code[i]);
      for (uint32_t t = r16 + kAhead * kRows16; t < to; t += kRows16)
        one(t, t < old ? *reinterpret_cast<const u4_t*>(keys_out + (size_t)t * D + c16 * 16) : u4_t{0u, 0u, 0u, 0u});
      uint32_t* const at = lds + r16 * (D / 2) + c16 * 4;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        at[w] = pack4(mx[4 * w], mx[4 * w + 1], mx[4 * w + 2], mx[4 * w + 3]);
        at[D / 4 + w] = pack4(mn[4 * w], mn[4 * w + 1], mn[4 * w + 2], mn[4 * w + 3]);
      }
    }
    __syncthreads();
    const int8_t* const part = reinterpret_cast<const int8_t*>(lds);
    const uint32_t n = min(kRows16, to);
    for (uint32_t i = tid; i < 2 * D; i += kAppendThreads) {
      int b = part[i];
#pragma unroll 8
      for (uint32_t r = 1; r < n; ++r) b = i < D ? max(b, (int)part[r * 2 * D + i]) : min(b, (int)part[r * 2 * D + i]);
      c.bound[cell * 2 * D + i] = (int8_t)b;
    }
  } else {
    // Values lie dims-major. Rows are read as they lie, four tokens x 8 dimensions
    // a thread, turned in LDS, and leave 16 tokens of a dimension at a time.
    constexpr uint32_t kStride = kMostTokens / 4 + 1;
    int8_t* const out = c.v + (cell * D << c.bsh);
    const uint32_t from = old && !grow ? old / 16 : 0u, to = old ? (old + cnt + 15) / 16 : (uint32_t)bs / 16;  // of 16 tokens
    const uint32_t quads = (to - from) * 4;
    for (uint32_t i = tid; i < quads * C8; i += kAppendThreads) {
      const uint32_t q = 4 * from + i / C8, e8 = i % C8;
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
      for (int d = 0; d < 8; ++d) lds[(e8 * 8 + d) * kStride + q] = pack4(got[0][d], got[1][d], got[2][d], got[3][d]);
    }
    __syncthreads();
    const uint32_t parts = to - from;
    for (uint32_t i = tid; i < parts * D; i += kAppendThreads) {
      const uint32_t p = from + i % parts, d = i / parts;
      u4_t* const at = reinterpret_cast<u4_t*>(out + ((size_t)d << c.bsh)) + p;
      u4_t w;
#pragma unroll
      for (int x = 0; x < 4; ++x) w[x] = lds[d * kStride + 4 * p + x];
      if (16 * p < old) {
        const u4_t o = *at;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          int b[4];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            b[r] = 16 * p + 4 * x + r < old ? shrink(byte_of(o[x], r), ratio) : byte_of(w[x], r);
          w[x] = pack4(b[0], b[1], b[2], b[3]);
        }
      }
      *at = w;
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
  const uint64_t blocks = batch->offsets ? batch->tokens / bs + 2ull * batch->seqs : batch->seqs;
  const uint64_t grid = blocks * cache->kv_heads * 2;
  if (grid * kAppendThreads > 0xFFFFFFFFull) KV_ERR("dance_kv_append", "batch is too large for one launch");
  const bool vec = rows_vector(keys) && rows_vector(values);
  with_kind(cache->dim, keys->dtype, [&](auto d, auto bf) {
    constexpr int D = decltype(d)::value;
    constexpr bool BF = decltype(bf)::value;
    if (vec)
      hipLaunchKernelGGL((k_append<D, BF, true>), dim3((uint32_t)grid), dim3(kAppendThreads), 0,
                         static_cast<hipStream_t>(stream), cache_args(cache), batch_args(batch), rows_args(keys),
                         rows_args(values));
    else
      hipLaunchKernelGGL((k_append<D, BF, false>), dim3((uint32_t)grid), dim3(kAppendThreads), 0,
                         static_cast<hipStream_t>(stream), cache_args(cache), batch_args(batch), rows_args(keys),
                         rows_args(values));
  });
  return launched("dance_kv_append");
}
