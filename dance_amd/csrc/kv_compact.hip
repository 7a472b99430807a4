// dance_kv_compact (include/dance_kv_pages.h): chosen tokens, densely, in blocks of
// their own scales.
//
// A token's code times its block's scale is exact in float32 where the scale is a power of two, and the new
// scale is one, so a code whose block keeps its scale stays as it is and the one
// rounding is that of a block that mixes scales.
//
// One workgroup per (sequence, new block, head) and for keys and values apart: the scale is a maximum over
// exactly that. Codes stay in registers from their one load to their rounding. Keys come 16 bytes of a token at
// a time. Values lie dims-major, so a token's are bytes of different lines: lanes stand for
// neighbouring tokens, which mostly lie in the same lines, and leave as words of four tokens that four lanes
// exchange by DPP.

#include "../../include/dance_kv_pages.h"
#include "kv_common.h"

namespace dance {
namespace kv {
namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kMostTokens = 128;  // of a block

struct Compact {
  Cache from, to;
  const int32_t* __restrict__ table;
  const int32_t* __restrict__ lengths;
  const int32_t* __restrict__ keep;
  const int32_t* __restrict__ counts;
  const int32_t* __restrict__ into;
  uint32_t width, keep_heads, keep_width, into_width;
};

__device__ __forceinline__ int byte_at(uint32_t w, int i) { return (int)(int8_t)(w >> (8 * i)); }
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)(d & 255) << 24;
}
__device__ __forceinline__ int largest(uint32_t w, int a) {
#pragma unroll
  for (int i = 0; i < 4; ++i) a = max(a, abs(byte_at(w, i)));
  return a;
}

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

template <int D>
__global__ __launch_bounds__(kThreads) void k_compact(Compact a, uint32_t places) {
  constexpr uint32_t C16 = D / 16, kRows = kThreads / C16;        // keys: pieces of a token, tokens at once
  constexpr uint32_t NP = (kMostTokens + kRows - 1) / kRows;      // pieces of a thread
  constexpr uint32_t NW = (D * kMostTokens / kThreads + 3) / 4;   // values: words of four dimensions of a thread
  __shared__ float wave_max[kWaves], t_scale[kMostTokens];
  __shared__ uint64_t t_at[kMostTokens];  // of a token: where its head's block begins, in codes, and its place in it
  __shared__ uint32_t t_slot[kMostTokens];
  __shared__ __attribute__((aligned(16))) uint32_t part[kRows * (D / 2)];  // each thread row's largest and least codes
  const uint32_t tid = threadIdx.x, bsh = a.from.bsh, bs = 1u << bsh;
  uint32_t id = blockIdx.x;
  const bool is_v = id & 1u;
  id >>= 1;
  const uint32_t h = id % a.from.kvh;
  id /= a.from.kvh;
  const uint32_t j = id % places, b = id / places;
  const uint32_t count = min((uint32_t)max(a.counts[b], 0), a.keep_width);
  if ((uint64_t)j << bsh >= count) return;
  const int32_t dst = a.into[(size_t)b * a.into_width + j];
  if ((uint32_t)dst >= a.to.blocks) return;
  const uint32_t live = min(bs, count - (j << bsh));
  if (tid < bs) {
    uint64_t at = 0;
    uint32_t slot = 0;
    float s = 0.f;
    if (tid < live) {
      const uint32_t hk = a.keep_heads == 1 ? 0u : h;
      const int32_t pos = a.keep[((size_t)b * a.keep_heads + hk) * a.keep_width + (j << bsh) + tid];
      const int64_t room = (int64_t)a.width << bsh;
      if (pos >= 0 && pos < a.lengths[b] && pos < room) {
        const int32_t p = a.table[(size_t)b * a.width + ((uint32_t)pos >> bsh)];
        if ((uint32_t)p < a.from.blocks) {
          const size_t cell = (size_t)p * a.from.kvh + h;
          at = (cell * D) << bsh;
          slot = (uint32_t)pos & (bs - 1u);
          s = a.from.scale[cell * 2 + (is_v ? 1 : 0)];
        }
      }
    }
    t_at[tid] = at;
    t_slot[tid] = slot;
    t_scale[tid] = s;  // 0: no such token, whatever is read for it
  }
  __syncthreads();

  const size_t cell = (size_t)dst * a.to.kvh + h;
  auto finish = [&](float most) {  // the new scale, from each thread's largest magnitude
    most = rows_max(cols_max(most));
    if ((tid & 63u) == 0) wave_max[tid >> 6] = most;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) most = fmaxf(most, wave_max[w]);
    const float now = exp2_int(scale_exp(most));
    if (tid == 0) a.to.scale[cell * 2 + (is_v ? 1 : 0)] = now;
    return 1.f / now;
  };
  float most = 0.f;
  if (!is_v) {
    const uint32_t c16 = tid % C16, r = tid / C16;
    u4_t w[NP];
#pragma unroll
    for (uint32_t i = 0; i < NP; ++i) {
      const uint32_t t = r + i * kRows;
      w[i] = u4_t{0u, 0u, 0u, 0u};
      if (r < kRows && t < live) w[i] = *reinterpret_cast<const u4_t*>(a.from.k + t_at[t] + t_slot[t] * D + c16 * 16);
    }
#pragma unroll
    for (uint32_t i = 0; i < NP; ++i) {
      const uint32_t t = r + i * kRows;
      if (r < kRows && t < live) {
        int m = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x) m = largest(w[i][x], m);
        most = fmaxf(most, finite_abs((float)m * t_scale[t]));
      }
    }
    const float inv = finish(most);
    int mx[16], mn[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) mx[i] = -128, mn[i] = 127;
    int8_t* const out = a.to.k + ((cell * D) << bsh);
#pragma unroll
    for (uint32_t i = 0; i < NP; ++i) {
      const uint32_t t = r + i * kRows;
      if (r >= kRows || t >= bs) continue;
      u4_t y = {0u, 0u, 0u, 0u};
      if (t < live) {
        const float s = t_scale[t];
        int q[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          q[x] = code_of((float)byte_at(w[i][x >> 2], x & 3) * s, inv);
          mx[x] = max(mx[x], q[x]);
          mn[x] = min(mn[x], q[x]);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) y[x] = pack4(q[4 * x], q[4 * x + 1], q[4 * x + 2], q[4 * x + 3]);
      }
      *reinterpret_cast<u4_t*>(out + t * D + c16 * 16) = y;
    }
    if (r < kRows) {
      uint32_t* const at = part + r * (D / 2) + c16 * 4;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        at[x] = pack4(mx[4 * x], mx[4 * x + 1], mx[4 * x + 2], mx[4 * x + 3]);
        at[D / 4 + x] = pack4(mn[4 * x], mn[4 * x + 1], mn[4 * x + 2], mn[4 * x + 3]);
      }
    }
    __syncthreads();
    const int8_t* const p8 = reinterpret_cast<const int8_t*>(part);
    const uint32_t n = min(kRows, live);
    for (uint32_t i = tid; i < 2 * D; i += kThreads) {
      int v = p8[i];
      for (uint32_t x = 1; x < n; ++x) v = i < D ? max(v, (int)p8[x * 2 * D + i]) : min(v, (int)p8[x * 2 * D + i]);
      a.to.bound[cell * 2 * D + i] = (int8_t)v;
    }
  } else {
    // thread: token t, dimensions 4 (g + i groups) ..
    const uint32_t t = tid & (bs - 1u), g = tid >> bsh, groups = kThreads >> bsh;
    const float s = t_scale[t];
    const int8_t* const src = a.from.v + t_at[t] + t_slot[t];
    uint32_t w[NW];
#pragma unroll
    for (uint32_t i = 0; i < NW; ++i) {
      const uint32_t d = 4 * (g + i * groups);
      w[i] = 0u;
      if (d < D && t < live) {
        const int8_t* const p = src + ((size_t)d << bsh);
        w[i] = pack4(p[0], p[(size_t)1 << bsh], p[(size_t)2 << bsh], p[(size_t)3 << bsh]);
      }
    }
    int m = 0;
#pragma unroll
    for (uint32_t i = 0; i < NW; ++i) m = largest(w[i], m);
    const float inv = finish(finite_abs((float)m * s));
    int8_t* const out = a.to.v + ((cell * D) << bsh) + (t & ~3u);
#pragma unroll
    for (uint32_t i = 0; i < NW; ++i) {
      const uint32_t d = 4 * (g + i * groups);
      if (d >= D) continue;  // the four lanes that exchange have one d
      int q[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) q[x] = code_of((float)byte_at(w[i], x) * s, inv);
      const uint32_t y = turn4(pack4(q[0], q[1], q[2], q[3]), tid);
      *reinterpret_cast<uint32_t*>(out + ((size_t)(d + (tid & 3u)) << bsh)) = y;
    }
  }
}

}  // namespace
}  // namespace kv
}  // namespace dance

extern "C" int dance_kv_compact(const DanceKvCache* from, const DanceKvCache* to, const int32_t* table, const int32_t* lengths,
                                uint32_t seqs, uint32_t width, const int32_t* keep, uint32_t keep_heads, uint32_t keep_width,
                                const int32_t* counts, const int32_t* into_table, uint32_t into_width, void* stream) {
  using namespace dance::kv;
  const DanceKvBatch source{table, lengths, nullptr, seqs, seqs, width, 1, 0}, target{into_table, counts, nullptr, seqs, seqs, into_width, 1, 0};
  const char* why = check_common(from, &source);
  if (!why) why = check_common(to, &target);
  if (!why && (from->kv_heads != to->kv_heads || from->dim != to->dim || from->block_tokens != to->block_tokens))
    why = "both caches must have one kv_heads, dim and block_tokens";
  if (!why && !keep) why = "null keep";
  if (!why && keep_heads != 1 && keep_heads != from->kv_heads) why = "keep_heads must be 1 or kv_heads";
  if (!why && (keep_width == 0 || keep_width > 0x7FFFFFFFu)) why = "keep_width must be in [1, 2^31)";
  if (why) KV_ERR("dance_kv_compact", "%s", why);
  // places that the lists can fill
  const uint32_t most = (keep_width - 1) / from->block_tokens + 1, places = most < into_width ? most : into_width;
  const uint64_t grid = (uint64_t)seqs * places * from->kv_heads * 2;
  if (grid > 0xFFFFFFFFull / kThreads) KV_ERR("dance_kv_compact", "batch is too large for one launch");
  const Compact a{cache_args(from), cache_args(to), table, lengths, keep, counts, into_table,
                  width, keep_heads, keep_width, into_width};
  with_kind(from->dim, DANCE_KV_F16, [&](auto d, auto) {
    hipLaunchKernelGGL((k_compact<decltype(d)::value>), dim3((uint32_t)grid), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), a, places);
  });
  return launched("dance_kv_compact");
}
