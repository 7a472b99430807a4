// dance_kv_join (include/dance_kv_parts.h): attentions over parts of a context
// become the attention over all of it.
//
// With m the largest of a row's logarithms l_i, w_i = exp(l_i - m) and s = sum w_i, the row is sum w_i o_i / s
// and its logarithm m + log s: float32, one rounding to the rows' type at the end. bfloat16 reaches float32's range, so that
// a sum of eight rows would pass it: their weights are held in eighths, which changes no bit of normal numbers. Every lane has
// eight dimensions of a row and forms the weights itself, so that nothing is exchanged. Bound by bytes: 8192 rows of 32
// heads of 128, one part whole and two of half the rows (204 MB), 41 us, 5.0 TB/s, a large copy's rate; 64 rows of two
// parts 3.5 us, a launch and three loads in turn.

#include "../../include/dance_kv_parts.h"
#include "kv_common.h"

namespace dance {
namespace kv {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMostParts = 8;

struct Part {
  const uint16_t* __restrict__ data;
  const float* __restrict__ lse;
  const int32_t* __restrict__ rows;
  int64_t token_stride, head_stride;
  uint32_t tokens;
};
template <int P>
struct Join {
  Part part[P];
  uint32_t heads, dim, pieces, rows, cover;  // pieces of eight dimensions in a row; rows x heads; rows that a workgroup covers
  uint16_t* __restrict__ out;
  float* __restrict__ lse;
};

template <int P, bool BF, bool VEC>
__global__ __launch_bounds__(kThreads) void k_join_parts(Join<P> a) {
  const uint32_t row = blockIdx.x * a.cover + threadIdx.x / a.pieces, piece = threadIdx.x % a.pieces;
  if (threadIdx.x >= a.cover * a.pieces || row >= a.rows) return;
  const uint32_t token = row / a.heads, head = row % a.heads;
  float l[P];
  uint32_t at[P];
  float m = -__builtin_inff();
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const Part& x = a.part[p];
    at[p] = x.rows ? (uint32_t)x.rows[token] : token;
    l[p] = at[p] < x.tokens ? x.lse[(size_t)at[p] * a.heads + head] : -__builtin_inff();
    m = l[p] > m || l[p] != l[p] ? l[p] : m;
  }
  constexpr float kUnit = BF ? 0.125f : 1.f;
  float w[P], sum = 0.f;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const float x = l[p] == -__builtin_inff() ? 0.f : expf(l[p] - m);
    sum += x;
    w[p] = x * kUnit;
  }
  if (a.lse && piece == 0) a.lse[row] = m + logf(sum);  // -infinity where all parts are
  const float inv = sum == 0.f ? 0.f : 1.f / sum * (1.f / kUnit);
  for (uint32_t d = piece * 8; d < a.dim; d += a.pieces * 8) {
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if constexpr (VEC) {
      u4_t raw[P];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        raw[p] = u4_t{0u, 0u, 0u, 0u};
        if (w[p] != 0.f)
          raw[p] = *reinterpret_cast<const u4_t*>(a.part[p].data + (int64_t)at[p] * a.part[p].token_stride +
                                                  (int64_t)head * a.part[p].head_stride + d);
      }
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          o[i] = __builtin_fmaf(w[p], load_val<BF>((uint16_t)(raw[p][i >> 1] >> (16 * (i & 1)))), o[i]);
      uint32_t y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        y[i] = store_val<BF>(o[2 * i] * inv) | (uint32_t)store_val<BF>(o[2 * i + 1] * inv) << 16;
      *reinterpret_cast<u4_t*>(a.out + (size_t)row * a.dim + d) = u4_t{y[0], y[1], y[2], y[3]};
    } else {
      const uint32_t n = min(8u, a.dim - d);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (w[p] == 0.f) continue;
        const uint16_t* const src = a.part[p].data + (int64_t)at[p] * a.part[p].token_stride +
                                    (int64_t)head * a.part[p].head_stride + d;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          if (i < n) o[i] = __builtin_fmaf(w[p], load_val<BF>(src[i]), o[i]);
      }
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (i < n) a.out[(size_t)row * a.dim + d + i] = store_val<BF>(o[i] * inv);
    }
  }
}

}  // namespace
}  // namespace kv
}  // namespace dance

extern "C" int dance_kv_join(const DanceKvPart* parts, uint32_t count, uint32_t tokens, uint32_t heads, uint32_t dim, int dtype,
                             void* out, float* lse, void* stream) {
  using namespace dance::kv;
  const char* why = nullptr;
  if (!parts || count == 0 || count > kMostParts) why = "1 to 8 parts must be given";
  if (!why && dtype != DANCE_KV_F16 && dtype != DANCE_KV_BF16) why = "rows must be float16 or bfloat16";
  if (!why && (heads == 0 || heads > 65535u || dim == 0 || dim > 65536u)) why = "heads must be in [1, 65535], dim in [1, 65536]";
  if (!why && (uint64_t)tokens * heads > 0x7FFFFFFFull) why = "batch is too large for one launch";
  if (!why && tokens && (!out || !aligned(out, 2))) why = "out must be given, aligned to its elements";
  bool vec = dim % 8 == 0 && aligned(out, 16);
  Join<kMostParts> a{};
  for (uint32_t i = 0; !why && i < count; ++i) {
    const DanceKvPart& p = parts[i];
    if (p.tokens > 0x7FFFFFFFull) why = "a part must have fewer than 2^31 rows";
    else if (!p.rows && p.tokens != tokens) why = "a part without rows has one row for each that is joined";
    else if (p.tokens && (!p.data || !p.lse || !aligned(p.data, 2))) why = "null part, or rows not aligned to their elements";
    vec = vec && aligned(p.data, 16) && p.token_stride % 8 == 0 && p.head_stride % 8 == 0;
    a.part[i] = Part{static_cast<const uint16_t*>(p.data), p.lse, p.rows, p.token_stride, p.head_stride, (uint32_t)p.tokens};
  }
  if (why) KV_ERR("dance_kv_join", "%s", why);
  if (tokens == 0) return 0;
  a.heads = heads, a.dim = dim, a.rows = tokens * heads;
  const uint32_t all = (dim + 7) / 8;
  a.pieces = all < kThreads ? all : kThreads;
  a.cover = kThreads / a.pieces;
  a.out = static_cast<uint16_t*>(out), a.lse = lse;
  const uint32_t grid = (a.rows + a.cover - 1) / a.cover;
  if ((uint64_t)grid * kThreads > 0xFFFFFFFFull) KV_ERR("dance_kv_join", "batch is too large for one launch");
  auto go = [&](auto n, auto bf, auto v) {
    constexpr int P = decltype(n)::value;
    Join<P> b;
    for (int i = 0; i < P; ++i) b.part[i] = a.part[i];
    b.heads = a.heads, b.dim = a.dim, b.pieces = a.pieces, b.rows = a.rows, b.cover = a.cover, b.out = a.out, b.lse = a.lse;
    hipLaunchKernelGGL((k_join_parts<P, decltype(bf)::value, decltype(v)::value>), dim3(grid), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), b);
  };
  auto kind = [&](auto n) {
    if (dtype == DANCE_KV_BF16)
      vec ? go(n, std::true_type{}, std::true_type{}) : go(n, std::true_type{}, std::false_type{});
    else
      vec ? go(n, std::false_type{}, std::true_type{}) : go(n, std::false_type{}, std::false_type{});
  };
  switch (count) {  // fewer parts than the kernel's have no rows
    case 1:
    case 2: kind(Int<2>{}); break;
    case 3:
    case 4: kind(Int<4>{}); break;
    default: kind(Int<8>{}); break;
  }
  return launched("dance_kv_join");
}
