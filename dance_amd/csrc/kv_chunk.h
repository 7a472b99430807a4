// dance_kv_attention for many rows of a sequence (prompts and their chunks):
// included by kv_attention.hip, whose notation this uses.
//
// A wave takes 32 rows, a workgroup W waves. The codes of 64 tokens become
// f16 in LDS once per workgroup (the conversion is then a tenth of a wave's
// instructions), two tiles deep, so that one barrier a tile is enough: around a tile's products the next one's codes
// go from registers to LDS and those of the one after set out.
// Products with 32x32x16 f16 MFMAs, S' = K Q' and O' += V' P'. Result
// register i of S' is token 8 (i / 4) + 4 (lane / 32) + i % 4 of 32; eight
// registers are one group of 16 tokens, which has one scale, and in their order the weights'
// operand of the second product. The value rows lie in LDS in the order that
// operand wants: within 16 tokens 0-3, 8-11, 4-7, 12-15, a swap of words.
//
// Bound by the softmax's and the conversion's vector instructions and the matrix units in turn: two chunks of
// 2048 tokens over 6,000 to 10,000, 8 kv heads of 4, 128 dimensions (491 GFLOP), 500 us, 980 TFLOP/s; a
// large f16 product reaches 1370. Vector instructions are 55 %, matrix instructions 45 % of the time.
#pragma once

// Waves per SIMD, by registers. At 64 dimensions, where a tile has half the products for as much softmax, more waves
// hide more: 8 sequences of 300 rows over 3000 tokens (8 kv heads of 4, bf16) take 104 us with three, 117 with two; four
// spill.
constexpr int chunk_occ(int d) { return d <= 64 ? 3 : d <= 128 ? 2 : 1; }

typedef float f16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float half_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// The order of N loads from LDS and the products that they feed: four loads ahead, then one for each product. Left to
// itself the compiler loads two and waits (two chunks of 2048 rows over 8000 tokens take 8 % less four ahead, two of 1024 over 4000 at 192
// dimensions 5 %).
template <int N, int GROUP>
__device__ __forceinline__ void operands_ahead() {
  constexpr int kProduct = 0x008, kLoad = 0x100, kFirst = 4;
  __builtin_amdgcn_sched_group_barrier(kLoad, kFirst, GROUP);
#pragma unroll
  for (int i = 0; i < N - kFirst; ++i) {
    __builtin_amdgcn_sched_group_barrier(kProduct, 1, GROUP);
    __builtin_amdgcn_sched_group_barrier(kLoad, 1, GROUP);
  }
  __builtin_amdgcn_sched_group_barrier(kProduct, kFirst, GROUP);
}

template <int D, bool BF, bool VEC, int W>
__global__ __launch_bounds__(64 * W)
    __attribute__((amdgpu_waves_per_eu(chunk_occ(D), chunk_occ(D)))) void k_chunk(StepArgs a) {
  constexpr int KS = D / 16;              // inner steps of the first product
  constexpr int DT = D / 32;              // row tiles of the second
  constexpr uint32_t KST = 2 * D + 16;    // bytes of a token's keys in LDS: rows of an operand in different banks
  constexpr uint32_t VST = 2 * 64 + 16;   // bytes of a dimension's values
  constexpr uint32_t kChunks = 4 * D;     // 16-byte pieces of a tile's key codes, and of its value codes
  constexpr int CN = (kChunks + 64 * W - 1) / (64 * W);
  constexpr uint32_t kRows = W * 32;
  // The next tile's codes go to LDS ahead of a tile's products, which hide the conversion; with one wave a SIMD, behind
  // them (two chunks of 1024 rows over 4000 tokens: at 128 dimensions 5 % less, at 192 and 256 21 and 7 % more).
  constexpr bool kAhead = D <= 128;
  // Blocks of a tile and more have addresses of their own (two chunks of 2048 rows over 8000 tokens take 3 % less so;
  // at 192 dimensions, where the registers then lie less well, two of 1024 over 4000 take 6 % more).
  constexpr bool kOneBlock = D != 192;
  __shared__ __attribute__((aligned(16))) char sk[2][64 * KST];
  __shared__ __attribute__((aligned(16))) char sv[2][D * VST];
  // of a tile's groups of 16 tokens: key scales (-infinity: a hole), log2 and inverses of the value scales
  __shared__ __attribute__((aligned(16))) float sg[2][3][4];
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t n = lane & 31u, hl = lane >> 5;
  const uint32_t bsh = a.c.bsh, bs = 1u << bsh;
  // Heads go round the XCDs, so that the workgroups that read the same tokens
  // share an L2 (with eight heads); a sequence's last rows, which see the most, first.
  uint32_t id = blockIdx.x;
  const uint32_t h = id % a.c.kvh;
  id /= a.c.kvh;
  const uint32_t split = id / a.slots;
  const TileAt at = tile_at(a.b, id % a.slots, a.group, kRows, a.tiles);
  if (at.sq >= a.b.seqs) return;
  const uint32_t sq = at.sq;
  const Seq s = seq_of(a.b, sq, bsh);
  const uint32_t r_end = s.n * a.group, tiles = (r_end + kRows - 1u) / kRows;
  if (at.tile >= tiles) return;
  const uint32_t r_first = (tiles - 1u - at.tile) * kRows;
  const uint32_t rows = min(kRows, r_end - r_first);
  auto pos_of = [&](uint32_t r) {
    const int64_t p = a.full ? s.len - 1 : min(s.first + r / a.group, s.len - 1);
    return p >= 0 ? (int32_t)p : -1;
  };
  auto row_of = [&](uint32_t rr) {
    const uint32_t rw = r_first + rr;
    return (size_t)(s.row + rw / a.group) * a.q.heads + h * a.group + rw % a.group;
  };
  const int32_t top = pos_of(r_first + rows - 1u);
  const int32_t seen = (int32_t)((uint32_t)(top + (int32_t)bs) >> bsh);  // blocks
  const uint32_t all = (uint32_t)(top + 64) / 64u;
  const uint32_t t_begin = split * a.per, t_end = split + 1 < a.splits ? min(all, t_begin + a.per) : all;
  float* const part_ml = a.part + (size_t)a.b.tokens * a.q.heads * a.splits * D;  // splits > 1
  if (a.splits > 1 && t_begin >= all) {
    for (uint32_t rr = tid; rr < rows; rr += 64 * W) {
      float* const pm = part_ml + (row_of(rr) * a.splits + split) * 2;
      pm[0] = -FLT_MAX;
      pm[1] = 0.f;
    }
    return;
  }
  const int32_t* const table = a.b.table + (size_t)sq * a.b.width;
  // Lane j of every wave keeps the block of group j % 4, as the table has it: what has just been asked for is not
  // looked at, since loads come back in order and to look at the last one is to wait for all.
  auto entry = [&](uint32_t tt) { return (int32_t)((tt * 64u + (lane & 3u) * 16u) >> bsh); };
  auto locate = [&](uint32_t tt) -> int32_t { return table[min(entry(tt), seen - 1)]; };
  u4_t kc[CN], vc[CN];
  float2 gs;    // of the lane's group: the scales
  bool hole;
  auto load_codes = [&](uint32_t tt, int32_t raw) {
    const int32_t ph = entry(tt) < seen && (uint32_t)raw < a.c.blocks ? raw : -1;
    if (kOneBlock && bsh >= 6) {  // the tile lies in one block: its place is the wave's, and a lane's offset in it stays
      const uint32_t one = (uint32_t)max(__builtin_amdgcn_readfirstlane(ph), 0);
      const size_t cell = (size_t)one * a.c.kvh + h;
      const uint32_t slot = (tt * 64u) & (bs - 1u);
      const int8_t* const k0 = a.c.k + ((cell << bsh) + slot) * D;
      const int8_t* const v0 = a.c.v + ((cell * D) << bsh) + slot;
#pragma unroll
      for (int i = 0; i < CN; ++i) {
        const uint32_t c = min(tid + i * 64 * W, kChunks - 1u);
        kc[i] = *reinterpret_cast<const u4_t*>(k0 + c * 16u);
        vc[i] = *reinterpret_cast<const u4_t*>(v0 + (((c >> 2) << bsh) + (c & 3u) * 16u));
      }
    } else {
#pragma unroll
    for (int i = 0; i < CN; ++i) {
      const uint32_t c = min(tid + i * 64 * W, kChunks - 1u);
      const uint32_t tok = c / (D / 16), off = c % (D / 16);
      const int32_t pk = max(__shfl(ph, (int)(tok >> 4)), 0), pv = max(__shfl(ph, (int)(c & 3u)), 0);
      const uint32_t slot_k = (tt * 64u + (tok & 48u)) & (bs - 1u), slot_v = (tt * 64u + (c & 3u) * 16u) & (bs - 1u);
      const size_t cell_k = (size_t)pk * a.c.kvh + h, cell_v = (size_t)pv * a.c.kvh + h;
      kc[i] = *reinterpret_cast<const u4_t*>(a.c.k + ((cell_k << bsh) + slot_k + (tok & 15u)) * D + off * 16);
      vc[i] = *reinterpret_cast<const u4_t*>(a.c.v + ((cell_v * D + (c >> 2)) << bsh) + slot_v);
    }
    }
    if (tid < 4) {
      gs = *reinterpret_cast<const float2*>(a.c.scale + ((size_t)max(ph, 0) * a.c.kvh + h) * 2);
      hole = ph < 0;
    }
  };
  auto store_codes = [&](uint32_t buf) {
#pragma unroll
    for (int i = 0; i < CN; ++i) {
      const uint32_t c = tid + i * 64 * W;
      if (kChunks % (64 * W) == 0 || c < kChunks) {
        const u2_t k0 = codes4(kc[i].x), k1 = codes4(kc[i].y), k2 = codes4(kc[i].z), k3 = codes4(kc[i].w);
        u4_t* const ko = reinterpret_cast<u4_t*>(sk[buf] + c / (D / 16) * KST + c % (D / 16) * 32);
        ko[0] = u4_t{k0.x, k0.y, k1.x, k1.y};
        ko[1] = u4_t{k2.x, k2.y, k3.x, k3.y};
        const u2_t v0 = codes4(vc[i].x), v1 = codes4(vc[i].y), v2 = codes4(vc[i].z), v3 = codes4(vc[i].w);
        u4_t* const vo = reinterpret_cast<u4_t*>(sv[buf] + (c >> 2) * VST + (c & 3u) * 32);
        vo[0] = u4_t{v0.x, v0.y, v2.x, v2.y};
        vo[1] = u4_t{v1.x, v1.y, v3.x, v3.y};
      }
    }
    if (tid < 4) {
      const float y = hole ? 1.f : fmaxf(gs.y, kLeastScale);
      sg[buf][0][tid] = hole ? -__builtin_inff() : gs.x;
      sg[buf][1][tid] = __builtin_amdgcn_logf(y);
      sg[buf][2][tid] = 1.f / y;
    }
  };

  int32_t ph = -1;  // of the tile after the one in the registers
  if (t_begin < t_end) {
    ph = locate(t_begin);
    load_codes(t_begin, ph);
    ph = locate(min(t_begin + 1, t_end - 1u));
  }

  // The wave's queries: dimensions 16 c + 8 (lane / 32) .., as f16 with a power of two taken out.
  h8_t qf[KS];
  const uint32_t r = r_first + min(wave * 32u + n, rows - 1u);
  const int32_t pos = pos_of(r);
  const uint16_t* const src = a.q.data + (int64_t)(s.row + r / a.group) * a.q.token_stride +
                              (int64_t)(h * a.group + r % a.group) * a.q.head_stride + 8 * hl;
  u4_t raw[KS];
#pragma unroll
  for (int c = 0; c < KS; ++c) {
    if constexpr (VEC) {
      raw[c] = *reinterpret_cast<const u4_t*>(src + 16 * c);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[c][i] = (uint32_t)src[16 * c + 2 * i] | (uint32_t)src[16 * c + 2 * i + 1] << 16;
    }
  }
  float qscale = fabsf(a.scale2);  // a negative scale turns the queries round, so that the largest product has the largest logit
  const uint32_t flip = a.scale2 < 0.f ? 0x80008000u : 0u;
  if constexpr (BF) {
    float mag = 0.f;
#pragma unroll
    for (int c = 0; c < KS; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        mag = fmaxf(mag, finite_abs(load_val<true>((uint16_t)(raw[c][i >> 1] >> (16 * (i & 1))))));
    mag = half_max(mag);
    int e = (int)(__float_as_uint(mag) >> 23) - 127 - 10;
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
  // first and last position of the wave's rows
  const uint32_t w_first = wave * 32u;
  const bool idle = w_first >= rows;
  const int32_t p_least = pos_of(r_first + min(w_first, rows - 1u));
  const int32_t p_most = idle ? -1 : pos_of(r_first + min(w_first + 32u, rows) - 1u);

  f16_t acc[DT];
  float R = -FLT_MAX;
  Sum l;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

  if (t_begin < t_end) {
    store_codes(0);
    load_codes(min(t_begin + 1, t_end - 1u), ph);
    ph = locate(min(t_begin + 2, t_end - 1u));
  }
  // Of the two waves that share a SIMD one goes first, so that its softmax meets the other's products (of eight waves; 1
  // to 4 %).
  if (wave & 4u) __builtin_amdgcn_s_setprio(1);
  auto stage = [&](uint32_t tt) {
    store_codes((tt - t_begin + 1) & 1u);  // behind the last tile: the last one again, which nobody reads
    load_codes(min(tt + 2, t_end - 1u), ph);
    ph = locate(min(tt + 3, t_end - 1u));
  };
  for (uint32_t tt = t_begin; tt < t_end; ++tt) {
    const uint32_t buf = (tt - t_begin) & 1u;
    const int32_t t0 = (int32_t)(tt * 64u);
    __syncthreads();
    if constexpr (kAhead) stage(tt);
    if (t0 <= p_most) {
      f16_t sc[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[u][i] = 0.f;
#pragma unroll
      for (int c = 0; c < KS; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const h8_t kf = *reinterpret_cast<const h8_t*>(sk[buf] + (u * 32u + n) * KST + c * 32 + hl * 16);
          sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[c], sc[u], 0, 0, 0);
        }
      operands_ahead<2 * KS, 0>();
      const f4_t gk = *reinterpret_cast<const f4_t*>(sg[buf][0]), gl = *reinterpret_cast<const f4_t*>(sg[buf][1]),
                 gi = *reinterpret_cast<const f4_t*>(sg[buf][2]);
      const bool holes = fminf(fminf(gk.x, gk.y), fminf(gk.z, gk.w)) == -__builtin_inff();
      const bool mask = __builtin_amdgcn_readfirstlane((int)holes) || t0 + 63 > p_least;
      h8_t pf[4];
      float kq[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) kq[j] = fmaxf(gk[j] * qscale, kLeastFactor);
      if (mask) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // tokens 8 x + y (y < 4) of this lane's in group j are seen up to this
          const int32_t m = gk[j] == -__builtin_inff() ? -1 : pos - (t0 + 16 * j + 4 * (int)hl);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (8 * (i >> 2) + (i & 3) > m) sc[j >> 1][8 * (j & 1) + i] = -__builtin_inff();
        }
      }
      float big = -FLT_MAX;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float m = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, sc[j >> 1][8 * (j & 1) + i]);
        big = fmaxf(big, __builtin_fmaf(m, kq[j], gl[j]));
      }
      if (__any(big > R + (kLift + kSlack))) {
        const float row_big = half_max(big);
        const float r_new = row_big > R + (kLift + kSlack) ? row_big - kLift : R;
        const float f = exp2f(R - r_new);
        l.scale(f);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] *= f;
        R = r_new;
      }
      float part = 0.f;  // at most 2^120: 32 tokens of the least scale
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float c = gl[j] - R;
        float add = 0.f, p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j >> 1][8 * (j & 1) + i], kq[j], c));
          add += p[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) pf[j][i] = (_Float16)p[i];
        part = __builtin_fmaf(add, gi[j], part);
      }
      l.add(part * kSumUnit);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const h8_t vf = *reinterpret_cast<const h8_t*>(sv[buf] + (d * 32u + n) * VST + j * 32 + hl * 16);
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[j], acc[d], 0, 0, 0);
        }
      operands_ahead<4 * DT, 1>();
    }
    if constexpr (!kAhead) stage(tt);
  }

  const float sum = half_sum(l.x);
  const uint32_t rr = wave * 32u + n;
  if (rr >= rows) return;
  const size_t row = row_of(rr);
  if (a.splits > 1) {
    float* const po = a.part + (row * a.splits + split) * D + 4 * hl;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<f4_t*>(po + 32 * d + 8 * x) =
            f4_t{acc[d][4 * x], acc[d][4 * x + 1], acc[d][4 * x + 2], acc[d][4 * x + 3]};
    if (hl == 0) {
      float* const pm = part_ml + (row * a.splits + split) * 2;
      pm[0] = R;
      pm[1] = sum;
    }
  } else {
    uint16_t* const out = a.out + row * D + 4 * hl;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<u2_t*>(out + 32 * d + 8 * x) =
            quotients<BF>(f4_t{acc[d][4 * x], acc[d][4 * x + 1], acc[d][4 * x + 2], acc[d][4 * x + 3]}, sum);
    if (a.lse && hl == 0) a.lse[row] = lse_of(R, sum);
  }
}
