// Attention of a few new tokens per sequence over the paged 4-bit cache (layout: kv4.cuh).
//
// With x_c = scale_j code_c + low_j for channel c of group j, and p = exp(s - m):
//   s   = sum_j scale^k_j (sum_{c in j} code_c q_c) + sum_j low^k_j (sum_{c in j} q_c)
//   o_c = sum_tau (p_tau scale^v_{tau j}) code_{tau c} + sum_tau p_tau low^v_{tau j}
// so the codes themselves feed the tensor cores and no value is ever rebuilt: a nibble left where
// it stands in a half-word is the fp16 subnormal code 2^-24 (or 16 code 2^-24, undone by a factor
// 1/16 on q, or on the output's row), which takes one AND per two values.  K's scales multiply the
// fp32 sums of a group, V's the fp16 probabilities, the lows are one more small product, with the
// row sum of p as a row of ones beside V's lows.
//
// m16n8k16: rows = 16 tokens (K) or 16 channels (V), columns = 8 of the query rows (new token,
// head of the group) that share a kv head.  q is scaled by a power of two per row to [2^8, 2^9)
// at its largest, so bf16's range fits fp16 and 32 q sum below 2^14; sums of q go in as a
// high and a low half.  The products accumulate in fp32, running maximum and sum are fp32; p is
// rounded to fp16 (2^-11 relative, against bf16's 2^-9 at the output).  A row's reference maximum
// moves when a score passes it by more than 2 (log2 units), so p <= 4 and p scale <= 4 x 8735
// stays finite for every scale that the append kernel writes.
//
// A CTA of 8 warps takes one split of one (sequence, kv head); each warp takes every eighth unit of
// 32 tokens with its own bulk-copy ring, running maximum, sum and accumulator, so nothing is
// exchanged until the warps' results meet in shared memory at the end.  Splits meet in a second
// kernel, in order, so the result does not depend on timing.
#include "host_util.h"
#include "kv4.cuh"

namespace rldx {

namespace {
constexpr int kDecWarps = 8;
constexpr int kDecStages = 2;
constexpr float kDecGrow = 2.0f;  // lazy move of the reference maximum (log2 units)

template <int D, int NT>
struct DecShape {
  static constexpr int kCols = 8 * NT;
  static constexpr int kRing = kDecWarps * kDecStages * Kv4Unit<D>::kBytes;
  static constexpr int kOLd = D + 4;  // floats of one column's partial result
  static constexpr int kMerge = kDecWarps * kCols * kOLd * 4;
  static constexpr int kBody = kRing > kMerge ? kRing : kMerge;
  static constexpr int kMl = kDecWarps * kCols * 8;  // (reference maximum, sum)
  static constexpr size_t kSmem = kBody + kMl + 8 * kDecWarps * kDecStages + 16;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ float2 h2_floats(uint32_t u) { return __half22float2(bits_h2(u)); }

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// 4 G bytes per lane: G words.
template <int G>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[G]) {
  if constexpr (G == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x, w[1] = u.y;
  }
}
}  // namespace

// Rows of a CTA's columns: column c of tile `tile` is new token (tile * kCols + c) / group, head
// (tile * kCols + c) % group of the kv head's group.
template <int D, int NT>
__global__ void __launch_bounds__(32 * kDecWarps, NT == 1 ? 2 : 1)
    kv4_decode_kernel(const __grid_constant__ Kv4AttnParams P) {
  using U = Kv4Unit<D>;
  using Sh = DecShape<D, NT>;
  constexpr int G = U::kG;
  constexpr int kCols = Sh::kCols;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* body = smem;
  float2* s_ml = reinterpret_cast<float2*>(smem + Sh::kBody);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Sh::kBody + Sh::kMl);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int tile = blockIdx.y / P.c.kv_heads, kvh = blockIdx.y - tile * P.c.kv_heads;
  const int b = blockIdx.z, split = blockIdx.x;

  if (threadIdx.x < kDecWarps * kDecStages) mbar_init(&bars[threadIdx.x], 1);
  if (threadIdx.x == 0) fence_mbar_init();
  griddep_wait();
  griddep_launch();
  const int q0 = P.c.cu[b], nq = P.c.cu[b + 1] - q0;
  const int c0 = tile * kCols, ncols = min(kCols, nq * P.group - c0);
  if (ncols <= 0) return;  // the whole CTA
  if (q0 < 0 || q0 + nq > P.c.tokens) {
    if (threadIdx.x == 0) record_error(kErrKv4Table);
    return;
  }
  const int len = P.c.lengths[b];
  const Kv4Span span = kv4_span(len, nq, c0 / P.group, (c0 + ncols - 1) / P.group, P.window, P.sinks);
  if (threadIdx.x == 0 && (nq > P.max_new || len > P.max_len)) record_error(kErrKv4Bound);
  const int u_begin = split * P.chunk_units, u_end = min(span.count, u_begin + P.chunk_units);
  if (split > 0 && u_begin >= u_end) return;  // the combine kernel counts the splits the same way

  // ---- this warp's units: lane i holds the place of the i-th (u_begin + warp + 8 i) ----
  const int mine = max(0, (u_end - u_begin - warp + kDecWarps - 1) / kDecWarps);  // <= 32
  long long my_off = -1;
  if (lane < mine) {
    my_off = kv4_unit_offset(P.c, b, kvh, span.unit(u_begin + warp + kDecWarps * lane), U::kBytes);
    if (my_off < 0) record_error(kErrKv4Table);
  }
  uint8_t* ring = body + warp * kDecStages * U::kBytes;
  uint64_t* bar = bars + warp * kDecStages;
  __syncthreads();
  const uint64_t policy = l2_policy_evict_first();
  auto fetch = [&](int i) {  // every lane calls it; a unit without a page is not fetched
    const long long off = __shfl_sync(0xffffffffu, my_off, i);
    if (lane == 0) {
      uint64_t* bb = &bar[i % kDecStages];
      if (off >= 0) {
        mbar_arrive_expect_tx(bb, U::kBytes);
        bulk_load(ring + (i % kDecStages) * U::kBytes, P.c.data + off, U::kBytes, bb, policy);
      } else {
        mbar_arrive(bb);
      }
    }
  };
  for (int i = 0; i < kDecStages && i < mine; ++i) fetch(i);

  // ---- q: B fragments of column 8 nt + g, channels 32 j + 8 t + 0..7 ----
  uint32_t qf[NT][G][4], qsum[NT];
  float colfac[NT][2];  // log2 score per unit of the products, for columns 2t, 2t + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = 8 * nt + g;
    const int row = c0 + col, tok = row / P.group;
    float v[G][8], mx = 0.0f;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (col < ncols)
        u = *reinterpret_cast<const uint4*>(P.q + (q0 + tok) * P.ldq +
                                            static_cast<long long>(kvh * P.group + row - tok * P.group) * D + 32 * j + 8 * t);
      unpack_bf16x2(u.x, v[j][0], v[j][1]);
      unpack_bf16x2(u.y, v[j][2], v[j][3]);
      unpack_bf16x2(u.z, v[j][4], v[j][5]);
      unpack_bf16x2(u.w, v[j][6], v[j][7]);
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(v[j][e]));
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // 2^e with e = 8 - exponent(mx), kept a normal number; a row of zeros keeps 1
    const int ex = static_cast<int>(__float_as_uint(mx) >> 23);
    const int e2 = mx > 0.0f ? min(max(262 - ex, 1), 253) : 127;
    const float up = __uint_as_float(static_cast<uint32_t>(e2) << 23);
    const float down = __uint_as_float(static_cast<uint32_t>(254 - e2) << 23);
    float part[G];
#pragma unroll
    for (int j = 0; j < G; ++j) {
      part[j] = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[j][e] *= up;
        part[j] += v[j][e];
      }
      part[j] += __shfl_xor_sync(0xffffffffu, part[j], 1);
      part[j] += __shfl_xor_sync(0xffffffffu, part[j], 2);
      // nibbles 0, 4 | 1, 5 (sixteen times their code) | 2, 6 | 3, 7
      qf[nt][j][0] = h2_bits(__floats2half2_rn(v[j][0], v[j][4]));
      qf[nt][j][1] = h2_bits(__floats2half2_rn(v[j][1] * 0.0625f, v[j][5] * 0.0625f));
      qf[nt][j][2] = h2_bits(__floats2half2_rn(v[j][2], v[j][6]));
      qf[nt][j][3] = h2_bits(__floats2half2_rn(v[j][3] * 0.0625f, v[j][7] * 0.0625f));
    }
    // sums of q for the lows: lanes t = 0, 1 hold the fp16 high halves of groups 0, 1 | 2, 3, lanes
    // t = 2, 3 what those leave
    float sa = part[0], sb = part[1];
    if constexpr (G == 4) {
      if (t & 1) sa = part[2], sb = part[3];
    } else {
      if (t & 1) sa = sb = 0.0f;
    }
    const __half2 hi = __floats2half2_rn(sa, sb);
    const float2 hf = __half22float2(hi);
    qsum[nt] = h2_bits(t < 2 ? hi : __floats2half2_rn(sa - hf.x, sb - hf.y));
    const float cf = P.scale_log2 * down;
    colfac[nt][0] = __shfl_sync(0xffffffffu, cf, 8 * t);
    colfac[nt][1] = __shfl_sync(0xffffffffu, cf, 8 * t + 4);
  }
  int pos[NT][2];  // position of columns 2t, 2t + 1 of each tile
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) pos[nt][i] = span.pos_lo + min(c0 + 8 * nt + 2 * t + i, c0 + ncols - 1) / P.group - c0 / P.group;

  float acc[NT][G][2][4], low[NT][4];  // O of channels 32 j + 4 g + 2 s (and + 1), low sums and row sum
  float m_ref[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][j][s][i] = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) low[nt][i] = 0.0f;
    m_ref[nt][0] = m_ref[nt][1] = -INFINITY;
  }

  bool ok = true;
  for (int i = 0; i < mine; ++i) {
    const int st = i % kDecStages;
    ok = mbar_wait(&bar[st], static_cast<uint32_t>(i / kDecStages) & 1u, kErrKv4Timeout);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    const uint8_t* un = ring + st * U::kBytes;
    const bool have = __shfl_sync(0xffffffffu, my_off, i) >= 0;
    const int key0 = kKv4Unit * span.unit(u_begin + warp + kDecWarps * i);
    const int key_hi = key0 + kKv4Unit - 1;
    const bool plain = have && key_hi <= span.pos_lo &&
                       (P.window <= 0 || span.pos_hi - key0 < P.window || key_hi < P.sinks);

    // ---- scores of 32 tokens (two tiles of 16) ----
    float sc[2][NT][4];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      uint32_t ka[G], kb[G], ma[G], mb[G];
      lds_words<G>(un + blk * 16 * U::kRow + lane * 4 * G, ka);
      lds_words<G>(un + blk * 16 * U::kRow + 8 * U::kRow + lane * 4 * G, kb);
      lds_words<G>(un + U::kKMeta + (blk * 16 + g) * 4 * G, ma);
      lds_words<G>(un + U::kKMeta + (blk * 16 + 8 + g) * 4 * G, mb);
      float sa[G], sb[G];
#pragma unroll
      for (int j = 0; j < G; j += 2) {
        const float2 a = h2_floats(ma[j / 2]), c = h2_floats(mb[j / 2]);
        sa[j] = a.x, sa[j + 1] = a.y, sb[j] = c.x, sb[j + 1] = c.y;
      }
      uint32_t la = ma[G / 2], lb = mb[G / 2];
      if constexpr (G == 4) {
        if (t & 1) la = ma[3], lb = mb[3];
      } else {
        if (t & 1) la = lb = 0u;
      }
      float sm[NT][4], sum[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sm[nt][e] = sum[nt][e] = 0.0f;
        mma_1688(sm[nt], la, lb, qsum[nt]);
      }
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const uint32_t wa = ka[j], wb = kb[j], va = wa >> 8, vb = wb >> 8;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma_16816(d, wa & 0x000f000fu, wb & 0x000f000fu, wa & 0x00f000f0u, wb & 0x00f000f0u, qf[nt][j][0], qf[nt][j][1]);
          mma_16816(d, va & 0x000f000fu, vb & 0x000f000fu, va & 0x00f000f0u, vb & 0x00f000f0u, qf[nt][j][2], qf[nt][j][3]);
          sum[nt][0] = fmaf(sa[j], d[0], sum[nt][0]);
          sum[nt][1] = fmaf(sa[j], d[1], sum[nt][1]);
          sum[nt][2] = fmaf(sb[j], d[2], sum[nt][2]);
          sum[nt][3] = fmaf(sb[j], d[3], sum[nt][3]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[blk][nt][e] = fmaf(16777216.0f, sum[nt][e], sm[nt][e]) * colfac[nt][e & 1];
    }
    if (!plain) {
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 16 * blk + 8 * (e >> 1) + g, ps = pos[nt][e & 1];
            const bool seen = have && key <= ps && (P.window <= 0 || ps - key < P.window || key < P.sinks);
            sc[blk][nt][e] = seen ? sc[blk][nt][e] : -INFINITY;
          }
    }
    // ---- running maximum ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) mx[e] = fmaxf(fmaxf(sc[0][nt][e], sc[0][nt][e + 2]), fmaxf(sc[1][nt][e], sc[1][nt][e + 2]));
      if (__any_sync(0xffffffffu, mx[0] > m_ref[nt][0] + kDecGrow || mx[1] > m_ref[nt][1] + kDecGrow)) {
        float al[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o <= 16; o <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], o));
          const float m = fmaxf(m_ref[nt][e], mx[e]);
          al[e] = m_ref[nt][e] == -INFINITY ? 0.0f : ex2_approx(m_ref[nt][e] - m);
          m_ref[nt][e] = m;
        }
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][j][s][e] *= al[e & 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) low[nt][e] *= al[e & 1];
      }
    }
    // ---- O += P V ----
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      uint32_t pb[NT][2];  // B fragments of p: tokens 2t, 2t + 1 of each half, column g
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float m0 = m_ref[nt][0] == -INFINITY ? 0.0f : m_ref[nt][0];
        const float m1 = m_ref[nt][1] == -INFINITY ? 0.0f : m_ref[nt][1];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          pb[nt][h] = transpose_8x8(h2_bits(
              __floats2half2_rn(ex2_approx(sc[blk][nt][2 * h] - m0), ex2_approx(sc[blk][nt][2 * h + 1] - m1))));
      }
      uint32_t v0[G], v1[G], s0[G], s1[G];
      lds_words<G>(un + U::kV + blk * 8 * D + lane * 4 * G, v0);
      lds_words<G>(un + U::kV + blk * 8 * D + 4 * D + lane * 4 * G, v1);
      lds_words<G>(un + U::kVScale + blk * 32 * G + t * 4 * G, s0);
      lds_words<G>(un + U::kVScale + blk * 32 * G + 16 * G + t * 4 * G, s1);
      uint32_t l0 = g == 4 ? 0x3c003c00u : 0u, l1 = l0;  // rows 0..G-1: lows of a group; row 4: ones
      if (g < G) {
        l0 = *reinterpret_cast<const uint32_t*>(un + U::kVLow + blk * 32 * G + t * 4 * G + 4 * g);
        l1 = *reinterpret_cast<const uint32_t*>(un + U::kVLow + blk * 32 * G + 16 * G + t * 4 * G + 4 * g);
        if (!plain) {  // a NaN low comes with a NaN scale, which reaches the columns that see the token
          l0 &= __hlt2_mask(__habs2(bits_h2(l0)), bits_h2(0x7c007c00u));
          l1 &= __hlt2_mask(__habs2(bits_h2(l1)), bits_h2(0x7c007c00u));
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_16816(low[nt], l0, 0u, l1, 0u, pb[nt][0], pb[nt][1]);
#pragma unroll
      for (int j = 0; j < G; ++j) {
        // half-words of group j of tokens 2t | 2t + 1
        const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
        const uint32_t x0 = __byte_perm(v0[j / 2], v0[G / 2 + j / 2], sel), x1 = __byte_perm(v1[j / 2], v1[G / 2 + j / 2], sel);
        const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          uint32_t b0 = h2_bits(__hmul2(bits_h2(pb[nt][0]), bits_h2(s0[j])));
          uint32_t b1 = h2_bits(__hmul2(bits_h2(pb[nt][1]), bits_h2(s1[j])));
          if (!plain) {  // p = 0 stays 0 beside whatever stands in a hidden token's scale
            b0 &= __hneu2_mask(bits_h2(pb[nt][0]), bits_h2(0u));
            b1 &= __hneu2_mask(bits_h2(pb[nt][1]), bits_h2(0u));
          }
          mma_16816(acc[nt][j][0], x0 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x000f000fu, x1 & 0x00f000f0u, b0, b1);
          mma_16816(acc[nt][j][1], y0 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x000f000fu, y1 & 0x00f000f0u, b0, b1);
        }
      }
    }
    __syncwarp();  // every lane has read the unit
    if (i + kDecStages < mine) fetch(i + kDecStages);
  }
  if (!ok) settle_issued_copies();

  // ---- the warps' results meet in shared memory ----
  __syncthreads();  // every ring is idle
  float* so = reinterpret_cast<float*>(body);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = 8 * nt + 2 * t + e;
      const float l = __shfl_sync(0xffffffffu, low[nt][e], 16 + t);
      if (g == 0) s_ml[warp * kCols + col] = make_float2(m_ref[nt][e], l);
      float* dst = so + (warp * kCols + col) * Sh::kOLd + 4 * g;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const float lw = __shfl_sync(0xffffffffu, low[nt][e], 4 * j + t);
        float4 o;
        o.x = fmaf(16777216.0f, acc[nt][j][0][e], lw);
        o.y = fmaf(1048576.0f, acc[nt][j][0][e + 2], lw);
        o.z = fmaf(16777216.0f, acc[nt][j][1][e], lw);
        o.w = fmaf(1048576.0f, acc[nt][j][1][e + 2], lw);
        *reinterpret_cast<float4*>(dst + 32 * j) = o;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ncols * (D / 4); i += 32 * kDecWarps) {
    const int col = i / (D / 4), ch = i % (D / 4) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) m = fmaxf(m, s_ml[w * kCols + col].x);
    const float m_use = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float2 ml = s_ml[w * kCols + col];
      if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // saw no visible token
      const float f = ex2_approx(ml.x - m_use);
      const float4 x = *reinterpret_cast<const float4*>(so + (w * kCols + col) * Sh::kOLd + ch);
      l = fmaf(f, ml.y, l);
      o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y), o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
    }
    const int row = c0 + col, tok = row / P.group;
    const long long orow = static_cast<long long>(q0 + tok) * P.q_heads + kvh * P.group + row - tok * P.group;
    if (P.chunks == 1) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no visible token: zeros
      uint2 u;
      u.x = pack_bf16x2(o.x * inv, o.y * inv);
      u.y = pack_bf16x2(o.z * inv, o.w * inv);
      *reinterpret_cast<uint2*>(P.out + orow * D + ch) = u;
    } else {
      *reinterpret_cast<float4*>(P.part_o + (orow * P.chunks + split) * D + ch) = o;
      if (ch == 0) P.part_ml[orow * P.chunks + split] = make_float2(m, l);
    }
  }
}

// out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s over a row's splits; D / 4 lanes per row.
template <int D>
__global__ void __launch_bounds__(128) kv4_combine_kernel(const __grid_constant__ Kv4AttnParams P, int cols_per_cta) {
  constexpr int kLanes = D / 4;
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.y;
  const int q0 = P.c.cu[b], nq = P.c.cu[b + 1] - q0;
  if (q0 < 0 || q0 + nq > P.c.tokens) return;
  const int r = (blockIdx.x * blockDim.x + threadIdx.x) / kLanes, ch = threadIdx.x % kLanes * 4;
  if (r >= nq * P.q_heads) return;
  const int tok = r / P.q_heads, head = r - tok * P.q_heads;
  const int col = tok * P.group + head % P.group;  // column of its kv head
  const int c0 = col / cols_per_cta * cols_per_cta, c1 = min(c0 + cols_per_cta, nq * P.group) - 1;
  const Kv4Span span = kv4_span(P.c.lengths[b], nq, c0 / P.group, c1 / P.group, P.window, P.sinks);
  const int n = min(P.chunks, max(1, (span.count + P.chunk_units - 1) / P.chunk_units));
  const long long row = static_cast<long long>(q0) * P.q_heads + r;
  const float2* ml = P.part_ml + row * P.chunks;
  const float* po = P.part_o + row * P.chunks * D + ch;
  float m = -INFINITY;
  for (int s = 0; s < n; ++s) m = fmaxf(m, ml[s].x);
  const float m_use = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int s = 0; s < n; ++s) {
    const float2 x = ml[s];
    const float4 v = *reinterpret_cast<const float4*>(po + static_cast<long long>(s) * D);
    const float f = x.x == -INFINITY && x.y == 0.0f ? 0.0f : ex2_approx(x.x - m_use);
    l = fmaf(f, x.y, l);
    o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint2 u;
  u.x = pack_bf16x2(o.x * inv, o.y * inv);
  u.y = pack_bf16x2(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(P.out + row * D + ch) = u;
}

namespace {
template <typename K, typename... A>
cudaError_t launch_pdl(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int D, int NT>
cudaError_t launch_decode(const Kv4AttnParams& p, cudaStream_t stream) {
  const int tiles = (p.max_new * p.group + 8 * NT - 1) / (8 * NT);
  cudaError_t e = launch_pdl(kv4_decode_kernel<D, NT>, dim3(p.chunks, tiles * p.c.kv_heads, p.c.seqs), 32 * kDecWarps,
                             DecShape<D, NT>::kSmem, stream, p);
  if (e != cudaSuccess || p.chunks == 1) return e;
  const int rows_per_block = 128 / (D / 4);
  return launch_pdl(kv4_combine_kernel<D>,
                    dim3((p.max_new * p.q_heads + rows_per_block - 1) / rows_per_block, p.c.seqs, 1), 128, 0, stream, p,
                    8 * NT);
}

template <int D, int NT>
cudaError_t decode_smem() {
  return cudaFuncSetAttribute(kv4_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(DecShape<D, NT>::kSmem));
}
}  // namespace

cudaError_t launch_kv4_decode(const Kv4AttnParams& p, int head_dim, int cols_per_cta, cudaStream_t stream) {
  if (head_dim == 128)
    return cols_per_cta == 8 ? launch_decode<128, 1>(p, stream) : launch_decode<128, 2>(p, stream);
  return cols_per_cta == 8 ? launch_decode<64, 1>(p, stream) : launch_decode<64, 2>(p, stream);
}

cudaError_t kv4_prepare_device() {
  cudaError_t e = decode_smem<128, 1>();
  if (e == cudaSuccess) e = decode_smem<128, 2>();
  if (e == cudaSuccess) e = decode_smem<64, 1>();
  if (e == cudaSuccess) e = decode_smem<64, 2>();
  return e;
}

namespace {
struct DecodePlan {
  int cols, chunk_units, chunks;
  uint64_t bytes;  // workspace of the splits' results
};

// Columns per CTA and the split over the length.  Splits until two rounds of the resident CTAs
// (two per SM) are full or a warp is left with one unit; a split has at most 256 units (each
// warp holds the places of its units in its 32 lanes).
DecodePlan decode_plan(const rldx_kv4_cache& c, int tokens, int q_heads, int max_new, int max_len, int window, int sinks) {
  DecodePlan p;
  const int group = q_heads / c.kv_heads;
  p.cols = max_new * group <= 8 ? 8 : 16;
  const long long tiles = (static_cast<long long>(max_new) * group + p.cols - 1) / p.cols;
  const long long base = tiles * c.kv_heads * c.seqs;
  long long keys = max_len;
  if (window > 0) keys = std::min<long long>(keys, static_cast<long long>(window) + max_new + std::min(sinks, max_len) + 3 * kKv4Unit);
  const long long units = std::max<long long>(1, (keys + kKv4Unit - 1) / kKv4Unit);
  const long long want = std::max<long long>(1, 4LL * sm_count() / base);
  long long per = std::max<long long>(kDecWarps, (units + want - 1) / want);
  per = std::min<long long>((per + kDecWarps - 1) / kDecWarps * kDecWarps, 32 * kDecWarps);
  p.chunk_units = static_cast<int>(per);
  p.chunks = static_cast<int>((units + per - 1) / per);
  const uint64_t rows = static_cast<uint64_t>(tokens) * q_heads;
  p.bytes = p.chunks == 1 ? 0 : rows * p.chunks * (static_cast<uint64_t>(c.head_dim) * 4 + 8);
  return p;
}

int attention_args(const rldx_kv4_cache* cache, const rldx_kv4_attention_desc* a, Kv4AttnParams* p) {
  if (!a) return set_error(RLDX_ERR_ARG, "kv4_attention: null description");
  int rc = kv4_cache(cache, a->tokens, "kv4_attention", &p->c);
  if (rc != RLDX_OK) return rc;
  if (a->q_heads <= 0 || a->q_heads % cache->kv_heads) return set_error(RLDX_ERR_ARG, "kv4_attention: kv_heads must divide q_heads");
  if (a->max_new <= 0 || a->max_len <= 0) return set_error(RLDX_ERR_ARG, "kv4_attention: max_new and max_len must be positive");
  if (a->window < 0 || a->sinks < 0) return set_error(RLDX_ERR_ARG, "kv4_attention: window and sinks must not be negative");
  if (!(a->scale > 0.0f) || !(a->scale < 1e30f)) return set_error(RLDX_ERR_ARG, "kv4_attention: the scale must be positive");
  if (cache->seqs > 65535) return set_error(RLDX_ERR_UNSUPPORTED, "kv4_attention: more than 65535 sequences");
  if (static_cast<long long>(a->tokens) * a->q_heads >= (1LL << 31) || static_cast<long long>(a->max_new) * a->q_heads >= (1LL << 19))
    return set_error(RLDX_ERR_UNSUPPORTED, "kv4_attention: too many rows");
  return RLDX_OK;
}
}  // namespace

}  // namespace rldx

using namespace rldx;

extern "C" {

int rldx_kv4_attention_workspace_size(const rldx_kv4_cache* cache, const rldx_kv4_attention_desc* a, uint64_t* bytes) {
  if (!bytes) return set_error(RLDX_ERR_ARG, "kv4_attention_workspace_size: null bytes");
  *bytes = 0;
  Kv4AttnParams p;
  int rc = attention_args(cache, a, &p);
  if (rc != RLDX_OK) return rc;
  *bytes = decode_plan(*cache, a->tokens, a->q_heads, a->max_new, std::min<long long>(a->max_len, static_cast<long long>(cache->table_width) * cache->page_size), a->window, a->sinks).bytes;
  return RLDX_OK;
}

int rldx_kv4_attention(const rldx_kv4_cache* cache, const rldx_kv4_attention_desc* a, void* workspace,
                       uint64_t workspace_bytes, void* stream) {
  int rc = ensure_device();
  if (rc != RLDX_OK) return rc;
  Kv4AttnParams p;
  rc = attention_args(cache, a, &p);
  if (rc != RLDX_OK) return rc;
  const int d = cache->head_dim;
  if (!a->q || !a->out || !aligned_to(a->q, 16) || !aligned_to(a->out, 16))
    return set_error(RLDX_ERR_ARG, "kv4_attention: q and out must be 16-byte aligned");
  if (a->ldq < static_cast<int64_t>(a->q_heads) * d || a->ldq % 8)
    return set_error(RLDX_ERR_ARG, "kv4_attention: q rows must be 16-byte aligned and hold every head");
  if (a->tokens == 0) return RLDX_OK;
  const int max_len = static_cast<int>(std::min<long long>(a->max_len, static_cast<long long>(cache->table_width) * cache->page_size));
  const DecodePlan plan = decode_plan(*cache, a->tokens, a->q_heads, a->max_new, max_len, a->window, a->sinks);
  if (plan.bytes > workspace_bytes || (plan.bytes > 0 && (!workspace || !aligned_to(workspace, 16))))
    return set_error(RLDX_ERR_ARG, "kv4_attention: needs a 16-byte aligned workspace of " + std::to_string(plan.bytes) + " bytes");
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.ldq = a->ldq;
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.q_heads = a->q_heads;
  p.group = a->q_heads / cache->kv_heads;
  p.window = a->window;
  p.sinks = a->window > 0 ? a->sinks : 0;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.max_new = a->max_new;
  p.max_len = max_len;
  p.chunk_units = plan.chunk_units;
  p.chunks = plan.chunks;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (plan.chunks > 1 ? static_cast<size_t>(a->tokens) * a->q_heads * plan.chunks * d : 0));
  cudaError_t e = launch_kv4_decode(p, d, plan.cols, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "kv4_attention launch");
  return RLDX_OK;
}

}  // extern "C"
