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
// high and a low half.  The products accumulate in fp32, running maximum and sum are fp32.  p and p scale
// are rounded to fp16 for the MMA (2^-11 relative each, against bf16's 2^-8 at the output; the row's sum takes
// the rounded p, so that the weights still add up to one).  That bound holds over fp16's normal numbers, so both
// are kept at their top: a row's p is held 2^11 times or more, its largest up to 2^15 (kDecSet, kDecMove), and V's scales
// go in times a power of two that each warp keeps for its units, the largest near 1/2.  What falls below is off by
// 2^-25 beside 2^11: a token counts with its bits down to 2^-25 of the largest weight, whatever the size of
// V.  8192 tokens, V of size 1 / 1e-3 / 1e-4 / 1e-5, error against 64 bits (the output's rounding alone 0.0017): 0.0017
// each; with p <= 4 and the scales as they are 0.0017 / 0.004 / 0.12 / 3.4, for 3 to 5 % less time.
//
// Work is split evenly over one wave of CTAs, whatever the lengths: a segment is one (sequence, kv
// head, tile of columns) with the units that it can see, all segments stand in one line and each
// CTA takes the same share of it, found by a prefix sum over the sequences that every CTA makes
// for itself.  Inside a CTA each of W = 4 (8) warps takes every W-th unit with its own bulk-copy ring,
// running maximum, sum and accumulator, so nothing is exchanged until the warps' results meet in
// shared memory at a segment's end.  A segment cut between CTAs is joined by a second kernel, in
// the CTAs' order, so the result does not depend on timing.
//
// Measured: 64 sequences of up to 8192 tokens, 16 / 2 heads, d = 128, 120 MB of cache: 32.0 us with the join,
// 3.73 TB/s, 0.57 of the copy's rate; 3 x 131077 27.7 us, 0.53.  Four warps a CTA and four CTAs an
// SM, 32 KB of copies in flight a CTA: 33.0 us against 35.7 with eight warps and two CTAs, when both were measured.  What is left is the
// start (lengths, prefix sums, q: about 3 us before the first unit is used), the shared-memory merge at a
// segment's end and the join's launch (3.5 us).
#include <type_traits>

#include "host_util.h"
#include "kv4.cuh"

namespace rldx {

namespace {
constexpr int kDecWarps = 4, kDecWarpsWide = 8;  // of a CTA; of one that has a short segment to itself
constexpr int dec_resident(int warps, int cols) { return 128 / (warps * cols); }  // CTAs per SM (128 registers a thread)
constexpr int kDecStages = 2;
// A row's reference (log2 units) stands 11 below the largest score when it is set and is set again once one passes it
// by more than 15, so that p = 2^(score - reference) is at most 2^15, and 2^11 or more for the largest.
constexpr float kDecSet = 11.0f, kDecMove = 15.0f;

constexpr int kDecMaxSeqs = 1024;        // sequences of one launch (their prefix sums stand in shared memory)
constexpr long long kDecMaxLine = 1 << 30;  // and units of all their segments (32-bit sums): pages may be shared, so memory sets no bound

// A segment's start counts as this many units of a CTA's share: its lookups, the wait for its first units
// and the merge of the one before (64 x 8192: 0 / 6 / 12 / 16 / 24 / 36 units 34.4 / 33.4 / 32.1 / 32.0 / 32.8 / 33.8 us).
constexpr int kDecStart = 12;

// What a CTA works on: units [u0, u0 + m) of the n that columns [c0, c0 + ncols) of kv head kvh of a
// sequence can see.
struct DecSegment {
  int b, q0, kvh, c0, ncols, n, u0, m, line, at;
  Kv4Span span;
};

template <int D, int NT, int W>
struct DecShape {
  static constexpr int kCols = 8 * NT;
  static constexpr int kRing = W * kDecStages * Kv4Unit<D>::kBytes;
  static constexpr int kOLd = D + 4;  // floats of one column's partial result
  static constexpr int kMerge = W * kCols * kOLd * 4;
  static constexpr int kBody = kRing > kMerge ? kRing : kMerge;
  static constexpr int kMl = W * kCols * 8;  // (reference maximum, sum)
  static constexpr int kQWords = 4 * Kv4Unit<D>::kG + 3;  // a lane's fragments, sums, factors of 8 columns
  static constexpr int kQ = NT * kQWords * 32 * 4;
  static constexpr size_t kSmem = kBody + kMl + kQ + 8 * W * kDecStages + sizeof(DecSegment) + 4 * (kDecMaxSeqs + 1) + 12;
};

// d += a b, and d = a b (no accumulator to clear).
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_1688_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.0f));
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

// (A call of its own: inlined, this code that hardly ever runs cost 0.1 us of an 8 us launch.)
__device__ __noinline__ void dec_zero_rows(const Kv4AttnParams& P, int d, int r0, int r1, int i, int n) {
  kv4_zero_rows(P, d, r0, r1, i, n);
}

// Units of all segments of sequence b: at least one per segment with a row, so that rows which see
// no key are written too.  In a launch that cuts no segment (P.whole) a segment counts as one.  A sequence that breaks
// the call's bounds has none: its rows are zeroed here, by one CTA.
__device__ __forceinline__ int tile_units(const Kv4AttnParams& P, int len, int nq, int c0, int cols) {
  const int c1 = min(c0 + cols, nq * P.group) - 1;
  return max(1, kv4_span(len, nq, c0 / P.group, c1 / P.group, P.window, P.sinks).count);
}
template <int D>
__device__ __forceinline__ int sequence_units(const Kv4AttnParams& P, int b, int cols, int* edge) {
  const int q0 = P.c.cu[b], q1 = P.c.cu[b + 1], nq = q1 - q0, len = P.c.lengths[b];
  if (b == 0) edge[0] = P.edges & 1 ? q0 : 0;  // rows of no sequence: [0, edge[0]) and [edge[1], tokens)
  if (b == P.c.seqs - 1) edge[1] = P.edges & 2 ? q1 : P.c.tokens;
  if (nq <= 0 || q0 < 0 || nq > P.max_new || len > P.max_len || q0 + nq > P.c.tokens) {
    if (nq != 0 && blockIdx.x == 0) {
      record_data_error(kErrKv4Bound);
      dec_zero_rows(P, D, q0, q1, 0, 1);
    }
    return 0;
  }
  int n = 0;
  for (int c0 = 0; c0 < nq * P.group; c0 += cols) n += P.whole ? 1 : kDecStart + tile_units(P, len, nq, c0, cols);
  return n * P.c.kv_heads;
}

template <int D, int NT, int W>
__global__ void __launch_bounds__(32 * W, dec_resident(W, 8 * NT))
    kv4_decode_kernel(const __grid_constant__ Kv4AttnParams P) {
  using U = Kv4Unit<D>;
  using Sh = DecShape<D, NT, W>;
  constexpr int G = U::kG;
  constexpr int kCols = Sh::kCols;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* body = smem;
  float2* s_ml = reinterpret_cast<float2*>(smem + Sh::kBody);
  uint32_t* s_q = reinterpret_cast<uint32_t*>(smem + Sh::kBody + Sh::kMl);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Sh::kBody + Sh::kMl + Sh::kQ);
  DecSegment& sg = *reinterpret_cast<DecSegment*>(bars + W * kDecStages);
  int* s_before = reinterpret_cast<int*>(&sg + 1);  // [seqs + 1] units before a sequence
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;

  if (threadIdx.x < W * kDecStages) mbar_init(&bars[threadIdx.x], 1);
  if (threadIdx.x == 0) fence_mbar_init();
  griddep_wait();
  griddep_launch();
  // ---- prefix sums of the sequences' units ----
  {
    int *s_warp = reinterpret_cast<int*>(s_ml), *s_edge = s_warp + W;
    int before = 0;
    for (int b0 = 0; b0 < P.c.seqs; b0 += 32 * W) {
      const int b = b0 + threadIdx.x;
      const int n = b < P.c.seqs ? sequence_units<D>(P, b, kCols, s_edge) : 0;
      int inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
      }
      if (lane == 31) s_warp[warp] = inc;
      __syncthreads();
      int mine = before + inc - n;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (w < warp) mine += s_warp[w];
        before += s_warp[w];
      }
      if (b < P.c.seqs) s_before[b] = mine;
      if (threadIdx.x == 0) s_before[P.c.seqs] = before;  // the last round's is the whole
      __syncthreads();
    }
#pragma unroll 1
    for (int r0 = 0, r1 = s_edge[0];; r0 = s_edge[1], r1 = P.c.tokens) {
      if (r0 < r1) dec_zero_rows(P, D, r0, r1, blockIdx.x * 32 * W + threadIdx.x, gridDim.x * 32 * W);
      if (r1 == P.c.tokens) break;
    }
  }
  const int total = s_before[P.c.seqs];
  const int quota = max(P.whole ? 1 : W, (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
  const int cta = blockIdx.x;
  const int begin = min(total, cta * quota), end = min(total, begin + quota);
  const uint64_t policy = l2_policy_evict_first();
  uint8_t* ring = body + warp * kDecStages * U::kBytes;
  uint64_t* bar = bars + warp * kDecStages;
  bool began = false;  // thread 0: a segment begins here and goes on
  int turn = 0;  // units this warp has fetched into its ring and consumed, over all segments
  bool ok = true;  // no wait of this warp has run out: else its ring is not used again and what it has a part in is NaN

  for (int at = begin; at < end;) {
    // ---- the segment that unit `at` of the line belongs to ----
    if (warp == 0) {
      int lo = 0, hi = P.c.seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_before[mid] <= at) lo = mid; else hi = mid;
      }
      const int b = lo;  // the last sequence that begins at or before `at`: it has units
      const int q0 = P.c.cu[b], nq = P.c.cu[b + 1] - q0, len = P.c.lengths[b];
      int rest = at - s_before[b], c0 = 0, n = 0, line = 0;
      for (;; c0 += kCols) {  // tiles of columns, each with all kv heads
        n = tile_units(P, len, nq, c0, kCols);
        line = P.whole ? 1 : kDecStart + n;
        if (rest < line * P.c.kv_heads) break;
        rest -= line * P.c.kv_heads;
      }
      const int kvh = rest / line, off = rest - kvh * line;  // units of the segment stand from kDecStart on
      const int here = min(line - off, end - at);
      const int u0 = P.whole ? 0 : max(0, off - kDecStart), m = P.whole ? n : max(0, off + here - kDecStart) - u0;
      if (lane == 0) {
        sg.b = b, sg.q0 = q0, sg.kvh = kvh, sg.c0 = c0, sg.ncols = min(kCols, nq * P.group - c0);
        sg.n = n, sg.u0 = u0, sg.m = m, sg.line = at - off + kDecStart, sg.at = at + here;
        sg.span = kv4_span(len, nq, c0 / P.group, (c0 + sg.ncols - 1) / P.group, P.window, P.sinks);
      }
    }
    __syncthreads();
    const int b = sg.b, q0 = sg.q0, kvh = sg.kvh, c0 = sg.c0, ncols = sg.ncols, n = sg.n, u0 = sg.u0, m = sg.m;
    const Kv4Span span = sg.span;
    at = sg.at;
    if (m == 0) {  // the CTA's share ends before the segment's first unit
      __syncthreads();
      continue;
    }

    // lane i holds the i-th of this warp's next 32 units: its index in the pool, and in a ballot
    // whether every column sees every token of it
    const int mine = ok ? (m - warp + W - 1) / W : 0;
    int index = -1;
    unsigned clear = 0u;
    auto look = [&](int round) {
      const int i = 32 * round + lane;
      index = -1;
      bool all = false;
      if (i < mine) {
        const int u = span.unit(u0 + warp + W * i), key0 = kKv4Unit * u, key1 = key0 + kKv4Unit - 1;
        if (span.count > 0) {
          index = kv4_unit_index(P.c, b, kvh, u);
          if (index < 0) record_data_error(kErrKv4Table);
        }
        all = index >= 0 && key1 <= span.pos_lo && (P.window <= 0 || span.pos_hi - key0 < P.window || key1 < P.sinks);
      }
      clear = __ballot_sync(0xffffffffu, all);
    };
    auto fetch = [&](int i, int slot) {  // every lane calls it; a unit without a page is not fetched
      const int x = __shfl_sync(0xffffffffu, index, i & 31);
      if (lane == 0) {
        if (x >= 0) {
          mbar_arrive_expect_tx(&bar[slot], U::kBytes);
          bulk_load(ring + slot * U::kBytes, P.c.data + static_cast<long long>(x) * U::kBytes, U::kBytes, &bar[slot], policy);
        } else {
          mbar_arrive(&bar[slot]);
        }
      }
    };
    look(0);
    for (int i = 0; i < kDecStages && i < mine; ++i) fetch(i, (turn + i) % kDecStages);

    // ---- q: B fragments of column 8 nt + g, channels 32 j + 8 t + 0..7, made by warp nt ----
    if (warp < NT) {
      const int nt = warp, col = 8 * nt + g;
      const int row = c0 + col, tok = row / P.group;
      uint32_t* dst = s_q + nt * Sh::kQWords * 32 + lane;
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
        dst[(4 * j + 0) * 32] = h2_bits(__floats2half2_rn(v[j][0], v[j][4]));
        dst[(4 * j + 1) * 32] = h2_bits(__floats2half2_rn(v[j][1] * 0.0625f, v[j][5] * 0.0625f));
        dst[(4 * j + 2) * 32] = h2_bits(__floats2half2_rn(v[j][2], v[j][6]));
        dst[(4 * j + 3) * 32] = h2_bits(__floats2half2_rn(v[j][3] * 0.0625f, v[j][7] * 0.0625f));
      }
      // sums of q for the lows: lanes t = 0, 1 hold the fp16 high halves of groups 0, 1 | 2, 3, lanes
      // t = 2, 3 what those leave
      float sa = part[0], sb = part[1];
      if constexpr (G == 4) {
        if (t & 1) sa = part[2], sb = part[3];
      } else {
        if (t & 1) sa = sb = 0.0f;
      }
      const __half2 hi2 = __floats2half2_rn(sa, sb);
      const float2 hf = __half22float2(hi2);
      dst[4 * G * 32] = h2_bits(t < 2 ? hi2 : __floats2half2_rn(sa - hf.x, sb - hf.y));
      const float cf = P.scale_log2 * down;  // log2 score per unit of the products, of columns 2t, 2t + 1
      dst[(4 * G + 1) * 32] = __float_as_uint(__shfl_sync(0xffffffffu, cf, 8 * t));
      dst[(4 * G + 2) * 32] = __float_as_uint(__shfl_sync(0xffffffffu, cf, 8 * t + 4));
    }
    __syncthreads();
    uint32_t qf[NT][G][4], qsum[NT];
    float colfac[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t* src = s_q + nt * Sh::kQWords * 32 + lane;
#pragma unroll
      for (int j = 0; j < G; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[nt][j][i] = src[(4 * j + i) * 32];
      qsum[nt] = src[4 * G * 32];
      colfac[nt][0] = __uint_as_float(src[(4 * G + 1) * 32]);
      colfac[nt][1] = __uint_as_float(src[(4 * G + 2) * 32]);
    }

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

    // V's scales go in times 2^vexp, which keeps them at 1 or below; a larger one moves it (and O) down, to leave
    // that one between 1/4 and 1/2.
    int vexp = 15;
    __half2 vmul = bits_h2(0x78007800u), vmax = bits_h2(0x02000200u);  // 2^vexp, 2^-vexp

    // One unit; kPlain: every column sees every token of it.  The two forms are separate code, so that
    // the plain one carries no masking.
    auto attend = [&](const uint8_t* un, int i, auto flag) {
      constexpr bool kPlain = decltype(flag)::value;
      // V's scales of the unit: a lane looks at G / 2 words of tokens 2 (lane / 2), + 1
      __half2 top;
      {
        const uint8_t* at = un + U::kVScale + lane * 2 * G;
        if constexpr (G == 4) {
          const uint2 x = *reinterpret_cast<const uint2*>(at);
          top = __hmax2(bits_h2(x.x), bits_h2(x.y));
        } else {
          top = bits_h2(*reinterpret_cast<const uint32_t*>(at));
        }
      }
      // ---- products of 32 tokens (two tiles of 16), before the column's factor ----
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
        float sum[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[nt][e] = 0.0f;
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const uint32_t wa = ka[j], wb = kb[j], va = wa >> 8, vb = wb >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float d[4];
            mma_16816_first(d, wa & 0x000f000fu, wb & 0x000f000fu, wa & 0x00f000f0u, wb & 0x00f000f0u, qf[nt][j][0], qf[nt][j][1]);
            mma_16816(d, va & 0x000f000fu, vb & 0x000f000fu, va & 0x00f000f0u, vb & 0x00f000f0u, qf[nt][j][2], qf[nt][j][3]);
            sum[nt][0] = fmaf(sa[j], d[0], sum[nt][0]);
            sum[nt][1] = fmaf(sa[j], d[1], sum[nt][1]);
            sum[nt][2] = fmaf(sb[j], d[2], sum[nt][2]);
            sum[nt][3] = fmaf(sb[j], d[3], sum[nt][3]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float sm[4];
          mma_1688_first(sm, la, lb, qsum[nt]);
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[blk][nt][e] = fmaf(16777216.0f, sum[nt][e], sm[e]);
        }
      }
      if constexpr (!kPlain) {
        const int key0 = kKv4Unit * span.unit(u0 + warp + W * i);
        const bool have = __shfl_sync(0xffffffffu, index, i & 31) >= 0;
        uint32_t some = 0u;  // the scale of a token that no column sees may be anything
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = key0 + (lane & ~1) + e;
          if (have && key <= span.pos_hi && (P.window <= 0 || span.pos_lo - key < P.window || key < P.sinks)) some |= 0xffffu << (16 * e);
        }
        top = bits_h2(h2_bits(top) & some);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // position of column 2t + e (columns past the rows repeat the last one)
            const int ps = span.pos_lo + min(c0 + 8 * nt + 2 * t + e, c0 + ncols - 1) / P.group - c0 / P.group;
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int key = key0 + 16 * blk + 8 * h + g;
                const bool seen = have && key <= ps && (P.window <= 0 || ps - key < P.window || key < P.sinks);
                if (!seen) sc[blk][nt][2 * h + e] = -INFINITY;
              }
          }
      }
      // ---- running maximum, and the power of two of V's scales ----
      const bool large = __hgt2_mask(top, vmax) != 0u;
      if (__any_sync(0xffffffffu, large)) {
        const uint32_t t2 = h2_bits(__hmax2(top, bits_h2(0u)));  // halves of at least 0, in the order of their bits
        const uint32_t most = __reduce_max_sync(0xffffffffu, max(t2 & 0xffffu, t2 >> 16));
        const int to = min(vexp, max(-14, 13 - static_cast<int>(most >> 10)));
        const float back = __uint_as_float(static_cast<uint32_t>(127 + to - vexp) << 23);
        vexp = to;
        vmul = bits_h2(static_cast<uint32_t>(15 + to) * 0x04000400u);
        vmax = bits_h2(static_cast<uint32_t>(15 - to) * 0x04000400u);
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
          for (int j = 0; j < G; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[c][j][s][e] *= back;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mx[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          mx[e] = fmaxf(fmaxf(sc[0][nt][e], sc[0][nt][e + 2]), fmaxf(sc[1][nt][e], sc[1][nt][e + 2])) * colfac[nt][e];
        if (__any_sync(0xffffffffu, mx[0] > m_ref[nt][0] + kDecMove || mx[1] > m_ref[nt][1] + kDecMove)) {
          float al[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], o));
            const float mm = fmaxf(m_ref[nt][e], mx[e] - kDecSet);
            al[e] = m_ref[nt][e] == -INFINITY ? 0.0f : ex2_approx(m_ref[nt][e] - mm);
            m_ref[nt][e] = mm;
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
      float neg[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) neg[nt][e] = m_ref[nt][e] == -INFINITY ? 0.0f : -m_ref[nt][e];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        uint32_t pb[NT][2];  // B fragments of p: tokens 2t, 2t + 1 of each half, column g
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            pb[nt][h] = transpose_8x8(h2_bits(__floats2half2_rn(ex2_approx(fmaf(sc[blk][nt][2 * h], colfac[nt][0], neg[nt][0])),
                                                                ex2_approx(fmaf(sc[blk][nt][2 * h + 1], colfac[nt][1], neg[nt][1])))));
        uint32_t v0[G], v1[G], s0[G], s1[G];
        lds_words<G>(un + U::kV + blk * 8 * D + lane * 4 * G, v0);
        lds_words<G>(un + U::kV + blk * 8 * D + 4 * D + lane * 4 * G, v1);
        lds_words<G>(un + U::kVScale + blk * 32 * G + t * 4 * G, s0);
        lds_words<G>(un + U::kVScale + blk * 32 * G + 16 * G + t * 4 * G, s1);
        uint32_t l0 = g == 4 ? 0x3c003c00u : 0u, l1 = l0;  // rows 0..G-1: lows of a group; row 4: ones
        if (g < G) {
          l0 = *reinterpret_cast<const uint32_t*>(un + U::kVLow + blk * 32 * G + t * 4 * G + 4 * g);
          l1 = *reinterpret_cast<const uint32_t*>(un + U::kVLow + blk * 32 * G + 16 * G + t * 4 * G + 4 * g);
          if constexpr (!kPlain) {  // a NaN low comes with a NaN scale, which reaches the columns that see the token
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
          const __half2 t0 = __hmul2(bits_h2(s0[j]), vmul), t1 = __hmul2(bits_h2(s1[j]), vmul);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint32_t b0 = h2_bits(__hmul2(bits_h2(pb[nt][0]), t0));
            uint32_t b1 = h2_bits(__hmul2(bits_h2(pb[nt][1]), t1));
            if constexpr (!kPlain) {  // p = 0 stays 0 beside whatever stands in a hidden token's scale
              b0 &= __hneu2_mask(bits_h2(pb[nt][0]), bits_h2(0u));
              b1 &= __hneu2_mask(bits_h2(pb[nt][1]), bits_h2(0u));
            }
            mma_16816(acc[nt][j][0], x0 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x000f000fu, x1 & 0x00f000f0u, b0, b1);
            mma_16816(acc[nt][j][1], y0 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x000f000fu, y1 & 0x00f000f0u, b0, b1);
          }
        }
      }
    };
    for (int i = 0; i < mine; ++i, ++turn) {
      const int st = turn % kDecStages;
      ok = mbar_wait(&bar[st], static_cast<uint32_t>(turn / kDecStages) & 1u, kErrKv4Timeout);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if ((clear >> (i & 31)) & 1u)
        attend(ring + st * U::kBytes, i, std::true_type{});
      else
        attend(ring + st * U::kBytes, i, std::false_type{});
      __syncwarp();  // every lane has read the unit
      if ((i & 31) == 31) {  // the next 32 places; those of the ring's units ahead are in the same round
        look((i + 1) >> 5);
        for (int k = 1; k <= kDecStages && i + k < mine; ++k) fetch(i + k, (turn + k) % kDecStages);
      } else if (i + kDecStages < mine && ((i + kDecStages) >> 5) == (i >> 5)) {
        fetch(i + kDecStages, st);
      }
    }
    if (!ok) {
      settle_issued_copies();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) low[nt][e] = NAN;
    }

    // ---- the warps' results meet in shared memory ----
    __syncthreads();  // every ring is idle
    float* so = reinterpret_cast<float*>(body);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + 24 - vexp) << 23), up16 = up * 0.0625f;  // 2^24 2^-vexp
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
          o.x = fmaf(up, acc[nt][j][0][e], lw);
          o.y = fmaf(up16, acc[nt][j][0][e + 2], lw);
          o.z = fmaf(up, acc[nt][j][1][e], lw);
          o.w = fmaf(up16, acc[nt][j][1][e + 2], lw);
          *reinterpret_cast<float4*>(dst + 32 * j) = o;
        }
      }
    }
    __syncthreads();
    const bool whole = m == n;
    if (u0 == 0 && threadIdx.x == 0 && (P.by_segment || !whole)) {  // for the join: who has a part of what begins here
      const int parts = (sg.line + n - 1) / quota - cta + 1;
      P.part_head[P.by_segment ? (b * P.tiles + c0 / kCols) * P.c.kv_heads + kvh : cta] =
          make_int4(q0, c0 | (ncols << 24), kvh, parts | cta << 16);
      began = !whole;
    }
    const long long slot = 2LL * cta + (u0 == 0 ? 1 : 0);  // 0: began in an earlier CTA; 1: goes on in the next
    for (int i = threadIdx.x; i < ncols * (D / 4); i += 32 * W) {
      const int col = i / (D / 4), ch = i % (D / 4) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) mm = fmaxf(mm, s_ml[w * kCols + col].x);
      const float m_use = mm == -INFINITY ? 0.0f : mm;
      float l = 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 ml = s_ml[w * kCols + col];
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // saw no visible token
        const float f = ex2_approx(ml.x - m_use);
        const float4 x = *reinterpret_cast<const float4*>(so + (w * kCols + col) * Sh::kOLd + ch);
        l = fmaf(f, ml.y, l);
        o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y), o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
      }
      if (whole) {
        const int row = c0 + col, tok = row / P.group;
        const long long orow = static_cast<long long>(q0 + tok) * P.q_heads + kvh * P.group + row - tok * P.group;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no visible token: zeros
        uint2 u;
        u.x = pack_bf16x2(o.x * inv, o.y * inv);
        u.y = pack_bf16x2(o.z * inv, o.w * inv);
        *reinterpret_cast<uint2*>(P.out + orow * D + ch) = u;
      } else {
        *reinterpret_cast<float4*>(P.part_o + (slot * kCols + col) * D + ch) = o;
        if (ch == 0) P.part_ml[slot * kCols + col] = make_float2(mm, l);
      }
    }
    if (at < end) {
      fence_proxy_async_smem();  // the rings are written by bulk copies again
      __syncthreads();
    }
  }
  if (threadIdx.x == 0 && !P.whole && !P.by_segment && !began) P.part_head[cta] = make_int4(0, 0, 0, 1);
}

// What a part with reference maximum x.x and sum x.y counts against the maximum m: nothing if it saw no token.
__device__ __forceinline__ float part_factor(float2 x, float m) {
  return x.x == -INFINITY && x.y == 0.0f ? 0.0f : ex2_approx(x.x - (m == -INFINITY ? 0.0f : m));
}

// out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s over parts from, from + step, ..., eight at a time so
// that their loads overlap: a warp's running maximum, sum and D / 32 channels a lane.  Part i stands in row
// row(i) of part_o and part_ml.  A part that saw no token may hold anything in part_o.
template <int D, typename Row>
__device__ __forceinline__ void join_parts(const Kv4AttnParams& P, Row row, int from, int step, int parts, float& m, float& l,
                                           float (&o)[D / 32]) {
  constexpr int kVec = D / 32, kBatch = 8;
  const int lane = threadIdx.x & 31;
  m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < kVec; ++e) o[e] = 0.0f;
  for (int i0 = from; i0 < parts; i0 += kBatch * step) {
    float2 x[kBatch];
    float v[kBatch][kVec];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u * step;
      x[u] = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[u][e] = 0.0f;
      if (i < parts) {
        x[u] = P.part_ml[row(i)];
        const float* src = P.part_o + row(i) * D + lane * kVec;
        if constexpr (kVec == 4) {
          const float4 y = *reinterpret_cast<const float4*>(src);
          v[u][0] = y.x, v[u][1] = y.y, v[u][2] = y.z, v[u][3] = y.w;
        } else {
          const float2 y = *reinterpret_cast<const float2*>(src);
          v[u][0] = y.x, v[u][1] = y.y;
        }
      }
    }
    float mb = m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) mb = fmaxf(mb, x[u].x);
    const float back = part_factor(make_float2(m, l), mb);
    l *= back;
#pragma unroll
    for (int e = 0; e < kVec; ++e) o[e] *= back;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (x[u].x == -INFINITY && x[u].y == 0.0f) continue;
      const float f = part_factor(x[u], mb);
      l = fmaf(f, x[u].y, l);
#pragma unroll
      for (int e = 0; e < kVec; ++e) o[e] = fmaf(f, v[u][e], o[e]);
    }
    m = mb;
  }
}
// Joins the segments that were cut between CTAs.  Few segments with many parts
// (P.by_segment): CTA (i, y) takes column y of segment i, its 16 warps every 16th part.  Otherwise CTA i
// takes the segment that begins in CTA i of the decode kernel and goes on, a warp per column.
template <int D>
__global__ void __launch_bounds__(512) kv4_combine_kernel(const __grid_constant__ Kv4AttnParams P, int cols) {
  constexpr int kVec = D / 32;  // channels of a lane
  __shared__ float s_o[16][D], s_l[16], s_m[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch();
  if (P.by_segment) {  // a segment without rows has no entry
    const int rest = blockIdx.x / P.c.kv_heads, b = rest / P.tiles, c0 = (rest - b * P.tiles) * cols;
    const int q0 = P.c.cu[b], nq = P.c.cu[b + 1] - q0;
    if (nq <= 0 || q0 < 0 || nq > P.max_new || P.c.lengths[b] > P.max_len || q0 + nq > P.c.tokens || c0 >= nq * P.group) return;
  }
  const int4 head = P.part_head[blockIdx.x];
  const int parts = head.w & 0xffff, cta = head.w >> 16, c0 = head.y & 0xffffff, ncols = head.y >> 24;
  if (parts <= 1) return;  // written by its CTA
  const int split = P.by_segment ? 16 : 1;
  const int col = P.by_segment ? blockIdx.y : warp, from = P.by_segment ? warp : 0;
  if (col >= ncols) return;
  // the first CTA kept its part as one that goes on, the others as one that began earlier
  auto slot = [&](int i) { return (2LL * (cta + i) + (i == 0 ? 1 : 0)) * cols + col; };
  float m, l, o[kVec];
  join_parts<D>(P, slot, from, split, parts, m, l, o);
  if (P.by_segment) {  // the warps' sums meet
#pragma unroll
    for (int e = 0; e < kVec; ++e) s_o[warp][lane * kVec + e] = o[e];
    if (lane == 0) s_l[warp] = l, s_m[warp] = m;
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 0; w < 16; ++w) m = fmaxf(m, s_m[w]);
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < kVec; ++e) o[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      const float f = part_factor(make_float2(s_m[w], s_l[w]), m);
      l = fmaf(f, s_l[w], l);
#pragma unroll
      for (int e = 0; e < kVec; ++e) o[e] = fmaf(f, s_o[w][lane * kVec + e], o[e]);
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no visible token: zeros
  const int row = c0 + col, tok = row / P.group;
  const long long orow = static_cast<long long>(head.x + tok) * P.q_heads + head.z * P.group + row - tok * P.group;
  __nv_bfloat16* dst = P.out + orow * D + lane * kVec;
  if constexpr (kVec == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(o[0] * inv, o[1] * inv);
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

template <int D, int NT, int W>
cudaError_t launch_decode(const Kv4AttnParams& whole, int ctas, int batch, cudaStream_t stream) {
  for (int b0 = 0; b0 < whole.c.seqs; b0 += batch) {
    Kv4AttnParams p = whole;
    p.c.seqs = std::min(batch, whole.c.seqs - b0);
    p.c.cu += b0;
    p.c.lengths += b0;
    p.c.table += static_cast<long long>(b0) * p.c.table_ld;
    p.edges = (b0 == 0 ? 1 : 0) | (b0 + p.c.seqs >= whole.c.seqs ? 2 : 0);
    p.tiles = (p.max_new * p.group + 8 * NT - 1) / (8 * NT);
    // A few segments are cut into many parts each: then a CTA of the join per segment and column, instead of one per
    // CTA of this launch with a warp per column (us, 592 CTAs, 400000 tokens in 2 / 8 / 16 / 24 / 32 / 48 / 74 segments
    // of d = 128: 32 / 30 / 30 / 33.0 / 33.6 / 36 / 38 against 67 / 40 / 35 / 33.8 / 33.2 / 33 / 32; 60000 tokens in 2 / 16 / 24 /
    // 32: 14.5 / 13.1 / 15.3 / 15.9 against 47 / 17 / 15.6 / 14.8).  A launch that cuts nothing has no join and no
    // workspace for its segments' heads, however few sequences the last one holds.
    p.by_segment = !p.whole && 16LL * p.tiles * p.c.kv_heads * p.c.seqs < ctas;
    cudaError_t e = launch_pdl(kv4_decode_kernel<D, NT, W>, dim3(ctas, 1, 1), 32 * W, DecShape<D, NT, W>::kSmem, stream, p);
    if (e != cudaSuccess) return e;
    if (p.whole) continue;
    e = p.by_segment ? launch_pdl(kv4_combine_kernel<D>, dim3(p.tiles * p.c.kv_heads * p.c.seqs, 8 * NT, 1), 512, 0, stream, p, 8 * NT)
                     : launch_pdl(kv4_combine_kernel<D>, dim3(ctas, 1, 1), 256 * NT, 0, stream, p, 8 * NT);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <int D, int NT>
cudaError_t decode_smem() {
  cudaError_t e = cudaFuncSetAttribute(kv4_decode_kernel<D, NT, kDecWarps>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(DecShape<D, NT, kDecWarps>::kSmem));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kv4_decode_kernel<D, NT, kDecWarpsWide>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(DecShape<D, NT, kDecWarpsWide>::kSmem));
  return e;
}
template <int D, int NT>
cudaError_t launch_decode(const Kv4AttnParams& p, int warps, int ctas, int batch, cudaStream_t stream) {
  return warps == kDecWarps ? launch_decode<D, NT, kDecWarps>(p, ctas, batch, stream)
                            : launch_decode<D, NT, kDecWarpsWide>(p, ctas, batch, stream);
}
}  // namespace

cudaError_t launch_kv4_decode(const Kv4AttnParams& p, int head_dim, int cols, int warps, int ctas, int batch, cudaStream_t stream) {
  if (head_dim == 128)
    return cols == 8 ? launch_decode<128, 1>(p, warps, ctas, batch, stream) : launch_decode<128, 2>(p, warps, ctas, batch, stream);
  return cols == 8 ? launch_decode<64, 1>(p, warps, ctas, batch, stream) : launch_decode<64, 2>(p, warps, ctas, batch, stream);
}

cudaError_t kv4_prepare_device() {
  cudaError_t e = decode_smem<128, 1>();
  if (e == cudaSuccess) e = decode_smem<128, 2>();
  if (e == cudaSuccess) e = decode_smem<64, 1>();
  if (e == cudaSuccess) e = decode_smem<64, 2>();
  if (e == cudaSuccess) e = kv4_chunk_prepare_device();
  return e;
}

namespace {
struct DecodePlan {
  int cols, ctas, whole;  // cols 0: kv4_chunk_kernel, its keys shared by `split` CTAs
  int split, warps;
  int batch;  // sequences of a launch, 0: one alone has too many units
  uint64_t part_rows, bytes;  // workspace of unfinished segments
};

// Columns per CTA, and one wave of resident CTAs (16 warps per SM with 8 columns, 8 with 16), or fewer when not
// every warp could have a unit.  A short segment is left whole, which spares the join (4 us with its launch):
//   - up to kDecWholeUnits units where segments are many;
//   - where a wave holds one each, with eight warps to a CTA, as long as a CTA's own time (4.5 us + 0.125 a unit, 0.09
//     with d = 64) stays below that of the cut (9 us + 0.00073 a unit and segment), or kDecWholeUnitsShared where
//     two CTAs share an SM.  us whole / cut, d = 128: 2 segments of 23 units 7.5 / 8.3, of 48 10.7 / 9.1, of 64 12.7 /
//     9.6; 128 of 64 14.3 / 17.9, of 134 24.0 / 25.2, of 256 40.2 / 36.9; 192 with d = 64, of 64 14.1 / 15.9, of 92 18.0 /
//     18.2, of 128 22.9 / 21.9.  Four warps a CTA instead of eight: 2 of 23 8.7, of 48 13.3.
constexpr int kDecWholeUnits = 48, kDecWholeUnitsShared = 110;
bool dec_whole(long long segments, long long units, bool wide, int head_dim) {
  if (!wide) return units <= kDecWholeUnits;
  if (segments > sm_count()) return units <= kDecWholeUnitsShared;
  return units <= (head_dim == 64 ? 50 : 36) + segments * (units + kDecStart) / 170;
}
// Which kernel, and how many CTAs share the keys of a tile of rows.  In steps of a 16-column tile over one
// unit (1.2 ns of the whole GPU with d = 128, 0.9 with 64) this file's kernel takes about kDecBase + tiles
// (units + kDecStart), spread evenly whatever the shape; kv4_chunk_kernel takes kChunkUnit (units + 10) for
// each wave of its CTAs of 256 rows (kChunkUnit2 with more than 128 rows: two query tiles), however few of a
// wave there are, and with keys shared out kChunkJoin + kChunkJoinTile for each 128 rows of a part.  d = 128, 8
// kv heads, us here / there with one CTA a tile / with as many as the rule takes: 1 x 8192 tokens, 96 rows 26
// / 147 / 22, 256 rows 53 / 180 / 29; 8 x 8192, 64 rows 89 / 150 / -, 128 rows 167 / 151 / 92, 256 rows 326 / 185 /
// 113; 8 x 512, 256 rows 48 / 22 / -, 28 if two shared; 32 x 2048, 32 rows 57 / 87 / -, 64 rows 103 / 88 / -, 256
// rows 387 / 114 / -.  Up to kDecMaxRows rows it was faster here at every shape.
constexpr int kDecMaxRows = 32;
constexpr long long kDecBase = 5000, kChunkUnit = 500, kChunkUnit2 = 640, kChunkJoin = 2000, kChunkJoinTile = 20;
constexpr int kChunkShare = 8;  // units of a part at least
DecodePlan decode_plan(const rldx_kv4_cache& c, int q_heads, int max_new, int max_len, int window, int sinks) {
  DecodePlan p;
  const long long rows = static_cast<long long>(max_new) * (q_heads / c.kv_heads);
  p = {};
  p.cols = rows <= 8 ? 8 : 16;
  const long long tiles = (rows + p.cols - 1) / p.cols;
  long long keys = max_len;
  if (window > 0) keys = std::min<long long>(keys, static_cast<long long>(window) + max_new + std::min(sinks, max_len) + 3 * kKv4Unit);
  const long long units = (keys + kKv4Unit - 1) / kKv4Unit;
  const long long line = tiles * c.kv_heads * ((static_cast<long long>(max_len) + kKv4Unit - 1) / kKv4Unit + kDecStart);
  p.batch = static_cast<int>(std::min<long long>(kDecMaxSeqs, kDecMaxLine / line));
  const long long segments = tiles * c.kv_heads * std::min(c.seqs, p.batch);
  if (rows > kDecMaxRows) {
    const long long heads = static_cast<long long>(c.kv_heads) * c.seqs, ctas = (rows + 255) / 256 * heads;
    long long least = p.batch > 0 ? kDecBase + tiles * heads * (units + kDecStart) : INT64_MAX;
    for (int split = 1; split == 1 || (split * ctas <= 2 * sm_count() && units >= split * kChunkShare); ++split) {
      const long long waves = (split * ctas + sm_count() - 1) / sm_count();
      const long long cost = waves * (rows > 128 ? kChunkUnit2 : kChunkUnit) * ((units + split - 1) / split + 10) +
                             (split > 1 ? kChunkJoin + kChunkJoinTile * split * ctas * (rows > 128 ? 2 : 1) : 0);
      if (cost < least) least = cost, p.cols = 0, p.split = split;
    }
    if (p.cols == 0) {
      p.part_rows = p.split > 1 ? 256ull * ctas * p.split : 0;
      p.bytes = p.part_rows * (static_cast<uint64_t>(c.head_dim) * 4 + 8);
      return p;
    }
  }
  const bool wide = segments <= dec_resident(kDecWarpsWide, p.cols) * sm_count();
  p.whole = dec_whole(segments, units, wide, c.head_dim);
  p.warps = p.whole && wide ? kDecWarpsWide : kDecWarps;
  const int wave = dec_resident(p.warps, p.cols) * sm_count();
  p.ctas = static_cast<int>(std::min<long long>(wave, p.whole ? segments : (units * segments + kDecWarps - 1) / kDecWarps));
  p.part_rows = p.whole ? 0 : 2ull * p.ctas * p.cols;
  p.bytes = p.part_rows * (static_cast<uint64_t>(c.head_dim) * 4 + 8) + (p.part_rows ? 16ull * p.ctas : 0);
  return p;
}

int plan_of(const rldx_kv4_cache& c, const rldx_kv4_attention_desc& a, const Kv4AttnParams& p, DecodePlan* plan) {
  *plan = decode_plan(c, a.q_heads, a.max_new, p.max_len, p.window, p.sinks);
  if (plan->cols > 0 && plan->batch == 0)
    return set_error(RLDX_ERR_UNSUPPORTED, "kv4_attention: max_len and the heads allow for more than 2^30 units of 32 tokens in a sequence");
  return RLDX_OK;
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
  p->max_len = static_cast<int>(std::min<long long>(a->max_len, static_cast<long long>(cache->table_width) * cache->page_size));
  // a window that no sequence is longer than hides nothing (and its differences of positions would not fit 32 bits)
  p->window = a->window < p->max_len ? a->window : 0;
  p->sinks = p->window > 0 ? a->sinks : 0;
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
  DecodePlan plan;
  rc = plan_of(*cache, *a, p, &plan);
  if (rc == RLDX_OK) *bytes = plan.bytes;
  return rc;
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
  DecodePlan plan;
  rc = plan_of(*cache, *a, p, &plan);
  if (rc != RLDX_OK) return rc;
  if (plan.bytes > workspace_bytes || (plan.bytes > 0 && (!workspace || !aligned_to(workspace, 16))))
    return set_error(RLDX_ERR_ARG, "kv4_attention: needs a 16-byte aligned workspace of " + std::to_string(plan.bytes) + " bytes");
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.ldq = a->ldq;
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.q_heads = a->q_heads;
  p.group = a->q_heads / cache->kv_heads;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.max_new = a->max_new;
  p.whole = plan.whole;
  p.split = plan.split;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + plan.part_rows * d);
  p.part_head = reinterpret_cast<int4*>(p.part_ml + plan.part_rows);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = plan.cols == 0 ? launch_kv4_chunk(p, d, st) : launch_kv4_decode(p, d, plan.cols, plan.warps, plan.ctas, plan.batch, st);
  if (e != cudaSuccess) return cuda_fail(e, "kv4_attention launch");
  return RLDX_OK;
}

}  // extern "C"
