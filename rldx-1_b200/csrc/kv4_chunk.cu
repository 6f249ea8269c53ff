// Attention of many new tokens per sequence over the paged 4-bit cache (layout: kv4.cuh), on
// tcgen05: one CTA takes 256 query rows (new token, head of the group) of one kv head, in two tiles
// of 128, and runs over the keys they can see in tiles of 64 (two units):
//   S = Q K^T (M = 128, N = 64, K = d), P = exp2(S - m), O += P V (M = 128, N = d, K = 64)
// with S, P and O in tensor memory and the codes rebuilt to fp16 on the way to shared memory:
// scale code + low in one fp16 fma, whose rounding (2^-11) is far inside the 4-bit step.  q goes to
// fp16 scaled by a power of two per row (largest in [2^14, 2^15)), p is at most 2^8 by the lazy
// reference maximum of joint_attention_kernel; sums and maxima are fp32.
//
// Warps: 0 fetches units by bulk copies, 1 issues the MMAs, 4-11 do the softmax (one row a thread),
// 12-13 rebuild K, 14-15 rebuild V^T; registers move from the first four to the softmax.  The order of channels inside 16 bytes of K (and q) is that of
// the nibbles under the masks (0 4 1 5 2 6 3 7), and tokens stand inside each group of eight in
// an order rotated by the group (chunk_token), so that neither side needs a shuffle and both the
// reads of the units and the writes of the swizzled tiles are free of bank conflicts.
//
// P_j takes the place of S_j in tensor memory, so S_{j+2} is issued once PV_j has finished; the
// other query tile's products keep the tensor cores busy meanwhile.
//
// A value of V that is not finite, of a token that some rows must not see, cannot go through a
// product with p = 0: it is rebuilt as 0, its place marked, and the rows that do see the token
// give NaN in the channels of its group (in every channel where K is not finite).
#include "host_util.h"
#include "kv4.cuh"

namespace rldx {

namespace {
constexpr unsigned int kErrKv4Chunk = 0x520;  // + role: a bounded wait ran out

template <int D>
struct ChunkShape {
  static constexpr int kG = D / 32;
  static constexpr int kKeys = 64;
  static constexpr int kQTile = 128 * D * 2;
  static constexpr int kQChunk = 128 * 128;
  static constexpr int kKTile = kKeys * D * 2;
  static constexpr int kKChunk = kKeys * 128;
  static constexpr int kVTile = D * 128;
  static constexpr int kRaw = 2 * Kv4Unit<D>::kBytes;
  static constexpr int kStages = 3;     // of K and of V^T
  static constexpr int kRawStages = 4;  // of unit pairs
  static constexpr int kThreads = 32 * 16;
  static constexpr uint32_t kOCol = 256;  // S / P: (2 g + buffer) 64 columns; O of tile g: 256 + g d
  static constexpr uint32_t kTmemCols = 512;
  static constexpr int kBars = 1 + 2 * kRawStages + 4 * kStages + 2 * 7 + 1;
  static constexpr int kBad = kStages * (kG + 2) * 8;  // marks of what is not finite, a bit per token: V's groups, K; any
  static constexpr size_t kSmem = 1024 + 2 * kQTile + kStages * (kKTile + kVTile) + kRawStages * kRaw + kBad + 8 * kBars + 16;
};

__host__ __device__ constexpr uint32_t umma_idesc_f16(int M, int N) {  // fp16 operands, fp32 accumulator, both K-major
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// Token (of the tile's 64) that stands at key position c.
__host__ __device__ constexpr int chunk_token(int c) { return (c & ~7) + 2 * (((c >> 1) + (c >> 3)) & 3) + (c & 1); }
// Its inverse inside a group of eight: pair (token / 2 % 4) of group o stands at pair position.
__device__ __forceinline__ int chunk_row(int token) {
  const int o = token >> 3;
  return (o << 3) + 2 * (((token >> 1) - o) & 3) + (token & 1);
}

// Codes of one word as fp16 pairs (nibbles 0 4 | 1 5 | 2 6 | 3 7).
__device__ __forceinline__ void codes_f16(uint32_t w, __half2 (&c)[4]) {
  const uint32_t v = w >> 8;
  const __half2 bias = bits_h2(0x64006400u);  // 1024
  const __half2 sixteenth = bits_h2(0x2c002c00u), shift = bits_h2(0xd400d400u);  // 1/16, -64
  c[0] = __hsub2(bits_h2((w & 0x000f000fu) | 0x64006400u), bias);
  c[1] = __hfma2(bits_h2((w & 0x00f000f0u) | 0x64006400u), sixteenth, shift);
  c[2] = __hsub2(bits_h2((v & 0x000f000fu) | 0x64006400u), bias);
  c[3] = __hfma2(bits_h2((v & 0x00f000f0u) | 0x64006400u), sixteenth, shift);
}
__device__ __forceinline__ void clamp_words(uint4* at) {  // NaN stays
  const __half2 top = bits_h2(0x7bff7bffu), bottom = bits_h2(0xfbfffbffu);
  uint32_t* w = reinterpret_cast<uint32_t*>(at);
#pragma unroll 1
  for (int i = 0; i < 4; ++i) w[i] = h2_bits(__hmax2_nan(__hmin2_nan(bits_h2(w[i]), top), bottom));
}
}  // namespace

// MMAs and commits that a converged warp reaches and the lane with `lead` issues.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e;
}
__device__ __forceinline__ void umma_f16_lead(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 e, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate),
      "r"(lead)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts_lead(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 e, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate),
      "r"(lead)
      : "memory");
}
__device__ __forceinline__ void umma_commit_lead(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(lead)
      : "memory");
}

// 16 consecutive 32-bit columns of one TMEM lane per thread.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
      "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
      "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
      "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15]))
      : "memory");
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
// Registers a thread of the four warpgroups: 72 + 160 + 160 + 120 = 4 x 128, what the block starts with.
constexpr int kChunkRegsIssue = 72, kChunkRegsSoftmax = 160, kChunkRegsRebuild = 120;

// What a row sees of a unit of 32 tokens: tau < hi and (tau > lo or tau < sinks), a bit per key position.
__device__ __forceinline__ uint32_t chunk_seen(int hi, int lo, int sinks) {
  auto below = [](int n) -> uint32_t { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); };
  const uint32_t m = below(hi) & (~below(lo + 1) | below(sinks));
  // token pair p of group o stands at pair (p - o) & 3: byte o turns right by 2 o bits
  uint32_t r = m & 0xffu;
#pragma unroll
  for (int o = 1; o < 4; ++o) {
    const uint32_t x = m >> (8 * o) & 0xffu;
    r |= ((x >> (2 * o) | x << (8 - 2 * o)) & 0xffu) << (8 * o);
  }
  return r;
}

template <int D>
__global__ void __launch_bounds__(ChunkShape<D>::kThreads, 1) kv4_chunk_kernel(const __grid_constant__ Kv4AttnParams P) {
  using U = Kv4Unit<D>;
  using Sh = ChunkShape<D>;
  constexpr int G = U::kG;
  constexpr int kS = Sh::kStages, kR = Sh::kRawStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * Sh::kQTile;
  uint8_t* sV = sK + kS * Sh::kKTile;
  uint8_t* sRaw = sV + kS * Sh::kVTile;
  uint8_t* sBad = sRaw + kR * Sh::kRaw;  // [stage][group of V, then K, then any][8] bytes
  uint64_t* bars = reinterpret_cast<uint64_t*>(sBad + Sh::kBad);
  uint64_t* q_full = bars;
  uint64_t* raw_full = bars + 1;
  uint64_t* raw_empty = raw_full + kR;
  uint64_t* k_full = raw_empty + kR;
  uint64_t* k_empty = k_full + kS;
  uint64_t* v_full = k_empty + kS;
  uint64_t* v_empty = v_full + kS;
  uint64_t* gbar = v_empty + kS;
  auto s_full = [&](int g) { return gbar + 7 * g; };
  auto p_full = [&](int g) { return gbar + 7 * g + 2; };
  auto o_done = [&](int g) { return gbar + 7 * g + 4; };
  auto o_final = [&](int g) { return gbar + 7 * g + 6; };
  uint64_t* drain = gbar + 14;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    for (int s = 0; s < kR; ++s) mbar_init(&raw_full[s], 1), mbar_init(&raw_empty[s], 4);
    for (int s = 0; s < kS; ++s) {
      mbar_init(&k_full[s], 2), mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 2), mbar_init(&v_empty[s], 1);
    }
    for (int g = 0; g < 2; ++g) {
      for (int i = 0; i < 2; ++i) mbar_init(&s_full(g)[i], 1), mbar_init(&p_full(g)[i], 4), mbar_init(&o_done(g)[i], 1);
      mbar_init(o_final(g), 1);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
  }
  griddep_wait();
  griddep_launch();
  // ---- this CTA's rows: the last tile of a sequence, which sees most keys, first ----
  const int b = blockIdx.z, kvh = blockIdx.y;
  const int q0 = P.c.cu[b], nq = P.c.cu[b + 1] - q0, len = P.c.lengths[b];
  if (nq <= 0 || q0 < 0 || nq > P.max_new || len > P.max_len || q0 + nq > P.c.tokens) {
    if (nq != 0 && threadIdx.x == 0) record_error(kErrKv4Bound);
    return;
  }
  const int tiles = (nq * P.group + 255) / 256;
  const int tile = tiles - 1 - static_cast<int>(blockIdx.x);
  if (tile < 0) return;
  const int c0 = tile * 256, nrows = min(256, nq * P.group - c0);
  const int ng = nrows > 128 ? 2 : 1;
  const Kv4Span span = kv4_span(len, nq, c0 / P.group, (c0 + nrows - 1) / P.group, P.window, P.sinks);
  const int nt = (span.count + 1) / 2;  // key tiles

  if (warp == 1) tmem_alloc(tmem_slot, Sh::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    reg_dec<kChunkRegsIssue>();
  if (warp == 0) {
    // ---------------- units: bulk copies; lane i looks up the i-th of the next 32 ----------------
    bool ok = true;
    int index = -1;
    const uint64_t policy = l2_policy_evict_last();
    for (int j = 0; j < nt; ++j) {
      if ((j & 15) == 0) {
        const int i = 2 * j + lane;
        index = i < span.count ? kv4_unit_index(P.c, b, kvh, span.unit(i)) : -1;
        if (i < span.count && index < 0) record_error(kErrKv4Table);
      }
      const int a = __shfl_sync(0xffffffffu, index, 2 * (j & 15)), c = __shfl_sync(0xffffffffu, index, 2 * (j & 15) + 1);
      const int s = j % kR;
      if (lane == 0) {
        ok = mbar_wait(&raw_empty[s], (static_cast<uint32_t>(j / kR) & 1u) ^ 1u, kErrKv4Chunk);
        if (ok) {
          const int n = (a >= 0) + (c >= 0);
          if (n)
            mbar_arrive_expect_tx(&raw_full[s], n * U::kBytes);
          else
            mbar_arrive(&raw_full[s]);
          uint8_t* dst = sRaw + s * Sh::kRaw;
          if (a >= 0) bulk_load(dst, P.c.data + static_cast<long long>(a) * U::kBytes, U::kBytes, &raw_full[s], policy);
          if (c >= 0) bulk_load(dst + U::kBytes, P.c.data + static_cast<long long>(c) * U::kBytes, U::kBytes, &raw_full[s], policy);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (!ok) break;
    }
    if (!ok) settle_issued_copies();
  } else if (warp == 1) {
    // ---------------- MMAs ----------------
    // the whole warp runs the loop, so that descriptors stay in uniform registers; one elected lane
    // issues
    const uint32_t lead = elect_one();
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const int tiles_k = __shfl_sync(0xffffffffu, nt, 0), groups = __shfl_sync(0xffffffffu, ng, 0);
    constexpr uint32_t idesc_s = umma_idesc_f16(128, 64), idesc_o = umma_idesc_f16(128, D);
    const uint64_t q_desc = umma_desc_sw128(smem_u32(sQ)), k_desc = umma_desc_sw128(smem_u32(sK)), v_desc = umma_desc_sw128(smem_u32(sV));
    bool ok = tiles_k > 0 && __all_sync(0xffffffffu, mbar_wait(q_full, 0u, kErrKv4Chunk + 1));
    tc_fence_after();
    // S runs two tiles ahead of PV
    int ks = 0, vs = 0;  // stages of S_{j+2} and PV_j, and their rounds' parity
    uint32_t kp = 0u, vp = 0u;
    for (int j = -2; ok && j < tiles_k; ++j) {
      const int b2 = j & 1;  // buffer of tiles j and j + 2
      if (j >= 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&v_full[vs], vp, kErrKv4Chunk + 1));
        for (int g = 0; ok && g < groups; ++g) {
          ok = __all_sync(0xffffffffu, mbar_wait(&p_full(g)[b2], static_cast<uint32_t>(j >> 1) & 1u, kErrKv4Chunk + 1));
          if (!ok) break;
          tc_fence_after();
          const uint64_t vd = v_desc + static_cast<uint32_t>(vs) * (Sh::kVTile >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16_ts_lead(lead, tm + Sh::kOCol + g * D, tm + (2 * g + b2) * 64 + 8 * k, vd + 2 * k, idesc_o, (j | k) != 0);
          umma_commit_lead(lead, &o_done(g)[b2]);
          if (j == tiles_k - 1) umma_commit_lead(lead, o_final(g));
        }
        if (!ok) break;
        umma_commit_lead(lead, &v_empty[vs]);
        if (++vs == kS) vs = 0, vp ^= 1u;
      }
      if (j + 2 < tiles_k) {
        ok = __all_sync(0xffffffffu, mbar_wait(&k_full[ks], kp, kErrKv4Chunk + 1));
        for (int g = 0; ok && g < groups; ++g) {
          // the buffer holds P_j until its product is done
          if (j >= 0) ok = __all_sync(0xffffffffu, mbar_wait(&o_done(g)[b2], static_cast<uint32_t>(j >> 1) & 1u, kErrKv4Chunk + 1));
          if (!ok) break;
          tc_fence_after();
          const uint64_t qd = q_desc + static_cast<uint32_t>(g) * (Sh::kQTile >> 4), kd = k_desc + static_cast<uint32_t>(ks) * (Sh::kKTile >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_f16_lead(lead, tm + (2 * g + b2) * 64, qd + (((k >> 2) * Sh::kQChunk + 32 * (k & 3)) >> 4),
                          kd + (((k >> 2) * Sh::kKChunk + 32 * (k & 3)) >> 4), idesc_s, k != 0);
          umma_commit_lead(lead, &s_full(g)[b2]);
        }
        if (!ok) break;
        umma_commit_lead(lead, &k_empty[ks]);
        if (++ks == kS) ks = 0, kp ^= 1u;
      }
    }
    if (!ok && tiles_k > 0) {  // the MMAs already issued finish before tensor memory is released
      umma_commit_lead(lead, drain);
      mbar_wait_teardown(drain, 0u);
    }
  }
  } else if (warp >= 12) {
    // ---------------- rebuild K (warps 12, 13) and V^T (warps 14, 15) ----------------
    reg_dec<kChunkRegsRebuild>();
    const bool is_v = warp >= 14;
    const int w = warp & 1;
    bool ok = true;
    for (int j = 0; ok && j < nt; ++j) {
      const int s = j % kS, rs = j % kR;
      ok = mbar_wait(&raw_full[rs], static_cast<uint32_t>(j / kR) & 1u, kErrKv4Chunk + 2) &&
           mbar_wait(is_v ? &v_empty[s] : &k_empty[s], (static_cast<uint32_t>(j / kS) & 1u) ^ 1u, kErrKv4Chunk + 2);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint8_t* raw = sRaw + rs * Sh::kRaw;
      if (!is_v) {
        // lane (quarter q, upper u, t): tokens r and r ^ 5 of a group of eight share a quarter, which
        // keeps both the loads (64-byte rows) and the swizzled stores free of conflicts
        const int t = lane & 3, r = (lane >> 3) ^ ((lane & 4) ? 5 : 0);
        uint8_t* dst = sK + s * Sh::kKTile;
#pragma unroll 1
        for (int p = 0; p < 4; ++p) {
          const int token = 8 * (4 * w + p) + r, tau = token & 31;
          const uint8_t* un = raw + (token >> 5) * U::kBytes;
          uint32_t code[G], meta[G];
          lds_words<G>(un + tau * U::kRow + t * 4 * G, code);
          lds_words<G>(un + U::kKMeta + 4 * G * tau, meta);
          __half2 z = bits_h2(0u);  // NaN once a value would not be finite
#pragma unroll
          for (int i = 0; i < G / 2; ++i)
            z = __hfma2(__hfma2(bits_h2(0x4b804b80u), bits_h2(meta[i]), bits_h2(meta[G / 2 + i])), bits_h2(0u), z);
          const int row = chunk_row(token);
          uint8_t* at = dst + row * 128;
#pragma unroll
          for (int gi = 0; gi < G; ++gi) {
            const uint32_t sel = (gi & 1) ? 0x3232u : 0x1010u;
            const __half2 sc = bits_h2(__byte_perm(meta[gi / 2], 0u, sel)), lo = bits_h2(__byte_perm(meta[G / 2 + gi / 2], 0u, sel));
            __half2 c[4];
            codes_f16(code[gi], c);
            uint4 u;
            u.x = h2_bits(__hfma2(c[0], sc, lo)), u.y = h2_bits(__hfma2(c[1], sc, lo));
            u.z = h2_bits(__hfma2(c[2], sc, lo)), u.w = h2_bits(__hfma2(c[3], sc, lo));
            *reinterpret_cast<uint4*>(at + (gi >> 1) * Sh::kKChunk + (((4 * (gi & 1) + t) ^ (row & 7)) << 4)) = u;
          }
          if (h2_bits(z) & 0x7fff7fffu) {  // a value outside fp16's range becomes its largest
#pragma unroll 1
            for (int gi = 0; gi < G; ++gi)
              clamp_words(reinterpret_cast<uint4*>(at + (gi >> 1) * Sh::kKChunk + (((4 * (gi & 1) + t) ^ (row & 7)) << 4)));
          }
        }
      } else {
        // lane (g, group of eight o): channels 32 j + 4 g + i of eight tokens, four 16-byte keys each
        const int o = 4 * w + (lane & 3), g = lane >> 2;
        const uint8_t* un = raw + (o >> 2) * U::kBytes;
        const int at = (o & 3) >> 1, hh = o & 1;  // block of 16, half
        uint32_t code[4][G], sc[4][G], lo[4][G];
        __half2 z = bits_h2(0u);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t = (k + o) & 3;
          lds_words<G>(un + U::kV + 8 * D * at + 4 * D * hh + 4 * G * (4 * g + t), code[k]);
          lds_words<G>(un + U::kVScale + 32 * G * at + 16 * G * hh + 4 * G * t, sc[k]);
          lds_words<G>(un + U::kVLow + 32 * G * at + 16 * G * hh + 4 * G * t, lo[k]);
#pragma unroll
          for (int gi = 0; gi < G; ++gi)
            z = __hfma2(__hfma2(bits_h2(0x4b804b80u), bits_h2(sc[k][gi]), bits_h2(lo[k][gi])), bits_h2(0u), z);
        }
        // lane g also looks at K of token 8 o + g
        uint32_t meta[G];
        lds_words<G>(un + U::kKMeta + 4 * G * ((8 * o + g) & 31), meta);
        __half2 zk = bits_h2(0u);
#pragma unroll
        for (int i = 0; i < G; ++i) zk = __hfma2(bits_h2(meta[i]), bits_h2(0u), zk);
        const unsigned bad_k = __ballot_sync(0xffffffffu, h2_bits(zk) & 0x7fff7fffu);
        const bool odd = (h2_bits(z) & 0x7fff7fffu) != 0u;  // a value would not be finite
        uint32_t bad[G];
#pragma unroll
        for (int gi = 0; gi < G; ++gi) bad[gi] = 0u;
        if (odd) {
          const __half2 inf = bits_h2(0x7c007c00u);
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int gi = 0; gi < G; ++gi) {
              const uint32_t fine = __hlt2_mask(__habs2(bits_h2(sc[k][gi])), inf) & __hlt2_mask(__habs2(bits_h2(lo[k][gi])), inf);
              sc[k][gi] &= fine, lo[k][gi] &= fine;
              bad[gi] |= ((~fine & 1u) | (~fine >> 15 & 2u)) << (2 * k);
            }
        }
        if (__any_sync(0xffffffffu, odd || bad_k != 0u)) {
          if (g == 0) {
#pragma unroll
            for (int gi = 0; gi < G; ++gi) sBad[(s * (G + 2) + gi) * 8 + o] = static_cast<uint8_t>(bad[gi]);
            uint32_t byte = 0u;
#pragma unroll 1
            for (int i = 0; i < 8; ++i) byte |= (bad_k >> (4 * i + lane) & 1u) << (chunk_row(8 * o + i) & 7);
            sBad[(s * (G + 2) + G) * 8 + o] = static_cast<uint8_t>(byte);
            sBad[(s * (G + 2) + G + 1) * 8 + o] = 1u;
          }
          __syncwarp();
        } else if (g == 0) {
          // the other warp's groups may be marked: then these are read too
#pragma unroll
          for (int gi = 0; gi <= G + 1; ++gi) sBad[(s * (G + 2) + gi) * 8 + o] = 0u;
        }
        uint8_t* dst = sV + s * Sh::kVTile;
#pragma unroll
        for (int gi = 0; gi < G; ++gi) {
          uint32_t out[4][4];  // [channel i][pair k]
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t x = __byte_perm(code[k][gi / 2], code[k][G / 2 + gi / 2], (gi & 1) ? 0x7632u : 0x5410u);
            __half2 c[4];
            codes_f16(x, c);  // channels 0..3 of tokens 2t | 2t + 1
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              out[i][k] = h2_bits(__hfma2(c[i], bits_h2(sc[k][gi]), bits_h2(lo[k][gi])));
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = 32 * gi + 4 * g + i;
            *reinterpret_cast<uint4*>(dst + row * 128 + ((o ^ (row & 7)) << 4)) = make_uint4(out[i][0], out[i][1], out[i][2], out[i][3]);
          }
        }
        if (odd) {
#pragma unroll 1
          for (int i = 0; i < 4 * G; ++i) {
            const int row = 32 * (i >> 2) + 4 * g + (i & 3);
            clamp_words(reinterpret_cast<uint4*>(dst + row * 128 + ((o ^ (row & 7)) << 4)));
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(is_v ? &v_full[s] : &k_full[s]);
        mbar_arrive(&raw_empty[rs]);
      }
    }
  } else {
    // ---------------- softmax: one row a thread ----------------
    reg_inc<kChunkRegsSoftmax>();
    const int g = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane;
    const int row = c0 + 128 * g + r;  // among the kv head's rows
    const bool live = 128 * g + r < nrows;
    const int tok = row / P.group, head = kvh * P.group + row - tok * P.group;
    const int ps = live ? len - nq + tok : -1;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    float fac;  // log2 score per unit of the products
    {
      uint4 u[D / 8];
      const uint4* src = reinterpret_cast<const uint4*>(P.q + static_cast<long long>(q0 + tok) * P.ldq + static_cast<long long>(head) * D);
      float mx = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        u[i] = live ? src[i] : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t x[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float lo, hi;
          unpack_bf16x2(x[e], lo, hi);
          mx = fmaxf(mx, fmaxf(fabsf(lo), fabsf(hi)));
        }
      }
      const int ex = static_cast<int>(__float_as_uint(mx) >> 23);
      const int e2 = mx > 0.0f ? min(max(268 - ex, 1), 253) : 127;  // 2^(14 - exponent), a normal number
      const float up = __uint_as_float(static_cast<uint32_t>(e2) << 23);
      fac = P.scale_log2 * __uint_as_float(static_cast<uint32_t>(254 - e2) << 23);
      uint8_t* dst = sQ + g * Sh::kQTile + r * 128;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        float v[8];
        unpack_bf16x2(u[i].x, v[0], v[1]);
        unpack_bf16x2(u[i].y, v[2], v[3]);
        unpack_bf16x2(u[i].z, v[4], v[5]);
        unpack_bf16x2(u[i].w, v[6], v[7]);
        uint4 o;  // the order of the nibbles
        o.x = h2_bits(__floats2half2_rn(v[0] * up, v[4] * up));
        o.y = h2_bits(__floats2half2_rn(v[1] * up, v[5] * up));
        o.z = h2_bits(__floats2half2_rn(v[2] * up, v[6] * up));
        o.w = h2_bits(__floats2half2_rn(v[3] * up, v[7] * up));
        *reinterpret_cast<uint4*>(dst + (i >> 3) * Sh::kQChunk + (((i & 7) ^ (r & 7)) << 4)) = o;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    // positions of the tile's first and last row
    const int pos_lo = len - nq + (c0 + 128 * g) / P.group;
    const int pos_hi = len - nq + (c0 + min(nrows, 128 * g + 128) - 1) / P.group;
    float m_ref = -INFINITY, l_run = 0.0f;
    uint32_t poison = 0u;  // groups in which a visible token has no finite value
    bool ok = g < ng;
    for (int j = 0; ok && j < nt; ++j) {
      const int sb = j & 1;
      const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u;
      const uint32_t s_col = tmem + lane_off + (2 * g + sb) * 64;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full(g)[sb], ph, kErrKv4Chunk + 3));
      if (!ok) break;
      tc_fence_after();
      // ---- masks: keys of the two units; a unit past the span is hidden ----
      bool plain = true;
      int key0[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool have = 2 * j + i < span.count;
        key0[i] = have ? kKv4Unit * span.unit(2 * j + i) : 0x40000000;
        plain &= key0[i] + 31 <= pos_lo && (P.window <= 0 || pos_hi - key0[i] < P.window || key0[i] + 31 < P.sinks);
      }
      uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
      if (!plain) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          seen[i] = P.window > 0 ? chunk_seen(ps - key0[i] + 1, ps - P.window - key0[i], P.sinks - key0[i])
                                 : chunk_seen(ps - key0[i] + 1, -1, 0);
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      float sv[64];
      tmem_ld32(s_col, *reinterpret_cast<float(*)[32]>(&sv[0]));
      tmem_ld32(s_col + 32, *reinterpret_cast<float(*)[32]>(&sv[32]));
      tmem_wait_ld();
      if (!plain) {
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (!(seen[c >> 5] >> (c & 31) & 1u)) sv[c] = -INFINITY;
      }
#pragma unroll
      for (int c = 0; c < 64; ++c) mx4[c & 3] = fmaxf(mx4[c & 3], sv[c]);
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * fac;
      const bool grow = mx > m_ref + kRescaleLog2;
      float alpha = 1.0f;
      if (grow) {
        alpha = m_ref == -INFINITY ? 0.0f : ex2_approx(m_ref - mx);
        m_ref = mx;
        l_run *= alpha;
      }
      if (j > 0 && __any_sync(0xffffffffu, grow)) {  // O holds PV_0 .. PV_{j-1}: scale the rows that moved
        ok = __all_sync(0xffffffffu, mbar_wait(&o_done(g)[sb ^ 1], static_cast<uint32_t>((j - 1) >> 1) & 1u, kErrKv4Chunk + 3));
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int h = 0; h < D / 32; ++h) {
          float o[32];
          tmem_ld32(tmem + lane_off + Sh::kOCol + g * D + 32 * h, o);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] *= alpha;
          tmem_st32(tmem + lane_off + Sh::kOCol + g * D + 32 * h, o);
        }
        tmem_wait_st();
      }
      const float m_use = m_ref == -INFINITY ? 0.0f : m_ref;
      const float2 f2 = make_float2(fac, fac), n2 = make_float2(-m_use, -m_use);
      float2 sum0 = make_float2(0.0f, 0.0f), sum1 = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float pk[16];
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const float2 x = fma_f32x2(make_float2(sv[32 * i + c], sv[32 * i + c + 1]), f2, n2);
          const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          if (c & 2) sum1 = add_f32x2(sum1, e); else sum0 = add_f32x2(sum0, e);
          pk[c >> 1] = __uint_as_float(h2_bits(__floats2half2_rn(e.x, e.y)));
        }
        tmem_st16(s_col + 16 * i, pk);  // P_j over S_j, two keys a column
      }
      l_run += (sum0.x + sum0.y) + (sum1.x + sum1.y);
      tmem_wait_st();
      // ---- values that are not finite (the marks are there once V_j is) ----
      ok = __all_sync(0xffffffffu, mbar_wait(&v_full[j % kS], static_cast<uint32_t>(j / kS) & 1u, kErrKv4Chunk + 3));
      if (!ok) break;
      const uint32_t* marks = reinterpret_cast<const uint32_t*>(sBad + (j % kS) * (G + 2) * 8);
      if (marks[2 * G + 2] | marks[2 * G + 3]) {
#pragma unroll 1
        for (int gi = 0; gi <= G; ++gi)
          if ((seen[0] & marks[2 * gi]) | (seen[1] & marks[2 * gi + 1])) poison |= gi < G ? 1u << gi : 0xffffffffu;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full(g)[sb]);
    }
    if (ok && nt > 0) ok = mbar_wait(o_final(g), 0u, kErrKv4Chunk + 3);
    if (__all_sync(0xffffffffu, ok) && g < ng) {
      tc_fence_after();
      const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;  // no visible key: zeros
      uint4* dst = reinterpret_cast<uint4*>(P.out + (static_cast<long long>(q0 + tok) * P.q_heads + head) * D);
#pragma unroll
      for (int h = 0; h < D / 32; ++h) {
        float o[32];
        if (nt > 0) {
          tmem_ld32(tmem + lane_off + Sh::kOCol + g * D + 32 * h, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = 0.0f;
        }
        const float f = (poison >> h & 1u) ? NAN : inv;
        if (live) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 u;
            u.x = pack_bf16x2(o[8 * i + 0] * f, o[8 * i + 1] * f);
            u.y = pack_bf16x2(o[8 * i + 2] * f, o[8 * i + 3] * f);
            u.z = pack_bf16x2(o[8 * i + 4] * f, o[8 * i + 5] * f);
            u.w = pack_bf16x2(o[8 * i + 6] * f, o[8 * i + 7] * f);
            dst[4 * h + i] = u;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kTmemCols);
  }
}

cudaError_t launch_kv4_chunk(const Kv4AttnParams& p, int head_dim, cudaStream_t stream) {
  const dim3 grid((p.max_new * p.group + 255) / 256, p.c.kv_heads, p.c.seqs);
  return head_dim == 128
             ? launch_pdl(kv4_chunk_kernel<128>, grid, ChunkShape<128>::kThreads, ChunkShape<128>::kSmem, stream, p)
             : launch_pdl(kv4_chunk_kernel<64>, grid, ChunkShape<64>::kThreads, ChunkShape<64>::kSmem, stream, p);
}

cudaError_t kv4_chunk_prepare_device() {
  cudaError_t e = cudaFuncSetAttribute(kv4_chunk_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(ChunkShape<128>::kSmem));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kv4_chunk_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(ChunkShape<64>::kSmem));
  return e;
}

}  // namespace rldx
