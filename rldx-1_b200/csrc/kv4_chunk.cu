// Attention of many new tokens per sequence over the paged 4-bit cache (layout: kv4.cuh), on
// tcgen05: one CTA takes 256 query rows (new token, head of the group) of one kv head, in two tiles
// of 128, and runs over the keys they can see in tiles of 64 (two units):
//   S = Q K^T (M = 128, N = 64, K = d), P = exp2(S - m), O += P V (M = 128, N = d, K = 64)
// with S, P and O in tensor memory and the codes rebuilt to fp16 on the way to shared memory:
// scale code + low in one fp16 fma, off by 2^-11 of the value.  q goes to
// fp16 scaled by a power of two per row (largest in [2^14, 2^15)).  p is fp16, off by 2^-11 and by 2^-25 beside a largest
// of 2^7 to 2^15 (a reference moved lazily, kChunkSet, kChunkMove); sums and maxima are fp32.  With a largest of 1
// to 2^8 a thousand tokens at 2^-24.4 of the largest weight counted a third too much.
//
// Warps: 0 fetches units by bulk copies, 1 issues the MMAs, 2-3 rebuild K, 4-11 do the softmax (one row a
// thread), 12-15 rebuild V^T; registers move from the first four to the softmax.  The order of
// channels inside 16 bytes of K (and q) is that of the nibbles under the masks (0 4 1 5 2 6 3 7), and tokens
// stand inside each group of eight in an order rotated by the group (chunk_token), so that neither
// side needs a shuffle and both the reads of the units and the writes of the swizzled tiles are free
// of bank conflicts.
//
// P_j takes the place of S_j in tensor memory, so S_{j+2} is issued once PV_j has finished; the
// other query tile's products keep the tensor cores busy meanwhile.
//
// A value of V that is not finite, of a token that some rows must not see, cannot go through a
// product with p = 0: it is rebuilt as 0, its place marked, and the rows that do see the token
// give NaN in the channels of its group (in every channel where K is not finite).  A unit without a page
// is marked the same way and hidden from every row, whatever its place in the ring holds.
//
// Few tiles of rows would leave most SMs idle, so up to two waves' worth of CTAs share a tile's keys evenly
// and a second kernel joins their parts (the rule and both sides' times: decode_plan).  With more than
// a wave of tiles each CTA has its own, longest first.
//
// Measured: 8 sequences of up to 2300 tokens, up to 1104 of them new, 16 / 2 heads, d = 128: 138 us, 32 % of
// cuBLAS's bf16 rate (44 us).  No role bounds it alone: without three quarters of K's rebuilding, of V's, or
// without nearly all exponentials it takes 138, 133 and 131 us.  K's tiles of 64 keys give an MMA of N = 64, P takes S's
// place, and the chain S, softmax, P V of the two query tiles covers each other's waits only in part.
#include "host_util.h"
#include "kv4.cuh"

namespace rldx {

namespace {
// A row's reference (log2 units) stands 7 below the largest score when it is set and is set again once one passes it
// by more than 15: p = 2^(score - reference) is at most 2^15, and 2^7 or more for the largest.
constexpr float kChunkSet = 7.0f, kChunkMove = 15.0f;
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
  // Marks of a stage of V: what is not finite, a bit per token, in V's groups and K; then a byte for each eight tokens,
  // 1: there is any, 2: their unit has no page.  Then a byte a raw stage: which of its units have none.
  static constexpr int kBad = kStages * (kG + 2) * 8 + 8;
  static constexpr size_t kSmem = 1024 + 2 * kQTile + kStages * (kKTile + kVTile) + kRawStages * kRaw + kBad + 8 * kBars + 16 + 64;
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

// Codes of one word as fp16 pairs: its nibbles 0 4 | 1 5, and with those of word >> 8 also 2 6 | 3 7.  A half of exponent
// 2^10 has a last bit of 1, so a nibble in its low bits makes it 1024 + code, and one four bits further up
// 1024 + 16 code; the difference, or the difference of a sixteenth and 64, is exact.
__device__ __forceinline__ void codes_f16_low(uint32_t w, __half2 (&c)[2]) {
  c[0] = __hsub2(bits_h2((w & 0x000f000fu) | 0x64006400u), bits_h2(0x64006400u));                                // 1024
  c[1] = __hfma2(bits_h2((w & 0x00f000f0u) | 0x64006400u), bits_h2(0x2c002c00u), bits_h2(0xd400d400u));  // 1/16, -64
}
__device__ __forceinline__ void codes_f16(uint32_t w, __half2 (&c)[4]) {
  codes_f16_low(w, *reinterpret_cast<__half2(*)[2]>(&c[0]));
  codes_f16_low(w >> 8, *reinterpret_cast<__half2(*)[2]>(&c[2]));
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

__device__ __forceinline__ bool chunk_in_bounds(const Kv4AttnParams& P, int q0, int nq, int len) {
  return nq > 0 && q0 >= 0 && nq <= P.max_new && len <= P.max_len && q0 + nq <= P.c.tokens;
}

// What a CTA works on, in shared memory, so that each role keeps no more of it in registers than it needs.
struct alignas(16) ChunkShare {
  int u0, sink_units, gap, count;  // unit i of the share stands at i + u0 among the span's `count`; kv4_span's unit()
  int q0, kvh, c0, nrows;          // first query row, kv head, first of the kv head's rows, rows
  int nt, ng, base, b;             // tiles of 64 keys, of 128 rows; position of the first new token; sequence
  __device__ __forceinline__ static int unit(const int4& span, int u) { return u < span.y ? u : span.z + u; }
  __device__ __forceinline__ int4 span() const { return *reinterpret_cast<const int4*>(this); }
};

// The (sequence, tile of rows) that comes at place `rank` when they stand by descending units, equal ones by
// ascending number; at most kChunkOrdered of them.  CTAs that run long start first, which evens out the last wave: 4 sequences of
// 2048 tokens, 1104 of them new, 32 / 8 heads, 184 us against 204 in their own order.
constexpr int kChunkOrdered = 512;
__device__ __forceinline__ int chunk_item_of_rank(const Kv4AttnParams& P, int rank, int max_tiles, int* s_units) {
  const int n = P.c.seqs * max_tiles, i = threadIdx.x;
  int mine = -1;
  if (i < n) {
    const int b = i / max_tiles, c0 = (i - b * max_tiles) * 256;
    const int q0 = P.c.cu[b], nq = P.c.cu[b + 1] - q0, len = P.c.lengths[b];
    mine = 0;
    if (chunk_in_bounds(P, q0, nq, len) && c0 < nq * P.group)
      mine = 1 + kv4_span(len, nq, c0 / P.group, (min(c0 + 256, nq * P.group) - 1) / P.group, P.window, P.sinks).count;
  }
  s_units[i] = mine;
  __syncthreads();
  if (i < n) {
    int before = 0;
#pragma unroll 8
    for (int k = 0; k < n; ++k) before += s_units[k] > mine || (s_units[k] == mine && k < i);
    if (before == rank) s_units[kChunkOrdered] = i;
  }
  __syncthreads();
  const int item = s_units[kChunkOrdered];
  __syncthreads();
  return item;
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
  uint8_t* sGone = sBad + kS * (G + 2) * 8;
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
  ChunkShare& share = *reinterpret_cast<ChunkShare*>((reinterpret_cast<uintptr_t>(tmem_slot) + 19) & ~static_cast<uintptr_t>(15));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    for (int s = 0; s < kR; ++s) mbar_init(&raw_full[s], 1), mbar_init(&raw_empty[s], 6);
    for (int s = 0; s < kS; ++s) {
      mbar_init(&k_full[s], 2), mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 4), mbar_init(&v_empty[s], 1);
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
  // ---- this CTA's rows and its share of their keys ----
  {
    const int max_tiles = (P.max_new * P.group + 255) / 256;
    const int part = static_cast<int>(blockIdx.x % P.split), unsplit = static_cast<int>(blockIdx.x / P.split);
    int item = unsplit / P.c.kv_heads;  // sequence, tile
    if (P.ordered) item = chunk_item_of_rank(P, item, max_tiles, reinterpret_cast<int*>(smem));
    const int b = item / max_tiles, c0 = (item - b * max_tiles) * 256;
    const int q0 = P.c.cu[b], nq = P.c.cu[b + 1] - q0, len = P.c.lengths[b];
    const bool fine = chunk_in_bounds(P, q0, nq, len);
    if (blockIdx.x == 0 || !fine) {  // zeros: in rows of no sequence, and of one that breaks the call's bounds
      if (!fine && nq != 0 && threadIdx.x == 0) record_data_error(kErrKv4Bound);
      const bool all = !fine && c0 == 0 && part == 0 && unsplit % P.c.kv_heads == 0;
#pragma unroll 1
      for (int k = blockIdx.x == 0 ? 0 : 2; k < (all ? 3 : 2); ++k)
        kv4_zero_rows(P, D, k == 0 ? 0 : k == 1 ? P.c.cu[P.c.seqs] : q0, k == 0 ? P.c.cu[0] : k == 1 ? P.c.tokens : q0 + nq, threadIdx.x,
                      blockDim.x);
      if (!fine) return;
    }
    const int nrows = min(256, nq * P.group - c0);
    if (nrows <= 0) return;
    if (threadIdx.x == 0) {
      const Kv4Span span = kv4_span(len, nq, c0 / P.group, (c0 + nrows - 1) / P.group, P.window, P.sinks);
      const int all = (span.count + 1) / 2;
      int t0 = 0, t1 = all;
      if (P.split > 1) {
        t0 = static_cast<int>(static_cast<long long>(all) * part / P.split);
        t1 = static_cast<int>(static_cast<long long>(all) * (part + 1) / P.split);
      }
      share.u0 = 2 * t0, share.sink_units = span.sink_units, share.gap = span.first - span.sink_units, share.count = span.count;
      share.q0 = q0, share.kvh = unsplit % P.c.kv_heads, share.c0 = c0, share.nrows = nrows;
      share.nt = t1 - t0, share.ng = nrows > 128 ? 2 : 1;
      share.base = len - nq, share.b = b;
    }
  }

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
    const int4 span = share.span();
    const int nt = share.nt, kvh = share.kvh, b = share.b;
    for (int j = 0; j < nt; ++j) {
      if ((j & 15) == 0) {
        const int u = span.x + 2 * j + lane;
        index = u < span.w ? kv4_unit_index(P.c, b, kvh, ChunkShare::unit(span, u)) : -2;
        if (index == -1) record_data_error(kErrKv4Table);
      }
      const int a = __shfl_sync(0xffffffffu, index, 2 * (j & 15)), c = __shfl_sync(0xffffffffu, index, 2 * (j & 15) + 1);
      const int s = j % kR;
      if (lane == 0) {
        ok = mbar_wait(&raw_empty[s], (static_cast<uint32_t>(j / kR) & 1u) ^ 1u, kErrKv4Chunk);
        if (ok) {
          const int n = (a >= 0) + (c >= 0);
          sGone[s] = (a == -1 ? 1 : 0) | (c == -1 ? 2 : 0);
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
    const int tiles_k = __shfl_sync(0xffffffffu, share.nt, 0), groups = __shfl_sync(0xffffffffu, share.ng, 0);
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
  } else {
    // ---------------- rebuild K (warps 2, 3) ----------------
    const int w = warp & 1, nt = share.nt;
    bool ok = true;
    for (int j = 0; ok && j < nt; ++j) {
      const int s = j % kS, rs = j % kR;
      ok = mbar_wait(&raw_full[rs], static_cast<uint32_t>(j / kR) & 1u, kErrKv4Chunk + 2) &&
           mbar_wait(&k_empty[s], (static_cast<uint32_t>(j / kS) & 1u) ^ 1u, kErrKv4Chunk + 2);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint8_t* raw = sRaw + rs * Sh::kRaw;
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
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&k_full[s]);
        mbar_arrive(&raw_empty[rs]);
      }
    }
  }
  } else if (warp >= 12) {
    // ---------------- rebuild V^T (warps 12 to 15) ----------------
    reg_dec<kChunkRegsRebuild>();
    const int w = warp & 3, nt = share.nt;
    bool ok = true;
    for (int j = 0; ok && j < nt; ++j) {
      const int s = j % kS, rs = j % kR;
      ok = mbar_wait(&raw_full[rs], static_cast<uint32_t>(j / kR) & 1u, kErrKv4Chunk + 2) &&
           mbar_wait(&v_empty[s], (static_cast<uint32_t>(j / kS) & 1u) ^ 1u, kErrKv4Chunk + 2);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint8_t* raw = sRaw + rs * Sh::kRaw;
      // lane (g, half h, group of eight o): channels 32 j + 4 g + 2 h + i of eight tokens
      const int o = 2 * w + (lane & 1), h = lane >> 1 & 1, g = lane >> 2;
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
      const uint32_t gone = (sGone[rs] >> (w >> 1) & 1u) << 1;  // (a warp's tokens are of one unit)
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
        if (g == 0 && h == 0) {
#pragma unroll
          for (int gi = 0; gi < G; ++gi) sBad[(s * (G + 2) + gi) * 8 + o] = static_cast<uint8_t>(bad[gi]);
          uint32_t byte = 0u;
#pragma unroll 1
          for (int i = 0; i < 8; ++i) byte |= (bad_k >> (4 * i + lane) & 1u) << (chunk_row(8 * o + i) & 7);
          sBad[(s * (G + 2) + G) * 8 + o] = static_cast<uint8_t>(byte);
          sBad[(s * (G + 2) + G + 1) * 8 + o] = static_cast<uint8_t>(1u | gone);
        }
        __syncwarp();
      } else if (g == 0 && h == 0) {
        // another warp's groups may be marked: then these are read too
#pragma unroll
        for (int gi = 0; gi <= G; ++gi) sBad[(s * (G + 2) + gi) * 8 + o] = 0u;
        sBad[(s * (G + 2) + G + 1) * 8 + o] = static_cast<uint8_t>(gone);
      }
      uint8_t* dst = sV + s * Sh::kVTile;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        uint32_t out[2][4];  // [channel i][pair k]
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t x = __byte_perm(code[k][gi / 2], code[k][G / 2 + gi / 2], (gi & 1) ? 0x7632u : 0x5410u);
          __half2 c[2];
          codes_f16_low(x >> (8 * h), c);  // channels 2 h, 2 h + 1 of tokens 2t | 2t + 1
#pragma unroll
          for (int i = 0; i < 2; ++i) out[i][k] = h2_bits(__hfma2(c[i], bits_h2(sc[k][gi]), bits_h2(lo[k][gi])));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = 32 * gi + 4 * g + 2 * h + i;
          *reinterpret_cast<uint4*>(dst + row * 128 + ((o ^ (row & 7)) << 4)) = make_uint4(out[i][0], out[i][1], out[i][2], out[i][3]);
        }
      }
      if (odd) {
#pragma unroll 1
        for (int i = 0; i < 2 * G; ++i) {
          const int row = 32 * (i >> 1) + 4 * g + 2 * h + (i & 1);
          clamp_words(reinterpret_cast<uint4*>(dst + row * 128 + ((o ^ (row & 7)) << 4)));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v_full[s]);
        mbar_arrive(&raw_empty[rs]);
      }
    }
  } else {
    // ---------------- softmax: one row a thread ----------------
    reg_inc<kChunkRegsSoftmax>();
    const int g = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane;
    const int nt = share.nt, ng = share.ng;
    int ps, pos_lo, pos_hi;  // positions of this row, and of the tile's first and last
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    float fac;  // log2 score per unit of the products
    {
      const int c0 = share.c0, nrows = share.nrows, base = share.base;
      const bool live = 128 * g + r < nrows;
      const int row = c0 + 128 * g + r, tok = row / P.group, head = share.kvh * P.group + row - tok * P.group;
      ps = live ? base + tok : -1;
      pos_lo = base + (c0 + 128 * g) / P.group;
      pos_hi = base + (c0 + min(nrows, 128 * g + 128) - 1) / P.group;
      uint4 u[D / 8];
      const uint4* src = reinterpret_cast<const uint4*>(P.q + static_cast<long long>(share.q0 + tok) * P.ldq + static_cast<long long>(head) * D);
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
    float m_ref = -INFINITY, l_run = 0.0f;
    uint32_t poison = 0u;  // groups in which a visible token has no finite value
    bool ok = g < ng;
    for (int j = 0; ok && j < nt; ++j) {
      const int sb = j & 1;
      const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u;
      const uint32_t s_col = tmem + lane_off + (2 * g + sb) * 64;
      // ---- masks: keys of the two units; a unit past the span is hidden, and one without a page (the marks are
      // there once V_j is) ----
      ok = __all_sync(0xffffffffu, mbar_wait(&v_full[j % kS], static_cast<uint32_t>(j / kS) & 1u, kErrKv4Chunk + 3));
      if (!ok) break;
      const uint32_t* marks = reinterpret_cast<const uint32_t*>(sBad + (j % kS) * (G + 2) * 8);
      const uint32_t mark[2] = {marks[2 * G + 2], marks[2 * G + 3]};
      bool plain = true;
      int key0[2];
      const int4 span = share.span();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int u = span.x + 2 * j + i;
        key0[i] = u < span.w ? kKv4Unit * ChunkShare::unit(span, u) : 0x40000000;
        plain &= key0[i] + 31 <= pos_lo && (P.window <= 0 || pos_hi - key0[i] < P.window || key0[i] + 31 < P.sinks);
      }
      plain &= ((mark[0] | mark[1]) & 0x02020202u) == 0u;
      uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
      if (!plain) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          seen[i] = P.window > 0 ? chunk_seen(ps - key0[i] + 1, ps - P.window - key0[i], P.sinks - key0[i])
                                 : chunk_seen(ps - key0[i] + 1, -1, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (mark[i] & 0x02020202u) seen[i] = 0u;
      }
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full(g)[sb], ph, kErrKv4Chunk + 3));
      if (!ok) break;
      tc_fence_after();
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
      const bool grow = mx > m_ref + kChunkMove;
      float alpha = 1.0f;
      if (grow) {
        alpha = m_ref == -INFINITY ? 0.0f : ex2_approx(m_ref - (mx - kChunkSet));
        m_ref = mx - kChunkSet;
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
      // ---- values that are not finite ----
      if (mark[0] | mark[1]) {
#pragma unroll 1
        for (int gi = 0; gi <= G; ++gi)
          if ((seen[0] & marks[2 * gi]) | (seen[1] & marks[2 * gi + 1])) poison |= gi < G ? 1u << gi : 0xffffffffu;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full(g)[sb]);
    }
    if (ok && nt > 0) ok = mbar_wait(o_final(g), 0u, kErrKv4Chunk + 3);
    if (g < ng) {
      const bool fine = __all_sync(0xffffffffu, ok);  // no wait has run out: else NaN
      tc_fence_after();
      if (!fine) l_run = NAN;
      const bool whole = P.split == 1;
      const int row = share.c0 + 128 * g + r, tok = row / P.group, head = share.kvh * P.group + row - tok * P.group;
      const bool live = 128 * g + r < share.nrows;
      const float inv = !whole ? 1.0f : l_run == 0.0f ? 0.0f : 1.0f / l_run;  // no visible key: zeros
      uint4* dst = reinterpret_cast<uint4*>(P.out + (static_cast<long long>(share.q0 + tok) * P.q_heads + head) * D);
      if (!whole && live) P.part_ml[256LL * blockIdx.x + 128 * g + r] = make_float2(m_ref, l_run);
#pragma unroll
      for (int h = 0; h < D / 32; ++h) {
        if (nt == 0 && !whole) break;  // (-inf, 0) says that there is nothing
        float o[32];
        if (nt > 0 && fine) {
          tmem_ld32(tmem + lane_off + Sh::kOCol + g * D + 32 * h, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = 0.0f;
        }
        const float f = !fine || (poison >> h & 1u) ? NAN : inv;
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] *= f;
        if (live && whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 u;
            u.x = pack_bf16x2(o[8 * i + 0], o[8 * i + 1]);
            u.y = pack_bf16x2(o[8 * i + 2], o[8 * i + 3]);
            u.z = pack_bf16x2(o[8 * i + 4], o[8 * i + 5]);
            u.w = pack_bf16x2(o[8 * i + 6], o[8 * i + 7]);
            dst[4 * h + i] = u;
          }
        } else if (live) {
          float4* po = reinterpret_cast<float4*>(P.part_o) + (static_cast<long long>(blockIdx.x) * (D / 4) + 8 * h) * 256 + 128 * g + r;
#pragma unroll
          for (int i = 0; i < 8; ++i) po[256 * i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
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

// Joins the parts of rows whose keys were shared out (split > 1): out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.
// A part lies as [d / 4][256 rows][4], so that both the softmax threads, a row each, and the threads here, a
// row and four channels each, read and write whole lines.  A part that saw no key holds nothing in part_o.
template <int D>
__global__ void __launch_bounds__(256) kv4_chunk_join_kernel(const __grid_constant__ Kv4AttnParams P) {
  constexpr int kBatch = 8;  // parts loaded at once
  griddep_wait();
  griddep_launch();
  const int max_tiles = (P.max_new * P.group + 255) / 256;
  const int unsplit = static_cast<int>(blockIdx.x) >> 3, r = (static_cast<int>(blockIdx.x) & 7) * 32 + (threadIdx.x & 31);
  const int four = 8 * blockIdx.y + (threadIdx.x >> 5);
  const int kvh = unsplit % P.c.kv_heads, item = unsplit / P.c.kv_heads;
  const int b = item / max_tiles, row = (item - b * max_tiles) * 256 + r;
  const int q0 = P.c.cu[b], nq = P.c.cu[b + 1] - q0;
  if (!chunk_in_bounds(P, q0, nq, P.c.lengths[b]) || row >= nq * P.group) return;
  const float2* ml = P.part_ml + static_cast<long long>(unsplit) * P.split * 256 + r;
  const float4* po = reinterpret_cast<const float4*>(P.part_o) + (static_cast<long long>(unsplit) * P.split * (D / 4) + four) * 256 + r;
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i0 = 0; i0 < P.split; i0 += kBatch) {
    float2 x[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      x[u] = make_float2(-INFINITY, 0.0f);
      v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (i0 + u < P.split) x[u] = ml[256 * (i0 + u)], v[u] = po[static_cast<long long>(i0 + u) * (D / 4) * 256];
    }
    float mb = m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) mb = fmaxf(mb, x[u].x);
    const float back = part_factor(make_float2(m, l), mb);
    m = mb;
    l *= back, o.x *= back, o.y *= back, o.z *= back, o.w *= back;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (x[u].x == -INFINITY && x[u].y == 0.0f) continue;  // saw no key: v may be anything
      const float f = part_factor(x[u], m);
      l = fmaf(f, x[u].y, l);
      o.x = fmaf(f, v[u].x, o.x), o.y = fmaf(f, v[u].y, o.y), o.z = fmaf(f, v[u].z, o.z), o.w = fmaf(f, v[u].w, o.w);
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no visible key: zeros
  const int tok = row / P.group, head = kvh * P.group + row - tok * P.group;
  *reinterpret_cast<uint2*>(P.out + (static_cast<long long>(q0 + tok) * P.q_heads + head) * D + 4 * four) =
      make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

namespace {
template <int D>
cudaError_t launch_chunk(const Kv4AttnParams& p, unsigned unsplit, cudaStream_t stream) {
  cudaError_t e = launch_pdl(kv4_chunk_kernel<D>, dim3(unsplit * p.split, 1, 1), ChunkShape<D>::kThreads, ChunkShape<D>::kSmem, stream, p);
  if (e != cudaSuccess || p.split == 1) return e;
  return launch_pdl(kv4_chunk_join_kernel<D>, dim3(unsplit * 8, D / 32, 1), 256, 0, stream, p);
}
}  // namespace

cudaError_t launch_kv4_chunk(Kv4AttnParams p, int head_dim, cudaStream_t stream) {
  const unsigned max_tiles = (p.max_new * p.group + 255) / 256, unsplit = max_tiles * p.c.kv_heads * p.c.seqs;
  p.ordered = p.split == 1 && unsplit > static_cast<unsigned>(sm_count()) && max_tiles * p.c.seqs <= kChunkOrdered;
  return head_dim == 128 ? launch_chunk<128>(p, unsplit, stream) : launch_chunk<64>(p, unsplit, stream);
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
