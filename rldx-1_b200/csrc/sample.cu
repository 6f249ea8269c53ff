// Token sampling: temperature, top-k, top-p, min-p, then one draw per row from a given number.
//
// With M the row's maximum, d_i = (x_i - M) / T in fp32 (0 where x_i = M) the weight of token i is the
// whole number w_i = floor(2^32 exp(d_i)), so every sum below is exact and the drawn token depends on
// no summation order, launch shape or batch.  In the order of descending logits, equal ones by
// ascending id, with B_i the weight before token i:
//   top-k   the first k tokens              top-p   those with B_i < p S, S the weight top-k left
//   min-p   w_i >= min_p 2^32               and never a token of weight 0 (exp(d) < 2^-32)
// The draw takes, in the order of ids, the first kept token whose inclusive sum passes floor(u S').
// Sums stay below 2^53 (V < 2^21), so comparisons with products in doubles are exact.
//
// A cluster of CTAs holds a row in shared memory, so the logits are read once.  The last token kept is
// found in one of two ways:
//   - a few candidates (top-k up to about a thousand): the k-th largest of the threads' maxima is a
//     lower bound of the k-th largest logit; the tokens that reach its bin go to rank 0's list, which
//     sorts them (bitonic, ordered bits and id in one word), scans the weights and draws alone.
//   - otherwise by histogram: 1024 bins linear in -d (every bin holds a run of the order), then by the
//     ordered bits of the logit inside the bin where count or weight crosses, until one value is left;
//     of the tokens that share it the first few by id stay.  Bins hold counts (top-k) or weights
//     (top-p: the low 16 and high 17 bits of a weight in two 32-bit sums); CTAs add theirs to rank 0's
//     through distributed shared memory, which finds the crossing and tells the others.
#include "host_util.h"

namespace rldx {

namespace {
constexpr int kSampThreads = 512;
constexpr int kSampWarps = kSampThreads / 32;
constexpr int kSampBins = 1024;
constexpr int kSampMaxCluster = 8;
constexpr int kSampMaxSlice = 49152;     // tokens of a CTA: its sums of 16-bit halves stay below 2^32
constexpr float kSampReach = 22.5f;      // exp(-22.5) < 2^-32: weights beyond are 0
typedef unsigned long long u64;
constexpr unsigned int kErrSampleTimeout = 0x530;

struct SampleParams {
  const void* logits;
  long long ld;
  int rows, vocab, cluster;
  const float* u;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  long long* token;
  float* logprob;
  int* kept;
};

// Where a cut of the order falls: tokens whose ordered bits are above `key` stay, and the first
// `ties` (by id) of those that equal it.
struct Cut {
  uint32_t key;
  float x;
  u64 weight;  // of one tied token
  u64 before;  // count or weight of the order before them
  uint32_t ties;
};

constexpr int kSampList = 2048;   // candidates of a row
constexpr int kSampLocal = 1024;  // and of one CTA

struct SampleShared {
  union {
    struct {
      uint32_t lo[kSampBins], hi[kSampBins];  // this CTA's bins (counts in lo)
      u64 g[kSampBins];                       // rank 0: the row's
    };
    u64 list[kSampList];  // rank 0: the row's candidates, ordered bits of the logit and ~id
  };
  u64 local[kSampLocal];             // this CTA's
  u64 slots[2][kSampMaxCluster][4];  // all-gather, two phases
  u64 found[4];                      // rank 0's answer, written to every CTA
  u64 red[kSampWarps][2];
  uint32_t red32[kSampWarps];
  uint32_t flag, nlocal, nlist, base;
  uint64_t loaded;  // the bulk copy
};

__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as 0
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void red_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void red_cluster_u64(uint32_t addr, u64 v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

__device__ __forceinline__ void unpack(const uint4& u, const __nv_bfloat16*, float (&x)[8]) {
  unpack_bf16x2(u.x, x[0], x[1]);
  unpack_bf16x2(u.y, x[2], x[3]);
  unpack_bf16x2(u.z, x[4], x[5]);
  unpack_bf16x2(u.w, x[6], x[7]);
}
__device__ __forceinline__ void unpack(const uint4& u, const float*, float (&x)[4]) {
  x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
}

__device__ __forceinline__ uint32_t atom_add_cluster(uint32_t addr, uint32_t v) {
  uint32_t old;
  asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
  return old;
}

template <typename T>
struct Sampler {
  static constexpr int kVec = 16 / sizeof(T);
  SampleShared& s;
  const uint4* row;  // this CTA's vectors in shared memory
  int nvec, first_id;  // vectors held, id of the first one's first token (negative: padding)
  int rank, cluster, phase;
  float top, temp, inv;  // maximum, temperature and its reciprocal

  // ---- reductions ----
  __device__ __forceinline__ void all_gather(u64 a, u64 b, u64 c, u64 d) {  // thread 0's values, to every CTA
    phase ^= 1;
    if (threadIdx.x == 0) {
      const u64 v[4] = {a, b, c, d};
      for (int r = 0; r < cluster; ++r)
        for (int i = 0; i < 4; ++i) st_cluster_u64(mapa_shared(smem_u32(&s.slots[phase][rank][i]), r), v[i]);
    }
    cluster_sync();
  }
  __device__ __forceinline__ u64 slot(int r, int i) const { return s.slots[phase][r][i]; }

  // sum over the block, in every thread
  __device__ __forceinline__ u64 block_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5][0] = v;
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int w = 0; w < kSampWarps; ++w) t += s.red[w][0];
    return t;
  }

  // ---- tokens ----
  // d = (x - top) / temp, correctly rounded: an approximate quotient improved twice by its exact
  // remainder (Markstein's division with a rounded reciprocal), or divided where a remainder could leave
  // the normal numbers.  Below -22.2 the weight is 0: -inf.
  __device__ __forceinline__ float distance(float x) const {
    const float n = x - top;
    if (!(temp > 1e-20f && temp < 1e20f)) return x == top ? 0.0f : __fdiv_rn(n, temp);
    float q = n * inv;
    if (!(q > -22.2f)) return x == top ? 0.0f : -INFINITY;  // also: inf - inf
    q = fmaf(fmaf(-q, temp, n), inv, q);
    return fmaf(fmaf(-q, temp, n), inv, q);
  }
  __device__ __forceinline__ static u64 weight_of(float d) {
    if (!(d > -22.2f)) return 0;
    const float f = expf(d) * 4294967296.0f;
    return static_cast<u64>(__float2uint_rz(f)) + (f >= 4294967296.0f ? 1u : 0u);
  }
  __device__ __forceinline__ static bool weighs(float d) { return d > -22.17f || weight_of(d) > 0; }
  __device__ __forceinline__ static int bin_of(float d) {
    return min(kSampBins - 1, static_cast<int>(-d * (kSampBins / kSampReach)));
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int v = threadIdx.x; v < nvec; v += kSampThreads) {
      float x[kVec];
      unpack(row[v], static_cast<const T*>(nullptr), x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) f(x[e]);
    }
  }

  // ---- histogram ----
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kSampBins; i += kSampThreads) s.lo[i] = s.hi[i] = 0u;
    __syncthreads();
  }
  __device__ __forceinline__ void add(bool by_count, int bin, u64 w) {
    if (by_count) {
      atomicAdd(&s.lo[bin], 1u);
    } else {
      const uint32_t l = static_cast<uint32_t>(w) & 0xffffu, h = static_cast<uint32_t>(w >> 16);
      if (l) atomicAdd(&s.lo[bin], l);
      if (h) atomicAdd(&s.hi[bin], h);
    }
  }
  // The first bin where the running sum passes `level`; found = {bin or ~0, sum before, sum of the
  // bin, whole}.  With `share` >= 0 the level is the last one below share x whole.  rank 0's sums are
  // zero before and after.
  __device__ __forceinline__ bool crossing(u64 level, float share) {
    __syncthreads();
    const uint32_t g = mapa_shared(smem_u32(s.g), 0);
    for (int i = threadIdx.x; i < kSampBins; i += kSampThreads) {
      const u64 v = (static_cast<u64>(s.hi[i]) << 16) + s.lo[i];
      if (v) red_cluster_u64(g + 8 * i, v);
    }
    cluster_sync();
    if (rank == 0) {
      constexpr int kPer = kSampBins / kSampThreads;
      u64 w[kPer], ws = 0;
      const int b0 = threadIdx.x * kPer;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        w[i] = s.g[b0 + i];
        s.g[b0 + i] = 0;
        ws += w[i];
      }
      u64 wi = ws;  // inclusive scan
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 b = __shfl_up_sync(0xffffffffu, wi, o);
        if (lane >= o) wi += b;
      }
      if (lane == 31) s.red[warp][0] = wi;
      if (threadIdx.x == 0) s.flag = 0u;
      __syncthreads();
      u64 wb = wi - ws, whole = 0;
#pragma unroll
      for (int k = 0; k < kSampWarps; ++k) {
        if (k < warp) wb += s.red[k][0];
        whole += s.red[k][0];
      }
      if (share >= 0.0f) level = last_below(share, whole);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (wb <= level && level < wb + w[i]) {
          s.flag = 1u;
          const u64 v[4] = {static_cast<u64>(b0 + i), wb, w[i], whole};
          for (int r = 0; r < cluster; ++r)
            for (int k = 0; k < 4; ++k) st_cluster_u64(mapa_shared(smem_u32(&s.found[k]), r), v[k]);
        }
        wb += w[i];
      }
      __syncthreads();
      if (threadIdx.x == 0 && s.flag == 0u)
        for (int r = 0; r < cluster; ++r) {
          st_cluster_u64(mapa_shared(smem_u32(&s.found[0]), r), ~0ull);
          st_cluster_u64(mapa_shared(smem_u32(&s.found[3]), r), whole);
        }
    }
    cluster_sync();
    return s.found[0] != ~0ull;
  }
  // Tokens with less than `share` of `whole` before them are those with at most this before them.
  __device__ __forceinline__ static u64 last_below(float share, u64 whole) {
    const double bound = static_cast<double>(share) * static_cast<double>(whole);
    return bound > 1.0 ? static_cast<u64>(ceil(bound)) - 1 : 0;
  }

  // Finds the cut where the count (or weight) of the order passes `level` among the tokens of positive
  // weight above `from` and its ties.  With `share` >= 0 the level comes from the whole weight, which
  // is returned in *whole.  False: never.
  __device__ __forceinline__ bool find(bool by_count, u64 level, float share, const Cut& from, Cut* out, u64* whole) {
    clear();
    each([&](float x) {
      if (order_bits(x) <= from.key) return;
      const float d = distance(x);
      if (by_count) {
        if (weighs(d)) add(true, bin_of(d), 1);
      } else {
        const u64 w = weight_of(d);
        if (w) add(false, bin_of(d), w);
      }
    });
    const bool has_ties = from.ties > 0;  // the ties of the cut so far count as that many tokens
    const int tie_bin = has_ties ? bin_of(distance(from.x)) : -1;
    const u64 tie_sum = by_count ? from.ties : from.ties * from.weight;
    __syncthreads();
    if (rank == 0 && threadIdx.x == 0 && has_ties) s.g[tie_bin] += tie_sum;
    if (has_ties) cluster_sync();  // before the others add to the same bin
    const bool hit = crossing(level, share);
    *whole = s.found[3];
    if (!hit) return false;
    if (share >= 0.0f) level = last_below(share, *whole);
    const int bin = static_cast<int>(s.found[0]);
    u64 before = s.found[1], sum = s.found[2];
    // the bin's range of ordered bits
    uint32_t lo = 0xffffffffu, hi = 0u;
    // (a little more than the bin's range of quotients, before the exact look)
    const float q_hi = -bin * (kSampReach / kSampBins) * 0.9999f + 1e-6f, q_lo = -(bin + 1) * (kSampReach / kSampBins) * 1.0001f - 1e-6f;
    const bool quick = temp > 1e-20f && temp < 1e20f;
    each([&](float x) {
      const float q = (x - top) * inv;
      if (quick && (q < q_lo || q > q_hi)) return;
      const uint32_t k = order_bits(x);
      if (k <= from.key) return;
      const float d = distance(x);
      if (bin_of(d) != bin || !weighs(d)) return;
      lo = min(lo, k), hi = max(hi, k);
    });
    if (has_ties && tie_bin == bin) lo = min(lo, from.key), hi = max(hi, from.key);
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5][0] = lo, s.red[threadIdx.x >> 5][1] = hi;
    __syncthreads();
    for (int w = 0; w < kSampWarps; ++w) lo = min(lo, static_cast<uint32_t>(s.red[w][0])), hi = max(hi, static_cast<uint32_t>(s.red[w][1]));
    all_gather(lo, hi, 0, 0);
    for (int r = 0; r < cluster; ++r) lo = min(lo, static_cast<uint32_t>(slot(r, 0))), hi = max(hi, static_cast<uint32_t>(slot(r, 1)));
    while (lo != hi) {
      const int shift = max(0, 32 - __clz(hi - lo) - 10);
      clear();
      each([&](float x) {
        const uint32_t k = order_bits(x);
        if (k < lo || k > hi || k <= from.key) return;
        const float d = distance(x);
        if (weighs(d)) add(by_count, (hi - k) >> shift, by_count ? 1 : weight_of(d));
      });
      const bool tie_in = has_ties && from.key >= lo && from.key <= hi;
      __syncthreads();
      if (rank == 0 && threadIdx.x == 0 && tie_in) s.g[(hi - from.key) >> shift] += tie_sum;
      if (tie_in) cluster_sync();
      if (!crossing(level - before, -1.0f)) return false;  // (a bin holds its crossing)
      const uint32_t b = static_cast<uint32_t>(s.found[0]);
      before += s.found[1], sum = s.found[2];
      hi -= b << shift;
      const uint32_t width = (1u << shift) - 1u;
      lo = hi - lo > width ? hi - width : lo;
    }
    out->key = lo;
    out->x = order_value(lo);
    out->weight = weight_of(distance(out->x));
    out->before = before;
    out->ties = static_cast<uint32_t>(by_count ? sum : sum / out->weight);  // the caller keeps as many as fit
    return true;
  }

  // ---- a few candidates ----
  // Sorts s.list[0, n) of this CTA descending, n a power of two.
  __device__ __forceinline__ void sort(int n) {
    for (int k = 2; k <= n; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (int i = threadIdx.x; i < n / 2; i += kSampThreads) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;  // a has bit j clear
          const u64 x = s.list[a], y = s.list[b];
          if ((x < y) == ((a & k) == 0)) s.list[a] = y, s.list[b] = x;
        }
      }
    __syncthreads();
  }
  // Inclusive sum over the block of the threads' v, in thread order.
  __device__ __forceinline__ u64 block_scan(u64 v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 b = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += b;
    }
    __syncthreads();
    if (lane == 31) s.red[warp][0] = v;
    __syncthreads();
    for (int k = 0; k < warp; ++k) v += s.red[k][0];
    return v;
  }

  // The tokens that may be among the first top_k go to rank 0's list.  Returns their number (rank 0's
  // list is complete), or -1 if they are too many.
  __device__ __forceinline__ int gather_candidates(int top_k, float best) {
    // lower bound: the bin of the top_k-th largest of the threads' maxima (of pairs of tokens, where a
    // thread has one vector)
    clear();
    if (nvec <= kSampThreads) {
      if (threadIdx.x < nvec) {
        float x[kVec];
        unpack(row[threadIdx.x], static_cast<const T*>(nullptr), x);
#pragma unroll
        for (int e = 0; e < kVec; e += 2) {
          const float d = distance(fmaxf(x[e], x[e + 1]));
          if (d > -22.2f) add(true, bin_of(d), 1);
        }
      }
    } else {
      const float d = distance(best);
      if (d > -22.2f) add(true, bin_of(d), 1);
    }
    if (threadIdx.x == 0) s.nlocal = 0u, s.nlist = 0u;
    const bool hit = crossing(static_cast<u64>(top_k) - 1, -1.0f);
    const int bound = hit ? static_cast<int>(s.found[0]) : kSampBins - 1;
    // bins are cut at -d x 1024 / 22.5 in fp32: monotone in the order, so the bound's bin holds a run;
    // what lies well below it is passed over on the approximate quotient
    const float q_lo = -(bound + 1) * (kSampReach / kSampBins) * 1.0001f - 1e-6f;
    const bool quick = temp > 1e-20f && temp < 1e20f;
    for (int v = threadIdx.x; v < nvec; v += kSampThreads) {
      float x[kVec];
      unpack(row[v], static_cast<const T*>(nullptr), x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (quick && (x[e] - top) * inv < q_lo) continue;
        const float d = distance(x[e]);
        if (d > -22.2f && bin_of(d) <= bound) {
          const uint32_t at = atomicAdd(&s.nlocal, 1u);
          if (at < kSampLocal)
            s.local[at] = (static_cast<u64>(order_bits(x[e])) << 32) | static_cast<uint32_t>(~(first_id + v * kVec + e));
        }
      }
    }
    __syncthreads();
    const uint32_t n = s.nlocal;
    if (threadIdx.x == 0) s.base = atom_add_cluster(mapa_shared(smem_u32(&s.nlist), 0), n > kSampLocal ? kSampList + 1u : n);
    __syncthreads();
    const uint32_t base = s.base, list = mapa_shared(smem_u32(s.list), 0);
    if (n <= kSampLocal && base + n <= kSampList)
      for (uint32_t i = threadIdx.x; i < n; i += kSampThreads) st_cluster_u64(list + 8 * (base + i), s.local[i]);
    cluster_sync();
    // everyone has to know: rank 0 tells
    if (rank == 0 && threadIdx.x == 0)
      for (int r = 0; r < cluster; ++r) st_cluster_u64(mapa_shared(smem_u32(&s.found[0]), r), s.nlist);
    cluster_sync();
    return s.found[0] <= kSampList ? static_cast<int>(s.found[0]) : -1;
  }
};

// The whole draw from rank 0's n candidates, which contain the first top_k tokens of positive weight.
template <typename T>
__device__ __forceinline__ void draw_from_list(Sampler<T>& S, const SampleParams& P, int r, int n, int top_k, float top_p,
                                               u64 least) {
  SampleShared& s = S.s;
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kSampThreads) s.list[i] = 0;
  S.sort(size);
  n = min(n, top_k);
  // four consecutive places of the order a thread
  constexpr int kPer = kSampList / kSampThreads;
  auto weight_at = [&](int i) -> u64 {
    return i < n ? Sampler<T>::weight_of(S.distance(order_value(static_cast<uint32_t>(s.list[i] >> 32)))) : 0;
  };
  u64 w[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum += w[i] = weight_at(kPer * threadIdx.x + i);
  const u64 inc = S.block_scan(sum);
  __syncthreads();
  if (threadIdx.x == kSampThreads - 1) s.found[0] = inc;
  if (threadIdx.x == 0) s.nlist = 0u;
  __syncthreads();
  const u64 level = top_p < 1.0f ? Sampler<T>::last_below(fmaxf(top_p, 0.0f), s.found[0]) : ~0ull;
  u64 before = inc - sum;
  uint32_t mine = 0;
  u64 kept_sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (w[i] > 0 && before <= level && w[i] >= least) ++mine, kept_sum += w[i];
    before += w[i];
  }
  mine = __reduce_add_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) atomicAdd(&s.nlist, mine);
  kept_sum = S.block_sum(kept_sum);  // (its barriers also order nlist)
  const int kept = static_cast<int>(s.nlist);  // a prefix of the order
  // the kept ones by id
  size = 2;
  while (size < kept) size <<= 1;
  __syncthreads();
  for (int i = threadIdx.x; i < size; i += kSampThreads)
    s.list[i] = i < kept ? (s.list[i] << 32) | (s.list[i] >> 32) : 0;  // ~id, ordered bits: descending is ascending id
  S.sort(size);
  n = kept;
  sum = 0;
  auto weight_by_id = [&](int i) -> u64 {
    return i < n ? Sampler<T>::weight_of(S.distance(order_value(static_cast<uint32_t>(s.list[i])))) : 0;
  };
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum += w[i] = weight_by_id(kPer * threadIdx.x + i);
  before = S.block_scan(sum) - sum;
  const double target = static_cast<double>(P.u[r]) * static_cast<double>(kept_sum);
  u64 goal = target > 0.0 ? static_cast<u64>(target) : 0;
  if (goal >= kept_sum) goal = kept_sum - 1;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (before <= goal && goal < before + w[i]) {
      P.token[r] = static_cast<int>(~static_cast<uint32_t>(s.list[kPer * threadIdx.x + i] >> 32));
      P.logprob[r] = static_cast<float>(log(static_cast<double>(w[i]) / static_cast<double>(kept_sum)));
      P.kept[r] = kept;
    }
    before += w[i];
  }
}

template <typename T>
__global__ void __launch_bounds__(kSampThreads, 2) sample_kernel(const __grid_constant__ SampleParams P) {
  constexpr int kVec = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(smem_raw);
  uint4* vecs = reinterpret_cast<uint4*>(smem_raw + (sizeof(SampleShared) + 15) / 16 * 16);
  const int rank = static_cast<int>(cluster_ctarank()), cluster = P.cluster;
  const int r = blockIdx.x / cluster;
  // another CTA's shared memory may be written only once that CTA runs: wait for this below
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  griddep_wait();
  griddep_launch();

  // ---- this CTA's share of the row: whole 16-byte vectors of memory, by one bulk copy; the edges
  // with tokens outside the row as -inf ----
  const T* src = static_cast<const T*>(P.logits) + r * P.ld;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));
  const int all = (P.vocab + mis + kVec - 1) / kVec, per = (all + cluster - 1) / cluster;
  const int v0 = min(all, rank * per), nvec = min(all, v0 + per) - v0;
  const int first_id = v0 * kVec - mis;
  const int head = first_id < 0 ? 1 : 0, tail = first_id + nvec * kVec > P.vocab ? 1 : 0;
  const int whole_vecs = max(0, nvec - head - tail);
  if (threadIdx.x == 0) {
    mbar_init(&s.loaded, 1);
    fence_mbar_init();
    mbar_arrive_expect_tx(&s.loaded, whole_vecs * 16);
    if (whole_vecs > 0) bulk_load(vecs + head, src + first_id + head * kVec, whole_vecs * 16, &s.loaded, l2_policy_evict_first());
  }
  if (threadIdx.x < 2 && nvec > 0 && (threadIdx.x == 0 ? head : tail)) {
    const int v = threadIdx.x == 0 ? 0 : nvec - 1;
    T* e = reinterpret_cast<T*>(vecs + v);
#pragma unroll 1
    for (int i = 0; i < kVec; ++i) {
      const int id = first_id + v * kVec + i;
      e[i] = (id >= 0 && id < P.vocab) ? src[id] : static_cast<T>(-INFINITY);
    }
  }
  for (int i = threadIdx.x; i < kSampBins; i += kSampThreads) s.g[i] = 0;
  Sampler<T> S{s, vecs, nvec, first_id, rank, cluster, 0, 0.0f, 0.0f, 0.0f};
  __syncthreads();  // the barrier is set up, the edges are written
  const bool ok = mbar_wait(&s.loaded, 0u, kErrSampleTimeout);
  // ---- maximum (NaN is passed over here and weighs nothing below) and, for a greedy row, its first id ----
  float best = -INFINITY;
  S.each([&](float x) { best = fmaxf(best, x); });
  const float temp = P.temperature ? P.temperature[r] : 1.0f;
  const bool greedy = !(temp > 0.0f);
  const uint32_t mine = order_bits(best);
  uint32_t m = __reduce_max_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) s.red32[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int w = 0; w < kSampWarps; ++w) m = max(m, s.red32[w]);
  uint32_t id = 0x7fffffffu;
  if (greedy) {
    const float top = order_value(m);
    if (mine == m)
      for (int v = threadIdx.x; v < nvec && id == 0x7fffffffu; v += kSampThreads) {
        float x[kVec];
        unpack(vecs[v], static_cast<const T*>(nullptr), x);
#pragma unroll
        for (int i = kVec - 1; i >= 0; --i)
          if (x[i] == top) id = first_id + v * kVec + i;
      }
    id = __reduce_min_sync(0xffffffffu, id);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red32[threadIdx.x >> 5] = id;
    __syncthreads();
    for (int w = 0; w < kSampWarps; ++w) id = min(id, s.red32[w]);
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  S.all_gather((static_cast<u64>(m) << 32) | static_cast<uint32_t>(~id), ok ? 0u : 1u, 0, 0);
  u64 first = 0, failed = 0;
  for (int k = 0; k < cluster; ++k) first = max(first, S.slot(k, 0)), failed |= S.slot(k, 1);
  m = static_cast<uint32_t>(first >> 32);
  S.top = order_value(m);
  const bool empty = S.top == -INFINITY;
  if (greedy || empty || failed) {  // failed: the copy's wait ran out, in whichever CTA
    if (!ok) settle_issued_copies();
    if (rank == 0 && threadIdx.x == 0) {
      P.token[r] = empty || failed ? -1 : static_cast<long long>(~static_cast<uint32_t>(first));
      P.logprob[r] = empty || failed ? -INFINITY : 0.0f;
      P.kept[r] = empty || failed ? 0 : 1;
    }
    return;  // nothing was written to another CTA since the last barrier
  }
  S.temp = fmaxf(temp, 1e-30f);
  S.inv = __fdiv_rn(1.0f, S.temp);

  const int top_k = P.top_k ? P.top_k[r] : 0;
  const float top_p = P.top_p ? P.top_p[r] : 1.0f;
  const float min_p = P.min_p ? P.min_p[r] : 0.0f;
  // w >= min_p 2^32 for whole w
  const u64 least = static_cast<u64>(ceil(static_cast<double>(min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f) * 4294967296.0));
  Cut cut{};  // below every logit
  cut.key = order_bits(-INFINITY);
  cut.x = -INFINITY;
  if (top_k > 0 && top_k < P.vocab) {
    // the list holds what the bound lets through, a little more than top_k
    const int n = top_k <= kSampList * 3 / 4 ? S.gather_candidates(top_k, best) : -1;
    if (n >= 0) {
      if (rank == 0) draw_from_list(S, P, r, n, top_k, top_p, least);
      return;  // rank 0 needs nothing more of the others
    }
    if (rank == 0) {  // the list stood where the sums are
      __syncthreads();
      for (int i = threadIdx.x; i < kSampBins; i += kSampThreads) s.g[i] = 0;
    }
    cluster_sync();
    Cut c;
    u64 whole;
    if (S.find(true, static_cast<u64>(top_k) - 1, -1.0f, cut, &c, &whole)) {
      c.ties = min(c.ties, static_cast<uint32_t>(static_cast<u64>(top_k) - c.before));
      cut = c;
    }
  }
  if (top_p < 1.0f) {
    Cut c;
    u64 whole;
    if (S.find(false, 0, top_p > 0.0f ? top_p : 0.0f, cut, &c, &whole)) {
      const u64 fit = (Sampler<T>::last_below(top_p > 0.0f ? top_p : 0.0f, whole) - c.before) / c.weight + 1;
      c.ties = static_cast<uint32_t>(min(static_cast<u64>(c.ties), fit));
      cut = c;
    }
  }
  const u64 tie_weight = (cut.ties > 0 && cut.weight >= least) ? cut.weight : 0;
  const uint32_t ties = tie_weight ? cut.ties : 0;
  auto kept_weight = [&](float x) -> u64 {  // of a token above the cut
    if (order_bits(x) <= cut.key) return 0;
    const u64 w = Sampler<T>::weight_of(S.distance(x));
    return w >= least ? w : 0;
  };

  // ---- sums of the CTA: weight and count above the cut, ties ----
  u64 w = 0;
  uint32_t n = 0, nt = 0;
  S.each([&](float x) {
    const u64 k = kept_weight(x);
    w += k;
    n += k > 0;
    nt += order_bits(x) == cut.key;
  });
  w = S.block_sum(w);
  const u64 nn = S.block_sum((static_cast<u64>(n) << 32) | nt);
  S.all_gather(w, nn, 0, 0);
  u64 sum = 0, count = 0;
  for (int k = 0; k < cluster; ++k) sum += S.slot(k, 0), count += S.slot(k, 1) >> 32;
  sum += static_cast<u64>(ties) * tie_weight;
  count += ties;
  const double target = static_cast<double>(P.u[r]) * static_cast<double>(sum);
  u64 goal = target > 0.0 ? static_cast<u64>(target) : 0;
  if (goal >= sum) goal = sum - 1;
  // inclusive sum after a token: weight above the cut + tie_weight * min(ties, tied tokens so far)
  u64 wb = 0;
  uint32_t tb = 0;
  int owner = 0;
  for (; owner < cluster - 1; ++owner) {
    const u64 w1 = wb + S.slot(owner, 0);
    const uint32_t t1 = tb + static_cast<uint32_t>(S.slot(owner, 1));
    if (w1 + static_cast<u64>(min(ties, t1)) * tie_weight > goal) break;
    wb = w1, tb = t1;
  }
  if (rank == owner) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int base = 0; base < nvec; base += kSampThreads) {
      const int v = base + threadIdx.x;
      float x[kVec];
      u64 ws = 0;
      uint32_t ts = 0;
      if (v < nvec) {
        unpack(vecs[v], static_cast<const T*>(nullptr), x);
#pragma unroll
        for (int e = 0; e < kVec; ++e) ws += kept_weight(x[e]), ts += order_bits(x[e]) == cut.key;
      }
      u64 wi = ws;
      uint32_t ti = ts;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 a = __shfl_up_sync(0xffffffffu, wi, o);
        const uint32_t b = __shfl_up_sync(0xffffffffu, ti, o);
        if (lane >= o) wi += a, ti += b;
      }
      __syncthreads();
      if (lane == 31) s.red[warp][0] = wi, s.red[warp][1] = ti;
      __syncthreads();
      u64 pw = wb;
      uint32_t pt = tb;
      for (int k = 0; k < kSampWarps; ++k) {
        if (k == warp) wi += pw, ti += pt;
        pw += s.red[k][0], pt += static_cast<uint32_t>(s.red[k][1]);
      }
      const u64 before = wi - ws + static_cast<u64>(min(ties, ti - ts)) * tie_weight;
      const u64 after = wi + static_cast<u64>(min(ties, ti)) * tie_weight;
      if (v < nvec && before <= goal && goal < after) {
        u64 cw = wi - ws;
        uint32_t ct = ti - ts;
        bool done = false;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const u64 k = kept_weight(x[e]);
          const bool tie = order_bits(x[e]) == cut.key;
          cw += k, ct += tie;
          if (!done && cw + static_cast<u64>(min(ties, ct)) * tie_weight > goal) {
            done = true;
            P.token[r] = first_id + v * kVec + e;
            P.logprob[r] = static_cast<float>(log(static_cast<double>(tie ? tie_weight : k) / static_cast<double>(sum)));
            P.kept[r] = static_cast<int>(count);
          }
        }
      }
      wb = pw, tb = pt;
      if (wb + static_cast<u64>(min(ties, tb)) * tie_weight > goal) break;
    }
  }
  cluster_sync();
}

template <typename T>
size_t sample_smem(int vocab, int cluster) {
  const int kVec = 16 / sizeof(T);
  const int per = ((vocab + kVec - 1 + kVec - 1) / kVec + cluster - 1) / cluster;
  return (sizeof(SampleShared) + 15) / 16 * 16 + static_cast<size_t>(per) * 16;
}

template <typename T>
cudaError_t launch_sample(const SampleParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows * p.cluster), 1, 1);
  cfg.blockDim = dim3(kSampThreads, 1, 1);
  cfg.dynamicSmemBytes = sample_smem<T>(p.vocab, p.cluster);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, p);
}
}  // namespace

constexpr int kSampSmemMax = 220 * 1024;

cudaError_t sample_prepare_device() {
  cudaError_t e = cudaFuncSetAttribute(sample_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampSmemMax);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(sample_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampSmemMax);
  return e;
}

}  // namespace rldx

using namespace rldx;

extern "C" int rldx_sample(const void* logits, int64_t ld, int rows, int vocab, int logits_fp32, const float* u,
                           const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                           int64_t* token, float* logprob, int32_t* kept, void* stream) {
  int rc = ensure_device();
  if (rc != RLDX_OK) return rc;
  if (rows < 0 || vocab <= 0 || ld < vocab) return set_error(RLDX_ERR_ARG, "sample: need rows >= 0, vocab > 0, ld >= vocab");
  if (vocab > kSampMaxCluster * kSampMaxSlice)
    return set_error(RLDX_ERR_UNSUPPORTED, "sample: a vocabulary has at most " + std::to_string(kSampMaxCluster * kSampMaxSlice) + " tokens");
  if (rows == 0) return RLDX_OK;
  if (!logits || !u || !token || !logprob || !kept) return set_error(RLDX_ERR_ARG, "sample: null pointer");
  if (reinterpret_cast<uintptr_t>(logits) % (logits_fp32 ? 4 : 2)) return set_error(RLDX_ERR_ARG, "sample: misaligned logits");
  if (static_cast<long long>(rows) * kSampMaxCluster >= (1LL << 31)) return set_error(RLDX_ERR_UNSUPPORTED, "sample: too many rows");
  SampleParams p;
  p.logits = logits;
  p.ld = ld;
  p.rows = rows;
  p.vocab = vocab;
  p.cluster = 1;
  while (p.cluster < kSampMaxCluster && vocab / p.cluster > 4096) p.cluster *= 2;
  p.u = u;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.token = reinterpret_cast<long long*>(token);
  p.logprob = logprob;
  p.kept = kept;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = logits_fp32 ? launch_sample<float>(p, st) : launch_sample<__nv_bfloat16>(p, st);
  if (e != cudaSuccess) return cuda_fail(e, "sample launch");
  return RLDX_OK;
}
