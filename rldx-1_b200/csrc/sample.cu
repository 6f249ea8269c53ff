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
// A cluster of CTAs holds a row in shared memory, so the logits are read once (one bulk copy a CTA).
// The last token kept is found in one of two ways:
//   - top-k up to 1536: each CTA finds, by bins, a value that the k / CTAs largest of its threads' maxima (four
//     a thread) reach; the least of these is a lower bound of the k-th largest logit.  The tokens that reach
//     it, a little more than k, go to rank 0's list, and the other CTAs are done.  Up to 192 are compared
//     with one another, a thread each; of more rank 0 finds the cut as below and draws by bins of ids.
//   - otherwise by histogram: 1024 bins linear in -d (every bin holds a run of the order), then by the
//     ordered bits of the logit (16 of bf16) inside the bin where count or weight crosses, until one value is left;
//     of the tokens that share it the first few by id stay.  Bins hold counts (top-k) or weights
//     (top-p: the low 16 and high 17 bits of a weight in two 32-bit sums); CTAs add theirs to rank 0's
//     through distributed shared memory, which finds the crossing and tells the others.
//
// Measured, bf16 rows of 151680, 1 row / 256 rows in us: greedy 3.0 / 21 (78 MB: 12 at the copy's rate), top-k 20
// 7.9 / 43, top-k 1000 15.5 / 77, top-k 3000 (by histogram) 23 / 160, temperature alone 11.4 / 82, top-p 0.9 at
// T = 1, 28914 kept, 26.3 / 193.  Few rows wait on the chain of passes and cluster barriers, and so do
// many: with mixed filters barriers and the fences beside them lead the stalls (2.7 and 1.1 of an issue's), DRAM is at 11
// % and the busiest unit of an SM at 36 %.  Rows drawn from the list keep one CTA of a cluster after the gather, so top-k
// 20 takes twice a greedy row; flat rows add a correctly rounded quotient and exponential a token and pass
// (about 40 instructions) and the histogram's atomics.
#include <cfloat>

#include "host_util.h"
#include "rows.cuh"

namespace rldx {

namespace {
constexpr int kSampBins = 1024;
constexpr int kSampMaxCluster = 8;
constexpr int kSampMaxSlice = 49152;  // tokens of a CTA: its sums of 16-bit halves stay below 2^32
constexpr float kSampReach = 22.5f;   // of the bins; exp(-22.2) < 2^-32: weights beyond are 0
constexpr int kSampList = 2048;       // candidates of a row
// Candidates that a thread each compares with all; more go through bins.  The limit at 128 / 256, us: 1 row of
// 151680, top-k 80 13.9 / 11.2, 100 15.4 / 12.0, 160 15.6 / 14.9; 256 rows 58.7 / 56.1, 63.3 / 64.6, 65.8 / 77.4.
constexpr int kSampFew = 192;
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

// Where a cut of the order falls: tokens above x stay, and the first `ties` (by id) of those that equal it.
struct Cut {
  float x;
  uint32_t ties;
  u64 weight;  // of one tied token
  u64 before;  // count or weight of the order before them
};

struct SampleShared {
  union {
    struct {
      uint32_t lo[kSampBins], hi[kSampBins];  // this CTA's bins (counts in lo)
      u64 g[kSampBins];                       // rank 0: the row's
    };
    u64 list[kSampList];  // rank 0: the row's candidates, ordered bits of the logit and ~id
  };
  u64 slots[2][kSampMaxCluster][2];  // all-gather, two phases
  u64 found[4];                      // rank 0's answer, written to every CTA
  u64 red[32][2];
  u64 warps[16][2];  // sums of a warp's vectors
  uint32_t red32[32];
  uint32_t flag, count;
  uint64_t loaded;  // the bulk copy
};

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
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
// The larger ones of two vectors, halves of a word apart (NaN gives way to any number).
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Four running maxima of a thread: of bf16 as two words.
struct MaximaBf16 {
  uint32_t a = 0xff80ff80u, b = 0xff80ff80u;  // -inf
  __device__ __forceinline__ void add(const uint4& u) {
    a = max_bf16x2(a, max_bf16x2(u.x, u.y));
    b = max_bf16x2(b, max_bf16x2(u.z, u.w));
  }
  __device__ __forceinline__ void get(float (&x)[4]) const { unpack_bf16x2(a, x[0], x[1]), unpack_bf16x2(b, x[2], x[3]); }
};
struct MaximaFloat {
  float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  __device__ __forceinline__ void add(const uint4& u) {
    x[0] = fmaxf(x[0], __uint_as_float(u.x)), x[1] = fmaxf(x[1], __uint_as_float(u.y));
    x[2] = fmaxf(x[2], __uint_as_float(u.z)), x[3] = fmaxf(x[3], __uint_as_float(u.w));
  }
  __device__ __forceinline__ void get(float (&y)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = x[i];
  }
};
template <typename T>
struct MaximaOf {
  using Type = MaximaBf16;
};
template <>
struct MaximaOf<float> {
  using Type = MaximaFloat;
};
__device__ __forceinline__ void unpack(const uint4& u, const float*, float (&x)[4]) {
  x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
}

// The order of the logits of a type: bf16 has 16 bits of it.
template <typename T>
__device__ __forceinline__ uint32_t key_bits(float x) {
  return order_bits(x) >> (sizeof(T) == 2 ? 16 : 0);
}
template <typename T>
__device__ __forceinline__ float key_float(uint32_t k) {
  return sizeof(T) == 2 ? order_value((k << 16) | ((k >> 15) ? 0u : 0xffffu)) : order_value(k);
}

// NT threads of one CTA of a row's cluster.
template <typename T, int NT>
struct Sampler {
  static constexpr int kVec = 16 / sizeof(T);
  static constexpr int kWarps = NT / 32;
  SampleShared& s;
  const uint4* row;    // this CTA's vectors in shared memory
  int nvec, first_id;  // vectors held, id of the first one's first token (negative: padding)
  int rank, cluster, phase;
  float top, temp, inv, scale;  // maximum; scaled temperature, its reciprocal and the scale
  float floor;                  // tokens below weigh 0

  __device__ __forceinline__ void load(int v, float (&x)[kVec]) const { unpack(row[v], static_cast<const T*>(nullptr), x); }
  __device__ __forceinline__ static uint32_t key_of(float x) { return key_bits<T>(x); }
  __device__ __forceinline__ static float key_value(uint32_t k) { return key_float<T>(k); }
  __device__ __forceinline__ static float largest(const uint4& u) {
    typename MaximaOf<T>::Type maxima;
    float x[4];
    maxima.add(u);
    maxima.get(x);
    return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  }
  // The tokens of the vectors that hold one of at least `least`.
  template <typename F>
  __device__ __forceinline__ void each(float least, F f) const {
    for (int v = threadIdx.x; v < nvec; v += NT) {
      const uint4 u = row[v];
      if (!(largest(u) >= least)) continue;
      float x[kVec];
      unpack(u, static_cast<const T*>(nullptr), x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) f(x[e]);
    }
  }

  // ---- reductions ----
  __device__ __forceinline__ void all_gather(u64 a, u64 b) {  // thread 0's values, to every CTA
    phase ^= 1;
    if (threadIdx.x < cluster) {
      const uint32_t at = mapa_shared(smem_u32(&s.slots[phase][rank][0]), threadIdx.x);
      st_cluster_u64(at, a);
      st_cluster_u64(at + 8, b);
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
    for (int w = 0; w < kWarps; ++w) t += s.red[w][0];
    return t;
  }
  // inclusive sums over the block of (a, b), in thread order; *all_a, *all_b: of the block
  __device__ __forceinline__ void block_scan(u64& a, u64& b, u64* all_a, u64* all_b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) a += x, b += y;
    }
    __syncthreads();
    if (lane == 31) s.red[warp][0] = a, s.red[warp][1] = b;
    __syncthreads();
    *all_a = *all_b = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      if (k == warp) a += *all_a, b += *all_b;
      *all_a += s.red[k][0], *all_b += s.red[k][1];
    }
  }

  // ---- tokens ----
  // d = (x - top) / temp, correctly rounded: an approximate quotient improved twice by its exact
  // remainder (Markstein's division with a rounded reciprocal); both sides are scaled by a power of two
  // that keeps the remainders normal numbers.  -inf and NaN logits, and quotients that overflow, give NaN
  // or -inf, which weighs 0 below.
  __device__ __forceinline__ float distance(float x) const {
    const float n = (x - top) * scale;
    const float q0 = n * inv, q1 = fmaf(fmaf(-q0, temp, n), inv, q0);
    return fmaf(fmaf(-q1, temp, n), inv, q1);
  }
  // The weight, with 2^32 - 1 for 2^32 (exponentials below 1 give at most 2^32 - 256); 0 for NaN.
  __device__ __forceinline__ static uint32_t weight32(float d) { return __float2uint_rz(expf(d) * 4294967296.0f); }
  __device__ __forceinline__ static u64 widen(uint32_t t) { return static_cast<u64>(t) + (t == 0xffffffffu ? 1u : 0u); }
  __device__ __forceinline__ static u64 weight_of(float d) { return widen(weight32(d)); }
  __device__ __forceinline__ u64 weight(float x) const { return weight_of(distance(x)); }
  __device__ __forceinline__ static bool weighs(float d) { return d > -22.17f || (d > -22.2f && weight_of(d) > 0); }
  __device__ __forceinline__ static int bin_of(float d) {
    return min(kSampBins - 1, static_cast<int>(-d * (kSampBins / kSampReach)));
  }

  // ---- histogram ----
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kSampBins; i += NT) s.lo[i] = s.hi[i] = 0u;
    __syncthreads();
  }
  __device__ __forceinline__ void add_weight(int bin, uint32_t t) {  // (2^32 - 1 is 2^32)
    const bool full = t == 0xffffffffu;
    const uint32_t l = full ? 0u : t & 0xffffu, h = full ? 0x10000u : t >> 16;
    if (l) atomicAdd(&s.lo[bin], l);
    if (h) atomicAdd(&s.hi[bin], h);
  }
  // Tokens with less than `share` of `whole` before them are those with at most this before them.
  __device__ __forceinline__ static u64 last_below(float share, u64 whole) {
    const double bound = static_cast<double>(share) * static_cast<double>(whole);
    return bound > 1.0 ? static_cast<u64>(ceil(bound)) - 1 : 0;
  }
  __device__ __forceinline__ u64 bin_sum(int i) const { return (static_cast<u64>(s.hi[i]) << 16) + s.lo[i]; }
  // One thread of rank 0 writes `found`, of every CTA or (kAlone) its own.
  template <bool kAlone>
  __device__ __forceinline__ void tell(const u64 (&v)[4]) {
    if constexpr (kAlone) {
#pragma unroll
      for (int k = 0; k < 4; ++k) s.found[k] = v[k];
    } else {
      for (int r = 0; r < cluster; ++r)
#pragma unroll
        for (int k = 0; k < 4; ++k) st_cluster_u64(mapa_shared(smem_u32(&s.found[k]), r), v[k]);
    }
  }
  // The first bin where the running sum passes `level`; found = {bin or ~0, sum before, sum of the
  // bin, whole}.  With `share` >= 0 the level is the last one below share x whole.  rank 0's sums are
  // zero before and after.
  // kAlone: rank 0 works without the others.
  template <bool kAlone>
  __device__ __forceinline__ bool crossing(u64 level, float share) {
    __syncthreads();
    if constexpr (!kAlone) {
      const uint32_t g = mapa_shared(smem_u32(s.g), 0);
      for (int i = threadIdx.x; i < kSampBins; i += NT) {
        const u64 v = bin_sum(i);
        if (v) red_cluster_u64(g + 8 * i, v);
      }
      cluster_sync();
    }
    if (rank == 0) {
      constexpr int kPer = kSampBins / NT;
      u64 w[kPer], ws = 0;
      const int b0 = threadIdx.x * kPer;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        w[i] = s.g[b0 + i] + (kAlone ? bin_sum(b0 + i) : 0);
        s.g[b0 + i] = 0;
        ws += w[i];
      }
      if (threadIdx.x == 0) s.flag = 0u;
      u64 wi = ws, none = 0, whole, other;
      block_scan(wi, none, &whole, &other);
      u64 wb = wi - ws;
      if (share >= 0.0f) level = last_below(share, whole);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (wb <= level && level < wb + w[i]) {
          s.flag = 1u;
          const u64 v[4] = {static_cast<u64>(b0 + i), wb, w[i], whole};
          tell<kAlone>(v);
        }
        wb += w[i];
      }
      __syncthreads();
      if (threadIdx.x == 0 && s.flag == 0u) {
        const u64 v[4] = {~0ull, 0, 0, whole};
        tell<kAlone>(v);
      }
    }
    if constexpr (kAlone)
      __syncthreads();
    else
      cluster_sync();
    return s.found[0] != ~0ull;
  }

  // Finds the cut where the count (or weight) of the order passes `level` among the tokens of positive
  // weight above `from` and its ties.  With `share` >= 0 the level comes from the whole weight, which
  // is returned in *whole.  False: never.  `each` visits the CTA's tokens, those of at least its first argument.
  template <bool kAlone, typename Each>
  __device__ __forceinline__ bool find(Each each, bool by_count, u64 level, float share, const Cut& from, Cut* out, u64* whole) {
    clear();
    each(fmaxf(floor, from.x), [&](float x) {
      const float d = distance(x);
      if (!by_count)
        add_weight(bin_of(d), x > from.x ? weight32(d) : 0u);
      else if (x > from.x && weighs(d))
        atomicAdd(&s.lo[bin_of(d)], 1u);
    });
    const bool has_ties = from.ties > 0;  // the ties of the cut so far count as that many tokens
    const int tie_bin = has_ties ? bin_of(distance(from.x)) : -1;
    const u64 tie_sum = by_count ? from.ties : from.ties * from.weight;
    __syncthreads();
    if (rank == 0 && threadIdx.x == 0 && has_ties) s.g[tie_bin] += tie_sum;
    if (has_ties && !kAlone) cluster_sync();  // before the others add to the same bin
    const bool hit = crossing<kAlone>(level, share);
    *whole = s.found[3];
    if (!hit) return false;
    if (share >= 0.0f) level = last_below(share, *whole);
    const int bin = static_cast<int>(s.found[0]);
    u64 before = s.found[1], sum = s.found[2];
    // keys that hold the bin's tokens, and a little more than them
    const float span = scale == 1.0f ? temp : temp / scale, slack = fabsf(top) * 0x1p-20f;
    const float x_min = top - (bin + 1) * (kSampReach / kSampBins) * span * 1.0001f - slack;
    const float x_max = fminf(top, top - bin * (kSampReach / kSampBins) * span * 0.9999f + slack);
    uint32_t lo = key_of(fmaxf(x_min, -FLT_MAX)), hi = key_of(fmaxf(x_max, -FLT_MAX));
    const uint32_t from_key = key_of(from.x);
    while (lo != hi) {
      const int shift = max(0, 32 - __clz(hi - lo) - 10);
      const float x_lo = key_value(lo), x_hi = key_value(hi);
      clear();
      each(x_lo, [&](float x) {
        if (!(x >= x_lo && x <= x_hi && x > from.x)) return;
        const float d = distance(x);
        if (!weighs(d) || bin_of(d) != bin) return;
        const int b = static_cast<int>((hi - key_of(x)) >> shift);
        if (by_count)
          atomicAdd(&s.lo[b], 1u);
        else
          add_weight(b, weight32(d));
      });
      const bool tie_in = has_ties && tie_bin == bin && from_key >= lo && from_key <= hi;
      __syncthreads();
      if (rank == 0 && threadIdx.x == 0 && tie_in) s.g[(hi - from_key) >> shift] += tie_sum;
      if (tie_in && !kAlone) cluster_sync();
      if (!crossing<kAlone>(level - before, -1.0f)) return false;  // (a bin holds its crossing)
      const uint32_t b = static_cast<uint32_t>(s.found[0]);
      before += s.found[1], sum = s.found[2];
      hi -= b << shift;
      const uint32_t width = (1u << shift) - 1u;
      lo = hi - lo > width ? hi - width : lo;
    }
    out->x = key_value(lo);
    out->weight = weight(out->x);
    out->before = before;
    out->ties = static_cast<uint32_t>(by_count ? sum : sum / out->weight);  // find_cut keeps as many as fit
    return true;
  }
  // The cut of top_k (0: off), then of top_p.
  template <bool kAlone, typename Each>
  __device__ __forceinline__ Cut find_cut(Each each, int top_k, float top_p) {
    Cut cut{}, c;  // below every logit
    cut.x = -INFINITY;
    u64 whole;
    const float share = fmaxf(top_p, 0.0f);
#pragma unroll 1
    for (int by_weight = top_k > 0 ? 0 : 1; by_weight < (top_p < 1.0f ? 2 : 1); ++by_weight) {  // (one copy of the code)
      const u64 last = static_cast<u64>(top_k) - 1;
      if (!find<kAlone>(each, !by_weight, last, by_weight ? share : -1.0f, cut, &c, &whole)) continue;
      const u64 fit = by_weight ? (last_below(share, whole) - c.before) / c.weight + 1 : static_cast<u64>(top_k) - c.before;
      c.ties = static_cast<uint32_t>(min(static_cast<u64>(c.ties), fit));
      cut = c;
    }
    return cut;
  }

  // ---- a few candidates ----
  // A value that at least `want` of the CTA's tokens reach, from the threads' four maxima each in bins of the
  // distance from the CTA's largest; or, if these do not show so many, one below which every token weighs 0.
  __device__ __forceinline__ float reached_by(int want, const float (&best)[4], float most, float t) {
    constexpr int kBins = 256;
    const int i = threadIdx.x, lane = i & 31, warp = i >> 5;
    if (i < kBins) s.lo[i] = 0u;
    if (i == 0) s.flag = kBins - 1;
    __syncthreads();
    const float per = kBins / (kSampReach * t);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float q = best[e] == most ? 0.0f : (most - best[e]) * per;
      if (q < kBins) atomicAdd(&s.lo[static_cast<int>(q)], 1u);
    }
    __syncthreads();
    const int n = i < kBins ? s.lo[i] : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s.red32[warp] = upto;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kBins / 32; ++w) upto += w < warp ? s.red32[w] : 0;
    if (i < kBins && upto - n < want && want <= upto) s.flag = i;
    __syncthreads();
    return most - (s.flag + 1) / per * 1.0001f - fabsf(most) * 0x1p-20f;  // a little below the bin
  }

  // The tokens that reach `bound` go to rank 0's list, in any order.  Returns their number, or -1 if they are
  // too many.
  __device__ __forceinline__ int gather_candidates(float bound) {
    if (threadIdx.x == 0) s.count = 0u;
    __syncthreads();
    for (int v = threadIdx.x; v < nvec; v += NT) {
      const uint4 u = row[v];
      if (!(largest(u) >= bound)) continue;
      float x[kVec];
      unpack(u, static_cast<const T*>(nullptr), x);
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (x[e] >= bound && x[e] > -INFINITY) {
          const uint32_t at = atomicAdd(&s.count, 1u);
          if (at < kSampList) s.list[at] = (static_cast<u64>(order_bits(x[e])) << 32) | static_cast<uint32_t>(~(first_id + v * kVec + e));
        }
    }
    __syncthreads();
    const uint32_t mine = s.count;
    all_gather(mine, 0);
    u64 base = 0, total = 0;
    for (int r = 0; r < cluster; ++r) {
      if (r < rank) base += slot(r, 0);
      total += slot(r, 0);
    }
    if (total > kSampList) {  // rank 0's part may have run into the row's bins
      if (rank == 0)
        for (int i = threadIdx.x; i < kSampBins; i += NT) s.g[i] = 0;
      cluster_sync();
      return -1;
    }
    if (rank > 0) {  // rank 0's stand where they are
      const uint32_t at = mapa_shared(smem_u32(s.list), 0) + 8 * static_cast<uint32_t>(base);
      for (uint32_t i = threadIdx.x; i < mine; i += NT) st_cluster_u64(at + 8 * i, s.list[i]);
    }
    cluster_sync();
    return static_cast<int>(total);
  }

  // The whole draw by rank 0 from its n <= kSampFew candidates, which contain the first top_k tokens of positive
  // weight: thread i takes candidate i and compares it with all.
  __device__ __forceinline__ void draw_from_few(const SampleParams& P, int r, int n, int top_k, float top_p, u64 least) {
    u64* ws = s.list + kSampFew;  // weights
    const int i = threadIdx.x;
    const u64 mine = i < n ? s.list[i] : 0;
    const u64 w = i < n ? weight(order_value(static_cast<uint32_t>(mine >> 32))) : 0;
    if (i < n) ws[i] = w;
    __syncthreads();
    u64 before = 0;  // in the order
    int place = 0;
    if (i < n) {
#pragma unroll 4
      for (int k = 0; k < n; ++k)
        if (s.list[k] > mine) before += ws[k], ++place;
      if (place == min(n, top_k) - 1) s.found[0] = before + w;  // what top-k left
    }
    __syncthreads();
    const u64 level = top_p < 1.0f ? last_below(fmaxf(top_p, 0.0f), s.found[0]) : ~0ull;
    if (i < n && !(place < top_k && before <= level && w >= least)) ws[i] = 0;
    __syncthreads();
    if (i < n && ws[i] > 0) {
      u64 sum = 0, kept = 0;
      before = 0;  // in the order of ids (the low word is ~id)
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const u64 x = ws[k];
        sum += x, kept += x > 0;
        if (static_cast<uint32_t>(s.list[k]) > static_cast<uint32_t>(mine)) before += x;
      }
      const u64 goal = goal_of(P.u[r], sum);
      if (before <= goal && goal < before + w) write(P, r, static_cast<int>(~static_cast<uint32_t>(mine)), w, sum, kept);
    }
  }

  // The draw by rank 0 among its n candidates (logits, then replaced by what they weigh, and ids) above the cut and its
  // ties: bins of ids, 1024 over the vocabulary and then the ids of one, hold weights and numbers of tied tokens.
  __device__ __forceinline__ void draw_from_list(const SampleParams& P, int r, uint2* list, int n, const Cut& cut, u64 least) {
    constexpr uint32_t kTied = 0xfffffffeu;  // (weights are at most 2^32 - 256, or 2^32 - 1 for 2^32)
    const u64 tie_weight = (cut.ties > 0 && cut.weight >= least) ? cut.weight : 0;
    const u64 ties = tie_weight ? cut.ties : 0;
    uint32_t* tied = reinterpret_cast<uint32_t*>(s.g);
    const uint32_t least32 = static_cast<uint32_t>(max(1ull, min(least, 0xffffffffull)));
    u64 count = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += NT) {
      const float x = __uint_as_float(list[i].x);
      const uint32_t t = weight32(distance(x)), w = x > cut.x && t >= least32 ? t : 0u;
      list[i].x = ties > 0 && x == cut.x ? kTied : w;
      count += w > 0u;
    }
    count = block_sum(count);
    auto reach = [&](u64 above, u64 tied) { return above + min(ties, tied) * tie_weight; };
    int base = 0, shift = max(0, 22 - __clz(P.vocab - 1));  // bins of 2^shift ids
    u64 wb = 0, tb = 0, whole = 0, goal = 0;
    for (bool first = true;; first = false) {
      for (int i = threadIdx.x; i < kSampBins; i += NT) s.lo[i] = s.hi[i] = tied[i] = 0u;
      __syncthreads();
#pragma unroll 1
      for (int i = threadIdx.x; i < n; i += NT) {
        const uint2 c = list[i];
        const int id = static_cast<int>(c.y), bin = (id - base) >> shift;
        if (id < base || bin >= kSampBins) continue;
        if (c.x == kTied)
          atomicAdd(&tied[bin], 1u);
        else
          add_weight(bin, c.x);
      }
      __syncthreads();
      constexpr int kPer = kSampBins / NT;
      const int b0 = threadIdx.x * kPer;
      u64 ws = 0, ts = 0, all_w, all_t;
#pragma unroll
      for (int i = 0; i < kPer; ++i) ws += bin_sum(b0 + i), ts += tied[b0 + i];
      u64 wi = ws, ti = ts;
      block_scan(wi, ti, &all_w, &all_t);
      if (first) whole = reach(all_w, all_t), goal = goal_of(P.u[r], whole), count += min(ties, all_t);
      wi += wb - ws, ti += tb - ts;  // before this thread's bins
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const u64 wn = wi + bin_sum(b0 + i), tn = ti + tied[b0 + i];
        if (reach(wi, ti) <= goal && goal < reach(wn, tn)) {
          if (shift == 0) {
            write(P, r, base + b0 + i, wn > wi ? wn - wi : tie_weight, whole, count);
          } else {
            s.found[0] = b0 + i, s.found[1] = wi, s.found[2] = ti;
          }
        }
        wi = wn, ti = tn;
      }
      if (shift == 0) return;
      __syncthreads();
      base += static_cast<int>(s.found[0]) << shift, wb = s.found[1], tb = s.found[2];
      shift = 0;
    }
  }

  __device__ __forceinline__ static u64 goal_of(float u, u64 sum) {
    const double target = static_cast<double>(u) * static_cast<double>(sum);
    const u64 goal = target > 0.0 ? static_cast<u64>(target) : 0;
    return goal >= sum ? sum - 1 : goal;
  }
  __device__ __forceinline__ static void write(const SampleParams& P, int r, int id, u64 w, u64 sum, u64 kept) {
    P.token[r] = id;
    P.logprob[r] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(sum)));
    P.kept[r] = static_cast<int>(kept);
  }

  // The draw among the tokens above the cut and its ties, everywhere in the row.
  __device__ __forceinline__ void draw_from_row(const SampleParams& P, int r, const Cut& cut, u64 least) {
    const u64 tie_weight = (cut.ties > 0 && cut.weight >= least) ? cut.weight : 0;
    const uint32_t ties = tie_weight ? cut.ties : 0;
    const uint32_t least32 = static_cast<uint32_t>(max(1ull, min(least, 0xffffffffull)));
    const float low = fmaxf(cut.x, floor);
    // weights of one vector's kept tokens above the cut; false: it has none, nor a tied one
    auto kept_of = [&](const uint4& u, float (&x)[kVec], uint32_t (&k)[kVec]) {
      if (!(largest(u) >= low)) return false;
      unpack(u, static_cast<const T*>(nullptr), x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const uint32_t t = weight32(distance(x[e]));
        k[e] = x[e] > cut.x && t >= least32 ? t : 0u;
      }
      return true;
    };
    // a warp takes consecutive vectors, so that the search below has one warp's to look through
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = (nvec + kWarps - 1) / kWarps;
    const float full = top + 1e-3f * (floor - top);  // tokens below (0.02 T from the top) weigh less than 2^32
    u64 sum = 0, num = 0;  // num: count above, and ties in the low half
    uint32_t above = 0u, tied = 0u;
    for (int v = warp * share + lane; v < min(nvec, (warp + 1) * share); v += 32) {
      float x[kVec];
      uint32_t k[kVec];
      const uint4 u = row[v];
      if (!kept_of(u, x, k)) continue;
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum += k[e], above += k[e] > 0u;
      if (largest(u) >= full) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) sum += k[e] == 0xffffffffu;
      }
      if (ties)
#pragma unroll
        for (int e = 0; e < kVec; ++e) tied += x[e] == cut.x;
    }
    above = __reduce_add_sync(0xffffffffu, above), tied = __reduce_add_sync(0xffffffffu, tied);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (lane == 0) s.warps[warp][0] = sum, s.warps[warp][1] = (static_cast<u64>(above) << 32) | tied;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += s.warps[w][0], num += s.warps[w][1];
    all_gather(sum, num);
    u64 whole = static_cast<u64>(ties) * tie_weight, count = ties;
    for (int k = 0; k < cluster; ++k) whole += slot(k, 0), count += slot(k, 1) >> 32;
    const u64 goal = goal_of(P.u[r], whole);
    // inclusive sum after a token: weight above the cut + tie_weight * min(ties, tied tokens so far)
    auto reach = [&](u64 above, u64 tied) { return above + min(static_cast<u64>(ties), tied) * tie_weight; };
    u64 wb = 0, tb = 0;
    int owner = 0;
    for (; owner < cluster - 1; ++owner) {
      const u64 w1 = wb + slot(owner, 0), t1 = tb + static_cast<uint32_t>(slot(owner, 1));
      if (reach(w1, t1) > goal) break;
      wb = w1, tb = t1;
    }
    if (rank != owner) return;
    int w0 = 0;
    for (; w0 < kWarps - 1; ++w0) {
      const u64 w1 = wb + s.warps[w0][0], t1 = tb + static_cast<uint32_t>(s.warps[w0][1]);
      if (reach(w1, t1) > goal) break;
      wb = w1, tb = t1;
    }
    const int end = min(nvec, (w0 + 1) * share);
    for (int base = w0 * share; base < end; base += NT) {
      const int v = base + threadIdx.x;
      float x[kVec];
      uint32_t k[kVec];
      u64 ws = 0, ts = 0, all_w, all_t;
      const bool some = v < end && kept_of(row[v], x, k);
      if (some) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) ws += widen(k[e]), ts += ties > 0u && x[e] == cut.x;
      }
      u64 wi = ws, ti = ts;
      block_scan(wi, ti, &all_w, &all_t);
      wi += wb - ws, ti += tb - ts;  // before this vector
      if (some && reach(wi, ti) <= goal && goal < reach(wi + ws, ti + ts)) {
        bool done = false;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const bool tie = ties > 0u && x[e] == cut.x;
          wi += widen(k[e]), ti += tie;
          if (!done && reach(wi, ti) > goal) {
            done = true;
            write(P, r, first_id + v * kVec + e, tie ? tie_weight : widen(k[e]), whole, count);
          }
        }
      }
      wb += all_w, tb += all_t;
      if (reach(wb, tb) > goal) break;
    }
  }
};

template <typename T, int NT>
__global__ void __launch_bounds__(NT, NT == 512 ? 1 : 4) sample_kernel(const __grid_constant__ SampleParams P) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kWarps = NT / 32;
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
  const int inner = max(0, nvec - head - tail);
  if (threadIdx.x == 0) {
    mbar_init(&s.loaded, 1);
    fence_mbar_init();
    mbar_arrive_expect_tx(&s.loaded, inner * 16);
    if (inner > 0) bulk_load(vecs + head, src + first_id + head * kVec, inner * 16, &s.loaded, l2_policy_evict_first());
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
  const float temp = P.temperature ? P.temperature[r] : 1.0f;
  const int top_k = P.top_k ? P.top_k[r] : 0;
  const float top_p = P.top_p ? P.top_p[r] : 1.0f;
  const float min_p = P.min_p ? P.min_p[r] : 0.0f;
  const bool greedy = !(temp > 0.0f);
  // the list holds what the bound lets through, a little more than top_k
  const bool few = !greedy && top_k > 0 && top_k < P.vocab && top_k <= kSampList * 3 / 4;
  for (int i = threadIdx.x; i < kSampBins; i += NT) s.g[i] = 0;
  Sampler<T, NT> S{s, vecs, nvec, first_id, rank, cluster, 0, 0.0f, 0.0f, 0.0f, 1.0f, -INFINITY};
  __syncthreads();  // the barrier is set up, the edges are written
  const bool ok = mbar_wait(&s.loaded, 0u, kErrSampleTimeout);
  // ---- maximum (NaN is passed over here and weighs nothing below) and, for a greedy row, its first id ----
  float best[4];
  {
    typename MaximaOf<T>::Type maxima;
    for (int v = threadIdx.x; v < nvec; v += NT) maxima.add(vecs[v]);
    maxima.get(best);
  }
  const uint32_t mine = order_bits(fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3])));
  uint32_t m = __reduce_max_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) s.red32[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) m = max(m, s.red32[w]);
  uint32_t id = 0x7fffffffu;
  float bound = -INFINITY;
  if (greedy) {
    const float top = order_value(m);
    if (mine == m)
      for (int v = threadIdx.x; v < nvec && id == 0x7fffffffu; v += NT) {
        float x[kVec];
        S.load(v, x);
#pragma unroll
        for (int i = kVec - 1; i >= 0; --i)
          if (x[i] == top) id = first_id + v * kVec + i;
      }
    id = __reduce_min_sync(0xffffffffu, id);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red32[threadIdx.x >> 5] = id;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) id = min(id, s.red32[w]);
  } else if (few) {
    __syncthreads();
    bound = S.reached_by((top_k + cluster - 1) / cluster, best, order_value(m), fminf(fmaxf(temp, 1e-30f), 3e38f));
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  S.all_gather((static_cast<u64>(m) << 32) | static_cast<uint32_t>(~id), (static_cast<u64>(ok ? 0u : 1u) << 32) | order_bits(bound));
  u64 first = 0, failed = 0;
  uint32_t least_bound = 0xffffffffu;
  for (int k = 0; k < cluster; ++k) {
    first = max(first, S.slot(k, 0)), failed |= S.slot(k, 1) >> 32;
    least_bound = min(least_bound, static_cast<uint32_t>(S.slot(k, 1)));
  }
  S.top = order_value(static_cast<uint32_t>(first >> 32));
  const bool empty = S.top == -INFINITY;
  if (greedy || empty || failed) {  // failed: the copy's wait ran out, in whichever CTA
    if (!ok) settle_issued_copies();
    if (rank == 0 && threadIdx.x == 0) {
      P.token[r] = empty || failed ? -1 : static_cast<long long>(~static_cast<uint32_t>(first));
      P.logprob[r] = empty || failed ? -INFINITY : 0.0f;
      P.kept[r] = empty || failed ? 0 : 1;
    }
    return;  // nothing is written to another CTA after the last barrier: so at every return here
  }
  if (S.top == INFINITY) {  // the infinite ones share the draw: as logits 0 and -inf
    for (int v = threadIdx.x; v < nvec; v += NT) {
      T* e = reinterpret_cast<T*>(vecs + v);
#pragma unroll 1
      for (int i = 0; i < kVec; ++i) e[i] = static_cast<T>(static_cast<float>(e[i]) == INFINITY ? 0.0f : -INFINITY);
    }
    __syncthreads();
    S.top = 0.0f;
    least_bound = order_bits(-INFINITY);
  }
  // temperatures of [1e-30, 3e38] at a scale where neither a quotient's remainder nor the reciprocal leaves
  // the normal numbers
  S.temp = fminf(fmaxf(temp, 1e-30f), 3e38f);
  S.scale = S.temp < 1e-20f ? 18446744073709551616.0f : S.temp > 1e20f ? 5.4210108624275222e-20f : 1.0f;  // 2^64, 2^-64
  S.floor = S.top - 22.21f * S.temp;  // exp(-22.2) < 2^-32, and room for what this rounds
  S.temp *= S.scale;
  S.inv = __fdiv_rn(1.0f, S.temp);

  // w >= min_p 2^32 for whole w
  const u64 least = static_cast<u64>(ceil(static_cast<double>(min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f) * 4294967296.0));
  auto in_row = [&](float least, auto f) { S.each(least, f); };
  const int n = few ? S.gather_candidates(order_value(least_bound)) : -1;
  Cut cut{};
  if (n < 0) {
    cut = S.template find_cut<false>(in_row, top_k < P.vocab ? top_k : 0, top_p);
  } else if (n <= kSampFew) {
    if (rank == 0) S.draw_from_few(P, r, n, top_k, top_p, least);
    return;
  } else {
    if (rank > 0) return;
    // the candidates move to where the logits were
    uint2* list = reinterpret_cast<uint2*>(vecs);
    for (int i = threadIdx.x; i < n; i += NT) {
      const u64 c = s.list[i];
      list[i] = make_uint2(__float_as_uint(order_value(static_cast<uint32_t>(c >> 32))), ~static_cast<uint32_t>(c));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kSampBins; i += NT) s.g[i] = 0;
    cut = S.template find_cut<true>(
        [&](float, auto f) {
#pragma unroll 1
          for (int i = threadIdx.x; i < n; i += NT) f(__uint_as_float(list[i].x));
        },
        top_k, top_p);
    __syncthreads();  // every warp has read the last answer in `found`
    S.draw_from_list(P, r, list, n, cut, least);
    return;
  }
  S.draw_from_row(P, r, cut, least);
}

template <typename T>
size_t sample_smem(int vocab, int cluster) {
  const int kVec = 16 / sizeof(T);
  const int per = ((vocab + kVec - 1 + kVec - 1) / kVec + cluster - 1) / cluster;
  return (sizeof(SampleShared) + 15) / 16 * 16 + std::max<size_t>(static_cast<size_t>(per) * 16, kSampList * 8);  // or the list
}

template <typename T, int NT>
cudaError_t launch_sample(const SampleParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows * p.cluster), 1, 1);
  cfg.blockDim = dim3(NT, 1, 1);
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
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, NT>, p);
}

constexpr int kSampSmemMax = 220 * 1024;
template <typename T, int NT>
cudaError_t sample_smem_limit() {
  return cudaFuncSetAttribute(sample_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampSmemMax);
}
}  // namespace

cudaError_t sample_prepare_device() {
  cudaError_t e = sample_smem_limit<__nv_bfloat16, 512>();
  if (e == cudaSuccess) e = sample_smem_limit<__nv_bfloat16, 256>();
  if (e == cudaSuccess) e = sample_smem_limit<float, 512>();
  if (e == cudaSuccess) e = sample_smem_limit<float, 256>();
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
  // As many CTAs a row, up to 8, as leave each 4096 tokens or fewer: right for few rows.  The number of rows does not
  // count yet, and many rows of a middling vocabulary would be faster with fewer (us, bf16, 1 / 2 / 4 / 8 CTAs a row: 1 row,
  // top-p 0.9, of 4096 15.4 / 15.4 / 15.5 / 15.9, 16384 23 / 18 / 15.5 / 16.3, 32003 34 / 24 / 18 / 16, 151680 - / - / 42 / 29;
  // 256 rows of 4096 30 / 20 / 36 / 69, 32003 70 / 53 / 62 / 87, 151680 - / - / 257 / 207).
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
  // Few CTAs: 512 threads each shorten a row's passes (1 x 151680 bf16, top-k 1000 14.8 us against 19.0 with 256,
  // temperature alone 11.6 against 13.8).  More than two an SM: 256 threads, four CTAs to an SM (256 x 151680, mixed
  // filters, 90 us against 120 with 512 threads, two to an SM, when both were measured; now 86).
  const bool wide = static_cast<long long>(rows) * p.cluster <= 2 * sm_count();
  cudaError_t e;
  if (logits_fp32)
    e = wide ? launch_sample<float, 512>(p, st) : launch_sample<float, 256>(p, st);
  else
    e = wide ? launch_sample<__nv_bfloat16, 512>(p, st) : launch_sample<__nv_bfloat16, 256>(p, st);
  if (e != cudaSuccess) return cuda_fail(e, "sample launch");
  return RLDX_OK;
}
