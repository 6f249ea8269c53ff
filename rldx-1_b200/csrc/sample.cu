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
// A cluster of CTAs holds a row in shared memory, so the logits are read once.  Top-k and top-p are
// searches for the last token kept, by histogram: 1024 bins linear in -d (every bin holds a run of
// the order), then by the ordered bits of the logit inside the bin where count or weight crosses,
// until one value is left; of the tokens that share it the first few by id stay.  Bins hold
// counts and weights (the low 16 and high 17 bits of a weight in two 32-bit sums); CTAs add theirs
// to rank 0's through distributed shared memory, which finds the crossing and tells the others.
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
  uint32_t ties;
  u64 before_weight;
  uint32_t before_count;
};

struct SampleShared {
  uint32_t count[kSampBins], lo[kSampBins], hi[kSampBins];  // this CTA's bins
  uint32_t g_count[kSampBins];                              // rank 0: the row's
  u64 g_weight[kSampBins];
  u64 slots[2][kSampMaxCluster][4];  // all-gather, two phases
  u64 found[8];                      // rank 0's answer, written to every CTA
  u64 red[kSampWarps][2];
  uint32_t red32[kSampWarps];
  uint32_t flag;
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

template <typename T>
struct Sampler {
  static constexpr int kVec = 16 / sizeof(T);
  SampleShared& s;
  const uint4* row;  // this CTA's vectors in shared memory
  int nvec, first_id;  // vectors held, id of the first one's first token (negative: padding)
  int rank, cluster, phase;
  float top, temp;

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
  __device__ __forceinline__ float distance(float x) const {  // d <= 0
    return x == top ? 0.0f : __fdiv_rn(x - top, temp);
  }
  __device__ __forceinline__ static u64 weight_of(float d) {
    if (!(d > -kSampReach)) return 0;
    const float f = expf(d) * 4294967296.0f;
    return static_cast<u64>(__float2uint_rz(f)) + (f >= 4294967296.0f ? 1u : 0u);
  }
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
    for (int i = threadIdx.x; i < kSampBins; i += kSampThreads) s.count[i] = s.lo[i] = s.hi[i] = 0u;
    __syncthreads();
  }
  __device__ __forceinline__ void add(int bin, u64 w) {
    atomicAdd(&s.count[bin], 1u);
    const uint32_t l = static_cast<uint32_t>(w) & 0xffffu, h = static_cast<uint32_t>(w >> 16);
    if (l) atomicAdd(&s.lo[bin], l);
    if (h) atomicAdd(&s.hi[bin], h);
  }
  // The first bin where the running count (or weight) passes `level`; found = {bin or ~0, count before,
  // weight before, count of the bin, weight of the bin}.  rank 0's sums are zero before and after.
  __device__ __forceinline__ bool crossing(bool by_count, u64 level) {
    __syncthreads();
    const uint32_t gc = mapa_shared(smem_u32(s.g_count), 0), gw = mapa_shared(smem_u32(s.g_weight), 0);
    for (int i = threadIdx.x; i < kSampBins; i += kSampThreads)
      if (s.count[i]) {
        red_cluster_u32(gc + 4 * i, s.count[i]);
        red_cluster_u64(gw + 8 * i, (static_cast<u64>(s.hi[i]) << 16) + s.lo[i]);
      }
    cluster_sync();
    if (rank == 0) {
      constexpr int kPer = kSampBins / kSampThreads;
      uint32_t c[kPer];
      u64 w[kPer], cs = 0, ws = 0;
      const int b0 = threadIdx.x * kPer;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        c[i] = s.g_count[b0 + i], w[i] = s.g_weight[b0 + i];
        s.g_count[b0 + i] = 0u, s.g_weight[b0 + i] = 0;
        cs += c[i], ws += w[i];
      }
      u64 ci = cs, wi = ws;  // inclusive scans
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 a = __shfl_up_sync(0xffffffffu, ci, o), b = __shfl_up_sync(0xffffffffu, wi, o);
        if (lane >= o) ci += a, wi += b;
      }
      if (lane == 31) s.red[warp][0] = ci, s.red[warp][1] = wi;
      if (threadIdx.x == 0) s.flag = 0u;
      __syncthreads();
      u64 cb = ci - cs, wb = wi - ws;
      for (int k = 0; k < warp; ++k) cb += s.red[k][0], wb += s.red[k][1];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const u64 before = by_count ? cb : wb, amount = by_count ? c[i] : w[i];
        if (before <= level && level < before + amount) {
          s.flag = 1u;
          const u64 v[5] = {static_cast<u64>(b0 + i), cb, wb, c[i], w[i]};
          for (int r = 0; r < cluster; ++r)
            for (int k = 0; k < 5; ++k) st_cluster_u64(mapa_shared(smem_u32(&s.found[k]), r), v[k]);
        }
        cb += c[i], wb += w[i];
      }
      __syncthreads();
      if (threadIdx.x == 0 && s.flag == 0u)
        for (int r = 0; r < cluster; ++r) st_cluster_u64(mapa_shared(smem_u32(&s.found[0]), r), ~0ull);
    }
    cluster_sync();
    return s.found[0] != ~0ull;
  }

  // Finds the cut where the count (or weight) of the order passes `level` among the tokens of positive
  // weight above `from` and its ties.  False: never.
  __device__ __forceinline__ bool find(bool by_count, u64 level, const Cut& from, Cut* out) {
    clear();
    each([&](float x) {
      if (order_bits(x) <= from.key) return;
      const float d = distance(x);
      if (!(d > -kSampReach)) return;
      const u64 w = weight_of(d);
      if (w) add(bin_of(d), w);
    });
    const bool has_ties = from.ties > 0;  // the ties of the cut so far count as that many tokens
    const int tie_bin = has_ties ? bin_of(distance(from.x)) : -1;
    __syncthreads();
    if (rank == 0 && threadIdx.x == 0 && has_ties) {
      s.g_count[tie_bin] += from.ties;
      s.g_weight[tie_bin] += from.ties * from.weight;
    }
    if (has_ties) cluster_sync();  // before the others add to the same bin
    if (!crossing(by_count, level)) return false;
    const int bin = static_cast<int>(s.found[0]);
    u64 cb = s.found[1], wb = s.found[2], cn = s.found[3], wn = s.found[4];
    // the bin's range of ordered bits
    uint32_t lo = 0xffffffffu, hi = 0u;
    each([&](float x) {
      const uint32_t k = order_bits(x);
      if (k <= from.key) return;
      const float d = distance(x);
      if (!(d > -kSampReach) || bin_of(d) != bin || weight_of(d) == 0) return;
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
        const u64 w = weight_of(distance(x));
        if (w) add((hi - k) >> shift, w);
      });
      const bool tie_in = has_ties && from.key >= lo && from.key <= hi;
      __syncthreads();
      if (rank == 0 && threadIdx.x == 0 && tie_in) {
        s.g_count[(hi - from.key) >> shift] += from.ties;
        s.g_weight[(hi - from.key) >> shift] += from.ties * from.weight;
      }
      if (tie_in) cluster_sync();
      if (!crossing(by_count, by_count ? level - cb : level - wb)) return false;  // (a bin holds its crossing)
      const uint32_t b = static_cast<uint32_t>(s.found[0]);
      cb += s.found[1], wb += s.found[2], cn = s.found[3], wn = s.found[4];
      hi -= b << shift;
      const uint32_t width = (1u << shift) - 1u;
      lo = hi - lo > width ? hi - width : lo;
    }
    out->key = lo;
    out->x = order_value(lo);
    out->weight = wn / cn;
    out->before_count = static_cast<uint32_t>(cb);
    out->before_weight = wb;
    out->ties = static_cast<uint32_t>(cn);  // the caller keeps as many as fit
    return true;
  }
};

template <typename T>
__global__ void __launch_bounds__(kSampThreads) sample_kernel(const __grid_constant__ SampleParams P) {
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

  // ---- this CTA's share of the row: whole 16-byte vectors of memory, tokens outside it -inf ----
  const T* src = static_cast<const T*>(P.logits) + r * P.ld;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));
  const int all = (P.vocab + mis + kVec - 1) / kVec, per = (all + cluster - 1) / cluster;
  const int v0 = min(all, rank * per), nvec = min(all, v0 + per) - v0;
  const int first_id = v0 * kVec - mis;
  float best = -INFINITY;
  for (int v = threadIdx.x; v < nvec; v += kSampThreads) {
    const int id = first_id + v * kVec;
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
    if (id >= 0 && id + kVec <= P.vocab) {
      u = __ldcs(reinterpret_cast<const uint4*>(src + id));
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        e[i] = (id + i >= 0 && id + i < P.vocab) ? src[id + i] : static_cast<T>(-INFINITY);
    }
    float x[kVec];
    unpack(u, static_cast<const T*>(nullptr), x);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if (x[i] != x[i]) e[i] = static_cast<T>(-INFINITY);  // NaN: never drawn
      best = fmaxf(best, x[i]);
    }
    vecs[v] = u;
  }
  for (int i = threadIdx.x; i < kSampBins; i += kSampThreads) s.g_count[i] = 0u, s.g_weight[i] = 0;
  Sampler<T> S{s, vecs, nvec, first_id, rank, cluster, 0, 0.0f, 0.0f};
  // ---- maximum and its first id ----
  const uint32_t mine = order_bits(best);
  uint32_t m = __reduce_max_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) s.red32[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int w = 0; w < kSampWarps; ++w) m = max(m, s.red32[w]);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  S.all_gather(m, 0, 0, 0);
  for (int k = 0; k < cluster; ++k) m = max(m, static_cast<uint32_t>(S.slot(k, 0)));
  S.top = order_value(m);
  const float temp = P.temperature ? P.temperature[r] : 1.0f;
  const bool greedy = !(temp > 0.0f), empty = S.top == -INFINITY;
  if (greedy || empty) {
    uint32_t id = 0x7fffffffu;
    if (mine == m)
      for (int v = threadIdx.x; v < nvec && id == 0x7fffffffu; v += kSampThreads) {
        float x[kVec];
        unpack(vecs[v], static_cast<const T*>(nullptr), x);
#pragma unroll
        for (int i = kVec - 1; i >= 0; --i)
          if (x[i] == S.top) id = first_id + v * kVec + i;
      }
    id = __reduce_min_sync(0xffffffffu, id);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red32[threadIdx.x >> 5] = id;
    __syncthreads();
    for (int w = 0; w < kSampWarps; ++w) id = min(id, s.red32[w]);
    S.all_gather(id, 0, 0, 0);
    if (rank == 0 && threadIdx.x == 0) {
      for (int k = 0; k < cluster; ++k) id = min(id, static_cast<uint32_t>(S.slot(k, 0)));
      P.token[r] = empty ? -1 : static_cast<long long>(id);
      P.logprob[r] = empty ? -INFINITY : 0.0f;
      P.kept[r] = empty ? 0 : 1;
    }
    cluster_sync();  // no CTA leaves while another may still write to it
    return;
  }
  S.temp = fmaxf(temp, 1e-30f);

  const int top_k = P.top_k ? P.top_k[r] : 0;
  const float top_p = P.top_p ? P.top_p[r] : 1.0f;
  const float min_p = P.min_p ? P.min_p[r] : 0.0f;
  Cut cut{};  // key 0: below every logit
  cut.key = order_bits(-INFINITY);
  cut.x = -INFINITY;
  u64 total = 0;
  if (top_k > 0 && top_k < P.vocab) {
    Cut c;
    if (S.find(true, static_cast<u64>(top_k) - 1, cut, &c)) {
      c.ties = min(c.ties, static_cast<uint32_t>(top_k) - c.before_count);
      cut = c;
      total = c.before_weight + c.ties * c.weight;
    }
  }
  if (top_p < 1.0f) {
    if (total == 0) {
      u64 w = 0;
      S.each([&](float x) { w += Sampler<T>::weight_of(S.distance(x)); });
      w = S.block_sum(w);
      S.all_gather(w, 0, 0, 0);
      for (int k = 0; k < cluster; ++k) total += S.slot(k, 0);
    }
    // kept: weight before < p total, and the first in any case
    const double bound = static_cast<double>(top_p) * static_cast<double>(total);
    const u64 level = bound > 1.0 ? static_cast<u64>(ceil(bound)) - 1 : 0;
    Cut c;
    if (S.find(false, level, cut, &c)) {
      const u64 fit = (level - c.before_weight) / c.weight + 1;
      c.ties = static_cast<uint32_t>(min(static_cast<u64>(c.ties), fit));
      cut = c;
    }
  }
  const double least = static_cast<double>(min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f) * 4294967296.0;
  const u64 tie_weight = (cut.ties > 0 && static_cast<double>(cut.weight) >= least) ? cut.weight : 0;
  const uint32_t ties = tie_weight ? cut.ties : 0;
  auto kept_weight = [&](float x) -> u64 {  // of a token above the cut
    if (order_bits(x) <= cut.key) return 0;
    const u64 w = Sampler<T>::weight_of(S.distance(x));
    return static_cast<double>(w) >= least ? w : 0;
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
