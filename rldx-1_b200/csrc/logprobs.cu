// Log probabilities of given tokens under rows of logits, with the entropy of each row, the token's rank and the
// top alternatives, in one pass over the logits (rows whose queue overflows are gone over again, see below).
//
// With M the row's maximum, d_i = x_i - M, S = sum exp(d_i) and T = sum exp(d_i) d_i:
//   log p_i = d_i - ln S,   H = ln S - T / S  (both terms positive: nothing cancels),
//   rank of t = the number of i with x_i > x_t, or x_i = x_t and i < t,
//   top: the k first in the order of descending logits, equal ones by ascending id.
// Sums and statistics are fp32, each thread's relative to the largest logit that it has seen; two of them are joined
// by moving the smaller reference to the larger.
//
// A row is shared out among the CTAs of a cluster, one where rows are many; each goes over its part in chunks that its
// threads hold in registers, the next one on the way.
// The top k of a part: after the chunks 0, 1, 3, 7, ... the k-th largest of 64 maxima, each of a few threads', is a bound
// that some more than k values reach (two warps find it by counting for each how many are larger).  Threads whose maximum
// of a chunk reaches it queue the vectors that do; at the end the queue's values that reach the last bound are put in order
// as (ordered bits of the logit, ~id), whose order is the answer's.  -inf is never queued: where fewer than k
// other values are in a row, the missing places go to the lowest ids of -inf.  A queue that overflows (many values share the
// bound, or logits rise along the row) is given up for lists of the warps that are cut down to k when they are full:
// exact whatever the row, and some times slower.
//
// Measured: 2208 x 151680 bf16 with 20 alternatives takes 167 us (670 MB: 4.0 TB/s; at the copy's rate 102), without 129, without a
// token to count before 120; 1104 x 151680 fp32 134; one row 7.2 with five alternatives; 64 x 50257 fp32 11.7.  Many rows are bound
// by the instructions of a value (about 8: unpacked, compared, exponential on the special-function unit, two sums); the
// alternatives add the barriers of the bounds and the end of a row, during which the CTA loads nothing.  512 x 151680: rows of
// random logits 55 us, flat 120, descending 85, ascending 183, masked but for a few 128 to 193.
#include <cfloat>

#include "host_util.h"
#include "rows.cuh"

namespace rldx {

namespace {
constexpr int kLogpTop = 32;        // alternatives at most
constexpr int kLogpMaxCluster = 8;
// 16-byte vectors of a thread and chunk: with four, 64 registers let four CTAs of 256 threads run on an SM (eight and three of
// them, us: 2208 x 151680 175 against 171, 256 rows 36.2 against 31.6, 64 x 50257 fp32 16.6 against 14.5, one row 6.1 against 6.8)
constexpr int kLogpVecs = 4;
constexpr int kLogpQueue = 512;     // vectors of a CTA
constexpr int kLogpShown = 8;       // threads that show their vectors to their warp at a time
constexpr int kLogpList = 2 * kLogpShown * kLogpVecs * 8;  // of a warp: room for theirs besides what is left of a full one
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
constexpr float kLogpLeast = -200.0f;  // of d in powers of two: its exponential is 0 all the same, and times it 0 too
constexpr int kLogpMaxVocab = 1 << 28;
constexpr unsigned int kErrLogprobsToken = 0x503;
typedef unsigned long long u64;

struct LogprobsParams {
  const void* logits;
  long long ld;
  int rows, vocab, cluster, top;
  const long long* tokens;
  float* logprob;
  float* entropy;
  int* rank;
  long long* top_ids;
  float* top_logprobs;
};

// Sum of exp2(d) and of exp2(d) d over values relative to m, d = (x - m) log2 e.
struct Partial {
  float m, s, t;
};
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void move_to(Partial& p, float m) {
  const float d = max_nan((p.m - m) * kLog2e, kLogpLeast), f = ex2_approx(d);
  p.t = f * fmaf(p.s, d, p.t);
  p.s *= f;
  p.m = m;
}
// The sums of a warp's threads, and of their counts.  (Called for a warp, a CTA and a cluster: code that runs once a row
// waits for its instructions more than for anything else, so there is one copy of it.)
struct Total {
  Partial p;
  uint32_t better;
};
__device__ __noinline__ Total warp_total(Total x) {
  move_to(x.p, order_value(__reduce_max_sync(0xffffffffu, order_bits(x.p.m))));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x.p.s += __shfl_xor_sync(0xffffffffu, x.p.s, o), x.p.t += __shfl_xor_sync(0xffffffffu, x.p.t, o);
  x.better = __reduce_add_sync(0xffffffffu, x.better);
  return x;
}
__device__ __forceinline__ uint4 words_of(const Total& x) {
  return make_uint4(__float_as_uint(x.p.m), __float_as_uint(x.p.s), __float_as_uint(x.p.t), x.better);
}
// The total of n of them in shared memory, for every thread of the warp that asks.
__device__ __forceinline__ Total total_of(const uint4* words, int n) {
  const int lane = threadIdx.x & 31;
  Total x{{-FLT_MAX, 0.0f, 0.0f}, 0};
  if (lane < n) {
    const uint4 w = words[lane];
    x = {{__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z)}, w.w};
  }
  return warp_total(x);
}

template <int NT>
struct LogprobsShared {
  static constexpr int kWarps = NT / 32;
  union {
    struct {
      uint4 queue[kLogpQueue];
      int queue_at[kLogpQueue];  // their places in the row
    };
    struct {  // where the queue is not enough
      u64 list[kWarps][kLogpList];
      uint4 shown[kWarps][kLogpShown * kLogpVecs];
      int from[kWarps][kLogpShown];
      int listed[kWarps];
    };
  };
  uint4 maxima[64 / 4];
  uint32_t bound[2];      // of a chunk, and of the next one that finds one
  uint4 totals[kWarps];   // of the warps
  u64 front[NT];          // keys that can be among the top, in any order
  int queued, fronts, finalists;
  long long token;
  float x_token;
  // rank 0's, of every CTA: the keys that it sends, their number and its bound, its totals
  u64 sent[kLogpMaxCluster * kLogpTop];
  uint2 sent_n[kLogpMaxCluster];
  uint4 sent_totals[kLogpMaxCluster];
  u64 final[kLogpMaxCluster * kLogpTop];  // those that reach every CTA's bound
};

// What differs between the types: a word of -inf, how many leading bits of the fp32 form tell values apart, how far from
// zero a reference may lie for the short form of the differences, and the value that stands for what is below it there.
template <typename T>
struct Logit;
template <>
struct Logit<__nv_bfloat16> {
  static constexpr uint32_t kLowest = 0xff80ff80u, kFloor = 0xf14af14au;  // -1e30
  static constexpr int kBits = 16;
  static constexpr float kNear = 65536.0f;
};
template <>
struct Logit<__half> {
  static constexpr uint32_t kLowest = 0xfc00fc00u, kFloor = 0xfbfffbffu;  // -65504
  static constexpr int kBits = 19;  // sign, 8 exponent and 10 mantissa bits
  static constexpr float kNear = 32768.0f;
};
template <>
struct Logit<float> {
  static constexpr uint32_t kLowest = 0xff800000u;
  static constexpr int kBits = 32;
  static constexpr float kNear = 65536.0f;
};

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, const __nv_bfloat16*) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, const __half*) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, const __nv_bfloat16*) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, const __half*) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint32_t w, const __nv_bfloat16*) {
  float2 x;
  unpack_bf16x2(w, x.x, x.y);
  return x;
}
__device__ __forceinline__ float2 unpack2(uint32_t w, const __half*) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
// Ones where a > b, added up in fp16 in halves of a word (whole numbers up to 2048 there).  bf16 patterns are compared as
// fp16 ones, whose order is the same up to 2^121 (2208 rows of 151680: 175 us, with bf16 comparisons 184).
__device__ __forceinline__ void count2(uint32_t& n, uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<__half2*>(&n), __hgt2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b)));
  n = *reinterpret_cast<const uint32_t*>(&r);
}
// The largest value of T below x (x finite).
__device__ __forceinline__ __nv_bfloat16 below(__nv_bfloat16 x) {
  const uint16_t b = __bfloat16_as_ushort(x);
  return __ushort_as_bfloat16((b & 0x7fffu) == 0 ? 0x8001u : b & 0x8000u ? b + 1 : b - 1);
}
__device__ __forceinline__ __half below(__half x) {
  const uint16_t b = __half_as_ushort(x);
  return __ushort_as_half((b & 0x7fffu) == 0 ? 0x8001u : b & 0x8000u ? b + 1 : b - 1);
}
__device__ __forceinline__ float below(float x) {
  const uint32_t b = __float_as_uint(x);
  return __uint_as_float((b & 0x7fffffffu) == 0 ? 0x80000001u : b & 0x80000000u ? b + 1 : b - 1);
}
template <typename T>
__device__ __forceinline__ uint32_t both(T x) {
  if constexpr (sizeof(T) == 4)
    return __float_as_uint(x);
  else
    return 0x10001u * *reinterpret_cast<const uint16_t*>(&x);
}

// The largest of a vector (NaN gives way).
template <typename T>
__device__ __forceinline__ float largest_of(const uint4& u) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  } else {
    const T* t = nullptr;
    const float2 x = unpack2(max2(max2(u.x, u.y, t), max2(u.z, u.w, t), t), t);
    return fmaxf(x.x, x.y);
  }
}
template <typename T>
__device__ __forceinline__ float largest_of(const uint4 (&raw)[kLogpVecs]) {
  if constexpr (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kLogpVecs; ++k) m = fmaxf(m, largest_of<T>(raw[k]));
    return m;
  } else {
    const T* t = nullptr;
    uint32_t m = Logit<T>::kLowest;
#pragma unroll
    for (int k = 0; k < kLogpVecs; ++k) m = max2(m, max2(max2(raw[k].x, raw[k].y, t), max2(raw[k].z, raw[k].w, t), t), t);
    const float2 x = unpack2(m, t);
    return fmaxf(x.x, x.y);
  }
}
// -inf in the place of other rows' values; the vector's ids count from `id0`.
template <typename T>
__device__ __forceinline__ void cut_vec(uint4& u, int id0, int vocab) {
  T* e = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i)
    if (id0 + i < 0 || id0 + i >= vocab) e[i] = from_float<T>(-INFINITY);
}

__device__ __forceinline__ u64 key_of(float x, int id) {
  return (static_cast<u64>(order_bits(x)) << 32) | static_cast<uint32_t>(~id);
}

__device__ __forceinline__ u64 pair_of(uint32_t lo, uint32_t hi) { return (static_cast<u64>(hi) << 32) | lo; }
// The largest t, in bits 31 to `low`, that `need` of the warp's numbers reach (of those there are at least so many).
// count(c): of a thread's those that reach c.
template <typename F>
__device__ __forceinline__ uint32_t warp_reached_by(int need, int low, F count) {
  uint32_t t = 0;
#pragma unroll 1
  for (int b = 31; b >= low; --b)
    if (static_cast<int>(__reduce_add_sync(0xffffffffu, count(t | (1u << b)))) >= need) t |= 1u << b;
  return t;
}
// Leaves the keys of a warp's list of n that reach `last`, and returns their number.
__device__ __forceinline__ int warp_keep(u64* list, int n, u64 last) {
  const int lane = threadIdx.x & 31;
  int kept = 0;
  __syncwarp();
  for (int base = 0; base < n; base += 32) {
    const u64 key = base + lane < n ? list[base + lane] : 0;
    const uint32_t keep = __ballot_sync(0xffffffffu, key >= last);  // (every key has been read by now)
    if (key >= last) list[kept + __popc(keep & ((1u << lane) - 1u))] = key;
    kept += __popc(keep);
    __syncwarp();
  }
  return kept;
}
// Cuts a warp's list of n > k keys down to the k best and returns the last of them.  kBits: as Logit's.
template <int kBits>
__device__ __noinline__ u64 warp_prune(u64* list, int n, int k) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  auto count = [&](auto f) {
    uint32_t c = 0;
    for (int i = lane; i < n; i += 32) c += f(static_cast<uint32_t>(list[i] >> 32), static_cast<uint32_t>(list[i]));
    return c;
  };
  uint32_t hi = warp_reached_by(k, 32 - kBits, [&](uint32_t c) { return count([c](uint32_t x, uint32_t) { return x >= c; }); });
  if (kBits < 32 && !(hi >> 31)) hi |= (1u << (32 - kBits)) - 1u;  // (negative values: the bits that the type does not have are ones)
  const int left = k - static_cast<int>(__reduce_add_sync(0xffffffffu, count([hi](uint32_t x, uint32_t) { return x > hi; })));
  const uint32_t lo = warp_reached_by(left, 0, [&](uint32_t c) { return count([hi, c](uint32_t x, uint32_t id) { return x == hi && id >= c; }); });
  const u64 last = pair_of(lo, hi);
  warp_keep(list, n, last);
  return last;
}

// Fills s.front with 32 keys at most of every warp, the part's top ones among them, whatever the row: the way of a queue that
// overflowed.  Every thread calls it.  bound_x: a value that they reach.
template <typename T, int NT>
__device__ __noinline__ void list_part(LogprobsShared<NT>& s, int vocab, int top, const uint4* vecs, int before, int begin, int end, int nvec,
                                       float bound_x) {
  constexpr int kVec = 16 / sizeof(T), NV = kLogpVecs;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __syncthreads();  // the queue and the count are done with
  if (tid == 0) s.fronts = 0;
  int bound_id = INT32_MAX;  // values that equal bound_x count up to this id
  int listed = 0;
  u64* list = s.list[warp];
#pragma unroll 1
  for (int base = begin; base < end; base += NT * NV) {
    uint4 raw[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = base + k * NT + tid;
      constexpr uint32_t low = Logit<T>::kLowest;
      raw[k] = v < end ? vecs[v] : make_uint4(low, low, low, low);
      if (v == 0 || v == nvec - 1) cut_vec<T>(raw[k], v * kVec - before, vocab);
    }
    float largest = -INFINITY;
#pragma unroll
    for (int k = 0; k < NV; ++k) largest = fmaxf(largest, largest_of<T>(raw[k]));
    const int id0 = (base + tid) * kVec - before;
    auto who_reach = [&] {
      return __ballot_sync(0xffffffffu, largest > -INFINITY && (largest > bound_x || (largest == bound_x && id0 <= bound_id)));
    };
    uint32_t who = who_reach();
    while (who) {
      if (listed > kLogpList / 2) {
        const u64 last = warp_prune<Logit<T>::kBits>(list, listed, top);
        listed = top;
        if (last > key_of(bound_x, bound_id)) bound_x = order_value(static_cast<uint32_t>(last >> 32)), bound_id = static_cast<int>(~static_cast<uint32_t>(last));
        who &= who_reach();
      }
      // the first few of these threads show their vectors, and every thread looks at one
      const int slot = __popc(who & ((1u << lane) - 1u));
      if ((who >> lane & 1u) && slot < kLogpShown) {
#pragma unroll
        for (int k = 0; k < NV; ++k) s.shown[warp][slot * NV + k] = raw[k];
        s.from[warp][slot] = lane;
      }
      if (lane == 0) s.listed[warp] = listed;
      __syncwarp();
      if (lane / NV < __popc(who)) {
        Raw<T, kVec> r;
        r.w[0] = s.shown[warp][lane];
        const int v = base + (lane % NV) * NT + warp * 32 + s.from[warp][lane / NV];
        float x[kVec];
        unpack_row<T, kVec>(r, x);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int id = v * kVec + i - before;
          if (x[i] > -INFINITY && (x[i] > bound_x || (x[i] == bound_x && id <= bound_id))) list[atomicAdd(&s.listed[warp], 1)] = key_of(x[i], id);
        }
      }
#pragma unroll
      for (int g = 0; g < kLogpShown; ++g) who &= who - 1;
      __syncwarp();
      listed = s.listed[warp];
    }
  }
  if (listed > 32) {
    warp_prune<Logit<T>::kBits>(list, listed, top);
    listed = top;
  }
  __syncthreads();
  int at = 0;
  if (lane == 0) at = atomicAdd(&s.fronts, listed);
  at = __shfl_sync(0xffffffffu, at, 0);
  if (lane < listed) s.front[at + lane] = list[lane];
}

// A row whose sum is good has a distribution: no NaN or +inf, and not -inf alone.
__device__ __forceinline__ bool good_sum(const Partial& p) { return p.s > 0.0f && p.s < INFINITY; }
__device__ __forceinline__ void finish(const LogprobsParams& P, int row, long long token, float x_token, const Total& x) {
  const bool good = good_sum(x.p), given = token >= 0 && token < P.vocab;
  const float log_s = logf(x.p.s);
  if (token >= P.vocab) record_data_error(kErrLogprobsToken);
  P.logprob[row] = token < 0 ? 0.0f : given && good ? (x_token - x.p.m) - log_s : NAN;
  P.rank[row] = given && good ? static_cast<int>(x.better) : -1;
  P.entropy[row] = good ? log_s - kLn2 * (x.p.t / x.p.s) : NAN;
}
// How many of n keys are larger.
__device__ __noinline__ int place_of(const u64* keys, int n, u64 key) {
  int place = 0;
#pragma unroll 4
  for (int i = 0; i < n; ++i) place += keys[i] > key;
  return place;
}
// Writes the row's top of n keys, `i` this thread's first of every `by`.  Where they are fewer the others are the lowest ids of
// -inf: with less than 32 other values they are among the first 64 (the first warp looks for them).
template <typename T>
__device__ __forceinline__ void write_top(const LogprobsParams& P, int row, const u64* keys, int n, int i, int by, const Total& x) {
  const long long at = static_cast<long long>(row) * P.top;
  const bool good = good_sum(x.p);
  const float log_s = logf(x.p.s);
  if (good)
    for (int k = i; k < n; k += by) {
      const u64 key = keys[k];
      const int place = place_of(keys, n, key);
      if (place >= P.top) continue;
      P.top_ids[at + place] = static_cast<long long>(~static_cast<uint32_t>(key));
      P.top_logprobs[at + place] = (order_value(static_cast<uint32_t>(key >> 32)) - x.p.m) - log_s;
    }
  if ((good && n >= P.top) || threadIdx.x >= 32) return;
  int place = good ? n : 0;
  const T* logits = static_cast<const T*>(P.logits) + row * P.ld;
  for (int base = 0; base < 64; base += 32) {
    const int id = base + static_cast<int>(threadIdx.x);
    const uint32_t b = __ballot_sync(0xffffffffu, !good || (id < P.vocab && to_float(logits[id]) == -INFINITY));
    const int mine = place + __popc(b & ((1u << threadIdx.x) - 1u));
    if ((b >> threadIdx.x & 1u) && mine < P.top) P.top_ids[at + mine] = good ? id : -1, P.top_logprobs[at + mine] = good ? -INFINITY : NAN;
    place += __popc(b);
  }
}

// NT threads a CTA.
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) logprobs_kernel(const __grid_constant__ LogprobsParams P) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int NV = kLogpVecs, kWarps = NT / 32;
  __shared__ LogprobsShared<NT> s;
  const int cluster = P.cluster;
  const int part = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  if (cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (rank 0 runs before it is written to)
  griddep_wait();
  griddep_launch();
  const int top = P.top;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = static_cast<int>(blockIdx.x / cluster);
  const T* logits = static_cast<const T*>(P.logits) + row * P.ld;
  // This part of the row: vectors on 16-byte boundaries, the first and the last of the row in part of other rows.
  const int before = static_cast<int>(reinterpret_cast<uintptr_t>(logits) % 16 / sizeof(T));
  const uint4* vecs = reinterpret_cast<const uint4*>(logits - before);
  const int nvec = static_cast<int>((static_cast<long long>(P.vocab) + before + kVec - 1) / kVec);
  const int per = (nvec + cluster - 1) / cluster;
  const int begin = min(nvec, part * per), end = min(nvec, begin + per);
  // vector v; past the part its last one, whose place a chunk fills with -inf before it is looked at
  auto load_vec = [&](int v) { return __ldcs(vecs + min(v, end - 1)); };
  uint4 raw[NV];
  if (begin < end)
#pragma unroll
    for (int k = 0; k < NV; ++k) raw[k] = load_vec(begin + k * NT + tid);

  // Tokens before the given one: of vectors before its own those at or above it, of the others those above, and those of
  // its own vector that equal it and come before it.  Where it is -inf, which also fills up vectors, or of a size that is
  // not compared by its bits, all are looked at.
  const long long token = P.tokens[row];
  const bool given = token >= 0 && token < P.vocab;
  const T t_token = given ? logits[token] : from_float<T>(INFINITY);
  const float x_token = to_float(t_token);
  const bool by_one = given && !(fabsf(x_token) < 1e36f);
  const int v_token = given ? static_cast<int>((token + before) / kVec) : 0;
  const uint32_t above = both(by_one ? from_float<T>(INFINITY) : t_token);
  const uint32_t at_or_above = both(given && !by_one ? below(t_token) : from_float<T>(INFINITY));
  uint32_t better = 0;
  if (given && !by_one && tid < kVec && v_token >= begin && v_token < end) {
    const long long id = static_cast<long long>(v_token) * kVec + tid - before;
    if (id >= 0 && id < token) better = to_float(logits[id]) == x_token;
  }

  if (tid == 0) s.fronts = 0, s.queued = 0, s.token = token, s.x_token = x_token;
  __syncthreads();
  Partial p{-FLT_MAX, 0.0f, 0.0f};
  float best = -INFINITY;  // this thread's largest logit so far, where it has seen one
  bool seen = false;
  float bound_x = -INFINITY;  // what can be among the top reaches it; the same for every thread
  int found = 0;              // such bounds

#pragma unroll 1
  for (int base = begin, chunk = 0; base < end; base += NT * NV, ++chunk) {
    if (base == 0 || base + NT * NV >= end) {  // other rows' values, and what is past the part
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int v = base + k * NT + tid;
        if (v == 0 || v == nvec - 1) cut_vec<T>(raw[k], v * kVec - before, P.vocab);
        constexpr uint32_t low = Logit<T>::kLowest;
        if (v >= end) raw[k] = make_uint4(low, low, low, low);
      }
    }
    const float largest = largest_of<T>(raw);
    if (largest > p.m) move_to(p, largest);
    if (top > 0) {
      const bool here = base + tid < end;  // the thread has values in this chunk
      best = fmaxf(best, largest);
      seen |= here;
      if (((chunk & (chunk + 1)) == 0 || bound_x == -INFINITY) && end - begin > top) {
        // a new bound: the top-th largest of 64 maxima, each of NT / 64 threads
        uint32_t m = seen ? order_bits(best) : 0u;
#pragma unroll
        for (int o = 1; o < NT / 64; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        uint32_t* maxima = reinterpret_cast<uint32_t*>(s.maxima);
        if (tid % (NT / 64) == 0) maxima[tid / (NT / 64)] = m;
        uint32_t* bound = &s.bound[found++ & 1];
        if (tid == 0) *bound = 0xffffffffu;
        __syncthreads();
        if (tid < 64) {
          const uint32_t mine = maxima[tid];
          int larger = 0;
#pragma unroll 4
          for (int i = 0; i < 16; ++i) {
            const uint4 u = s.maxima[i];
            larger += (u.x > mine) + (u.y > mine) + (u.z > mine) + (u.w > mine);
          }
          const uint32_t least = __reduce_min_sync(0xffffffffu, larger < top ? mine : 0xffffffffu);
          if (lane == 0) atomicMin(bound, least);
        }
        __syncthreads();
        const float x = order_value(*bound);
        if (x > bound_x) bound_x = x;
      }
      if (here && largest >= bound_x && largest > -INFINITY) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if (largest_of<T>(raw[k]) >= bound_x && base + k * NT + tid < end) {
            const int at = atomicAdd(&s.queued, 1);
            if (at < kLogpQueue) s.queue[at] = raw[k], s.queue_at[at] = base + k * NT + tid;
          }
      }
    }
    if (by_one) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        Raw<T, kVec> r;
        r.w[0] = raw[k];
        float x[kVec];
        unpack_row<T, kVec>(r, x);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int v = base + k * NT + tid, id = v * kVec + i - before;
          better += x[i] > x_token || (x[i] == x_token && v < end && id >= 0 && id < token);
        }
      }
    }
    uint32_t count = 0;
    const T* t = nullptr;
    const int next = base + NT * NV + tid;  // on the way while this chunk is summed
    // a likely token has few before it: most warps have none to count (2208 rows of 151680 where none has, 120 us against 130)
    const bool counting = __any_sync(0xffffffffu, largest >= x_token);
    if (fabsf(p.m) <= Logit<T>::kNear) {
      // exp2(x log2 e - c) with c = m log2 e rounded: one product a value, and what the rounding left out, rho, is put right
      // for all of the chunk.  Of values so far from the reference that they count as nothing it takes a finite one.
      const float c = p.m * kLog2e;
      const float rho = fmaf(p.m, kLog2e, -c);
      // (one value at a time: packed pairs took 140 us where this takes 126, 2208 rows of 151680 without alternatives)
      float sum0 = 0.0f, sum1 = 0.0f, dot0 = 0.0f, dot1 = 0.0f;
      auto add = [&](float x, float& sum, float& dot) {
        const float d = fmaf(x, kLog2e, -c), e = ex2_approx(d);
        sum += e;
        dot = fmaf(e, d, dot);
      };
      auto take = [&](int k, auto counts) {
        const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
        raw[k] = load_vec(next + k * NT);
        const uint32_t limit = base + k * NT + tid < v_token ? at_or_above : above;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float a = __uint_as_float(w[i]), b = __uint_as_float(w[i + 1]);
            if constexpr (counts.value) count += a > __uint_as_float(limit), count += b > __uint_as_float(limit);
            add(max_nan(a, -1e30f), sum0, dot0);
            add(max_nan(b, -1e30f), sum1, dot1);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (counts.value) count2(count, w[i], limit);
            const float2 x = unpack2(max2_nan(w[i], Logit<T>::kFloor, t), t);
            add(x.x, sum0, dot0);
            add(x.y, sum1, dot1);
          }
        }
      };
      auto take_all = [&](auto counts) {
        if (base + NT * (NV - 1) < end) {
#pragma unroll
          for (int k = 0; k < NV; ++k) take(k, counts);
        } else {  // a row's last chunk, or its only one
#pragma unroll
          for (int k = 0; k < NV - 1; ++k)
            if (base + k * NT < end) take(k, counts);
        }
      };
      if (counting)
        take_all(std::true_type{});
      else
        take_all(std::false_type{});
      const float f = ex2_approx(-rho), sum = f * (sum0 + sum1);
      p.s += sum;
      p.t += fmaf(-rho, sum, f * (dot0 + dot1));
    } else {
      float sum = 0.0f, sum_d = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        Raw<T, kVec> r, l;
        r.w[0] = raw[k];
        raw[k] = load_vec(next + k * NT);
        const uint32_t limit = base + k * NT + tid < v_token ? at_or_above : above;
        l.w[0] = make_uint4(limit, limit, limit, limit);
        float x[kVec], y[kVec];
        unpack_row<T, kVec>(r, x);
        unpack_row<T, kVec>(l, y);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const float d = max_nan((x[i] - p.m) * kLog2e, kLogpLeast), e = ex2_approx(d);
          sum += e;
          sum_d = fmaf(e, d, sum_d);
          better += x[i] > y[i];
        }
      }
      p.s += sum, p.t += sum_d;
    }
    if constexpr (sizeof(T) == 4) {
      better += count;
    } else {
      const float2 n = unpack2(count, static_cast<const __half*>(nullptr));
      better += static_cast<uint32_t>(n.x + n.y);
    }
  }

  // The warps leave their totals; of the queue's values those that reach the last bound go to the front.
  const Total mine = warp_total({p, better});
  if (lane == 0) s.totals[warp] = words_of(mine);
  if (top > 0) {
    __syncthreads();
    const int queued = s.queued;
    if (queued <= kLogpQueue)
      for (int i = tid; i < queued; i += NT) {
        Raw<T, kVec> r;
        r.w[0] = s.queue[i];
        float x[kVec];
        unpack_row<T, kVec>(r, x);
        const int id0 = s.queue_at[i] * kVec - before;
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (x[k] >= bound_x && x[k] > -INFINITY) {
            const int at = atomicAdd(&s.fronts, 1);
            if (at < NT) s.front[at] = key_of(x[k], id0 + k);
          }
      }
    __syncthreads();
    if (queued > kLogpQueue || s.fronts > NT) list_part<T, NT>(s, P.vocab, top, vecs, before, begin, end, nvec, bound_x);
  }
  if (cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  __syncthreads();
  const Total total = total_of(s.totals, kWarps);
  const int fronts = s.fronts;
  if (cluster == 1) {
    if (tid == 0) finish(P, row, s.token, s.x_token, total);
    if (top > 0) write_top<T>(P, row, s.front, fronts, tid, NT, total);
    return;
  }
  // Rank 0 gets up to 32 keys of every CTA: all, or where they are more the top ones.
  if (tid < fronts) {
    const u64 key = s.front[tid];
    const int place = fronts > kLogpTop ? place_of(s.front, fronts, key) : tid;
    if (place < kLogpTop) st_cluster_u64(mapa_shared(smem_u32(&s.sent[part * kLogpTop + place]), 0), key);
  }
  if (tid == 0) {
    const uint4 w = words_of(total);
    st_cluster_u64(mapa_shared(smem_u32(&s.sent_totals[part]), 0), pair_of(w.x, w.y));
    st_cluster_u64(mapa_shared(smem_u32(&s.sent_totals[part]) + 8, 0), pair_of(w.z, w.w));
    st_cluster_u64(mapa_shared(smem_u32(&s.sent_n[part]), 0), pair_of(min(fronts, kLogpTop), found ? s.bound[(found - 1) & 1] : 0u));
    s.finalists = 0;
  }
  cluster_sync();
  if (part > 0) return;  // nothing is written to another CTA from here on
  const Total row_total = total_of(s.sent_totals, cluster);
  if (tid == 0) finish(P, row, s.token, s.x_token, row_total);
  const uint2 mine_n = lane < cluster ? s.sent_n[lane] : make_uint2(0, 0);
  const uint32_t row_bound = __reduce_max_sync(0xffffffffu, mine_n.y);
  for (int e = tid; e < cluster * kLogpTop; e += NT)
    if (e % kLogpTop < static_cast<int>(s.sent_n[e / kLogpTop].x) && static_cast<uint32_t>(s.sent[e] >> 32) >= row_bound)
      s.final[atomicAdd(&s.finalists, 1)] = s.sent[e];
  __syncthreads();
  if (top > 0) write_top<T>(P, row, s.final, s.finalists, tid, NT, row_total);
}

template <typename T, int NT>
cudaError_t launch_logprobs(const LogprobsParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * static_cast<unsigned>(p.cluster), 1, 1);
  cfg.blockDim = dim3(NT, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, NT>, p);
}
template <typename T>
cudaError_t launch_logprobs(LogprobsParams p, cudaStream_t stream) {
  // Threads of a CTA.  A row's latency is shortest with 256, the search for its top costs least with 64, so the most threads are
  // taken with which all rows run at once (1024 threads an SM), or in two turns if the rows are past 8 KB; no more than a row has
  // vectors, and 256 past 64 KB, where the search no longer counts.  us with 64, 128 and 256, bf16:
  //   x 4096: 300 rows 15.0  9.8  7.3, 600 rows 14.7  8.8 10.1, 4000 rows 26.3 28.3 42.7
  //   x 16331: 300 rows 18.8 14.5 11.5, 1200 rows 30.4 26.0 25.7, 4000 rows 59.9 61.4 69.9;  4000 x 40000: 111 111 115
  // CTAs of a row: up to 8, until they would take a quarter of the threads that run at once, and none with less
  // than a vector a thread.  (Up to half of them, us: 64 x 50257 fp32 14.3 against 11.6, 64 x 20000 12.2 against 7.8, 256 x
  // 151680 31.8 against 33.3; up to 16 CTAs a row: 8 x 151680 17.4 against 11.4, one row 14.6 against 10.5.)
  const long long vecs = static_cast<long long>(p.vocab) * sizeof(T) / 16;
  const long long at_once = (vecs <= 512 ? 1024LL : 2048LL) * sm_count();
  int nt = 256;
  while (nt > 64 && vecs <= 4096 && (vecs < nt || static_cast<long long>(p.rows) * nt > at_once)) nt /= 2;
  p.cluster = 1;
  while (p.cluster < kLogpMaxCluster && static_cast<long long>(p.rows) * p.cluster * nt < 384LL * sm_count() && vecs / (2 * p.cluster) >= nt) p.cluster *= 2;
  if (nt == 64) return launch_logprobs<T, 64>(p, stream);
  if (nt == 128) return launch_logprobs<T, 128>(p, stream);
  return launch_logprobs<T, 256>(p, stream);
}
}  // namespace

}  // namespace rldx

using namespace rldx;

extern "C" int rldx_token_logprobs(const void* logits, int64_t ld, int rows, int vocab, int dtype, const int64_t* tokens, int top,
                                   float* logprob, float* entropy, int32_t* rank, int64_t* top_ids, float* top_logprobs, void* stream) {
  auto bad = [](const char* what) { return set_error(RLDX_ERR_ARG, std::string("token_logprobs: ") + what); };
  if (rows < 0 || vocab <= 0 || ld < 0) return bad("need rows >= 0, vocab > 0, ld >= 0");
  if (!known_dtype(dtype)) return set_error(RLDX_ERR_UNSUPPORTED, "token_logprobs: unknown type");
  if (vocab > kLogpMaxVocab) return set_error(RLDX_ERR_UNSUPPORTED, "token_logprobs: a vocabulary has at most 2^28 tokens");
  if (top < 0 || top > kLogpTop || top > vocab)
    return set_error(RLDX_ERR_UNSUPPORTED, "token_logprobs: 0 to " + std::to_string(kLogpTop) + " alternatives, no more than tokens");
  if (rows > INT32_MAX / kLogpMaxCluster) return set_error(RLDX_ERR_UNSUPPORTED, "token_logprobs: too many rows");
  if (rows == 0) return RLDX_OK;
  if (!logits || !tokens || !logprob || !entropy || !rank || (top && (!top_ids || !top_logprobs))) return bad("null pointer");
  if (reinterpret_cast<uintptr_t>(logits) % dtype_bytes(dtype)) return bad("misaligned logits");
  auto off = [](const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; };
  if (off(tokens, 8) || off(logprob, 4) || off(entropy, 4) || off(rank, 4) || (top && (off(top_ids, 8) || off(top_logprobs, 4))))
    return bad("misaligned tokens or results");
  int rc = ensure_device();
  if (rc != RLDX_OK) return rc;
  LogprobsParams p;
  p.logits = logits, p.ld = ld, p.rows = rows, p.vocab = vocab, p.top = top;
  p.tokens = reinterpret_cast<const long long*>(tokens);
  p.logprob = logprob, p.entropy = entropy, p.rank = rank;
  p.top_ids = reinterpret_cast<long long*>(top_ids), p.top_logprobs = top_logprobs;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == RLDX_F32   ? launch_logprobs<float>(p, st)
                        : dtype == RLDX_F16 ? launch_logprobs<__half>(p, st)
                                            : launch_logprobs<__nv_bfloat16>(p, st);
  if (e != cudaSuccess) return cuda_fail(e, "token_logprobs launch");
  return RLDX_OK;
}
