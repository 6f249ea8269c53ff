// Log probabilities of given tokens under rows of logits, with the entropy of each row, the token's rank and the
// top alternatives, in one pass over the logits.
//
// With M the row's maximum, d_i = x_i - M, S = sum exp(d_i) and T = sum exp(d_i) d_i:
//   log p_i = d_i - ln S,   H = ln S - T / S  (both terms positive: nothing cancels),
//   rank of t = the number of i with x_i > x_t, or x_i = x_t and i < t,
//   top: the k first in the order of descending logits, equal ones by ascending id.
// Sums and statistics are fp32, each thread's relative to the largest logit that it has seen; two of them are joined
// by moving the smaller reference to the larger.
//
// A row is shared out among the CTAs of a cluster, each of which goes over its part in chunks of 32 KB that its threads
// hold in registers.  The top k of a part: the k-th largest of the threads' maxima is a lower bound of the k-th largest
// value, so what reaches it is a little more than k tokens, and it comes from at most k threads.  Those go to a list in
// shared memory as (ordered bits of the logit, ~id), whose order is the answer's.  Bounds only rise, and where more
// threads share the bounding value than are needed the lowest ids decide, so a row of equal logits lists no more.
#include <cfloat>

#include "host_util.h"
#include "rows.cuh"

namespace rldx {

namespace {
constexpr int kLogpTop = 32;        // alternatives at most
constexpr int kLogpMaxCluster = 8;
constexpr int kLogpVecs = 8;        // 16-byte vectors of a thread and chunk
// A list is cut down to k before it could overflow: a chunk adds the values of at most k threads.
constexpr int kLogpRoom = kLogpTop * kLogpVecs * 8;
constexpr int kLogpList = kLogpRoom + 512;
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
__device__ __forceinline__ void join(Partial& a, Partial b) {
  const float m = fmaxf(a.m, b.m);
  move_to(a, m);
  move_to(b, m);
  a.s += b.s, a.t += b.t;
}

struct LogprobsShared {
  u64 list[kLogpList];
  u64 top[kLogpMaxCluster][kLogpTop];  // rank 0: every CTA's, in order
  u64 stats[kLogpMaxCluster][2];       // rank 0: m, s, t and the count of better tokens of every CTA
  u64 tops[kLogpMaxCluster];           // rank 0: the lengths of the lists
  float4 warps[16];
  u64 kept[kLogpTop];
  u64 bound;
  int count;
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
// Ones where a > b, added up in halves of a word (whole numbers up to 256 there).
__device__ __forceinline__ void count2(uint32_t& n, uint32_t a, uint32_t b, const __nv_bfloat16*) {
  const __nv_bfloat162 r = __hadd2(*reinterpret_cast<__nv_bfloat162*>(&n), __hgt2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b)));
  n = *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void count2(uint32_t& n, uint32_t a, uint32_t b, const __half*) {
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
__device__ __forceinline__ float largest_of(const uint4 (&raw)[kLogpVecs]) {
  if constexpr (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kLogpVecs; ++k)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(raw[k].x), __uint_as_float(raw[k].y)), fmaxf(__uint_as_float(raw[k].z), __uint_as_float(raw[k].w))));
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

__device__ __forceinline__ u64 key_of(float x, int id) {
  return (static_cast<u64>(order_bits(x)) << 32) | static_cast<uint32_t>(~id);
}

__device__ __forceinline__ u64 pair_of(uint32_t lo, uint32_t hi) { return (static_cast<u64>(hi) << 32) | lo; }
// Writes to the same place of the cluster's first CTA.
__device__ __forceinline__ void store_to_first(u64* place, u64 v, int cluster) {
  if (cluster > 1)
    st_cluster_u64(mapa_shared(smem_u32(place), 0), v);
  else
    *place = v;
}

// The largest t, in bits top_bit to low_bit, that at least `need` of the threads' numbers reach; 0 where there are fewer.
template <typename F>
__device__ __forceinline__ uint32_t reached_by(int need, int top_bit, int low_bit, F reaches) {
  uint32_t t = 0;
#pragma unroll 1
  for (int b = top_bit; b >= low_bit; --b)
    if (__syncthreads_count(reaches(t | (1u << b))) >= need) t |= 1u << b;
  return t;
}

// Cuts the list down to the k best, s.bound the last of them.  Every thread calls it after a barrier; s.count >= k.
template <int NT>
__device__ __forceinline__ void prune(LogprobsShared& s, int k) {
  const int n = min(s.count, kLogpList);
  int* sums = reinterpret_cast<int*>(s.warps);
  // keys differ: the k-th largest, bit by bit
  u64 t = 0;
#pragma unroll 1
  for (int b = 63; b >= 0; --b) {
    const u64 c = t | (1ull << b);
    int reach = 0;
    for (int i = threadIdx.x; i < n; i += NT) reach += s.list[i] >= c;
    reach = __reduce_add_sync(0xffffffffu, reach);
    int* at = sums + (b & 1) * (NT / 32);
    if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = reach;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < NT / 32; ++w) all += at[w];
    if (all >= k) t = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0, s.bound = t;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT)
    if (s.list[i] >= t) s.kept[atomicAdd(&s.count, 1)] = s.list[i];
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < k) s.list[threadIdx.x] = s.kept[threadIdx.x];
  __syncthreads();
}

// NT threads a CTA.
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 768 / NT) logprobs_kernel(const __grid_constant__ LogprobsParams P) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int NV = kLogpVecs;
  __shared__ LogprobsShared s;
  const int cluster = P.cluster;
  const int part = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const long long row = blockIdx.x / cluster;
  if (cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (rank 0 runs before it is written to)
  griddep_wait();
  griddep_launch();
  const int top = P.top;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) s.count = 0;
  const T* logits = static_cast<const T*>(P.logits) + row * P.ld;
  // vectors on 16-byte boundaries, the first and the last in part of other rows
  const int before = static_cast<int>(reinterpret_cast<uintptr_t>(logits) % 16 / sizeof(T));
  const uint4* vecs = reinterpret_cast<const uint4*>(logits - before);
  const int nvec = static_cast<int>((static_cast<long long>(P.vocab) + before + kVec - 1) / kVec);
  const int per = (nvec + cluster - 1) / cluster;
  const int v_begin = part * per, v_end = min(nvec, v_begin + per);

  // vector v of this part, -inf where there is none
  auto load_vec = [&](int v) {
    constexpr uint32_t low = Logit<T>::kLowest;
    uint4 u = make_uint4(low, low, low, low);
    if (v < v_end) u = __ldcs(vecs + v);
    return u;
  };
  // and -inf in the place of other rows' values
  auto cut = [&](uint4& u, int v) {
    if (v == 0 || v == nvec - 1) {
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const int id = v * kVec + i - before;
        if (id < 0 || id >= P.vocab) e[i] = from_float<T>(-INFINITY);
      }
    }
  };
  uint4 raw[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) raw[k] = load_vec(v_begin + k * NT + tid);

  const long long token = P.tokens[row];
  const bool given = token >= 0 && token < P.vocab;
  const T t_token = given ? logits[token] : from_float<T>(INFINITY);
  const float x_token = to_float(t_token);
  // Tokens before the given one: of vectors before its own those at or above it, of the others those above, and those of
  // its own vector that equal it and come before it.  Where it is -inf, which also fills up vectors, all are looked at.
  const bool by_one = given && x_token == -INFINITY;
  const int v_token = given ? static_cast<int>((token + before) / kVec) : 0;
  const uint32_t above = both(by_one ? from_float<T>(INFINITY) : t_token);
  const uint32_t at_or_above = both(given && x_token < INFINITY && !by_one ? below(t_token) : from_float<T>(INFINITY));
  uint32_t better = 0;
  if (given && !by_one && tid < kVec && part == v_token / per) {
    const long long id = static_cast<long long>(v_token) * kVec + tid - before;
    if (id >= 0 && id < token) better = to_float(logits[id]) == x_token;
  }

  Partial p{-FLT_MAX, 0.0f, 0.0f};
  float best = -INFINITY;  // this thread's largest logit so far, where it has seen one
  bool seen = false;
  // What can be among the top: values above bound_x, and those that equal it up to bound_id.  The same for every thread.
  float bound_x = -INFINITY;
  int bound_id = INT32_MAX;
  int room = kLogpList;  // in the list, at least
  __syncthreads();

#pragma unroll 1
  for (int base = v_begin; base < v_end; base += NT * NV) {
    if (base == 0 || base + NT * NV >= nvec)
#pragma unroll
      for (int k = 0; k < NV; ++k) cut(raw[k], base + k * NT + tid);
    const float largest = largest_of<T>(raw);
    if (largest > p.m) move_to(p, largest);
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
          better += x[i] > -INFINITY || (x[i] == -INFINITY && v < v_end && id >= 0 && id < token);
        }
      }
    }
    uint32_t count = 0;
    const T* t = nullptr;
    const int next = base + NT * NV + tid;
    if (fabsf(p.m) <= Logit<T>::kNear) {
      // exp2(x log2 e - c) with c = m log2 e rounded: one product a value, and what the rounding left out, rho, is put right
      // for all of the chunk.  Of values so far from the reference that they count as nothing it takes a finite one.
      const float c = p.m * kLog2e;
      const float rho = fmaf(p.m, kLog2e, -c);
      const float2 l2 = make_float2(kLog2e, kLog2e), c2 = make_float2(-c, -c);
      float2 s2 = make_float2(0.0f, 0.0f), t2 = s2;
      auto add = [&](float2 x) {
        const float2 d = fma_f32x2(x, l2, c2);
        const float2 e = make_float2(ex2_approx(d.x), ex2_approx(d.y));
        s2 = add_f32x2(s2, e);
        t2 = fma_f32x2(e, d, t2);
      };
      auto take = [&](int k) {
        const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
        raw[k] = load_vec(next + k * NT);
        const uint32_t limit = base + k * NT + tid < v_token ? at_or_above : above;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float a = __uint_as_float(w[i]), b = __uint_as_float(w[i + 1]);
            count += a > __uint_as_float(limit), count += b > __uint_as_float(limit);
            add(make_float2(max_nan(a, -1e30f), max_nan(b, -1e30f)));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            count2(count, w[i], limit, t);
            add(unpack2(max2_nan(w[i], Logit<T>::kFloor, t), t));
          }
        }
      };
      if (base + NT * (NV - 1) < v_end) {
#pragma unroll
        for (int k = 0; k < NV; ++k) take(k);
      } else {  // a row's last chunk, or its only one
#pragma unroll
        for (int k = 0; k < NV - 1; ++k)
          if (base + k * NT < v_end) take(k);
      }
      const float f = ex2_approx(-rho), sum = f * (s2.x + s2.y);
      p.s += sum;
      p.t += fmaf(-rho, sum, f * (t2.x + t2.y));
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
      const float2 n = unpack2(count, t);
      better += static_cast<uint32_t>(n.x + n.y);
    }

    if (top == 0) continue;
    const int id0 = (base + tid) * kVec - before;
    const bool here = base + tid < v_end;  // the thread has values in this chunk
    const bool rises = here && (largest > bound_x || (largest == bound_x && id0 <= bound_id));
    const bool earlier = seen;
    const float earlier_best = best;
    best = fmaxf(best, largest);
    seen |= here;
    const int rising = __syncthreads_count(rises);
    if (rising == 0) continue;
    if (rising > top) {
      // a new bound: the top-th largest of the threads' maxima
      constexpr int low = 32 - Logit<T>::kBits;
      const uint32_t bits = seen ? order_bits(best) : 0u;
      uint32_t reach = reached_by(top, 31, low, [&](uint32_t c) { return bits >= c; });
      if (!(reach >> 31)) reach |= (1u << low) - 1u;  // (negative values: the bits that the type does not have are ones)
      const float tx = order_value(reach);
      if (tx >= bound_x) {
        const int higher = __syncthreads_count(bits > reach), tied = __syncthreads_count(bits == reach);
        if (tx > bound_x) bound_id = INT32_MAX;
        bound_x = tx;
        if (tied > top - higher) {
          // of those that share the value the lowest ids; one of an earlier chunk counts as lower than any here
          int id = INT32_MAX;
          if (earlier && earlier_best == tx) {
            id = 0;
          } else if (bits == reach) {
#pragma unroll 1
            for (int k = NV - 1; k >= 0; --k) {
              Raw<T, kVec> r;
              r.w[0] = load_vec(base + k * NT + tid);
              float x[kVec];
              unpack_row<T, kVec>(r, x);
#pragma unroll
              for (int i = kVec - 1; i >= 0; --i) {
                const int at = id0 + k * NT * kVec + i;
                if (x[i] == tx && base + k * NT + tid < v_end && at >= 0 && at < P.vocab) id = at;
              }
            }
          }
          const uint32_t order = bits == reach ? static_cast<uint32_t>(INT32_MAX - id) : 0u;
          const uint32_t r = reached_by(top - higher, 30, 0, [&](uint32_t c) { return order >= c; });
          bound_id = min(bound_id, INT32_MAX - static_cast<int>(r));
        }
      }
    }
    // At most `top` threads add values now, whose bound is as good as that of the list's last.
    const int added = min(rising, top) * NV * kVec;
    if (room < added) {  // (counted anew, it is more: a thread seldom adds all its values)
      __syncthreads();
      const int free = kLogpList - s.count;
      if (free < added) {
        prune<NT>(s, top);
        if (s.bound > key_of(bound_x, bound_id))
          bound_x = order_value(static_cast<uint32_t>(s.bound >> 32)), bound_id = static_cast<int>(~static_cast<uint32_t>(s.bound));
      }
      room = kLogpList - s.count;
      __syncthreads();
    }
    room -= added;
    // what reaches the bound: a warp reads the vectors of four such threads at a time again
    uint32_t who = __ballot_sync(0xffffffffu, rises && largest >= bound_x);
    while (who) {
      int mine = -1;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (who && lane >> 3 == g) mine = __ffs(who) - 1;
        who &= who - 1;
      }
      const int v = base + (lane & 7) * NT + warp * 32 + mine;
      if (mine >= 0 && v < v_end) {
        Raw<T, kVec> r;
        r.w[0] = load_vec(v);
        float x[kVec];
        unpack_row<T, kVec>(r, x);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int id = v * kVec + i - before;
          if ((x[i] > bound_x || (x[i] == bound_x && id <= bound_id)) && id >= 0 && id < P.vocab) {
            const int at = atomicAdd(&s.count, 1);
            if (at < kLogpList) s.list[at] = key_of(x[i], id);
          }
        }
      }
    }
  }

  // the part's sums
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Partial q{__shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.s, o), __shfl_xor_sync(0xffffffffu, p.t, o)};
    join(p, q);
  }
  better = __reduce_add_sync(0xffffffffu, better);
  __syncthreads();
  if (s.count > NT) prune<NT>(s, top);  // (NT >= 64 > top)
  if (lane == 0) s.warps[warp] = make_float4(p.m, p.s, p.t, __uint_as_float(better));
  __syncthreads();
  // and its list go to rank 0
  if (cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int listed = s.count;  // a thread each
  if (tid < listed) {
    const u64 mine = s.list[tid];
    int place = 0;
    for (int i = 0; i < listed; ++i) place += s.list[i] > mine;
    if (place < top) store_to_first(&s.top[part][place], mine, cluster);
  }
  if (warp == 0) {
    const float4 w = lane < NT / 32 ? s.warps[lane] : make_float4(-FLT_MAX, 0.0f, 0.0f, 0.0f);
    p = Partial{w.x, w.y, w.z};
    better = __float_as_uint(w.w);
#pragma unroll
    for (int o = NT / 64; o > 0; o >>= 1) {
      const Partial q{__shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.s, o), __shfl_xor_sync(0xffffffffu, p.t, o)};
      join(p, q);
      better += __shfl_xor_sync(0xffffffffu, better, o);
    }
    if (lane == 0) {
      store_to_first(&s.stats[part][0], pair_of(__float_as_uint(p.m), __float_as_uint(p.s)), cluster);
      store_to_first(&s.stats[part][1], pair_of(__float_as_uint(p.t), better), cluster);
      store_to_first(&s.tops[part], static_cast<u64>(min(listed, top)), cluster);
    }
  }
  if (cluster > 1) {
    cluster_sync();
    if (part > 0) return;  // nothing is written to another CTA from here on
  } else {
    __syncthreads();
  }

  // every warp joins the parts
  p = Partial{-FLT_MAX, 0.0f, 0.0f};
  better = 0;
  for (int c = 0; c < cluster; ++c) {
    const u64 a = s.stats[c][0], b = s.stats[c][1];
    join(p, Partial{__uint_as_float(static_cast<uint32_t>(a)), __uint_as_float(static_cast<uint32_t>(a >> 32)), __uint_as_float(static_cast<uint32_t>(b))});
    better += static_cast<uint32_t>(b >> 32);
  }
  const bool good = p.s > 0.0f && p.s < INFINITY;  // else NaN or +inf is in the row, or nothing but -inf
  const float log_s = logf(p.s);
  if (threadIdx.x == 0) {
    if (token >= P.vocab) record_data_error(kErrLogprobsToken);
    P.logprob[row] = token < 0 ? 0.0f : given && good ? (x_token - p.m) - log_s : NAN;
    P.rank[row] = given && good ? static_cast<int>(better) : -1;
    P.entropy[row] = good ? log_s - kLn2 * (p.t / p.s) : NAN;
  }
  for (int e = threadIdx.x; e < cluster * top; e += NT) {
    const int c = e / top, i = e - c * top;
    if (!good) {
      if (c == 0) P.top_ids[row * top + i] = -1, P.top_logprobs[row * top + i] = NAN;
      continue;
    }
    if (i >= static_cast<int>(s.tops[c])) continue;
    const u64 mine = s.top[c][i];
    int place = i;
    for (int o = 0; o < cluster; ++o) {
      if (o == c) continue;
      int lo = 0, hi = static_cast<int>(s.tops[o]);  // the keys of list o before mine
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s.top[o][mid] > mine)
          lo = mid + 1;
        else
          hi = mid;
      }
      place += lo;
    }
    if (place < top) {
      P.top_ids[row * top + place] = static_cast<long long>(~static_cast<uint32_t>(mine));
      P.top_logprobs[row * top + place] = (order_value(static_cast<uint32_t>(mine >> 32)) - p.m) - log_s;
    }
  }
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
  // Threads of a CTA: 64, of many small rows to an SM, where they hold one at a time; else 256.  CTAs of a row: as few as
  // fill the SMs, and none with less than a vector a thread.
  const long long vecs = static_cast<long long>(p.vocab) * sizeof(T) / 16;
  const int nt = vecs <= 64 * kLogpVecs ? 64 : 256;
  p.cluster = 1;
  while (p.cluster < kLogpMaxCluster && static_cast<long long>(p.rows) * p.cluster * nt < 768LL * sm_count() && vecs / (2 * p.cluster) >= nt)
    p.cluster *= 2;
  return nt == 64 ? launch_logprobs<T, 64>(p, stream) : launch_logprobs<T, 256>(p, stream);
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
