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
constexpr int kLogpThreads = 256;
constexpr int kLogpVecs = 8;        // 16-byte vectors of a thread and chunk
// A list is cut down to k when it is longer than kLogpPrune after a chunk; a chunk adds the values of at most k threads.
constexpr int kLogpPrune = 256;
constexpr int kLogpMaxValues = kLogpVecs * 8;  // of a thread and chunk
constexpr int kLogpList = kLogpPrune + kLogpTop * kLogpMaxValues;
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
  float4 warps[kLogpThreads / 32];
  u64 bound;
  int count;
};

template <typename T>
struct LogitBits;  // a vector's worth of -inf, and how many leading bits tell values of T apart
template <>
struct LogitBits<__nv_bfloat16> {
  static constexpr uint32_t kLowest = 0xff80ff80u;
  static constexpr int kBits = 16;
};
template <>
struct LogitBits<__half> {
  static constexpr uint32_t kLowest = 0xfc00fc00u;
  static constexpr int kBits = 19;  // of its fp32 form: sign, 8 exponent and 10 mantissa bits
};
template <>
struct LogitBits<float> {
  static constexpr uint32_t kLowest = 0xff800000u;
  static constexpr int kBits = 32;
};

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

// Cuts the list down to the k best, s.bound the last of them.  Every thread calls it; s.count > k.
__device__ __forceinline__ void prune(LogprobsShared& s, int k) {
  constexpr int kEach = (kLogpList + kLogpThreads - 1) / kLogpThreads;
  const int n = min(s.count, kLogpList);
  u64 mine[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int at = threadIdx.x + i * kLogpThreads;
    mine[i] = at < n ? s.list[at] : 0;
  }
  // keys differ: the k-th largest, bit by bit
  u64 t = 0;
#pragma unroll 1
  for (int b = 63; b >= 0; --b) {
    const u64 c = t | (1ull << b);
    int mine_reach = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) mine_reach += mine[i] >= c;
    // sums of more than one a thread: by warps, then over them
    mine_reach = __reduce_add_sync(0xffffffffu, mine_reach);
    int* sums = reinterpret_cast<int*>(s.warps) + (b & 1) * (kLogpThreads / 32);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = mine_reach;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < kLogpThreads / 32; ++w) all += sums[w];
    if (all >= k) t = c;
  }
  if (threadIdx.x == 0) s.count = 0, s.bound = t;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (mine[i] >= t) s.list[atomicAdd(&s.count, 1)] = mine[i];
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kLogpThreads) logprobs_kernel(const __grid_constant__ LogprobsParams P) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int NT = kLogpThreads, NV = kLogpVecs;
  __shared__ LogprobsShared s;
  const int cluster = P.cluster;
  const int part = cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const long long row = blockIdx.x / cluster;
  if (cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (rank 0 runs before it is written to)
  griddep_wait();
  griddep_launch();
  const int top = P.top;
  if (threadIdx.x == 0) s.count = 0, s.bound = 0;
  const T* logits = static_cast<const T*>(P.logits) + row * P.ld;
  // vectors on 16-byte boundaries, the first and the last in part of other rows
  const int before = static_cast<int>(reinterpret_cast<uintptr_t>(logits) % 16 / sizeof(T));
  const uint4* vecs = reinterpret_cast<const uint4*>(logits - before);
  const int nvec = static_cast<int>((static_cast<long long>(P.vocab) + before + kVec - 1) / kVec);
  const int per = (nvec + cluster - 1) / cluster;
  const int v_end = min(nvec, (part + 1) * per);
  const long long token = P.tokens[row];
  const bool given = token >= 0 && token < P.vocab;
  const float x_token = given ? to_float(logits[token]) : INFINITY;
  // equal logits count up to here: before the token, and in this part (what fills up its last chunk is -inf too)
  const int id_token = given ? static_cast<int>(min(token, static_cast<long long>(v_end) * kVec - before)) : 0;

  Partial p{-FLT_MAX, 0.0f, 0.0f};
  float best = -INFINITY;  // this thread's largest logit so far, where it has seen one
  bool seen = false;
  uint32_t better = 0;  // tokens before the given one
  __syncthreads();

#pragma unroll 1
  for (int base = part * per; base < v_end; base += NT * NV) {
    uint4 raw[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = base + k * NT + static_cast<int>(threadIdx.x);
      if (v < v_end)
        raw[k] = __ldcs(vecs + v);
      else
        raw[k] = make_uint4(LogitBits<T>::kLowest, LogitBits<T>::kLowest, LogitBits<T>::kLowest, LogitBits<T>::kLowest);
      if (v == 0 || v == nvec - 1) {  // values of other rows
        T* e = reinterpret_cast<T*>(&raw[k]);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int id = v * kVec + i - before;
          if (id < 0 || id >= P.vocab) e[i] = from_float<T>(-INFINITY);
        }
      }
    }
    auto values = [&](int k, float (&x)[kVec]) {
      Raw<T, kVec> r;
      r.w[0] = raw[k];
      unpack_row<T, kVec>(r, x);
    };
    float largest = -INFINITY;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float x[kVec];
      values(k, x);
#pragma unroll
      for (int i = 0; i < kVec; ++i) largest = fmaxf(largest, x[i]);
    }
    if (largest > p.m) move_to(p, largest);
    float chunk_s = 0.0f, chunk_t = 0.0f;  // (short sums: a thread of a long row adds hundreds of values)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float x[kVec];
      values(k, x);
      const int id0 = (base + k * NT + static_cast<int>(threadIdx.x)) * kVec - before;  // (before the row: x is -inf there)
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float d = max_nan((x[i] - p.m) * kLog2e, kLogpLeast), e = ex2_approx(d);
        chunk_s += e;
        chunk_t = fmaf(e, d, chunk_t);
        better += x[i] > x_token || (x[i] == x_token && id0 + i >= 0 && id0 + i < id_token);
      }
    }
    p.s += chunk_s, p.t += chunk_t;
    if (top == 0) continue;
    const u64 bound = s.bound;  // 0: none yet
    const float bound_x = bound ? order_value(static_cast<uint32_t>(bound >> 32)) : -INFINITY;
    const int bound_id = bound ? static_cast<int>(~static_cast<uint32_t>(bound)) : INT32_MAX;
    const int id0 = (base + static_cast<int>(threadIdx.x)) * kVec - before;
    const bool here = base + static_cast<int>(threadIdx.x) < v_end;  // the thread has values in this chunk
    const bool rises = here && (largest > bound_x || (largest == bound_x && id0 <= bound_id));
    const bool earlier = seen;
    const float earlier_best = best;
    best = fmaxf(best, largest);
    seen |= here;
    const int rising = __syncthreads_count(rises);
    if (rising == 0) continue;
    float new_x = bound_x;
    int new_id = bound_id;
    if (rising > top) {
      // a new bound: the top-th largest of the threads' maxima
      constexpr int low = 32 - LogitBits<T>::kBits;
      const uint32_t bits = seen ? order_bits(best) : 0u;
      uint32_t t = reached_by(top, 31, low, [&](uint32_t c) { return bits >= c; });
      if (!(t >> 31)) t |= (1u << low) - 1u;  // (negative values: the bits that the type does not have are ones)
      const float tx = order_value(t);
      if (tx >= bound_x) {
        const int above = __syncthreads_count(bits > t), tied = __syncthreads_count(bits == t);
        new_id = tx > bound_x ? INT32_MAX : bound_id;
        new_x = tx;
        if (tied > top - above) {
          // of those that share the value the lowest ids; one of an earlier chunk counts as lower than any here
          int id = INT32_MAX;
          if (earlier && earlier_best == tx) {
            id = 0;
          } else if (bits == t) {
#pragma unroll
            for (int k = NV - 1; k >= 0; --k) {
              float x[kVec];
              values(k, x);
#pragma unroll
              for (int i = kVec - 1; i >= 0; --i) {
                const int at = id0 + k * NT * kVec + i;
                if (x[i] == tx && at >= 0 && at < P.vocab) id = at;
              }
            }
          }
          const uint32_t order = bits == t ? static_cast<uint32_t>(INT32_MAX - id) : 0u;
          const uint32_t r = reached_by(top - above, 30, 0, [&](uint32_t c) { return order >= c; });
          new_id = min(new_id, INT32_MAX - static_cast<int>(r));
        }
      }
    }
    if (rises && largest >= new_x) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float x[kVec];
        values(k, x);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int id = id0 + k * NT * kVec + i;
          if ((x[i] > new_x || (x[i] == new_x && id <= new_id)) && id >= 0 && base + k * NT + static_cast<int>(threadIdx.x) < v_end && id < P.vocab) {
            const int at = atomicAdd(&s.count, 1);
            if (at < kLogpList) s.list[at] = key_of(x[i], id);
          }
        }
      }
    }
    __syncthreads();
    const int listed = s.count;
    if (threadIdx.x == 0 && (new_x != bound_x || new_id != bound_id)) s.bound = key_of(new_x, new_id);
    __syncthreads();
    if (listed > kLogpPrune) prune(s, top);
  }

  // the part's sums
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Partial q{__shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.s, o), __shfl_xor_sync(0xffffffffu, p.t, o)};
    join(p, q);
  }
  better = __reduce_add_sync(0xffffffffu, better);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) s.warps[warp] = make_float4(p.m, p.s, p.t, __uint_as_float(better));
  __syncthreads();
  // and its list go to rank 0
  if (cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int listed = s.count;  // at most kLogpPrune, a thread each
  if (static_cast<int>(threadIdx.x) < listed) {
    const u64 mine = s.list[threadIdx.x];
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

template <typename T>
cudaError_t launch_logprobs(const LogprobsParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * static_cast<unsigned>(p.cluster), 1, 1);
  cfg.blockDim = dim3(kLogpThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, p);
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
  // CTAs of a row: as few as fill the SMs, and none with less than a vector a thread
  const long long vecs = static_cast<long long>(vocab) * dtype_bytes(dtype) / 16;
  p.cluster = 1;
  while (p.cluster < kLogpMaxCluster && static_cast<long long>(rows) * p.cluster < 3LL * sm_count() && vecs / (2 * p.cluster) >= kLogpThreads)
    p.cluster *= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == RLDX_F32   ? launch_logprobs<float>(p, st)
                        : dtype == RLDX_F16 ? launch_logprobs<__half>(p, st)
                                            : launch_logprobs<__nv_bfloat16>(p, st);
  if (e != cudaSuccess) return cuda_fail(e, "token_logprobs launch");
  return RLDX_OK;
}
