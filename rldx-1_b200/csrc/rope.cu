// Rotary positions: pairs (a, b) of a head's values turned by the angle p f_i of their pair i,
//   a' = m (a cos - b sin),  b' = m (b cos + a sin),
// with p the token's position on the pair's axis, f_i radians a position (double) and m a factor.  Pairs are
// (i, i + r / 2) or (2 i, 2 i + 1) of the head's first r values; the others pass unchanged.
//
// Angles: p f_i is reduced to a fraction of a turn in doubles, off by less than 2^-51 |p f_i| (two products and the constant 1 / (2 pi)):
// below fp32's own 2^-24 up to 2^27 radians.  (In fp32 the angle of a position of a million would be off by 0.06.)  The sine and
// cosine of that fraction come in fp32 with the part of it that fp32 drops added to first order.  Everything else is fp32 with one rounding to the output's type.
//
// A block takes a few tokens: its threads make each token's cos and sin once, in shared memory, while their first
// values are on the way, then turn the heads, V pairs a thread and step.  Bound by memory: every value is read and
// written once.  65536 tokens of 16 / 16 heads of 128 in bf16 take 154 us (6.97 TB/s; 1.07 GB at the copy's rate: 164), 8832
// of 16 / 2 heads 13.5 (floor 12.5), 20011 of 24 / 24 heads of 64 in fp32, 32 of each turned, 73.6 (75.1).
#include "host_util.h"
#include "rows.cuh"

namespace rldx {

namespace {
constexpr int kRopeMaxAxes = 4;
constexpr int kRopeMaxPairs = 512;
constexpr int kRopeItems = 2;  // of a thread and step, loaded before the first is turned

// n / d for n d < 2^32 by one multiplication: with m = ceil(2^32 / d) the quotient is off by n (m d - 2^32) / (2^32 d)
// < n / 2^32, less than the 1 / d that the next whole number is away.
struct SmallDiv {
  uint32_t m, d;
};
SmallDiv small_div(uint32_t d) { return {d == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + d - 1) / d), d}; }
__device__ __forceinline__ uint32_t quotient(uint32_t n, const SmallDiv& s) { return s.d == 1 ? n : __umulhi(n, s.m); }

struct RopeAngles {
  const void* pos;
  long long pos_ld;
  int pos64, axes;
  int sections[kRopeMaxAxes];
  int sections_interleaved;
  const double* freqs;
  int pairs;
  float factor;
  int inverse;
};
struct RopePart {
  const void* in;
  void* out;
  long long in_tok, in_head, out_tok, out_head;
  int heads;
};
struct RopeParams {
  RopePart part[2];
  RopeAngles a;
  long long tokens;
  int head_dim, tokens_per_block;
  int chunks;  // of V pairs in a head
  SmallDiv per_head, per_token;
};

__device__ __forceinline__ int rope_axis(const RopeAngles& a, int pair) {
  if (a.axes == 1) return 0;
  if (a.sections_interleaved) {
    const int x = pair % a.axes;
    return pair < a.axes * a.sections[x] ? x : 0;
  }
  int x = 0, end = 0;
#pragma unroll
  for (int i = 0; i < kRopeMaxAxes - 1; ++i) {
    end += a.sections[i];
    if (i + 1 < a.axes && pair >= end) x = i + 1;
  }
  return x;
}

// cos and sin of one pair of one token, with the factor and the direction.
__device__ __forceinline__ float2 rope_turn(const RopeAngles& a, long long token, int pair) {
  const long long at = rope_axis(a, pair) * a.pos_ld + token;
  const double p = a.pos64 ? static_cast<double>(__ldg(static_cast<const long long*>(a.pos) + at))
                           : static_cast<double>(__ldg(static_cast<const int*>(a.pos) + at));
  const double turns = p * __ldg(a.freqs + pair) * 0.15915494309189533577;  // 1 / (2 pi)
  const double halves = 2.0 * (turns - rint(turns));
  const float x = static_cast<float>(halves);
  const float rest = static_cast<float>(halves - static_cast<double>(x)) * 3.14159265f;
  float s, c;
  sincospif(x, &s, &c);
  const float cc = fmaf(-s, rest, c) * a.factor, ss = fmaf(c, rest, s) * a.factor;
  return make_float2(cc, a.inverse ? -ss : ss);
}

// Where the turn of pair j of chunk c stands among a token's: chunks of the same pair side by side, so that threads
// of neighbouring chunks read neighbouring words.
template <int V>
__device__ __forceinline__ int turn_place(int c, int j, int chunks) {
  return V == 1 ? c : ((j >> 1) * chunks + c) * 2 + (j & 1);
}

template <typename T, int V, bool kHalves>
__global__ void __launch_bounds__(512) rope_kernel(const __grid_constant__ RopeParams P) {
  extern __shared__ __align__(16) float2 turns[];  // [tokens of the block][pairs]
  griddep_wait();
  griddep_launch();
  const long long tok0 = static_cast<long long>(blockIdx.x) * P.tokens_per_block;
  const int ntok = static_cast<int>(min(static_cast<long long>(P.tokens_per_block), P.tokens - tok0));
  const uint32_t items = static_cast<uint32_t>(ntok) * P.per_token.d;
  const int pairs = P.a.pairs;
  for (uint32_t base = 0; base < items; base += kRopeItems * blockDim.x) {
    Raw<T, V> a[kRopeItems], b[kRopeItems];
    T* dst[kRopeItems];
    int tok[kRopeItems], chunk[kRopeItems], second[kRopeItems];  // second: where b lies from a, 0: there is none
#pragma unroll
    for (int u = 0; u < kRopeItems; ++u) {
      const uint32_t it = base + u * blockDim.x + threadIdx.x;
      dst[u] = nullptr;
      if (it >= items) continue;
      tok[u] = static_cast<int>(quotient(it, P.per_token));
      const uint32_t in_tok = it - tok[u] * P.per_token.d;
      int head = static_cast<int>(quotient(in_tok, P.per_head));
      chunk[u] = static_cast<int>(in_tok - head * P.per_head.d);
      const bool other = head >= P.part[0].heads;
      const RopePart& part = P.part[other ? 1 : 0];
      if (other) head -= P.part[0].heads;
      int e;
      if (chunk[u] < P.chunks) {
        e = kHalves ? chunk[u] * V : 2 * chunk[u] * V;
        second[u] = kHalves ? pairs : V;
      } else {  // values that are not turned, two vectors an item
        e = 2 * pairs + 2 * (chunk[u] - P.chunks) * V;
        second[u] = e + V < P.head_dim ? V : 0;
      }
      const T* src = static_cast<const T*>(part.in) + (tok0 + tok[u]) * part.in_tok + head * part.in_head + e;
      dst[u] = static_cast<T*>(part.out) + (tok0 + tok[u]) * part.out_tok + head * part.out_head + e;
      a[u] = load_once<T, V>(src);
      if (second[u]) b[u] = load_once<T, V>(src + second[u]);
    }
    if (base == 0) {
      for (int i = threadIdx.x; i < ntok * pairs; i += blockDim.x) {
        const int t = i / pairs, pair = i - t * pairs;
        turns[t * pairs + turn_place<V>(pair / V, pair % V, P.chunks)] = rope_turn(P.a, tok0 + t, pair);
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kRopeItems; ++u) {
      if (!dst[u]) continue;
      if (chunk[u] < P.chunks) {
        const float2* w = turns + tok[u] * pairs;
        float x[V], y[V];
        unpack_row<T, V>(a[u], x);
        unpack_row<T, V>(b[u], y);
        if constexpr (kHalves || V == 1) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float2 t = w[turn_place<V>(chunk[u], j, P.chunks)];
            const float p = x[j], q = y[j];
            x[j] = fmaf(p, t.x, -q * t.y);
            y[j] = fmaf(q, t.x, p * t.y);
          }
        } else {  // x and y hold V / 2 pairs each
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float2 t = w[turn_place<V>(chunk[u], j, P.chunks)];
            float(&z)[V] = j < V / 2 ? x : y;
            const int k = 2 * (j % (V / 2));
            const float p = z[k], q = z[k + 1];
            z[k] = fmaf(p, t.x, -q * t.y);
            z[k + 1] = fmaf(q, t.x, p * t.y);
          }
        }
        a[u] = pack_row<T, V>(x);
        b[u] = pack_row<T, V>(y);
      }
      store_once<T, V>(dst[u], a[u]);
      if (second[u]) store_once<T, V>(dst[u] + second[u], b[u]);
    }
  }
}

// cos and sin rows [tokens, 2 pairs], each value twice: the tables of a kernel that turns halves.
template <typename T, int V>
__global__ void __launch_bounds__(256) rope_rows_kernel(const __grid_constant__ RopeAngles A, long long tokens, T* cos, T* sin) {
  griddep_wait();
  griddep_launch();
  const int chunks = A.pairs / V;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= tokens * chunks) return;
  const long long token = i / chunks;
  const int pair = static_cast<int>(i - token * chunks) * V;
  float c[V], s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float2 t = rope_turn(A, token, pair + j);
    c[j] = t.x, s[j] = t.y;
  }
  const Raw<T, V> rc = pack_row<T, V>(c), rs = pack_row<T, V>(s);
  const long long at = token * 2 * A.pairs + pair;
  *reinterpret_cast<Raw<T, V>*>(cos + at) = rc;  // (read soon: not streamed past the caches)
  *reinterpret_cast<Raw<T, V>*>(cos + at + A.pairs) = rc;
  *reinterpret_cast<Raw<T, V>*>(sin + at) = rs;
  *reinterpret_cast<Raw<T, V>*>(sin + at + A.pairs) = rs;
}


template <typename T, int V>
cudaError_t launch_rope(const RopeParams& p, bool halves, unsigned grid, unsigned block, size_t smem, cudaStream_t stream) {
  return halves ? launch_overlapped(rope_kernel<T, V, true>, grid, block, smem, stream, p)
                : launch_overlapped(rope_kernel<T, V, false>, grid, block, smem, stream, p);
}
template <typename T>
cudaError_t launch_rope(const RopeParams& p, int v, bool halves, unsigned grid, unsigned block, size_t smem, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (v == 8) return launch_rope<T, 8>(p, halves, grid, block, smem, stream);
  switch (v) {
    case 4: return launch_rope<T, 4>(p, halves, grid, block, smem, stream);
    case 2: return launch_rope<T, 2>(p, halves, grid, block, smem, stream);
    default: return launch_rope<T, 1>(p, halves, grid, block, smem, stream);
  }
}
template <typename T>
cudaError_t launch_rope_rows(const RopeAngles& a, long long tokens, void* cos, void* sin, bool wide, cudaStream_t stream) {
  const long long n = tokens * (wide ? a.pairs / 4 : a.pairs);
  const unsigned grid = static_cast<unsigned>((n + 255) / 256);
  return wide ? launch_overlapped(rope_rows_kernel<T, 4>, grid, 256u, 0, stream, a, tokens, static_cast<T*>(cos), static_cast<T*>(sin))
              : launch_overlapped(rope_rows_kernel<T, 1>, grid, 256u, 0, stream, a, tokens, static_cast<T*>(cos), static_cast<T*>(sin));
}

int rope_angles(const rldx_rope_plan* plan, const char* who, RopeAngles* a) {
  const std::string w = std::string(who) + ": ";
  if (!plan) return set_error(RLDX_ERR_ARG, w + "null plan");
  if (!plan->positions || !plan->freqs) return set_error(RLDX_ERR_ARG, w + "null positions or freqs");
  if (reinterpret_cast<uintptr_t>(plan->freqs) % 8 || reinterpret_cast<uintptr_t>(plan->positions) % (plan->positions_int64 ? 8 : 4))
    return set_error(RLDX_ERR_ARG, w + "misaligned positions or freqs");
  if (plan->pairs < 1 || plan->pairs > kRopeMaxPairs)
    return set_error(RLDX_ERR_UNSUPPORTED, w + "1 to " + std::to_string(kRopeMaxPairs) + " pairs of a head are turned");
  if (plan->axes < 1 || plan->axes > kRopeMaxAxes)
    return set_error(RLDX_ERR_UNSUPPORTED, w + "positions have 1 to " + std::to_string(kRopeMaxAxes) + " axes");
  if (plan->axes > 1) {
    int sum = 0;
    for (int i = 0; i < plan->axes; ++i) {
      if (plan->sections[i] < 0 || plan->sections[i] > plan->pairs) return set_error(RLDX_ERR_ARG, w + "sections must be pairs of the head");
      sum += plan->sections[i];
    }
    if (sum != plan->pairs) return set_error(RLDX_ERR_ARG, w + "sections must add up to the pairs");
    if (plan->positions_ld < 0) return set_error(RLDX_ERR_ARG, w + "negative stride of positions");
  }
  a->pos = plan->positions;
  a->pos_ld = plan->positions_ld;
  a->pos64 = plan->positions_int64 ? 1 : 0;
  a->axes = plan->axes;
  for (int i = 0; i < kRopeMaxAxes; ++i) a->sections[i] = plan->axes > 1 && i < plan->axes ? plan->sections[i] : 0;
  a->sections_interleaved = plan->sections_interleaved ? 1 : 0;
  a->freqs = plan->freqs;
  a->pairs = plan->pairs;
  a->factor = plan->factor;
  a->inverse = plan->inverse ? 1 : 0;
  return RLDX_OK;
}
}  // namespace

}  // namespace rldx

using namespace rldx;

extern "C" {

int rldx_rope(const rldx_rope_plan* plan, const rldx_rope_heads* heads, int nheads, int64_t tokens, int head_dim, int dtype,
              void* stream) {
  RopeParams p = {};
  if (tokens < 0 || tokens >= (1LL << 31)) return set_error(RLDX_ERR_ARG, "rope: 0 to 2^31 - 1 tokens");
  int rc = rope_angles(plan, "rope", &p.a);
  if (rc != RLDX_OK) return rc;
  if (!heads || nheads < 1 || nheads > 2) return set_error(RLDX_ERR_ARG, "rope: one or two groups of heads");
  if (!known_dtype(dtype)) return set_error(RLDX_ERR_UNSUPPORTED, "rope: unknown type");
  if (head_dim < 2 * plan->pairs || head_dim > 4096)
    return set_error(RLDX_ERR_ARG, "rope: a head has at least the values that are turned, 4096 at most");
  const int size = dtype_bytes(dtype);
  long long all_heads = 0;
  bool in_place = true;
  // V pairs an item: as many as the addresses' common alignment and the counts allow
  int v = dtype == RLDX_F32 ? 4 : 8;
  auto halve_until = [&](auto fits) {
    while (v > 1 && !fits()) v /= 2;
  };
  for (int i = 0; i < nheads; ++i) {
    const rldx_rope_heads& h = heads[i];
    if (!h.in || !h.out) return set_error(RLDX_ERR_ARG, "rope: null heads");
    if (h.heads < 1 || h.heads > 65536) return set_error(RLDX_ERR_ARG, "rope: 1 to 65536 heads");
    if (h.in_tok < 0 || h.in_head < 0 || h.out_tok < 0 || h.out_head < 0) return set_error(RLDX_ERR_ARG, "rope: negative strides");
    // tokens of heads, or heads of tokens: written values have places of their own (read ones may share theirs)
    const bool of_tokens = (h.heads == 1 || h.out_head >= head_dim) && (tokens <= 1 || h.out_tok >= (h.heads - 1) * h.out_head + head_dim);
    const bool of_heads = (tokens <= 1 || h.out_tok >= head_dim) && (h.heads == 1 || h.out_head >= (tokens - 1) * h.out_tok + head_dim);
    if (!of_tokens && !of_heads) return set_error(RLDX_ERR_ARG, "rope: heads of the output overlap");
    if (reinterpret_cast<uintptr_t>(h.in) % size || reinterpret_cast<uintptr_t>(h.out) % size) return set_error(RLDX_ERR_ARG, "rope: misaligned heads");
    p.part[i] = {h.in, h.out, h.in_tok, h.in_head, h.out_tok, h.out_head, h.heads};
    all_heads += h.heads;
    in_place &= h.in == h.out && h.in_tok == h.out_tok && h.in_head == h.out_head;
    halve_until([&] {
      const int bytes = v * size > 16 ? 16 : v * size;
      return h.in_tok % v == 0 && h.in_head % v == 0 && h.out_tok % v == 0 && h.out_head % v == 0 &&
             reinterpret_cast<uintptr_t>(h.in) % bytes == 0 && reinterpret_cast<uintptr_t>(h.out) % bytes == 0;
    });
  }
  halve_until([&] { return plan->pairs % v == 0 && head_dim % v == 0; });
  p.tokens = tokens;
  p.head_dim = head_dim;
  p.chunks = plan->pairs / v;
  const int rest = in_place ? 0 : (head_dim - 2 * plan->pairs) / v;  // vectors that are only copied
  const uint32_t per_head = static_cast<uint32_t>(p.chunks + (rest + 1) / 2);
  const long long per_token = per_head * all_heads;
  if (per_token > (1 << 16)) return set_error(RLDX_ERR_UNSUPPORTED, "rope: too many values a token");
  if (tokens == 0) return RLDX_OK;
  rc = ensure_device();
  if (rc != RLDX_OK) return rc;
  // Tokens of a block: up to 384 items (us, 256 / 384 / 512 / 1024: 8832 tokens of 16 / 2 heads of 128 13.8 / 13.5 / 13.0 / 15.4, 65536 of
  // 16 / 16 154 / 154 / 165 / 179, 11524 of 12 / 4 heads of 96 in fp32 21.5 / 23.5 / 23.5 / 28.5), but so few that there are two blocks
  // an SM (one token a block while tokens are fewer than four times the SMs), and turns of 16 KB at most.
  long long tpb = std::max(1LL, std::min<long long>(384 / per_token, 2048 / plan->pairs));
  tpb = std::min(tpb, std::max(1LL, tokens / (2LL * sm_count())));
  p.tokens_per_block = static_cast<int>(tpb);
  p.per_head = small_div(per_head);
  p.per_token = small_div(static_cast<uint32_t>(per_token));
  const long long per_thread = (tpb * per_token + kRopeItems - 1) / kRopeItems;
  const unsigned block = static_cast<unsigned>(std::min(512LL, std::max(64LL, (per_thread + 31) / 32 * 32)));
  const unsigned grid = static_cast<unsigned>((tokens + tpb - 1) / tpb);
  const size_t smem = sizeof(float2) * tpb * plan->pairs;
  const bool halves = !plan->interleaved;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == RLDX_F32   ? launch_rope<float>(p, v, halves, grid, block, smem, st)
                        : dtype == RLDX_F16 ? launch_rope<__half>(p, v, halves, grid, block, smem, st)
                                            : launch_rope<__nv_bfloat16>(p, v, halves, grid, block, smem, st);
  if (e != cudaSuccess) return cuda_fail(e, "rope launch");
  return RLDX_OK;
}

int rldx_rope_rows(const rldx_rope_plan* plan, int64_t tokens, void* cos, void* sin, int dtype, void* stream) {
  RopeAngles a;
  if (tokens < 0 || tokens >= (1LL << 31)) return set_error(RLDX_ERR_ARG, "rope_rows: 0 to 2^31 - 1 tokens");
  int rc = rope_angles(plan, "rope_rows", &a);
  if (rc != RLDX_OK) return rc;
  if (!cos || !sin) return set_error(RLDX_ERR_ARG, "rope_rows: null rows");
  if (!known_dtype(dtype)) return set_error(RLDX_ERR_UNSUPPORTED, "rope_rows: unknown type");
  const uintptr_t at = reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin);
  if (at % dtype_bytes(dtype)) return set_error(RLDX_ERR_ARG, "rope_rows: misaligned rows");
  if (tokens * a.pairs >= (1LL << 38)) return set_error(RLDX_ERR_UNSUPPORTED, "rope_rows: too many rows");
  if (tokens == 0) return RLDX_OK;
  rc = ensure_device();
  if (rc != RLDX_OK) return rc;
  const bool wide = a.pairs % 4 == 0 && at % (4 * dtype_bytes(dtype)) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == RLDX_F32   ? launch_rope_rows<float>(a, tokens, cos, sin, wide, st)
                        : dtype == RLDX_F16 ? launch_rope_rows<__half>(a, tokens, cos, sin, wide, st)
                                            : launch_rope_rows<__nv_bfloat16>(a, tokens, cos, sin, wide, st);
  if (e != cudaSuccess) return cuda_fail(e, "rope_rows launch");
  return RLDX_OK;
}

}  // extern "C"
