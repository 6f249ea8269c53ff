// Writing and reading the paged 4-bit cache (layout: kv4.cuh).
//
//   kv4_append_kernel  q = rope(rms(q) wq), k = rope(rms(k) wk), v of projected [q | k | v] rows;
//                      q to bf16, k and v quantised into the cache.  Per head of d channels:
//                        rms(x)_i = x_i / sqrt(mean(x^2) + eps)
//                        rope(y)_i = y_i cos_i - y_{i+d/2} sin_i (i < d/2), y_i cos_i + y_{i-d/2} sin_i
//                      and per token and group of 32 channels of k and v:
//                        low = h(min x), scale = h((max x - min x) / 15), h: round to fp16
//                        code = clamp(rint((x - low) / scale), 0, 15)
//                      all in fp32.  The rounded low and scale choose the codes, so a value is
//                      off by half a step plus what their rounding takes from the range's ends.
//                      A NaN in a group makes its scale and low NaN; values past +-65504 saturate.
//   kv4_read_kernel    scale * code + low of the newest tokens, as bf16.
#include "host_util.h"
#include "kv4.cuh"

namespace rldx {

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  unpack_bf16x2(u.x, v[0], v[1]);
  unpack_bf16x2(u.y, v[2], v[3]);
  unpack_bf16x2(u.z, v[4], v[5]);
  unpack_bf16x2(u.w, v[6], v[7]);
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float2 (&v)[2]) {
  const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
  unpack_bf16x2(u.x, v[0].x, v[0].y);
  unpack_bf16x2(u.y, v[1].x, v[1].y);
}
__device__ __forceinline__ void load4(const float* p, float2 (&v)[2]) {
  const float4 u = __ldg(reinterpret_cast<const float4*>(p));
  v[0] = make_float2(u.x, u.y), v[1] = make_float2(u.z, u.w);
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// Sequence of row `row`: the number of cu entries 1..seqs that are <= row.
__device__ __forceinline__ int seq_of_row(const int* cu, int seqs, int row) {
  int lo = 0, hi = seqs;  // cu[lo] <= row < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

constexpr int kKv4SmemSeqs = 1024;  // batches up to this size keep cu and lengths in shared memory

// Where new-token row `row` stands in the cache: index of its unit for head 0 (-1: nowhere, recorded; a row before
// the first sequence's or past the last one's is none of theirs) and its token in the unit; head h's unit is
// units_per_page h further.
__device__ __forceinline__ int kv4_token_place(const Kv4Cache& c, const int* cu, const int* lengths, int row, int* tau) {
  const int b = seq_of_row(cu, c.seqs, row);
  const int pos = lengths[b] - cu[b + 1] + row;
  *tau = pos & (kKv4Unit - 1);
  if (row < cu[b] || row >= cu[b + 1]) {
    record_data_error(kErrKv4Bound);
    return -1;
  }
  const int index = pos >= 0 ? kv4_unit_index(c, b, 0, pos / kKv4Unit) : -1;
  if (index < 0) record_data_error(kErrKv4Table);
  return index;
}

// Copies cu and lengths to shared memory where they fit and returns where to read them.
__device__ __forceinline__ void stage_seqs(const Kv4Cache& c, int* smem, const int** cu, const int** lengths) {
  *cu = c.cu;
  *lengths = c.lengths;
  if (c.seqs <= kKv4SmemSeqs) {
    for (int i = threadIdx.x; i <= c.seqs; i += blockDim.x) smem[i] = c.cu[i];
    for (int i = threadIdx.x; i < c.seqs; i += blockDim.x) smem[kKv4SmemSeqs + 1 + i] = c.lengths[i];
    *cu = smem;
    *lengths = smem + kKv4SmemSeqs + 1;
  }
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  unpack_bf16x2(u.x, v[0], v[1]);
  unpack_bf16x2(u.y, v[2], v[3]);
  unpack_bf16x2(u.z, v[4], v[5]);
  unpack_bf16x2(u.w, v[6], v[7]);
}

// A head of one token, D / 8 lanes with 8 channels each: v = rope(rms(v) w).  c, s: this lane's part of the
// rotation's row, s with the sign of rotate_half = cat(-x2, x1).
template <int D>
__device__ __forceinline__ void norm_rope(float (&v)[8], const float (&w)[8], const float (&c)[8], const float (&s)[8], float eps) {
  constexpr int kLanes = D / 8;
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float rstd = rsqrtf(ss * (1.0f / D) + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = __fmul_rn(__fmul_rn(v[e], rstd), w[e]);
    const float o = __shfl_xor_sync(0xffffffffu, y, kLanes / 2);  // the channel half a head away
    v[e] = __fadd_rn(__fmul_rn(y, c[e]), __fmul_rn(o, s[e]));
  }
}

// Codes of this lane's 8 channels (lowest first), and scale and low of the group that four lanes share.
__device__ __forceinline__ uint32_t quantise8(const float (&v)[8], __half* scale_h, __half* low_h) {
  float mn = v[0], mx = v[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) mn = min_nan(mn, v[e]), mx = max_nan(mx, v[e]);
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  mn = max_nan(min_nan(mn, 65504.0f), -65504.0f);
  mx = max_nan(min_nan(mx, 65504.0f), -65504.0f);
  *low_h = __float2half_rn(mn);
  *scale_h = __float2half_rn(__fmul_rn(mx - mn, 1.0f / 15.0f));
  const float low = __half2float(*low_h), scale = __half2float(*scale_h);
  const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(v[e], low), inv)), 0.0f), 15.0f);  // NaN: 0
    codes |= static_cast<uint32_t>(q) << (4 * e);
  }
  return codes;
}

// D / 8 lanes own an item: four query heads of a token, or (blocks from q_blocks on) k and v of one kv
// head.  The rotation's row is read once for an item, all loads are issued before any arithmetic, and
// every block runs straight-line code of one kind.  8 prompts of up to 1104 tokens, 16 / 2 heads, d = 128,
// appended and read back: 24.2 us (12.0 at the copy's rate; captured 20.9).  Before the query heads' arithmetic was
// paired it was 26, and then 39 with one head an item, 39 with q, k and v heads mixed in a block, 27 with two heads an
// item and more CTAs an SM.  No unit is busy (DRAM 22 %, the busiest of an SM 44 %) and waits for loads lead the
// stalls: each block of 128 threads pays a chain of them, lengths, place, page, data.
constexpr int kAppendHeads = 4;

template <int D, typename Rope>
__global__ void __launch_bounds__(128) kv4_append_kernel(const __grid_constant__ Kv4AppendParams P, unsigned q_blocks) {
  using U = Kv4Unit<D>;
  constexpr int kLanes = D / 8;
  __shared__ int s_seq[2 * kKv4SmemSeqs + 1];
  griddep_wait();
  const int hq = P.q_heads, hkv = P.c.kv_heads, l = threadIdx.x % kLanes;
  const bool of_q = blockIdx.x < q_blocks;
  const unsigned item = ((of_q ? blockIdx.x : blockIdx.x - q_blocks) * 128u + threadIdx.x) / kLanes;
  const unsigned per_token = of_q ? (hq + kAppendHeads - 1) / kAppendHeads : hkv;
  const bool live = item < static_cast<unsigned>(P.c.tokens) * per_token;  // (an item past the end repeats the last token)
  const int tok = live ? static_cast<int>(item / per_token) : P.c.tokens - 1;
  const int at = static_cast<int>(item % per_token);
  const __nv_bfloat16* src = P.qkv + tok * P.ld + 8 * l;
  int rp = __ldg(P.rope_pos + tok);
  if (of_q) {
    // a lane's channels: four, and the four half a head away that the rotation pairs them with
    const int h0 = at * kAppendHeads;
    uint2 x[kAppendHeads][2];
#pragma unroll
    for (int r = 0; r < kAppendHeads; ++r)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        x[r][i] = __ldcs(reinterpret_cast<const uint2*>(P.qkv + tok * P.ld + min(h0 + r, hq - 1) * D + i * (D / 2) + 4 * l));
    if (static_cast<unsigned>(rp) >= static_cast<unsigned>(P.rope_rows)) {
      if (live) record_data_error(kErrKv4Rope);
      rp = 0;
    }
    float2 w[2][2], c[2][2], s[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int ch = i * (D / 2) + 4 * l;
      load4(P.wq + ch, w[i]);
      load4(static_cast<const Rope*>(P.cos) + static_cast<long long>(rp) * D + ch, c[i]);
      load4(static_cast<const Rope*>(P.sin) + static_cast<long long>(rp) * D + ch, s[i]);
    }
    griddep_launch();
    float2 v[kAppendHeads][2][2];
    float ss[kAppendHeads];
#pragma unroll
    for (int r = 0; r < kAppendHeads; ++r) {
      float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        unpack_bf16x2(x[r][i].x, v[r][i][0].x, v[r][i][0].y);
        unpack_bf16x2(x[r][i].y, v[r][i][1].x, v[r][i][1].y);
#pragma unroll
        for (int e = 0; e < 2; ++e) sum = fma_f32x2(v[r][i][e], v[r][i][e], sum);
      }
      ss[r] = sum.x + sum.y;
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
      for (int r = 0; r < kAppendHeads; ++r) ss[r] += __shfl_xor_sync(0xffffffffu, ss[r], o);
#pragma unroll
    for (int r = 0; r < kAppendHeads; ++r) {
      const float rstd = rsqrtf(ss[r] * (1.0f / D) + P.eps);
      const float2 rr = make_float2(rstd, rstd);
      uint2 u[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 y0 = mul_f32x2(mul_f32x2(v[r][0][e], rr), w[0][e]), y1 = mul_f32x2(mul_f32x2(v[r][1][e], rr), w[1][e]);
        const float2 n = mul_f32x2(y1, s[0][e]);
        const float2 a = add_f32x2(mul_f32x2(y0, c[0][e]), make_float2(-n.x, -n.y));
        const float2 b = add_f32x2(mul_f32x2(y1, c[1][e]), mul_f32x2(y0, s[1][e]));
        (e ? u[0].y : u[0].x) = pack_bf16x2(a.x, a.y);
        (e ? u[1].y : u[1].x) = pack_bf16x2(b.x, b.y);
      }
      if (live && h0 + r < hq)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<uint2*>(P.q + (static_cast<long long>(tok) * hq + h0 + r) * D + i * (D / 2) + 4 * l) = u[i];
    }
    return;
  }
  float w[8], c[8], s[8];
  load8(P.wk + 8 * l, w);
  if (static_cast<unsigned>(rp) >= static_cast<unsigned>(P.rope_rows)) {
    if (live) record_data_error(kErrKv4Rope);
    rp = 0;
  }
  const uint4 xk = __ldcs(reinterpret_cast<const uint4*>(src + (hq + at) * D));
  const uint4 xv = __ldcs(reinterpret_cast<const uint4*>(src + (hq + hkv + at) * D));
  const int *cu = P.c.cu, *lengths = P.c.lengths;
  stage_seqs(P.c, s_seq, &cu, &lengths);
  load8(static_cast<const Rope*>(P.cos) + static_cast<long long>(rp) * D + 8 * l, c);
  load8(static_cast<const Rope*>(P.sin) + static_cast<long long>(rp) * D + 8 * l, s);
  if (l < kLanes / 2)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = -s[e];
  __syncthreads();
  griddep_launch();
  int tau = 0;
  const int place = live ? kv4_token_place(P.c, cu, lengths, tok, &tau) : -1;
  float k[8], v[8];
  unpack8(xk, k);
  unpack8(xv, v);
  norm_rope<D>(k, w, c, s, P.eps);
  __half k_scale, k_low, v_scale, v_low;
  const uint32_t kc = quantise8(k, &k_scale, &k_low), vc = quantise8(v, &v_scale, &v_low);
  if (place < 0) return;
  uint8_t* unit = P.c.data + static_cast<long long>(place + at * P.c.units_per_page) * U::kBytes;
  const int j = l / 4, t4 = l % 4;  // group, position in the group
  const int blk = tau / 16, hh = tau / 8 % 2, t = tau / 2 % 4, e = tau % 2;
  *reinterpret_cast<uint32_t*>(unit + tau * U::kRow + 4 * (t4 * U::kG + j)) = kc;
  uint8_t* va = unit + U::kV + 8 * D * blk + 4 * D * hh + 4 * U::kG * t + 2 * U::kG * e + 2 * j;
  *reinterpret_cast<uint16_t*>(va + 16 * U::kG * (2 * t4)) = static_cast<uint16_t>(vc);
  *reinterpret_cast<uint16_t*>(va + 16 * U::kG * (2 * t4 + 1)) = static_cast<uint16_t>(vc >> 16);
  if (t4 == 0) {
    __half* meta = reinterpret_cast<__half*>(unit + U::kKMeta + 4 * U::kG * tau);
    meta[j] = k_scale;
    meta[U::kG + j] = k_low;
    const int m = 32 * U::kG * blk + 16 * U::kG * hh + 4 * U::kG * t + 4 * j + 2 * e;
    *reinterpret_cast<__half*>(unit + U::kVScale + m) = v_scale;
    *reinterpret_cast<__half*>(unit + U::kVLow + m) = v_low;
  }
}

// 8 channels: scale * code + low, rounded to bf16.
__device__ __forceinline__ uint4 rebuild8(uint32_t codes, __half scale_h, __half low_h) {
  const float scale = __half2float(scale_h), low = __half2float(low_h);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = fmaf(scale, static_cast<float>(codes >> (4 * i) & 15u), low);
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// D / 8 lanes own k and v of one kv head of a token: one search for the token's place serves both, and all
// loads are issued together.  8 prompts, 6789 tokens, 2 heads of 128, the cache in L2: 5.0 us captured for 2.1 MB read
// and 7.0 MB written (1.4 at the copy's rate); one token 2.0.  The same chain of loads in every block bounds it.
template <int D>
__global__ void __launch_bounds__(128) kv4_read_kernel(const __grid_constant__ Kv4ReadParams P) {
  using U = Kv4Unit<D>;
  constexpr int kLanes = D / 8;
  __shared__ int s_seq[2 * kKv4SmemSeqs + 1];
  griddep_wait();
  griddep_launch();
  const int hkv = P.c.kv_heads;
  const int *cu, *lengths;
  stage_seqs(P.c, s_seq, &cu, &lengths);
  __syncthreads();
  const long long row = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / kLanes;
  if (row >= static_cast<long long>(P.c.tokens) * hkv) return;
  const int l = threadIdx.x % kLanes, j = l / 4, t4 = l % 4;
  const int tok = static_cast<int>(row / hkv), h = static_cast<int>(row - static_cast<long long>(tok) * hkv);
  int tau;
  const int place = kv4_token_place(P.c, cu, lengths, tok, &tau);
  uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
  if (place >= 0) {
    const uint8_t* unit = P.c.data + static_cast<long long>(place + h * P.c.units_per_page) * U::kBytes;
    const int blk = tau / 16, hh = tau / 8 % 2, t = tau / 2 % 4, e = tau % 2;
    const uint8_t* at = unit + U::kV + 8 * D * blk + 4 * D * hh + 4 * U::kG * t + 2 * U::kG * e + 2 * j;
    const int m = 32 * U::kG * blk + 16 * U::kG * hh + 4 * U::kG * t + 4 * j + 2 * e;
    const __half* meta = reinterpret_cast<const __half*>(unit + U::kKMeta + 4 * U::kG * tau);
    const uint32_t kc = *reinterpret_cast<const uint32_t*>(unit + tau * U::kRow + 4 * (t4 * U::kG + j));
    const __half k_scale = meta[j], k_low = meta[U::kG + j];
    const uint32_t v0 = *reinterpret_cast<const uint16_t*>(at + 16 * U::kG * (2 * t4));
    const uint32_t v1 = *reinterpret_cast<const uint16_t*>(at + 16 * U::kG * (2 * t4 + 1));
    const __half v_scale = *reinterpret_cast<const __half*>(unit + U::kVScale + m);
    const __half v_low = *reinterpret_cast<const __half*>(unit + U::kVLow + m);
    k = rebuild8(kc, k_scale, k_low);
    v = rebuild8(v0 | v1 << 16, v_scale, v_low);
  }
  const long long to = (static_cast<long long>(tok) * hkv + h) * D + 8 * l;
  *reinterpret_cast<uint4*>(P.k + to) = k;
  *reinterpret_cast<uint4*>(P.v + to) = v;
}

namespace {
template <typename... Args>
cudaError_t launch_blocks(void (*kernel)(Args...), unsigned blocks, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, 1, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
// blocks of 128 threads for `items` of `lanes` threads
unsigned blocks_of(long long items, int lanes) { return static_cast<unsigned>((items * lanes + 127) / 128); }

template <int D>
cudaError_t launch_append(const Kv4AppendParams& p, cudaStream_t stream) {
  const unsigned q_blocks = blocks_of(static_cast<long long>(p.c.tokens) * ((p.q_heads + kAppendHeads - 1) / kAppendHeads), D / 8);
  const unsigned kv_blocks = blocks_of(static_cast<long long>(p.c.tokens) * p.c.kv_heads, D / 8);
  return p.rope_f32 ? launch_blocks<Kv4AppendParams, unsigned>(kv4_append_kernel<D, float>, q_blocks + kv_blocks, stream, p, q_blocks)
                    : launch_blocks<Kv4AppendParams, unsigned>(kv4_append_kernel<D, __nv_bfloat16>, q_blocks + kv_blocks, stream, p, q_blocks);
}
}  // namespace

cudaError_t launch_kv4_append(const Kv4AppendParams& p, int head_dim, cudaStream_t stream) {
  return head_dim == 128 ? launch_append<128>(p, stream) : launch_append<64>(p, stream);
}

cudaError_t launch_kv4_read(const Kv4ReadParams& p, int head_dim, cudaStream_t stream) {
  const unsigned blocks = blocks_of(static_cast<long long>(p.c.tokens) * p.c.kv_heads, head_dim / 8);
  return head_dim == 128 ? launch_blocks<Kv4ReadParams>(kv4_read_kernel<128>, blocks, stream, p)
                         : launch_blocks<Kv4ReadParams>(kv4_read_kernel<64>, blocks, stream, p);
}

namespace {
bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Checks a cache description and turns it into the kernels' form.
int kv4_cache(const rldx_kv4_cache* d, int tokens, const char* what, Kv4Cache* c) {
  const std::string w = what;
  if (!d) return set_error(RLDX_ERR_ARG, w + ": null cache");
  if (!d->data || !d->table || !d->lengths || !d->cu_seqlens) return set_error(RLDX_ERR_ARG, w + ": null cache pointer");
  if (d->head_dim != 64 && d->head_dim != 128) return set_error(RLDX_ERR_UNSUPPORTED, w + ": head_dim must be 64 or 128");
  if (d->page_size <= 0 || d->page_size % kKv4Unit) return set_error(RLDX_ERR_ARG, w + ": page_size must be a multiple of 32");
  if (d->pages <= 0 || d->pages >= (1LL << 31) || d->kv_heads <= 0 || d->table_width <= 0 ||
      d->table_ld < d->table_width || d->seqs <= 0)
    return set_error(RLDX_ERR_ARG, w + ": pages, kv_heads, seqs and table_width must be positive, table_ld >= table_width");
  if (static_cast<long long>(d->table_width) * d->page_size >= (1LL << 31))
    return set_error(RLDX_ERR_UNSUPPORTED, w + ": a sequence holds less than 2^31 tokens");
  if (d->pages * d->kv_heads * (d->page_size / kKv4Unit) >= (1LL << 31))
    return set_error(RLDX_ERR_UNSUPPORTED, w + ": a pool has fewer than 2^31 units of 32 tokens of a head");
  if (tokens < 0) return set_error(RLDX_ERR_ARG, w + ": negative token count");
  if (!aligned_to(d->data, 16)) return set_error(RLDX_ERR_ARG, w + ": the cache must be 16-byte aligned");
  c->data = static_cast<uint8_t*>(d->data);
  c->pages = d->pages;
  c->kv_heads = d->kv_heads;
  c->units_per_page = d->page_size / kKv4Unit;
  c->table = d->table;
  c->table_width = d->table_width;
  c->table_ld = d->table_ld;
  c->lengths = d->lengths;
  c->cu = d->cu_seqlens;
  c->seqs = d->seqs;
  c->tokens = tokens;
  return RLDX_OK;
}
}  // namespace

}  // namespace rldx

using namespace rldx;

extern "C" {

int rldx_kv4_append(const rldx_kv4_cache* cache, const void* qkv, int64_t ld, int tokens, int q_heads,
                    const void* q_norm, const void* k_norm, const void* rope_cos, const void* rope_sin,
                    int rope_fp32, int rope_rows, const int32_t* rope_pos, void* q_out, float eps, void* stream) {
  int rc = ensure_device();
  if (rc != RLDX_OK) return rc;
  Kv4AppendParams p;
  rc = kv4_cache(cache, tokens, "kv4_append", &p.c);
  if (rc != RLDX_OK) return rc;
  const int d = cache->head_dim;
  if (!qkv || !q_norm || !k_norm || !rope_cos || !rope_sin || !rope_pos || !q_out)
    return set_error(RLDX_ERR_ARG, "kv4_append: null pointer");
  if (q_heads <= 0 || q_heads % cache->kv_heads) return set_error(RLDX_ERR_ARG, "kv4_append: kv_heads must divide q_heads");
  const long long width = static_cast<long long>(q_heads + 2 * cache->kv_heads) * d;
  if (ld < width || ld % 8) return set_error(RLDX_ERR_ARG, "kv4_append: rows must be 16-byte aligned and hold q, k and v");
  if (rope_rows <= 0) return set_error(RLDX_ERR_ARG, "kv4_append: empty RoPE table");
  for (const void* x : {qkv, q_norm, k_norm, rope_cos, rope_sin, static_cast<const void*>(q_out)})
    if (!aligned_to(x, 16)) return set_error(RLDX_ERR_ARG, "kv4_append: pointers must be 16-byte aligned");
  if (static_cast<long long>(tokens) * (q_heads + 2 * cache->kv_heads) >= (1LL << 27))
    return set_error(RLDX_ERR_UNSUPPORTED, "kv4_append: too many rows");
  if (tokens == 0) return RLDX_OK;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.ld = ld;
  p.q_heads = q_heads;
  p.wq = static_cast<const __nv_bfloat16*>(q_norm);
  p.wk = static_cast<const __nv_bfloat16*>(k_norm);
  p.cos = rope_cos;
  p.sin = rope_sin;
  p.rope_f32 = rope_fp32 ? 1 : 0;
  p.rope_rows = rope_rows;
  p.rope_pos = rope_pos;
  p.q = static_cast<__nv_bfloat16*>(q_out);
  p.eps = eps;
  cudaError_t e = launch_kv4_append(p, d, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "kv4_append launch");
  return RLDX_OK;
}

int rldx_kv4_read(const rldx_kv4_cache* cache, int tokens, void* k, void* v, void* stream) {
  int rc = ensure_device();
  if (rc != RLDX_OK) return rc;
  Kv4ReadParams p;
  rc = kv4_cache(cache, tokens, "kv4_read", &p.c);
  if (rc != RLDX_OK) return rc;
  if (!k || !v || !aligned_to(k, 16) || !aligned_to(v, 16))
    return set_error(RLDX_ERR_ARG, "kv4_read: k and v must be 16-byte aligned");
  if (static_cast<long long>(tokens) * 2 * cache->kv_heads >= (1LL << 31))
    return set_error(RLDX_ERR_UNSUPPORTED, "kv4_read: too many rows");
  if (tokens == 0) return RLDX_OK;
  p.k = static_cast<__nv_bfloat16*>(k);
  p.v = static_cast<__nv_bfloat16*>(v);
  cudaError_t e = launch_kv4_read(p, cache->head_dim, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "kv4_read launch");
  return RLDX_OK;
}

}  // extern "C"
