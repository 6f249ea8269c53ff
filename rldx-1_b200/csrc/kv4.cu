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

// Unit of the cache (start, or null) and token in the unit of new-token row `row`.
__device__ __forceinline__ uint8_t* kv4_token_unit(const Kv4Cache& c, const int* cu, const int* lengths, int row,
                                                   int head, int unit_bytes, int* tau) {
  const int b = seq_of_row(cu, c.seqs, row);
  const int pos = lengths[b] - cu[b + 1] + row;
  *tau = pos & (kKv4Unit - 1);
  const int index = pos >= 0 ? kv4_unit_index(c, b, head, pos / kKv4Unit) : -1;
  if (index < 0) {
    record_error(kErrKv4Table);
    return nullptr;
  }
  return c.data + static_cast<long long>(index) * unit_bytes;
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

// D / 8 lanes own a (token, head) row, 8 channels each; kRows rows per lane group, their loads
// issued before any arithmetic.  Heads of a token are ordered [q | k | v].
template <int D, int kRows, typename Rope>
__global__ void __launch_bounds__(128) kv4_append_kernel(const __grid_constant__ Kv4AppendParams P) {
  using U = Kv4Unit<D>;
  constexpr int kLanes = D / 8;
  __shared__ int s_seq[2 * kKv4SmemSeqs + 1];
  griddep_wait();
  const int hq = P.q_heads, hkv = P.c.kv_heads, heads = hq + 2 * hkv;
  const long long nrows = static_cast<long long>(P.c.tokens) * heads;
  const long long group = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / kLanes;
  const int l = threadIdx.x % kLanes;
  const long long row0 = group * kRows;
  float x[kRows][8];
  int tok[kRows], head[kRows], rp[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const long long row = min(row0 + r, nrows - 1);  // clamped: rows past the end are not stored
    tok[r] = static_cast<int>(row / heads);
    head[r] = static_cast<int>(row - static_cast<long long>(tok[r]) * heads);
    load8(P.qkv + tok[r] * P.ld + head[r] * D + 8 * l, x[r]);
    rp[r] = __ldg(P.rope_pos + tok[r]);
  }
  const int *cu, *lengths;
  stage_seqs(P.c, s_seq, &cu, &lengths);
  __syncthreads();
  griddep_launch();
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const bool live = row0 + r < nrows;
    const bool is_v = head[r] >= hq + hkv;
    if (!is_v) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[r][e], x[r][e], ss);
      // rows of one warp may be q / k in one lane group and v in another: the mask names the group
      const unsigned lanes = (kLanes == 16 ? 0xffffu : 0xffu) << ((threadIdx.x & 31) / kLanes * kLanes);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(lanes, ss, o);
      const float rstd = rsqrtf(ss * (1.0f / D) + P.eps);
      float w[8], c[8], s[8];
      load8((head[r] < hq ? P.wq : P.wk) + 8 * l, w);
      if (static_cast<unsigned>(rp[r]) >= static_cast<unsigned>(P.rope_rows)) {
        if (live) record_error(kErrKv4Rope);
        rp[r] = 0;
      }
      load8(static_cast<const Rope*>(P.cos) + static_cast<long long>(rp[r]) * D + 8 * l, c);
      load8(static_cast<const Rope*>(P.sin) + static_cast<long long>(rp[r]) * D + 8 * l, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __fmul_rn(__fmul_rn(x[r][e], rstd), w[e]);
        const float o = __shfl_xor_sync(lanes, y, kLanes / 2);  // the channel half a head away
        x[r][e] = __fadd_rn(__fmul_rn(y, c[e]), __fmul_rn(l < kLanes / 2 ? -o : o, s[e]));
      }
    }
    if (head[r] < hq) {
      if (live) {
        uint4 u;
        u.x = pack_bf16x2(x[r][0], x[r][1]);
        u.y = pack_bf16x2(x[r][2], x[r][3]);
        u.z = pack_bf16x2(x[r][4], x[r][5]);
        u.w = pack_bf16x2(x[r][6], x[r][7]);
        *reinterpret_cast<uint4*>(P.q + (static_cast<long long>(tok[r]) * hq + head[r]) * D + 8 * l) = u;
      }
      continue;
    }
    // four lanes share a group of 32 channels
    const unsigned quad = 0xfu << (threadIdx.x & 28);
    float mn = x[r][0], mx = x[r][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mn = min_nan(mn, x[r][e]), mx = max_nan(mx, x[r][e]);
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
      mn = min_nan(mn, __shfl_xor_sync(quad, mn, o));
      mx = max_nan(mx, __shfl_xor_sync(quad, mx, o));
    }
    mn = max_nan(min_nan(mn, 65504.0f), -65504.0f);
    mx = max_nan(min_nan(mx, 65504.0f), -65504.0f);
    const __half low_h = __float2half_rn(mn);
    const __half scale_h = __float2half_rn(__fmul_rn(mx - mn, 1.0f / 15.0f));
    const float low = __half2float(low_h), scale = __half2float(scale_h);
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
    uint32_t codes = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[r][e], low), inv)), 0.0f), 15.0f);  // NaN: 0
      codes |= static_cast<uint32_t>(c) << (4 * e);
    }
    if (!live) continue;
    const int h = head[r] - hq - (is_v ? hkv : 0);
    int tau;
    uint8_t* unit = kv4_token_unit(P.c, cu, lengths, tok[r], h, U::kBytes, &tau);
    if (unit == nullptr) continue;
    const int j = l / 4, t4 = l % 4;  // group, position in the group
    if (!is_v) {
      *reinterpret_cast<uint32_t*>(unit + tau * U::kRow + 4 * (t4 * U::kG + j)) = codes;
      if (t4 == 0) {
        __half* meta = reinterpret_cast<__half*>(unit + U::kKMeta + 4 * U::kG * tau);
        meta[j] = scale_h;
        meta[U::kG + j] = low_h;
      }
    } else {
      const int blk = tau / 16, hh = tau / 8 % 2, t = tau / 2 % 4, e = tau % 2;
      uint8_t* at = unit + U::kV + 8 * D * blk + 4 * D * hh + 4 * U::kG * t + 2 * U::kG * e + 2 * j;
      *reinterpret_cast<uint16_t*>(at + 16 * U::kG * (2 * t4)) = static_cast<uint16_t>(codes);
      *reinterpret_cast<uint16_t*>(at + 16 * U::kG * (2 * t4 + 1)) = static_cast<uint16_t>(codes >> 16);
      if (t4 == 0) {
        const int m = 32 * U::kG * blk + 16 * U::kG * hh + 4 * U::kG * t + 4 * j + 2 * e;
        *reinterpret_cast<__half*>(unit + U::kVScale + m) = scale_h;
        *reinterpret_cast<__half*>(unit + U::kVLow + m) = low_h;
      }
    }
  }
}

// D / 8 lanes own one (token, kv head, K or V) row.
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
  if (row >= static_cast<long long>(P.c.tokens) * hkv * 2) return;
  const int l = threadIdx.x % kLanes, j = l / 4, t4 = l % 4;
  const int tok = static_cast<int>(row / (2 * hkv)), which = static_cast<int>(row - static_cast<long long>(tok) * 2 * hkv);
  const bool is_v = which >= hkv;
  const int h = is_v ? which - hkv : which;
  int tau;
  const uint8_t* unit = kv4_token_unit(P.c, cu, lengths, tok, h, U::kBytes, &tau);
  uint4 o = make_uint4(0u, 0u, 0u, 0u);
  if (unit != nullptr) {
    uint32_t codes;
    float scale, low;
    if (!is_v) {
      codes = *reinterpret_cast<const uint32_t*>(unit + tau * U::kRow + 4 * (t4 * U::kG + j));
      const __half* meta = reinterpret_cast<const __half*>(unit + U::kKMeta + 4 * U::kG * tau);
      scale = __half2float(meta[j]);
      low = __half2float(meta[U::kG + j]);
    } else {
      const int blk = tau / 16, hh = tau / 8 % 2, t = tau / 2 % 4, e = tau % 2;
      const uint8_t* at = unit + U::kV + 8 * D * blk + 4 * D * hh + 4 * U::kG * t + 2 * U::kG * e + 2 * j;
      codes = *reinterpret_cast<const uint16_t*>(at + 16 * U::kG * (2 * t4));
      codes |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(at + 16 * U::kG * (2 * t4 + 1))) << 16;
      const int m = 32 * U::kG * blk + 16 * U::kG * hh + 4 * U::kG * t + 4 * j + 2 * e;
      scale = __half2float(*reinterpret_cast<const __half*>(unit + U::kVScale + m));
      low = __half2float(*reinterpret_cast<const __half*>(unit + U::kVLow + m));
    }
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(scale, static_cast<float>(codes >> (4 * i) & 15u), low);
    o.x = pack_bf16x2(v[0], v[1]);
    o.y = pack_bf16x2(v[2], v[3]);
    o.z = pack_bf16x2(v[4], v[5]);
    o.w = pack_bf16x2(v[6], v[7]);
  }
  __nv_bfloat16* dst = (is_v ? P.v : P.k) + (static_cast<long long>(tok) * hkv + h) * D + 8 * l;
  *reinterpret_cast<uint4*>(dst) = o;
}

namespace {
template <typename Params>
cudaError_t launch_rows(void (*kernel)(Params), const Params& p, long long groups, int lanes, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((groups * lanes + 127) / 128), 1, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int D, int kRows>
cudaError_t launch_append(const Kv4AppendParams& p, long long rows, cudaStream_t stream) {
  const long long groups = (rows + kRows - 1) / kRows;
  return p.rope_f32 ? launch_rows<Kv4AppendParams>(kv4_append_kernel<D, kRows, float>, p, groups, D / 8, stream)
                    : launch_rows<Kv4AppendParams>(kv4_append_kernel<D, kRows, __nv_bfloat16>, p, groups, D / 8, stream);
}
}  // namespace

cudaError_t launch_kv4_append(const Kv4AppendParams& p, int head_dim, cudaStream_t stream) {
  const long long rows = static_cast<long long>(p.c.tokens) * (p.q_heads + 2 * p.c.kv_heads);
  return head_dim == 128 ? launch_append<128, 1>(p, rows, stream) : launch_append<64, 1>(p, rows, stream);
}

cudaError_t launch_kv4_read(const Kv4ReadParams& p, int head_dim, cudaStream_t stream) {
  const long long rows = static_cast<long long>(p.c.tokens) * p.c.kv_heads * 2;
  return head_dim == 128 ? launch_rows<Kv4ReadParams>(kv4_read_kernel<128>, p, rows, 16, stream)
                         : launch_rows<Kv4ReadParams>(kv4_read_kernel<64>, p, rows, 8, stream);
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
  if (static_cast<long long>(tokens) * (q_heads + 2 * cache->kv_heads) >= (1LL << 31))
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
