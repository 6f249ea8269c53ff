// The norms after and before a block, with its gate and residual scale, of rows [rows, D]:
//   h' = h + scale * gate * post(y)            y the block's output, h the residual stream
//   n  = pre(h') * (1 + mod_scale) + mod_shift  what the next block reads
// post and pre are none, RMSNorm x / sqrt(mean(x^2) + eps) * w or LayerNorm (x - mean) / sqrt(var + eps) * w + b (w may
// count from one: 1 + w).  gate, mod_scale and mod_shift are vectors of all rows or of each group of rows.
//
// Everything is fp32 until the two results are rounded, once each; pre takes the sum before its rounding.  The
// variance is the mean square of what the mean leaves, from registers.
//
// A row lies in the registers of a team: 4 to 32 lanes, or as many warps as 16 values a thread ask for.  Bound by memory: y
// and h are read and h' and n written once; the vectors come from the caches.
#include "host_util.h"
#include "rows.cuh"

namespace rldx {

namespace {
constexpr int kNormValues = 16;  // of a thread
constexpr int kNormMaxWidth = 1024 * kNormValues;

struct NormsParams {
  const void* y;
  const void* h;
  void* h_out;
  void* n_out;  // null: pre is none
  long long ld_y, ld_h, ld_h_out, ld_n;
  const void* post_w;
  const void* post_b;
  const void* gate;
  const void* pre_w;
  const void* pre_b;
  const void* mod_scale;
  const void* mod_shift;
  long long ld_gate, ld_scale, ld_shift;  // of the groups' vectors; 0: one for all rows
  long long rows, group;
  int width, post, pre;      // RLDX_NORM_*
  int vectors_f32, aligned;  // the vectors' type; V of them may be loaded at once
  int team, warps;           // lanes of a row (4 to 32), warps of a row
  float scale, eps, plus_one;
};

template <int V>
__device__ __forceinline__ void each(float (&x)[V], float v) {
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = v;
}

// Values e .. e + V of a vector (of fp32 or the rows' type), `n` of them there.
template <typename T, int V>
__device__ __forceinline__ void vector_at(const NormsParams& P, const void* base, long long e, int n, float (&x)[V]) {
  if (P.vectors_f32) {
    const float* p = static_cast<const float*>(base) + e;
    if (P.aligned && n >= V)
      unpack_row<float, V>(load_shared_by_rows<float, V>(p), x);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = i < n ? __ldg(p + i) : 0.0f;
  } else {
    const T* p = static_cast<const T*>(base) + e;
    if (P.aligned && n >= V)
      unpack_row<T, V>(load_shared_by_rows<T, V>(p), x);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = i < n ? to_float(__ldg(p + i)) : 0.0f;
  }
}

template <typename T, int V>
__device__ __forceinline__ void row_at(const T* p, int n, float (&x)[V]) {
  if (n >= V)
    unpack_row<T, V>(load_once<T, V>(p), x);
  else
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = i < n ? to_float(p[i]) : 0.0f;
}
template <typename T, int V>
__device__ __forceinline__ void row_to(T* p, int n, const float (&x)[V]) {
  if (n >= V)
    store_once<T, V>(p, pack_row<T, V>(x));
  else
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = from_float<T>(x[i]);
}

// Sum over a row's team.  Of several warps: each leaves its sum, and all read them after a barrier; two sets of
// places take turns, so one barrier a sum is enough.
struct TeamSum {
  float* places;  // [2][warps of the row]
  int team, warps, warp, barrier, turn;
  __device__ __forceinline__ float operator()(float x) {
    for (int o = team >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (warps == 1) return x;
    float* p = places + turn * warps;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) p[warp] = x;
    named_bar_sync(barrier, 32 * warps);
    x = 0.0f;
    for (int w = 0; w < warps; ++w) x += p[w];
    return x;
  }
};

template <typename TY, typename TH, int V>
__global__ void __launch_bounds__(1024) block_norms_kernel(const __grid_constant__ NormsParams P) {
  constexpr int K = kNormValues / V;  // vectors of a thread
  __shared__ float places[2 * 32];
  griddep_wait();
  griddep_launch();
  const int threads = P.warps > 1 ? 32 * P.warps : P.team;  // of a row
  const int slot = threadIdx.x / threads, at = threadIdx.x - slot * threads;
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / threads) + slot;
  const bool real = row < P.rows;
  TeamSum sum{places + 2 * slot * (P.warps > 1 ? P.warps : 0), P.team, P.warps, at >> 5, 1 + slot, 0};
  const int D = P.width;
  const float inv_d = 1.0f / static_cast<float>(D), root_inv_d = rsqrtf(static_cast<float>(D));
  auto left = [&](int k) { return real ? D - (at + k * threads) * V : 0; };  // values there, V at most
  auto first = [&](int k) { return (at + k * threads) * V; };
  float x[K][V], h[K][V];
  const TY* y = static_cast<const TY*>(P.y) + row * P.ld_y;
  const TH* hin = static_cast<const TH*>(P.h) + row * P.ld_h;
#pragma unroll
  for (int k = 0; k < K; ++k) row_at<TY, V>(y + first(k), left(k), x[k]);
#pragma unroll
  for (int k = 0; k < K; ++k) row_at<TH, V>(hin + first(k), left(k), h[k]);

  // mean (of a LayerNorm) and 1 / sqrt of the mean square of what it leaves
  auto statistics = [&](int kind, float& mean, float& inv) {
    mean = 0.0f;
    if (kind == RLDX_NORM_LAYER) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s += x[k][i];  // (zeros where there is nothing)
      mean = sum(s) * inv_d;
    }
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = (x[k][i] - mean) * root_inv_d;  // (a mean, not a sum, of squares stays in range up to 1.8e19)
        s += i < left(k) ? d * d : 0.0f;
      }
    inv = rsqrtf(sum(s) + P.eps);
  };
  auto normed = [&](const void* w, const void* b, float mean, float inv) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (left(k) <= 0) continue;
      float wv[V], bv[V];
      each(wv, 1.0f), each(bv, 0.0f);
      if (w) {
        vector_at<TY, V>(P, w, first(k), left(k), wv);
#pragma unroll
        for (int i = 0; i < V; ++i) wv[i] += P.plus_one;
      }
      if (b) vector_at<TY, V>(P, b, first(k), left(k), bv);
#pragma unroll
      for (int i = 0; i < V; ++i) x[k][i] = fmaf((x[k][i] - mean) * inv, wv[i], bv[i]);
    }
  };

  float mean, inv;
  if (P.post != RLDX_NORM_NONE) {
    statistics(P.post, mean, inv);
    normed(P.post_w, P.post_b, mean, inv);
  }
  const long long g = real && P.group > 0 ? row / P.group : 0;
  TH* hout = static_cast<TH*>(P.h_out) + row * P.ld_h_out;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (left(k) > 0) {
      float gv[V];
      each(gv, 1.0f);
      if (P.gate) vector_at<TY, V>(P, P.gate, g * P.ld_gate + first(k), left(k), gv);
#pragma unroll
      for (int i = 0; i < V; ++i) x[k][i] = i < left(k) ? fmaf(P.scale * gv[i], x[k][i], h[k][i]) : 0.0f;
      row_to<TH, V>(hout + first(k), left(k), x[k]);
    }
  }
  if (P.pre == RLDX_NORM_NONE) return;  // (the same for every thread)
  statistics(P.pre, mean, inv);
  normed(P.pre_w, P.pre_b, mean, inv);
  TY* nout = static_cast<TY*>(P.n_out) + row * P.ld_n;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (left(k) <= 0) continue;
    if (P.mod_scale) {
      float sv[V];
      vector_at<TY, V>(P, P.mod_scale, g * P.ld_scale + first(k), left(k), sv);
#pragma unroll
      for (int i = 0; i < V; ++i) x[k][i] = fmaf(x[k][i], sv[i], x[k][i]);
    }
    if (P.mod_shift) {
      float sv[V];
      vector_at<TY, V>(P, P.mod_shift, g * P.ld_shift + first(k), left(k), sv);
#pragma unroll
      for (int i = 0; i < V; ++i) x[k][i] += sv[i];
    }
    row_to<TY, V>(nout + first(k), left(k), x[k]);
  }
}

template <typename TY, typename TH>
cudaError_t launch_block_norms(const NormsParams& p, int v, unsigned grid, unsigned block, cudaStream_t stream) {
  if constexpr (sizeof(TY) == 2)
    if (v == 8) return launch_overlapped(block_norms_kernel<TY, TH, 8>, grid, block, 0, stream, p);
  switch (v) {
    case 4: return launch_overlapped(block_norms_kernel<TY, TH, 4>, grid, block, 0, stream, p);
    case 2: return launch_overlapped(block_norms_kernel<TY, TH, 2>, grid, block, 0, stream, p);
    default: return launch_overlapped(block_norms_kernel<TY, TH, 1>, grid, block, 0, stream, p);
  }
}
}  // namespace

}  // namespace rldx

using namespace rldx;

extern "C" int rldx_block_norms(const rldx_block_norms_desc* d, void* stream) {
  auto bad = [](const char* what) { return set_error(RLDX_ERR_ARG, std::string("block_norms: ") + what); };
  if (!d) return bad("null description");
  if (!known_dtype(d->dtype) || (d->residual_dtype != d->dtype && d->residual_dtype != RLDX_F32) ||
      (d->vector_dtype != d->dtype && d->vector_dtype != RLDX_F32))
    return set_error(RLDX_ERR_UNSUPPORTED, "block_norms: residual and vectors have the branch's type or float32");
  if (d->rows < 0 || d->rows >= (1LL << 31)) return bad("0 to 2^31 - 1 rows");
  if (d->width < 1 || d->width > kNormMaxWidth)
    return set_error(RLDX_ERR_UNSUPPORTED, "block_norms: rows have 1 to " + std::to_string(kNormMaxWidth) + " values");
  for (int kind : {d->post, d->pre})
    if (kind != RLDX_NORM_NONE && kind != RLDX_NORM_RMS && kind != RLDX_NORM_LAYER) return bad("unknown norm");
  if (!d->branch || !d->residual || !d->residual_out || (d->pre != RLDX_NORM_NONE && !d->out)) return bad("null rows");
  if (d->pre == RLDX_NORM_NONE && (d->out || d->pre_weight || d->pre_bias || d->mod_scale || d->mod_shift))
    return bad("without a pre norm there are no out, weights or modulation of it");
  if (d->post == RLDX_NORM_NONE && (d->post_weight || d->post_bias)) return bad("without a post norm there are no weights of it");
  if (d->weight_plus_one && ((d->post != RLDX_NORM_NONE && !d->post_weight) || (d->pre != RLDX_NORM_NONE && !d->pre_weight)))
    return bad("weights that count from one need to be given");
  const int sy = dtype_bytes(d->dtype), sh = dtype_bytes(d->residual_dtype), sv = dtype_bytes(d->vector_dtype);
  const int64_t lds[4] = {d->ld_branch, d->ld_residual, d->ld_residual_out, d->pre != RLDX_NORM_NONE ? d->ld_out : d->width};
  if (lds[0] < 0 || lds[1] < 0) return bad("negative strides");  // (0: one row for all)
  if (lds[2] < d->width || lds[3] < d->width) return bad("rows of a result overlap");
  const bool grouped = d->ld_gate || d->ld_scale || d->ld_shift;
  if (d->rows_per_group < 0 || (grouped && d->rows_per_group < 1)) return bad("vectors of groups need rows_per_group");
  for (int64_t ld : {d->ld_gate, d->ld_scale, d->ld_shift})
    if (ld < 0 || (ld > 0 && ld < d->width)) return bad("vectors of groups overlap");
  const void* rows_at[4] = {d->branch, d->residual, d->residual_out, d->out};
  const int row_size[4] = {sy, sh, sh, sy};
  const void* vectors[7] = {d->post_weight, d->post_bias, d->gate, d->pre_weight, d->pre_bias, d->mod_scale, d->mod_shift};
  for (int i = 0; i < 4; ++i)
    if (reinterpret_cast<uintptr_t>(rows_at[i]) % row_size[i]) return bad("misaligned rows");
  for (const void* p : vectors)
    if (reinterpret_cast<uintptr_t>(p) % sv) return bad("a misaligned vector");
  if (d->rows == 0) return RLDX_OK;
  int rc = ensure_device();
  if (rc != RLDX_OK) return rc;

  NormsParams p;
  p.y = d->branch, p.h = d->residual, p.h_out = d->residual_out, p.n_out = d->out;
  p.ld_y = lds[0], p.ld_h = lds[1], p.ld_h_out = lds[2], p.ld_n = lds[3];
  p.post_w = d->post_weight, p.post_b = d->post_bias, p.gate = d->gate, p.pre_w = d->pre_weight, p.pre_b = d->pre_bias;
  p.mod_scale = d->mod_scale, p.mod_shift = d->mod_shift;
  p.ld_gate = d->ld_gate, p.ld_scale = d->ld_scale, p.ld_shift = d->ld_shift;
  p.rows = d->rows, p.group = d->rows_per_group;
  p.width = d->width, p.post = d->post, p.pre = d->pre;
  p.vectors_f32 = d->vector_dtype == RLDX_F32;
  p.scale = d->scale, p.eps = d->eps, p.plus_one = d->weight_plus_one ? 1.0f : 0.0f;
  // V values at a time: as many as the rows' common alignment allows.  The end of a row that they do not divide goes
  // value by value, and so do vectors whose own alignment is less.
  int v = d->dtype == RLDX_F32 ? 4 : 8;
  auto fits = [](const void* at, int64_t ld, int size, int v) {
    return ld % v == 0 && reinterpret_cast<uintptr_t>(at) % std::min(16, v * size) == 0;
  };
  for (int i = 0; i < 4; ++i)
    while (v > 1 && !fits(rows_at[i], lds[i], row_size[i], v)) v /= 2;
  p.aligned = 1;
  const int64_t vector_ld[7] = {0, 0, d->ld_gate, 0, 0, d->ld_scale, d->ld_shift};
  for (int i = 0; i < 7; ++i)
    if (!fits(vectors[i], vector_ld[i], sv, v)) p.aligned = 0;
  const int lanes = (d->width + kNormValues - 1) / kNormValues;
  p.warps = (lanes + 31) / 32;
  p.team = 4;
  while (p.team < 32 && p.team < lanes) p.team *= 2;
  const int threads = p.warps > 1 ? 32 * p.warps : p.team;
  const int teams = p.warps > 1 ? std::max(1, 4 / p.warps) : 128 / threads;
  const unsigned block = static_cast<unsigned>(teams * threads);
  const unsigned grid = static_cast<unsigned>((d->rows + teams - 1) / teams);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = d->residual_dtype == RLDX_F32;
  cudaError_t e;
  if (d->dtype == RLDX_F32)
    e = launch_block_norms<float, float>(p, v, grid, block, st);
  else if (d->dtype == RLDX_F16)
    e = wide ? launch_block_norms<__half, float>(p, v, grid, block, st) : launch_block_norms<__half, __half>(p, v, grid, block, st);
  else
    e = wide ? launch_block_norms<__nv_bfloat16, float>(p, v, grid, block, st)
             : launch_block_norms<__nv_bfloat16, __nv_bfloat16>(p, v, grid, block, st);
  if (e != cudaSuccess) return cuda_fail(e, "block_norms launch");
  return RLDX_OK;
}
