// The norms after and before a block, with its gate and residual scale, of rows [rows, D]:
//   h' = h + scale * gate * post(y)            y the block's output, h the residual stream
//   n  = pre(h') * (1 + mod_scale) + mod_shift  what the next block reads
// post and pre are none, RMSNorm x / sqrt(mean(x^2) + eps) * w or LayerNorm (x - mean) / sqrt(var + eps) * w + b (w may
// count from one: 1 + w).  gate, mod_scale and mod_shift are vectors of all rows or of each group of rows.
//
// Everything is fp32 until the two results are rounded, once each; pre takes the sum before its rounding.  The
// variance is the mean square of what the mean leaves, from registers.
//
// A row lies in the registers of a team: 8 lanes, a warp or several, 16 values a thread.  The vectors come down
// to four numbers a value, h' = h + (a y^ + b) and n = c h^ + d with a = scale gate (w + 1), b = scale gate b, c = (w + 1)
// (1 + mod_scale), d = b (1 + mod_scale) + mod_shift, kept in shared memory and made once by a CTA.  Vectors of groups are
// read beside the rows, as they are, where they have the rows' type and alignment, rows are of at most 4096 values
// and either a group has fewer than 16 rows or a row is 8 lanes' (128 values); else each team makes its own four numbers
// whenever it comes to another group.  A CTA goes over a run of rows, the next of which is on the way while one is
// normed.  Bound by memory: y and h are read and h' and n written once.  8832 x 2048 bf16 with norms on both sides takes 26 us
// (5.6 TB/s; at the copy's rate 22), with channel gates 27, 35968 x 1536 with a modulation of each 562 rows 83 (68), 4999 x
// 1001 fp16 with an fp32 stream 16.3 (9.2: one value at a time, and 450 instructions a warp and row of 512 values).
#include <utility>

#include "host_util.h"
#include "rows.cuh"

namespace rldx {

namespace {
constexpr int kNormMaxWidth = 14336;  // four vectors of it fill the shared memory
constexpr int kNormShared = 4 * 4 * kNormMaxWidth;
// Values of a thread: 16, and 8 of those taken one by one, whose rows are often narrow (100000 x 157 bf16: 75 us with 16, 44 with 8;
// 4999 x 1001 fp16 with an fp32 stream 18.7 and 16.2; 20000 x 1001 bf16 41 and 43).
template <int V, int kThreads>
constexpr int kNormValues = V == 1 && kThreads == 256 ? 8 : 16;
enum { kNormA = 0, kNormB = 1, kNormC = 2, kNormD = 3 };

struct NormsParams {
  const void* y;
  const void* h;
  void* h_out;
  void* n_out;
  long long ld_y, ld_h, ld_h_out, ld_n;
  const void* post_w;
  const void* post_b;
  const void* gate;
  const void* pre_w;
  const void* pre_b;
  const void* mod_scale;
  const void* mod_shift;
  long long ld_gate, ld_scale, ld_shift;  // of the groups' vectors
  long long rows, group;
  // of groups, read beside the rows (the ones above are null then)
  const void* row_gate;
  const void* row_scale;
  const void* row_shift;
  int run;                 // rows of a team
  int width, post, pre;    // RLDX_NORM_*
  int place[4];            // of a, b, c, d in shared memory (values); -1: a is scale, c one, b and d zero
  int copy;                // and of a team's own copy of them; 0: one for all
  int padded;              // values of one of them there
  int vectors_f32, aligned;  // the vectors' type; four of them may be loaded at once
  int warps;               // of a row
  float scale, eps, plus_one;
};

// Values e .. e + V of a vector (of fp32 or the rows' type) that begins `from` values past base; what is past the width stays.
template <typename T, int V>
__device__ __forceinline__ void vector_at(const NormsParams& P, const void* base, long long from, int e, float (&x)[V]) {
  auto read = [&](auto* p) {
    using S = std::remove_cv_t<std::remove_reference_t<decltype(*p)>>;
    p += from + e;
    if (P.aligned && e + V <= P.width)
      unpack_row<S, V>(load_shared_by_rows<S, V>(p), x);
    else
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (e + i < P.width) x[i] = to_float(__ldg(p + i));
  };
  if (P.vectors_f32)
    read(static_cast<const float*>(base));
  else
    read(static_cast<const T*>(base));
}

// Sum over a row's team.  Several warps are all of the CTA: each leaves its sum, and all read them after a barrier; two
// sets of places take turns, so one barrier a sum is enough.
template <int kLanes, int kWarps>
struct TeamSum {
  float* places;  // [2][kWarps], zeros past the row's warps
  bool several;
  int turn = 0;
  __device__ __forceinline__ float operator()(float x) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (kLanes < 32 || !several) return x;
    float* p = places + turn;
    turn ^= kWarps;
    if ((threadIdx.x & 31) == 0) p[threadIdx.x >> 5] = x;
    __syncthreads();
    x = p[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
  }
};

// Threads that run on an SM at once, from their registers: 80 with vectors of eight and with single values, 64 in CTAs of up to
// 1024, 128 else.
template <int V, int kThreads>
constexpr int kNormResident = kThreads > 256 ? 1024 : V == 8 || V == 1 ? 768 : 512;  // (V == 0: with vectors of groups)

// V values at a time, which divides the width; kLanes: of a row, or of one of its warps; kDirect: vectors of groups are
// read beside the rows.
template <typename TY, typename TH, int V, int kLanes, int kThreads, bool kDirect>
__global__ void __launch_bounds__(kThreads, kNormResident<kDirect ? 0 : V, kThreads> / kThreads) block_norms_kernel(const __grid_constant__ NormsParams P) {
  constexpr int E = kNormValues<V, kThreads>, K = E / V, kStep = kLanes * V;
  constexpr int kWarps = kThreads / 32;
  extern __shared__ __align__(16) float shared[];  // a, b, c, d
  __shared__ float places[2 * kWarps];
  griddep_wait();
  griddep_launch();
  const int threads = P.warps > 1 ? 32 * P.warps : kLanes;  // of a row
  const int teams = blockDim.x / threads, slot = P.warps > 1 ? 0 : threadIdx.x / kLanes, at = threadIdx.x - slot * threads;
  if (threadIdx.x < 2 * kWarps) places[threadIdx.x] = 0.0f;
  TeamSum<kLanes, kWarps> sum{places, P.warps > 1};
  long long row = static_cast<long long>(blockIdx.x) * teams * P.run + slot;
  const long long row_end = min(P.rows, row - slot + teams * P.run);
  // Vector k of a thread begins at value first + k kStep; `have` of them are there.
  const int width = P.width, first = at / kLanes * (kLanes * E) + at % kLanes * V;
  const int have = min(K, max(0, (width - first + kStep - 1) / kStep));
  const float inv_d = 1.0f / static_cast<float>(width), root_inv_d = rsqrtf(static_cast<float>(width));

  const TY* y_at = static_cast<const TY*>(P.y) + row * P.ld_y + first;
  const TH* h_at = static_cast<const TH*>(P.h) + row * P.ld_h + first;
  TH* h_to = static_cast<TH*>(P.h_out) + row * P.ld_h_out + first;
  TY* n_to = static_cast<TY*>(P.n_out) + row * P.ld_n + first;
  Raw<TY, V> y[K];
  Raw<TH, V> h[K];
  auto load_y = [&](int have) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      y[k] = Raw<TY, V>{};
      if (k < have) y[k] = load_once<TY, V>(y_at + k * kStep);
    }
    y_at += teams * P.ld_y;
  };
  auto load_h = [&](int have) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      h[k] = Raw<TH, V>{};
      if (k < have) h[k] = load_once<TH, V>(h_at + k * kStep);
    }
    h_at += teams * P.ld_h;
  };
  load_y(row < row_end ? have : 0);
  load_h(row < row_end ? have : 0);
  constexpr int kDirectVecs = kDirect ? K : 1;
  Raw<TY, V> gate[kDirectVecs], scale[kDirectVecs], shift[kDirectVecs];
  auto load_vector = [&](auto& to, const void* base, long long ld, long long of_row, int have) {
    if constexpr (kDirect) {
      if (!base) return;
      const TY* from = static_cast<const TY*>(base) + static_cast<uint32_t>(of_row) / static_cast<uint32_t>(P.group) * ld + first;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (k < have) to[k] = load_shared_by_rows<TY, V>(from + k * kStep);
    }
  };
  if (row < row_end) {
    load_vector(gate, P.row_gate, P.ld_gate, row, have);
    load_vector(scale, P.row_scale, P.ld_scale, row, have);
    load_vector(shift, P.row_shift, P.ld_shift, row, have);
  }

  // a, b, c, d of group g, by `by` threads of which this is the `me`-th, four values at a time; threads of eight values
  // read theirs in two halves, each side by side with the other threads' (half: where the second ones begin)
  float* const mine = shared + slot * P.copy;
  const int half = V == 8 ? P.padded / 2 : 0;
  auto make_vectors = [&](long long g, int me, int by) {
#pragma unroll 2
    for (int e = 4 * me; e < P.padded; e += 4 * by) {
      auto values = [&](const void* base, long long ld, float otherwise, float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = otherwise;
        if (base) vector_at<TY, 4>(P, base, g * ld, e, v);
      };
      const int to = V == 8 ? (e >> 1 & ~3) + (e & 4 ? half : 0) : e;
      auto put = [&](int which, const float (&v)[4]) {
        *reinterpret_cast<float4*>(mine + P.place[which] + to) = make_float4(v[0], v[1], v[2], v[3]);
      };
      float v[4], w[4];
      if (P.place[kNormA] >= 0 || P.place[kNormB] >= 0) {
        float gate[4];
        values(P.gate, P.ld_gate, 1.0f, gate);
        values(P.post_w, 0, 1.0f - P.plus_one, v);
        values(P.post_b, 0, 0.0f, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) gate[i] *= P.scale, v[i] = gate[i] * (v[i] + P.plus_one), w[i] *= gate[i];
        if (P.place[kNormA] >= 0) put(kNormA, v);
        if (P.place[kNormB] >= 0) put(kNormB, w);
      }
      if (P.place[kNormC] >= 0 || P.place[kNormD] >= 0) {
        float scale[4], shift[4];
        values(P.mod_scale, P.ld_scale, 0.0f, scale);
        values(P.mod_shift, P.ld_shift, 0.0f, shift);
        values(P.pre_w, 0, 1.0f - P.plus_one, v);
        values(P.pre_b, 0, 0.0f, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += P.plus_one, v[i] = fmaf(v[i], scale[i], v[i]), w[i] = fmaf(w[i], scale[i], w[i]) + shift[i];
        if (P.place[kNormC] >= 0) put(kNormC, v);
        if (P.place[kNormD] >= 0) put(kNormD, w);
      }
    }
  };
  const bool grouped = P.copy > 0;
  long long group_end = 0;
  if (grouped) {
    const long long g = min(row, P.rows - 1) / P.group;
    group_end = (g + 1) * P.group;
    make_vectors(g, at, threads);
  } else {
    make_vectors(0, threadIdx.x, blockDim.x);
  }
  __syncthreads();

#pragma unroll 1
  for (int left = P.run; left > 0; --left) {  // (the same count for every team: lanes of a warp stay together)
    asm volatile("" ::: "memory");  // (a to d are read anew for each row: kept in registers they would take most of them)
    const int next = left > 1 && row + teams < row_end ? have : 0, here = row < row_end ? have : 0;
    float2 x[E / 2];  // two by two, in packed arithmetic
#pragma unroll
    for (int k = 0; k < K; ++k) unpack_row<TY, V>(y[k], *reinterpret_cast<float(*)[V]>(reinterpret_cast<float*>(x) + k * V));
    load_y(next);
    auto each = [&](auto f) {
#pragma unroll
      for (int j = 0; j < E / 2; ++j) x[j] = f(x[j]);
    };
    auto times = [&](float v) { each([v](float2 a) { return mul_f32x2(a, make_float2(v, v)); }); };
    // 1 / sqrt of the mean square of x, centred first for a LayerNorm (x is zero where nothing is, and then again)
    auto inverse_size = [&](int kind) {
      auto total = [&](float2 s) { return sum(s.x + s.y); };
      if (kind == RLDX_NORM_LAYER) {
        float2 s = x[0];
#pragma unroll
        for (int j = 1; j < E / 2; ++j) s = add_f32x2(s, x[j]);
        const float mean = total(s) * inv_d;
        each([mean](float2 a) { return add_f32x2(a, make_float2(-mean, -mean)); });
        if (have < K) {
          float* v = reinterpret_cast<float*>(x);
#pragma unroll
          for (int k = 0; k < K; ++k)
            if (k >= have)
#pragma unroll
              for (int i = 0; i < V; ++i) v[k * V + i] = 0.0f;
        }
      }
      float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        const float2 v = mul_f32x2(x[j], make_float2(root_inv_d, root_inv_d));  // (a mean, not a sum, of squares is in range up to 1.8e19)
        s = fma_f32x2(v, v, s);
      }
      return rsqrtf(total(s) + P.eps);
    };
    // f(x, numbers) with those of a vector in shared memory (past the width x is 0, and b and d are)
    auto with = [&](int which, auto f) {
      const int place = P.place[which];
      if (place < 0) return;
      const float* from = mine + place + (V == 8 ? first / 2 : first);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float2 v[(V + 1) / 2];
        if constexpr (V == 1) {
          if (k % 2 == 0) x[k / 2] = f(x[k / 2], make_float2(from[k * kStep], from[(k + 1) * kStep]));
        } else {
#pragma unroll
          for (int i = 0; i < V / 4; ++i)
            *reinterpret_cast<float4*>(v + 2 * i) = *reinterpret_cast<const float4*>(from + (V == 8 ? k * kStep / 2 : k * kStep) + (i ? half : 0));
#pragma unroll
          for (int i = 0; i < V / 2; ++i) x[k * V / 2 + i] = f(x[k * V / 2 + i], v[i]);
        }
      }
    };
    auto product = [](float2 a, float2 b) { return mul_f32x2(a, b); };
    auto plus = [](float2 a, float2 b) { return add_f32x2(a, b); };
    // f(x, numbers) with those of the row's group
    auto with_group = [&](const void* base, const auto& of, auto f) {
      if constexpr (kDirect) {
        if (!base) return;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (k >= have) continue;
          float v[V];
          unpack_row<TY, V>(of[k], v);
#pragma unroll
          for (int i = 0; i < V / 2; ++i) x[k * V / 2 + i] = f(x[k * V / 2 + i], make_float2(v[2 * i], v[2 * i + 1]));
        }
      }
    };
    auto vector = [&](int k) -> const float(&)[V] { return *reinterpret_cast<const float(*)[V]>(reinterpret_cast<const float*>(x) + k * V); };

    const float post = P.post != RLDX_NORM_NONE ? inverse_size(P.post) : 1.0f;
    times(P.place[kNormA] < 0 ? P.scale * post : post);
    with(kNormA, product);
    with(kNormB, plus);
    with_group(P.row_gate, gate, product);
    load_vector(gate, P.row_gate, P.ld_gate, row + teams, next);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float r[V];
      unpack_row<TH, V>(h[k], r);
      float* v = reinterpret_cast<float*>(x) + k * V;
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += r[i];
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k < here) store_once<TH, V>(h_to + k * kStep, pack_row<TH, V>(vector(k)));
    load_h(next);
    if (P.pre != RLDX_NORM_NONE) {  // (the same for every thread)
      times(inverse_size(P.pre));
      with(kNormC, product);
      with(kNormD, plus);
      with_group(P.row_scale, scale, [](float2 a, float2 b) { return fma_f32x2(a, b, a); });
      with_group(P.row_shift, shift, plus);
      load_vector(scale, P.row_scale, P.ld_scale, row + teams, next);
      load_vector(shift, P.row_shift, P.ld_shift, row + teams, next);
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (k < here) store_once<TY, V>(n_to + k * kStep, pack_row<TY, V>(vector(k)));
      n_to += teams * P.ld_n;
    }
    h_to += teams * P.ld_h_out;
    row += teams;
    const bool next_group = grouped && row >= group_end && left > 1 && row < row_end;
    if (__any_sync(0xffffffffu, next_group)) {  // (several warps are one team, and agree)
      const auto wait = [&] {
        if (P.warps > 1)
          __syncthreads();
        else
          __syncwarp();
      };
      wait();  // the last row's numbers have been read
      if (next_group) {
        const long long g = row / P.group;
        group_end = (g + 1) * P.group;
        make_vectors(g, at, threads);
      }
      wait();
    }
  }
}

template <typename TY, typename TH, int V, int kLanes, int kThreads, bool kDirect>
cudaError_t launch_norms(NormsParams p, int values, cudaStream_t stream) {
  // as many teams as run at once, each with its run of rows
  const int block = p.warps > 1 ? 32 * p.warps : 128, teams = p.warps > 1 ? 1 : block / kLanes;
  const long long resident = static_cast<long long>(sm_count()) * std::max(1, kNormResident<kDirect ? 0 : V, kThreads> / block) * teams;
  p.run = static_cast<int>(std::max(1LL, (p.rows + resident - 1) / resident));
  const long long all_teams = (p.rows + p.run - 1) / p.run;
  const size_t smem = sizeof(float) * values * (p.copy ? teams : 1);
  auto* kernel = block_norms_kernel<TY, TH, V, kLanes, kThreads, kDirect>;
  if (smem > 47 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormShared);
    if (e != cudaSuccess) return e;
  }
  return launch_overlapped(kernel, static_cast<unsigned>((all_teams + teams - 1) / teams), static_cast<unsigned>(block), smem, stream, p);
}
template <typename TY, typename TH, int V>
cudaError_t launch_block_norms(NormsParams p, bool grouped, bool direct, cudaStream_t stream) {
  // a row of up to 8 lanes' values is theirs, else a warp's or several
  constexpr int e = kNormValues<V, 256>;
  const int lanes = p.width <= 8 * e ? 8 : 32;
  const bool wide = p.width > 256 * e;
  const int ev = wide ? kNormValues<V, 1024> : e;
  p.warps = (p.width + lanes * ev - 1) / (lanes * ev);
  p.padded = lanes * p.warps * ev;  // 14336 at most
  p.row_gate = p.row_scale = p.row_shift = nullptr;
  // Read beside the rows, the vectors of groups cost registers and their bytes with every row; made into four numbers, a barrier
  // and a pass over the row's width with every group (us, 8832 x 2048 bf16, gate and modulation of groups of 1, 4, 16, 50 rows: 50, 40,
  // 37, 36 against 112, 49, 35, 28; 100000 x 128, groups of 100: 21 against 29).
  direct = direct && V > 1 && !wide && (lanes == 8 || p.group < 16);
  if (direct) {
    if (p.ld_gate) std::swap(p.gate, p.row_gate);
    if (p.ld_scale || p.ld_shift) std::swap(p.mod_scale, p.row_scale), std::swap(p.mod_shift, p.row_shift);
    grouped = false;
  }
  const bool held[4] = {p.post_w || p.gate, p.post_b != nullptr, p.pre_w || p.mod_scale, p.pre_b || p.mod_shift};
  int values = 0;
  for (int i = 0; i < 4; ++i) {
    p.place[i] = held[i] ? values : -1;
    values += held[i] ? p.padded : 0;
  }
  if (!values) p.padded = 0;
  p.copy = grouped ? values : 0;
  if constexpr (V > 1)
    if (direct) return lanes == 8 ? launch_norms<TY, TH, V, 8, 256, true>(p, values, stream) : launch_norms<TY, TH, V, 32, 256, true>(p, values, stream);
  return lanes == 8 ? launch_norms<TY, TH, V, 8, 256, false>(p, values, stream)
         : !wide   ? launch_norms<TY, TH, V, 32, 256, false>(p, values, stream)
                   : launch_norms<TY, TH, V, 32, 1024, false>(p, values, stream);
}
template <typename TY, typename TH>
cudaError_t launch_block_norms(const NormsParams& p, bool whole, bool grouped, bool direct, cudaStream_t stream) {
  return whole ? launch_block_norms<TY, TH, 16 / sizeof(TY)>(p, grouped, direct, stream) : launch_block_norms<TY, TH, 1>(p, grouped, false, stream);
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
  const bool grouped = (d->gate && d->ld_gate) || (d->mod_scale && d->ld_scale) || (d->mod_shift && d->ld_shift);
  if (d->rows_per_group < 0 || ((d->ld_gate || d->ld_scale || d->ld_shift) && d->rows_per_group < 1)) return bad("vectors of groups need rows_per_group");
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
  p.rows = d->rows, p.group = std::min(d->rows_per_group, d->rows);  // (fits 31 bits)
  p.width = d->width, p.post = d->post, p.pre = d->pre;
  p.vectors_f32 = d->vector_dtype == RLDX_F32;
  p.scale = d->scale, p.eps = d->eps, p.plus_one = d->weight_plus_one ? 1.0f : 0.0f;
  // 16 bytes of y at a time where the rows' alignment and the width allow it, else one value
  const int v = 16 / sy;
  auto fits = [](const void* at, int64_t ld, int size, int v) {
    return ld % v == 0 && reinterpret_cast<uintptr_t>(at) % std::min(16, v * size) == 0;
  };
  bool whole = d->width % v == 0;
  for (int i = 0; i < 4; ++i) whole &= fits(rows_at[i], lds[i], row_size[i], v);
  p.aligned = 1;
  const int64_t vector_ld[7] = {0, 0, d->ld_gate, 0, 0, d->ld_scale, d->ld_shift};
  for (int i = 0; i < 7; ++i)
    if (!fits(vectors[i], vector_ld[i], sv, 4)) p.aligned = 0;
  bool direct = grouped && sv == sy;  // the groups' vectors as the rows
  for (int i : {2, 5, 6}) direct &= fits(vectors[i], vector_ld[i], sv, v);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = d->residual_dtype == RLDX_F32;
  cudaError_t e;
  if (d->dtype == RLDX_F32)
    e = launch_block_norms<float, float>(p, whole, grouped, direct, st);
  else if (d->dtype == RLDX_F16)
    e = wide ? launch_block_norms<__half, float>(p, whole, grouped, direct, st) : launch_block_norms<__half, __half>(p, whole, grouped, direct, st);
  else
    e = wide ? launch_block_norms<__nv_bfloat16, float>(p, whole, grouped, direct, st)
             : launch_block_norms<__nv_bfloat16, __nv_bfloat16>(p, whole, grouped, direct, st);
  if (e != cudaSuccess) return cuda_fail(e, "block_norms launch");
  return RLDX_OK;
}
