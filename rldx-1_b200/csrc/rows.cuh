// Typed vectors of a row (bf16, fp16, fp32, 2 to 32 bytes) and the order of floats as whole numbers, shared by
// the row operators (rope.cu, block_norms.cu, logprobs.cu) and sampling.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/rldx_b200.h"
#include "common.cuh"

namespace rldx {

// V values of type T as they lie in memory, in 16-byte words where they fill them.
template <int kBytes>
struct RawBytes;
template <>
struct RawBytes<2> {
  uint16_t w[1];
};
template <>
struct RawBytes<4> {
  uint32_t w[1];
};
template <>
struct RawBytes<8> {
  uint2 w[1];
};
template <>
struct RawBytes<16> {
  uint4 w[1];
};
template <>
struct RawBytes<32> {
  uint4 w[2];
};
template <typename T, int V>
using Raw = RawBytes<V * static_cast<int>(sizeof(T))>;

// Values read once (streamed past the caches) and values that every row reads.
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_once(const T* p) {
  Raw<T, V> r;
  using W = std::remove_reference_t<decltype(r.w[0])>;
  constexpr int n = sizeof(r) / sizeof(W);
#pragma unroll
  for (int i = 0; i < n; ++i) {
    if constexpr (sizeof(W) == 2)
      r.w[i] = __ldcs(reinterpret_cast<const unsigned short*>(p) + i);
    else
      r.w[i] = __ldcs(reinterpret_cast<const W*>(p) + i);
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_shared_by_rows(const T* p) {
  Raw<T, V> r;
  using W = std::remove_reference_t<decltype(r.w[0])>;
  constexpr int n = sizeof(r) / sizeof(W);
#pragma unroll
  for (int i = 0; i < n; ++i) {
    if constexpr (sizeof(W) == 2)
      r.w[i] = __ldg(reinterpret_cast<const unsigned short*>(p) + i);
    else
      r.w[i] = __ldg(reinterpret_cast<const W*>(p) + i);
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_once(T* p, const Raw<T, V>& r) {
  using W = std::remove_cv_t<std::remove_reference_t<decltype(r.w[0])>>;
  constexpr int n = sizeof(r) / sizeof(W);
#pragma unroll
  for (int i = 0; i < n; ++i) {
    if constexpr (sizeof(W) == 2)
      __stcs(reinterpret_cast<unsigned short*>(p) + i, r.w[i]);
    else
      __stcs(reinterpret_cast<W*>(p) + i, r.w[i]);
  }
}

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }
template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    return __float2bfloat16_rn(x);
  else if constexpr (std::is_same_v<T, __half>)
    return __float2half_rn(x);
  else
    return x;
}

template <typename T, int V>
__device__ __forceinline__ void unpack_row(const Raw<T, V>& r, float (&x)[V]) {
  if constexpr (std::is_same_v<T, float> || V == 1) {
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = to_float(e[i]);
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        unpack_bf16x2(w[i], x[2 * i], x[2 * i + 1]);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(w + i));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      }
    }
  }
}
// One rounding to T, to the nearest (past fp16's range to infinity).
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> pack_row(const float (&x)[V]) {
  Raw<T, V> r;
  if constexpr (std::is_same_v<T, float> || V == 1) {
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_float<T>(x[i]);
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
      } else {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
  return r;
}

// Order of floats as whole numbers (-0 counts as 0).
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

// A launch that may begin while the one before it ends: its kernel waits (griddep_wait) before it touches memory.
template <typename... A>
cudaError_t launch_overlapped(void (*kernel)(A...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline int dtype_bytes(int dtype) { return dtype == RLDX_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == RLDX_BF16 || dtype == RLDX_F16 || dtype == RLDX_F32; }

}  // namespace rldx
