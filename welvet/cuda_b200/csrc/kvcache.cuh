// kvcache.cuh -- conversions of the key-value cache's storage types, and small helpers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kvcache.hpp"

#include <cstdint>
#include <type_traits>

namespace wb {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__nv_fp8_e4m3 x) { return static_cast<float>(x); }

// Round to nearest even; E4M3 saturates at +-448 (NaN stays NaN). E4M3 pages hold the OCP format
// with its subnormals, unlike the weight codec, which follows the reference's flush to zero.
template <typename T>
__device__ __forceinline__ T to_stored(float x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(x);
  else return __nv_fp8_e4m3(x);
}

// What a page's values are divided by. The reciprocal of a power of two is exact, and one product
// gives the quotient; other scales divide (kDiv), so that a value between two codes goes to the side
// that x / scale rounds to.
template <bool kDiv>
__device__ __forceinline__ float over(float x, float scale, float inv) {
  return kDiv ? __fdiv_rn(x, scale) : x * inv;
}

// Four values over the scale to consecutive elements (aligned to four elements).
template <typename T, bool kDiv>
__device__ __forceinline__ void store4(T* dst, const float (&x)[4], float scale, float inv) {
  auto f = [&](int i) { return over<kDiv>(x[i], scale, inv); };
  if constexpr (std::is_same_v<T, float>) {
    *reinterpret_cast<float4*>(dst) = make_float4(f(0), f(1), f(2), f(3));
  } else if constexpr (sizeof(T) == 2) {
    union { T t[4]; uint2 u; } o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.t[i] = to_stored<T>(f(i));
    *reinterpret_cast<uint2*>(dst) = o.u;
  } else {
    const __nv_fp8x4_e4m3 o(make_float4(f(0), f(1), f(2), f(3)));
    *reinterpret_cast<__nv_fp8x4_e4m3*>(dst) = o;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The MHA cell's slope of head h (src/cuda/kernels.cu:520-528): 2^(-8 (h + 1) / heads).
__device__ __forceinline__ float alibi_slope(int h, int heads) {
  return exp2f(-8.0f * static_cast<float>(h + 1) / static_cast<float>(heads));
}

// f(T*) with the C++ type of the pages.
template <typename F>
Status by_type(KvType t, F&& f) {
  switch (t) {
  case KvType::F32: return f(static_cast<float*>(nullptr));
  case KvType::F16: return f(static_cast<__half*>(nullptr));
  case KvType::BF16: return f(static_cast<__nv_bfloat16*>(nullptr));
  case KvType::E4M3: return f(static_cast<__nv_fp8_e4m3*>(nullptr));
  }
  return Status::Internal("kv: type");
}

// A launch that may start while the kernel before it still runs (it waits for its results itself).
template <typename K, typename P>
Status launch_after(K* kernel, dim3 grid, int threads, int smem, cudaStream_t st, const P& p, int cluster = 0) {
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, p), "kv launch");
}

} // namespace wb
