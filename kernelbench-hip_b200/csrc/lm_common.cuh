// lm_common.cuh — helpers shared by the language-model operators: element
// types, pairs of fp32 values, and launches that begin while the one before ends.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kb_common.cuh"

namespace kb {
namespace lm {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// round to nearest even; the only rounding an output sees
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two fp32 values in a 64-bit register, and operations on both at once.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

inline int dtype_size(int dtype) { return dtype == KB_F32 ? 4 : (dtype == KB_F16 || dtype == KB_BF16) ? 2 : 0; }

// Calls f with a null pointer of the element type that `dtype` names.
template <typename F>
int with_dtype(int dtype, F f) {
  switch (dtype) {
    case KB_F32: return f(static_cast<float*>(nullptr));
    case KB_F16: return f(static_cast<__half*>(nullptr));
    default: return f(static_cast<__nv_bfloat16*>(nullptr));
  }
}

// Programmatic dependent launch, for every launch of these operators: it may
// begin once all CTAs of the launch before it have passed allow_next() (or
// ended), and nothing of that launch, nor of those before it, is read or
// written before wait_for_previous() returns.  A decoding step is a chain of
// launches of a few microseconds each, and their starts are a good part of it.
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), dim3 blocks, unsigned threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.gridDim = blocks, config.blockDim = dim3(threads), config.dynamicSmemBytes = smem, config.stream = stream;
  config.attrs = &attr, config.numAttrs = 1;
  KB_CUDA(cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...));
  return KB_OK;
}

}  // namespace lm
}  // namespace kb
