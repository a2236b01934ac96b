// Shared pieces of the attention kernels: 16-bit element types (1 bf16, 2 f16,
// the codes of v1x.h) and their conversions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "common.cuh"

namespace v1x {
namespace attn {

// Weights that go into a product in f16, whose range ends at 2^16 above and, with steps
// of 2^-24, at 2^-25 below: taken against a reference 2^lift below the running maximum
// they use that range up, and many small ones beside a large one are not lost (without
// it 65536 tokens 17.5 below the largest score lost their 1.6e-3 of the sum).  `lazy`:
// how far, in powers of two, weights may outgrow their reference.
template <typename T>
constexpr float lift(float lazy) {
  return std::is_same<T, __half>::value ? 15.0f - lazy : 0.0f;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
__device__ __forceinline__ float2 to_float2(uint32_t two);
template <>
__device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t two) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&two));
}
template <>
__device__ __forceinline__ float2 to_float2<__half>(uint32_t two) {
  return __half22float2(*reinterpret_cast<__half2*>(&two));
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- two floats in one 64-bit register, one instruction for both ----------------
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 two(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 both(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// two floats rounded to nearest even, the first in the low half
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// The driver's encoder of TMA tensor maps; null where it has none.
inline PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// A kernel that joins what the one launched before it on the stream leaves: its launch
// is prepared while that one drains, and its first statement, wait_for_previous, holds
// it until that one is complete.
template <typename... KArgs, typename... Args>
inline void launch_join(void (*kernel)(KArgs...), dim3 grid, dim3 block, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A scale that is finite, also times log2 e (NaN is not).
inline bool scale_in_range(float scale) { return scale > -0x1p127f && scale < 0x1p127f; }

__host__ __device__ inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace attn
}  // namespace v1x
