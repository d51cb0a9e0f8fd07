// What the kernels behind a forest's leaves share: element types, to fp32 and, rounded to nearest, back; the
// order of a call's kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <type_traits>

namespace tb {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Adds two 16-bit elements to two fp32 sums: widened (exactly) and added by one instruction each.
template <class T> __device__ __forceinline__ void add_halves(unsigned long long &sums, uint32_t halves) {
  if constexpr (std::is_same<T, __half>::value)
    asm("{\n .reg .b16 c, d;\n .reg .f32 a, b;\n mov.b64 {a, b}, %0;\n mov.b32 {c, d}, %1;\n add.rn.f32.f16 a, c, a;\n add.rn.f32.f16 b, d, b;\n"
        " mov.b64 %0, {a, b};\n}" : "+l"(sums) : "r"(halves));
  else
    asm("{\n .reg .b16 c, d;\n .reg .f32 a, b;\n mov.b64 {a, b}, %0;\n mov.b32 {c, d}, %1;\n add.rn.f32.bf16 a, c, a;\n add.rn.f32.bf16 b, d, b;\n"
        " mov.b64 %0, {a, b};\n}" : "+l"(sums) : "r"(halves));
}

// Kernels of one call follow one another closely: each is launched while the one before still runs, prepares itself
// and waits here until that one's results are there (and lets its own follower come).  What is read afterwards is read
// by plain loads: __ldg is for data that nothing writes while the grid is resident.
__device__ __forceinline__ void after_previous_kernel() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Loads of such results.  (As statements of their own, which stay behind the wait but may be moved past shuffles and
// past stores to shared memory, where those of plain expressions may not.)
__device__ __forceinline__ uint4 load_result(const uint4 *p) {
  uint4 v;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load_result(const uint2 *p) {
  uint2 v;
  asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t load_result(const uint32_t *p) {
  uint32_t v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint16_t load_result(const uint16_t *p) {
  uint16_t v;
  asm volatile("ld.global.b16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}

} // namespace tb
