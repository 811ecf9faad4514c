// Device helpers shared by the token-stream operators: element types by tag,
// conversions to and from f32, and the 8-bit codes.
#pragma once

#include <stdexcept>
#include <string>
#include <type_traits>

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "tessera_b200_ops.h"
#include "token_ops.h"

namespace tcb {

using f16 = __half;
using e4m3 = __nv_fp8_e4m3;

inline void need(bool ok, const char *what) {
    if (!ok) throw std::runtime_error(what);
}
// A pointer (or NULL) that its elements can be read through.
inline bool on(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline int type_bytes(int type) {
    return type == TCB_I8 || type == TCB_E4M3 ? 1 : type == TCB_BF16 || type == TCB_F16 ? 2 : type == TCB_I64 ? 8 : 4;
}
inline void check_token_launch(const char *what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(f16 v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(int8_t v) { return (float)v; }
__device__ __forceinline__ float to_f32(e4m3 v) { return float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (std::is_same_v<T, bf16>) return __float2bfloat16_rn(v);
    else if constexpr (std::is_same_v<T, f16>) return __float2half_rn(v);
    else return v;
}

// Asynchronous copies of 16 bytes into shared memory; a thread sees its own after the wait.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Largest magnitude of an 8-bit code.
template <class T>
__host__ __device__ constexpr float code_top() {
    return std::is_same_v<T, int8_t> ? 127.f : 448.f;
}

// The larger of two magnitudes, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

}  // namespace tcb
