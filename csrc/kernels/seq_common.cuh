// seq_common.cuh — element types, asynchronous row copies and the small math
// shared by the sequence operators (causal convolution, selective scan).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "surf_cuda.cuh"

namespace seqk {

using bf16 = __nv_bfloat16;

// dtype codes of the exported entry points
enum : int { kF32 = 0, kBf16 = 1 };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }

// elements of T in 16 bytes
template <typename T> constexpr int kVec16 = 16 / static_cast<int>(sizeof(T));

// V consecutive elements as floats; V * sizeof(T) is a power of two up to 16
// bytes and the address is a multiple of it (the caller's alignment rule).
template <typename T, int V> __device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f(*p);
  } else {
    constexpr int kBytes = V * static_cast<int>(sizeof(T));
    alignas(16) T raw[V];
    if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
    else *reinterpret_cast<uint32_t*>(raw) = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f(raw[i]);
  }
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f<T>(v[0]);
  } else {
    constexpr int kBytes = V * static_cast<int>(sizeof(T));
    alignas(16) T raw[V];
#pragma unroll
    for (int i = 0; i < V; ++i) raw[i] = from_f<T>(v[i]);
    if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(raw);
    else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(raw);
    else *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(raw);
  }
}

// ---- asynchronous 16-byte copies to shared memory ------------------------------
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// dst[r][0, cols) = src[r * stride + (0, cols)] for `rows` rows (dst row pitch:
// `pitch` elements), by all NT threads. kAsync: 16-byte pieces (cols, pitch and
// stride are multiples of a piece, both bases aligned), in flight on return;
// else element by element, done on return.
template <typename T, int NT, bool kAsync>
__device__ __forceinline__ void copy_rows(T* dst, int pitch, const T* src, int64_t stride, int rows, int cols) {
  if constexpr (kAsync) {
    constexpr int V = kVec16<T>;
    const int per = cols / V;
    for (int i = threadIdx.x; i < rows * per; i += NT) {
      const int r = i / per, c = (i - r * per) * V;
      cp_async16(dst + r * pitch + c, src + r * stride + c);
    }
  } else {
    for (int i = threadIdx.x; i < rows * cols; i += NT) {
      const int r = i / cols, c = i - r * cols;
      dst[r * pitch + c] = src[r * stride + c];
    }
  }
}

// ---- launches -----------------------------------------------------------------------
// Raises the kernel's dynamic shared-memory limit once per device.
template <auto Kern> int allow_smem(size_t bytes) {
  static bool done[64] = {};
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return static_cast<int>(e);
  if (dev < 64 && done[dev]) return 0;
  const cudaError_t e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess && dev < 64) done[dev] = true;
  return static_cast<int>(e);
}

// ---- math ---------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 2^x by the hardware's approximation (relative error 2^-22, denormals to 0)
__device__ __forceinline__ float exp2_hw(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.0f, 1.0f + exp2_hw(-kLog2e * v)); }

// log(1 + e^v)
__device__ __forceinline__ float softplus(float v) { return v > 20.0f ? v : log1pf(expf(v)); }

}  // namespace seqk
