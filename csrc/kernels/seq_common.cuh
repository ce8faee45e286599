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
  } else if constexpr (sizeof(T) == 4) {
    if constexpr (V == 4) {
      const float4 q = *reinterpret_cast<const float4*>(p);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      const float2 q = *reinterpret_cast<const float2*>(p);
      v[0] = q.x; v[1] = q.y;
    }
  } else {
    uint32_t w[V / 2];
    if constexpr (V == 8) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (V == 4) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = surfk::pack_bf16x2(v[2 * i], v[2 * i + 1]);
    if constexpr (V == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
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

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}

// How rows may be copied: pieces of 16 or 4 bytes (bases, strides and the row's length
// are multiples of it), else element by element.
enum : int { kPlain = 0, kPieces4 = 4, kPieces16 = 16 };

// dst[r][0, cols) = src[r * stride + (0, cols)] for `rows` rows of pitch P, by all NT
// threads; in pieces it is still in flight on return.
template <typename T, int NT, int P>
__device__ __forceinline__ void copy_rows(T* dst, const T* src, int64_t stride, int rows, int cols, int mode) {
  if (mode == kPieces16) {
    constexpr int V = kVec16<T>, W = (P + V - 1) / V;
    for (int i = threadIdx.x; i < rows * W; i += NT) {
      const int r = i / W, c = (i - r * W) * V;
      if (c < cols) cp_async16(dst + r * P + c, src + r * stride + c);
    }
  } else if (mode == kPieces4) {
    constexpr int V = 4 / static_cast<int>(sizeof(T)), W = P / V;
    for (int i = threadIdx.x; i < rows * W; i += NT) {
      const int r = i / W, c = (i - r * W) * V;
      if (c < cols) cp_async4(dst + r * P + c, src + r * stride + c);
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * P; i += NT) {
      const int r = i / P, c = i - r * P;
      if (c < cols) dst[i] = src[r * stride + c];
    }
  }
}

// One thread's share of a tile's rows of channels in 16-byte pieces: piece column `c`, rows
// r0, r0 + kStep, ... of R. The pointer moves with the tiles, so a tile costs no index
// arithmetic.
template <typename T, int NT, int CH, int R> struct RowPieces {
  static constexpr int kPer = CH / kVec16<T>, kStep = NT / kPer;         // pieces of a row, rows between two of a thread's
  static constexpr int kCount = (R + kStep - 1) / kStep;
  static __device__ __forceinline__ int column() { return static_cast<int>(threadIdx.x) % kPer * kVec16<T>; }
  static __device__ __forceinline__ int row() { return static_cast<int>(threadIdx.x) / kPer; }
  // dst: the tile; src: this thread's first piece; rows: how many are there
  static __device__ __forceinline__ void copy(T* dst, const T* src, int64_t stride, int rows) {
    T* d = dst + row() * CH + column();
#pragma unroll
    for (int k = 0; k < kCount; ++k)
      if (row() + k * kStep < rows) cp_async16(d + k * kStep * CH, src + k * kStep * stride);
  }
};

// The same for the two short rows of a token (B and C, NP elements each): one piece for each
// of the first 2 R NP / V threads, B's first.
template <typename T, int NT, int NP, int R> struct TwinPieces {
  static constexpr int kPer = NP >= kVec16<T> ? NP / kVec16<T> : 1, kEach = R * kPer;
  static constexpr bool kFits = NP % kVec16<T> == 0 && 2 * kEach <= NT;
  static __device__ __forceinline__ int which() { return static_cast<int>(threadIdx.x) / kEach; }        // 0: B, 1: C
  static __device__ __forceinline__ int row() { return static_cast<int>(threadIdx.x) % kEach / kPer; }
  static __device__ __forceinline__ int column() { return static_cast<int>(threadIdx.x) % kPer * kVec16<T>; }
};

// ---- launches -----------------------------------------------------------------------
// Raises the kernel's dynamic shared-memory limit (and, if wide, its cluster limit to 16
// blocks) once per device.
template <auto Kern, bool kWide = false> int allow_smem(size_t bytes) {
  static bool done[64] = {};
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return static_cast<int>(e);
  if (dev < 64 && done[dev]) return 0;
  cudaError_t e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (kWide && e == cudaSuccess) e = cudaFuncSetAttribute(Kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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
// The hardware's 2^x is 2e-8 too small on average between 2^-1 and 1, where the decays of
// long memories lie: over the hundreds of factors of a state's life that was the largest
// error of the scan (1.3e-6 of the final states' norm, 7e-7 with an exact exponential). An
// argument 3e-8 larger takes it out (mean -4e-10 for x in [-0.02, -0.002], 2e-9 in
// [-0.1, -0.02]) at no cost: the multiplication that makes it becomes a multiply-add.
constexpr float kExp2Shift = 3e-8f;
// The rate of a state, A log2(e). -inf (a state that forgets at once) becomes the largest finite
// rate: with a step of zero, which a dt of -inf is and every token that fills up a row's last
// tile, it would be 0 * -inf, not a number. Steps above 4e-37 forget all the same.
__device__ __forceinline__ float rate_of(float A) {
  const float r = A * kLog2e;
  return r < -3.4028235e38f ? -3.4028235e38f : r;
}
// exp(delta * A) with A2 = rate_of(A); exactly 1 for a step of zero
__device__ __forceinline__ float decay(float delta, float A2) { return exp2_hw(fmaf(delta, A2, kExp2Shift)); }
// 1 / x by the hardware's approximation (relative error 2^-23; 0 for infinity). The divisors
// here lie between 1 and infinity: a division, even the approximate one, guards a range that
// they never reach with four instructions more.
__device__ __forceinline__ float rcp_hw(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid(float v) { return rcp_hw(1.0f + exp2_hw(-kLog2e * v)); }

// log(1 + e^v) = max(v, 0) + log(1 + e^-|v|); with s = e / (2 + e) <= 1/3 the logarithm is
// 2 atanh(s) = 2 s g(s^2), g fitted on [0, 1/9] to 4e-9: as exact for small e as for e = 1.
__device__ __forceinline__ float softplus(float v) {
  const float e = exp2_hw(-kLog2e * fabsf(v));
  const float s = e * rcp_hw(2.0f + e), q = s * s;
  float g = fmaf(q, 0.14089155197143555f, 0.13980303704738617f);
  g = fmaf(g, q, 0.20012454688549042f);
  g = fmaf(g, q, 0.3333315849304199f);
  g = fmaf(g, q, 1.0f);
  return fmaf(2.0f * s, g, fmaxf(v, 0.0f));
}

// dt -> delta for 4 channels
__device__ __forceinline__ void step_of(float (&v)[4], const float (&bias)[4], int through_softplus) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] += bias[j];
  if (through_softplus) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = softplus(v[j]);
  }
}

// ---- pairs of floats in one 64-bit register: one instruction for both ---------------
struct f2 { unsigned long long v; };
__device__ __forceinline__ f2 pack2(float lo, float hi) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
// four floats of shared memory as two pairs
__device__ __forceinline__ void load_pairs(const float* p, f2& a, f2& b) {
  const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(p);
  a.v = q.x;
  b.v = q.y;
}
__device__ __forceinline__ f2 decay_arg(f2 delta, f2 A2) { return fma2(delta, A2, pack2(kExp2Shift, kExp2Shift)); }
__device__ __forceinline__ f2 decay2(f2 delta, f2 A2) {
  float lo, hi;
  unpack2(decay_arg(delta, A2), lo, hi);
  return pack2(exp2_hw(lo), exp2_hw(hi));
}
}  // namespace seqk
