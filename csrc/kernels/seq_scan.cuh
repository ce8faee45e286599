// seq_scan.cuh — arguments and thread layout shared by the selective scan's
// forward (seq_scan.cu) and gradient (seq_scan_grad.cu).
#pragma once
#include <type_traits>

#include "seq_common.cuh"

namespace seqk {

// States are kept for the gradient before every kSave-th token.
constexpr int kSave = 8;

// Everything 8 bytes wide first, then 32-bit numbers: the binding packs it flat.
struct ScanArgs {
  const void *x, *dt, *z, *B, *C, *dout;       // z null: no gate
  const float *A, *D, *bias, *state, *dfinal;  // D, bias, state, dfinal may be null
  const uint8_t* reset;                        // [B, T] or null
  const int* lengths;                          // [B] or null
  void* out;                                   // forward
  float *final_state, *saved;                  // [B, D, N]; [B, ceil(T / kSave), D, N] (null: not kept)
  float *carry, *sumd;                         // [B, chunks, D, N], [B, chunks, D]: length split only
  uint8_t* cut;                                // [B, chunks]
  void *dx, *ddt, *dz, *dB, *dC;               // gradient: dense [B, T, D] and [B, T, G, N]
  float *part_bc;                              // [blocks of a group][B, T, G, 2 N]
  float *part_a, *part_v;                      // [B * chunks][D, N], [B * chunks][2][D] (dD, ddt_bias)
  float *dA, *dD, *dbias, *dstate;
  int64_t x_b, x_t, dt_b, dt_t, z_b, z_t, B_b, B_t, B_g, C_b, C_t, C_g, do_b, do_t, out_b, out_t, r_b;
  int batch, T, dim, N, G, softplus;
  int chunk, chunks;                           // tokens of a chunk (a multiple of 16), chunks of a row
  int mode_d, mode_n;                          // how rows of channels and of states are copied (copy_rows)
};
static_assert(sizeof(ScanArgs) == 48 * 8 + 10 * 4, "as the caller packs it");

// A warp's 32 lanes are 32 / LN channel rows of LN lanes; a lane holds 4 states of
// each of K channels, so 4 * LN >= N states of a channel sit in LN neighbouring lanes.
__device__ __forceinline__ float4 load_state4(const float* p, int n0, int N) {
  if ((N & 3) == 0) return n0 < N ? *reinterpret_cast<const float4*>(p + n0) : make_float4(0.f, 0.f, 0.f, 0.f);
  float4 v;
  v.x = n0 + 0 < N ? p[n0 + 0] : 0.0f;
  v.y = n0 + 1 < N ? p[n0 + 1] : 0.0f;
  v.z = n0 + 2 < N ? p[n0 + 2] : 0.0f;
  v.w = n0 + 3 < N ? p[n0 + 3] : 0.0f;
  return v;
}
__device__ __forceinline__ void store_state4(float* p, int n0, int N, const float (&h)[4]) {
  if ((N & 3) == 0) {
    if (n0 < N) *reinterpret_cast<float4*>(p + n0) = make_float4(h[0], h[1], h[2], h[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n0 + i < N) p[n0 + i] = h[i];
}

// Sums v[0..K) over the LN lanes of a channel row, halving what a lane carries with
// every exchange (K = 4, LN = 4: 3 exchanges instead of 8). Afterwards v[0] is the sum of
// channel reduced_channel<LN, K>(lane); with LN > K several lanes hold the same one.
template <int LN, int K> __device__ __forceinline__ void reduce_lanes(float (&v)[K], int lane) {
  int k = K;
#pragma unroll
  for (int off = LN / 2; off >= 1; off /= 2) {
    if (k > 1) {
      k /= 2;
#pragma unroll
      for (int i = 0; i < K / 2; ++i) {
        if (i < k) {
          const bool up = lane & off;
          const float give = up ? v[i] : v[i + k];
          const float keep = up ? v[i + k] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
        }
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
    }
  }
}
template <int LN, int K> __device__ __forceinline__ int reduced_channel(int lane) {
  int c = 0, k = K;
#pragma unroll
  for (int off = LN / 2; off >= 1; off /= 2)
    if (k > 1) {
      k /= 2;
      if (lane & off) c += k;
    }
  return c;
}
// the lanes that write sums, and how many each of them holds
template <int LN, int K> __device__ __forceinline__ bool reduced_writer(int lane) {
  return LN <= K || (lane & (LN / K - 1)) == 0;
}
template <int LN, int K> constexpr int kReduced = K > LN ? K / LN : 1;

// The states at the borders of a row's chunks, strung together for one (channel, state):
// slot c of `ends` (per apart) holds what chunk c adds to the state that passes through it,
// and gets the state that comes in. kDown: from the last chunk to the first (the adjoint).
// Two batches of loads are in flight ahead of the chain, which is what this waits for (one
// at a time, and the sums of delta behind their reset flags, took 22 us for 37 chunks).
template <bool kDown>
__device__ __forceinline__ float string_chunks(float v, float A2, float* ends, int64_t per, const float* sumd, int dim,
                                               const uint8_t* cut, int chunks) {
  constexpr int kAhead = 16;
  float e[2][kAhead], d[2][kAhead];
  bool z[2][kAhead];
  auto load = [&](int c0, float (&eb)[kAhead], float (&db)[kAhead], bool (&zb)[kAhead]) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (c0 + j < chunks) {
        const int c = kDown ? chunks - 1 - (c0 + j) : c0 + j;
        eb[j] = ends[c * per];
        db[j] = sumd[static_cast<int64_t>(c) * dim];
        zb[j] = cut[c] != 0;
      }
  };
  auto pass = [&](int c0, const float (&eb)[kAhead], const float (&db)[kAhead], const bool (&zb)[kAhead]) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (c0 + j < chunks) {
        const int c = kDown ? chunks - 1 - (c0 + j) : c0 + j;
        ends[c * per] = v;
        v = zb[j] ? eb[j] : fmaf(exp2_hw(A2 * db[j]), v, eb[j]);
      }
  };
  load(0, e[0], d[0], z[0]);
  for (int c = 0; c < chunks; c += 2 * kAhead) {
    load(c + kAhead, e[1], d[1], z[1]);
    pass(c, e[0], d[0], z[0]);
    load(c + 2 * kAhead, e[0], d[0], z[0]);
    pass(c + kAhead, e[1], d[1], z[1]);
  }
  return v;
}

// up to 4 channels of a row: one store where it is aligned and whole
template <typename T> __device__ __forceinline__ void store_quad(T* p, const float (&v)[4], int left, bool whole) {
  if (whole && left >= 4) {
    store_vec<T, 4>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = from_f<T>(v[j]);
  }
}

// Threads of a block. A block's channels lie in one group, so a group that fills at most half
// of the ordinary block's channels gets blocks of one warp (two for the widest states, whose
// rows of channels stay whole 16-byte pieces): 119 x 1047 tokens of 4 groups of 5 channels
// would leave 59 of 64 channel places idle.
template <int LN> constexpr int kSmallBlock = LN == 16 ? 64 : 32;
template <int LN> constexpr int kScanBlock = 128;
template <int LN> constexpr int kGradBlock = LN < 4 ? 128 : 256;
template <int LN> constexpr int scan_channels(int threads) { return threads / LN * (LN < 4 ? 2 : 4); }
template <int LN> constexpr int grad_channels(int threads) { return threads / LN * 2; }

// states -> lanes of a channel row; f gets the count as a compile-time constant
template <typename F> int by_lanes(int N, F f) {
  if (N < 1 || N > 64) return static_cast<int>(cudaErrorInvalidValue);
  if (N <= 4) return f(std::integral_constant<int, 1>{});
  if (N <= 8) return f(std::integral_constant<int, 2>{});
  if (N <= 16) return f(std::integral_constant<int, 4>{});
  if (N <= 32) return f(std::integral_constant<int, 8>{});
  return f(std::integral_constant<int, 16>{});
}

}  // namespace seqk
