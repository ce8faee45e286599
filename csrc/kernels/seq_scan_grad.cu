// seq_scan_grad.cu — gradient of the selective state space scan (sm_100a).
//
// With a = exp(delta A), g = dout * silu(z) and the adjoint state running backwards,
//   dh[t] = g[t] C[t] + a[t + 1] dh[t + 1]          (dfinal behind the last token)
//   dz = dout * y * silu'(z)          y = C . h + D x
//   dC[n] = sum_d g h[n]              dB[n] = sum_d dh[n] delta x
//   q = dh * a[t] * h[t - 1]          dA[d, n] = sum_t q delta
//   ddelta = sum_n q A + x sum_n dh B, through the softplus into ddt
//   dx = delta sum_n dh B + g D       dD = sum g x
//
// A block walks a stretch of channels backwards over tiles of kSave tokens. The
// forward kept the state before every tile, so the tile's states are run again from
// it into registers (kSave + 1 states of 4 x K per thread) and used at once by the
// backward sweep. Sums over the states go across the LN lanes of a channel; sums over
// the channels go across the warp, then the block's warps, then (dB, dC) over the
// blocks of a group: always in a fixed order, without atomics.
//
// Long rows are cut into chunks as in the forward: a first pass leaves each chunk's
// adjoint from nothing behind it, a small kernel strings the chunks together.
#include "seq_scan.cuh"

namespace {

using namespace seqk;

template <typename T, int LN> struct GradLayout {
  static constexpr int K = LN < 2 ? 1 : 2;
  static constexpr int NT = LN < 4 ? 128 : 256;
  static constexpr int CH = NT / LN * K;
  static constexpr int NP = 4 * LN;
  static constexpr int R = kSave;                         // tokens of a tile
  struct Smem {
    alignas(16) T x[2][R * CH], dt[2][R * CH], z[2][R * CH], dout[2][R * CH], B[2][R * NP], C[2][R * NP];
    alignas(16) float delta[R * CH], u[R * CH], g[R * CH], y[R * CH], ub[R * CH], qa[R * CH], Bf[R * NP], Cf[R * NP];
    alignas(16) float red[NT / 32][R][2 * NP];            // the warps' sums of dB and dC
    int cut[R];
  };
};

// Sums v[0..8) over the 32 / LN channel rows of a warp, halving what a lane carries with
// every exchange. Returns how many sums the lane holds (in v[0..)), the first of them
// being value `first`; lanes with `writer` false hold copies.
template <int LN> __device__ __forceinline__ void reduce_rows(float (&v)[8], int lane, int& first, bool& writer) {
  int k = 8;
  first = 0;
  writer = true;
#pragma unroll
  for (int off = 16; off >= LN; off /= 2) {
    const bool up = lane & off;
    if (k > 1) {
      k /= 2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < k) {
          const float give = up ? v[i] : v[i + k];
          const float keep = up ? v[i + k] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
        }
      }
      if (up) first += k;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
      if (up) writer = false;
    }
  }
}
// The backward sweep's decays, made again: as an ordinary expression the compiler would
// keep the forward run's (4 K values for each of the tile's tokens) and spill.
__device__ __forceinline__ float exp2_again(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int LN> constexpr int kRowSums = LN <= 4 ? 1 : (LN == 8 ? 2 : 4);

template <typename T, int LN, bool kAsync, bool kCarry>
__global__ void __launch_bounds__(GradLayout<T, LN>::NT, kCarry ? 1 : 512 / GradLayout<T, LN>::NT)
scan_grad_kernel(ScanArgs a, int blocks_per_group) {
  using L = GradLayout<T, LN>;
  constexpr int K = L::K, CH = L::CH, NP = L::NP, R = L::R, NT = L::NT;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  typename L::Smem& sm = *reinterpret_cast<typename L::Smem*>(smem_raw);
  const int blocks = blocks_per_group * a.G;
  const int b = blockIdx.x / blocks, blk = blockIdx.x - b * blocks;
  const int g = blk / blocks_per_group, per_group = a.dim / a.G, sub = blk - g * blocks_per_group;
  const int c0 = sub * CH;
  const int nch = min(CH, per_group - c0);
  const int d0 = g * per_group + c0;
  const int chunk = blockIdx.y;
  const int t_lo = chunk * a.chunk, t_hi = min(a.T, t_lo + a.chunk);
  const int len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  const int t_live = min(t_hi, len);
  const int64_t bchunk = static_cast<int64_t>(b) * a.chunks + chunk;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nl = lane & (LN - 1);
  const int ch = threadIdx.x / LN * K;
  const int n0 = nl * 4;

  float A2[K][4], dh[K][4], dA[K][4], sumd[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool on = ch + k < nch;
    const int64_t row = static_cast<int64_t>(d0 + ch + k) * a.N, bd = static_cast<int64_t>(a.dim) * a.N;
    const float4 v = on ? load_state4<LN>(a.A + row, n0, a.N) : make_float4(0.f, 0.f, 0.f, 0.f);
    A2[k][0] = v.x * kLog2e; A2[k][1] = v.y * kLog2e; A2[k][2] = v.z * kLog2e; A2[k][3] = v.w * kLog2e;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!kCarry && on) {
      if (a.chunks > 1) s = load_state4<LN>(a.carry + bchunk * bd + row, n0, a.N);
      else if (a.dfinal) s = load_state4<LN>(a.dfinal + b * bd + row, n0, a.N);
    }
    dh[k][0] = s.x; dh[k][1] = s.y; dh[k][2] = s.z; dh[k][3] = s.w;
    dA[k][0] = dA[k][1] = dA[k][2] = dA[k][3] = 0.0f;
    sumd[k] = 0.0f;
  }
  const T* gx = static_cast<const T*>(a.x) + b * a.x_b + d0;
  const T* gdt = static_cast<const T*>(a.dt) + b * a.dt_b + d0;
  const T* gz = a.z ? static_cast<const T*>(a.z) + b * a.z_b + d0 : nullptr;
  const T* gdo = static_cast<const T*>(a.dout) + b * a.do_b + d0;
  const T* gB = static_cast<const T*>(a.B) + b * a.B_b + g * a.B_g;
  const T* gC = static_cast<const T*>(a.C) + b * a.C_b + g * a.C_g;
  const int64_t dense = static_cast<int64_t>(b) * a.T * a.dim + d0;      // outputs are dense [B, T, D]
  T* gdx = static_cast<T*>(a.dx) + dense;
  T* gddt = static_cast<T*>(a.ddt) + dense;
  T* gdz = a.dz ? static_cast<T*>(a.dz) + dense : nullptr;
  const uint8_t* reset = a.reset ? a.reset + b * a.r_b : nullptr;
  const int64_t save_rows = (a.T + kSave - 1) / kSave;

  auto fetch = [&](int t, int buf) {
    const int rows = min(R, t_live - t);
    if (t >= t_lo && rows > 0) {
      if (!kCarry) {
        copy_rows<T, NT, kAsync>(sm.x[buf], CH, gx + t * a.x_t, a.x_t, rows, nch);
        copy_rows<T, NT, kAsync>(sm.B[buf], NP, gB + t * a.B_t, a.B_t, rows, a.N);
      }
      copy_rows<T, NT, kAsync>(sm.dt[buf], CH, gdt + t * a.dt_t, a.dt_t, rows, nch);
      copy_rows<T, NT, kAsync>(sm.dout[buf], CH, gdo + t * a.do_t, a.do_t, rows, nch);
      copy_rows<T, NT, kAsync>(sm.C[buf], NP, gC + t * a.C_t, a.C_t, rows, a.N);
      if (gz) copy_rows<T, NT, kAsync>(sm.z[buf], CH, gz + t * a.z_t, a.z_t, rows, nch);
    }
    cp_async_commit();
  };
  auto load_saved = [&](int t, float (&h0)[K][4]) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float* s = a.saved + ((b * save_rows + t / kSave) * a.dim + d0 + ch + k) * a.N;
      const float4 v = t >= t_lo && ch + k < nch ? load_state4<LN>(s, n0, a.N) : make_float4(0.f, 0.f, 0.f, 0.f);
      h0[k][0] = v.x; h0[k][1] = v.y; h0[k][2] = v.z; h0[k][3] = v.w;
    }
  };

  // the epilogue's channels of this thread, and their sums of g x and ddt
  constexpr int VE = kAsync ? 4 : 1;
  const int ec = static_cast<int>(threadIdx.x % (CH / VE)) * VE;
  float sD[VE], sV[VE];
#pragma unroll
  for (int j = 0; j < VE; ++j) sD[j] = sV[j] = 0.0f;

  bool any_cut = false;
  const int last = t_live > t_lo ? t_lo + (t_live - 1 - t_lo) / R * R : t_lo - R;
  float h0[K][4];
  if (!kCarry) load_saved(last, h0);
  fetch(last, 0);
  int buf = 0;
  for (int t0 = last; t0 >= t_lo; t0 -= R, buf ^= 1) {
    cp_async_wait<0>();
    __syncthreads();
    fetch(t0 - R, buf ^ 1);
    const int rows = min(R, t_live - t0);
    for (int i = threadIdx.x; i < R * CH; i += NT) {
      const int r = i / CH, c = i - r * CH;
      float dv = 0.0f, uv = 0.0f, gv = 0.0f;
      if (r < rows && c < nch) {
        dv = to_f(sm.dt[buf][i]) + (a.bias ? a.bias[d0 + c] : 0.0f);
        if (a.softplus) dv = softplus(dv);
        if (!kCarry) uv = dv * to_f(sm.x[buf][i]);
        gv = to_f(sm.dout[buf][i]);
        if (gz) {
          const float z = to_f(sm.z[buf][i]);
          gv *= z * sigmoid(z);
        }
      }
      sm.delta[i] = dv;
      if (!kCarry) sm.u[i] = uv;
      sm.g[i] = gv;
    }
    for (int i = threadIdx.x; i < R * NP; i += NT) {
      const int r = i / NP, n = i - r * NP;
      const bool in = r < rows && n < a.N;
      if (!kCarry) sm.Bf[i] = in ? to_f(sm.B[buf][i]) : 0.0f;
      sm.Cf[i] = in ? to_f(sm.C[buf][i]) : 0.0f;
    }
    if (threadIdx.x < R) sm.cut[threadIdx.x] = reset && threadIdx.x < rows && reset[t0 + threadIdx.x] ? 1 : 0;
    __syncthreads();
    if constexpr (kCarry) {
      for (int r = rows - 1; r >= 0; --r) {
        const bool cut = sm.cut[r];
        any_cut |= cut;
        const float4 Cv = *reinterpret_cast<const float4*>(sm.Cf + r * NP + n0);
        const float Ct[4] = {Cv.x, Cv.y, Cv.z, Cv.w};
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float dl = sm.delta[r * CH + ch + k], gv = sm.g[r * CH + ch + k];
          sumd[k] += dl;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = fmaf(gv, Ct[i], dh[k][i]);
            dh[k][i] = cut ? 0.0f : v * exp2_hw(dl * A2[k][i]);
          }
        }
      }
    } else {
      // the states of the tile: h[r] before token r, h[R] behind the last (tokens past the
      // row's end have delta = 0 and change nothing)
      float h[R + 1][K][4];
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) h[0][k][i] = h0[k][i];
      load_saved(t0 - R, h0);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 Bv = *reinterpret_cast<const float4*>(sm.Bf + r * NP + n0);
        const float Bt[4] = {Bv.x, Bv.y, Bv.z, Bv.w};
        const bool cut = sm.cut[r];
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float dl = sm.delta[r * CH + ch + k], u = sm.u[r * CH + ch + k];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            h[r + 1][k][i] = fmaf(exp2_hw(dl * A2[k][i]), cut ? 0.0f : h[r][k][i], u * Bt[i]);
        }
      }
#pragma unroll
      for (int r = R - 1; r >= 0; --r) {
        if (r < rows) {
          const float4 Bv = *reinterpret_cast<const float4*>(sm.Bf + r * NP + n0);
          const float4 Cv = *reinterpret_cast<const float4*>(sm.Cf + r * NP + n0);
          const float Bt[4] = {Bv.x, Bv.y, Bv.z, Bv.w}, Ct[4] = {Cv.x, Cv.y, Cv.z, Cv.w};
          float y[K], ub[K], qa[K], bc[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) bc[i] = 0.0f;
          const bool cut = sm.cut[r];
#pragma unroll
          for (int k = 0; k < K; ++k) {
            const float dl = sm.delta[r * CH + ch + k], u = sm.u[r * CH + ch + k], gv = sm.g[r * CH + ch + k];
            y[k] = ub[k] = qa[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float ad = exp2_again(dl * A2[k][i]);
              const float v = fmaf(gv, Ct[i], dh[k][i]);
              y[k] = fmaf(h[r + 1][k][i], Ct[i], y[k]);
              bc[4 + i] = fmaf(h[r + 1][k][i], gv, bc[4 + i]);
              bc[i] = fmaf(v, u, bc[i]);
              ub[k] = fmaf(v, Bt[i], ub[k]);
              const float va = v * ad;
              const float q = va * (cut ? 0.0f : h[r][k][i]);
              qa[k] = fmaf(q, A2[k][i], qa[k]);
              dA[k][i] = fmaf(q, dl, dA[k][i]);
              dh[k][i] = cut ? 0.0f : va;
            }
          }
          reduce_lanes<LN, K>(y, lane);
          reduce_lanes<LN, K>(ub, lane);
          reduce_lanes<LN, K>(qa, lane);
          if (reduced_writer<LN, K>(lane)) {
            const int at = r * CH + ch + reduced_channel<LN, K>(lane);
            sm.y[at] = y[0];
            sm.ub[at] = ub[0];
            sm.qa[at] = qa[0] * kLn2;
          }
          int first;
          bool writer;
          reduce_rows<LN>(bc, lane, first, writer);
          if (writer) {
#pragma unroll
            for (int i = 0; i < kRowSums<LN>; ++i) {
              const int q = first + i;
              sm.red[warp][r][(q < 4 ? 0 : NP) + n0 + (q & 3)] = bc[i];
            }
          }
        }
      }
      __syncthreads();
      for (int r = threadIdx.x / (CH / VE); r < rows; r += NT / (CH / VE)) {
        if (ec >= nch) break;
        float xv[VE], tv[VE], zv[VE], ov[VE], dx[VE], ddt[VE], dz[VE];
        const int at = r * CH + ec;
        load_vec<T, VE>(sm.x[buf] + at, xv);
        load_vec<T, VE>(sm.dt[buf] + at, tv);
        load_vec<T, VE>(sm.dout[buf] + at, ov);
        if (gz) load_vec<T, VE>(sm.z[buf] + at, zv);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float D = a.D ? a.D[d0 + ec + j] : 0.0f;
          const float gv = sm.g[at + j], ub = sm.ub[at + j];
          if (gz) {
            const float s = sigmoid(zv[j]);
            dz[j] = ov[j] * fmaf(D, xv[j], sm.y[at + j]) * s * fmaf(zv[j], 1.0f - s, 1.0f);
          }
          dx[j] = fmaf(ub, sm.delta[at + j], gv * D);
          const float dd = fmaf(ub, xv[j], sm.qa[at + j]);
          ddt[j] = a.softplus ? dd * sigmoid(tv[j] + (a.bias ? a.bias[d0 + ec + j] : 0.0f)) : dd;
          sD[j] = fmaf(gv, xv[j], sD[j]);
          sV[j] += ddt[j];
        }
        const int64_t o = static_cast<int64_t>(t0 + r) * a.dim + ec;
        store_vec<T, VE>(gdx + o, dx);
        store_vec<T, VE>(gddt + o, ddt);
        if (gz) store_vec<T, VE>(gdz + o, dz);
      }
      for (int i = threadIdx.x; i < rows * 2 * a.N; i += NT) {
        const int r = i / (2 * a.N), q = i - r * (2 * a.N);
        const int at = q < a.N ? q : NP + q - a.N;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) s += sm.red[w][r][at];
        a.part_bc[(((static_cast<int64_t>(sub) * a.batch + b) * a.T + t0 + r) * a.G + g) * (2 * a.N) + q] = s;
      }
    }
  }
  cp_async_wait<0>();
  if constexpr (kCarry) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (ch + k < nch) {
        store_state4(a.carry + (bchunk * a.dim + d0 + ch + k) * a.N, n0, a.N, dh[k]);
        if (nl == 0) a.sumd[bchunk * a.dim + d0 + ch + k] = sumd[k];
      }
    if (threadIdx.x == 0) a.cut[bchunk] = any_cut;               // the same from every block
  } else {
    for (int t = max(t_lo, t_live); t < t_hi; ++t) {             // tokens that are not there
      for (int c = threadIdx.x; c < nch; c += NT) {
        const int64_t o = static_cast<int64_t>(t) * a.dim + c;
        gdx[o] = gddt[o] = from_f<T>(0.0f);
        if (gz) gdz[o] = from_f<T>(0.0f);
      }
      for (int q = threadIdx.x; q < 2 * a.N; q += NT)
        a.part_bc[(((static_cast<int64_t>(sub) * a.batch + b) * a.T + t) * a.G + g) * (2 * a.N) + q] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (ch + k < nch) {
        const int64_t row = static_cast<int64_t>(d0 + ch + k) * a.N;
        if (a.dstate && a.chunks == 1) store_state4(a.dstate + static_cast<int64_t>(b) * a.dim * a.N + row, n0, a.N, dh[k]);
        store_state4(a.part_a + bchunk * a.dim * a.N + row, n0, a.N, dA[k]);
      }
    // the channels' sums over the threads that share them: within the warp, then in warp order
    constexpr int kSpan = CH / VE, kWide = kSpan < 32 ? 32 : kSpan, kRows = NT / kWide;
    static_assert(kRows <= R, "the sums of a block fit one array of the tile");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VE; ++j) {
#pragma unroll
      for (int off = 16; off >= kSpan; off /= 2) {
        sD[j] += __shfl_xor_sync(0xffffffffu, sD[j], off);
        sV[j] += __shfl_xor_sync(0xffffffffu, sV[j], off);
      }
      if (kSpan >= 32 || lane < kSpan) {
        sm.delta[(threadIdx.x / kWide) * CH + ec + j] = sD[j];
        sm.u[(threadIdx.x / kWide) * CH + ec + j] = sV[j];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < nch; c += NT) {
      float s = 0.0f, v = 0.0f;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        s += sm.delta[r * CH + c];
        v += sm.u[r * CH + c];
      }
      a.part_v[(bchunk * 2 + 0) * a.dim + d0 + c] = s;
      a.part_v[(bchunk * 2 + 1) * a.dim + d0 + c] = v;
    }
  }
}

// carry[b, c] <- the adjoint behind chunk c, dstate <- the one before the first token
__global__ void __launch_bounds__(256) grad_carry_kernel(ScanArgs a) {
  const int64_t per = static_cast<int64_t>(a.dim) * a.N;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (id >= per * a.batch) return;
  const int b = static_cast<int>(id / per);
  const int64_t dn = id - b * per;
  const int d = static_cast<int>(dn / a.N);
  const float A2 = a.A[dn] * kLog2e;
  float dh = a.dfinal ? a.dfinal[id] : 0.0f;
  float* carry = a.carry + static_cast<int64_t>(b) * a.chunks * per + dn;
  const float* sumd = a.sumd + static_cast<int64_t>(b) * a.chunks * a.dim + d;
  const uint8_t* cut = a.cut + static_cast<int64_t>(b) * a.chunks;
  constexpr int kAhead = 8;
  for (int c = a.chunks - 1; c >= 0; c -= kAhead) {
    float e[kAhead], p[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (c - j >= 0) {
        e[j] = carry[(c - j) * per];
        p[j] = cut[c - j] ? 0.0f : exp2_hw(A2 * sumd[static_cast<int64_t>(c - j) * a.dim]);
      }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (c - j >= 0) {
        carry[(c - j) * per] = dh;
        dh = cut[c - j] ? e[j] : fmaf(p[j], dh, e[j]);
      }
  }
  if (a.dstate) a.dstate[id] = dh;
}

// dB, dC: the sum over a group's channel blocks, in block order
template <typename T> __global__ void __launch_bounds__(256) finish_bc_kernel(ScanArgs a, int blocks) {
  const int64_t n = static_cast<int64_t>(a.batch) * a.T * a.G * 2 * a.N;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    float s = 0.0f;
    for (int k = 0; k < blocks; ++k) s += a.part_bc[k * n + i];
    const int64_t row = i / (2 * a.N);
    const int q = static_cast<int>(i - row * (2 * a.N));
    if (q < a.N) static_cast<T*>(a.dB)[row * a.N + q] = from_f<T>(s);
    else static_cast<T*>(a.dC)[row * a.N + q - a.N] = from_f<T>(s);
  }
}

// dA, dD, ddt_bias: the sum over rows and chunks, 8 row sums side by side, joined in order
__global__ void __launch_bounds__(256) finish_weights_kernel(ScanArgs a) {
  __shared__ float red[8][33];
  const int64_t na = static_cast<int64_t>(a.dim) * a.N, total = na + 2 * static_cast<int64_t>(a.dim);
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.chunks;
  float s = 0.0f;
  if (e < total) {
    const float* p = e < na ? a.part_a + e : a.part_v + (e - na);
    const int64_t step = e < na ? na : 2 * static_cast<int64_t>(a.dim);
    for (int64_t r = threadIdx.y; r < rows; r += 8) s += p[r * step];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && e < total) {
#pragma unroll
    for (int r = 1; r < 8; ++r) s += red[r][threadIdx.x];
    if (e < na) a.dA[e] = s;
    else if (e - na < a.dim) { if (a.dD) a.dD[e - na] = s; }
    else if (a.dbias) a.dbias[e - na - a.dim] = s;
  }
}

template <typename T, int LN, bool kAsync> int launch_grad(const ScanArgs& a, cudaStream_t s) {
  using L = GradLayout<T, LN>;
  const int bpg = static_cast<int>(surfk::ceil_div(a.dim / a.G, L::CH));
  const int64_t gx = static_cast<int64_t>(bpg) * a.G * a.batch;
  if (gx > 0x7fffffffLL || a.chunks > 65535) return static_cast<int>(cudaErrorInvalidValue);
  constexpr size_t smem = sizeof(typename L::Smem);
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(a.chunks));
  if (a.chunks > 1) {
    if (const int rc = allow_smem<scan_grad_kernel<T, LN, kAsync, true>>(smem)) return rc;
    scan_grad_kernel<T, LN, kAsync, true><<<grid, L::NT, smem, s>>>(a, bpg);
    grad_carry_kernel<<<static_cast<unsigned>(surfk::ceil_div(static_cast<int64_t>(a.batch) * a.dim * a.N, 256)), 256, 0, s>>>(a);
  }
  if (const int rc = allow_smem<scan_grad_kernel<T, LN, kAsync, false>>(smem)) return rc;
  scan_grad_kernel<T, LN, kAsync, false><<<grid, L::NT, smem, s>>>(a, bpg);
  const int64_t n = static_cast<int64_t>(a.batch) * a.T * a.G * 2 * a.N;
  const int64_t blocks = surfk::ceil_div(n, 256);
  finish_bc_kernel<T><<<static_cast<unsigned>(blocks < 148 * 16 ? (blocks > 0 ? blocks : 1) : 148 * 16), 256, 0, s>>>(a, bpg);
  finish_weights_kernel<<<static_cast<unsigned>(surfk::ceil_div(static_cast<int64_t>(a.dim) * (a.N + 2), 32)), dim3(32, 8), 0, s>>>(a);
  SURF_RETURN_LAUNCH();
}

}  // namespace

SURF_EXPORT int surf_seq_scan_grad(const void* args, int dtype, int aligned, void* stream) {
  const ScanArgs a = *static_cast<const ScanArgs*>(args);
  if (a.batch <= 0 || a.dim <= 0) return static_cast<int>(cudaErrorInvalidValue);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_lanes(a.N, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    if (dtype == kBf16) return aligned ? launch_grad<bf16, LN, true>(a, s) : launch_grad<bf16, LN, false>(a, s);
    return aligned ? launch_grad<float, LN, true>(a, s) : launch_grad<float, LN, false>(a, s);
  });
}

// channel blocks of a group (the caller sizes part_bc with it)
SURF_EXPORT int surf_seq_scan_grad_blocks(int per_group, int N) {
  return by_lanes(N, [&](auto ln) {
    return static_cast<int>(surfk::ceil_div(per_group, GradLayout<float, decltype(ln)::value>::CH));
  });
}
