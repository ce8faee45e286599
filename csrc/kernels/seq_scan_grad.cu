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
//
// Measured on a B200, 16 states, back to back: 256 x 128 x 512 bf16 369 us, f32 397 us, 2 x 4096
// x 1024 in 37 chunks 257 and 270 us (launched one by one, bf16: first pass 65, stringing 10,
// sweeps 187, last sums 7 us). The two sweeps alone take
// 404 cycles for 512 states (exponentials 256, multiply-adds about 260 on their own units),
// 206 us for 256 x 128 x 512; the other half is the work on every (token, channel) around
// them (80 of 240 M warp instructions) and the waits between the two at 16 warps on an SM.
#include "seq_scan.cuh"

namespace {

using namespace seqk;

template <typename T, int LN, int kThreads> struct GradLayout {
  static constexpr int NT = kThreads;
  static constexpr int CH = grad_channels<LN>(NT);        // two channels a thread, 4 states of each in two f32x2 pairs
  static constexpr int NP = 4 * LN;
  static constexpr int R = kSave;                         // tokens of a tile
  struct Smem {
    alignas(16) T x[2][R * CH], dt[2][R * CH], z[2][R * CH], dout[2][R * CH], B[2][R * NP], C[2][R * NP];
    alignas(16) float delta[R * CH], u[R * CH], g[R * CH], y[R * CH], ub[R * CH], qa[R * CH];
    alignas(16) float dgate[R * CH], dstep[R * CH];       // dout silu'(z), d delta / d dt
    alignas(16) float Bf[R * 4 * NP], Cf[R * 4 * NP];     // 32-bit, in the four orders of the lanes
    alignas(16) float red[NT / 32][R][2 * NP];            // the warps' sums of dB and dC
    alignas(16) float bias[CH], skip[CH];
    alignas(16) float hs[2][CH * NP];                     // the states kept before a tile, as in memory
  };
};

// The order of a lane's 4 states. Sums over the 32 / LN channel rows of a warp halve what a
// lane carries with every exchange; so that no lane has to choose which half it gives, lanes
// hold their states in different orders: slot s is state s ^ order_of(lane).
template <int LN> __device__ __forceinline__ int order_of(int lane) {
  return (LN <= 16 && (lane & LN) ? 2 : 0) | (LN <= 8 && (lane & (2 * LN)) ? 1 : 0);
}
// where B and C lie in that order: neighbouring channel rows read neighbouring copies
__device__ __forceinline__ int copy_of(int order) { return (order >> 1) | (order & 1) << 1; }
__device__ __forceinline__ float4 in_order(float4 v, int order) {
  if (order & 2) v = make_float4(v.z, v.w, v.x, v.y);
  if (order & 1) v = make_float4(v.y, v.x, v.w, v.z);
  return v;
}

// dB and dC of one token: b and c summed over the warp's channel rows into red[0, NP) and
// red[NP, 2 NP).
template <int LN> __device__ __forceinline__ void reduce_rows(float (&b)[4], float (&c)[4], int lane, int n, float* red) {
  constexpr int NP = 4 * LN;
  constexpr unsigned kFull = 0xffffffffu;
  b[0] += __shfl_xor_sync(kFull, b[2], LN);
  b[1] += __shfl_xor_sync(kFull, b[3], LN);
  c[0] += __shfl_xor_sync(kFull, c[2], LN);
  c[1] += __shfl_xor_sync(kFull, c[3], LN);
  if constexpr (LN <= 8) {
    b[0] += __shfl_xor_sync(kFull, b[1], 2 * LN);
    c[0] += __shfl_xor_sync(kFull, c[1], 2 * LN);
  } else {
    red[n ^ 1] = b[1];
    red[NP + (n ^ 1)] = c[1];
  }
  if constexpr (LN <= 4) {
    const bool up = lane & (4 * LN);
    float keep = up ? c[0] : b[0];
    keep += __shfl_xor_sync(kFull, up ? b[0] : c[0], 4 * LN);
#pragma unroll
    for (int off = 8 * LN; off <= 16; off *= 2) keep += __shfl_xor_sync(kFull, keep, off);
    if (LN == 4 || lane < 8 * LN) red[(up ? NP : 0) + n] = keep;
  } else {
    red[n] = b[0];
    red[NP + n] = c[0];
  }
}

// The backward sweep's decays, made again: as an ordinary expression the compiler would
// keep the forward run's (8 values for each of the tile's tokens), for which there are no
// registers: the nine states of a thread's two channels take 72 of its 128, and every instance
// spills 128 to 248 bytes of what lies around the sweeps as it is.
__device__ __forceinline__ f2 decay2_again(f2 delta, f2 A2) {
  float lo, hi;
  unpack2(decay_arg(delta, A2), lo, hi);
  asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(lo));
  asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(hi));
  return pack2(lo, hi);
}

__device__ __forceinline__ float sum_of(f2 v) {
  float lo, hi;
  unpack2(v, lo, hi);
  return lo + hi;
}

// Per state and token the two sweeps cost 13 multiply-adds (in pairs of states) and two
// exponentials, the sums across lanes 13 exchanges for 8 states. A tile's resets choose one of
// two copies of the sweeps: selecting in every tile costs 1.5%.
template <typename T, int LN, int NT, bool kCarry>
__global__ void __launch_bounds__(NT, (kCarry ? 768 : 512) / NT) scan_grad_kernel(ScanArgs a, int blocks_per_group) {
  using L = GradLayout<T, LN, NT>;
  constexpr int CH = L::CH, NP = L::NP, R = L::R;
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
  const int ch = threadIdx.x / LN * 2;
  const int n0 = nl * 4;

  const int order = order_of<LN>(lane);
  // 4 states of the two channels, from memory into pairs and back
  auto load_h = [&](const float* src, f2 (&v)[2][2], auto rate) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
      if (src && ch + k < nch) q = in_order(load_state4(src + static_cast<int64_t>(d0 + ch + k) * a.N, n0, a.N), order);
      if constexpr (decltype(rate)::value) q = make_float4(rate_of(q.x), rate_of(q.y), rate_of(q.z), rate_of(q.w));
      v[k][0] = pack2(q.x, q.y);
      v[k][1] = pack2(q.z, q.w);
    }
  };
  auto store_h = [&](float* dst, const f2 (&v)[2][2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float4 q;
      unpack2(v[k][0], q.x, q.y);
      unpack2(v[k][1], q.z, q.w);
      q = in_order(q, order);
      const float f[4] = {q.x, q.y, q.z, q.w};
      if (ch + k < nch) store_state4(dst + static_cast<int64_t>(d0 + ch + k) * a.N, n0, a.N, f);
    }
  };
  const int64_t per_row = static_cast<int64_t>(a.dim) * a.N;

  f2 A2[2][2], dh[2][2], dA[2][2];
  float sumd[2] = {0.0f, 0.0f};
  load_h(a.A, A2, std::true_type{});
  load_h(kCarry ? nullptr : a.chunks > 1 ? a.carry + bchunk * per_row : a.dfinal ? a.dfinal + b * per_row : nullptr, dh, std::false_type{});
  dA[0][0].v = dA[0][1].v = dA[1][0].v = dA[1][1].v = 0;

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
  const float* saved = kCarry ? nullptr : a.saved + static_cast<int64_t>(b) * ((a.T + kSave - 1) / kSave) * per_row;

  // rows of channels in 16-byte pieces: this thread's first piece of the next tile
  using Pieces = RowPieces<T, NT, CH, R>;
  const int last = t_live > t_lo ? t_lo + (t_live - 1 - t_lo) / R * R : t_lo - R;
  const bool pieces = a.mode_d == kPieces16, mine = Pieces::column() < nch;
  const T *px = gx + (last + Pieces::row()) * a.x_t + Pieces::column(), *pdt = gdt + (last + Pieces::row()) * a.dt_t + Pieces::column();
  const T* pdo = gdo + (last + Pieces::row()) * a.do_t + Pieces::column();
  const T* pz = gz ? gz + (last + Pieces::row()) * a.z_t + Pieces::column() : nullptr;
  const float* psaved = kCarry ? nullptr : saved + last / kSave * per_row + static_cast<int64_t>(d0) * a.N;
  const bool all_states = nch == CH && a.N == NP;
  using Twin = TwinPieces<T, NT, NP, R>;
  const bool twin = Twin::kFits && a.mode_n == kPieces16 && a.N == NP;
  const bool my_twin = kCarry ? Twin::which() == 1 : Twin::which() < 2;
  const int64_t twin_t = Twin::which() == 0 ? a.B_t : a.C_t;
  const T* ptwin = (Twin::which() == 0 ? gB : gC) + (last + Twin::row()) * twin_t + Twin::column();
  auto fetch = [&](int t, int buf) {
    const int rows = min(R, t_live - t);
    if (t >= t_lo && rows > 0) {
      if (pieces) {
        if (mine) {
          if (!kCarry) Pieces::copy(sm.x[buf], px, a.x_t, rows);
          Pieces::copy(sm.dt[buf], pdt, a.dt_t, rows);
          Pieces::copy(sm.dout[buf], pdo, a.do_t, rows);
          if (gz) Pieces::copy(sm.z[buf], pz, a.z_t, rows);
        }
        px -= R * a.x_t;
        pdt -= R * a.dt_t;
        pdo -= R * a.do_t;
        if (gz) pz -= R * a.z_t;
      } else {
#pragma unroll 1
        for (int i = kCarry ? 1 : 0; i < (gz ? 4 : 3); ++i) {
          const int64_t stride = i == 0 ? a.x_t : i == 1 ? a.dt_t : i == 2 ? a.do_t : a.z_t;
          copy_rows<T, NT, CH>(i == 0 ? sm.x[buf] : i == 1 ? sm.dt[buf] : i == 2 ? sm.dout[buf] : sm.z[buf],
                               (i == 0 ? gx : i == 1 ? gdt : i == 2 ? gdo : gz) + t * stride, stride, rows, nch, a.mode_d);
        }
      }
      if (twin) {
        if (my_twin && Twin::row() < rows)
          cp_async16((Twin::which() == 0 ? sm.B[buf] : sm.C[buf]) + Twin::row() * NP + Twin::column(), ptwin);
        ptwin -= R * twin_t;
      } else {
#pragma unroll 1
        for (int i = kCarry ? 1 : 0; i < 2; ++i) {
          const int64_t stride = i == 0 ? a.B_t : a.C_t;
          copy_rows<T, NT, NP>(i == 0 ? sm.B[buf] : sm.C[buf], (i == 0 ? gB : gC) + t * stride, stride, rows, a.N, a.mode_n);
        }
      }
      if (!kCarry) {
        if (all_states) {
          constexpr int kStates = CH * NP / (4 * NT);
#pragma unroll
          for (int k = 0; k < kStates; ++k) cp_async16(sm.hs[buf] + (threadIdx.x + k * NT) * 4, psaved + (threadIdx.x + k * NT) * 4);
        } else if ((a.N & 3) == 0) {
          for (int i = threadIdx.x * 4; i < nch * a.N; i += NT * 4) cp_async16(sm.hs[buf] + i, psaved + i);
        } else {
          for (int i = threadIdx.x; i < nch * a.N; i += NT) cp_async4(sm.hs[buf] + i, psaved + i);
        }
        psaved -= per_row;
      }
    }
    cp_async_commit();
  };

  // before and behind the sweeps a thread works on 4 channels of every kStep-th token
  constexpr int kQuads = CH / 4, kStep = NT / kQuads;
  const int ec = threadIdx.x % kQuads * 4, er = threadIdx.x / kQuads;
  float sD[4] = {0.f, 0.f, 0.f, 0.f}, sV[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c = threadIdx.x; c < CH; c += NT) {
    sm.bias[c] = a.bias && c < nch ? a.bias[d0 + c] : 0.0f;
    sm.skip[c] = a.D && c < nch ? a.D[d0 + c] : 0.0f;
  }

  // dB and dC of the tile: a thread sums one state of every kBcStep-th token over the warps
  constexpr int kBcStep = NT / (2 * NP) > 0 ? NT / (2 * NP) : 1;
  const int bq = threadIdx.x % (2 * NP), br = threadIdx.x / (2 * NP), bn = bq % NP;
  const int64_t bc_stride = static_cast<int64_t>(a.G) * 2 * a.N;
  float* const pbc = kCarry ? nullptr : a.part_bc + ((static_cast<int64_t>(sub) * a.batch + b) * a.T * a.G + g) * (2 * a.N) +
                                        (NT < 2 * NP ? 0 : bq < NP ? bn : a.N + bn);

  bool any_cut = false;
  int buf = 1;
  for (int t0 = last + R; t0 >= t_lo; t0 -= R, buf ^= 1) {
    f2 h[R + 1][2][2];                                     // h[r]: the state before token r, h[R] behind the last
    cp_async_wait<0>();
    __syncthreads();
    fetch(t0 - R, buf ^ 1);
    if (t0 > last) continue;                               // the first round only fetches
    const int rows = min(R, t_live - t0);
    // bit r: token r starts an episode (every warp finds them for itself)
    const unsigned cuts = __ballot_sync(0xffffffffu, reset && lane < rows && reset[t0 + lane]);
    any_cut |= cuts != 0;
    for (int r = er; r < R; r += kStep) {
      float dv[4], gv[4], uv[4], dg[4], ds[4], bias[4];
      const int at = r * CH + ec;
      load_vec<float, 4>(sm.bias + ec, bias);
      load_vec<T, 4>(sm.dt[buf] + at, dv);
      load_vec<T, 4>(sm.dout[buf] + at, gv);
      if (gz) {
        float zv[4];
        load_vec<T, 4>(sm.z[buf] + at, zv);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float s = sigmoid(zv[j]), w = gv[j] * s;
          dg[j] = w * fmaf(zv[j], 1.0f - s, 1.0f);
          gv[j] = w * zv[j];
        }
        if (!kCarry) store_vec<float, 4>(sm.dgate + at, dg);
      }
      if (!kCarry && a.softplus) {
#pragma unroll
        for (int j = 0; j < 4; ++j) ds[j] = sigmoid(dv[j] + bias[j]);
        store_vec<float, 4>(sm.dstep + at, ds);
      }
      step_of(dv, bias, a.softplus);
      if (!kCarry) {
        load_vec<T, 4>(sm.x[buf] + at, uv);
#pragma unroll
        for (int j = 0; j < 4; ++j) uv[j] *= dv[j];
      }
      if (r >= rows || ec + 4 > nch) {                     // what is not there adds nothing and changes nothing
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r >= rows || ec + j >= nch) dv[j] = gv[j] = uv[j] = 0.0f;
      }
      store_vec<float, 4>(sm.delta + at, dv);
      store_vec<float, 4>(sm.g + at, gv);
      if (!kCarry) store_vec<float, 4>(sm.u + at, uv);
    }
    for (int i = threadIdx.x; i < R * NP; i += NT) {
      const int r = i / NP, n = i % NP;
      const bool in = r < rows && n < a.N;
      const float Cv = in ? to_f(sm.C[buf][i]) : 0.0f, Bv = !kCarry && in ? to_f(sm.B[buf][i]) : 0.0f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sm.Cf[(r * 4 + copy_of(q)) * NP + (n ^ q)] = Cv;
        if (!kCarry) sm.Bf[(r * 4 + copy_of(q)) * NP + (n ^ q)] = Bv;
      }
    }
    __syncthreads();
    const float* const Bl = sm.Bf + copy_of(order) * NP + n0;
    const float* const Cl = sm.Cf + copy_of(order) * NP + n0;
    auto twice = [](const float* p, f2 (&v)[2], float (&x)[2]) {       // the two channels' numbers
      const float2 q = *reinterpret_cast<const float2*>(p);
      x[0] = q.x;
      x[1] = q.y;
      v[0] = pack2(q.x, q.x);
      v[1] = pack2(q.y, q.y);
    };
    if constexpr (kCarry) {
#pragma unroll
      for (int r = R - 1; r >= 0; --r) {
        f2 Ct[2], dl[2], gv[2];
        float dx[2], gx2[2];
        load_pairs(Cl + r * 4 * NP, Ct[0], Ct[1]);
        twice(sm.delta + r * CH + ch, dl, dx);
        twice(sm.g + r * CH + ch, gv, gx2);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          sumd[k] += dx[k];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            dh[k][q] = mul2(fma2(gv[k], Ct[q], dh[k][q]), decay2(dl[k], A2[k][q]));
            if (cuts >> r & 1u) dh[k][q].v = 0;
          }
        }
      }
    } else {
      load_h(sm.hs[buf] - static_cast<int64_t>(d0) * a.N, h[0], std::false_type{});
      auto sweeps = [&](auto with_cuts) {
        constexpr bool kCuts = decltype(with_cuts)::value;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          f2 Bt[2], dl[2], u[2];
          float x0[2], x1[2];
          load_pairs(Bl + r * 4 * NP, Bt[0], Bt[1]);
          twice(sm.delta + r * CH + ch, dl, x0);
          twice(sm.u + r * CH + ch, u, x1);
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              f2 before = h[r][k][q];
              if (kCuts && (cuts >> r & 1u)) before.v = 0;
              h[r + 1][k][q] = fma2(decay2(dl[k], A2[k][q]), before, mul2(u[k], Bt[q]));
            }
        }
#pragma unroll
        for (int r = R - 1; r >= 0; --r) {
          f2 Bt[2], Ct[2], dl[2], u[2], gv[2], dB[2], dC[2];
          float x0[2], x1[2], x2[2], s3[3][2];
          load_pairs(Bl + r * 4 * NP, Bt[0], Bt[1]);
          load_pairs(Cl + r * 4 * NP, Ct[0], Ct[1]);
          twice(sm.delta + r * CH + ch, dl, x0);
          twice(sm.u + r * CH + ch, u, x1);
          twice(sm.g + r * CH + ch, gv, x2);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            f2 y, ub, qa;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const f2 v = fma2(gv[k], Ct[q], dh[k][q]), now = h[r + 1][k][q];
              dB[q] = k == 0 ? mul2(v, u[k]) : fma2(v, u[k], dB[q]);
              dC[q] = k == 0 ? mul2(now, gv[k]) : fma2(now, gv[k], dC[q]);
              y = q == 0 ? mul2(now, Ct[q]) : fma2(now, Ct[q], y);
              ub = q == 0 ? mul2(v, Bt[q]) : fma2(v, Bt[q], ub);
              f2 va = mul2(v, decay2_again(dl[k], A2[k][q]));
              f2 w = mul2(va, h[r][k][q]);
              if (kCuts && (cuts >> r & 1u)) va.v = w.v = 0;
              qa = q == 0 ? mul2(w, A2[k][q]) : fma2(w, A2[k][q], qa);
              dA[k][q] = fma2(w, dl[k], dA[k][q]);
              dh[k][q] = va;
            }
            s3[0][k] = sum_of(y);
            s3[1][k] = sum_of(ub);
            s3[2][k] = sum_of(qa);
          }
#pragma unroll
          for (int e = 0; e < 3; ++e) reduce_lanes<LN, 2>(s3[e], lane);
          if (reduced_writer<LN, 2>(lane)) {
            const int at = r * CH + ch + reduced_channel<LN, 2>(lane);
#pragma unroll
            for (int e = 0; e < kReduced<LN, 2>; ++e) {
              sm.y[at + e] = s3[0][e];
              sm.ub[at + e] = s3[1][e];
              sm.qa[at + e] = s3[2][e];
            }
          }
          float b4[4], c4[4];
          unpack2(dB[0], b4[0], b4[1]);
          unpack2(dB[1], b4[2], b4[3]);
          unpack2(dC[0], c4[0], c4[1]);
          unpack2(dC[1], c4[2], c4[3]);
          reduce_rows<LN>(b4, c4, lane, n0 + order, sm.red[warp][r]);
        }
      };
      if (cuts) sweeps(std::true_type{});
      else sweeps(std::false_type{});
      __syncthreads();
      for (int r = er; r < rows; r += kStep) {
        if (ec >= nch) break;
        float xv[4], gv[4], dl[4], y[4], ub[4], qa[4], dx[4], ddt[4], skip[4];
        const int at = r * CH + ec;
        const int64_t o = static_cast<int64_t>(t0 + r) * a.dim + ec;
        load_vec<T, 4>(sm.x[buf] + at, xv);
        load_vec<float, 4>(sm.skip + ec, skip);
        if (gz) {
          float dz[4];
          load_vec<float, 4>(sm.y + at, y);
          load_vec<float, 4>(sm.dgate + at, dz);
#pragma unroll
          for (int j = 0; j < 4; ++j) dz[j] *= fmaf(skip[j], xv[j], y[j]);
          store_quad<T>(gdz + o, dz, nch - ec, a.mode_d == kPieces16);
        }
        load_vec<float, 4>(sm.g + at, gv);
        load_vec<float, 4>(sm.delta + at, dl);
        load_vec<float, 4>(sm.ub + at, ub);
        load_vec<float, 4>(sm.qa + at, qa);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          dx[j] = fmaf(ub[j], dl[j], gv[j] * skip[j]);
          ddt[j] = fmaf(ub[j], xv[j], qa[j] * kLn2);
        }
        if (a.softplus) {
          float ds[4];
          load_vec<float, 4>(sm.dstep + at, ds);
#pragma unroll
          for (int j = 0; j < 4; ++j) ddt[j] *= ds[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {                      // channels past the last are never looked at
          sD[j] = fmaf(gv[j], xv[j], sD[j]);
          sV[j] += ddt[j];
        }
        store_quad<T>(gdx + o, dx, nch - ec, a.mode_d == kPieces16);
        store_quad<T>(gddt + o, ddt, nch - ec, a.mode_d == kPieces16);
      }
      if constexpr (NT >= 2 * NP) {
        if (bn < a.N) {
          for (int r = br; r < rows; r += kBcStep) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < NT / 32; ++w) s += sm.red[w][r][bq];
            pbc[(t0 + r) * bc_stride] = s;
          }
        }
      } else {
        for (int i = threadIdx.x; i < rows * 2 * NP; i += NT) {
          const int r = i / (2 * NP), q = i % (2 * NP), n = q % NP;
          if (n >= a.N) continue;
          float s = 0.0f;
#pragma unroll
          for (int w = 0; w < NT / 32; ++w) s += sm.red[w][r][q];
          pbc[(t0 + r) * bc_stride + (q < NP ? n : a.N + n)] = s;
        }
      }
    }
  }
  cp_async_wait<0>();
  if constexpr (kCarry) {
    store_h(a.carry + bchunk * per_row, dh);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (nl == 0 && ch + e < nch) a.sumd[bchunk * a.dim + d0 + ch + e] = sumd[e];
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
    if (a.dstate && a.chunks == 1) store_h(a.dstate + b * per_row, dh);
    store_h(a.part_a + bchunk * per_row, dA);
    // the channels' sums over the threads that share them: within the warp, then in warp order
    constexpr int kWide = kQuads < 32 ? 32 : kQuads, kRows = NT / kWide;
    static_assert(kRows <= R, "the sums of a block fit one array of the tile");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int off = 16; off >= kQuads; off /= 2) {
        sD[j] += __shfl_xor_sync(0xffffffffu, sD[j], off);
        sV[j] += __shfl_xor_sync(0xffffffffu, sV[j], off);
      }
      if (kQuads >= 32 || lane < kQuads) {
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
__global__ void __launch_bounds__(128) grad_carry_kernel(ScanArgs a) {
  const int64_t per = static_cast<int64_t>(a.dim) * a.N;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (id >= per * a.batch) return;
  const int b = static_cast<int>(id / per);
  const int64_t dn = id - b * per, row = static_cast<int64_t>(b) * a.chunks;
  const int d = static_cast<int>(dn / a.N);
  const float dh = string_chunks<true>(a.dfinal ? a.dfinal[id] : 0.0f, rate_of(a.A[dn]), a.carry + row * per + dn, per,
                                       a.sumd + row * a.dim + d, a.dim, a.cut + row, a.chunks);
  if (a.dstate) a.dstate[id] = dh;
}

// The last sums, in a fixed order. Blocks below bc_blocks: dB and dC, over a group's channel
// blocks. The others: dA, dD and ddt_bias over rows and chunks, 32 numbers a block, 8 row
// sums side by side.
template <typename T> __global__ void __launch_bounds__(256) finish_kernel(ScanArgs a, int blocks, int bc_blocks) {
  if (static_cast<int>(blockIdx.x) < bc_blocks) {
    const int64_t n = static_cast<int64_t>(a.batch) * a.T * a.G * 2 * a.N;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(bc_blocks) * 256) {
      float s = 0.0f;
      for (int k = 0; k < blocks; ++k) s += a.part_bc[k * n + i];
      const int64_t row = i / (2 * a.N);
      const int q = static_cast<int>(i - row * (2 * a.N));
      if (q < a.N) static_cast<T*>(a.dB)[row * a.N + q] = from_f<T>(s);
      else static_cast<T*>(a.dC)[row * a.N + q - a.N] = from_f<T>(s);
    }
    return;
  }
  __shared__ float red[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t na = static_cast<int64_t>(a.dim) * a.N, total = na + 2 * static_cast<int64_t>(a.dim);
  const int64_t e = static_cast<int64_t>(blockIdx.x - bc_blocks) * 32 + tx;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.chunks;
  float s = 0.0f;
  if (e < total) {
    const float* p = e < na ? a.part_a + e : a.part_v + (e - na);
    const int64_t step = e < na ? na : 2 * static_cast<int64_t>(a.dim);
    for (int64_t r = ty; r < rows; r += 8) s += p[r * step];
  }
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && e < total) {
#pragma unroll
    for (int r = 1; r < 8; ++r) s += red[r][tx];
    if (e < na) a.dA[e] = s;
    else if (e - na < a.dim) { if (a.dD) a.dD[e - na] = s; }
    else if (a.dbias) a.dbias[e - na - a.dim] = s;
  }
}

template <typename T, int LN, int NT> int launch_grad(const ScanArgs& a, cudaStream_t s) {
  using L = GradLayout<T, LN, NT>;
  const int bpg = static_cast<int>(surfk::ceil_div(a.dim / a.G, L::CH));
  const int64_t gx = static_cast<int64_t>(bpg) * a.G * a.batch;
  if (gx > 0x7fffffffLL || a.chunks > 65535) return static_cast<int>(cudaErrorInvalidValue);
  constexpr size_t smem = sizeof(typename L::Smem);
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(a.chunks));
  if (a.chunks > 1) {
    if (const int rc = allow_smem<scan_grad_kernel<T, LN, NT, true>>(smem)) return rc;
    scan_grad_kernel<T, LN, NT, true><<<grid, NT, smem, s>>>(a, bpg);
    grad_carry_kernel<<<static_cast<unsigned>(surfk::ceil_div(static_cast<int64_t>(a.batch) * a.dim * a.N, 128)), 128, 0, s>>>(a);
  }
  if (const int rc = allow_smem<scan_grad_kernel<T, LN, NT, false>>(smem)) return rc;
  scan_grad_kernel<T, LN, NT, false><<<grid, NT, smem, s>>>(a, bpg);
  const int64_t bc = surfk::ceil_div(static_cast<int64_t>(a.batch) * a.T * a.G * 2 * a.N, 256);
  const int bc_blocks = static_cast<int>(bc < 148 * 16 ? bc : 148 * 16);
  const int64_t weights = surfk::ceil_div(static_cast<int64_t>(a.dim) * (a.N + 2), 32);
  finish_kernel<T><<<static_cast<unsigned>(bc_blocks + weights), 256, 0, s>>>(a, bpg, bc_blocks);
  SURF_RETURN_LAUNCH();
}

// whether a group's channels leave half of an ordinary block idle
template <int LN> bool small_blocks(int per_group) { return 2 * per_group <= grad_channels<LN>(kGradBlock<LN>); }

template <typename T, int LN> int launch_grad(const ScanArgs& a, cudaStream_t s) {
  return small_blocks<LN>(a.dim / a.G) ? launch_grad<T, LN, kSmallBlock<LN>>(a, s) : launch_grad<T, LN, kGradBlock<LN>>(a, s);
}

}  // namespace

SURF_EXPORT int surf_seq_scan_grad(const void* args, int dtype, void* stream) {
  const ScanArgs a = *static_cast<const ScanArgs*>(args);
  if (a.batch <= 0 || a.dim <= 0) return static_cast<int>(cudaErrorInvalidValue);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_lanes(a.N, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    return dtype == kBf16 ? launch_grad<bf16, LN>(a, s) : launch_grad<float, LN>(a, s);
  });
}

// channel blocks of a group (the caller sizes part_bc with it)
SURF_EXPORT int surf_seq_scan_grad_blocks(int per_group, int N) {
  return by_lanes(N, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    return static_cast<int>(surfk::ceil_div(per_group, grad_channels<LN>(small_blocks<LN>(per_group) ? kSmallBlock<LN> : kGradBlock<LN>)));
  });
}
