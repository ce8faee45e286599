// seq_scan.cu — selective state space scan: whole sequences and single tokens (sm_100a).
//
//   delta = softplus(dt + bias)
//   h[n] <- exp(delta * A[d, n]) * h[n] + delta * x * B[n]        (32-bit state)
//   out  = (sum_n C[n] * h[n] + D[d] * x) * silu(z)
//
// for every channel d of every row, token by token. reset[b, t] empties the state
// before token t; tokens from lengths[b] on leave it alone, give zeros and are never
// read. A block takes a stretch of channels through its tokens in tiles of kTile: the
// tile's x, dt, z, B, C arrive by asynchronous copies while the tile before is worked
// on, delta and delta * x are made once per channel, and the recurrence runs with the
// states in registers (4 states of K channels a thread).
//
// Long rows with too few channels to fill the GPU are cut into chunks: a first pass
// leaves each chunk's state from an empty start and its sum of delta (the chunk's
// whole decay is exp(A * sum), 0 across a reset), a small kernel strings the chunks
// together, and the scan then runs in all chunks at once.
//
// Measured on a B200, 16 states, back to back: 256 x 128 x 512 bf16 117 us, f32 143 us (127 and
// 158 us with the states kept for the gradient), a prompt of 8191 x 1024 in 74 chunks 114 and
// 138 us (launched one by one: first pass 49, stringing 13, scan 62 us), one token of 2048 envs
// x 1024 67 us in both types (285 MB, 4.3 TB/s). The recurrence's exponentials alone take the
// SMs' units 60 us for 256 x 128 x 512 (2^28 of them, 16 a cycle and SM), softplus and gate,
// four of their kind a (token, channel), 15 us more; the rest is the other work on every (token,
// channel), which shares the issue slots with the recurrence, and waits at 16 warps on an SM
// (0.52 issued a cycle and scheduler; 24 warps with tiles of 8 tokens were no faster: 120 us
// against 121 us for every 2^28 at 1184 rows).
#include "seq_scan.cuh"

namespace {

using namespace seqk;

constexpr int kTile = 16;

template <typename T, int LN, int kThreads> struct Layout {
  static constexpr int K = LN < 4 ? 2 : 4;               // channels of a thread, taken in pairs
  static constexpr int CH = scan_channels<LN>(kThreads); // channels of a block
  static constexpr int NP = 4 * LN;                      // states, padded
  struct Smem {
    alignas(16) T x[2][kTile * CH], dt[2][kTile * CH], z[2][kTile * CH], B[2][kTile * NP], C[2][kTile * NP];
    alignas(16) float delta[kTile * CH], u[kTile * CH];  // u: delta * x, then y = C . h of the token
    alignas(16) float Bd[kTile * NP * 2], Cd[kTile * NP * 2];    // 32-bit, every value twice
  };
};

// kCarry: only the chunk's end state from an empty start and its sum of delta.
//
// The recurrence of a token costs 4 multiply-adds and an exponential per state. Two
// channels share an instruction (f32x2), which leaves the exponential unit's 16 a cycle
// and SM as the bound: the loop below takes 143 to 153 cycles for 512 states where that unit
// takes 128.
template <typename T, int LN, int kThreads, bool kCarry>
__global__ void __launch_bounds__(kThreads, 512 / kThreads) scan_kernel(ScanArgs a, int blocks_per_group) {
  using L = Layout<T, LN, kThreads>;
  constexpr int K = L::K, P = K / 2, CH = L::CH, NP = L::NP;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  typename L::Smem& sm = *reinterpret_cast<typename L::Smem*>(smem_raw);
  const int blocks = blocks_per_group * a.G;
  const int b = blockIdx.x / blocks, blk = blockIdx.x - b * blocks;
  const int g = blk / blocks_per_group, per_group = a.dim / a.G;
  const int c0 = (blk - g * blocks_per_group) * CH;
  const int nch = min(CH, per_group - c0);
  const int d0 = g * per_group + c0;                     // first channel of the block
  const int chunk = blockIdx.y;
  const int t_lo = chunk * a.chunk, t_hi = min(a.T, t_lo + a.chunk);
  const int len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
  const int t_live = min(t_hi, len);

  const int lane = threadIdx.x & 31;
  const int nl = lane & (LN - 1);
  const int ch = threadIdx.x / LN * K;                   // the thread's first channel within the block
  const int n0 = nl * 4;

  f2 A2[P][4], h[P][4], sumd[P];                         // pairs of channels (ch + 2 p, ch + 2 p + 1)
#pragma unroll
  for (int p = 0; p < P; ++p) {
    float4 av[2], hv[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool on = ch + 2 * p + e < nch;
      const int64_t row = static_cast<int64_t>(d0 + ch + 2 * p + e) * a.N, bd = static_cast<int64_t>(a.dim) * a.N;
      av[e] = hv[e] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (on) {
        av[e] = load_state4(a.A + row, n0, a.N);
        if (!kCarry) {
          if (a.chunks > 1) hv[e] = load_state4(a.carry + (static_cast<int64_t>(b) * a.chunks + chunk) * bd + row, n0, a.N);
          else if (a.state) hv[e] = load_state4(a.state + b * bd + row, n0, a.N);
        }
      }
    }
    const float a0[4] = {av[0].x, av[0].y, av[0].z, av[0].w}, a1[4] = {av[1].x, av[1].y, av[1].z, av[1].w};
    const float h0[4] = {hv[0].x, hv[0].y, hv[0].z, hv[0].w}, h1[4] = {hv[1].x, hv[1].y, hv[1].z, hv[1].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      A2[p][i] = pack2(rate_of(a0[i]), rate_of(a1[i]));
      h[p][i] = pack2(h0[i], h1[i]);
    }
    sumd[p] = pack2(0.0f, 0.0f);
  }
  auto store_h = [&](float* dst) {                       // dst: the first channel's states
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (ch + k >= nch) continue;
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float lo, hi;
        unpack2(h[k / 2][i], lo, hi);
        v[i] = k & 1 ? hi : lo;
      }
      store_state4(dst + static_cast<int64_t>(k) * a.N, n0, a.N, v);
    }
  };
  const T* gx = static_cast<const T*>(a.x) + b * a.x_b + d0;
  const T* gdt = static_cast<const T*>(a.dt) + b * a.dt_b + d0;
  const T* gz = a.z ? static_cast<const T*>(a.z) + b * a.z_b + d0 : nullptr;
  const T* gB = static_cast<const T*>(a.B) + b * a.B_b + g * a.B_g;
  const T* gC = static_cast<const T*>(a.C) + b * a.C_b + g * a.C_g;
  T* gout = static_cast<T*>(a.out) + b * a.out_b + d0;
  const uint8_t* reset = a.reset ? a.reset + b * a.r_b : nullptr;
  float* saved = a.saved ? a.saved + (static_cast<int64_t>(b) * ((a.T + kSave - 1) / kSave) * a.dim + d0 + ch) * a.N : nullptr;

  // rows of channels in 16-byte pieces: this thread's first piece of the next tile
  using Pieces = RowPieces<T, kThreads, CH, kTile>;
  const bool pieces = a.mode_d == kPieces16, mine = Pieces::column() < nch;
  const T *px = gx + (t_lo + Pieces::row()) * a.x_t + Pieces::column(), *pdt = gdt + (t_lo + Pieces::row()) * a.dt_t + Pieces::column();
  const T* pz = gz ? gz + (t_lo + Pieces::row()) * a.z_t + Pieces::column() : nullptr;
  using Twin = TwinPieces<T, kThreads, NP, kTile>;
  const bool twin = Twin::kFits && a.mode_n == kPieces16 && a.N == NP;
  const bool my_twin = kCarry ? Twin::which() == 0 : Twin::which() < 2;
  const int64_t twin_t = Twin::which() == 0 ? a.B_t : a.C_t;
  const T* ptwin = (Twin::which() == 0 ? gB : gC) + (t_lo + Twin::row()) * twin_t + Twin::column();
  auto fetch = [&](int t, int buf) {
    const int rows = min(kTile, t_live - t);
    if (rows > 0) {
      if (pieces) {
        if (mine) {
          Pieces::copy(sm.x[buf], px, a.x_t, rows);
          Pieces::copy(sm.dt[buf], pdt, a.dt_t, rows);
          if (!kCarry && gz) Pieces::copy(sm.z[buf], pz, a.z_t, rows);
        }
        px += kTile * a.x_t;
        pdt += kTile * a.dt_t;
        if (!kCarry && gz) pz += kTile * a.z_t;
      } else {
#pragma unroll 1
        for (int i = 0; i < (kCarry || !gz ? 2 : 3); ++i) {
          const int64_t stride = i == 0 ? a.x_t : i == 1 ? a.dt_t : a.z_t;
          copy_rows<T, kThreads, CH>(i == 0 ? sm.x[buf] : i == 1 ? sm.dt[buf] : sm.z[buf], (i == 0 ? gx : i == 1 ? gdt : gz) + t * stride, stride,
                                     rows, nch, a.mode_d);
        }
      }
      if (twin) {
        if (my_twin && Twin::row() < rows)
          cp_async16((Twin::which() == 0 ? sm.B[buf] : sm.C[buf]) + Twin::row() * NP + Twin::column(), ptwin);
        ptwin += kTile * twin_t;
      } else {
#pragma unroll 1
        for (int i = 0; i < (kCarry ? 1 : 2); ++i) {
          const int64_t stride = i == 0 ? a.B_t : a.C_t;
          copy_rows<T, kThreads, NP>(i == 0 ? sm.B[buf] : sm.C[buf], (i == 0 ? gB : gC) + t * stride, stride, rows, a.N, a.mode_n);
        }
      }
    }
    cp_async_commit();
  };

  // before and behind the recurrence a thread works on 4 channels of every kStep-th token
  constexpr int kQuads = CH / 4, kStep = kThreads / kQuads;
  const int ec = threadIdx.x % kQuads * 4, er = threadIdx.x / kQuads;
  float bias[4], skip[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bias[j] = a.bias && ec + j < nch ? a.bias[d0 + ec + j] : 0.0f;
    skip[j] = a.D && ec + j < nch ? a.D[d0 + ec + j] : 0.0f;
  }

  // the tile's reset flags, a token a lane, on their way a tile ahead
  auto flag_of = [&](int t) { return reset && lane < kTile && t + lane < t_live && reset[t + lane] != 0; };
  bool any_cut = false, flag = flag_of(t_lo);
  int buf = 1;
  for (int t0 = t_lo - kTile; t0 < t_live; t0 += kTile, buf ^= 1) {
    cp_async_wait<0>();
    __syncthreads();
    fetch(t0 + kTile, buf ^ 1);
    if (t0 < t_lo) continue;                             // the first round only fetches
    const int rows = min(kTile, t_live - t0);
    // bit r: token r starts an episode (every warp finds them for itself)
    static_assert(kTile <= 32, "a warp's lanes look at a tile's tokens");
    const unsigned cuts = __ballot_sync(0xffffffffu, flag);
    any_cut |= cuts != 0;
    flag = flag_of(t0 + kTile);
    // delta and delta * x (channels past the block's last are never looked at)
#pragma unroll 2
    for (int r = er; r < kTile; r += kStep) {
      float dv[4], xv[4];
      load_vec<T, 4>(sm.dt[buf] + r * CH + ec, dv);
      load_vec<T, 4>(sm.x[buf] + r * CH + ec, xv);
      step_of(dv, bias, a.softplus);
#pragma unroll
      for (int j = 0; j < 4; ++j) xv[j] *= dv[j];
      store_vec<float, 4>(sm.delta + r * CH + ec, dv);
      store_vec<float, 4>(sm.u + r * CH + ec, xv);
    }
    if (rows < kTile) {                                  // past the last token the state stays as it is
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      for (int r = er; r < kTile; r += kStep)
        if (r >= rows) {
          store_vec<float, 4>(sm.delta + r * CH + ec, zero);
          store_vec<float, 4>(sm.u + r * CH + ec, zero);
        }
    }
    for (int i = threadIdx.x; i < kTile * NP; i += kThreads) {
      const int r = i / NP, n = i % NP;
      const bool in = r < rows && n < a.N;
      const float Bv = in ? to_f(sm.B[buf][i]) : 0.0f;
      *reinterpret_cast<float2*>(sm.Bd + 2 * i) = make_float2(Bv, Bv);
      if (!kCarry) {
        const float Cv = in ? to_f(sm.C[buf][i]) : 0.0f;
        *reinterpret_cast<float2*>(sm.Cd + 2 * i) = make_float2(Cv, Cv);
      }
    }
    __syncthreads();
#pragma unroll 8
    for (int r = 0; r < kTile; ++r) {
      if (cuts >> r & 1u) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) h[p][i].v = 0;
      }
      if (!kCarry && (r % kSave) == 0 && saved && r < rows)
        store_h(saved + static_cast<int64_t>((t0 + r) / kSave) * a.dim * a.N);
      f2 dl[P], u[P], y[P], Bt[4], Ct[4];
      if constexpr (P == 2) {
        load_pairs(sm.delta + r * CH + ch, dl[0], dl[1]);
        load_pairs(sm.u + r * CH + ch, u[0], u[1]);
      } else {
        dl[0].v = *reinterpret_cast<const unsigned long long*>(sm.delta + r * CH + ch);
        u[0].v = *reinterpret_cast<const unsigned long long*>(sm.u + r * CH + ch);
      }
      load_pairs(sm.Bd + (r * NP + n0) * 2, Bt[0], Bt[1]);
      load_pairs(sm.Bd + (r * NP + n0) * 2 + 4, Bt[2], Bt[3]);
      if (!kCarry) {
        load_pairs(sm.Cd + (r * NP + n0) * 2, Ct[0], Ct[1]);
        load_pairs(sm.Cd + (r * NP + n0) * 2 + 4, Ct[2], Ct[3]);
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (kCarry) sumd[p] = add2(sumd[p], dl[p]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h[p][i] = fma2(decay2(dl[p], A2[p][i]), h[p][i], mul2(u[p], Bt[i]));
          if (!kCarry) y[p] = i == 0 ? mul2(h[p][i], Ct[i]) : fma2(h[p][i], Ct[i], y[p]);
        }
      }
      if (!kCarry) {
        float acc[K];
#pragma unroll
        for (int p = 0; p < P; ++p) unpack2(y[p], acc[2 * p], acc[2 * p + 1]);
        reduce_lanes<LN, K>(acc, lane);
        // u of this token and these channels has been read by the lanes whose sums are here
        if (reduced_writer<LN, K>(lane)) {
#pragma unroll
          for (int q = 0; q < kReduced<LN, K>; ++q) sm.u[r * CH + ch + reduced_channel<LN, K>(lane) + q] = acc[q];
        }
      }
    }
    __syncthreads();
    if (!kCarry) {
#pragma unroll 2
      for (int r = er; r < rows; r += kStep) {
        if (ec >= nch) break;
        float o[4], xv[4];
        load_vec<float, 4>(sm.u + r * CH + ec, o);
        load_vec<T, 4>(sm.x[buf] + r * CH + ec, xv);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(skip[j], xv[j], o[j]);
        if (gz) {
          float zv[4];
          load_vec<T, 4>(sm.z[buf] + r * CH + ec, zv);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] *= zv[j] * sigmoid(zv[j]);
        }
        store_quad<T>(gout + (t0 + r) * a.out_t + ec, o, nch - ec, a.mode_d == kPieces16);
      }
    }
  }
  cp_async_wait<0>();
  if (!kCarry) {
    for (int t = max(t_lo, t_live); t < t_hi; ++t)
      for (int c = threadIdx.x; c < nch; c += kThreads) gout[t * a.out_t + c] = from_f<T>(0.0f);
  }
  if (kCarry) store_h(a.carry + ((static_cast<int64_t>(b) * a.chunks + chunk) * a.dim + d0 + ch) * a.N);
  else if (a.final_state && chunk == a.chunks - 1) store_h(a.final_state + (static_cast<int64_t>(b) * a.dim + d0 + ch) * a.N);
  if (kCarry) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float v[2];
      unpack2(sumd[p], v[0], v[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (nl == 0 && ch + 2 * p + e < nch)
          a.sumd[(static_cast<int64_t>(b) * a.chunks + chunk) * a.dim + d0 + ch + 2 * p + e] = v[e];
    }
    if (threadIdx.x == 0) a.cut[static_cast<int64_t>(b) * a.chunks + chunk] = any_cut;   // the same from every block
  }
}

// carry[b, c] <- the state before chunk c. One thread per (b, d, n).
__global__ void __launch_bounds__(128) carry_kernel(ScanArgs a) {
  const int64_t per = static_cast<int64_t>(a.dim) * a.N;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (id >= per * a.batch) return;
  const int b = static_cast<int>(id / per);
  const int64_t dn = id - b * per, row = static_cast<int64_t>(b) * a.chunks;
  const int d = static_cast<int>(dn / a.N);
  string_chunks<false>(a.state ? a.state[id] : 0.0f, rate_of(a.A[dn]), a.carry + row * per + dn, per, a.sumd + row * a.dim + d, a.dim,
                       a.cut + row, a.chunks);
}

template <typename T, int LN, int kThreads> int launch_scan(const ScanArgs& a, cudaStream_t s) {
  using L = Layout<T, LN, kThreads>;
  const int bpg = static_cast<int>(surfk::ceil_div(a.dim / a.G, L::CH));
  const int64_t gx = static_cast<int64_t>(bpg) * a.G * a.batch;
  if (gx > 0x7fffffffLL || a.chunks > 65535) return static_cast<int>(cudaErrorInvalidValue);
  constexpr size_t smem = sizeof(typename L::Smem);
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(a.chunks));
  if (a.chunks > 1) {
    if (const int rc = allow_smem<scan_kernel<T, LN, kThreads, true>>(smem)) return rc;
    scan_kernel<T, LN, kThreads, true><<<grid, kThreads, smem, s>>>(a, bpg);
    const int64_t n = static_cast<int64_t>(a.batch) * a.dim * a.N;
    carry_kernel<<<static_cast<unsigned>(surfk::ceil_div(n, 128)), 128, 0, s>>>(a);
  }
  if (const int rc = allow_smem<scan_kernel<T, LN, kThreads, false>>(smem)) return rc;
  scan_kernel<T, LN, kThreads, false><<<grid, kThreads, smem, s>>>(a, bpg);
  SURF_RETURN_LAUNCH();
}

// whether a group's channels leave half of an ordinary block idle
template <int LN> bool small_blocks(int per_group) { return 2 * per_group <= scan_channels<LN>(kScanBlock<LN>); }

template <typename T, int LN> int launch_scan(const ScanArgs& a, cudaStream_t s) {
  return small_blocks<LN>(a.dim / a.G) ? launch_scan<T, LN, kSmallBlock<LN>>(a, s) : launch_scan<T, LN, kScanBlock<LN>>(a, s);
}

// ---- single tokens -----------------------------------------------------------------------
// Row r is the next token of the env in slot slots[r] of the state pool (-1: none, its output
// is zero); the slot's state is moved on in place. LN lanes hold a channel's states.
struct StepArgs {
  const void *x, *dt, *z, *B, *C;
  const float *A, *D, *bias;
  float* pool;                                 // [slots, D, N]
  const uint8_t* reset;                        // [rows] or null
  const int* slots;                            // [rows] or null: row r is slot r
  void* out;
  int* err;
  int64_t x_r, dt_r, z_r, B_r, B_g, C_r, C_g, out_r;
  int rows, dim, N, G, softplus, n_slots;
  int whole, pad;                              // rows of B and C start on 4-element boundaries, N is a multiple of 4
};
static_assert(sizeof(StepArgs) == 21 * 8 + 8 * 4, "as the caller packs it");

// Four neighbouring values of a row of B or C as they are in memory, zeros past the N-th
template <typename T> struct Quad {
  T v[4];
  __device__ __forceinline__ void load(const T* p, int left, bool whole) {
    if (whole) {
      if (left >= 4) *reinterpret_cast<std::conditional_t<sizeof(T) == 2, uint2, uint4>*>(v) = *reinterpret_cast<const std::conditional_t<sizeof(T) == 2, uint2, uint4>*>(p);
      else v[0] = v[1] = v[2] = v[3] = from_f<T>(0.0f);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = i < left ? p[i] : from_f<T>(0.0f);
    }
  }
};

// One pass over the states, 8 bytes a state to move. A thread moves 4 states of K channels
// that lie 32 / LN apart, so a warp's loads are whole 128-byte lines; of a channel's LN lanes
// one makes delta, delta * x and the gated output and hands them round (with a thread for 4
// states of one channel, every lane made its own: 66 instructions a state, 109 us at
// 2048x1024x16; now 67 us, 4.3 TB/s).
template <typename T, int LN> __global__ void __launch_bounds__(128) step_kernel(StepArgs a) {
  constexpr int K = LN < 4 ? LN : 4, kRowsOfWarp = 32 / LN;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nl = lane & (LN - 1), n0 = nl * 4, row = lane / LN;
  const int r = blockIdx.x;
  const int slot = a.slots ? a.slots[r] : r;
  const int base = (blockIdx.y * 4 + warp) * (kRowsOfWarp * K) + row;      // channel k: base + k * kRowsOfWarp
  const int mine = base + reduced_channel<LN, K>(lane) * kRowsOfWarp;
  if (slot < 0 || slot >= a.n_slots) {                                     // the same for the whole block
    if (mine < a.dim) static_cast<T*>(a.out)[r * a.out_r + mine] = from_f<T>(0.0f);
    if (slot >= 0 && threadIdx.x == 0) surfk::report_error(a.err, surfk::kErrSlotIndex);
    return;
  }
  float* pool = a.pool + static_cast<int64_t>(slot) * a.dim * a.N;
  const bool cut = a.reset && a.reset[r];
  float4 h4[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int d = base + k * kRowsOfWarp;
    h4[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d < a.dim && !cut) h4[k] = load_state4(pool + static_cast<int64_t>(d) * a.N, n0, a.N);
  }
  alignas(16) Quad<T> B, C;
  const T* rowB = static_cast<const T*>(a.B) + r * a.B_r + n0;
  const T* rowC = static_cast<const T*>(a.C) + r * a.C_r + n0;
  B.load(rowB, a.N - n0, a.whole);
  C.load(rowC, a.N - n0, a.whole);
  float x = 0.0f, dv = 0.0f, z = 0.0f;
  if (mine < a.dim) {
    x = to_f(static_cast<const T*>(a.x)[r * a.x_r + mine]);
    dv = to_f(static_cast<const T*>(a.dt)[r * a.dt_r + mine]) + (a.bias ? a.bias[mine] : 0.0f);
    if (a.z) z = to_f(static_cast<const T*>(a.z)[r * a.z_r + mine]);
    if (a.softplus) dv = softplus(dv);
  }
  const float ux = dv * x;
  float acc[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int d = base + k * kRowsOfWarp, from = row * LN + k * (LN / K);
    const float dl = __shfl_sync(0xffffffffu, dv, from), u = __shfl_sync(0xffffffffu, ux, from);
    acc[k] = 0.0f;
    if (d < a.dim) {
      if (a.G > 1) {
        const int g = d / (a.dim / a.G);
        B.load(rowB + g * a.B_g, a.N - n0, a.whole);
        C.load(rowC + g * a.C_g, a.N - n0, a.whole);
      }
      const float4 A4 = load_state4(a.A + static_cast<int64_t>(d) * a.N, n0, a.N);
      const float Av[4] = {A4.x, A4.y, A4.z, A4.w};
      float h[4] = {h4[k].x, h4[k].y, h4[k].z, h4[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {                      // states past the N-th stay zero: A, B and h are there
        h[i] = fmaf(decay(dl, rate_of(Av[i])), h[i], u * to_f(B.v[i]));
        acc[k] = fmaf(h[i], to_f(C.v[i]), acc[k]);
      }
      store_state4(pool + static_cast<int64_t>(d) * a.N, n0, a.N, h);
    }
  }
  reduce_lanes<LN, K>(acc, lane);
  if (mine < a.dim && reduced_writer<LN, K>(lane)) {
    float o = acc[0] + (a.D ? a.D[mine] * x : 0.0f);
    if (a.z) o *= z * sigmoid(z);
    static_cast<T*>(a.out)[r * a.out_r + mine] = from_f<T>(o);
  }
}

template <typename T, int LN> int launch_step(const StepArgs& a, cudaStream_t s) {
  constexpr int kChannels = 4 * (32 / LN) * (LN < 4 ? LN : 4);
  const int64_t across = surfk::ceil_div(a.dim, kChannels);
  if (across > 65535) return static_cast<int>(cudaErrorInvalidValue);
  step_kernel<T, LN><<<dim3(static_cast<unsigned>(a.rows), static_cast<unsigned>(across)), 128, 0, s>>>(a);
  SURF_RETURN_LAUNCH();
}

}  // namespace

SURF_EXPORT int surf_seq_scan(const void* args, int dtype, void* stream) {
  const ScanArgs a = *static_cast<const ScanArgs*>(args);
  if (a.batch <= 0 || a.dim <= 0) return 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_lanes(a.N, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    return dtype == kBf16 ? launch_scan<bf16, LN>(a, s) : launch_scan<float, LN>(a, s);
  });
}

SURF_EXPORT int surf_seq_scan_step(const void* args, int dtype, void* stream) {
  const StepArgs a = *static_cast<const StepArgs*>(args);
  if (a.rows <= 0 || a.dim <= 0) return 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_lanes(a.N, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    return dtype == kBf16 ? launch_step<bf16, LN>(a, s) : launch_step<float, LN>(a, s);
  });
}

// The forward's blocks of a row, in threads (the caller cuts rows where they do not fill the GPU).
SURF_EXPORT int surf_seq_scan_threads(int per_group, int groups, int N) {
  return by_lanes(N, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    const int threads = small_blocks<LN>(per_group) ? kSmallBlock<LN> : kScanBlock<LN>;
    return static_cast<int>(surfk::ceil_div(per_group, scan_channels<LN>(threads))) * groups * threads;
  });
}
