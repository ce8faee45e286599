// delta_grad.cu — gradient of the gated delta rule (sm_100a). Notation of delta.cuh.
//
// Back through the chunks with dS the gradient of the state behind one (rows values), a chunk
// starting from S with W, U = beta W of the forward pass made again:
//   dU = P^T dO + tail K dS^T                    Z = (I + M beta)^-T (beta dU) = dV
//   dS <- end dS + sum_i scale head_i dO_i q_i^T - head_i Z_i k_i^T
//   dM = -Z U^T (j < i)   dP = dO U^T (j <= i)   dbeta_i = W_i.dU_i - sum_l M_li (Z_l.W_i)
//   dq_i = scale head_i S^T dO_i + sum_j scale dP_ij D_ij k_j
//   dk_i = -head_i S^T Z_i + tail_i beta_i dS^T W_i + sum_j scale dP_ji D_ji q_j + (dM_ij D_ij + dM_ji D_ji) k_j
// and of a token's log decay, with E = dP P + dM M, e_i = head_i's terms, f_j = tail_j's:
//   dg_m = sum_{j < m <= i} E_ij + sum_{i >= m} e_i + sum_{j < m} f_j + end <dS, S>.
// These are sums of what each pair's decay contributes; none is a difference of larger ones.
//
// A block for up to 64 values of a sequence's value head: two warps make the chunks ready in turn, as
// in the forward pass, four carry them out, one makes the matrices and gates of 16 x 16. By values
// (a warp for 16 rows of dS, its accumulators): the chain from dS to dS; by keys (a warp for a
// quarter of the columns): dq and dk, which sum over the values; the chain's results pass
// through shared memory as planes. S and W are the forward pass's. Blocks of one head, and heads
// that share keys, leave parts of dq and dk that a second kernel sums in order.
//
// Neither memory nor the tensor pipe bounds it (256x128x8x64x64: 518 us, 0.16 of the copy rate, tensor pipe
// 20%): each warp's instructions wait for the ones before, and many warps with code of their own
// for the instruction cache. See Plan.
#include "delta.cuh"

namespace {

using namespace delta;

constexpr int kPrep = 2, kMain = 4, kValues = 64;      // warps that make chunks ready, of the chain and of the keys; values of a block

// How a block is made up. Either teams of one head each, whose four main warps follow the chain and then the
// keys; or (kApart) one head whose chain is four warps' and whose keys are four others', a chunk behind. The
// first where there are more heads of sequences than SMs: main warps of two teams meet before each tile and run the
// same instructions at the same time, 256x128x8x64x64 518 us (apart about 700), 16x2048x16x64x64 986 (1573); apart
// where there are fewer, 2x4096x16x64x64 861 us (one head a block, nothing apart: 1326).
template <int kTeams_, bool kApart_> struct Plan {
  static constexpr int kTeams = kTeams_;
  static constexpr bool kApart = kApart_;
  static constexpr int kAll = (kApart ? 2 : 1) * kMain;                // main warps of a team
  static constexpr int kThreads = kTeams * (kAll + kPrep + 1) * 32;
  static constexpr int kStages = kApart ? 2 * kPrep : kPrep;           // a stage's barriers are one preparing warp's alone
  static constexpr int kCopies = kApart ? 2 : 1;                       // of what the chain leaves
  // a team's barriers, and how many threads meet at them: stage s ready (chain, the warp that made it),
  // stage s free (all of them), the chain's results (main, matrices), their place free (the
  // same), the matrices (keys, matrices); one for the main warps of all teams
  static constexpr int kReady = 0, kFree = kStages, kChain = 2 * kStages, kPlace = kChain + kCopies, kMatrices = kPlace + (kApart ? 2 : 0);
  static constexpr int kBars = kMatrices + 1, kEvery = 1 + kTeams * kBars;
  static_assert(kEvery < 16, "barriers of a block");
  static constexpr int kAtReady = (kMain + 1) * 32, kAtFree = (kAll + 2) * 32, kAtChain = (kAll + 1) * 32, kAtMatrices = (kMain + 1) * 32;
};

template <typename T, int DK> struct Backward {
  static constexpr int NT = Planes<T>::kToken, NI = Planes<T>::kInner, NS = Planes<T>::kShort;
  using Keys = Tile<T, DK>;
  using Values = Tile<T, kValues>;
  static constexpr int kPitchS = DK + 4, kPitchD = DK + 8;
  static constexpr int kColumns = DK / kMain < 16 ? 16 : DK / kMain;     // of a warp by keys
  struct Stage {
    Chunk<T, NI> c;
    Wide wide;                                         // in the end E's parts of P and M, and M Z W^T
    int t0, n, more;                                   // more: the tile's next episode follows in this stage
    unsigned marks;
    alignas(16) bf16 tk[Keys::kSize], tq[Keys::kSize], tdo[Values::kSize];
  };
  struct Chain {                                       // what the chain leaves of a chunk
    alignas(16) bf16 w[NI][kValues][kTile], z[NI][kValues][kTile];     // rows values, columns tokens; see swap8
    alignas(16) bf16 d[NS][kValues][kPitchD];          // dS
    // of each warp: Z W^T and dO W^T, or its outputs
    alignas(16) union { float product[2][kTile][kMat]; T out[kTile][16 + 16 / sizeof(T)]; } part[kMain];
    float by_value[kMain][2][kTile], inner[kMain];     // sums over its values: W.dU, the tails' terms; <dS, S>
  };
  template <typename P> struct Shared {
    Stage stage[P::kStages];
    // the forward pass's S and W (rows values, columns tokens) of a tile: the chain's, and where the keys' warps
    // are others, theirs
    alignas(16) float s[P::kCopies][kValues][kPitchS];
    alignas(16) float saved_w[kValues][kMat];
    alignas(16) Scratch scratch[kPrep];
    Chain chain[P::kCopies];
    alignas(16) bf16 x1[NS][kTile][kSide], x2[NS][kTile][kSide], x3[NS][kTile][kSide];
    // outputs, where other warps have the chain's place in use: the chain's dV, the keys' dq and dk
    alignas(16) T dv[P::kApart ? P::kCopies * kMain : 1][kTile][16 + 16 / sizeof(T)], out[P::kApart ? kMain : 1][kTile][16 + 16 / sizeof(T)];
    float by_key[2][kMain][kTile];                     // the head's terms of q and k
    float nq[kTile], nk[kTile];                        // q.dq and k.dk but for those
  };
  template <typename P> static constexpr bool kFits = P::kTeams * sizeof(Shared<P>) <= 227 * 1024;
  static_assert(kFits<Plan<1, false>>, "a block's shared memory");
};

// Rows of 16 tokens lie 32 bytes apart, their halves swapped in every other four rows: eight rows of
// 16 bytes, as ldmatrix reads them, are in all banks.
__device__ __forceinline__ int swap8(int row, int token) { return token ^ ((row & 4) << 1); }

__device__ __forceinline__ float quad_sum(float v) {   // over a row's four lanes
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
template <int N, int R, int P> __device__ __forceinline__ void put_planes(bf16 (&m)[N][R][P], int i, int j, const uint32_t (&p)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) *reinterpret_cast<uint32_t*>(&m[n][i][j]) = p[n];
}
// A fragment's tiles (rows i .. i + 15, columns j .. j + 15) to rows of m; of w and z with swap8.
template <int N, int NF, int R, int P> __device__ __forceinline__ void put_frag(bf16 (&m)[N][R][P], int i, int j, const Frag<NF>& f) {
  const int lane = threadIdx.x & 31;
  const uint32_t at = smem_of(&m[0][i + (lane & 15)][j + ((lane & 16) >> 1)]);
#pragma unroll
  for (int n = 0; n < N; ++n) stsm4(at + n * R * P * 2, f.r[n]);
}
template <int N, int NF, int R> __device__ __forceinline__ void put_tokens(bf16 (&m)[N][R][kTile], int i, const Frag<NF>& f) {
  const int lane = threadIdx.x & 31, r = lane & 15;
  const uint32_t at = smem_of(&m[0][i + r][swap8(r, (lane & 16) >> 1)]);
#pragma unroll
  for (int n = 0; n < N; ++n) stsm4(at + n * R * kTile * 2, f.r[n]);
}
// Addresses of ldmatrix in such rows, of a left operand's columns (a_cols) and a right one's (at_cols).
__device__ __forceinline__ uint32_t tokens_a(int lane) {
  const int r = ((lane & 16) >> 1) + (lane & 7);
  return (r * kTile + swap8(r, lane & 8)) * 2;
}
__device__ __forceinline__ uint32_t tokens_b(int lane) {
  const int r = lane & 15;
  return (r * kTile + swap8(r, (lane & 16) >> 1)) * 2;
}
// A warp's 16 x 16 of `out` (rows tokens) to the first n rows of memory, `cols` of its columns.
template <typename T, int P>
__device__ __forceinline__ void put_rows(T* to, int64_t stride, const T (&out)[kTile][P], int n, int cols, bool pieces) {
  const int lane = threadIdx.x & 31;
  if (pieces) {
    constexpr int V = kVec16<T>;
    for (int j = lane; j < n * (16 / V); j += 32) {
      const int r = j / (16 / V), c = j % (16 / V) * V;
      if (c < cols) *reinterpret_cast<uint4*>(to + r * stride + c) = *reinterpret_cast<const uint4*>(&out[r][c]);
    }
  } else {
    for (int j = lane; j < n * 16; j += 32)
      if (j % 16 < cols) to[j / 16 * stride + j % 16] = out[j / 16][j % 16];
  }
}

template <typename T, int DK, typename P> __global__ void __launch_bounds__(P::kThreads) delta_backward(DeltaArgs a, int splits) {
  using B = Backward<T, DK>;
  constexpr int NT = B::NT, NI = B::NI, NS = B::NS, kSteps = DK / 16, kStages = P::kStages, kTeams = P::kTeams;
  using Keys = typename B::Keys;
  using Values = typename B::Values;
  extern __shared__ __align__(16) char smem[];
  // Main warps first (warp w of every team, and of the chain and the keys, on the same quarter of the SM:
  // warps of the same task then run the same instructions at the same time), then the ones that
  // make chunks ready, then those of the matrices.
  enum { kFollow, kPrepare, kSquares };
  int warp = threadIdx.x >> 5, team, role;
  if (warp < kTeams * P::kAll) {
    role = kFollow;
    team = warp / P::kAll;
    warp %= P::kAll;
  } else if (warp < kTeams * (P::kAll + kPrep)) {
    role = kPrepare;
    team = (warp - kTeams * P::kAll) / kPrep;
    warp = (warp - kTeams * P::kAll) % kPrep;
  } else {
    role = kSquares;
    team = warp - kTeams * (P::kAll + kPrep);
  }
  const int64_t items = static_cast<int64_t>(a.batch) * a.heads * splits, item = static_cast<int64_t>(blockIdx.x) * kTeams + team;
  if (item >= items) return;
  auto& sh = reinterpret_cast<typename B::template Shared<P>*>(smem)[team];
  const int bars = 1 + team * P::kBars;
  const int block = static_cast<int>(item % splits), bh = static_cast<int>(item / splits), bi = bh / a.heads, h = bh % a.heads, gr = h / (a.heads / a.groups);
  const int lane = threadIdx.x & 31, row = lane >> 2, col = (lane & 3) * 2;
  const int vb = block * kValues, mine = min(kValues, a.values - vb);
  auto length_of = [&](int b) { return a.lengths ? max(0, min(a.lengths[b], a.length)) : a.length; };
  const int length = length_of(bi);
  const int tiles = (a.length + kTile - 1) / kTile, count = (length + kTile - 1) / kTile;
  const int64_t row0 = static_cast<int64_t>(bi) * a.length;
  const T* dt = static_cast<const T*>(a.dt) + bi * a.dt_b + h;
  const T* gb = static_cast<const T*>(a.b) + bi * a.b_b + h;
  const float rate = rate_at(a.A, h), bias = a.bias ? a.bias[h] : 0.0f;

  if (role == kPrepare) {
    const int w = warp, pitch = a.keys + kTile;
    const T* q = static_cast<const T*>(a.q) + bi * a.q_b + gr * a.q_g;
    const T* k = static_cast<const T*>(a.k) + bi * a.k_b + gr * a.k_g;
    const T* dout = static_cast<const T*>(a.dout) + bi * a.do_b + h * a.do_h + vb;
    Marks look{a.reset ? a.reset + static_cast<int64_t>(bi) * a.length : nullptr, length, 0u};
    // resets and gates a tile of this warp's ahead of the rest
    T raw_dt = from_f<T>(0.0f), raw_b = raw_dt;
    auto ahead = [&](int tile) {
      look.look(tile * kTile);
      if (tile >= 0 && lane < kTile && tile * kTile + lane < length) {
        raw_dt = dt[(tile * kTile + lane) * a.dt_t];
        raw_b = gb[(tile * kTile + lane) * a.b_t];
      }
    };
    ahead(count - 1 - w);
    for (int i = w; i < count; i += kPrep) {
      const int at = i % kStages;
      typename B::Stage& st = sh.stage[at];
      const int tile = count - 1 - i, end = min(kTile, length - tile * kTile);
      const unsigned marks = look.get();
      const float now_dt = to_f(raw_dt), now_b = to_f(raw_b);
      ahead(tile - kPrep);
      if (i >= kStages) bar_sync(bars + P::kFree + at, P::kAtFree);
      const float* saved = a.saved + (((static_cast<int64_t>(bi) * tiles + tile) * a.heads + h) * a.values + vb) * pitch;
      bool bad = false;
      auto fetch = [&](int from, int n, unsigned mark, float x, float y) {
        const int t0 = tile * kTile + from;
        Keys::load(st.tk, k + t0 * a.k_t, a.k_t, n, a.keys, a.piece_k == 16);
        Keys::load(st.tq, q + t0 * a.q_t, a.q_t, n, a.keys, a.piece_k == 16);
        Values::load(st.tdo, dout + t0 * a.do_t, a.do_t, n, mine, a.piece_v == 16);
        cp_async_commit();
        Gate e{};
        if (lane < n) e = gate_of(x, y, bias, rate);
        decays(st.c, e.g, e.beta, mark);
        if (lane == 0) {
          st.t0 = t0;
          st.n = n;
          st.marks = mark;
          st.more = 0;
        }
        bad = __any_sync(0xffffffffu, fmaf(e.g, 0.0f, e.beta * 0.0f) != 0.0f);
        cp_async_wait<0>();
        __syncwarp();
      };
      auto ready = [&](unsigned mark) {
        prepare<T, DK, true>(st.c, sh.scratch[w], &st.wide, st.tk, st.tq, mark, a.scale, a.unit);
        bar_arrive(bars + P::kReady + at, P::kAtReady);
      };
      fetch(0, end, marks, now_dt, now_b);
      bool split = false;
      if (marks & ~1u) {
        float w_bad = 0.0f;                            // a value that is not finite makes its token's W so
        for (int x = lane; x < mine * end; x += 32) w_bad = fmaf(saved[x / end * pitch + a.keys + x % end], 0.0f, w_bad);
        split = bad || __any_sync(0xffffffffu, w_bad != 0.0f) || not_finite(st.tk, Keys::kPitch, DK, end) ||
                not_finite(st.tq, Keys::kPitch, DK, end) || not_finite(st.tdo, Values::kPitch, kValues, end);
      }
      if (!split) {
        ready(marks);
        continue;
      }
      for (int to = end; to > 0;) {                    // the last episode first
        const int from = 31 - __clz((marks | 1u) & ((1u << to) - 1u));
        const unsigned mark = (marks >> from) & 1u;
        if (to < end) bar_sync(bars + P::kFree + at, P::kAtFree);
        const int token = tile * kTile + from + lane;
        const bool on = from + lane < to;
        fetch(from, to - from, mark, on ? to_f(dt[token * a.dt_t]) : 0.0f, on ? to_f(gb[token * a.b_t]) : 0.0f);
        if (lane == 0) st.more = from > 0;
        ready(mark);
        to = from;
      }
    }
    return;
  }

  if (role == kSquares) {
    // the matrices and gates of 16 x 16
    const int64_t g_t = static_cast<int64_t>(a.heads) * splits, g_at = row0 * g_t + static_cast<int64_t>(h) * splits + block;
    double sum_a = 0.0, sum_bias = 0.0;
    for (int i = 0, more = 0, unit = 0; i < count; i += more ? 0 : 1, ++unit) {
      const int at = i % kStages, copy = unit % P::kCopies;
      typename B::Stage& st = sh.stage[at];
      const typename B::Chain& chain = sh.chain[copy];
      // the chunk was ready for the chain, which does not wait for this warp
      bar_sync(bars + P::kChain + copy, P::kAtChain);
      const int t0 = st.t0, n = st.n;
      const unsigned marks = st.marks;
      more = st.more;
      T raw_dt = from_f<T>(0.0f), raw_b = raw_dt;      // on their way until the end
      if (lane < n) {
        raw_dt = dt[(t0 + lane) * a.dt_t];
        raw_b = gb[(t0 + lane) * a.b_t];
      }
      // lane: row r, columns j0 .. j0 + 7 of Z W^T and dO W^T. By rows: sums of E's part of P, of M
      const int r = lane >> 1, j0 = (lane & 1) * 8;
      const float rqr = st.c.rq[r], rkr = st.c.rk[r];
      float row_p = 0.0f, row_m = 0.0f;
#pragma unroll
      for (int j = j0; j < j0 + 8; j += 4) {
        auto four = [](float (&x)[4], const float* from) { *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(from); };
        float zw[4] = {}, ow[4] = {}, bt[4], rk[4], d[4], p[4], m[4], ep[4], em[4], mz[4], pd[4], md[4];
#pragma unroll
        for (int x = 0; x < kMain; ++x) {
          float y[4];
          four(y, &chain.part[x].product[0][r][j]);
#pragma unroll
          for (int e = 0; e < 4; ++e) zw[e] += y[e];
          four(y, &chain.part[x].product[1][r][j]);
#pragma unroll
          for (int e = 0; e < 4; ++e) ow[e] += y[e];
        }
        four(bt, &st.c.beta[j]);
        four(rk, &st.c.rk[j]);
        four(d, &st.wide.d[r][j]);
        four(p, &st.wide.p[r][j]);
        four(m, &st.wide.m[r][j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = j + e;
          const bool one = d[e] != 0.0f;               // across a reset Z or W need not be finite
          const float dp = one && c <= r ? ow[e] * bt[e] : 0.0f, dm = one && c < r ? -zw[e] * bt[e] : 0.0f;
          ep[e] = dp * p[e];
          em[e] = dm * m[e];
          pd[e] = a.scale * dp * d[e];
          md[e] = dm * d[e];
          mz[e] = one && c < r ? m[e] * zw[e] : 0.0f;
          row_p += ep[e];
          row_m += em[e];
        }
        *reinterpret_cast<float4*>(&st.wide.p[r][j]) = make_float4(ep[0], ep[1], ep[2], ep[3]);
        *reinterpret_cast<float4*>(&st.wide.m[r][j]) = make_float4(em[0], em[1], em[2], em[3]);
        *reinterpret_cast<float4*>(&st.wide.d[r][j]) = make_float4(mz[0], mz[1], mz[2], mz[3]);
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          uint32_t y[NS];
          split2<NS>(pd[e] * rk[e], pd[e + 1] * rk[e + 1], y);
          put_planes(sh.x1, r, j + e, y);
          split2<NS>(pd[e] * rqr, pd[e + 1] * rqr, y);
          put_planes(sh.x2, r, j + e, y);
#pragma unroll
          for (int o = e; o < e + 2; ++o)
            if (j + o <= r) {                          // below the diagonal, and what it gives above it
              split2<NS>(md[o] * rk[o], md[o] * rkr, y);
#pragma unroll
              for (int x = 0; x < NS; ++x) {
                if (j + o < r) sh.x3[x][j + o][r] = __ushort_as_bfloat16(static_cast<unsigned short>(y[x] >> 16));
                sh.x3[x][r][j + o] = __ushort_as_bfloat16(static_cast<unsigned short>(y[x]));
              }
            }
        }
      }
      row_p += __shfl_xor_sync(0xffffffffu, row_p, 1);
      row_m += __shfl_xor_sync(0xffffffffu, row_m, 1);
      __syncwarp();
      // lane: column and token c; columns from below
      const int c = lane & 15;
      float wd = 0.0f, f = 0.0f, inner = 0.0f;
#pragma unroll
      for (int x = 0; x < kMain; ++x) {
        wd += chain.by_value[x][0][c];
        f += chain.by_value[x][1][c];
        inner += chain.inner[x];
      }
      float column = 0.0f, below = 0.0f, dbeta = wd;
#pragma unroll
      for (int y = kTile - 1; y >= 0; --y) {
        const float ep = st.wide.p[y][c], em = st.wide.m[y][c];
        dbeta -= st.wide.d[y][c];
        column += ep + em;
        if (y > c) below += ep + em;
        __syncwarp();
        if (lane < kTile) st.wide.p[y][c] = y > c ? below : 0.0f;
      }
      row_p = __shfl_sync(0xffffffffu, row_p, 2 * c);
      row_m = __shfl_sync(0xffffffffu, row_m, 2 * c);
      if (lane < kTile) {
        sh.nq[c] = row_p;
        sh.nk[c] = f + row_m + column;
      }
      bar_sync(bars + P::kMatrices, P::kAtMatrices);
      if constexpr (P::kApart) bar_arrive(bars + P::kPlace + copy, P::kAtChain);
      float e = 0.0f;
#pragma unroll
      for (int x = 0; x < kMain; ++x) e += sh.by_key[0][x][c] + sh.by_key[1][x][c];
      float dg = marks ? 0.0f : st.c.head[kTile - 1] * inner;
#pragma unroll
      for (int j = 0; j < kTile; ++j) {
        const float ej = __shfl_sync(0xffffffffu, e, j), fj = __shfl_sync(0xffffffffu, f, j);
        dg += j >= c ? ej : fj + st.wide.p[c][j];
      }
      if (lane < n) {
        const Gate gate = gate_of(to_f(raw_dt), to_f(raw_b), bias, rate);
        const float back = dg * rate * sigmoid(gate.pre), b_back = dbeta * gate.beta * (1.0f - gate.beta);
        const int64_t to = g_at + (t0 + lane) * g_t;
        if (a.part_g) {
          *reinterpret_cast<float2*>(a.part_g + 2 * to) = make_float2(back, b_back);
        } else {
          static_cast<T*>(a.ddt)[to] = from_f<T>(back);
          static_cast<T*>(a.db)[to] = from_f<T>(b_back);
        }
        sum_a += static_cast<double>(dg) * gate.delta;
        sum_bias += back;
      }
      __syncwarp();
      bar_arrive(bars + P::kFree + at, P::kAtFree);
    }
    for (int o = 16; o; o >>= 1) {
      sum_a += __shfl_xor_sync(0xffffffffu, sum_a, o);
      sum_bias += __shfl_xor_sync(0xffffffffu, sum_bias, o);
    }
    if (lane == 0) {
      const int64_t to = item * 2;
      a.part_h[to] = static_cast<float>(sum_a);
      a.part_h[to + 1] = static_cast<float>(sum_bias);
    }
    for (int t = length + lane; t < a.length; t += 32) {
      const int64_t to = g_at + t * g_t;
      if (a.part_g) *reinterpret_cast<float2*>(a.part_g + 2 * to) = make_float2(0.0f, 0.0f);
      else static_cast<T*>(a.ddt)[to] = static_cast<T*>(a.db)[to] = from_f<T>(0.0f);
    }
    return;
  }

  // gradients are dense; parts of dq and dk by heads and blocks
  const int qk_heads = a.part_q ? a.heads * splits : a.groups, qk_head = a.part_q ? h * splits + block : gr;
  const int64_t qk_t = static_cast<int64_t>(qk_heads) * a.keys, qk_at = (row0 * qk_heads + qk_head) * a.keys;
  const int64_t v_t = static_cast<int64_t>(a.heads) * a.values;
  T* dv = static_cast<T*>(a.dv) + (row0 * a.heads + h) * a.values + vb;
  const bool pieces_v = a.values * sizeof(T) % 16 == 0, pieces_k = a.keys * sizeof(T) % 16 == 0;
  const bool follows = !P::kApart || warp < kMain, keys = !P::kApart || warp >= kMain;       // the chain, the keys
  warp %= kMain;
  const int vl = warp * 16, c0 = warp * B::kColumns, vsteps = (mine + 15) / 16;
  const bool by_v = vl < mine, by_k = c0 < DK && c0 < a.keys;
  constexpr int kPairs = B::kColumns / 16;
  float* dstate = a.dstate ? a.dstate + ((static_cast<int64_t>(bi) * a.heads + h) * a.values + vb) * a.keys : nullptr;
  const float* dfinal = a.dfinal ? a.dfinal + ((static_cast<int64_t>(bi) * a.heads + h) * a.values + vb) * a.keys : nullptr;

  // S and W of the tiles from the last on, by the chain its own rows, on their way while the tile before is finished
  const int pitch = a.keys + kTile;
  const bool pieces_s = a.keys % 4 == 0;
  const int64_t saved_tile = static_cast<int64_t>(a.heads) * a.values * pitch;
  const float* saved = a.saved + (static_cast<int64_t>(bi) * tiles * a.heads + h) * a.values * pitch + static_cast<int64_t>(vb + vl) * pitch;
  auto take = [&](int copy, int tile, bool w_too) {
    if (!by_v) return;
    const float* from = saved + tile * saved_tile;
    load_rows(&sh.s[copy][vl][0], B::kPitchS, 16, DK, from, pitch, min(16, mine - vl), a.keys, pieces_s);
    if (w_too) load_rows(&sh.saved_w[vl][0], kMat, 16, kTile, from + a.keys, pitch, min(16, mine - vl), kTile, pieces_s);
    cp_async_commit();
  };

  // d[n]: rows vl + row, + 8; keys 8 n + col, + 1
  float d[DK / 8][4];
#pragma unroll
  for (int n = 0; n < DK / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = vl + row + (e >> 1) * 8, kc = 8 * n + col + (e & 1);
      d[n][e] = dfinal && r < mine && kc < a.keys ? dfinal[r * a.keys + kc] : 0.0f;
    }
  // what a warp without values or columns leaves
  if (follows)
    for (int copy = 0; copy < P::kCopies; ++copy) {
      for (int i = lane; i < 2 * kTile; i += 32) (&sh.chain[copy].by_value[warp][0][0])[i] = 0.0f;
      if (lane == 0) sh.chain[copy].inner[warp] = 0.0f;
    }
  if (P::kApart && !by_v) {
    for (int copy = 0; copy < P::kCopies; ++copy) {
      auto zero = [&](auto& rows) {
        for (int n = 0; n < NI; ++n)
          for (int x = lane; x < 16 * kTile; x += 32) (&rows[n][vl][0])[x] = bf16(0.0f);
      };
      if (follows) {
        zero(sh.chain[copy].w);
        zero(sh.chain[copy].z);
        for (int n = 0; n < NS; ++n)
          for (int x = lane; x < 16 * B::kPitchD; x += 32) (&sh.chain[copy].d[n][vl][0])[x] = bf16(0.0f);
      } else {
        for (int x = lane; x < 16 * B::kPitchS; x += 32) (&sh.s[copy][vl][0])[x] = 0.0f;  // copy 1 is the keys'
      }
    }
  }
  if (keys && lane < kTile) sh.by_key[0][warp][lane] = sh.by_key[1][warp][lane] = 0.0f;
  __syncwarp();

  // tiles that all teams of the block have
  int common = 0;
  if constexpr (kTeams > 1) {
    const int64_t other = item ^ 1;
    if (other < items) common = min(count, (length_of(static_cast<int>(other / splits) / a.heads) + kTile - 1) / kTile);
  }

  auto follow_chain = [&](const typename B::Stage& st, typename B::Chain& chain, int copy) {
    const Chunk<T, NI>& c = st.c;
    const int t0 = st.t0, n = st.n;
    const unsigned marks = st.marks;
    const bool fresh = marks & 1u;                     // no token sees S
    if (by_v) {
      // K dS^T (rows values, columns tokens), <dS, S>; dS's planes to shared memory
      float ds[2][4] = {}, inner = 0.0f;
      const uint32_t ka = smem_of(st.tk) + at_rows(lane, Keys::kPitch);
#pragma unroll
      for (int x = 0; x < kSteps; ++x) {
        Frag<NI> f;
        f.from(d[2 * x], d[2 * x + 1]);
        uint32_t b[NT][4];
        load_planes<NT, false>(b, ka + x * 32, Keys::kPlane * 2);
        mma_planes<NI, NT>(ds[0], ds[1], f.r, b);
        put_frag(chain.d, vl, 16 * x, f);
        if (!marks)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 s = *reinterpret_cast<const float2*>(&sh.s[0][vl + row + 8 * e][16 * x + 8 * t + col]);
              inner = fmaf(s.x, d[2 * x + t][2 * e], fmaf(s.y, d[2 * x + t][2 * e + 1], inner));
            }
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) inner += __shfl_xor_sync(0xffffffffu, inner, o);
      if (lane == 0) chain.inner[warp] = inner;
      // dU, Z
      float w[2][4], du[2][4] = {}, z[2][4] = {};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 y = *reinterpret_cast<const float2*>(&sh.saved_w[vl + row + 8 * e][8 * t + col]);
          w[t][2 * e] = y.x;
          w[t][2 * e + 1] = y.y;
        }
      if (n < kTile)                                   // a part of the tile
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tok = 8 * t + col + (e & 1);
            w[t][e] = tok < n ? sh.saved_w[vl + row + (e >> 1) * 8][t0 % kTile + tok] : 0.0f;
          }
      {
        uint32_t o[NT][4], b[NI][4];
        load_planes<NT, true>(o, smem_of(st.tdo) + a_cols(lane, Values::kPitch) + vl * 2, Values::kPlane * 2);
        load_planes<NI, true>(b, smem_of(c.p) + at_cols(lane, kSide), kTile * kSide * 2);
        mma_planes<NT, NI>(du[0], du[1], o, b);
        if (marks)                                     // no token before the last reset gets of dS
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (marks >> (t * 8 + col + (e & 1) + 1)) ds[t][e] = 0.0f;
        float x[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float2 tail = *reinterpret_cast<const float2*>(&c.tail_k[t * 8 + col]), beta = *reinterpret_cast<const float2*>(&c.beta[t * 8 + col]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ds[t][e] *= e & 1 ? tail.y : tail.x;
            du[t][e] += ds[t][e];
            x[t][e] = (e & 1 ? beta.y : beta.x) * du[t][e];
          }
        }
        Frag<NI> f;
        load_planes<NI, true>(b, smem_of(c.inv) + at_cols(lane, kSide), kTile * kSide * 2);
        // A gradient of the state that is not finite reaches the last episode's tokens alone: with
        // others in the chunk, theirs is a sum without them.
        float bad = 0.0f;
        if (marks & ~1u) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) bad = fmaf(x[t][e], 0.0f, bad);
        }
        if (!__any_sync(0xffffffffu, bad != 0.0f)) {
          f.from(x[0], x[1]);
          mma_planes<NI, NI>(z[0], z[1], f.r, b);
        } else {
          for (int last = 0; last < 2; ++last) {
            float y[2][4], to[2][4] = {};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) y[t][e] = (marks >> (t * 8 + col + (e & 1) + 1) == 0) == (last != 0) ? x[t][e] : 0.0f;
            f.from(y[0], y[1]);
            mma_planes<NI, NI>(to[0], to[1], f.r, b);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((marks >> (t * 8 + col + (e & 1) + 1) == 0) == (last != 0)) z[t][e] = to[t][e];
          }
        }
        f.from(z[0], z[1]);
        put_tokens(chain.z, vl, f);
        f.from(w[0], w[1]);
        put_tokens(chain.w, vl, f);
      }
      // sums over the warp's values, by tokens: halves of the sums change lanes until each has one token's
      {
        T (&so)[kTile][16 + 16 / sizeof(T)] = *(P::kApart ? &sh.dv[P::kApart ? copy * kMain + warp : 0] : &chain.part[warp].out);
        float sum[2][2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int tok = t * 8 + col + e;
            sum[0][t][e] = fmaf(w[t][e], du[t][e], w[t][e + 2] * du[t][e + 2]);
            sum[1][t][e] = fmaf(w[t][e], ds[t][e], w[t][e + 2] * ds[t][e + 2]);
            so[tok][row] = from_f<T>(z[t][e]);
            so[tok][row + 8] = from_f<T>(z[t][e + 2]);
          }
        const bool t1 = lane & 16, e1 = lane & 8;
        const int tok = (t1 ? 8 : 0) + col + (e1 ? 1 : 0);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float y[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) y[e] = (t1 ? sum[x][1][e] : sum[x][0][e]) + __shfl_xor_sync(0xffffffffu, t1 ? sum[x][0][e] : sum[x][1][e], 16);
          float one = (e1 ? y[1] : y[0]) + __shfl_xor_sync(0xffffffffu, e1 ? y[0] : y[1], 8);
          one += __shfl_xor_sync(0xffffffffu, one, 4);
          if (!(lane & 4)) chain.by_value[warp][x][tok] = x == 1 ? c.beta[tok] * one : one;
        }
        if constexpr (!P::kApart) {
          __syncwarp();
          put_rows(dv + t0 * v_t + vl, v_t, so, n, mine - vl, pieces_v);
        }
      }
      __syncwarp();
      // the warp's part of Z W^T and dO W^T
      {
        uint32_t b[NI][4], x[NI][4], o[NT][4];
        float zw[2][4] = {}, ow[2][4] = {};
        load_planes<NI, true>(b, smem_of(chain.w) + tokens_b(lane) + vl * kTile * 2, kValues * kTile * 2);
        load_planes<NI, true>(x, smem_of(chain.z) + tokens_a(lane) + vl * kTile * 2, kValues * kTile * 2);
        mma_planes<NI, NI>(zw[0], zw[1], x, b);
        load_planes<NT, false>(o, smem_of(st.tdo) + a_rows(lane, Values::kPitch) + vl * 2, Values::kPlane * 2);
        mma_planes<NT, NI>(ow[0], ow[1], o, b);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            *reinterpret_cast<float2*>(&chain.part[warp].product[0][row + 8 * e][8 * t + col]) = make_float2(zw[t][2 * e], zw[t][2 * e + 1]);
            *reinterpret_cast<float2*>(&chain.part[warp].product[1][row + 8 * e][8 * t + col]) = make_float2(ow[t][2 * e], ow[t][2 * e + 1]);
          }
      }
      // dS one chunk on
      if (fresh) {
#pragma unroll
        for (int x = 0; x < DK / 8; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[x][e] = 0.0f;
      } else {
        float x[2][4];
        if (marks) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (marks & ((2u << (t * 8 + col + (e & 1))) - 1u)) z[t][e] = 0.0f;
#pragma unroll
          for (int y = 0; y < DK / 8; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[y][e] = 0.0f;
        } else {
          const float end = c.head[kTile - 1];
#pragma unroll
          for (int y = 0; y < DK / 8; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[y][e] *= end;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float2 hk = *reinterpret_cast<const float2*>(&c.head_k[t * 8 + col]), hq = *reinterpret_cast<const float2*>(&c.head_q[t * 8 + col]);
          const bf16* from = st.tdo + (t * 8 + col) * Values::kPitch + vl + row;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            z[t][e] *= e & 1 ? -hk.y : -hk.x;
            x[t][e] = (e & 1 ? hq.y : hq.x) * tile_at<T>(from, Values::kPlane, (e & 1) * Values::kPitch + (e >> 1) * 8);
          }
        }
        Frag<NI> fz, fo;
        fz.from(z[0], z[1]);
        fo.from(x[0], x[1]);
        const uint32_t kt = smem_of(st.tk) + at_cols(lane, Keys::kPitch), qt = smem_of(st.tq) + at_cols(lane, Keys::kPitch);
#pragma unroll
        for (int y = 0; y < kSteps; ++y) {
          uint32_t b[NT][4];
          load_planes<NT, true>(b, kt + y * 32, Keys::kPlane * 2);
          mma_planes<NI, NT>(d[2 * y], d[2 * y + 1], fz.r, b);
          load_planes<NT, true>(b, qt + y * 32, Keys::kPlane * 2);
          mma_planes<NI, NT>(d[2 * y], d[2 * y + 1], fo.r, b);
        }
      }
    }
    else
      for (int x = lane; x < 2 * kTile * kMat; x += 32) (&chain.part[warp].product[0][0][0])[x] = 0.0f;
  };

  auto follow_keys = [&](const typename B::Stage& st, typename B::Chain& chain, int i, int copy) {
    const Chunk<T, NI>& c = st.c;
    const int t0 = st.t0, n = st.n;
    const unsigned marks = st.marks;
    const bool fresh = marks & 1u;                     // no token sees S
    const int more = st.more;
    // by keys: rows tokens, columns c0 ..
    float aq[kPairs][2][4] = {}, ak[kPairs][2][4] = {};
    if (P::kApart && by_v) put_rows(dv + t0 * v_t + vl, v_t, sh.dv[P::kApart ? copy * kMain + warp : 0], n, mine - vl, pieces_v);
    if (by_k) {
      float as[kPairs][2][4] = {};
      // apart, all of a block's values unrolled, those that it does not have as zeros (4% at
      // 2x4096x16x64x64); teams of two are bound by fetching instructions
#pragma unroll (P::kApart ? kMain : 1)
      for (int x = 0; x < (P::kApart ? kMain : vsteps); ++x) {
        uint32_t o[NT][4], z[NI][4], w[NS][4];
        load_planes<NS, true>(w, smem_of(chain.w) + tokens_a(lane) + x * 16 * kTile * 2, kValues * kTile * 2);
        if (!fresh) {
          load_planes<NT, false>(o, smem_of(st.tdo) + a_rows(lane, Values::kPitch) + x * 32, Values::kPlane * 2);
          load_planes<NI, true>(z, smem_of(chain.z) + tokens_a(lane) + x * 16 * kTile * 2, kValues * kTile * 2);
        }
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
          uint32_t b[NS][4];
          load_planes<NS, true>(b, smem_of(chain.d) + at_cols(lane, B::kPitchD) + (x * 16 * B::kPitchD + c0 + 16 * p) * 2,
                                kValues * B::kPitchD * 2);
          mma_planes<NS, NS>(as[p][0], as[p][1], w, b);
          if (!fresh) {
            uint32_t s[NI][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float* from = &sh.s[P::kCopies - 1][16 * x + (e & 1) * 8 + col][c0 + 16 * p + (e >> 1) * 8 + row];
              uint32_t y[NI];
              split2<NI>(from[0], from[B::kPitchS], y);
#pragma unroll
              for (int m = 0; m < NI; ++m) s[m][e] = y[m];
            }
            mma_planes<NT, NI>(aq[p][0], aq[p][1], o, s);
            mma_planes<NI, NI>(ak[p][0], ak[p][1], z, s);    // all planes: the decays' gradients are made of it
          }
        }
      }
      float e0[2] = {}, e1[2] = {}, hq[2], hk[2], tk[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int tok = row + 8 * e;
        hk[e] = -c.head[tok];
        hq[e] = a.scale * c.head[tok];
        tk[e] = c.tail[tok] * c.beta[tok];
        if (marks) {
#pragma unroll
          for (int p = 0; p < kPairs; ++p)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int x = 2 * e; x < 2 * e + 2; ++x) {
                if (marks & ((2u << tok) - 1u)) aq[p][t][x] = ak[p][t][x] = 0.0f;
                if (marks >> (tok + 1)) as[p][t][x] = 0.0f;
              }
        }
      }
#pragma unroll
      for (int p = 0; p < kPairs; ++p)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float q0, q1;
            tile_pair<T>(st.tq, Keys::kPlane, (row + 8 * e) * Keys::kPitch + c0 + 16 * p + t * 8 + col, q0, q1);
            float k0, k1;
            tile_pair<T>(st.tk, Keys::kPlane, (row + 8 * e) * Keys::kPitch + c0 + 16 * p + t * 8 + col, k0, k1);
            e1[e] = fmaf(ak[p][t][2 * e], k0, fmaf(ak[p][t][2 * e + 1], k1, e1[e]));
#pragma unroll
            for (int x = 2 * e; x < 2 * e + 2; ++x) {
              aq[p][t][x] *= hq[e];
              ak[p][t][x] = fmaf(hk[e], ak[p][t][x], tk[e] * as[p][t][x]);
              e0[e] = fmaf(aq[p][t][x], x & 1 ? q1 : q0, e0[e]);
            }
          }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        e0[e] = quad_sum(e0[e]);
        if ((lane & 3) == 0) sh.by_key[0][warp][row + 8 * e] = e0[e] * c.rq[row + 8 * e];
        e1[e] = quad_sum(e1[e]);
        if ((lane & 3) == 0) sh.by_key[1][warp][row + 8 * e] = e1[e] * hk[e] * c.rk[row + 8 * e];
      }
    }
    bar_sync(bars + P::kMatrices, P::kAtMatrices);     // S is read no more
    if constexpr (P::kApart) bar_arrive(bars + P::kPlace + copy, P::kAtChain);
    if (!more && i + 1 < count) take(P::kCopies - 1, count - 2 - i, !P::kApart);

    if (by_k) {
      float nq[2] = {}, nk[2] = {}, rq[2], rk[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        rq[e] = c.rq[row + 8 * e];
        rk[e] = c.rk[row + 8 * e];
        if (!a.unit) continue;
        nq[e] = sh.nq[row + 8 * e];
#pragma unroll
        for (int x = 0; x < kMain; ++x) {
          nq[e] += sh.by_key[0][x][row + 8 * e];
          nk[e] += sh.by_key[1][x][row + 8 * e];
        }
        nq[e] *= rq[e];                                // what takes the part along q out of dq, for q itself
        nk[e] = (nk[e] + sh.nk[row + 8 * e]) * rk[e];
      }
      uint32_t x1[NS][4], x2[NS][4], x3[NS][4];
      load_planes<NS, false>(x1, smem_of(sh.x1) + a_rows(lane, kSide), kTile * kSide * 2);
      load_planes<NS, true>(x2, smem_of(sh.x2) + a_cols(lane, kSide), kTile * kSide * 2);
      load_planes<NS, false>(x3, smem_of(sh.x3) + a_rows(lane, kSide), kTile * kSide * 2);
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
        const int cp = c0 + 16 * p;
        uint32_t b[NT][4];
        load_planes<NT, true>(b, smem_of(st.tk) + at_cols(lane, Keys::kPitch) + cp * 2, Keys::kPlane * 2);
        mma_planes<NS, NT>(aq[p][0], aq[p][1], x1, b);
        mma_planes<NS, NT>(ak[p][0], ak[p][1], x3, b);
        load_planes<NT, true>(b, smem_of(st.tq) + at_cols(lane, Keys::kPitch) + cp * 2, Keys::kPlane * 2);
        mma_planes<NS, NT>(ak[p][0], ak[p][1], x2, b);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int x = (row + 8 * e) * Keys::kPitch + cp + t * 8 + col;
            float q0, q1, k0, k1;
            tile_pair<T>(st.tq, Keys::kPlane, x, q0, q1);
            tile_pair<T>(st.tk, Keys::kPlane, x, k0, k1);
            aq[p][t][2 * e] = rq[e] * fmaf(-nq[e], q0, aq[p][t][2 * e]);
            aq[p][t][2 * e + 1] = rq[e] * fmaf(-nq[e], q1, aq[p][t][2 * e + 1]);
            ak[p][t][2 * e] = rk[e] * fmaf(-nk[e], k0, ak[p][t][2 * e]);
            ak[p][t][2 * e + 1] = rk[e] * fmaf(-nk[e], k1, ak[p][t][2 * e + 1]);
          }
        if (a.part_q) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int tok = row + (e >> 1) * 8, kc = cp + t * 8 + col + (e & 1);
              if (tok >= n || kc >= a.keys) continue;
              a.part_q[qk_at + (t0 + tok) * qk_t + kc] = aq[p][t][e];
              a.part_k[qk_at + (t0 + tok) * qk_t + kc] = ak[p][t][e];
            }
        } else {
          T (&so)[kTile][16 + 16 / sizeof(T)] = *(P::kApart ? &sh.out[P::kApart ? warp : 0] : &chain.part[warp].out);
#pragma unroll
          for (int turn2 = 0; turn2 < 2; ++turn2) {
            __syncwarp();
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float pair[2] = {turn2 ? ak[p][t][2 * e] : aq[p][t][2 * e], turn2 ? ak[p][t][2 * e + 1] : aq[p][t][2 * e + 1]};
                store_vec<T, 2>(&so[row + 8 * e][t * 8 + col], pair);
              }
            __syncwarp();
            put_rows(static_cast<T*>(turn2 ? a.dk : a.dq) + qk_at + t0 * qk_t + cp, qk_t, so, n, a.keys - cp, pieces_k);
          }
        }
      }
    }
  };

  if constexpr (P::kApart) {
    if (follows) {
      if (count > 0) take(0, count - 1, true);
      for (int i = 0, more = 0, unit = 0; i < count; i += more ? 0 : 1, ++unit) {
        const int at = i % kStages, copy = unit & 1;
        bar_sync(bars + P::kReady + at, P::kAtReady);
        more = sh.stage[at].more;
        if (unit > 1) bar_sync(bars + P::kPlace + copy, P::kAtChain);
        cp_async_wait<0>();
        __syncwarp();
        follow_chain(sh.stage[at], sh.chain[copy], copy);
        __syncwarp();
        bar_arrive(bars + P::kChain + copy, P::kAtChain);
        bar_arrive(bars + P::kFree + at, P::kAtFree);
        if (!more && i + 1 < count) take(0, count - 2 - i, true);
      }
    } else {
      if (count > 0) take(1, count - 1, false);
      for (int i = 0, more = 0, unit = 0; i < count; i += more ? 0 : 1, ++unit) {
        const int at = i % kStages, copy = unit & 1;
        cp_async_wait<0>();                            // this warp's rows of S; all warps' with the barrier
        bar_sync(bars + P::kChain + copy, P::kAtChain);
        more = sh.stage[at].more;
        follow_keys(sh.stage[at], sh.chain[copy], i, copy);
        __syncwarp();
        bar_arrive(bars + P::kFree + at, P::kAtFree);
      }
    }
  } else {
    if (count > 0) take(0, count - 1, true);
    for (int i = 0, more = 0, next = 1; i < count; i += more ? 0 : 1) {
      const int at = i % kStages;
      if (next && i < common) bar_sync(P::kEvery, kTeams * kMain * 32);
      bar_sync(bars + P::kReady + at, P::kAtReady);
      more = sh.stage[at].more;
      next = !more;
      cp_async_wait<0>();
      __syncwarp();
      follow_chain(sh.stage[at], sh.chain[0], 0);
      bar_sync(bars + P::kChain, P::kAtChain);
      follow_keys(sh.stage[at], sh.chain[0], i, 0);
      __syncwarp();
      bar_arrive(bars + P::kFree + at, P::kAtFree);
    }
  }

  if (dstate && by_v && follows) {
#pragma unroll
    for (int n = 0; n < DK / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = vl + row + (e >> 1) * 8, kc = 8 * n + col + (e & 1);
        if (r < mine && kc < a.keys) dstate[r * a.keys + kc] = d[n][e];
      }
  }
  // tokens that are not there
  if (!keys) return;
  for (int t = length + warp; t < a.length; t += kMain) {
    for (int x = lane; x < a.keys; x += 32) {
      const int64_t to = qk_at + t * qk_t + x;
      if (a.part_q) a.part_q[to] = a.part_k[to] = 0.0f;
      else static_cast<T*>(a.dq)[to] = static_cast<T*>(a.dk)[to] = from_f<T>(0.0f);
    }
    for (int x = lane; x < mine; x += 32) dv[t * v_t + x] = from_f<T>(0.0f);
  }
}

// dA and dbias: the sequences' in order.
__global__ void __launch_bounds__(32) delta_rates(DeltaArgs a, int splits) {
  const int h = blockIdx.x, lane = threadIdx.x;
  double x = 0.0, y = 0.0;
  for (int i = lane; i < a.batch * splits; i += 32) {
    const int64_t at = ((static_cast<int64_t>(i / splits) * a.heads + h) * splits + i % splits) * 2;
    x += a.part_h[at];
    y += a.part_h[at + 1];
  }
  for (int o = 16; o; o >>= 1) {
    x += __shfl_xor_sync(0xffffffffu, x, o);
    y += __shfl_xor_sync(0xffffffffu, y, o);
  }
  if (lane == 0) {
    a.dA[h] = static_cast<float>(x);
    if (a.dbias) a.dbias[h] = static_cast<float>(y);
  }
}

// Parts of dq and dk (of the value heads of a key head, of their blocks) and of ddt and db, summed in order.
template <typename T> __global__ void __launch_bounds__(256) delta_parts(DeltaArgs a, int splits) {
  const int64_t tokens = static_cast<int64_t>(a.batch) * a.length, total = tokens * a.groups * a.keys;
  const int parts = a.heads / a.groups * splits;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = first; i < total; i += step) {
    const int64_t head = i / a.keys, at = head * parts * a.keys + (i - head * a.keys);
    float x = 0.0f, y = 0.0f;
    for (int r = 0; r < parts; ++r) {
      x += a.part_q[at + static_cast<int64_t>(r) * a.keys];
      y += a.part_k[at + static_cast<int64_t>(r) * a.keys];
    }
    static_cast<T*>(a.dq)[i] = from_f<T>(x);
    static_cast<T*>(a.dk)[i] = from_f<T>(y);
  }
  if (a.part_g)
    for (int64_t i = first; i < tokens * a.heads; i += step) {
      float x = 0.0f, y = 0.0f;
      for (int r = 0; r < splits; ++r) {
        x += a.part_g[(i * splits + r) * 2];
        y += a.part_g[(i * splits + r) * 2 + 1];
      }
      static_cast<T*>(a.ddt)[i] = from_f<T>(x);
      static_cast<T*>(a.db)[i] = from_f<T>(y);
    }
}

template <typename T, int DK> int backward(const DeltaArgs& a, cudaStream_t s) {
  using B = Backward<T, DK>;
  const int splits = (a.values + kValues - 1) / kValues;
  // parts of as many elements as there are tokens: rows of none need no memory for them
  if (a.length > 0 && ((splits > 1 && !a.part_g) || (splits * a.heads != a.groups && !a.part_q))) return static_cast<int>(cudaErrorInvalidValue);
  const int64_t items = static_cast<int64_t>(a.batch) * a.heads * splits;
  auto go = [&](auto plan) {
    using P = decltype(plan);
    constexpr size_t bytes = P::kTeams * sizeof(typename B::template Shared<P>);
    if (const int e = allow_smem<delta_backward<T, DK, P>>(bytes)) return e;
    delta_backward<T, DK, P><<<static_cast<unsigned>((items + P::kTeams - 1) / P::kTeams), P::kThreads, bytes, s>>>(a, splits);
    return static_cast<int>(cudaGetLastError());
  };
  using One = Plan<1, false>;
  using Two = std::conditional_t<B::template kFits<Plan<2, false>>, Plan<2, false>, One>;
  using Apart = std::conditional_t<B::template kFits<Plan<1, true>>, Plan<1, true>, One>;
  if (const int e = items > 148 ? go(Two()) : go(Apart())) return e;            // see Plan
  delta_rates<<<a.heads, 32, 0, s>>>(a, splits);
  if (a.part_q && a.length > 0) {
    const int64_t grid = (static_cast<int64_t>(a.batch) * a.length * a.groups * a.keys + 255) / 256;
    delta_parts<T><<<grid < 148 * 16 ? static_cast<unsigned>(grid) : 148 * 16, 256, 0, s>>>(a, splits);
  }
  return static_cast<int>(cudaGetLastError());
}
template <typename T> int backward_by(const DeltaArgs& a, cudaStream_t s) {
  if (a.keys <= 32) return backward<T, 32>(a, s);
  if (a.keys <= 64) return backward<T, 64>(a, s);
  return backward<T, 128>(a, s);
}

}  // namespace

SURF_EXPORT int surf_delta_grad(const void* args, int dtype, void* stream) {
  const DeltaArgs& a = *static_cast<const DeltaArgs*>(args);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == kBf16 ? backward_by<bf16>(a, s) : backward_by<float>(a, s);
}
