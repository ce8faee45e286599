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
// A block for a sequence's value head. By values (a warp for 16 rows of S and dS, dS its
// accumulators): the chain from dS to dS. By keys (a warp for 16 columns): dq and dk, which sum
// over the values; the chain's results pass through shared memory as planes.
#include "delta.cuh"

namespace {

using namespace delta;

template <typename T, int DK> struct Backward {
  static constexpr int NI = Planes<T>::kInner;
  using Keys = Tile<T, DK>;
  using Values = Tile<T, 128>;
  static constexpr int kState = DK + 8;                // pitch of S and dS
  struct Shared {
    Chunk<T> c;
    alignas(16) bf16 tk[Keys::kSize], tq[Keys::kSize], tv[Values::kSize], tdo[Values::kSize];
    alignas(16) bf16 w[NI][128][kSide], z[NI][128][kSide];       // rows values, columns tokens
    alignas(16) bf16 x1[NI][kTile][kSide], x2[NI][kTile][kSide], x3[NI][kTile][kSide];
    float zw[kTile][kTile + 1], ow[kTile][kTile + 1];            // Z W^T and dO W^T
    float by_value[8][3][kTile];                       // of each warp: W.dU, head's and tail's terms of k
    float by_key[8][3][kTile];                         // head's term of q, q.dq, k.dk
    float inner[8];                                    // <dS, S>
    alignas(16) bf16 st[NI][128][kState];              // S, then dS
  };
  static constexpr size_t kBytes = sizeof(Shared);
  static_assert(kBytes <= 227 * 1024, "a block's shared memory");
};

__device__ __forceinline__ float quad_sum(float v) {   // over a row's four lanes
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float column_sum(float v) { // over a column's eight lanes
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

template <int N, int R> __device__ __forceinline__ void put_planes(bf16 (&m)[N][kTile][R], int i, int j, float x) {
  uint32_t p[N];
  split2<N>(x, 0.0f, p);
#pragma unroll
  for (int n = 0; n < N; ++n) m[n][i][j] = __ushort_as_bfloat16(static_cast<unsigned short>(p[n]));
}

template <typename T, int DK> __global__ void __launch_bounds__(256) delta_backward(DeltaArgs a) {
  constexpr int NT = Planes<T>::kToken, NI = Planes<T>::kInner, kSteps = DK / 16;
  using B = Backward<T, DK>;
  using Keys = typename B::Keys;
  using Values = typename B::Values;
  extern __shared__ __align__(16) char smem[];
  typename B::Shared& sh = *reinterpret_cast<typename B::Shared*>(smem);
  Chunk<T>& c = sh.c;
  const int bi = blockIdx.x / a.heads, h = blockIdx.x % a.heads, rep = a.heads / a.groups, gr = h / rep;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = lane >> 2, col = (lane & 3) * 2;
  const int vwarps = (a.values + 15) / 16, kwarps = (a.keys + 15) / 16, warps = blockDim.x / 32;
  const int v0 = warp * 16, k0 = warp * 16;
  const bool by_v = warp < vwarps, by_k = warp < kwarps;
  const int length = a.lengths ? max(0, min(a.lengths[bi], a.length)) : a.length;
  const uint8_t* reset = a.reset ? a.reset + static_cast<int64_t>(bi) * a.length : nullptr;
  const T* q = static_cast<const T*>(a.q) + bi * a.q_b + gr * a.q_g;
  const T* k = static_cast<const T*>(a.k) + bi * a.k_b + gr * a.k_g;
  const T* v = static_cast<const T*>(a.v) + bi * a.v_b + h * a.v_h;
  const T* dt = static_cast<const T*>(a.dt) + bi * a.dt_b + h;
  const T* gb = static_cast<const T*>(a.b) + bi * a.b_b + h;
  const T* dout = static_cast<const T*>(a.dout) + bi * a.do_b + h * a.do_h;
  // gradients are dense
  const int64_t row0 = static_cast<int64_t>(bi) * a.length;
  T* dq = static_cast<T*>(a.dq) + (row0 * a.groups + gr) * a.keys;
  T* dk = static_cast<T*>(a.dk) + (row0 * a.groups + gr) * a.keys;
  float* pq = a.part_q ? a.part_q + (row0 * a.heads + h) * a.keys : nullptr;
  float* pk = a.part_q ? a.part_k + (row0 * a.heads + h) * a.keys : nullptr;
  const int64_t qk_t = static_cast<int64_t>(pq ? a.heads : a.groups) * a.keys, v_t = static_cast<int64_t>(a.heads) * a.values;
  T* dv = static_cast<T*>(a.dv) + (row0 * a.heads + h) * a.values;
  T* ddt = static_cast<T*>(a.ddt) + row0 * a.heads + h;
  T* db = static_cast<T*>(a.db) + row0 * a.heads + h;
  const float rate = rate_at(a.A, h), bias = a.bias ? a.bias[h] : 0.0f;
  const int64_t head_size = static_cast<int64_t>(a.values) * a.keys;
  const int64_t head_at = (static_cast<int64_t>(bi) * a.heads + h) * head_size;
  const int tiles = (a.length + kTile - 1) / kTile;

  // d[n]: rows v0 + row, + 8; keys 8 n + col, + 1
  float d[DK / 8][4];
#pragma unroll
  for (int n = 0; n < DK / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = v0 + row + (e >> 1) * 8, kc = 8 * n + col + (e & 1);
      d[n][e] = a.dfinal && r < a.values && kc < a.keys ? a.dfinal[head_at + static_cast<int64_t>(r) * a.keys + kc] : 0.0f;
    }
  double sum_a = 0.0, sum_bias = 0.0;

  int t1 = length;                                     // the chunk's end
  while (t1 > 0) {
    // its start: the tile's, or the last reset before its end
    int t0 = (t1 - 1) / kTile * kTile;
    bool fresh = false;
    if (reset) {
      const unsigned cuts = __ballot_sync(0xffffffffu, lane < t1 - t0 && reset[t0 + lane]);
      if (cuts) {
        t0 += 31 - __clz(cuts);
        fresh = true;
      }
    }
    const int n = t1 - t0;
    const float* S = !fresh ? a.saved + ((static_cast<int64_t>(bi) * tiles + t0 / kTile) * a.heads + h) * head_size : nullptr;
    __syncthreads();
    Keys::load(sh.tk, k + t0 * a.k_t, a.k_t, n, a.keys, a.piece_k, threadIdx.x, blockDim.x);
    Keys::load(sh.tq, q + t0 * a.q_t, a.q_t, n, a.keys, a.piece_k, threadIdx.x, blockDim.x);
    Values::load(sh.tv, v + t0 * a.v_t, a.v_t, n, a.values, a.piece_v, threadIdx.x, blockDim.x);
    Values::load(sh.tdo, dout + t0 * a.do_t, a.do_t, n, a.values, a.piece_v, threadIdx.x, blockDim.x);
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    Gate gate{};
    if (warp == 0) {
      if (lane < n) gate = gate_of(to_f(dt[(t0 + lane) * a.dt_t]), to_f(gb[(t0 + lane) * a.b_t]), bias, rate);
      prepare<T, DK, true>(c, sh.tk, sh.tq, gate.g, gate.beta, a.scale, a.unit);
    }
    __syncthreads();

    float z[2][4] = {};
    if (by_v) {
      // K S^T and K dS^T (rows values, columns tokens), <dS, S>; S's planes to shared memory
      float sk[2][4] = {}, dsk[2][4] = {}, inner = 0.0f;
      const uint32_t ka = smem_of(sh.tk) + at_rows(lane, Keys::kPitch);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = v0 + row + (e >> 1) * 8, kc = 16 * i + 8 * t + col + (e & 1);
            s[t][e] = S && r < a.values && kc < a.keys ? S[static_cast<int64_t>(r) * a.keys + kc] : 0.0f;
            inner = fmaf(s[t][e], d[2 * i + t][e], inner);
          }
        uint32_t b[NT][4];
        load_planes<NT, false>(b, ka + i * 32, Keys::kPlane * 2);
        Frag<NI> f;
        f.from(s[0], s[1]);
        mma_planes<NI, NT>(sk[0], sk[1], f.r, b);
#pragma unroll
        for (int p = 0; p < NI; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint32_t*>(&sh.st[p][v0 + row + (e & 1) * 8][16 * i + (e >> 1) * 8 + col]) = f.r[p][e];
        f.from(d[2 * i], d[2 * i + 1]);
        mma_planes<NI, NT>(dsk[0], dsk[1], f.r, b);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) inner += __shfl_xor_sync(0xffffffffu, inner, o);
      if (lane == 0) sh.inner[warp] = inner;
      // W
      float w[2][4] = {}, du[2][4] = {};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = t * 8 + col + (e & 1), r = v0 + row + (e >> 1) * 8;
          sk[t][e] *= c.head[tok] * c.rk[tok];
          dsk[t][e] *= c.tail[tok] * c.rk[tok];
          z[t][e] = tile_at<T>(sh.tv, Values::kPlane, tok * Values::kPitch + r) - sk[t][e];
        }
      {
        Frag<NI> f;
        f.from(z[0], z[1]);
        uint32_t b[NI][4];
        load_planes<NI, false>(b, smem_of(c.inv) + at_rows(lane, kSide), kTile * kSide * 2);
        mma_planes<NI, NI>(w[0], w[1], f.r, b);
        f.from(w[0], w[1]);
#pragma unroll
        for (int p = 0; p < NI; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint32_t*>(&sh.w[p][v0 + row + (e & 1) * 8][(e >> 1) * 8 + col]) = f.r[p][e];
      }
      // dU, Z
      {
        uint32_t o[NT][4], b[NI][4];
        load_planes<NT, true>(o, smem_of(sh.tdo) + a_cols(lane, Values::kPitch) + v0 * 2, Values::kPlane * 2);
        load_planes<NI, true>(b, smem_of(c.p) + at_cols(lane, kSide), kTile * kSide * 2);
        mma_planes<NT, NI>(du[0], du[1], o, b);
        float x[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            du[t][e] += dsk[t][e];
            x[t][e] = c.beta[t * 8 + col + (e & 1)] * du[t][e];
            z[t][e] = 0.0f;
          }
        Frag<NI> f;
        f.from(x[0], x[1]);
        load_planes<NI, true>(b, smem_of(c.inv) + at_cols(lane, kSide), kTile * kSide * 2);
        mma_planes<NI, NI>(z[0], z[1], f.r, b);
        f.from(z[0], z[1]);
#pragma unroll
        for (int p = 0; p < NI; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint32_t*>(&sh.z[p][v0 + row + (e & 1) * 8][(e >> 1) * 8 + col]) = f.r[p][e];
      }
      // sums over the warp's values, by tokens; dv
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tok = t * 8 + col + e;
          const float wd = column_sum(fmaf(w[t][e], du[t][e], w[t][e + 2] * du[t][e + 2]));
          const float keep = column_sum(fmaf(z[t][e], sk[t][e], z[t][e + 2] * sk[t][e + 2]));
          const float send = column_sum(fmaf(w[t][e], dsk[t][e], w[t][e + 2] * dsk[t][e + 2]));
          if (row == 0) {
            sh.by_value[warp][0][tok] = wd;
            sh.by_value[warp][1][tok] = -keep;
            sh.by_value[warp][2][tok] = c.beta[tok] * send;
          }
          if (tok < n) {
            if (v0 + row < a.values) dv[(t0 + tok) * v_t + v0 + row] = from_f<T>(z[t][e]);
            if (v0 + row + 8 < a.values) dv[(t0 + tok) * v_t + v0 + row + 8] = from_f<T>(z[t][e + 2]);
          }
        }
    }
    __syncthreads();

    // by keys: S^T dO and S^T Z
    float aq[2][4] = {}, ak[2][4] = {};
    if (by_k) {
      for (int i = 0; i < vwarps; ++i) {
        uint32_t b[NI][4], o[NT][4], zz[NI][4];
        load_planes<NI, true>(b, smem_of(sh.st) + at_cols(lane, B::kState) + (i * 16 * B::kState + k0) * 2, 128 * B::kState * 2);
        load_planes<NT, false>(o, smem_of(sh.tdo) + a_rows(lane, Values::kPitch) + i * 32, Values::kPlane * 2);
        mma_planes<NT, NI>(aq[0], aq[1], o, b);
        load_planes<NI, true>(zz, smem_of(sh.z) + a_cols(lane, kSide) + i * 16 * kSide * 2, 128 * kSide * 2);
        mma_planes<NI, NI>(ak[0], ak[1], zz, b);
      }
      float e0 = 0.0f, e1 = 0.0f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = row + (e >> 1) * 8;
          aq[t][e] *= a.scale * c.head[tok];
          ak[t][e] *= -c.head[tok];
          const float x = aq[t][e] * tile_at<T>(sh.tq, Keys::kPlane, tok * Keys::kPitch + k0 + t * 8 + col + (e & 1));
          if (e < 2) e0 += x;
          else e1 += x;
        }
      e0 = quad_sum(e0);
      e1 = quad_sum(e1);
      if ((lane & 3) == 0) {
        sh.by_key[warp][0][row] = e0 * c.rq[row];
        sh.by_key[warp][0][row + 8] = e1 * c.rq[row + 8];
      }
    }
    // Z W^T and dO W^T
    for (int m = warp; m < 2; m += warps) {
      float r[2][4] = {};
      for (int i = 0; i < vwarps; ++i) {
        uint32_t b[NI][4];
        load_planes<NI, true>(b, smem_of(sh.w) + at_cols(lane, kSide) + i * 16 * kSide * 2, 128 * kSide * 2);
        if (m == 0) {
          uint32_t x[NI][4];
          load_planes<NI, true>(x, smem_of(sh.z) + a_cols(lane, kSide) + i * 16 * kSide * 2, 128 * kSide * 2);
          mma_planes<NI, NI>(r[0], r[1], x, b);
        } else {
          uint32_t x[NT][4];
          load_planes<NT, false>(x, smem_of(sh.tdo) + a_rows(lane, Values::kPitch) + i * 32, Values::kPlane * 2);
          mma_planes<NT, NI>(r[0], r[1], x, b);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) (m ? sh.ow : sh.zw)[row + (e >> 1) * 8][t * 8 + col + (e & 1)] = r[t][e];
    }
    __syncthreads();

    // dS to shared memory and one chunk on; a warp makes the 16 x 16 matrices of dq and dk
    if (by_v) {
      const float end = c.head[kTile - 1];
      Frag<NI> fz, fo;
      float x[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = t * 8 + col + (e & 1), r = v0 + row + (e >> 1) * 8;
          z[t][e] *= -c.head[tok] * c.rk[tok];
          x[t][e] = a.scale * c.head[tok] * c.rq[tok] * tile_at<T>(sh.tdo, Values::kPlane, tok * Values::kPitch + r);
        }
      fz.from(z[0], z[1]);
      fo.from(x[0], x[1]);
      const uint32_t kt = smem_of(sh.tk) + at_cols(lane, Keys::kPitch), qt = smem_of(sh.tq) + at_cols(lane, Keys::kPitch);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        Frag<NI> f;
        f.from(d[2 * i], d[2 * i + 1]);
#pragma unroll
        for (int p = 0; p < NI; ++p)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint32_t*>(&sh.st[p][v0 + row + (e & 1) * 8][16 * i + (e >> 1) * 8 + col]) = f.r[p][e];
        if (fresh) {
#pragma unroll
          for (int e = 0; e < 4; ++e) d[2 * i][e] = d[2 * i + 1][e] = 0.0f;
          continue;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d[2 * i][e] *= end;
          d[2 * i + 1][e] *= end;
        }
        uint32_t b[NT][4];
        load_planes<NT, true>(b, kt + i * 32, Keys::kPlane * 2);
        mma_planes<NI, NT>(d[2 * i], d[2 * i + 1], fz.r, b);
        load_planes<NT, true>(b, qt + i * 32, Keys::kPlane * 2);
        mma_planes<NI, NT>(d[2 * i], d[2 * i + 1], fo.r, b);
      }
    }
    if (warp == warps - 1) {
      for (int x = lane; x < kTile * kTile; x += 32) {
        const int i = x / kTile, j = x % kTile;
        const float dec = i >= j ? c.scratch[2][i][j] : 0.0f;
        const float pd = a.scale * sh.ow[i][j] * c.beta[j] * dec;
        const int lo = min(i, j), hi = max(i, j);
        const float md = i == j ? 0.0f : -sh.zw[hi][lo] * c.beta[lo] * c.scratch[2][hi][lo];
        put_planes<NI>(sh.x1, i, j, i >= j ? pd * c.rk[j] : 0.0f);
        put_planes<NI>(sh.x2, j, i, i >= j ? pd * c.rq[i] : 0.0f);
        put_planes<NI>(sh.x3, i, j, md * c.rk[j]);
      }
    }
    __syncthreads();

    if (by_k) {
      float as[2][4] = {};
      for (int i = 0; i < vwarps; ++i) {
        uint32_t b[NI][4], ww[NI][4];
        load_planes<NI, true>(b, smem_of(sh.st) + at_cols(lane, B::kState) + (i * 16 * B::kState + k0) * 2, 128 * B::kState * 2);
        load_planes<NI, true>(ww, smem_of(sh.w) + a_cols(lane, kSide) + i * 16 * kSide * 2, 128 * kSide * 2);
        mma_planes<NI, NI>(as[0], as[1], ww, b);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = row + (e >> 1) * 8;
          ak[t][e] = fmaf(c.tail[tok] * c.beta[tok], as[t][e], ak[t][e]);
        }
      uint32_t bk[NT][4], x[NI][4];
      load_planes<NT, true>(bk, smem_of(sh.tk) + at_cols(lane, Keys::kPitch) + k0 * 2, Keys::kPlane * 2);
      load_planes<NI, false>(x, smem_of(sh.x1) + a_rows(lane, kSide), kTile * kSide * 2);
      mma_planes<NI, NT>(aq[0], aq[1], x, bk);
      load_planes<NI, false>(x, smem_of(sh.x3) + a_rows(lane, kSide), kTile * kSide * 2);
      mma_planes<NI, NT>(ak[0], ak[1], x, bk);
      load_planes<NT, true>(bk, smem_of(sh.tq) + at_cols(lane, Keys::kPitch) + k0 * 2, Keys::kPlane * 2);
      load_planes<NI, false>(x, smem_of(sh.x2) + a_rows(lane, kSide), kTile * kSide * 2);
      mma_planes<NI, NT>(ak[0], ak[1], x, bk);
      if (a.unit) {
        float nq[2] = {}, nk[2] = {};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = (row + (e >> 1) * 8) * Keys::kPitch + k0 + t * 8 + col + (e & 1);
            nq[e >> 1] = fmaf(aq[t][e], tile_at<T>(sh.tq, Keys::kPlane, at), nq[e >> 1]);
            nk[e >> 1] = fmaf(ak[t][e], tile_at<T>(sh.tk, Keys::kPlane, at), nk[e >> 1]);
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          nq[e] = quad_sum(nq[e]);
          nk[e] = quad_sum(nk[e]);
          if ((lane & 3) == 0) {
            sh.by_key[warp][1][row + 8 * e] = nq[e];
            sh.by_key[warp][2][row + 8 * e] = nk[e];
          }
        }
      }
    }
    __syncthreads();

    if (by_k) {
      float nq[2] = {}, nk[2] = {};
      if (a.unit)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          for (int i = 0; i < kwarps; ++i) {
            nq[e] += sh.by_key[i][1][row + 8 * e];
            nk[e] += sh.by_key[i][2][row + 8 * e];
          }
          nq[e] *= c.rq[row + 8 * e] * c.rq[row + 8 * e];
          nk[e] *= c.rk[row + 8 * e] * c.rk[row + 8 * e];
        }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = row + (e >> 1) * 8, kc = k0 + t * 8 + col + (e & 1);
          if (tok >= n || kc >= a.keys) continue;
          const int at = tok * Keys::kPitch + kc;
          const float x = c.rq[tok] * (aq[t][e] - nq[e >> 1] * tile_at<T>(sh.tq, Keys::kPlane, at));
          const float y = c.rk[tok] * (ak[t][e] - nk[e >> 1] * tile_at<T>(sh.tk, Keys::kPlane, at));
          const int64_t to = (t0 + tok) * qk_t + kc;
          if (pq) {
            pq[to] = x;
            pk[to] = y;
          } else {
            dq[to] = from_f<T>(x);
            dk[to] = from_f<T>(y);
          }
        }
    }
    if (warp == 0) {
      // the gates: lane m < 16 token m's
      const int m = lane & 15;
      float wd = 0.0f, e = 0.0f, f = 0.0f, inner = 0.0f, dbeta, dg;
      for (int i = 0; i < vwarps; ++i) {
        wd += sh.by_value[i][0][m];
        e += sh.by_value[i][1][m];
        f += sh.by_value[i][2][m];
        inner += sh.inner[i];
      }
      for (int i = 0; i < kwarps; ++i) e += sh.by_key[i][0][m];
      dbeta = wd;
      // column m: E's sums from below, into the place of M
      float below = 0.0f;
#pragma unroll
      for (int i = kTile - 1; i >= 0; --i) {
        if (i > m) {
          const float zw = sh.zw[i][m], mm = c.scratch[0][i][m];
          dbeta = fmaf(-mm, zw, dbeta);
          below += c.beta[m] * fmaf(sh.ow[i][m], c.scratch[1][i][m], -zw * mm);
        }
        __syncwarp();
        if (lane < 16) c.scratch[0][i][m] = i > m ? below : 0.0f;
      }
      __syncwarp();
      dg = c.head[kTile - 1] * inner;
#pragma unroll
      for (int j = 0; j < kTile; ++j) {
        const float ej = __shfl_sync(0xffffffffu, e, j), fj = __shfl_sync(0xffffffffu, f, j);
        if (j >= m) dg += ej;
        else dg += fj + c.scratch[0][m][j];
      }
      if (lane < n) {
        const float back = dg * rate * sigmoid(gate.pre);
        db[(t0 + lane) * static_cast<int64_t>(a.heads)] = from_f<T>(dbeta * gate.beta * (1.0f - gate.beta));
        ddt[(t0 + lane) * static_cast<int64_t>(a.heads)] = from_f<T>(back);
        sum_a += static_cast<double>(dg) * gate.delta;
        sum_bias += back;
      }
    }
    t1 = t0;
  }

  if (a.dstate && by_v) {
#pragma unroll
    for (int n = 0; n < DK / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = v0 + row + (e >> 1) * 8, kc = 8 * n + col + (e & 1);
        if (r < a.values && kc < a.keys) a.dstate[head_at + static_cast<int64_t>(r) * a.keys + kc] = d[n][e];
      }
  }
  if (warp == 0) {
    for (int o = 16; o; o >>= 1) {
      sum_a += __shfl_xor_sync(0xffffffffu, sum_a, o);
      sum_bias += __shfl_xor_sync(0xffffffffu, sum_bias, o);
    }
    if (lane == 0) {
      a.part_h[blockIdx.x * 2] = static_cast<float>(sum_a);
      a.part_h[blockIdx.x * 2 + 1] = static_cast<float>(sum_bias);
    }
  }
  // tokens that are not there
  for (int t = length; t < a.length; ++t) {
    for (int i = threadIdx.x; i < a.keys; i += blockDim.x) {
      if (pq) pq[t * qk_t + i] = pk[t * qk_t + i] = 0.0f;
      else dq[t * qk_t + i] = dk[t * qk_t + i] = from_f<T>(0.0f);
    }
    for (int i = threadIdx.x; i < a.values; i += blockDim.x) dv[t * v_t + i] = from_f<T>(0.0f);
    if (threadIdx.x == 0) ddt[t * static_cast<int64_t>(a.heads)] = db[t * static_cast<int64_t>(a.heads)] = from_f<T>(0.0f);
  }
}

// dA and dbias: the sequences' in order.
__global__ void __launch_bounds__(32) delta_rates(DeltaArgs a) {
  const int h = blockIdx.x, lane = threadIdx.x;
  double x = 0.0, y = 0.0;
  for (int b = lane; b < a.batch; b += 32) {
    x += a.part_h[(static_cast<int64_t>(b) * a.heads + h) * 2];
    y += a.part_h[(static_cast<int64_t>(b) * a.heads + h) * 2 + 1];
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

// dq and dk of key heads that value heads share: theirs summed, in order.
template <typename T> __global__ void __launch_bounds__(256) delta_shared(DeltaArgs a) {
  const int64_t total = static_cast<int64_t>(a.batch) * a.length * a.groups * a.keys;
  const int rep = a.heads / a.groups;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t head = i / a.keys, at = head * rep * a.keys + (i - head * a.keys);
    float x = 0.0f, y = 0.0f;
    for (int r = 0; r < rep; ++r) {
      x += a.part_q[at + static_cast<int64_t>(r) * a.keys];
      y += a.part_k[at + static_cast<int64_t>(r) * a.keys];
    }
    static_cast<T*>(a.dq)[i] = from_f<T>(x);
    static_cast<T*>(a.dk)[i] = from_f<T>(y);
  }
}

template <typename T, int DK> int backward(const DeltaArgs& a, cudaStream_t s) {
  using B = Backward<T, DK>;
  if (const int e = allow_smem<delta_backward<T, DK>>(B::kBytes)) return e;
  const int warps = max((a.values + 15) / 16, (a.keys + 15) / 16);
  delta_backward<T, DK><<<a.batch * a.heads, warps * 32, B::kBytes, s>>>(a);
  if (const cudaError_t e = cudaGetLastError()) return static_cast<int>(e);
  delta_rates<<<a.heads, 32, 0, s>>>(a);
  if (a.part_q && a.length > 0) {
    const int64_t blocks = (static_cast<int64_t>(a.batch) * a.length * a.groups * a.keys + 255) / 256;
    delta_shared<T><<<blocks < 148 * 16 ? static_cast<unsigned>(blocks) : 148 * 16, 256, 0, s>>>(a);
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
