// delta.cu — the gated delta rule over sequences and for single tokens (sm_100a). The formulas
// of a chunk are in delta.cuh.
#include "delta.cuh"

namespace {

using namespace delta;

// ---- sequences --------------------------------------------------------------------------
template <typename T, int DK> struct Forward {
  using Keys = Tile<T, DK>;
  using Values = Tile<T, 128>;                         // pitch of the values' rows, whatever their number
  static constexpr size_t kBytes = sizeof(Chunk<T>) + (2 * Keys::kSize + Values::kSize) * sizeof(bf16) +
                                   static_cast<size_t>(kTile) * (128 + 16 / sizeof(T)) * sizeof(T);
};

// A block for a sequence's value head, a warp for 16 of its values: their rows of the state are
// the warp's accumulators from the first token to the last.
template <typename T, int DK> __global__ void __launch_bounds__(256) delta_forward(DeltaArgs a) {
  constexpr int NT = Planes<T>::kToken, NI = Planes<T>::kInner, kSteps = DK / 16;
  using Keys = Tile<T, DK>;
  using Values = Tile<T, 128>;
  extern __shared__ __align__(16) char smem[];
  Chunk<T>& c = *reinterpret_cast<Chunk<T>*>(smem);
  bf16* tk = reinterpret_cast<bf16*>(smem + sizeof(Chunk<T>));
  bf16* tq = tk + Keys::kSize;
  bf16* tv = tq + Keys::kSize;
  T* so = reinterpret_cast<T*>(tv + Values::kSize);
  constexpr int kOut = 128 + 16 / static_cast<int>(sizeof(T));
  const int bi = blockIdx.x / a.heads, h = blockIdx.x % a.heads, gr = h / (a.heads / a.groups);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = lane >> 2, col = (lane & 3) * 2;
  const int v0 = warp * 16;
  const int length = a.lengths ? max(0, min(a.lengths[bi], a.length)) : a.length;
  const uint8_t* reset = a.reset ? a.reset + static_cast<int64_t>(bi) * a.length : nullptr;
  const T* q = static_cast<const T*>(a.q) + bi * a.q_b + gr * a.q_g;
  const T* k = static_cast<const T*>(a.k) + bi * a.k_b + gr * a.k_g;
  const T* v = static_cast<const T*>(a.v) + bi * a.v_b + h * a.v_h;
  const T* dt = static_cast<const T*>(a.dt) + bi * a.dt_b + h;
  const T* gb = static_cast<const T*>(a.b) + bi * a.b_b + h;
  T* out = static_cast<T*>(a.out) + bi * a.o_b + h * a.o_h;
  const float rate = rate_at(a.A, h), bias = a.bias ? a.bias[h] : 0.0f;
  const int64_t head_size = static_cast<int64_t>(a.values) * a.keys;
  const int64_t head_at = (static_cast<int64_t>(bi) * a.heads + h) * head_size;
  const bool pairs = (a.keys & 1) == 0;

  // s[n]: rows v0 + row, + 8; keys 8 n + col, + 1
  float s[DK / 8][4];
  auto each = [&](auto f) {
#pragma unroll
    for (int n = 0; n < DK / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) f(s[n][2 * e], s[n][2 * e + 1], v0 + row + 8 * e, 8 * n + col);
  };
  auto store = [&](float* to) {
    each([&](float x, float y, int r, int kc) {
      if (r >= a.values || kc >= a.keys) return;
      float* p = to + static_cast<int64_t>(r) * a.keys + kc;
      if (pairs) {
        *reinterpret_cast<float2*>(p) = make_float2(x, y);
      } else {
        p[0] = x;
        if (kc + 1 < a.keys) p[1] = y;
      }
    });
  };
  each([&](float& x, float& y, int r, int kc) {
    const bool on = a.state && r < a.values;
    const float* p = a.state + head_at + static_cast<int64_t>(r) * a.keys + kc;
    x = on && kc < a.keys ? p[0] : 0.0f;
    y = on && kc + 1 < a.keys ? p[1] : 0.0f;
  });

  const int tiles = (a.length + kTile - 1) / kTile;
  int t0 = 0;
  while (t0 < length) {
    const int n = chunk_tokens(reset, t0, length);
    const bool fresh = reset && reset[t0];
    if (a.saved && t0 % kTile == 0)
      store(a.saved + ((static_cast<int64_t>(bi) * tiles + t0 / kTile) * a.heads + h) * head_size);
    if (fresh) each([&](float& x, float& y, int, int) { x = y = 0.0f; });
    __syncthreads();
    Keys::load(tk, k + t0 * a.k_t, a.k_t, n, a.keys, a.piece_k, threadIdx.x, blockDim.x);
    Keys::load(tq, q + t0 * a.q_t, a.q_t, n, a.keys, a.piece_k, threadIdx.x, blockDim.x);
    Values::load(tv, v + t0 * a.v_t, a.v_t, n, a.values, a.piece_v, threadIdx.x, blockDim.x);
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    if (warp == 0) {
      float g = 0.0f, beta = 0.0f;
      if (lane < n) {
        const Gate e = gate_of(to_f(dt[(t0 + lane) * a.dt_t]), to_f(gb[(t0 + lane) * a.b_t]), bias, rate);
        g = e.g;
        beta = e.beta;
      }
      prepare<T, DK, false>(c, tk, tq, g, beta, a.scale, a.unit);
    }
    __syncthreads();

    // K S^T and Q S^T, transposed: rows values, columns tokens
    float sk[2][4] = {}, sq[2][4] = {};
    const uint32_t ka = smem_of(tk) + at_rows(lane, Keys::kPitch), qa = smem_of(tq) + at_rows(lane, Keys::kPitch);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      Frag<NI> f;
      f.from(s[2 * i], s[2 * i + 1]);
      uint32_t b[NT][4];
      load_planes<NT, false>(b, ka + i * 32, Keys::kPlane * 2);
      mma_planes<NI, NT>(sk[0], sk[1], f.r, b);
      load_planes<NT, false>(b, qa + i * 32, Keys::kPlane * 2);
      mma_planes<NI, NT>(sq[0], sq[1], f.r, b);
    }
    float w[2][4] = {};
    {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = t * 8 + col + (e & 1), r = v0 + row + (e >> 1) * 8;
          sk[t][e] = tile_at<T>(tv, Values::kPlane, tok * Values::kPitch + r) - c.head[tok] * c.rk[tok] * sk[t][e];
          sq[t][e] *= a.scale * c.head[tok] * c.rq[tok];
        }
      Frag<NI> f;
      f.from(sk[0], sk[1]);
      uint32_t b[NI][4];
      load_planes<NI, false>(b, smem_of(c.inv) + at_rows(lane, kSide), kTile * kSide * 2);
      mma_planes<NI, NI>(w[0], w[1], f.r, b);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[t][e] *= c.beta[t * 8 + col + (e & 1)];
    {
      Frag<NI> f;
      f.from(w[0], w[1]);
      uint32_t b[NI][4];
      load_planes<NI, false>(b, smem_of(c.p) + at_rows(lane, kSide), kTile * kSide * 2);
      mma_planes<NI, NI>(sq[0], sq[1], f.r, b);
    }
    // the state
    const float end = c.head[kTile - 1];
    {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = t * 8 + col + (e & 1);
          w[t][e] *= c.tail[tok] * c.rk[tok];
        }
      Frag<NI> f;
      f.from(w[0], w[1]);
      const uint32_t kt = smem_of(tk) + at_cols(lane, Keys::kPitch);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[2 * i][e] *= end;
          s[2 * i + 1][e] *= end;
        }
        uint32_t b[NT][4];
        load_planes<NT, true>(b, kt + i * 32, Keys::kPlane * 2);
        mma_planes<NI, NT>(s[2 * i], s[2 * i + 1], f.r, b);
      }
    }
    // the outputs, by tokens
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) so[(t * 8 + col + (e & 1)) * kOut + v0 + row + (e >> 1) * 8] = from_f<T>(sq[t][e]);
    __syncwarp();
    if (a.piece_v == 16) {
      constexpr int V = kVec16<T>;
      for (int i = lane; i < n * (16 / V); i += 32) {
        const int r = i / (16 / V), cc = v0 + i % (16 / V) * V;
        if (cc < a.values)
          *reinterpret_cast<uint4*>(out + (t0 + r) * a.o_t + cc) = *reinterpret_cast<const uint4*>(so + r * kOut + cc);
      }
    } else {
      for (int i = lane; i < n * 16; i += 32) {
        const int r = i / 16, cc = v0 + i % 16;
        if (cc < a.values) out[(t0 + r) * a.o_t + cc] = so[r * kOut + cc];
      }
    }
    t0 += n;
  }
  store(a.final_ + head_at);
  // tokens that are not there give zeros
  for (int64_t i = threadIdx.x; i < static_cast<int64_t>(a.length - length) * a.values; i += blockDim.x)
    out[(length + i / a.values) * a.o_t + i % a.values] = from_f<T>(0.0f);
}

template <typename T, int DK> int forward(const DeltaArgs& a, cudaStream_t s) {
  using F = Forward<T, DK>;
  if (const int e = allow_smem<delta_forward<T, DK>>(F::kBytes)) return e;
  delta_forward<T, DK><<<a.batch * a.heads, (a.values + 15) / 16 * 32, F::kBytes, s>>>(a);
  return static_cast<int>(cudaGetLastError());
}
template <typename T> int forward_by(const DeltaArgs& a, cudaStream_t s) {
  if (a.keys <= 32) return forward<T, 32>(a, s);
  if (a.keys <= 64) return forward<T, 64>(a, s);
  return forward<T, 128>(a, s);
}

// ---- single tokens ------------------------------------------------------------------------
struct StepArgs {
  const void *q, *k, *v, *dt, *b;
  const float *A, *bias;
  float* state;
  const uint8_t* reset;
  const int* slots;
  void* out;
  int* err;
  int64_t q_r, q_g, k_r, k_g, v_r, v_h, dt_r, b_r, o_r, o_h;
  float scale;
  int rows, groups, heads, keys, values, unit, pools;
};
static_assert(sizeof(StepArgs) == 12 * 8 + 10 * 8 + 8 * 4, "as the caller packs it");

// A warp for a head of a row: its lanes hold the key and the query, LK lanes a value's row of the
// state. S k and S q come from one look at the state:
//   u = beta (v - e^g S k),  S <- e^g S + u k^T,  o = scale (e^g S q + u k.q).
template <typename T, int LK> __global__ void __launch_bounds__(256) delta_step(StepArgs a) {
  constexpr int kRows = 32 / LK;                       // values that a warp takes at once
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5);
  if (item >= static_cast<int64_t>(a.rows) * a.heads) return;
  const int r = static_cast<int>(item / a.heads), h = static_cast<int>(item % a.heads), gr = h / (a.heads / a.groups);
  T* out = static_cast<T*>(a.out) + r * a.o_r + h * a.o_h;
  const int slot = a.slots ? a.slots[r] : r;
  if (slot < 0 || slot >= a.pools) {
    if (slot >= a.pools && h == 0 && lane == 0) surfk::report_error(a.err, surfk::kErrSlotIndex);
    for (int i = lane; i < a.values; i += 32) out[i] = from_f<T>(0.0f);
    return;
  }
  const int l = lane % LK, k0 = l * 4;
  float k[4], q[4], kk = 0.0f, qq = 0.0f, kq = 0.0f;
  const T* pk = static_cast<const T*>(a.k) + r * a.k_r + gr * a.k_g;
  const T* pq = static_cast<const T*>(a.q) + r * a.q_r + gr * a.q_g;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool on = k0 + j < a.keys;
    k[j] = on ? to_f(pk[k0 + j]) : 0.0f;
    q[j] = on ? to_f(pq[k0 + j]) : 0.0f;
    kk = fmaf(k[j], k[j], kk);
    qq = fmaf(q[j], q[j], qq);
  }
#pragma unroll
  for (int o = LK / 2; o; o >>= 1) {
    kk += __shfl_xor_sync(0xffffffffu, kk, o);
    qq += __shfl_xor_sync(0xffffffffu, qq, o);
  }
  if (a.unit) {
    const float rk = rsqrtf(kk + kNormEps), rq = rsqrtf(qq + kNormEps);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      k[j] *= rk;
      q[j] *= rq;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) kq = fmaf(k[j], q[j], kq);
#pragma unroll
  for (int o = LK / 2; o; o >>= 1) kq += __shfl_xor_sync(0xffffffffu, kq, o);
  const float pre = to_f(static_cast<const T*>(a.dt)[r * a.dt_r + h]) + (a.bias ? a.bias[h] : 0.0f);
  const bool fresh = a.reset && a.reset[r];
  const float decay = exp2_hw(fmaf(rate_at(a.A, h) * softplus(pre), kLog2e, kExp2Shift));
  const float beta = sigmoid(to_f(static_cast<const T*>(a.b)[r * a.b_r + h]));
  const T* pv = static_cast<const T*>(a.v) + r * a.v_r + h * a.v_h;
  float* state = a.state + (static_cast<int64_t>(slot) * a.heads + h) * a.values * a.keys;
  const bool whole = a.keys % 4 == 0;
  for (int v0 = 0; v0 < a.values; v0 += kRows) {
    const int vr = v0 + lane / LK;
    const bool on = vr < a.values;
    float* p = state + static_cast<int64_t>(vr) * a.keys + k0;
    float s[4] = {};
    if (on && !fresh) {
      if (whole) {
        if (k0 < a.keys) *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = k0 + j < a.keys ? p[j] : 0.0f;
      }
    }
    float sk = 0.0f, sq = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j] *= decay;
      sk = fmaf(s[j], k[j], sk);
      sq = fmaf(s[j], q[j], sq);
    }
#pragma unroll
    for (int o = LK / 2; o; o >>= 1) {
      sk += __shfl_xor_sync(0xffffffffu, sk, o);
      sq += __shfl_xor_sync(0xffffffffu, sq, o);
    }
    if (!on) continue;
    const float u = beta * (to_f(pv[vr]) - sk);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = fmaf(u, k[j], s[j]);
    if (whole) {
      if (k0 < a.keys) *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(s);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k0 + j < a.keys) p[j] = s[j];
    }
    if (l == 0) out[vr] = from_f<T>(a.scale * fmaf(u, kq, sq));
  }
}

template <typename T> int step(const StepArgs& a, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.rows) * a.heads + 7) / 8);
  if (a.keys <= 16) delta_step<T, 4><<<grid, 256, 0, s>>>(a);
  else if (a.keys <= 32) delta_step<T, 8><<<grid, 256, 0, s>>>(a);
  else if (a.keys <= 64) delta_step<T, 16><<<grid, 256, 0, s>>>(a);
  else delta_step<T, 32><<<grid, 256, 0, s>>>(a);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

SURF_EXPORT int surf_delta(const void* args, int dtype, void* stream) {
  const DeltaArgs& a = *static_cast<const DeltaArgs*>(args);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == kBf16 ? forward_by<bf16>(a, s) : forward_by<float>(a, s);
}

SURF_EXPORT int surf_delta_step(const void* args, int dtype, void* stream) {
  const StepArgs& a = *static_cast<const StepArgs*>(args);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == kBf16 ? step<bf16>(a, s) : step<float>(a, s);
}
