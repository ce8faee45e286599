// delta.cuh — what the kernels of the gated delta rule share: the formulas of a chunk, token
// tiles, and matrix products of numbers split into bfloat16 planes.
//
// The rule, per sequence and value head, S [values, keys] in 32 bits:
//   S <- e^g S,  w = v - S k,  S <- S + beta w k^T,  o = scale S q
// with g = A softplus(dt + bias) <= 0, beta = sigmoid(b), k and q divided by their lengths.
//
// A chunk: up to 16 tokens of one episode within one tile of 16. With D_ij = exp(g_j+1 + .. + g_i),
// head_i = exp(g_1 + .. + g_i), tail_i = D_last,i, end = head_last and
//   M_ij = D_ij k_i.k_j (j < i),  P_ij = scale D_ij q_i.k_j (j <= i):
//   R = V - head (K S^T),  W = (I + M beta)^-1 R,  U = beta W
//   O = scale head (Q S^T) + P U,  S+ = end S + sum_i tail_i U_i k_i^T.
// Every exponent is a sum of terms <= 0 taken afresh for its pair of tokens (never a difference of
// running sums), so that nothing overflows and a strong decay costs the others no digits.
// A reset ends a chunk: what stood before it is never multiplied by zero, it is not there, so
// that infinities and NaN end with their episode.
//
// Products run on the tensor cores as mma.sync.m16n8k16 with bfloat16 operands and 32-bit sums. A
// 32-bit number enters as the sum of its planes, each the bfloat16 next to what the ones before
// leave. tcgen05 does not fit: a chunk's products have 16 tokens for a side where its
// instructions take 128, and each of the chain's four products would go through tensor
// memory and shared memory to become the next one's operand. Here an accumulator is the next
// product's operand in the registers that it lies in, and a warp's 16 rows of the state never leave them.
#pragma once
#include <type_traits>

#include "seq_common.cuh"

namespace delta {

using namespace seqk;

constexpr int kTile = 16;                     // tokens of a chunk at most; states are kept before each tile
constexpr float kNormEps = 1e-6f;             // added to the square of a key's or query's length

struct DeltaArgs {
  const void *q, *k, *v, *dt, *b;
  const float *A, *bias, *state;
  const uint8_t* reset;
  const int* lengths;
  void* out;
  float *final_, *saved;
  // gradient
  const void* dout;
  const float* dfinal;
  void *dq, *dk, *dv, *ddt, *db;
  float *dstate, *part_q, *part_k, *part_h;
  float *dA, *dbias;
  int64_t q_b, q_t, q_g, k_b, k_t, k_g, v_b, v_t, v_h, dt_b, dt_t, b_b, b_t, o_b, o_t, o_h, do_b, do_t, do_h;
  float scale;
  int batch, length, groups, heads, keys, values, unit, piece_k, piece_v;
};
static_assert(sizeof(DeltaArgs) == 26 * 8 + 19 * 8 + 10 * 4, "as the caller packs it");

// Planes of a token (its own type: exact) and of a 32-bit number that is an operand. bfloat16 tokens:
// one plane, and two for what is computed, 16 bits of mantissa against the 8 of the results; the
// sums, states and decays keep 32 bits. 32-bit tokens: three planes of either, 24 bits.
template <typename T> struct Planes { static constexpr int kToken = 1, kInner = 2; };
template <> struct Planes<float> { static constexpr int kToken = 3, kInner = 3; };

__device__ __forceinline__ uint32_t smem_of(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x, y -> their planes, packed
template <int N> __device__ __forceinline__ void split2(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = surfk::pack_bf16x2(x, y);
    if (i + 1 < N) {
      x -= __uint_as_float(p[i] << 16);
      y -= __uint_as_float(p[i] & 0xffff0000u);
    }
  }
}

// Operand of 16 x 16 from an accumulator's two tiles of 16 x 8.
template <int N> struct Frag {
  uint32_t r[N][4];
  __device__ __forceinline__ void from(const float (&lo)[4], const float (&hi)[4]) {
    uint32_t p[N];
    split2<N>(lo[0], lo[1], p);
#pragma unroll
    for (int i = 0; i < N; ++i) r[i][0] = p[i];
    split2<N>(lo[2], lo[3], p);
#pragma unroll
    for (int i = 0; i < N; ++i) r[i][1] = p[i];
    split2<N>(hi[0], hi[1], p);
#pragma unroll
    for (int i = 0; i < N; ++i) r[i][2] = p[i];
    split2<N>(hi[2], hi[3], p);
#pragma unroll
    for (int i = 0; i < N; ++i) r[i][3] = p[i];
  }
};

// A matrix of 16-bit planes in shared memory: rows of kPitch elements, planes kPlane apart.
// Both pitches are odd multiples of 16 bytes, so that eight rows of 16 bytes lie in all banks.
//
// As the second operand of 16 x (two tiles of 8): rows are its columns (n), contiguous along k, ...
__device__ __forceinline__ uint32_t at_rows(int lane, int pitch) {
  return (((lane & 16) >> 1) + (lane & 7)) * pitch * 2 + (lane & 8) * 2;
}
// ... or rows are along k, contiguous along n (loaded transposed).
__device__ __forceinline__ uint32_t at_cols(int lane, int pitch) {
  return (lane & 15) * pitch * 2 + (lane & 16);
}
// As the first operand (rows m): contiguous along k; or rows along k, contiguous along m (transposed).
__device__ __forceinline__ uint32_t a_rows(int lane, int pitch) { return (lane & 15) * pitch * 2 + (lane & 16); }
__device__ __forceinline__ uint32_t a_cols(int lane, int pitch) {
  return (((lane & 16) >> 1) + (lane & 7)) * pitch * 2 + (lane & 8) * 2;
}

// c0, c1 (columns 0-7 and 8-15) += A B over 16 of k. NA and NB planes; products of planes i and j
// with i + j >= max(NA, NB) are below what the planes leave out.
template <int NA, int NB>
__device__ __forceinline__ void mma_planes(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][4]) {
  constexpr int kMost = NA > NB ? NA : NB;
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < kMost) {
        mma(c0, a[i], b[j][0], b[j][1]);
        mma(c1, a[i], b[j][2], b[j][3]);
      }
}
template <int N, bool kTrans> __device__ __forceinline__ void load_planes(uint32_t (&r)[N][4], uint32_t at, uint32_t plane) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (kTrans) ldsm4t(r[i], at + i * plane);
    else ldsm4(r[i], at + i * plane);
  }
}

// ---- token tiles ------------------------------------------------------------------------
// Rows [0, n) of `cols` elements, planes kPlane apart with a pitch of W + 8; the rest of 16 x W zero.
template <typename T, int W> struct Tile {
  static constexpr int kPitch = W + 8, kPlane = kTile * kPitch, kSize = Planes<T>::kToken * kPlane;
  static __device__ __forceinline__ void load(bf16* dst, const T* src, int64_t stride, int n, int cols, int piece, int tid, int threads) {
    if constexpr (sizeof(T) == 2) {
      if (piece == 16) {
        for (int i = tid; i < kTile * W / 8; i += threads) {
          const int r = i / (W / 8), c = i % (W / 8) * 8;
          bf16* d = dst + r * kPitch + c;
          if (r < n && c < cols) cp_async16(d, src + r * stride + c);
          else *reinterpret_cast<uint4*>(d) = make_uint4(0, 0, 0, 0);
        }
      } else {
        for (int i = tid; i < kTile * W; i += threads) {
          const int r = i / W, c = i % W;
          dst[r * kPitch + c] = r < n && c < cols ? src[r * stride + c] : from_f<bf16>(0.0f);
        }
      }
    } else {
      for (int i = tid; i < kTile * W / 2; i += threads) {
        const int r = i / (W / 2), c = i % (W / 2) * 2;
        const float x = r < n && c < cols ? src[r * stride + c] : 0.0f;
        const float y = r < n && c + 1 < cols ? src[r * stride + c + 1] : 0.0f;
        uint32_t p[Planes<T>::kToken];
        split2<Planes<T>::kToken>(x, y, p);
#pragma unroll
        for (int j = 0; j < Planes<T>::kToken; ++j) *reinterpret_cast<uint32_t*>(dst + j * kPlane + r * kPitch + c) = p[j];
      }
    }
  }
};
// A token tile's element, from its planes.
template <typename T> __device__ __forceinline__ float tile_at(const bf16* t, int plane, int at) {
  float v = to_f(t[at]);
#pragma unroll
  for (int i = 1; i < Planes<T>::kToken; ++i) v += to_f(t[i * plane + at]);
  return v;
}

// ---- a chunk's matrices -----------------------------------------------------------------
constexpr int kSide = kTile + 8;                       // pitch of 16 x 16 matrices of planes
template <typename T> struct Chunk {
  static constexpr int kInner = Planes<T>::kInner;
  float beta[kTile], head[kTile], tail[kTile], rk[kTile], rq[kTile];
  float scratch[3][kTile][20];                         // K K^T, Q K^T, Q Q^T; then M beta, M, P
  alignas(16) bf16 inv[kInner][kTile][kSide];          // (I + M beta)^-1
  alignas(16) bf16 p[kInner][kTile][kSide];            // P
};

// By one warp, from the tiles of K and Q and each lane's gates (lane < 16: token lane's log decay and
// beta, zero behind the chunk). scratch holds M and P as 32-bit numbers then and, with kKeep, D.
template <typename T, int DK, bool kKeep>
__device__ __forceinline__ void prepare(Chunk<T>& c, const bf16* tk, const bf16* tq, float g, float beta, float scale, int unit) {
  constexpr int NT = Planes<T>::kToken, NI = Planes<T>::kInner;
  using Keys = Tile<T, DK>;
  const int lane = threadIdx.x & 31, row = lane >> 2, col = (lane & 3) * 2;
  {
    float kk[2][4] = {}, qk[2][4] = {}, qq[2][4] = {};
    const uint32_t ka = smem_of(tk), qa = smem_of(tq);
    const uint32_t b_at = at_rows(lane, Keys::kPitch), a_at = a_rows(lane, Keys::kPitch);
#pragma unroll
    for (int s = 0; s < DK / 16; ++s) {
      uint32_t ak[NT][4], aq[NT][4], bk[NT][4];
      load_planes<NT, false>(ak, ka + a_at + s * 32, Keys::kPlane * 2);
      load_planes<NT, false>(aq, qa + a_at + s * 32, Keys::kPlane * 2);
      load_planes<NT, false>(bk, ka + b_at + s * 32, Keys::kPlane * 2);
      mma_planes<NT, NT>(kk[0], kk[1], ak, bk);
      mma_planes<NT, NT>(qk[0], qk[1], aq, bk);
      load_planes<NT, false>(bk, qa + b_at + s * 32, Keys::kPlane * 2);
      mma_planes<NT, NT>(qq[0], qq[1], aq, bk);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = row + (e >> 1) * 8, j = t * 8 + col + (e & 1);
        c.scratch[0][i][j] = kk[t][e];
        c.scratch[1][i][j] = qk[t][e];
        c.scratch[2][i][j] = qq[t][e];
      }
  }
  __syncwarp();
  const int j = lane & 15;
  const bool upper = lane >= 16;
  const float rk = unit ? rsqrtf(c.scratch[0][j][j] + kNormEps) : 1.0f;
  const float rq = unit ? rsqrtf(c.scratch[2][j][j] + kNormEps) : 1.0f;
  __syncwarp();
  // lanes 0-15 make M's column, 16-31 P's; d: the sum of the decays behind token j up to token i
  float d = 0.0f, h = 0.0f, last = 1.0f, decay[kKeep ? kTile : 1];
#pragma unroll
  for (int i = 0; i < kTile; ++i) {
    const float gi = __shfl_sync(0xffffffffu, g, i);
    const float ri = __shfl_sync(0xffffffffu, upper ? rq : rk, i + (lane & 16));
    if (i <= j) h += gi;
    if (i > j) d += gi;
    float x = 0.0f;
    if (i > j || (upper && i == j)) {
      last = exp2_hw(fmaf(d, kLog2e, kExp2Shift));
      x = c.scratch[upper ? 1 : 0][i][j] * (last * ri * rk) * (upper ? scale : 1.0f);
    }
    if constexpr (kKeep) decay[i] = i == j ? 1.0f : i > j ? last : 0.0f;
    c.scratch[upper ? 1 : 0][i][j] = x;
    if (upper) {
      float y = x, z = 0.0f;
      uint32_t p[NI];
      split2<NI>(y, z, p);
#pragma unroll
      for (int n = 0; n < NI; ++n) c.p[n][i][j] = __ushort_as_bfloat16(static_cast<unsigned short>(p[n]));
    } else {
      c.scratch[2][i][j] = x * beta;
    }
  }
  if (!upper) {
    c.beta[j] = beta;
    c.head[j] = exp2_hw(fmaf(h, kLog2e, kExp2Shift));
    c.tail[j] = last;
    c.rk[j] = rk;
    c.rq[j] = rq;
  }
  __syncwarp();
  // column j of (I + M beta)^-1, row by row
  float t[kTile];
#pragma unroll
  for (int i = 0; i < kTile; ++i) {
    float s = i == j ? 1.0f : 0.0f;
#pragma unroll
    for (int m = 0; m < i; m += 4) {
      const float4 a = *reinterpret_cast<const float4*>(&c.scratch[2][i][m]);
      s = fmaf(-a.x, t[m], s);
      if (m + 1 < i) s = fmaf(-a.y, t[m + 1], s);
      if (m + 2 < i) s = fmaf(-a.z, t[m + 2], s);
      if (m + 3 < i) s = fmaf(-a.w, t[m + 3], s);
    }
    t[i] = s;
  }
  if (!upper) {
#pragma unroll
    for (int i = 0; i < kTile; ++i) {
      uint32_t p[NI];
      split2<NI>(t[i], 0.0f, p);
#pragma unroll
      for (int n = 0; n < NI; ++n) c.inv[n][i][j] = __ushort_as_bfloat16(static_cast<unsigned short>(p[n]));
    }
  }
  __syncwarp();
  if constexpr (kKeep) {
    if (!upper) {
#pragma unroll
      for (int i = 0; i < kTile; ++i) c.scratch[2][i][j] = decay[i];
    }
    __syncwarp();
  }
}

// A log decay and its gate from a token's dt and b.
struct Gate { float pre, delta, g, beta; };
__device__ __forceinline__ Gate gate_of(float dt, float b, float bias, float rate) {
  Gate r;
  r.pre = dt + bias;
  r.delta = softplus(r.pre);
  r.g = rate * r.delta;
  r.beta = sigmoid(b);
  return r;
}
// A[h]; -inf as the lowest finite number, so that a step of zero decays by e^0
__device__ __forceinline__ float rate_at(const float* A, int h) { return fmaxf(A[h], -3.4028235e38f); }

// The tokens [t0, t0 + n) of a chunk: up to the end of its tile, the row's end, the next reset.
__device__ __forceinline__ int chunk_tokens(const uint8_t* reset, int t0, int length) {
  const int lane = threadIdx.x & 31;
  int n = min(kTile - t0 % kTile, length - t0);
  if (reset) {
    const bool cut = lane > 0 && lane < n && reset[t0 + lane];
    const unsigned cuts = __ballot_sync(0xffffffffu, cut);
    if (cuts) n = __ffs(cuts) - 1;
  }
  return n;
}

}  // namespace delta
