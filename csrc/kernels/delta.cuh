// delta.cuh — what the kernels of the gated delta rule share: the formulas of a chunk, token
// tiles, and matrix products of numbers split into bfloat16 planes.
//
// The rule, per sequence and value head, S [values, keys] in 32 bits:
//   S <- e^g S,  w = v - S k,  S <- S + beta w k^T,  o = scale S q
// with g = A softplus(dt + bias) <= 0, beta = sigmoid(b), k and q divided by their lengths.
//
// A chunk: a tile of 16 tokens, or what a row has of it. With D_ij = exp(g_j+1 + .. + g_i) within an
// episode and 0 across a reset, head_i = exp(g_1 + .. + g_i) up to the chunk's first reset, tail_i =
// D_last,i, end = head_last and
//   M_ij = D_ij k_i.k_j (j < i),  P_ij = scale D_ij q_i.k_j (j <= i):
//   R = V - head (K S^T),  W = (I + M beta)^-1 R,  U = beta W
//   O = scale head (Q S^T) + P U,  S+ = end S + sum_i tail_i U_i k_i^T.
// Every exponent is the sum of its tokens' own terms <= 0, so that nothing overflows and a strong
// decay costs the others no digits.
// Infinities and NaN end with their episode: where head, tail or end is 0 nothing is multiplied by
// it, and a chunk with a reset inside and tokens that are not finite is taken episode by episode.
//
// Products run on the tensor cores as mma.sync.m16n8k16 with bfloat16 operands and 32-bit sums. A
// 32-bit number enters as the sum of its planes, each the bfloat16 next to what the ones before
// leave. tcgen05 does not fit: a chunk's products have 16 tokens for a side where its
// instructions take 64 or 128, and each of the chain's four products would go through tensor
// memory and shared memory to become the next one's operand. Here an accumulator is the next
// product's operand in the registers that it lies in, and a warp's 16 rows of the state never leave them.
#pragma once
#include <type_traits>

#include "seq_common.cuh"

namespace delta {

using namespace seqk;

constexpr int kTile = 16;                     // tokens of a chunk at most, and of the tiles that it ends with
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
  float *dstate, *part_q, *part_k, *part_g, *part_h;
  float *dA, *dbias;
  int64_t q_b, q_t, q_g, k_b, k_t, k_g, v_b, v_t, v_h, dt_b, dt_t, b_b, b_t, o_b, o_t, o_h, do_b, do_t, do_h;
  float scale;
  int batch, length, groups, heads, keys, values, unit, piece_k, piece_v;
};
static_assert(sizeof(DeltaArgs) == 27 * 8 + 19 * 8 + 10 * 4, "as the caller packs it");

// Planes of a token (its own type: exact) and of a 32-bit number that is an operand: kInner on the way
// from state to state and into anything that stays 32-bit, 24 bits of mantissa; kShort where the
// result is rounded to the tokens' type at once, 16 bits against bfloat16's 8: one rounding in 2000 falls
// the other way, out and dk 1e-4 of their norm from where three planes have them (both 0.0017 from 64 bits). With
// three 1x8191x8x128x128 takes 901 us (two: 760), 256x128x8x64x64 174 + 741 us (164 + 532: two teams no
// longer fit a block's shared memory), 2x4096x16x64x64 391 + 979 us (369 + 918).
template <typename T> struct Planes { static constexpr int kToken = 1, kInner = 3, kShort = 2; };
template <> struct Planes<float> { static constexpr int kToken = 3, kInner = 3, kShort = 3; };

__device__ __forceinline__ uint32_t smem_of(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// What these read was written before a barrier of the warp or the block, across which the compiler moves
// neither; without a memory clobber it may move other accesses about them.
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
// four 8 x 8 tiles, one register of each lane's a tile, to rows of 16 bytes
__device__ __forceinline__ void stsm4(uint32_t at, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x, y -> their planes, packed. What a plane leaves is one multiply-add of mixed types a number.
template <int N> __device__ __forceinline__ void split2(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = surfk::pack_bf16x2(x, y);
    if (i + 1 < N)
      asm("{.reg .b16 lo, hi, m;\n mov.b16 m, 0xbf80;\n mov.b32 {lo, hi}, %2;\n fma.rn.f32.bf16 %0, lo, m, %0;\n fma.rn.f32.bf16 %1, hi, m, %1;}"
          : "+f"(x), "+f"(y) : "r"(p[i]));
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

// c0, c1 (columns 0-7 and 8-15) += A B over 16 of k, of the first PA and PB planes, smaller products
// first; products of planes i and j with i + j >= max(PA, PB) are below what the planes leave out.
template <int PA, int PB, int NA, int NB>
__device__ __forceinline__ void mma_planes(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][4]) {
  static_assert(PA <= NA && PB <= NB, "planes that are there");
  constexpr int kLevels = PA > PB ? PA : PB;
#pragma unroll
  for (int l = kLevels - 1; l >= 0; --l)
#pragma unroll
    for (int i = 0; i < PA; ++i)
      if (l - i >= 0 && l - i < PB) {
        mma(c0, a[i], b[l - i][0], b[l - i][1]);
        mma(c1, a[i], b[l - i][2], b[l - i][3]);
      }
}
// The same for one left operand and two right ones (c += A B, d += A D), planes in turn.
template <int PC, int PD, int NA, int NB>
__device__ __forceinline__ void mma_planes2(float (&c0)[4], float (&c1)[4], float (&d0)[4], float (&d1)[4], const uint32_t (&a)[NA][4],
                                            const uint32_t (&b)[NB][4], const uint32_t (&d)[NB][4]) {
  if constexpr (NB == 1) {
#pragma unroll
    for (int i = 0; i < PC; ++i) {
      mma(c0, a[i], b[0][0], b[0][1]);
      mma(c1, a[i], b[0][2], b[0][3]);
      if (i < PD) {
        mma(d0, a[i], d[0][0], d[0][1]);
        mma(d1, a[i], d[0][2], d[0][3]);
      }
    }
  } else {
    mma_planes<PC, NB>(c0, c1, a, b);
    mma_planes<PD, NB>(d0, d1, a, d);
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
// 16 bytes, or zeros (nothing is read then)
__device__ __forceinline__ void cp_async16_or_zero(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_of(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}
// By one warp: rows [0, n) of `cols` elements, planes kPlane apart with a pitch of W + 8; the rest of 16 x W zero.
template <typename T, int W> struct Tile {
  static constexpr int kPitch = W + 8, kPlane = kTile * kPitch, kSize = Planes<T>::kToken * kPlane;
  static __device__ __forceinline__ void load(bf16* dst, const T* src, int64_t stride, int n, int cols, bool pieces) {
    const int lane = threadIdx.x & 31;
    if constexpr (sizeof(T) == 2) {
      if (pieces) {
        constexpr int kPer = W / 8, kRows = 32 / kPer;
        const int r0 = lane / kPer, c = lane % kPer * 8;
        const T* from = src + r0 * stride + c;
        bf16* to = dst + r0 * kPitch + c;
        const int rows = c < cols ? n : 0;
#pragma unroll
        for (int r = 0; r < kTile; r += kRows) {
          cp_async16_or_zero(to + r * kPitch, r0 + r < rows ? from : src, r0 + r < rows);
          from += kRows * stride;
        }
      } else {
        for (int i = lane; i < kTile * W; i += 32) {
          const int r = i / W, c = i % W;
          dst[r * kPitch + c] = r < n && c < cols ? src[r * stride + c] : from_f<bf16>(0.0f);
        }
      }
    } else {
      for (int i = lane; i < kTile * W / 2; i += 32) {
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

// Two neighbouring ones, the first on an even place.
template <typename T> __device__ __forceinline__ void tile_pair(const bf16* t, int plane, int at, float& x, float& y) {
  x = y = 0.0f;
#pragma unroll
  for (int i = 0; i < Planes<T>::kToken; ++i) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(t + i * plane + at);
    x += __uint_as_float(w << 16);
    y += __uint_as_float(w & 0xffff0000u);
  }
}

// By one warp: rows [0, n) of `cols` elements as they are, `pitch` apart; the rest of `rows` x `width` zero.
// A row's pieces are spread over a power of two of lanes.
template <typename T>
__device__ __forceinline__ void load_rows(T* dst, int pitch, int rows, int width, const T* src, int64_t stride, int n, int cols, bool pieces) {
  constexpr int V = kVec16<T>;
  const int lane = threadIdx.x & 31;
  if (pieces) {
    const int bits = min(5, 32 - __clz(width / V - 1)), c = (lane & ((1 << bits) - 1)) * V, r0 = lane >> bits, step = 32 >> bits;
    for (int x = c; x < width; x += 32 * V) {
      const T* from = src + r0 * stride + x;
      T* to = dst + r0 * pitch + x;
      const int last = x < cols ? n : 0;
#pragma unroll 4
      for (int r = r0; r < rows; r += step) {
        cp_async16_or_zero(to, r < last ? from : src, r < last);
        from += step * stride;
        to += step * pitch;
      }
    }
  } else {
    for (int i = lane; i < rows * width; i += 32) {
      const int r = i / width, c = i - r * width;
      dst[r * pitch + c] = r < n && c < cols ? src[r * stride + c] : from_f<T>(0.0f);
    }
  }
}

// ---- a chunk's matrices -----------------------------------------------------------------
constexpr int kSide = kTile + 8;                       // pitch of 16 x 16 matrices of planes
constexpr int kMat = kTile + 4;                        // and of 32-bit numbers
template <typename T, int NP> struct Chunk {           // NP: planes of P
  float beta[kTile], head[kTile], tail[kTile], rk[kTile], rq[kTile];
  float head_k[kTile], head_q[kTile], tail_k[kTile];   // head rk, scale head rq, tail rk
  float g_hi[kTile], g_lo[kTile];                      // running sums of the log decays
  alignas(16) bf16 inv[Planes<T>::kInner][kTile][kSide];         // (I + M beta)^-1
  alignas(16) bf16 p[NP][kTile][kSide];                // P
};
using Scratch = float[2][kTile][kMat];
struct Wide { float m[kTile][kMat], p[kTile][kMat], d[kTile][kMat]; };   // M, P, D as 32-bit numbers

// The chunk's decays, by one warp, from each lane's gates (lane < 16: token lane's log decay and beta,
// zero behind the chunk) and the chunk's resets. Running sums are kept as two floats, of which
// differences lose nothing: the larger halves' is exact where they are close. Decays below e^-104 are
// 0 in 32 bits; -10^4 stands for all of them, and NaN stays.
template <typename T, int NP> __device__ __forceinline__ void decays(Chunk<T, NP>& c, float g, float beta, unsigned marks) {
  const int lane = threadIdx.x & 31;
  double sum = g < -1e4f ? -1e4f : g;
#pragma unroll
  for (int o = 1; o < kTile; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, sum, o, kTile);
    if ((lane & 15) >= o) sum += x;
  }
  const double all = __shfl_sync(0xffffffffu, sum, 15);
  if (lane < kTile) {
    const float hi = static_cast<float>(sum);
    c.g_hi[lane] = hi;
    c.g_lo[lane] = static_cast<float>(sum - hi);
    c.beta[lane] = beta;
    c.head[lane] = marks & ((2u << lane) - 1u) ? 0.0f : exp2_hw(fmaf(hi, kLog2e, kExp2Shift));
    c.tail[lane] = marks >> (lane + 1) ? 0.0f : exp2_hw(fmaf(static_cast<float>(all - sum), kLog2e, kExp2Shift));
  }
}

// The chunk's matrices, by the same warp, from the tiles of K and Q; with kKeep into `wide` too.
// The inverse goes by blocks of 8: [[A, 0], [C, B]]^-1 = [[A', 0], [-B' C A', B']], the blocks' own
// column by column.
template <typename T, int DK, bool kKeep, int NP>
__device__ __forceinline__ void prepare(Chunk<T, NP>& c, Scratch& s, Wide* wide, const bf16* tk, const bf16* tq, unsigned marks, float scale,
                                        int unit) {
  constexpr int NT = Planes<T>::kToken, NI = Planes<T>::kInner;
  using Keys = Tile<T, DK>;
  const int lane = threadIdx.x & 31, row = lane >> 2, col = (lane & 3) * 2;
  float kk[2][4] = {}, qk[2][4] = {};
  {
    float qq[2][4] = {};
    const uint32_t ka = smem_of(tk), qa = smem_of(tq);
    const uint32_t b_at = at_rows(lane, Keys::kPitch), a_at = a_rows(lane, Keys::kPitch);
#pragma unroll
    for (int i = 0; i < DK / 16; ++i) {
      uint32_t ak[NT][4], aq[NT][4], bk[NT][4];
      load_planes<NT, false>(ak, ka + a_at + i * 32, Keys::kPlane * 2);
      load_planes<NT, false>(aq, qa + a_at + i * 32, Keys::kPlane * 2);
      load_planes<NT, false>(bk, ka + b_at + i * 32, Keys::kPlane * 2);
      mma_planes<NT, NT>(kk[0], kk[1], ak, bk);
      mma_planes<NT, NT>(qk[0], qk[1], aq, bk);
      if (unit) {
        load_planes<NT, false>(bk, qa + b_at + i * 32, Keys::kPlane * 2);
        mma_planes<NT, NT>(qq[0], qq[1], aq, bk);
      }
    }
    // the lanes that hold the diagonals
    if (row == col || row == col + 1) {
      const bool odd = row != col;
      c.rk[row] = unit ? rsqrtf((odd ? kk[0][1] : kk[0][0]) + kNormEps) : 1.0f;
      c.rk[row + 8] = unit ? rsqrtf((odd ? kk[1][3] : kk[1][2]) + kNormEps) : 1.0f;
      c.rq[row] = unit ? rsqrtf((odd ? qq[0][1] : qq[0][0]) + kNormEps) : 1.0f;
      c.rq[row + 8] = unit ? rsqrtf((odd ? qq[1][3] : qq[1][2]) + kNormEps) : 1.0f;
    }
  }
  __syncwarp();
  if (lane < kTile) {
    const float rk = c.rk[lane], head = c.head[lane];
    c.head_k[lane] = head * rk;
    c.head_q[lane] = scale * head * c.rq[lane];
    c.tail_k[lane] = c.tail[lane] * rk;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = row + 8 * r;
    const float hi = c.g_hi[i], lo = c.g_lo[i], rk = c.rk[i], rq = scale * c.rq[i];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int j = 8 * t + col;
      float x[2] = {}, y[2] = {}, d[2] = {};
      if (t <= r) {
        const float2 hj = *reinterpret_cast<const float2*>(&c.g_hi[j]), lj = *reinterpret_cast<const float2*>(&c.g_lo[j]);
        const float2 rj = *reinterpret_cast<const float2*>(&c.rk[j]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float sum = (hi - (e ? hj.y : hj.x)) + (lo - (e ? lj.y : lj.x));
          const float dec = exp2_hw(fmaf(sum, kLog2e, kExp2Shift)), f = dec * (e ? rj.y : rj.x);
          const bool one = i >= j + e && !(marks & ((2u << i) - 1u) & ~((2u << (j + e)) - 1u));          // episode
          d[e] = one ? dec : 0.0f;
          x[e] = one && i > j + e ? kk[t][2 * r + e] * (f * rk) : 0.0f;
          y[e] = one ? qk[t][2 * r + e] * (f * rq) : 0.0f;
        }
      }
      const float2 bj = *reinterpret_cast<const float2*>(&c.beta[j]);
      *reinterpret_cast<float2*>(&s[0][i][j]) = make_float2(x[0] * bj.x, x[1] * bj.y);
      uint32_t p[NP];
      split2<NP>(y[0], y[1], p);
#pragma unroll
      for (int n = 0; n < NP; ++n) *reinterpret_cast<uint32_t*>(&c.p[n][i][j]) = p[n];
      if constexpr (kKeep) {
        *reinterpret_cast<float2*>(&wide->m[i][j]) = make_float2(x[0], x[1]);
        *reinterpret_cast<float2*>(&wide->p[i][j]) = make_float2(y[0], y[1]);
        *reinterpret_cast<float2*>(&wide->d[i][j]) = make_float2(d[0], d[1]);
      }
    }
  }
  __syncwarp();
  if (lane < kTile) {
    const int b = lane & 8, j = lane & 7;
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = i == j ? 1.0f : 0.0f;
      const float4 lo = *reinterpret_cast<const float4*>(&s[0][b + i][b]), hi = *reinterpret_cast<const float4*>(&s[0][b + i][b + 4]);
      const float a[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int e = 0; e < i; ++e) v = fmaf(-a[e], t[e], v);
      t[i] = v;
      s[1][b + i][b + j] = v;
    }
  }
  __syncwarp();
  const int j = lane & 7, r0 = (lane >> 3) * 2;
  auto product = [&](const float* left, int pitch_r, const float* right, float& x, float& y) {
    x = y = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const float4 l0 = *reinterpret_cast<const float4*>(left + r0 * kMat + e), l1 = *reinterpret_cast<const float4*>(left + (r0 + 1) * kMat + e);
      const float* r = right + e * pitch_r + j;
      const float b0 = r[0], b1 = r[pitch_r], b2 = r[2 * pitch_r], b3 = r[3 * pitch_r];
      x = fmaf(l0.x, b0, fmaf(l0.y, b1, fmaf(l0.z, b2, fmaf(l0.w, b3, x))));
      y = fmaf(l1.x, b0, fmaf(l1.y, b1, fmaf(l1.z, b2, fmaf(l1.w, b3, y))));
    }
  };
  float x, y;
  product(&s[0][8][0], kMat, &s[1][0][0], x, y);       // C A'
  s[0][r0][8 + j] = x;
  s[0][r0 + 1][8 + j] = y;
  __syncwarp();
  product(&s[1][8][8], kMat, &s[0][0][8], x, y);
  s[1][8 + r0][j] = -x;
  s[1][8 + r0 + 1][j] = -y;
  __syncwarp();
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float2 v = t <= r ? *reinterpret_cast<const float2*>(&s[1][row + 8 * r][8 * t + col]) : make_float2(0.0f, 0.0f);
      uint32_t p[NI];
      split2<NI>(v.x, v.y, p);
#pragma unroll
      for (int n = 0; n < NI; ++n) *reinterpret_cast<uint32_t*>(&c.inv[n][row + 8 * r][8 * t + col]) = p[n];
    }
  __syncwarp();
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
// A[h]; -inf as the lowest finite number, so that a step of zero decays by e^0. NaN stays.
__device__ __forceinline__ float rate_at(const float* A, int h) { return A[h] < -3.4028235e38f ? -3.4028235e38f : A[h]; }

// The resets of the tile at t (bit i: token t + i), as each lane's own flag, on its way until it is
// asked for by all lanes of the warp.
struct Marks {
  const uint8_t* reset;
  int length;
  unsigned coming;
  __device__ __forceinline__ void look(int t) {
    const int lane = threadIdx.x & 31;
    coming = reset && t >= 0 && lane < kTile && t + lane < length ? reset[t + lane] : 0u;
  }
  __device__ __forceinline__ unsigned get() const { return __ballot_sync(0xffffffffu, coming != 0); }
};

// Whether a warp's tile (rows of `pitch` elements, `width` of them, on 16-byte boundaries) holds a number
// that is not finite: 0 times it is not 0.
template <typename T> __device__ __forceinline__ bool not_finite(const T* tile, int pitch, int width, int n) {
  constexpr int V = kVec16<T>;
  const int lane = threadIdx.x & 31, per = width / V;
  float bad = 0.0f;
  for (int i = lane; i < n * per; i += 32) {
    float v[V];
    load_vec<T, V>(tile + i / per * pitch + i % per * V, v);
#pragma unroll
    for (int j = 0; j < V; ++j) bad = fmaf(v[j], 0.0f, bad);
  }
  return __any_sync(0xffffffffu, bad != 0.0f);
}

// ---- hardware barriers by number ----------------------------------------------------------
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

}  // namespace delta
