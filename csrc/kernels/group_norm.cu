// group_norm.cu — group norm with an activation on channels-last tensors, and its
// gradient (sm_100a).
//
// x [N, P, C]: N samples of P positions of C channels, G groups of C / G channels. With mean
// and rstd = 1 / sqrt(var + eps) over a sample's P positions and a group's channels,
//   xh = (x - mean) rstd,  pre = xh w[c] + b[c],  y = act(pre),
// and for the gradient d = dy act'(pre), a = d w:
//   dx = rstd (a - mean(a) - xh mean(a xh)),  dw[c] = sum d xh,  db[c] = sum d.
//
// The variance is the mean square distance from the mean, from a second look at the values
// that the first left in registers or shared memory; parts are joined by their counts, means
// and square sums. Sums are 32-bit, in a fixed order: no atomics.
//
// A piece is V consecutive channels of one group (V divides C / G), loaded at once. Three forms:
//   lanes  a (sample, group) of at most 4 pieces for each of L <= 32 lanes: a warp's registers;
//   block  a sample's slab of whole groups, at most 8 (gradient: 4) pieces a thread: a block's registers;
//   parts  anything larger, or too few slabs for the GPU: a pass over parts for their
//          statistics (or sums), one that applies them.
// Forward and gradient, bfloat16: 32768x512 g8 20 + 37 us (lanes; 0.52 and 0.42 of the copy rate, short
// kernels on what is partly in the L2 cache), 2048x512x64 g8 79 + 135 (block; 0.52 and 0.46: the sums'
// barriers, and rows of 32 bytes).
// In the first two x and dy are read once: a thread's loads are all on their way before the first is
// used, which is what keeps memory busy.
#include "seq_common.cuh"

namespace {

using namespace seqk;

enum : int { kNone = 0, kRelu = 1, kSilu = 2 };

struct NormArgs {
  const void *x, *dy;
  const float *w, *b;          // [C] or null
  void* y;                     // forward: y; gradient: dx
  float* stats;                // [N, G, 2]: mean, rstd
  float* part;                 // the parts' statistics, or the channels' sums
  float *dw, *db;
  int64_t xs_n, xs_p, ds_n, ds_p, ys_n, ys_p;
  int64_t n, p;
  int c, g;
  float eps;
  int act;
  int slab, parts;             // groups of a slab; parts of a sample (or blocks along the samples)
  int64_t span;                // positions of a part
};
static_assert(sizeof(NormArgs) == 9 * 8 + 8 * 8 + 6 * 4 + 8, "as the caller packs it");

// V numbers; from two on in pairs, one instruction for both.
template <int V> struct Nums {
  f2 p[V / 2];
  template <typename F> __device__ __forceinline__ static Nums of(F f) {
    Nums r;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = f(i);
    return r;
  }
  __device__ __forceinline__ static Nums all(float x) { return of([&](int) { return pack2(x, x); }); }
  __device__ __forceinline__ static Nums get(const float (&v)[V]) { return of([&](int i) { return pack2(v[2 * i], v[2 * i + 1]); }); }
  __device__ __forceinline__ void put(float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) unpack2(p[i], v[2 * i], v[2 * i + 1]);
  }
  template <typename F> __device__ __forceinline__ Nums each(F f) const {
    return of([&](int i) {
      float a, b;
      unpack2(p[i], a, b);
      return pack2(f(a), f(b));
    });
  }
  __device__ __forceinline__ float sum() const {
    f2 s = p[0];
#pragma unroll
    for (int i = 1; i < V / 2; ++i) s = add2(s, p[i]);
    float a, b;
    unpack2(s, a, b);
    return a + b;
  }
};
template <> struct Nums<1> {
  float p;
  __device__ __forceinline__ static Nums all(float x) { return {x}; }
  __device__ __forceinline__ static Nums get(const float (&v)[1]) { return {v[0]}; }
  __device__ __forceinline__ void put(float (&v)[1]) const { v[0] = p; }
  template <typename F> __device__ __forceinline__ Nums each(F f) const { return {f(p)}; }
  __device__ __forceinline__ float sum() const { return p; }
};
template <int V> __device__ __forceinline__ Nums<V> operator+(const Nums<V>& a, const Nums<V>& b) {
  if constexpr (V == 1) return {a.p + b.p};
  else return Nums<V>::of([&](int i) { return add2(a.p[i], b.p[i]); });
}
template <int V> __device__ __forceinline__ Nums<V> operator*(const Nums<V>& a, const Nums<V>& b) {
  if constexpr (V == 1) return {a.p * b.p};
  else return Nums<V>::of([&](int i) { return mul2(a.p[i], b.p[i]); });
}
template <int V> __device__ __forceinline__ Nums<V> fma(const Nums<V>& a, const Nums<V>& b, const Nums<V>& c) {
  if constexpr (V == 1) return {fmaf(a.p, b.p, c.p)};
  else return Nums<V>::of([&](int i) { return fma2(a.p[i], b.p[i], c.p[i]); });
}
template <int V> __device__ __forceinline__ Nums<V> sigmoid_of(const Nums<V>& v) {
  return ((v * Nums<V>::all(-kLog2e)).each([](float x) { return exp2_hw(x); }) + Nums<V>::all(1.0f)).each([](float x) { return rcp_hw(x); });
}

// act(xh w + b) with xh = (x - mean) rstd; NaN stays under relu
template <int V>
__device__ __forceinline__ Nums<V> apply(const Nums<V>& x, float mean, float rstd, const Nums<V>& w, const Nums<V>& b, int act) {
  const Nums<V> pre = fma((x + Nums<V>::all(-mean)) * Nums<V>::all(rstd), w, b);
  if (act == kSilu) return pre * sigmoid_of(pre);
  return act == kRelu ? pre.each([](float v) { return v < 0.0f ? 0.0f : v; }) : pre;
}
// dy act'(pre)
template <int V>
__device__ __forceinline__ Nums<V> gradient(const Nums<V>& x, const Nums<V>& dy, float mean, float rstd, const Nums<V>& w, const Nums<V>& b,
                                            int act, Nums<V>& xh) {
  const Nums<V> one = Nums<V>::all(1.0f);
  xh = (x + Nums<V>::all(-mean)) * Nums<V>::all(rstd);
  if (act == kNone) return dy;
  const Nums<V> pre = fma(xh, w, b);
  if (act == kRelu) return dy * pre.each([](float v) { return v > 0.0f ? 1.0f : 0.0f; });
  const Nums<V> s = sigmoid_of(pre);
  return dy * (s * fma(pre, fma(s, Nums<V>::all(-1.0f), one), one));
}

// (count, mean, sum of squares about it) of two sets
struct Moments { float n, mean, m2; };
__device__ __forceinline__ Moments join(const Moments& a, const Moments& b) {
  const float n = a.n + b.n;
  if (n == 0.0f) return a;
  const float d = b.mean - a.mean, f = b.n / n;
  return {n, fmaf(d, f, a.mean), a.m2 + b.m2 + d * d * a.n * f};
}

template <int L> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---- pieces in registers ------------------------------------------------------------------
// A piece as it was loaded.
template <typename T, int V> struct Piece {
  static constexpr int kWords = V * static_cast<int>(sizeof(T)) < 4 ? 1 : V * static_cast<int>(sizeof(T)) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) * V == 16) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (sizeof(T) * V == 8) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    else if constexpr (sizeof(T) * V == 4) w[0] = *reinterpret_cast<const uint32_t*>(p);
    else w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ Nums<V> get() const {
    float v[V];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = __uint_as_float(w[i]);
    } else if constexpr (V == 1) {
      v[0] = __uint_as_float(w[0] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
    return Nums<V>::get(v);
  }
};
template <typename T, int V> __device__ __forceinline__ void store(T* p, const Nums<V>& x) {
  float v[V];
  x.put(v);
  store_vec<T, V>(p, v);
}
template <typename T, int V> __device__ __forceinline__ Nums<V> load(const T* p) {
  Piece<T, V> r;
  r.load(p);
  return r.get();
}
template <int V> struct Weights {
  Nums<V> w, b;
  __device__ __forceinline__ void load(const float* pw, const float* pb, int c, bool on) {
    float x[V], y[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      x[j] = pw && on ? pw[c + j] : 1.0f;
      y[j] = pb && on ? pb[c + j] : 0.0f;
    }
    w = Nums<V>::get(x);
    b = Nums<V>::get(y);
  }
};

// ---- lanes ------------------------------------------------------------------------------
constexpr int kLaneThreads = 256;

// L lanes for a (sample, group): lane l holds pieces l, l + L, ... of at most H L; piece q is position
// q / (pieces of a group), whose channels follow. A block's warps take the samples of one set of
// 32 / L groups in turn, several at a time where a lane has one piece, so that a lane's channels stay
// the same and their sums stay in registers.
template <typename T, int V, int L, int H, bool kGrad>
__global__ void __launch_bounds__(kLaneThreads) norm_lanes(NormArgs a) {
  constexpr int kSets = 32 / L, kWarps = kLaneThreads / 32, U = H == 1 ? (kGrad ? 2 : 4) : 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % L;
  const int gi = blockIdx.x * kSets + lane / L, cg = a.c / a.g, per = cg / V;
  const int items = static_cast<int>(a.p) * per;
  const bool on = gi < a.g;
  int64_t xo[H], dofs[H], yo[H];
  bool have[H];
  Weights<V> wb[H];
#pragma unroll
  for (int k = 0; k < H; ++k) {
    const int q = l + k * L;
    have[k] = on && q < items;
    const int pos = have[k] ? q / per : 0, c = have[k] ? gi * cg + (q - pos * per) * V : 0;
    xo[k] = pos * a.xs_p + c;
    dofs[k] = pos * a.ds_p + c;
    yo[k] = pos * a.ys_p + c;
    wb[k].load(a.w, a.b, c, have[k]);
  }
  const float inv = 1.0f / (static_cast<float>(a.p) * cg);
  Nums<V> sw[kGrad ? H : 1], sb[kGrad ? H : 1];
#pragma unroll
  for (int k = 0; k < (kGrad ? H : 1); ++k) sw[k] = sb[k] = Nums<V>::all(0.0f);
  const int64_t step = static_cast<int64_t>(gridDim.y) * kWarps;
  for (int64_t n0 = static_cast<int64_t>(blockIdx.y) * kWarps + warp; n0 < a.n; n0 += U * step) {
    Piece<T, V> rx[U][H], rd[U][H];
    float2 st[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = n0 + u * step;
      const bool live = n < a.n;
#pragma unroll
      for (int k = 0; k < H; ++k) {
        if (live && have[k]) rx[u][k].load(static_cast<const T*>(a.x) + n * a.xs_n + xo[k]);
        else rx[u][k].zero();
        if constexpr (kGrad) {
          if (live && have[k]) rd[u][k].load(static_cast<const T*>(a.dy) + n * a.ds_n + dofs[k]);
          else rd[u][k].zero();
        }
      }
      st[u] = make_float2(0.0f, 0.0f);
      if (kGrad && live && on) st[u] = *reinterpret_cast<const float2*>(a.stats + (n * a.g + gi) * 2);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = n0 + u * step;
      const bool live = n < a.n;
      T* y = static_cast<T*>(a.y) + n * a.ys_n;
      if constexpr (!kGrad) {
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int k = 0; k < H; ++k) s += rx[u][k].get().sum();
        const float mean = lanes_sum<L>(s) * inv;
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const Nums<V> d = rx[u][k].get() + Nums<V>::all(-mean);
          if (have[k]) q += (d * d).sum();
        }
        const float rstd = rsqrtf(lanes_sum<L>(q) * inv + a.eps);
        if (a.stats && live && on && l == 0) *reinterpret_cast<float2*>(a.stats + (n * a.g + gi) * 2) = make_float2(mean, rstd);
#pragma unroll
        for (int k = 0; k < H; ++k)
          if (live && have[k]) store<T, V>(y + yo[k], apply<V>(rx[u][k].get(), mean, rstd, wb[k].w, wb[k].b, a.act));
      } else {
        // pieces that are not there have dy = 0
        Nums<V> xh[H], d[H];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const Nums<V> e = gradient<V>(rx[u][k].get(), rd[u][k].get(), st[u].x, st[u].y, wb[k].w, wb[k].b, a.act, xh[k]);
          sw[k] = fma(e, xh[k], sw[k]);
          sb[k] = sb[k] + e;
          d[k] = e * wb[k].w;
          s1 += d[k].sum();
          s2 += (d[k] * xh[k]).sum();
        }
        const float m1 = lanes_sum<L>(s1) * inv, m2 = lanes_sum<L>(s2) * inv;
#pragma unroll
        for (int k = 0; k < H; ++k)
          if (live && have[k])
            store<T, V>(y + yo[k], (d[k] + fma(xh[k], Nums<V>::all(-m2), Nums<V>::all(-m1))) * Nums<V>::all(st[u].y));
      }
    }
  }
  if constexpr (kGrad) {
    // the block's channels: warps, and positions of a channel in order
    __shared__ float sum[kWarps][32 * H * V + 1];
    float* out = a.part + static_cast<int64_t>(blockIdx.y) * 2 * a.c;
    const int width = min(kSets, a.g - static_cast<int>(blockIdx.x) * kSets) * cg;
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < H; ++k) {
        float v[V];
        (turn ? sb[k] : sw[k]).put(v);
#pragma unroll
        for (int j = 0; j < V; ++j) sum[warp][(lane / L * L * H + l + k * L) * V + j] = v[j];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < width; c += kLaneThreads) {
        const int set = c / cg, in = c - set * cg;
        float s = 0.0f;
        for (int i = 0; i < kWarps; ++i)
          for (int pos = 0; pos < static_cast<int>(a.p); ++pos) s += sum[i][set * L * H * V + pos * cg + in];
        out[turn * a.c + blockIdx.x * kSets * cg + c] = s;
      }
    }
  }
}

// ---- blocks -----------------------------------------------------------------------------
constexpr int kBlockThreads = 512;                     // at most

// v summed over the threads of each of the slab's groups; res[group] for all threads. Thread t <
// walkers stands at piece t % per of its row; the order of the sum is the threads'. The block is
// whole warps.
__device__ __forceinline__ void sum_groups(float v, float* red, float* res, int groups, int per, int per_group, int walkers) {
  __syncthreads();
  red[threadIdx.x] = static_cast<int>(threadIdx.x) < walkers ? v : 0.0f;
  __syncthreads();
  const int lane = threadIdx.x & 31, warps = blockDim.x / 32, rows = walkers / per;
  for (int g = threadIdx.x >> 5; g < groups; g += warps) {
    float s = 0.0f;
    for (int i = lane; i < rows * per_group; i += 32) {
      const int r = i / per_group;
      s += red[r * per + g * per_group + i - r * per_group];
    }
    s = lanes_sum<32>(s);
    if (lane == 0) res[g] = s;
  }
  __syncthreads();
}

// The place of a thread in a slab of `groups` groups: rows of `per` pieces, a piece of its own.
struct Place {
  int per_group, g0, groups, per, c0, rows, walkers, piece, row, own;
  bool on;
  __device__ __forceinline__ Place(const NormArgs& a, int slab_index, int vec) {
    const int cg = a.c / a.g;
    per_group = cg / vec;
    g0 = slab_index * a.slab;
    groups = min(a.slab, a.g - g0);
    per = groups * per_group;
    rows = static_cast<int>(blockDim.x) / per;
    walkers = rows * per;
    row = static_cast<int>(threadIdx.x) / per;
    piece = static_cast<int>(threadIdx.x) - row * per;
    own = piece / per_group;
    c0 = g0 * cg + piece * vec;
    on = static_cast<int>(threadIdx.x) < walkers;
  }
};

// A thread's pieces of a sample on their way to places of its own in shared memory, a sample ahead;
// pieces of two bytes are loaded when they are needed.
template <typename T, int V, int H> struct Ahead {
  static constexpr int kBytes = V * static_cast<int>(sizeof(T));
  static constexpr bool kAsync = kBytes >= 4;
  static __device__ __forceinline__ void copy(char* to, const T* from, int64_t step, int count) {
    if constexpr (kAsync) {
#pragma unroll
      for (int k = 0; k < H; ++k)
        if (k < count) {
          const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to + static_cast<size_t>(k * blockDim.x) * kBytes));
          if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from + k * step) : "memory");
          else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from + k * step), "n"(kBytes) : "memory");
        }
    }
  }
  static __device__ __forceinline__ void take(Piece<T, V> (&r)[H], const char* from, const T* memory, int64_t step, int count) {
#pragma unroll
    for (int k = 0; k < H; ++k) {
      if (k >= count) r[k].zero();
      else if constexpr (kAsync) r[k].load(reinterpret_cast<const T*>(from + static_cast<size_t>(k * blockDim.x) * kBytes));
      else r[k].load(memory + k * step);
    }
  }
};

// A slab of samples blockIdx.x / slabs, + gridDim.x / slabs, ... (slabs are the faster index, so that a
// sample's are read together); the next sample is on its way while one is normalised.
template <typename T, int V, int H> __global__ void __launch_bounds__(kBlockThreads) norm_block(NormArgs a) {
  using A = Ahead<T, V, H>;
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[kBlockThreads], res[kBlockThreads];
  const int slabs = (a.g + a.slab - 1) / a.slab;
  const Place at(a, blockIdx.x % slabs, V);
  const int64_t blocks = gridDim.x / slabs;
  const float inv = 1.0f / (static_cast<float>(a.p) * (a.c / a.g));
  const int count = at.on ? max(0, static_cast<int>((a.p - at.row + at.rows - 1) / at.rows)) : 0;       // this thread's pieces
  const T* x = static_cast<const T*>(a.x) + at.row * a.xs_p + at.c0;
  const int64_t step = at.rows * a.xs_p;
  char* mine = smem + threadIdx.x * A::kBytes;
  const size_t turn = static_cast<size_t>(H) * blockDim.x * A::kBytes;
  Weights<V> wb;
  wb.load(a.w, a.b, at.c0, at.on);
  const int64_t first = blockIdx.x / slabs;
  if (first < a.n) A::copy(mine, x + first * a.xs_n, step, count);
  cp_async_commit();
  int odd = 0;
  for (int64_t n = first; n < a.n; n += blocks, odd ^= 1) {
    if (n + blocks < a.n) A::copy(mine + (odd ^ 1) * turn, x + (n + blocks) * a.xs_n, step, count);
    cp_async_commit();
    cp_async_wait<1>();
    Piece<T, V> r[H];
    A::take(r, mine + odd * turn, x + n * a.xs_n, step, count);
    Nums<V> s = Nums<V>::all(0.0f);
#pragma unroll
    for (int k = 0; k < H; ++k) s = s + r[k].get();
    sum_groups(s.sum(), red, res, at.groups, at.per, at.per_group, at.walkers);
    const float mean = res[at.own] * inv;
    s = Nums<V>::all(0.0f);
#pragma unroll
    for (int k = 0; k < H; ++k)
      if (k < count) {
        const Nums<V> d = r[k].get() + Nums<V>::all(-mean);
        s = fma(d, d, s);
      }
    sum_groups(s.sum(), red, res, at.groups, at.per, at.per_group, at.walkers);
    const float rstd = rsqrtf(res[at.own] * inv + a.eps);
    if (a.stats && at.on && at.row == 0 && at.piece % at.per_group == 0)
      *reinterpret_cast<float2*>(a.stats + (n * a.g + at.g0 + at.own) * 2) = make_float2(mean, rstd);
    T* y = static_cast<T*>(a.y) + n * a.ys_n + at.row * a.ys_p + at.c0;
#pragma unroll
    for (int k = 0; k < H; ++k)
      if (k < count) store<T, V>(y + k * (at.rows * a.ys_p), apply<V>(r[k].get(), mean, rstd, wb.w, wb.b, a.act));
  }
}

// The rows' sums of each of `per` pieces, from threads row * per + piece, to out[0 .. ] and out[c .. ] for columns
// below `cols`: through 2 V floats a thread of shared memory, with as many lanes an output as there are rows, 32 at
// most (by one thread an output the rows' chain took 15 us at 128 rows).
template <int V> __device__ __forceinline__ void sum_rows(const Nums<V>& sw, const Nums<V>& sb, float* all, int rows, int per, int cols,
                                                          int c, float* out) {
  float both[2][V];
  sw.put(both[0]);
  sb.put(both[1]);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    all[j * blockDim.x + threadIdx.x] = both[0][j];
    all[(V + j) * blockDim.x + threadIdx.x] = both[1][j];
  }
  __syncthreads();
  int share = 32;
  while (share > rows) share >>= 1;
  const int outs = per * 2 * V, lane = threadIdx.x & 31;
  for (int first = (threadIdx.x & ~31u) / share; first < outs; first += blockDim.x / share) {
    const int o = first + lane / share, piece = o % per, slot = o / per;
    float s = 0.0f;
    if (o < outs)
      for (int i = lane % share; i < rows; i += share) s += all[slot * blockDim.x + i * per + piece];
    for (int x = share >> 1; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    if (o < outs && lane % share == 0 && piece * V < cols) out[(slot >= V ? c : 0) + piece * V + slot % V] = s;
  }
}

// Its gradient, x and dy a sample ahead.
template <typename T, int V, int H> __global__ void __launch_bounds__(kBlockThreads / 2, 2) norm_block_grad(NormArgs a) {
  using A = Ahead<T, V, H>;
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[kBlockThreads / 2], res[kBlockThreads / 2];
  const int slabs = (a.g + a.slab - 1) / a.slab, blocks = gridDim.x / slabs, block = blockIdx.x / slabs;
  const Place at(a, blockIdx.x % slabs, V);
  const float inv = 1.0f / (static_cast<float>(a.p) * (a.c / a.g));
  const int count = at.on ? max(0, static_cast<int>((a.p - at.row + at.rows - 1) / at.rows)) : 0;
  const T* x = static_cast<const T*>(a.x) + at.row * a.xs_p + at.c0;
  const T* dy = static_cast<const T*>(a.dy) + at.row * a.ds_p + at.c0;
  const int64_t xstep = at.rows * a.xs_p, dstep = at.rows * a.ds_p;
  char* mine = smem + threadIdx.x * A::kBytes;
  const size_t half = static_cast<size_t>(H) * blockDim.x * A::kBytes, turn = 2 * half;
  Weights<V> wb;
  wb.load(a.w, a.b, at.c0, at.on);
  Nums<V> sw = Nums<V>::all(0.0f), sb = sw;
  if (block < a.n) {
    A::copy(mine, x + block * a.xs_n, xstep, count);
    A::copy(mine + half, dy + block * a.ds_n, dstep, count);
  }
  cp_async_commit();
  int odd = 0;
  for (int64_t n = block; n < a.n; n += blocks, odd ^= 1) {
    if (n + blocks < a.n) {
      A::copy(mine + (odd ^ 1) * turn, x + (n + blocks) * a.xs_n, xstep, count);
      A::copy(mine + (odd ^ 1) * turn + half, dy + (n + blocks) * a.ds_n, dstep, count);
    }
    cp_async_commit();
    const float2 st = *reinterpret_cast<const float2*>(a.stats + (n * a.g + at.g0 + at.own) * 2);
    cp_async_wait<1>();
    Piece<T, V> rx[H], rd[H];
    A::take(rx, mine + odd * turn, x + n * a.xs_n, xstep, count);
    A::take(rd, mine + odd * turn + half, dy + n * a.ds_n, dstep, count);
    Nums<V> xh[H], d[H], s1 = Nums<V>::all(0.0f), s2 = s1;       // pieces that are not there have dy = 0
#pragma unroll
    for (int k = 0; k < H; ++k) {
      const Nums<V> e = gradient<V>(rx[k].get(), rd[k].get(), st.x, st.y, wb.w, wb.b, a.act, xh[k]);
      sw = fma(e, xh[k], sw);
      sb = sb + e;
      d[k] = e * wb.w;
      s1 = s1 + d[k];
      s2 = fma(d[k], xh[k], s2);
    }
    sum_groups(s1.sum(), red, res, at.groups, at.per, at.per_group, at.walkers);
    const float m1 = res[at.own] * inv;
    sum_groups(s2.sum(), red, res, at.groups, at.per, at.per_group, at.walkers);
    const float m2 = res[at.own] * inv;
    T* y = static_cast<T*>(a.y) + n * a.ys_n + at.row * a.ys_p + at.c0;
#pragma unroll
    for (int k = 0; k < H; ++k)
      if (k < count)
        store<T, V>(y + k * (at.rows * a.ys_p), (d[k] + fma(xh[k], Nums<V>::all(-m2), Nums<V>::all(-m1))) * Nums<V>::all(st.y));
  }
  // the channels' sums
  __syncthreads();
  sum_rows<V>(sw, sb, reinterpret_cast<float*>(smem), at.rows, at.per, a.c - at.c0 + at.piece * V, a.c,
              a.part + static_cast<int64_t>(block) * 2 * a.c + at.c0 - at.piece * V);
}

// ---- parts ------------------------------------------------------------------------------
// Moments of the positions of a part: [N, G, parts, 3]. A slab as above, or one group whose pieces are
// more than a block's threads.
template <typename T, int V> __global__ void __launch_bounds__(kBlockThreads) norm_part_stats(NormArgs a) {
  __shared__ float red[kBlockThreads], res[kBlockThreads];
  const Place at(a, blockIdx.y, V);
  const bool wide = at.rows == 0;
  const int cg = a.c / a.g, walkers = wide ? static_cast<int>(blockDim.x) : at.walkers;
  const int64_t n = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t first = part * a.span, last = min(a.p, first + a.span);
  const T* x = static_cast<const T*>(a.x) + n * a.xs_n + at.g0 * cg;
  const float inv = 1.0f / (static_cast<float>(last - first) * cg);
  auto each = [&](auto f) {
    if (wide) {
      for (int64_t p = first; p < last; ++p)
        for (int i = threadIdx.x; i < at.per; i += blockDim.x) f(x + p * a.xs_p + i * V);
    } else if (at.on) {
#pragma unroll 4
      for (int64_t p = first + at.row; p < last; p += at.rows) f(x + p * a.xs_p + at.piece * V);
    }
  };
  const int group_pieces = wide ? 1 : at.per_group, row_pieces = wide ? 1 : at.per, own = wide ? 0 : at.own;
  Nums<V> s = Nums<V>::all(0.0f);
  each([&](const T* from) { s = s + load<T, V>(from); });
  sum_groups(s.sum(), red, res, at.groups, row_pieces, group_pieces, walkers);
  const float mean = res[own] * inv;
  s = Nums<V>::all(0.0f);
  each([&](const T* from) {
    const Nums<V> d = load<T, V>(from) + Nums<V>::all(-mean);
    s = fma(d, d, s);
  });
  sum_groups(s.sum(), red, res, at.groups, row_pieces, group_pieces, walkers);
  if (wide ? threadIdx.x == 0 : at.on && at.row == 0 && at.piece % at.per_group == 0) {
    float* out = a.part + ((n * a.g + at.g0 + own) * a.parts + part) * 3;
    out[0] = static_cast<float>(last - first) * cg;
    out[1] = mean;
    out[2] = res[own];
  }
}

// (mean, rstd) of group g of sample n from its parts by one warp: a lane's in order, then lane by lane.
__device__ __forceinline__ float2 joined(const NormArgs& a, int64_t n, int g) {
  const float* m = a.part + (n * a.g + g) * a.parts * 3;
  Moments all{0.0f, 0.0f, 0.0f};
  for (int i = threadIdx.x & 31; i < a.parts; i += 32) all = join(all, {m[3 * i], m[3 * i + 1], m[3 * i + 2]});
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    Moments x = all, y{__shfl_xor_sync(0xffffffffu, all.n, o), __shfl_xor_sync(0xffffffffu, all.mean, o), __shfl_xor_sync(0xffffffffu, all.m2, o)};
    all = threadIdx.x & o ? join(y, x) : join(x, y);   // both lanes the same, to the bit
  }
  return make_float2(all.mean, rsqrtf(all.m2 / all.n + a.eps));
}

template <typename T, int V> __global__ void __launch_bounds__(kBlockThreads) norm_part_apply(NormArgs a) {
  __shared__ float2 st[kBlockThreads];
  const Place at(a, blockIdx.y, V);
  const bool wide = at.rows == 0;
  const int cg = a.c / a.g;
  const int64_t n = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t first = part * a.span, last = min(a.p, first + a.span);
  for (int i = threadIdx.x >> 5; i < at.groups; i += blockDim.x / 32) {
    const float2 v = joined(a, n, at.g0 + i);
    if (threadIdx.x & 31) continue;
    st[i] = v;
    if (a.stats && part == 0) *reinterpret_cast<float2*>(a.stats + (n * a.g + at.g0 + i) * 2) = v;
  }
  __syncthreads();
  const float2 m = st[wide ? 0 : at.own];
  const T* x = static_cast<const T*>(a.x) + n * a.xs_n + at.g0 * cg;
  T* y = static_cast<T*>(a.y) + n * a.ys_n + at.g0 * cg;
  auto one = [&](int64_t p, int i, const Weights<V>& wb) {
    store<T, V>(y + p * a.ys_p + i * V, apply<V>(load<T, V>(x + p * a.xs_p + i * V), m.x, m.y, wb.w, wb.b, a.act));
  };
  Weights<V> wb;
  if (wide) {
    for (int i = threadIdx.x; i < at.per; i += blockDim.x) {
      wb.load(a.w, a.b, at.g0 * cg + i * V, true);
      for (int64_t p = first; p < last; ++p) one(p, i, wb);
    }
  } else if (at.on) {
    wb.load(a.w, a.b, at.c0, true);
#pragma unroll 4
    for (int64_t p = first + at.row; p < last; p += at.rows) one(p, at.piece, wb);
  }
}

// A block of the gradient by parts: 32 pieces of channels by 8 positions, or fewer by more where
// the channels are fewer.
constexpr int kPartThreads = 256;
struct Cells {
  int cols, rows, piece, row;
  __device__ __forceinline__ explicit Cells(int pieces) {
    int log = 5;
    while (log > 0 && 1 << (log - 1) >= pieces) --log;
    cols = 1 << log;
    rows = kPartThreads >> log;
    piece = threadIdx.x & (cols - 1);
    row = threadIdx.x >> log;
  }
};

// Sums of d xh and d over the positions of a part: [N, parts, 2, C].
template <typename T, int V> __global__ void __launch_bounds__(kPartThreads) norm_part_sums(NormArgs a) {
  const int cg = a.c / a.g;
  const int64_t n = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t first = part * a.span, last = min(a.p, first + a.span);
  __shared__ float all[2 * V * kPartThreads];
  const Cells at(a.c / V);
  const int col0 = blockIdx.y * 32 * V, col = col0 + at.piece * V;
  const bool on = col < a.c;
  Nums<V> sw = Nums<V>::all(0.0f), sb = sw;
  Weights<V> wb;
  wb.load(a.w, a.b, col, on);
  if (on) {
    const float2 st = *reinterpret_cast<const float2*>(a.stats + (n * a.g + col / cg) * 2);
    const T* x = static_cast<const T*>(a.x) + n * a.xs_n + col;
    const T* dy = static_cast<const T*>(a.dy) + n * a.ds_n + col;
#pragma unroll 2
    for (int64_t p = first + at.row; p < last; p += at.rows) {
      Nums<V> xh;
      const Nums<V> e = gradient<V>(load<T, V>(x + p * a.xs_p), load<T, V>(dy + p * a.ds_p), st.x, st.y, wb.w, wb.b, a.act, xh);
      sw = fma(e, xh, sw);
      sb = sb + e;
    }
  }
  sum_rows<V>(sw, sb, all, at.rows, at.cols, a.c - col0, a.c, a.part + blockIdx.x * static_cast<int64_t>(2 * a.c) + col0);
}

// From those, of every (sample, group): mean(a), mean(a xh): [N, G, 2] behind the parts' sums.
__global__ void __launch_bounds__(128) norm_part_means(NormArgs a, float* means) {
  const int cg = a.c / a.g;
  const int64_t n = blockIdx.x / a.g;
  const int g = static_cast<int>(blockIdx.x % a.g);
  __shared__ float red[4][2];
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t i = threadIdx.x; i < static_cast<int64_t>(a.parts) * cg; i += 128) {
    const int part = static_cast<int>(i / cg), c = g * cg + static_cast<int>(i - static_cast<int64_t>(part) * cg);
    const float* s = a.part + (n * a.parts + part) * 2 * a.c;
    const float w = a.w ? a.w[c] : 1.0f;
    s1 = fmaf(s[a.c + c], w, s1);
    s2 = fmaf(s[c], w, s2);
  }
  s1 = lanes_sum<32>(s1);
  s2 = lanes_sum<32>(s2);
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5][0] = s1;
    red[threadIdx.x >> 5][1] = s2;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    const float inv = 1.0f / (static_cast<float>(a.p) * cg);
    means[blockIdx.x * 2 + threadIdx.x] =
        ((red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x])) * inv;
  }
}

template <typename T, int V> __global__ void __launch_bounds__(kPartThreads) norm_part_grad(NormArgs a, const float* means) {
  const int cg = a.c / a.g;
  const int64_t n = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t first = part * a.span, last = min(a.p, first + a.span);
  const Cells cell(a.c / V);
  const int col = (blockIdx.y * 32 + cell.piece) * V;
  if (col >= a.c) return;
  const int64_t at = (n * a.g + col / cg) * 2;
  const float2 st = *reinterpret_cast<const float2*>(a.stats + at);
  const float m1 = means[at], m2 = means[at + 1];
  Weights<V> wb;
  wb.load(a.w, a.b, col, true);
  const T* x = static_cast<const T*>(a.x) + n * a.xs_n + col;
  const T* dy = static_cast<const T*>(a.dy) + n * a.ds_n + col;
  T* y = static_cast<T*>(a.y) + n * a.ys_n + col;
#pragma unroll 2
  for (int64_t p = first + cell.row; p < last; p += cell.rows) {
    Nums<V> xh;
    const Nums<V> e = gradient<V>(load<T, V>(x + p * a.xs_p), load<T, V>(dy + p * a.ds_p), st.x, st.y, wb.w, wb.b, a.act, xh);
    store<T, V>(y + p * a.ys_p, (e * wb.w + fma(xh, Nums<V>::all(-m2), Nums<V>::all(-m1))) * Nums<V>::all(st.y));
  }
}

// dw, db [C] from rows of [2, C] sums, in order: a warp's lanes take every 32nd row.
__global__ void __launch_bounds__(256) norm_channels(const float* part, int64_t rows, int c, float* dw, float* db) {
  const int col = blockIdx.x * 8 + (threadIdx.x & 7), r0 = threadIdx.x >> 3;
  __shared__ float red[32][17];
  float s1 = 0.0f, s2 = 0.0f;
  if (col < c)
    for (int64_t r = r0; r < rows; r += 32) {
      s1 += part[r * 2 * c + col];
      s2 += part[r * 2 * c + c + col];
    }
  red[r0][threadIdx.x & 7] = s1;
  red[r0][8 + (threadIdx.x & 7)] = s2;
  __syncthreads();
  if (threadIdx.x < 16) {
    const int at = blockIdx.x * 8 + (threadIdx.x & 7);
    float s = 0.0f;
    for (int r = 0; r < 32; ++r) s += red[r][threadIdx.x];
    float* out = threadIdx.x < 8 ? dw : db;
    if (out && at < c) out[at] = s;
  }
}

// ---- launches -----------------------------------------------------------------------------
template <typename F> int by_vec(int v, F f) {
  switch (v) {
    case 8: return f(std::integral_constant<int, 8>());
    case 4: return f(std::integral_constant<int, 4>());
    case 2: return f(std::integral_constant<int, 2>());
    case 1: return f(std::integral_constant<int, 1>());
  }
  return static_cast<int>(cudaErrorInvalidValue);
}

template <typename T, int V, int L> int lanes_go(const NormArgs& a, bool grad, int hold, int blocks, cudaStream_t s) {
  const dim3 grid((a.g + 32 / L - 1) / (32 / L), blocks);
  auto go = [&](auto h) {
    constexpr int H = decltype(h)::value;
    if (grad) norm_lanes<T, V, L, H, true><<<grid, kLaneThreads, 0, s>>>(a);
    else norm_lanes<T, V, L, H, false><<<grid, kLaneThreads, 0, s>>>(a);
    return static_cast<int>(cudaGetLastError());
  };
  // fewer lanes than 32 hold one piece each
  if constexpr (L == 32) {
    if (hold == 4) return go(std::integral_constant<int, 4>());
    if (hold == 2) return go(std::integral_constant<int, 2>());
  }
  return hold == 1 ? go(std::integral_constant<int, 1>()) : static_cast<int>(cudaErrorInvalidValue);
}

template <typename T, int V> int lanes_by(const NormArgs& a, bool grad, int lanes, int hold, int blocks, cudaStream_t s) {
  switch (lanes) {
    case 1: return lanes_go<T, V, 1>(a, grad, hold, blocks, s);
    case 2: return lanes_go<T, V, 2>(a, grad, hold, blocks, s);
    case 4: return lanes_go<T, V, 4>(a, grad, hold, blocks, s);
    case 8: return lanes_go<T, V, 8>(a, grad, hold, blocks, s);
    case 16: return lanes_go<T, V, 16>(a, grad, hold, blocks, s);
    case 32: return lanes_go<T, V, 32>(a, grad, hold, blocks, s);
  }
  return static_cast<int>(cudaErrorInvalidValue);
}

// mode 0 lanes, 1 block, 2 parts; threads: of a block (modes 1 and 2); blocks: of the samples
template <typename T, int V> int forward(const NormArgs& a, int mode, int lanes, int hold, int threads, int blocks, cudaStream_t s) {
  if (mode == 0) return lanes_by<T, V>(a, false, lanes, hold, blocks, s);
  const int slabs = (a.g + a.slab - 1) / a.slab;
  if (threads > kBlockThreads || threads % 32) return static_cast<int>(cudaErrorInvalidValue);
  if (mode == 1) {
    auto go = [&](auto h) {
      constexpr int H = decltype(h)::value;
      const size_t bytes = 2 * static_cast<size_t>(H) * threads * V * sizeof(T);       // this sample's and the next one's
      if (const int e = allow_smem<norm_block<T, V, H>>(2 * H * kBlockThreads * 16)) return e;
      norm_block<T, V, H><<<static_cast<unsigned>(blocks) * slabs, threads, bytes, s>>>(a);
      return static_cast<int>(cudaGetLastError());
    };
    if (hold == 2) return go(std::integral_constant<int, 2>());
    if (hold == 4) return go(std::integral_constant<int, 4>());
    if (hold == 8) return go(std::integral_constant<int, 8>());
    return static_cast<int>(cudaErrorInvalidValue);
  } else {
    const dim3 grid(static_cast<unsigned>(a.n * a.parts), slabs);
    norm_part_stats<T, V><<<grid, threads, 0, s>>>(a);
    norm_part_apply<T, V><<<grid, threads, 0, s>>>(a);
  }
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int V> int backward(const NormArgs& a, int mode, int lanes, int hold, int threads, int blocks, cudaStream_t s) {
  int64_t rows = blocks;
  if (mode == 0) {
    if (const int e = lanes_by<T, V>(a, true, lanes, hold, blocks, s)) return e;
  } else if (mode == 1) {
    if (threads > kBlockThreads / 2 || threads % 32) return static_cast<int>(cudaErrorInvalidValue);
    const unsigned grid = static_cast<unsigned>(blocks) * ((a.g + a.slab - 1) / a.slab);
    auto go = [&](auto h) {
      constexpr int H = decltype(h)::value;
      const size_t bytes = 4 * static_cast<size_t>(H) * threads * V * sizeof(T);
      if (const int e = allow_smem<norm_block_grad<T, V, H>>(4 * H * kBlockThreads / 2 * 16)) return e;
      norm_block_grad<T, V, H><<<grid, threads, bytes, s>>>(a);
      return static_cast<int>(cudaGetLastError());
    };
    const int e = hold == 2 ? go(std::integral_constant<int, 2>()) : hold == 4 ? go(std::integral_constant<int, 4>())
                                                                             : static_cast<int>(cudaErrorInvalidValue);
    if (e) return e;
  } else {
    rows = a.n * a.parts;
    float* means = a.part + rows * 2 * a.c;
    const dim3 grid(static_cast<unsigned>(rows), (a.c / V + 31) / 32);
    norm_part_sums<T, V><<<grid, kPartThreads, 0, s>>>(a);
    norm_part_means<<<static_cast<unsigned>(a.n * a.g), 128, 0, s>>>(a, means);
    norm_part_grad<T, V><<<grid, kPartThreads, 0, s>>>(a, means);
  }
  if (a.dw || a.db) norm_channels<<<(a.c + 7) / 8, 256, 0, s>>>(a.part, rows, a.c, a.dw, a.db);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

// args: a NormArgs; vec: channels of a piece; mode, lanes, hold, threads, blocks: the form and its launch
SURF_EXPORT int surf_group_norm(const void* args, int dtype, int grad, int vec, int mode, int lanes, int hold, int threads, int blocks,
                                void* stream) {
  const NormArgs& a = *static_cast<const NormArgs*>(args);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_vec(vec, [&](auto v) {
    constexpr int V = decltype(v)::value;
    if (dtype == kBf16) return grad ? backward<bf16, V>(a, mode, lanes, hold, threads, blocks, s)
                                    : forward<bf16, V>(a, mode, lanes, hold, threads, blocks, s);
    if constexpr (V <= 4) return grad ? backward<float, V>(a, mode, lanes, hold, threads, blocks, s)
                                      : forward<float, V>(a, mode, lanes, hold, threads, blocks, s);
    return static_cast<int>(cudaErrorInvalidValue);
  });
}
