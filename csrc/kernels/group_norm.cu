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

__device__ __forceinline__ float act_of(float v, int act) {
  if (act == kSilu) return v * sigmoid(v);
  return act == kRelu ? fmaxf(v, 0.0f) : v;
}
__device__ __forceinline__ float slope_of(float v, int act) {
  if (act == kSilu) {
    const float s = sigmoid(v);
    return s * fmaf(v, 1.0f - s, 1.0f);
  }
  return act == kRelu && !(v > 0.0f) ? 0.0f : 1.0f;
}
// relu as torch's: NaN stays
__device__ __forceinline__ float apply(float x, float mean, float rstd, float w, float b, int act) {
  const float pre = fmaf((x - mean) * rstd, w, b);
  return act == kRelu && !(pre > 0.0f) ? (pre == pre ? 0.0f : pre) : act_of(pre, act);
}
__device__ __forceinline__ float gradient(float x, float dy, float mean, float rstd, float w, float b, int act, float& xh) {
  xh = (x - mean) * rstd;
  return act == kNone ? dy : dy * slope_of(fmaf(xh, w, b), act);
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
  __device__ __forceinline__ void get(float (&v)[V]) const {
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
  }
};
template <int V> struct Weights {
  float w[V], b[V];
  __device__ __forceinline__ void load(const float* pw, const float* pb, int c, bool on) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[j] = pw && on ? pw[c + j] : 1.0f;
      b[j] = pb && on ? pb[c + j] : 0.0f;
    }
  }
};

// ---- lanes ------------------------------------------------------------------------------
constexpr int kLaneThreads = 256;

// L lanes for a (sample, group): lane l holds pieces l, l + L, ... of at most H L; piece q is position
// q / (pieces of a group), whose channels follow. A block's warps take the samples of one set of
// 32 / L groups in turn, two at a time where a lane has one piece, so that a lane's channels stay
// the same and their sums stay in registers.
template <typename T, int V, int L, int H, bool kGrad>
__global__ void __launch_bounds__(kLaneThreads) norm_lanes(NormArgs a) {
  constexpr int kSets = 32 / L, kWarps = kLaneThreads / 32, U = H == 1 ? 2 : 1;
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
  float sw[kGrad ? H : 1][V] = {}, sb[kGrad ? H : 1][V] = {};
  const int64_t step = static_cast<int64_t>(gridDim.y) * kWarps;
  for (int64_t n0 = static_cast<int64_t>(blockIdx.y) * kWarps + warp; n0 < a.n; n0 += U * step) {
    Piece<T, V> rx[U][H], rd[U][H];
    float mean[U], rstd[U];
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
      mean[u] = rstd[u] = 0.0f;
      if (kGrad && live && on) {
        const float2 st = *reinterpret_cast<const float2*>(a.stats + (n * a.g + gi) * 2);
        mean[u] = st.x;
        rstd[u] = st.y;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = n0 + u * step;
      const bool live = n < a.n;
      T* y = static_cast<T*>(a.y) + n * a.ys_n;
      if constexpr (!kGrad) {
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int k = 0; k < H; ++k) {
          float v[V];
          rx[u][k].get(v);
#pragma unroll
          for (int j = 0; j < V; ++j) s += v[j];
        }
        const float m = lanes_sum<L>(s) * inv;
#pragma unroll
        for (int k = 0; k < H; ++k) {
          float v[V];
          rx[u][k].get(v);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float d = v[j] - m;
            if (have[k]) q = fmaf(d, d, q);
          }
        }
        const float r = rsqrtf(lanes_sum<L>(q) * inv + a.eps);
        if (a.stats && live && on && l == 0) *reinterpret_cast<float2*>(a.stats + (n * a.g + gi) * 2) = make_float2(m, r);
#pragma unroll
        for (int k = 0; k < H; ++k) {
          if (!live || !have[k]) continue;
          float v[V];
          rx[u][k].get(v);
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = apply(v[j], m, r, wb[k].w[j], wb[k].b[j], a.act);
          store_vec<T, V>(y + yo[k], v);
        }
      } else {
        float xh[H][V], d[H][V], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < H; ++k) {
          float v[V], e[V];
          rx[u][k].get(v);
          rd[u][k].get(e);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float g = gradient(v[j], e[j], mean[u], rstd[u], wb[k].w[j], wb[k].b[j], a.act, xh[k][j]);
            if (live && have[k]) {
              sw[k][j] = fmaf(g, xh[k][j], sw[k][j]);
              sb[k][j] += g;
            }
            d[k][j] = have[k] ? g * wb[k].w[j] : 0.0f;
            s1 += d[k][j];
            s2 = fmaf(d[k][j], xh[k][j], s2);
          }
        }
        const float m1 = lanes_sum<L>(s1) * inv, m2 = lanes_sum<L>(s2) * inv;
#pragma unroll
        for (int k = 0; k < H; ++k) {
          if (!live || !have[k]) continue;
          float v[V];
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = rstd[u] * (d[k][j] - fmaf(xh[k][j], m2, m1));
          store_vec<T, V>(y + yo[k], v);
        }
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
      for (int k = 0; k < H; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) sum[warp][(lane / L * L * H + l + k * L) * V + j] = turn ? sb[k][j] : sw[k][j];
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

// Slabs (the faster index, so that a sample's are read together) of samples.
template <typename T, int V, int H> __global__ void __launch_bounds__(kBlockThreads) norm_block(NormArgs a) {
  __shared__ float red[kBlockThreads], res[kBlockThreads];
  const int slabs = (a.g + a.slab - 1) / a.slab;
  const Place at(a, blockIdx.x % slabs, V);
  const int64_t n = blockIdx.x / slabs;
  const float inv = 1.0f / (static_cast<float>(a.p) * (a.c / a.g));
  const int count = at.on ? max(0, static_cast<int>((a.p - at.row + at.rows - 1) / at.rows)) : 0;       // this thread's pieces
  Piece<T, V> r[H];
  const T* x = static_cast<const T*>(a.x) + n * a.xs_n + at.row * a.xs_p + at.c0;
#pragma unroll
  for (int k = 0; k < H; ++k) {
    if (k < count) r[k].load(x + k * (at.rows * a.xs_p));
    else r[k].zero();
  }
  Weights<V> wb;
  wb.load(a.w, a.b, at.c0, at.on);
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < H; ++k) {
    float v[V];
    r[k].get(v);
#pragma unroll
    for (int j = 0; j < V; ++j) s += v[j];
  }
  sum_groups(s, red, res, at.groups, at.per, at.per_group, at.walkers);
  const float mean = res[at.own] * inv;
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < H; ++k) {
    float v[V];
    r[k].get(v);
    if (k < count)
#pragma unroll
      for (int j = 0; j < V; ++j) s = fmaf(v[j] - mean, v[j] - mean, s);
  }
  sum_groups(s, red, res, at.groups, at.per, at.per_group, at.walkers);
  const float rstd = rsqrtf(res[at.own] * inv + a.eps);
  if (a.stats && at.on && at.row == 0 && at.piece % at.per_group == 0)
    *reinterpret_cast<float2*>(a.stats + (n * a.g + at.g0 + at.own) * 2) = make_float2(mean, rstd);
  T* y = static_cast<T*>(a.y) + n * a.ys_n + at.row * a.ys_p + at.c0;
#pragma unroll
  for (int k = 0; k < H; ++k) {
    if (k >= count) continue;
    float v[V];
    r[k].get(v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = apply(v[j], mean, rstd, wb.w[j], wb.b[j], a.act);
    store_vec<T, V>(y + k * (at.rows * a.ys_p), v);
  }
}

// Gradient of a slab of samples blockIdx.x / slabs, + gridDim.x / slabs, ...
template <typename T, int V, int H> __global__ void __launch_bounds__(kBlockThreads / 2, 2) norm_block_grad(NormArgs a) {
  __shared__ float red[kBlockThreads], res[kBlockThreads];
  const int slabs = (a.g + a.slab - 1) / a.slab, blocks = gridDim.x / slabs, block = blockIdx.x / slabs;
  const Place at(a, blockIdx.x % slabs, V);
  const float inv = 1.0f / (static_cast<float>(a.p) * (a.c / a.g));
  const int count = at.on ? max(0, static_cast<int>((a.p - at.row + at.rows - 1) / at.rows)) : 0;
  Weights<V> wb;
  wb.load(a.w, a.b, at.c0, at.on);
  float sw[V] = {}, sb[V] = {};
  for (int64_t n = block; n < a.n; n += blocks) {
    Piece<T, V> rx[H], rd[H];
    const T* x = static_cast<const T*>(a.x) + n * a.xs_n + at.row * a.xs_p + at.c0;
    const T* dy = static_cast<const T*>(a.dy) + n * a.ds_n + at.row * a.ds_p + at.c0;
#pragma unroll
    for (int k = 0; k < H; ++k) {
      if (k < count) {
        rx[k].load(x + k * (at.rows * a.xs_p));
        rd[k].load(dy + k * (at.rows * a.ds_p));
      } else {
        rx[k].zero();
        rd[k].zero();
      }
    }
    const float2 st = *reinterpret_cast<const float2*>(a.stats + (n * a.g + at.g0 + at.own) * 2);
    float xh[H][V], d[H][V], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < H; ++k) {
      float v[V], e[V];
      rx[k].get(v);
      rd[k].get(e);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float g = gradient(v[j], e[j], st.x, st.y, wb.w[j], wb.b[j], a.act, xh[k][j]);
        if (k < count) {
          sw[j] = fmaf(g, xh[k][j], sw[j]);
          sb[j] += g;
        }
        d[k][j] = k < count ? g * wb.w[j] : 0.0f;
        s1 += d[k][j];
        s2 = fmaf(d[k][j], xh[k][j], s2);
      }
    }
    sum_groups(s1, red, res, at.groups, at.per, at.per_group, at.walkers);
    const float m1 = res[at.own] * inv;
    sum_groups(s2, red, res, at.groups, at.per, at.per_group, at.walkers);
    const float m2 = res[at.own] * inv;
    T* y = static_cast<T*>(a.y) + n * a.ys_n + at.row * a.ys_p + at.c0;
#pragma unroll
    for (int k = 0; k < H; ++k) {
      if (k >= count) continue;
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = st.y * (d[k][j] - fmaf(xh[k][j], m2, m1));
      store_vec<T, V>(y + k * (at.rows * a.ys_p), v);
    }
  }
  // the channels' sums, the block's rows in order
  float* out = a.part + static_cast<int64_t>(block) * 2 * a.c + at.c0 - at.piece * V;
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
      __syncthreads();
      red[threadIdx.x] = at.on ? (turn ? sb[j] : sw[j]) : 0.0f;
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < at.per) {
        float s = 0.0f;
        for (int i = 0; i < at.rows; ++i) s += red[i * at.per + threadIdx.x];
        out[turn * a.c + threadIdx.x * V + j] = s;
      }
    }
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
  float s = 0.0f;
  each([&](const T* from) {
    float v[V];
    load_vec<T, V>(from, v);
#pragma unroll
    for (int j = 0; j < V; ++j) s += v[j];
  });
  sum_groups(s, red, res, at.groups, row_pieces, group_pieces, walkers);
  const float mean = res[own] * inv;
  s = 0.0f;
  each([&](const T* from) {
    float v[V];
    load_vec<T, V>(from, v);
#pragma unroll
    for (int j = 0; j < V; ++j) s = fmaf(v[j] - mean, v[j] - mean, s);
  });
  sum_groups(s, red, res, at.groups, row_pieces, group_pieces, walkers);
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
    float v[V];
    load_vec<T, V>(x + p * a.xs_p + i * V, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = apply(v[j], m.x, m.y, wb.w[j], wb.b[j], a.act);
    store_vec<T, V>(y + p * a.ys_p + i * V, v);
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

// Sums of d xh and d over the positions of a part: [N, parts, 2, C].
constexpr int kPartThreads = 256;
template <typename T, int V> __global__ void __launch_bounds__(kPartThreads) norm_part_sums(NormArgs a) {
  const int cg = a.c / a.g;
  const int64_t n = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t first = part * a.span, last = min(a.p, first + a.span);
  __shared__ float red[kPartThreads];
  // 32 pieces of channels by 8 rows of positions
  const int col = (blockIdx.y * 32 + (threadIdx.x & 31)) * V, row = threadIdx.x >> 5;
  const bool on = col < a.c;
  float sw[V], sb[V], w[V], b[V], mean = 0.0f, rstd = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    sw[j] = sb[j] = 0.0f;
    w[j] = a.w && on ? a.w[col + j] : 1.0f;
    b[j] = a.b && on ? a.b[col + j] : 0.0f;
  }
  if (on) {
    mean = a.stats[(n * a.g + col / cg) * 2];
    rstd = a.stats[(n * a.g + col / cg) * 2 + 1];
    const T* x = static_cast<const T*>(a.x) + n * a.xs_n + col;
    const T* dy = static_cast<const T*>(a.dy) + n * a.ds_n + col;
#pragma unroll 2
    for (int64_t p = first + row; p < last; p += 8) {
      float v[V], d[V];
      load_vec<T, V>(x + p * a.xs_p, v);
      load_vec<T, V>(dy + p * a.ds_p, d);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float xh;
        const float e = gradient(v[j], d[j], mean, rstd, w[j], b[j], a.act, xh);
        sw[j] = fmaf(e, xh, sw[j]);
        sb[j] += e;
      }
    }
  }
  float* out = a.part + blockIdx.x * static_cast<int64_t>(2 * a.c);
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
      __syncthreads();
      red[threadIdx.x] = turn ? sb[j] : sw[j];
      __syncthreads();
      if (row == 0 && on) {
        float s = 0.0f;
        for (int r = 0; r < 8; ++r) s += red[r * 32 + threadIdx.x];
        out[turn * a.c + col + j] = s;
      }
    }
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
  const int col = (blockIdx.y * 32 + (threadIdx.x & 31)) * V, row = threadIdx.x >> 5;
  if (col >= a.c) return;
  const int64_t at = (n * a.g + col / cg) * 2;
  const float mean = a.stats[at], rstd = a.stats[at + 1], m1 = means[at], m2 = means[at + 1];
  float w[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    w[j] = a.w ? a.w[col + j] : 1.0f;
    b[j] = a.b ? a.b[col + j] : 0.0f;
  }
  const T* x = static_cast<const T*>(a.x) + n * a.xs_n + col;
  const T* dy = static_cast<const T*>(a.dy) + n * a.ds_n + col;
  T* y = static_cast<T*>(a.y) + n * a.ys_n + col;
#pragma unroll 2
  for (int64_t p = first + row; p < last; p += 8) {
    float v[V], d[V];
    load_vec<T, V>(x + p * a.xs_p, v);
    load_vec<T, V>(dy + p * a.ds_p, d);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float xh;
      const float e = gradient(v[j], d[j], mean, rstd, w[j], b[j], a.act, xh);
      v[j] = rstd * (e * w[j] - fmaf(xh, m2, m1));
    }
    store_vec<T, V>(y + p * a.ys_p, v);
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
    const unsigned grid = static_cast<unsigned>(a.n * slabs);
    if (hold == 2) norm_block<T, V, 2><<<grid, threads, 0, s>>>(a);
    else if (hold == 4) norm_block<T, V, 4><<<grid, threads, 0, s>>>(a);
    else if (hold == 8) norm_block<T, V, 8><<<grid, threads, 0, s>>>(a);
    else return static_cast<int>(cudaErrorInvalidValue);
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
    if (hold == 2) norm_block_grad<T, V, 2><<<grid, threads, 0, s>>>(a);
    else if (hold == 4) norm_block_grad<T, V, 4><<<grid, threads, 0, s>>>(a);
    else return static_cast<int>(cudaErrorInvalidValue);
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
