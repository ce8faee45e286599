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
//   lanes  a (sample, group) of at most 4 pieces for each of L <= 32 lanes stays in registers;
//   block  a sample's slab of whole groups stays in a block's shared memory: one pass over memory;
//   parts  anything larger, or too few slabs for the GPU: a pass over parts for their
//          statistics (or sums), one that applies them.
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

// ---- lanes ------------------------------------------------------------------------------
constexpr int kLaneThreads = 256, kHold = 4;

// L lanes for a (sample, group): lane l holds pieces l, l + L, ...; piece q is position
// q / (pieces of a group), whose channels follow. A block's warps take the samples of one set of
// 32 / L groups in turn, so that a lane's channels stay the same and their sums stay in registers.
template <typename T, int V, int L, bool kGrad>
__global__ void __launch_bounds__(kLaneThreads) norm_lanes(NormArgs a) {
  constexpr int kSets = 32 / L, kWarps = kLaneThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % L;
  const int gi = blockIdx.x * kSets + lane / L, cg = a.c / a.g, per = cg / V;
  const int items = static_cast<int>(a.p) * per;
  const bool on = gi < a.g;
  int64_t xo[kHold], dofs[kHold], yo[kHold];
  int ch[kHold];
  bool have[kHold];
  float w[kHold][V], b[kHold][V];
#pragma unroll
  for (int k = 0; k < kHold; ++k) {
    const int q = l + k * L;
    have[k] = on && q < items;
    const int pos = have[k] ? q / per : 0, c = have[k] ? gi * cg + (q - pos * per) * V : 0;
    ch[k] = c;
    xo[k] = pos * a.xs_p + c;
    dofs[k] = pos * a.ds_p + c;
    yo[k] = pos * a.ys_p + c;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[k][j] = a.w && have[k] ? a.w[c + j] : 1.0f;
      b[k][j] = a.b && have[k] ? a.b[c + j] : 0.0f;
    }
  }
  const float inv = 1.0f / (static_cast<float>(a.p) * cg);
  float sw[kGrad ? kHold : 1][V] = {}, sb[kGrad ? kHold : 1][V] = {};
  const int64_t step = static_cast<int64_t>(gridDim.y) * kWarps;
  for (int64_t n = static_cast<int64_t>(blockIdx.y) * kWarps + warp; n < a.n; n += step) {
    float v[kHold][V];
    const T* x = static_cast<const T*>(a.x) + n * a.xs_n;
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      if (have[k]) {
        load_vec<T, V>(x + xo[k], v[k]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[k][j] = 0.0f;
      }
    }
    if constexpr (!kGrad) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < kHold; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) s += v[k][j];
      const float mean = lanes_sum<L>(s) * inv;
      float q = 0.0f;
#pragma unroll
      for (int k = 0; k < kHold; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = v[k][j] - mean;
          if (have[k]) q = fmaf(d, d, q);
        }
      const float rstd = rsqrtf(lanes_sum<L>(q) * inv + a.eps);
      if (a.stats && on && l == 0) {
        a.stats[(n * a.g + gi) * 2] = mean;
        a.stats[(n * a.g + gi) * 2 + 1] = rstd;
      }
      T* y = static_cast<T*>(a.y) + n * a.ys_n;
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        if (!have[k]) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) v[k][j] = apply(v[k][j], mean, rstd, w[k][j], b[k][j], a.act);
        store_vec<T, V>(y + yo[k], v[k]);
      }
    } else {
      float mean = 0.0f, rstd = 0.0f;
      if (on) {
        mean = a.stats[(n * a.g + gi) * 2];
        rstd = a.stats[(n * a.g + gi) * 2 + 1];
      }
      const T* dy = static_cast<const T*>(a.dy) + n * a.ds_n;
      float d[kHold][V], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        if (have[k]) {
          load_vec<T, V>(dy + dofs[k], d[k]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) d[k][j] = 0.0f;
        }
      }
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        if (!have[k]) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float xh;
          const float e = gradient(v[k][j], d[k][j], mean, rstd, w[k][j], b[k][j], a.act, xh);
          sw[k][j] = fmaf(e, xh, sw[k][j]);
          sb[k][j] += e;
          v[k][j] = xh;
          d[k][j] = e * w[k][j];
          s1 += d[k][j];
          s2 = fmaf(d[k][j], xh, s2);
        }
      }
      const float m1 = lanes_sum<L>(s1) * inv, m2 = lanes_sum<L>(s2) * inv;
      T* y = static_cast<T*>(a.y) + n * a.ys_n;
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        if (!have[k]) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) v[k][j] = rstd * (d[k][j] - fmaf(v[k][j], m2, m1));
        store_vec<T, V>(y + yo[k], v[k]);
      }
    }
  }
  if constexpr (kGrad) {
    // the block's channels: warps, and positions of a channel in order
    __shared__ float sum[kWarps][32 * kHold * V + 1];
    float* out = a.part + static_cast<int64_t>(blockIdx.y) * 2 * a.c;
    const int width = min(kSets, a.g - static_cast<int>(blockIdx.x) * kSets) * cg;
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kHold; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) sum[warp][(lane / L * L * kHold + l + k * L) * V + j] = turn ? sb[k][j] : sw[k][j];
      __syncthreads();
      for (int c = threadIdx.x; c < width; c += kLaneThreads) {
        const int set = c / cg, in = c - set * cg;
        float s = 0.0f;
        for (int i = 0; i < kWarps; ++i)
          for (int pos = 0; pos < static_cast<int>(a.p); ++pos) s += sum[i][set * L * kHold * V + pos * cg + in];
        out[turn * a.c + blockIdx.x * kSets * cg + c] = s;
      }
    }
  }
}

// ---- blocks -----------------------------------------------------------------------------
constexpr int kBlockThreads = 256;

// Threads that walk a slab: with several groups whole rows of its pieces, so that a thread's piece
// (and group) stays the same; with one group all of them.
__device__ __forceinline__ int walkers(int groups, int per) {
  return groups == 1 ? static_cast<int>(blockDim.x) : static_cast<int>(blockDim.x) / per * per;
}
// The pieces of a slab in a thread's order, `step` further each time.
struct Walk {
  int per, piece, dpos, dpiece;
  int64_t pos;
  __device__ __forceinline__ Walk(int per_, int64_t first, int step) : per(per_) {
    dpos = step / per;
    dpiece = step - dpos * per;
    const int p0 = static_cast<int>(threadIdx.x) / per;
    piece = static_cast<int>(threadIdx.x) - p0 * per;
    pos = first + p0;
  }
  __device__ __forceinline__ void next() {
    pos += dpos;
    piece += dpiece;
    if (piece >= per) {
      piece -= per;
      ++pos;
    }
  }
};

// red[i] summed over the threads of each of the slab's groups; res[group] for all threads.
// A thread's group is piece / (pieces of a group); the order of the sum is the threads'. The block
// is whole warps.
__device__ __forceinline__ void sum_groups(float v, float* red, float* res, int groups, int per, int per_group) {
  __syncthreads();
  red[threadIdx.x] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31, warps = blockDim.x / 32;
  for (int g = threadIdx.x >> 5; g < groups; g += warps) {
    float s = 0.0f;
    if (groups == 1) {
      for (int i = lane; i < static_cast<int>(blockDim.x); i += 32) s += red[i];
    } else {
      const int rows = blockDim.x / per;
      for (int i = lane; i < rows * per_group; i += 32) {
        const int r = i / per_group;
        s += red[r * per + g * per_group + i - r * per_group];
      }
    }
    s = lanes_sum<32>(s);
    if (lane == 0) res[g] = s;
  }
  __syncthreads();
}

// One slab of one sample: first sums, then squares, then values, from shared memory.
template <typename T, int V> __global__ void __launch_bounds__(kBlockThreads) norm_block(NormArgs a) {
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[kBlockThreads], res[kBlockThreads];
  T* hold = reinterpret_cast<T*>(smem);
  const int cg = a.c / a.g, per_group = cg / V;
  const int g0 = blockIdx.y * a.slab, groups = min(a.slab, a.g - g0), per = groups * per_group;
  const int c0 = g0 * cg;
  const float inv = 1.0f / (static_cast<float>(a.p) * cg);
  const int own = groups == 1 ? 0 : static_cast<int>(threadIdx.x) % per / per_group;
  const int step = walkers(groups, per);
  const bool fits = static_cast<int>(threadIdx.x) < step;
  const int64_t n = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + n * a.xs_n + c0;
  T* y = static_cast<T*>(a.y) + n * a.ys_n + c0;
  float s = 0.0f;
  if (fits) {
    Walk it(per, 0, step);
    T* h = hold + static_cast<size_t>(threadIdx.x) * V;
    for (; it.pos < a.p; it.next(), h += step * V) {
      float v[V];
      load_vec<T, V>(x + it.pos * a.xs_p + it.piece * V, v);
      store_vec<T, V>(h, v);
#pragma unroll
      for (int j = 0; j < V; ++j) s += v[j];
    }
  }
  sum_groups(s, red, res, groups, per, per_group);
  const float mean = res[own] * inv;
  s = 0.0f;
  if (fits) {
    Walk it(per, 0, step);
    const T* h = hold + static_cast<size_t>(threadIdx.x) * V;
    for (; it.pos < a.p; it.next(), h += step * V) {
      float v[V];
      load_vec<T, V>(h, v);
#pragma unroll
      for (int j = 0; j < V; ++j) s = fmaf(v[j] - mean, v[j] - mean, s);
    }
  }
  sum_groups(s, red, res, groups, per, per_group);
  const float rstd = rsqrtf(res[own] * inv + a.eps);
  if (a.stats && fits && static_cast<int>(threadIdx.x) < per && static_cast<int>(threadIdx.x) % per_group == 0 &&
      (groups > 1 || threadIdx.x == 0)) {
    a.stats[(n * a.g + g0 + own) * 2] = mean;
    a.stats[(n * a.g + g0 + own) * 2 + 1] = rstd;
  }
  if (fits) {
    Walk it(per, 0, step);
    const T* h = hold + static_cast<size_t>(threadIdx.x) * V;
    for (; it.pos < a.p; it.next(), h += step * V) {
      float v[V];
      load_vec<T, V>(h, v);
      const int c = c0 + it.piece * V;
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = apply(v[j], mean, rstd, a.w ? a.w[c + j] : 1.0f, a.b ? a.b[c + j] : 0.0f, a.act);
      store_vec<T, V>(y + it.pos * a.ys_p + it.piece * V, v);
    }
  }
}

// The channels' sums of a thread's pieces, joined over the block's rows in order.
template <int V> struct ChannelSums {
  float w[V], b[V];
  __device__ __forceinline__ ChannelSums() {
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = b[j] = 0.0f;
  }
  __device__ __forceinline__ void store(float* red, float* out, int c, int per, bool fits) {
    const int rows = blockDim.x / per;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int turn = 0; turn < 2; ++turn) {
        __syncthreads();
        red[threadIdx.x] = fits ? (turn ? b[j] : w[j]) : 0.0f;
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < per) {
          float s = 0.0f;
          for (int r = 0; r < rows; ++r) s += red[r * per + threadIdx.x];
          out[turn * c + threadIdx.x * V + j] = s;
        }
      }
  }
};

// Gradient of slabs of samples blockIdx.x, + gridDim.x, ...; the block is a multiple of the
// slab's pieces, so that a thread's channels stay the same.
template <typename T, int V> __global__ void __launch_bounds__(kBlockThreads) norm_block_grad(NormArgs a) {
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[kBlockThreads], res[kBlockThreads];
  const int cg = a.c / a.g, per_group = cg / V;
  const int g0 = blockIdx.y * a.slab, groups = min(a.slab, a.g - g0), per = groups * per_group;
  const int c0 = g0 * cg;
  const float inv = 1.0f / (static_cast<float>(a.p) * cg);
  const bool fits = static_cast<int>(threadIdx.x) < static_cast<int>(blockDim.x) / per * per;
  const int piece = static_cast<int>(threadIdx.x) % per, rows = blockDim.x / per, own = piece / per_group;
  const int row = static_cast<int>(threadIdx.x) / per;
  T* hx = reinterpret_cast<T*>(smem);
  T* hd = hx + static_cast<size_t>((a.p + rows - 1) / rows) * rows * per * V;
  float w[V], b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    w[j] = a.w ? a.w[c0 + piece * V + j] : 1.0f;
    b[j] = a.b ? a.b[c0 + piece * V + j] : 0.0f;
  }
  ChannelSums<V> sums;
  for (int64_t n = blockIdx.x; n < a.n; n += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + n * a.xs_n + c0 + piece * V;
    const T* dy = static_cast<const T*>(a.dy) + n * a.ds_n + c0 + piece * V;
    T* y = static_cast<T*>(a.y) + n * a.ys_n + c0 + piece * V;
    const float mean = a.stats[(n * a.g + g0 + own) * 2], rstd = a.stats[(n * a.g + g0 + own) * 2 + 1];
    float s1 = 0.0f, s2 = 0.0f;
    if (fits) {
      for (int64_t p = row; p < a.p; p += rows) {
        float v[V], d[V];
        load_vec<T, V>(x + p * a.xs_p, v);
        load_vec<T, V>(dy + p * a.ds_p, d);
        store_vec<T, V>(hx + (p * per + piece) * V, v);
        store_vec<T, V>(hd + (p * per + piece) * V, d);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float xh;
          const float e = gradient(v[j], d[j], mean, rstd, w[j], b[j], a.act, xh);
          sums.w[j] = fmaf(e, xh, sums.w[j]);
          sums.b[j] += e;
          s1 = fmaf(e, w[j], s1);
          s2 = fmaf(e * w[j], xh, s2);
        }
      }
    }
    sum_groups(s1, red, res, groups, per, per_group);
    const float m1 = res[own] * inv;
    sum_groups(s2, red, res, groups, per, per_group);
    const float m2 = res[own] * inv;
    if (fits) {
      for (int64_t p = row; p < a.p; p += rows) {
        float v[V], d[V];
        load_vec<T, V>(hx + (p * per + piece) * V, v);
        load_vec<T, V>(hd + (p * per + piece) * V, d);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float xh;
          const float e = gradient(v[j], d[j], mean, rstd, w[j], b[j], a.act, xh);
          v[j] = rstd * (e * w[j] - fmaf(xh, m2, m1));
        }
        store_vec<T, V>(y + p * a.ys_p, v);
      }
    }
  }
  sums.store(red, a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.c + c0, a.c, per, fits);
}

// ---- parts ------------------------------------------------------------------------------
// Moments of the positions of a part: [N, G, parts, 3]. A slab as above.
template <typename T, int V> __global__ void __launch_bounds__(kBlockThreads) norm_part_stats(NormArgs a) {
  __shared__ float red[kBlockThreads], res[kBlockThreads];
  const int cg = a.c / a.g, per_group = cg / V;
  const int g0 = blockIdx.y * a.slab, groups = min(a.slab, a.g - g0), per = groups * per_group;
  const int own = groups == 1 ? 0 : static_cast<int>(threadIdx.x) % per / per_group;
  const int step = walkers(groups, per);
  const bool fits = static_cast<int>(threadIdx.x) < step;
  const int64_t n = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t first = part * a.span, last = min(a.p, first + a.span);
  const T* x = static_cast<const T*>(a.x) + n * a.xs_n + g0 * cg;
  const float inv = 1.0f / (static_cast<float>(last - first) * cg);
  float s = 0.0f;
  if (fits)
    for (Walk it(per, first, step); it.pos < last; it.next()) {
      float v[V];
      load_vec<T, V>(x + it.pos * a.xs_p + it.piece * V, v);
#pragma unroll
      for (int j = 0; j < V; ++j) s += v[j];
    }
  sum_groups(s, red, res, groups, per, per_group);
  const float mean = res[own] * inv;
  s = 0.0f;
  if (fits)
    for (Walk it(per, first, step); it.pos < last; it.next()) {
      float v[V];
      load_vec<T, V>(x + it.pos * a.xs_p + it.piece * V, v);
#pragma unroll
      for (int j = 0; j < V; ++j) s = fmaf(v[j] - mean, v[j] - mean, s);
    }
  sum_groups(s, red, res, groups, per, per_group);
  if (fits && static_cast<int>(threadIdx.x) < per && static_cast<int>(threadIdx.x) % per_group == 0 &&
      (groups > 1 || threadIdx.x == 0)) {
    float* out = a.part + ((n * a.g + g0 + own) * a.parts + part) * 3;
    out[0] = static_cast<float>(last - first) * cg;
    out[1] = mean;
    out[2] = res[own];
  }
}

// The moments of group g of sample n from its parts, in order: (mean, rstd).
__device__ __forceinline__ float2 joined(const NormArgs& a, int64_t n, int g) {
  const float* m = a.part + (n * a.g + g) * a.parts * 3;
  Moments all{0.0f, 0.0f, 0.0f};
  for (int i = 0; i < a.parts; ++i) all = join(all, {m[3 * i], m[3 * i + 1], m[3 * i + 2]});
  return make_float2(all.mean, rsqrtf(all.m2 / all.n + a.eps));
}

template <typename T, int V> __global__ void __launch_bounds__(kBlockThreads) norm_part_apply(NormArgs a) {
  __shared__ float2 st[kBlockThreads];
  const int cg = a.c / a.g, per_group = cg / V;
  const int g0 = blockIdx.y * a.slab, groups = min(a.slab, a.g - g0), per = groups * per_group;
  const int own = groups == 1 ? 0 : static_cast<int>(threadIdx.x) % per / per_group;
  const int step = walkers(groups, per);
  const bool fits = static_cast<int>(threadIdx.x) < step;
  const int64_t n = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t first = part * a.span, last = min(a.p, first + a.span);
  for (int i = threadIdx.x; i < groups; i += blockDim.x) {
    st[i] = joined(a, n, g0 + i);
    if (a.stats && part == 0) {
      a.stats[(n * a.g + g0 + i) * 2] = st[i].x;
      a.stats[(n * a.g + g0 + i) * 2 + 1] = st[i].y;
    }
  }
  __syncthreads();
  const float mean = st[own].x, rstd = st[own].y;
  const T* x = static_cast<const T*>(a.x) + n * a.xs_n + g0 * cg;
  T* y = static_cast<T*>(a.y) + n * a.ys_n + g0 * cg;
  if (fits)
    for (Walk it(per, first, step); it.pos < last; it.next()) {
      float v[V];
      load_vec<T, V>(x + it.pos * a.xs_p + it.piece * V, v);
      const int c = g0 * cg + it.piece * V;
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = apply(v[j], mean, rstd, a.w ? a.w[c + j] : 1.0f, a.b ? a.b[c + j] : 0.0f, a.act);
      store_vec<T, V>(y + it.pos * a.ys_p + it.piece * V, v);
    }
}

// Sums of d xh and d over the positions of a part: [N, parts, 2, C].
template <typename T, int V> __global__ void __launch_bounds__(kBlockThreads) norm_part_sums(NormArgs a) {
  const int cg = a.c / a.g;
  const int64_t n = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t first = part * a.span, last = min(a.p, first + a.span);
  __shared__ float red[kBlockThreads];
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

template <typename T, int V> __global__ void __launch_bounds__(kBlockThreads) norm_part_grad(NormArgs a, const float* means) {
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

template <typename T, int V, int L> int lanes_go(const NormArgs& a, bool grad, int blocks, cudaStream_t s) {
  const dim3 grid((a.g + 32 / L - 1) / (32 / L), blocks);
  if (grad) norm_lanes<T, V, L, true><<<grid, kLaneThreads, 0, s>>>(a);
  else norm_lanes<T, V, L, false><<<grid, kLaneThreads, 0, s>>>(a);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int V> int lanes_by(const NormArgs& a, bool grad, int lanes, int blocks, cudaStream_t s) {
  switch (lanes) {
    case 1: return lanes_go<T, V, 1>(a, grad, blocks, s);
    case 2: return lanes_go<T, V, 2>(a, grad, blocks, s);
    case 4: return lanes_go<T, V, 4>(a, grad, blocks, s);
    case 8: return lanes_go<T, V, 8>(a, grad, blocks, s);
    case 16: return lanes_go<T, V, 16>(a, grad, blocks, s);
    case 32: return lanes_go<T, V, 32>(a, grad, blocks, s);
  }
  return static_cast<int>(cudaErrorInvalidValue);
}

// mode 0 lanes, 1 block, 2 parts; threads: of a block of mode 1 and of the parts' forward
template <typename T, int V> int forward(const NormArgs& a, int mode, int lanes, int threads, int blocks, size_t smem, cudaStream_t s) {
  if (mode == 0) return lanes_by<T, V>(a, false, lanes, blocks, s);
  const int slabs = (a.g + a.slab - 1) / a.slab;
  if (mode == 1) {
    if (const int e = allow_smem<norm_block<T, V>>(200 * 1024)) return e;
    norm_block<T, V><<<dim3(static_cast<unsigned>(a.n), slabs), threads, smem, s>>>(a);
  } else {
    const dim3 grid(static_cast<unsigned>(a.n * a.parts), slabs);
    norm_part_stats<T, V><<<grid, threads, 0, s>>>(a);
    norm_part_apply<T, V><<<grid, threads, 0, s>>>(a);
  }
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int V> int backward(const NormArgs& a, int mode, int lanes, int threads, int blocks, size_t smem, cudaStream_t s) {
  int64_t rows = blocks;
  if (mode == 0) {
    if (const int e = lanes_by<T, V>(a, true, lanes, blocks, s)) return e;
  } else if (mode == 1) {
    if (const int e = allow_smem<norm_block_grad<T, V>>(200 * 1024)) return e;
    norm_block_grad<T, V><<<dim3(blocks, (a.g + a.slab - 1) / a.slab), threads, smem, s>>>(a);
  } else {
    rows = a.n * a.parts;
    float* means = a.part + rows * 2 * a.c;
    const dim3 grid(static_cast<unsigned>(rows), (a.c / V + 31) / 32);
    norm_part_sums<T, V><<<grid, kBlockThreads, 0, s>>>(a);
    norm_part_means<<<static_cast<unsigned>(a.n * a.g), 128, 0, s>>>(a, means);
    norm_part_grad<T, V><<<grid, kBlockThreads, 0, s>>>(a, means);
  }
  if (a.dw || a.db) norm_channels<<<(a.c + 7) / 8, 256, 0, s>>>(a.part, rows, a.c, a.dw, a.db);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

// args: a NormArgs; vec: channels of a piece; mode, lanes, threads, blocks, smem: the form and its launch
SURF_EXPORT int surf_group_norm(const void* args, int dtype, int grad, int vec, int mode, int lanes, int threads, int blocks,
                                int smem, void* stream) {
  const NormArgs& a = *static_cast<const NormArgs*>(args);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_vec(vec, [&](auto v) {
    constexpr int V = decltype(v)::value;
    if (dtype == kBf16) return grad ? backward<bf16, V>(a, mode, lanes, threads, blocks, smem, s)
                                    : forward<bf16, V>(a, mode, lanes, threads, blocks, smem, s);
    if constexpr (V <= 4) return grad ? backward<float, V>(a, mode, lanes, threads, blocks, smem, s)
                                      : forward<float, V>(a, mode, lanes, threads, blocks, smem, s);
    return static_cast<int>(cudaErrorInvalidValue);
  });
}
