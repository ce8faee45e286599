// policy_loss.cu — clipped policy loss with a KL term from rows of logits, and its gradient
// (sm_100a).
//
// Row n: logits z, temperature t, y = z / t, lse = log sum e^y, p = e^(y - lse); of its answer a
//   lp = y_a - lse,  r = exp(lp - old),  d = ref - lp,  H = -sum p log p
//   L  = -min(r A, clip(r, 1 - lo, 1 + hi) A) + kl (e^d - d - 1) - ent H
//   loss = sum_n w_n L_n
// and with c = w (kl (1 - e^d) - [r A <= clip(r) A] r A)
//   dz_j = (c ([j = a] - p_j) + w ent p_j (log p_j + H)) / t.
//
// One pass over memory: a row's logits stay in shared memory (registers, where a warp takes a
// row) between the pass that sums and the one that writes the gradient. 4096x32003 bfloat16: 139 us, 0.58 of
// the copy rate; 22 instructions a candidate, three blocks an SM that wait at the row's barriers.
#include <cooperative_groups.h>
#include <type_traits>

#include "seq_common.cuh"

namespace {

using namespace seqk;
namespace cg = cooperative_groups;

struct LossArgs {
  const void* z;
  const void* answers;         // int32 or int64
  const float *old_logp, *adv, *ref, *weight;       // ref, weight: null for none, 1 / rows
  void* dz;                    // or null
  float* rows;                 // [3, R]: log-probability, KL, entropy
  float* each;                 // [R]: w L
  float* loss;
  int* err;
  int64_t z_ld, d_ld;
  int64_t n;
  int v, wide;                 // candidates; 1: int64 answers
  float lo, hi, kl, ent, inv_t, share;
};
static_assert(sizeof(LossArgs) == 11 * 8 + 3 * 8 + 8 * 4, "as the caller packs it");

struct Row {
  int64_t n;
  int a;                       // the answer, -1: counts nothing
};

__device__ __forceinline__ Row row_of(const LossArgs& p, int64_t n, bool report) {
  const int64_t a = p.wide ? static_cast<const int64_t*>(p.answers)[n] : static_cast<const int*>(p.answers)[n];
  if (a >= p.v && report) surfk::report_error(p.err, surfk::kErrLossIndex);
  return {n, a >= 0 && a < p.v ? static_cast<int>(a) : -1};
}

// A row's exponents in powers of two: with c = log2(e) / t and the maximum m, x = z c - m c and e^(y - max y)
// = 2^x. The product m c is rounded once and is then what all of the row is measured from, so that its
// rounding cancels; where it would be as large as the differences themselves (and for infinite
// maxima) x is (z - m) c instead. -1000 stands for what has no probability: -inf and NaN (which the
// maximum of two numbers drops).
struct Shift {
  float m, c, mc;
  bool far;
  __device__ __forceinline__ double from() const { return far ? static_cast<double>(m) * c : static_cast<double>(mc); }   // finite m
};
__device__ __forceinline__ Shift shift_of(float m, float inv_t) {
  const float c = __fmul_rn(inv_t, kLog2e), mc = __fmul_rn(m, c);
  return {m, c, mc, !(fabsf(mc) <= 1048576.0f)};
}
template <bool kFar> __device__ __forceinline__ float power_of(float z, const Shift& h) {
  if constexpr (kFar) return z == h.m ? 0.0f : fmaxf((z - h.m) * h.c, -1000.0f);
  else return fmaxf(fmaf(z, h.c, -h.mc), -1000.0f);
}
// sums of 2^x and of x 2^x, x measured from m
struct Sums { float m, s, t; };
template <bool kFar> __device__ __forceinline__ void add(Sums& a, float z, const Shift& h) {
  const float x = power_of<kFar>(z, h), e = exp2_hw(x);
  a.s += e;
  a.t = fmaf(e, x, a.t);
}
// NaN logits count as -inf
__device__ __forceinline__ float clean(float z) { return fmaxf(z, -INFINITY); }
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float inv_t) {
  const Sums &hi = a.m >= b.m ? a : b, &lo = a.m >= b.m ? b : a;
  if (!(lo.s > 0.0f) || (hi.m == INFINITY && lo.m < hi.m)) return hi;
  const float x = hi.m == lo.m ? 0.0f : static_cast<float>(shift_of(lo.m, inv_t).from() - shift_of(hi.m, inv_t).from()), f = exp2f(x);
  return {hi.m, fmaf(lo.s, f, hi.s), hi.t + f * fmaf(lo.s, x, lo.t)};
}

// What the gradient needs of a row: dz = 2^x (ax x + b), + ka at the answer
struct Slopes { float m, ax, b, ka; };

// The row's numbers from its sums; `za` the answer's logit. Written by one thread.
__device__ __forceinline__ Slopes finish(const LossArgs& p, const Row& row, const Sums& s, float za, bool write) {
  Slopes g{s.m, 0.0f, 0.0f, 0.0f};
  float lp = 0.0f, kl = 0.0f, ent = 0.0f, each = 0.0f;
  if (row.a >= 0 && za > -INFINITY) {
    const float w = p.weight ? p.weight[row.n] : p.share, adv = p.adv[row.n];
    // the logarithm of the sum and what is subtracted from it in 64 bits: log-probabilities and
    // small KL terms are differences of larger numbers
    constexpr double kLn2d = 0.69314718055994530942;
    const Shift h = shift_of(s.m, p.inv_t);
    const double log_s = log(static_cast<double>(s.s)), power = static_cast<double>(s.t) / s.s;
    const double l = (za == s.m && h.far ? 0.0 : static_cast<double>(za) * h.c - h.from()) * kLn2d - log_s;
    lp = static_cast<float>(l);
    ent = static_cast<float>(log_s - power * kLn2d);
    const float ratio = expf(static_cast<float>(l - p.old_logp[row.n]));
    // by comparisons that NaN fails, so that it stays; no advantage makes nothing of an infinite ratio
    const float held = ratio < 1.0f - p.lo ? 1.0f - p.lo : ratio > 1.0f + p.hi ? 1.0f + p.hi : ratio;
    const float free = adv == 0.0f && ratio >= 0.0f ? 0.0f : ratio * adv, cut = held * adv;
    float c = cut < free ? 0.0f : -free;
    each = cut < free ? -cut : -free;
    if (p.ref) {
      const double d = p.ref[row.n] - l;
      const double e = expm1(d);
      kl = static_cast<float>(e - d);
      if (p.kl != 0.0f) {                              // e^d of a row may be infinite in 32 bits: 0 times it is not 0
        each = fmaf(p.kl, kl, each);
        c = fmaf(p.kl, -static_cast<float>(e), c);
      }
    }
    each = w * fmaf(-p.ent, ent, each);
    c *= w;
    // p = 2^x / s, log p = x ln 2 - log s:  (w ent p (log p + H) - c p) / t
    const float ke = w * p.ent * p.inv_t / s.s;
    g.ka = c * p.inv_t;
    g.ax = ke * kLn2;
    g.b = ke * (ent - static_cast<float>(log_s)) - g.ka / s.s;
  }
  if (write) {
    p.rows[row.n] = lp;
    p.rows[p.n + row.n] = kl;
    p.rows[2 * p.n + row.n] = ent;
    p.each[row.n] = each;
  }
  return g;
}
template <bool kFar> __device__ __forceinline__ float slope(const Slopes& g, float z, const Shift& h) {
  const float x = power_of<kFar>(z, h);
  return exp2_hw(x) * fmaf(g.ax, x, g.b);
}

// The rows' losses summed in a fixed order: a kernel of its own, since a counter of arrivals would
// have to be shared by calls on different streams or cleared by a launch too.
constexpr int kSumThreads = 512;
__global__ void __launch_bounds__(kSumThreads) loss_sum(const float* each, int64_t n, float* loss) {
  __shared__ double red[kSumThreads / 32];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += kSumThreads) s += each[i];
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kSumThreads / 32; ++i) s += red[i];
    *loss = static_cast<float>(s);
  }
}

// ---- a warp for a row -----------------------------------------------------------------
constexpr int kWarpThreads = 256;

template <typename T, int H> __global__ void __launch_bounds__(kWarpThreads) loss_warp(LossArgs p) {
  const int lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (kWarpThreads / 32) + (threadIdx.x >> 5);
  if (n >= p.n) return;
  const Row row = row_of(p, n, lane == 0);
  const T* z = static_cast<const T*>(p.z) + n * p.z_ld;
  float v[H], m = -INFINITY;
#pragma unroll
  for (int k = 0; k < H; ++k) {
    v[k] = k * 32 + lane < p.v ? to_f(z[k * 32 + lane]) : -INFINITY;
    m = fmaxf(m, v[k]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  Sums s{m, 0.0f, 0.0f};
  const Shift h = shift_of(m, p.inv_t);
  float za = -INFINITY;
#pragma unroll
  for (int k = 0; k < H; ++k) {
    if (h.far) add<true>(s, v[k], h);
    else add<false>(s, v[k], h);
    if (k * 32 + lane == row.a) za = clean(v[k]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s.s += __shfl_xor_sync(0xffffffffu, s.s, o);
    s.t += __shfl_xor_sync(0xffffffffu, s.t, o);
    za = fmaxf(za, __shfl_xor_sync(0xffffffffu, za, o));
  }
  const Slopes g = finish(p, row, s, za, lane == 0);
  if (!p.dz) return;
  T* d = static_cast<T*>(p.dz) + n * p.d_ld;
#pragma unroll
  for (int k = 0; k < H; ++k) {
    const int at = k * 32 + lane;
    if (at < p.v) d[at] = from_f<T>((h.far ? slope<true>(g, v[k], h) : slope<false>(g, v[k], h)) + (at == row.a ? g.ka : 0.0f));
  }
}

// ---- a cluster of blocks for a row ------------------------------------------------------
constexpr int kRowThreads = 384;

__device__ __forceinline__ float max_of(const uint4& q, float m) {
  return fmaxf(fmaxf(m, fmaxf(__uint_as_float(q.x), __uint_as_float(q.y))), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
}
__device__ __forceinline__ __nv_bfloat162 pair_of(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }

// A block takes candidates [first, first + count) of its row; shared memory mirrors their place within 16
// bytes of global memory, so that all but the ends move in pieces of 16 bytes.
template <typename T> __global__ void __launch_bounds__(kRowThreads, 3) loss_row(LossArgs p, int per) {
  constexpr int V = kVec16<T>;
  extern __shared__ __align__(16) char smem[];
  __shared__ Sums part[kRowThreads / 32], mine;
  __shared__ float answer;
  __shared__ Slopes slopes;
  cg::cluster_group cl = cg::this_cluster();
  const int ranks = cl.num_blocks(), rank = cl.block_rank();
  const int64_t n = blockIdx.x / ranks;
  const Row row = row_of(p, n, rank == 0 && threadIdx.x == 0);
  const int first = min(rank * per, p.v), count = min(per, p.v - first);
  const T* z = static_cast<const T*>(p.z) + n * p.z_ld + first;
  T* hold = reinterpret_cast<T*>(smem) + (reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T);
  const int head = min(count, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) / sizeof(T)) % V);
  const int whole = (count - head) / V;
  const int rest = count - whole * V;                  // the ends: [0, head) and behind the pieces
  float m = -INFINITY;
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat16 low = __ushort_as_bfloat16(0xff80);
    __nv_bfloat162 top = {low, low};
#pragma unroll 4
    for (int i = threadIdx.x; i < whole; i += kRowThreads) {
      const uint4 q = *reinterpret_cast<const uint4*>(z + head + i * V);
      *reinterpret_cast<uint4*>(hold + head + i * V) = q;
      top = __hmax2(top, __hmax2(__hmax2(pair_of(q.x), pair_of(q.y)), __hmax2(pair_of(q.z), pair_of(q.w))));
    }
    m = fmaxf(m, fmaxf(__low2float(top), __high2float(top)));
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < whole; i += kRowThreads) {
      const uint4 q = *reinterpret_cast<const uint4*>(z + head + i * V);
      *reinterpret_cast<uint4*>(hold + head + i * V) = q;
      m = max_of(q, m);
    }
  }
  for (int i = threadIdx.x; i < rest; i += kRowThreads) {
    const int at = i < head ? i : i + whole * V;
    hold[at] = z[at];
    m = fmaxf(m, to_f(z[at]));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5].m = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowThreads / 32; ++i) m = fmaxf(m, part[i].m);
  __syncthreads();
  Sums s{m, 0.0f, 0.0f};
  auto sum = [&](auto far) {
    constexpr bool kFar = decltype(far)::value;
    const Shift h = shift_of(m, p.inv_t);
#pragma unroll 2
    for (int i = threadIdx.x; i < whole; i += kRowThreads) {
      float v[V];
      load_vec<T, V>(hold + head + i * V, v);
#pragma unroll
      for (int j = 0; j < V; ++j) add<kFar>(s, v[j], h);
    }
    for (int i = threadIdx.x; i < rest; i += kRowThreads) add<kFar>(s, to_f(hold[i < head ? i : i + whole * V]), h);
  };
  if (m > -INFINITY) {
    if (shift_of(m, p.inv_t).far) sum(std::true_type());
    else sum(std::false_type());
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s.s += __shfl_xor_sync(0xffffffffu, s.s, o);
    s.t += __shfl_xor_sync(0xffffffffu, s.t, o);
  }
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kRowThreads / 32; ++i) {
      s.s += part[i].s;
      s.t += part[i].t;
    }
    mine = s;
    answer = row.a >= first && row.a < first + count ? clean(to_f(hold[row.a - first])) : -INFINITY;
  }
  if (ranks > 1) cl.sync(); else __syncthreads();
  if (threadIdx.x == 0) {
    Sums all = mine;
    float za = answer;
    if (ranks > 1) {
      all = *cl.map_shared_rank(&mine, 0);
      za = *cl.map_shared_rank(&answer, 0);
      for (int i = 1; i < ranks; ++i) {
        all = join(all, *cl.map_shared_rank(&mine, i), p.inv_t);
        za = fmaxf(za, *cl.map_shared_rank(&answer, i));
      }
    }
    slopes = finish(p, row, all, za, rank == 0);
  }
  if (ranks > 1) cl.sync(); else __syncthreads();      // the others' shared memory is read no more
  if (!p.dz) return;
  const Slopes g = slopes;
  const int answer_at = row.a - first;                 // in this block's candidates, if at all
  T* d = static_cast<T*>(p.dz) + n * p.d_ld + first;
  const bool same = ((reinterpret_cast<uintptr_t>(d) ^ reinterpret_cast<uintptr_t>(z)) & 15) == 0;
  auto write = [&](auto far) {
    constexpr bool kFar = decltype(far)::value;
    const Shift h = shift_of(g.m, p.inv_t);
#pragma unroll 2
    for (int i = threadIdx.x; i < whole; i += kRowThreads) {
      const int at = head + i * V;
      float v[V];
      load_vec<T, V>(hold + at, v);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = slope<kFar>(g, v[j], h);
      if (static_cast<unsigned>(answer_at - at) < static_cast<unsigned>(V) && row.a >= 0)
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += at + j == answer_at ? g.ka : 0.0f;
      if (same) {
        store_vec<T, V>(d + at, v);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) d[at + j] = from_f<T>(v[j]);
      }
    }
    for (int i = threadIdx.x; i < rest; i += kRowThreads) {
      const int at = i < head ? i : i + whole * V;
      d[at] = from_f<T>(slope<kFar>(g, to_f(hold[at]), h) + (at == answer_at && row.a >= 0 ? g.ka : 0.0f));
    }
  };
  if (shift_of(g.m, p.inv_t).far) write(std::true_type());
  else write(std::false_type());
}

template <typename T> int run(const LossArgs& a, int ranks, int per, cudaStream_t s) {
  if (ranks == 0) {
    const unsigned grid = static_cast<unsigned>((a.n + kWarpThreads / 32 - 1) / (kWarpThreads / 32));
    if (a.v <= 32) loss_warp<T, 1><<<grid, kWarpThreads, 0, s>>>(a);
    else if (a.v <= 128) loss_warp<T, 4><<<grid, kWarpThreads, 0, s>>>(a);
    else if (a.v <= 512) loss_warp<T, 16><<<grid, kWarpThreads, 0, s>>>(a);
    else return static_cast<int>(cudaErrorInvalidValue);
    if (const cudaError_t e = cudaGetLastError()) return static_cast<int>(e);
    loss_sum<<<1, kSumThreads, 0, s>>>(a.each, a.n, a.loss);
    return static_cast<int>(cudaGetLastError());
  }
  const size_t smem = (static_cast<size_t>(per) * sizeof(T) + 31) / 16 * 16;
  if (smem > 200 * 1024 || ranks > 8) return static_cast<int>(cudaErrorInvalidValue);
  if (const int e = allow_smem<loss_row<T>>(200 * 1024)) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.n * ranks));
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (const cudaError_t e = cudaLaunchKernelEx(&cfg, loss_row<T>, a, per)) return static_cast<int>(e);
  loss_sum<<<1, kSumThreads, 0, s>>>(a.each, a.n, a.loss);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

// args: a LossArgs; ranks: blocks of a row (0: a warp), per: candidates of a block
SURF_EXPORT int surf_policy_loss(const void* args, int dtype, int ranks, int per, void* stream) {
  const LossArgs& a = *static_cast<const LossArgs*>(args);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == kBf16 ? run<bf16>(a, ranks, per, s) : run<float>(a, ranks, per, s);
}
