// tokens.cu — sampled answers from rows of logits: temperature, top-k, top-p, min-p,
// one given uniform number per answer (sm_100a).
//
// A row's candidates are ordered by (logit falling, index rising). With m the largest
// logit and e = exp((z - m) / temperature), a candidate's weight is the whole number
// w = floor(e * 2^40), so every sum below is exact and does not depend on the order it
// is taken in. Kept are the candidates with e >= min_p, of these the first top_k, and of
// these the ones with less than ceil(top_p * their total) of weight before them. The
// answer is the first index whose running kept weight exceeds floor(u * W), W the kept
// total; its log-probability is log(w / W). NaN logits count as -inf; a row that has
// nothing else answers -1 with log-probability -inf. Temperature 0 takes the largest.
//
// The kept set is a prefix of the order: all candidates above a threshold key and the
// first few equal to it. The threshold is found without sorting, by histograms of count
// and weight: one over the distance from the largest logit (in 1/64 of a temperature),
// then three over the digits of the key within one bin of the first.
#include <cooperative_groups.h>

#include "seq_common.cuh"

namespace {

using namespace seqk;
namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kMaxHeads = 16;

struct TokenArgs {
  const void* logits;
  const float* u;             // [rows, heads]
  const float *temperature, *top_p, *min_p;    // [rows] or null: the number below
  const int* top_k;                            // [rows] or null
  int* token;                 // [rows, heads]
  float* logp;                // [rows, heads]
  int64_t ld;
  float t0, p0, m0;
  int k0;
  int rows, heads;
  int offset[kMaxHeads], size[kMaxHeads];
};

struct Rule {                 // of one row
  float inv, min_p;
  int k;                      // 0: no limit
  double p;                   // >= 1: no limit
};

__device__ __forceinline__ Rule rule_of(const TokenArgs& a, int r) {
  const float t = a.temperature ? a.temperature[r] : a.t0;
  Rule q;
  q.k = a.top_k ? a.top_k[r] : a.k0;
  if (q.k < 0) q.k = 0;
  if (t > 0.0f) {
    q.inv = __fdiv_rn(1.0f, t);
  } else {
    q.inv = 1.0f;
    q.k = 1;
  }
  q.p = static_cast<double>(a.top_p ? a.top_p[r] : a.p0);
  if (!(q.p < 1.0)) q.p = 1.0;
  q.min_p = fminf(a.min_p ? a.min_p[r] : a.m0, 1.0f);      // the largest always stays
  return q;
}

// -inf for NaN, +0 for -0
__device__ __forceinline__ float clean(float z) { return z == z ? z + 0.0f : -INFINITY; }
// distance from the largest logit, in temperatures (<= 0)
__device__ __forceinline__ float below(float z, float m, float inv) { return z == m ? 0.0f : __fmul_rn(__fsub_rn(z, m), inv); }
__device__ __forceinline__ u64 weight(float z, float m, const Rule& q) {
  const float e = expf(below(z, m, q.inv));
  return z > -INFINITY && (e >= q.min_p) ? static_cast<u64>(__fmul_rn(e, 1099511627776.0f)) : 0ull;
}
// larger logit <-> larger key
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ u64 mass_limit(double p, u64 total) {
  const u64 v = static_cast<u64>(ceil(p * static_cast<double>(total)));
  return v < 1 ? 1 : v;
}
__device__ __forceinline__ u64 draw_at(float u, u64 total) {
  const u64 at = static_cast<u64>(static_cast<double>(fmaxf(u, 0.0f)) * static_cast<double>(total));
  return at < total ? at : total - 1;
}
__device__ __forceinline__ float log_share(u64 w, u64 total) {
  return static_cast<float>(log(static_cast<double>(w) / static_cast<double>(total)));
}

__device__ __forceinline__ float warp_max(float v) {
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename V> __device__ __forceinline__ V warp_scan(V v, int lane) {     // inclusive
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

// ---- up to 32 candidates: one warp, a lane each ---------------------------------------
template <typename T> __global__ void __launch_bounds__(128) small_kernel(TokenArgs a) {
  const int64_t id = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (id >= static_cast<int64_t>(a.rows) * a.heads) return;
  const int r = static_cast<int>(id / a.heads), h = static_cast<int>(id - static_cast<int64_t>(r) * a.heads);
  const int n = a.size[h];
  const Rule q = rule_of(a, r);
  const float z = lane < n ? clean(to_f(static_cast<const T*>(a.logits)[r * a.ld + a.offset[h] + lane])) : -INFINITY;
  const float m = warp_max(z);
  u64 w = weight(z, m, q);
  int rank = 0;
  for (int j = 0; j < n; ++j) {
    const float zj = __shfl_sync(0xffffffffu, z, j);
    if (zj > z || (zj == z && j < lane)) ++rank;
  }
  if (q.k && rank >= q.k) w = 0;
  u64 total = warp_sum(w);
  if (q.p < 1.0 && total) {
    const u64 lim = mass_limit(q.p, total);
    u64 before = 0;
    for (int j = 0; j < n; ++j) {
      const int rj = __shfl_sync(0xffffffffu, rank, j);
      const u64 wj = __shfl_sync(0xffffffffu, w, j);
      if (rj < rank) before += wj;
    }
    if (before >= lim) w = 0;
    total = warp_sum(w);
  }
  if (!total) {
    if (lane == 0) {
      a.token[id] = -1;
      a.logp[id] = -INFINITY;
    }
    return;
  }
  const u64 at = draw_at(a.u[id], total);
  const u64 upto = warp_scan(w, lane);
  if (upto > at && upto - w <= at) {
    a.token[id] = lane;
    a.logp[id] = log_share(w, total);
  }
}

// ---- many candidates: a cluster of CS blocks, the row's slices in shared memory -----------
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kPerThread = kBins / kThreads;
constexpr int kMaxSlice = 32768;

struct Found { u64 mass_before, mass; unsigned count_before, count; int bin; };

struct TokenSmem {
  u64 hist_m[kBins];
  unsigned hist_c[kBins];
  u64 warp_m[kWarps];
  unsigned warp_c[kWarps];
  Found found;
  float x_max[2];
  u64 x_m[2];                 // what the block tells the cluster; two slots in turn
  unsigned x_c[2];
  float red[kWarps];
};

template <typename T, int CS> __global__ void __launch_bounds__(kThreads) large_kernel(TokenArgs a, int slice) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  TokenSmem& sm = *reinterpret_cast<TokenSmem*>(smem_raw);
  float* zs = reinterpret_cast<float*>(smem_raw + sizeof(TokenSmem));
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = CS > 1 ? static_cast<int>(cluster.block_rank()) : 0;
  const int64_t id = blockIdx.x / CS;
  const int r = static_cast<int>(id / a.heads), h = static_cast<int>(id - static_cast<int64_t>(r) * a.heads);
  const int V = a.size[h];
  const int lo = min(V, rank * slice), n = min(V, lo + slice) - lo;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Rule q = rule_of(a, r);
  auto sync = [&] {
    if constexpr (CS > 1) cluster.sync();
    else __syncthreads();
  };
  auto peer = [&](auto* p, int c) {
    if constexpr (CS > 1) return cluster.map_shared_rank(p, c);
    else return p;
  };

  const T* row = static_cast<const T*>(a.logits) + r * a.ld + a.offset[h] + lo;
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float z = clean(to_f(row[i]));
    zs[i] = z;
    mx = fmaxf(mx, z);
  }
  mx = warp_max(mx);
  if (lane == 0) sm.red[warp] = mx;
  __syncthreads();
  if (warp == 0) {
    mx = warp_max(lane < kWarps ? sm.red[lane] : -INFINITY);
    if (lane == 0) sm.x_max[0] = mx;
  }
  sync();
  float m = -INFINITY;
#pragma unroll
  for (int c = 0; c < CS; ++c) m = fmaxf(m, *peer(&sm.x_max[0], c));

  if (m == -INFINITY) {                      // the same in every block of the cluster
    if (rank == 0 && threadIdx.x == 0) {
      a.token[id] = -1;
      a.logp[id] = -INFINITY;
    }
    sync();                                  // nobody leaves while others read its memory
    return;
  }

  auto bin_of = [&](float z) {               // 0 holds the largest logit; rising with falling z
    const float v = -below(z, m, q.inv) * 64.0f;
    return v < static_cast<float>(kBins - 1) ? static_cast<int>(v) : kBins - 1;
  };
  auto clear = [&] {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      sm.hist_m[i] = 0;
      sm.hist_c[i] = 0;
    }
    __syncthreads();
  };
  // the first bin at which the running count reaches `lim` (by_mass: the running weight),
  // over the cluster's histograms; `at_m`, `at_c`: what is above the first bin
  auto find = [&](bool by_mass, u64 lim, u64 at_m, unsigned at_c) {
    sync();
    u64 bm[kPerThread], tm = 0;
    unsigned bc[kPerThread], tc = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      bm[j] = 0;
      bc[j] = 0;
#pragma unroll
      for (int c = 0; c < CS; ++c) {
        bm[j] += peer(sm.hist_m, c)[threadIdx.x * kPerThread + j];
        bc[j] += peer(sm.hist_c, c)[threadIdx.x * kPerThread + j];
      }
      tm += bm[j];
      tc += bc[j];
    }
    const u64 sm_ = warp_scan(tm, lane);
    const unsigned sc = warp_scan(tc, lane);
    if (lane == 31) {
      sm.warp_m[warp] = sm_;
      sm.warp_c[warp] = sc;
    }
    if (threadIdx.x == 0) sm.found.bin = -1;
    sync();                                  // the histograms may change again after this
    u64 cm = at_m + sm_ - tm;
    unsigned cc = at_c + sc - tc;
    for (int w = 0; w < warp; ++w) {
      cm += sm.warp_m[w];
      cc += sm.warp_c[w];
    }
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const u64 before = by_mass ? cm : cc, upto = by_mass ? cm + bm[j] : cc + bc[j];
      if (before < lim && lim <= upto) sm.found = Found{cm, bm[j], cc, bc[j], static_cast<int>(threadIdx.x) * kPerThread + j};
      cm += bm[j];
      cc += bc[j];
    }
    __syncthreads();
    const Found f = sm.found;
    __syncthreads();
    return f;
  };
  // the key at which the limit falls, within bin `b0` of the first histogram
  auto refine = [&](bool by_mass, u64 lim, Found f, Found& end) {
    uint32_t prefix = 0;
    const int b0 = f.bin;
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : (level == 1 ? 10 : 0), width = level == 2 ? 1024 : 2048;
      clear();
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const float z = zs[i];
        const uint32_t key = key_of(z);
        if (bin_of(z) == b0 && (level == 0 || key >> (level == 1 ? 21 : 10) == prefix)) {
          const u64 w = weight(z, m, q);
          if (w) {
            const int digit = width - 1 - static_cast<int>((key >> shift) & (width - 1));
            atomicAdd(&sm.hist_m[digit], w);
            atomicAdd(&sm.hist_c[digit], 1u);
          }
        }
      }
      f = find(by_mass, lim, f.mass_before, f.count_before);
      prefix = (prefix << (level == 2 ? 10 : 11)) | static_cast<uint32_t>(width - 1 - f.bin);
    }
    end = f;
    return prefix;
  };

  // kept: keys above `tau`, and the first `ties` of those equal to it
  uint32_t tau = 0;
  u64 ties = ~0ull;
  if (q.k || q.p < 1.0) {
    clear();
    u64 tm = 0;
    unsigned tc = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float z = zs[i];
      const u64 w = weight(z, m, q);
      if (w) {
        const int b = bin_of(z);
        atomicAdd(&sm.hist_m[b], w);
        atomicAdd(&sm.hist_c[b], 1u);
        tm += w;
        ++tc;
      }
    }
    // totals of the cluster
    tm = warp_sum(tm);
    tc = __reduce_add_sync(0xffffffffu, tc);
    __syncthreads();
    if (lane == 0) {
      sm.warp_m[warp] = tm;
      sm.warp_c[warp] = tc;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      tm = 0;
      tc = 0;
      for (int w = 0; w < kWarps; ++w) {
        tm += sm.warp_m[w];
        tc += sm.warp_c[w];
      }
      sm.x_m[0] = tm;
      sm.x_c[0] = tc;
    }
    sync();
    u64 total = 0;
    unsigned count = 0;
#pragma unroll
    for (int c = 0; c < CS; ++c) {
      total += *peer(&sm.x_m[0], c);
      count += *peer(&sm.x_c[0], c);
    }
    const bool by_k = q.k && count > static_cast<unsigned>(q.k), by_p = q.p < 1.0;
    Found first{}, end{};
    if (by_k) {
      first = find(false, q.k, 0, 0);
      tau = refine(false, q.k, first, end);
      ties = static_cast<u64>(q.k) - end.count_before;
      total = end.mass_before + ties * (end.mass / end.count);      // equal keys, equal weights
    }
    if (by_p) {
      const u64 lim = mass_limit(q.p, total);
      if (by_k) {                                                   // the first histogram once more
        clear();
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const float z = zs[i];
          const u64 w = weight(z, m, q);
          if (w) {
            const int b = bin_of(z);
            atomicAdd(&sm.hist_m[b], w);
            atomicAdd(&sm.hist_c[b], 1u);
          }
        }
      }
      first = find(true, lim, 0, 0);
      tau = refine(true, lim, first, end);
      const u64 each = end.mass / end.count;
      ties = (lim - end.mass_before + each - 1) / each;
    }
  }

  // the draw: every warp owns a run of the slice, so sums are in index order
  const int run = ((n + kThreads - 1) / kThreads) * 32;
  const int w_lo = min(n, warp * run), w_hi = min(n, w_lo + run);
  u64 above = 0, each = 0;
  unsigned equal = 0;
  for (int i = w_lo + lane; i < w_hi; i += 32) {
    const float z = zs[i];
    const uint32_t key = key_of(z);
    if (key >= tau) {
      const u64 w = weight(z, m, q);
      if (w && key == tau) {
        ++equal;
        each = w;
      } else {
        above += w;
      }
    }
  }
  above = warp_sum(above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  for (int o = 16; o; o >>= 1) each = max(each, __shfl_xor_sync(0xffffffffu, each, o));
  __syncthreads();
  if (lane == 0) {
    sm.warp_m[warp] = above;
    sm.warp_c[warp] = equal;
    if (each) sm.found.mass = each;          // the same from every warp that has one
  }
  if (threadIdx.x == 0) sm.x_m[1] = sm.x_c[1] = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    u64 s = 0;
    unsigned c = 0;
    for (int w = 0; w < kWarps; ++w) {
      s += sm.warp_m[w];
      c += sm.warp_c[w];
    }
    sm.x_m[1] = s;
    sm.x_c[1] = c;
    sm.found.mass_before = c ? sm.found.mass : 0;
  }
  sync();
  u64 total = 0, mass_at = 0, ties_at = 0, all_ties = 0;
  u64 tie_w = 0;
#pragma unroll
  for (int c = 0; c < CS; ++c) {
    const u64 am = *peer(&sm.x_m[1], c);
    const u64 ac = *peer(&sm.x_c[1], c);
    tie_w = max(tie_w, *peer(&sm.found.mass_before, c));
    if (c < rank) {
      mass_at += am;
      ties_at += ac;
    }
    total += am;
    all_ties += ac;
  }
  total += min(all_ties, ties) * tie_w;
  mass_at += min(ties_at, ties) * tie_w;
  const u64 at = draw_at(a.u[id], total);
  // this warp's start
  for (int w = 0; w < warp; ++w) {
    const u64 c = sm.warp_c[w];
    mass_at += sm.warp_m[w] + (min(ties_at + c, ties) - min(ties_at, ties)) * tie_w;
    ties_at += c;
  }
  const u64 mine = sm.warp_m[warp] + (min(ties_at + sm.warp_c[warp], ties) - min(ties_at, ties)) * tie_w;
  if (at >= mass_at && at < mass_at + mine) {
    for (int i0 = w_lo; i0 < w_hi; i0 += 32) {
      const int i = i0 + lane;
      const float z = i < w_hi ? zs[i] : -INFINITY;
      const uint32_t key = key_of(z);
      u64 w = i < w_hi && key >= tau ? weight(z, m, q) : 0;
      const unsigned eq = __ballot_sync(0xffffffffu, w && key == tau);
      if (w && key == tau && ties_at + __popc(eq & ((1u << lane) - 1u)) >= ties) w = 0;
      ties_at += __popc(eq);
      const u64 upto = mass_at + warp_scan(w, lane);
      if (w && upto > at && upto - w <= at) {
        a.token[id] = lo + i;
        a.logp[id] = log_share(w, total);
      }
      mass_at = __shfl_sync(0xffffffffu, upto, 31);
      if (mass_at > at) break;
    }
  }
  sync();                                    // nobody leaves while others read its memory
}

template <typename T, int CS> int launch_large(const TokenArgs& a, int slice, cudaStream_t s) {
  const size_t smem = sizeof(TokenSmem) + static_cast<size_t>(slice) * sizeof(float);
  const int64_t blocks = static_cast<int64_t>(a.rows) * a.heads * CS;
  if (blocks > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
  if (const int rc = allow_smem<large_kernel<T, CS>>(sizeof(TokenSmem) + kMaxSlice * sizeof(float))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CS > 1 ? 1 : 0;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, large_kernel<T, CS>, a, slice));
}

template <typename T> int launch_tokens(const TokenArgs& a, int widest, cudaStream_t s) {
  if (widest <= 32) {
    const int64_t blocks = surfk::ceil_div(static_cast<int64_t>(a.rows) * a.heads, 4);
    if (blocks > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
    small_kernel<T><<<static_cast<unsigned>(blocks), 128, 0, s>>>(a);
    SURF_RETURN_LAUNCH();
  }
  int cs = 1;
  while (cs < 8 && widest > cs * 8192) cs *= 2;
  const int slice = static_cast<int>(surfk::ceil_div(widest, cs));
  if (slice > kMaxSlice) return static_cast<int>(cudaErrorInvalidValue);
  switch (cs) {
    case 1: return launch_large<T, 1>(a, slice, s);
    case 2: return launch_large<T, 2>(a, slice, s);
    case 4: return launch_large<T, 4>(a, slice, s);
    default: return launch_large<T, 8>(a, slice, s);
  }
}

}  // namespace

SURF_EXPORT int surf_sample_tokens(const void* args, int dtype, int widest, void* stream) {
  const TokenArgs a = *static_cast<const TokenArgs*>(args);
  if (a.rows <= 0 || a.heads <= 0) return 0;
  if (a.heads > kMaxHeads || widest < 1) return static_cast<int>(cudaErrorInvalidValue);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == kBf16 ? launch_tokens<bf16>(a, widest, s) : launch_tokens<float>(a, widest, s);
}
