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
// The kept set is a prefix of the order: all candidates above a threshold and the first few
// equal to it. The threshold is found without sorting: a histogram of weight (and count) over
// the leading bits of e, then the order within the one bin where the limit falls.
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
// One exponential per candidate: e is kept in shared memory in the logit's place, and all
// later passes work on its bits (e orders the candidates except where several logits share
// an e; only there the logits are looked at again).
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxSlice = 32768;
constexpr int kBinShift = 17;                        // 64 bins an octave of e, 40 octaves
constexpr int kBins = 2592;                          // > 40 * 64, whole shares for 1, 2, 4, 8 blocks
constexpr int kList = 1024;

struct Found { u64 mass_before; unsigned count_before, count; int bin; };
struct Cut { uint32_t key; unsigned count_before; u64 ties, mass_upto; };     // kept: keys above, `ties` equal ones

struct TokenSmem {
  unsigned hist_lo[kBins], hist_hi[kBins], hist_c[kBins];      // weight in two words, count
  u64 list_w[kList];
  uint32_t list_key[kList];
  int list_at[kList];
  u64 warp_m[kWarps], share_m[8], x_m[8];
  unsigned warp_c[kWarps], share_c[8], x_c[8];
  float x_max[8], red[kWarps];
  Found found;
  Cut cut;
  unsigned list_n;
};

// w = floor(e * 2^40) from the bits of e in [0, 1]
__device__ __forceinline__ u64 weight_of_bits(uint32_t e) {
  return (static_cast<u64>((e & 0x7fffffu) | 0x800000u) << 17) >> min(127u - (e >> 23), 63u);
}
__device__ __forceinline__ int bin_of_bits(uint32_t e) { return static_cast<int>((0x3f800000u - e) >> kBinShift); }

template <typename T, int CS> __global__ void __launch_bounds__(kThreads) large_kernel(TokenArgs a, int slice) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  TokenSmem& sm = *reinterpret_cast<TokenSmem*>(smem_raw);
  float* zs = reinterpret_cast<float*>(smem_raw + (sizeof(TokenSmem) + 15) / 16 * 16);
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

  if constexpr (CS > 1) cluster.barrier_arrive();    // waited for before the first look into another block
  // the slice into shared memory: candidate i at zs[off + i], so that 16-byte pieces of the
  // row fall on 16-byte pieces there; -inf before and behind
  const T* row = static_cast<const T*>(a.logits) + r * a.ld + a.offset[h] + lo;
  constexpr int W = kVec16<T>;
  const int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T));
  const int off = (W - head) % W;
  const int total_slots = (off + n + 3) / 4 * 4;
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < off; i += kThreads) zs[i] = -INFINITY;
  for (int i = off + n + threadIdx.x; i < total_slots; i += kThreads) zs[i] = -INFINITY;
  for (int i = threadIdx.x; i < min(head, n); i += kThreads) {
    const float z = clean(to_f(row[i]));
    zs[off + i] = z;
    mx = fmaxf(mx, z);
  }
  const int whole = n > head ? (n - head) / W * W : 0;
#pragma unroll 2
  for (int i = threadIdx.x * W; i < whole; i += kThreads * W) {
    float v[W];
    load_vec<T, W>(row + head + i, v);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      v[j] = clean(v[j]);
      mx = fmaxf(mx, v[j]);
    }
#pragma unroll
    for (int j = 0; j < W; j += 4)
      *reinterpret_cast<float4*>(zs + off + head + i + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  }
  for (int i = head + whole + threadIdx.x; i < n; i += kThreads) {
    const float z = clean(to_f(row[i]));
    zs[off + i] = z;
    mx = fmaxf(mx, z);
  }
  auto clear = [&] {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sm.hist_lo[i] = sm.hist_hi[i] = sm.hist_c[i] = 0;
    __syncthreads();
  };
  mx = warp_max(mx);
  if (lane == 0) sm.red[warp] = mx;
  clear();
  if constexpr (CS > 1) cluster.barrier_wait();
  if (warp == 0) {
    mx = warp_max(lane < kWarps ? sm.red[lane] : -INFINITY);
    if (lane < CS) *peer(&sm.x_max[rank], lane) = mx;
  }
  sync();
  float m = sm.x_max[0];
#pragma unroll
  for (int c = 1; c < CS; ++c) m = fmaxf(m, sm.x_max[c]);

  if (m == -INFINITY) {                      // the same in every block of the cluster
    if (rank == 0 && threadIdx.x == 0) {
      a.token[id] = -1;
      a.logp[id] = -INFINITY;
    }
    return;
  }

  const bool limited = q.k || q.p < 1.0;
  auto add = [&](int bin, u64 w) {           // two 32-bit additions: shared memory has no 64-bit one
    const unsigned w0 = static_cast<unsigned>(w);
    const unsigned old = atomicAdd(&sm.hist_lo[bin], w0);
    const unsigned up = static_cast<unsigned>(w >> 32) + (old + w0 < old ? 1u : 0u);
    if (up) atomicAdd(&sm.hist_hi[bin], up);
    if (q.k) atomicAdd(&sm.hist_c[bin], 1u);
  };
  // logits -> e; weights into the histogram
  for (int i = threadIdx.x * 4; i < total_slots; i += kThreads * 4) {
    float4 v = *reinterpret_cast<float4*>(zs + i);
    float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float z = e[j];
      e[j] = expf(below(z, m, q.inv));
      if (!(e[j] >= q.min_p) || z == -INFINITY) e[j] = 0.0f;
    }
    *reinterpret_cast<float4*>(zs + i) = make_float4(e[0], e[1], e[2], e[3]);
    if (limited) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t bits = __float_as_uint(e[j]);
        const u64 w = weight_of_bits(bits);
        if (w) add(bin_of_bits(bits), w);
      }
    }
  }
  __syncthreads();
  auto rebuild = [&] {
    clear();
    for (int i = threadIdx.x; i < total_slots; i += kThreads) {
      const uint32_t bits = __float_as_uint(zs[i]);
      const u64 w = weight_of_bits(bits);
      if (w) add(bin_of_bits(bits), w);
    }
  };

  // The first bin at which the running weight (by_mass) or count reaches `lim`, over the
  // cluster's histograms; total_m, total_c: all of them. A block sums its share of the bins
  // over the cluster; the block whose share holds the bin tells the others.
  u64 total_m = 0;
  unsigned total_c = 0;
  constexpr int kShare = kBins / CS, kEach = (kShare + kThreads - 1) / kThreads;
  auto find = [&](auto limit_of, u64 at_m, unsigned at_c) {
    sync();
    u64 bm[kEach], tm = 0;
    unsigned bc[kEach], tc = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      bm[j] = 0;
      bc[j] = 0;
      const int bin = threadIdx.x * kEach + j;
      if (bin < kShare) {
#pragma unroll
        for (int c = 0; c < CS; ++c) {
          bm[j] += (static_cast<u64>(peer(sm.hist_hi, c)[rank * kShare + bin]) << 32) + peer(sm.hist_lo, c)[rank * kShare + bin];
          if (q.k) bc[j] += peer(sm.hist_c, c)[rank * kShare + bin];
        }
      }
      tm += bm[j];
      tc += bc[j];
    }
    const u64 s_m = warp_scan(tm, lane);
    const unsigned s_c = warp_scan(tc, lane);
    if (lane == 31) {
      sm.warp_m[warp] = s_m;
      sm.warp_c[warp] = s_c;
    }
    __syncthreads();
    u64 all_m = 0, cm = s_m - tm;
    unsigned all_c = 0, cc = s_c - tc;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) {
        cm += sm.warp_m[w];
        cc += sm.warp_c[w];
      }
      all_m += sm.warp_m[w];
      all_c += sm.warp_c[w];
    }
    if (threadIdx.x < CS) {
      peer(sm.share_m, threadIdx.x)[rank] = all_m;
      peer(sm.share_c, threadIdx.x)[rank] = all_c;
    }
    if (threadIdx.x == 0) sm.found.bin = -1;
    sync();
    total_m = at_m;
    total_c = at_c;
    for (int c = 0; c < CS; ++c) {
      if (c == rank) {
        cm += total_m;
        cc += total_c;
      }
      total_m += sm.share_m[c];
      total_c += sm.share_c[c];
    }
    bool by_mass;
    const u64 lim = limit_of(by_mass);       // may depend on the totals; 0: no limit
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const u64 before = by_mass ? cm : cc, upto = by_mass ? cm + bm[j] : cc + bc[j];
      if (before < lim && lim <= upto) {
        const Found f{cm, cc, bc[j], rank * kShare + static_cast<int>(threadIdx.x) * kEach + j};
        for (int c = 0; c < CS; ++c) *peer(&sm.found, c) = f;
      }
      cm += bm[j];
      cc += bc[j];
    }
    sync();
    return sm.found;
  };

  bool intact = true;                        // the histogram of e
  // the place within bin f at which the limit falls
  auto refine = [&](bool by_mass, u64 lim, Found f) {
    if (rank == 0 && threadIdx.x == 0) sm.list_n = 0;
    sync();
    for (int i = threadIdx.x; i < total_slots; i += kThreads) {
      const uint32_t bits = __float_as_uint(zs[i]);
      if (bin_of_bits(bits) == f.bin) {
        const u64 w = weight_of_bits(bits);
        if (w) {
          const unsigned at = atomicAdd(peer(&sm.list_n, 0), 1u);
          if (at < kList) {
            peer(sm.list_w, 0)[at] = w;
            peer(sm.list_key, 0)[at] = key_of(clean(to_f(row[i - off])));
            peer(sm.list_at, 0)[at] = lo + i - off;
          }
        }
      }
    }
    sync();
    const unsigned listed = *peer(&sm.list_n, 0);
    if (listed <= kList) {                   // few: their order by counting, in the first block
      if (rank == 0) {
        for (unsigned i = threadIdx.x; i < listed; i += kThreads) {
          const uint32_t key = sm.list_key[i];
          const int at = sm.list_at[i];
          u64 before = f.mass_before;
          unsigned count = f.count_before, same = 0;
          for (unsigned j = 0; j < listed; ++j) {
            const uint32_t kj = sm.list_key[j];
            const bool equal = kj == key && sm.list_at[j] < at;
            if (kj > key || equal) {
              before += sm.list_w[j];
              ++count;
            }
            same += equal;
          }
          const u64 w = sm.list_w[i];
          if (by_mass ? before < lim && lim <= before + w : count + 1 == lim) {
            const Cut cut{key, count, static_cast<u64>(same) + 1, before + w};
            for (int c = 0; c < CS; ++c) *peer(&sm.cut, c) = cut;
          }
        }
      }
      sync();
      return sm.cut;
    }
    // many (equal or nearly equal logits): three digits of the key, by histograms
    intact = false;
    uint32_t prefix = 0;
    const int b0 = f.bin;
    Found g = f;
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : (level == 1 ? 10 : 0), width = level == 2 ? 1024 : 2048;
      clear();
      for (int i = threadIdx.x; i < total_slots; i += kThreads) {
        const uint32_t bits = __float_as_uint(zs[i]);
        const u64 w = bin_of_bits(bits) == b0 ? weight_of_bits(bits) : 0;
        if (w) {
          const uint32_t key = key_of(clean(to_f(row[i - off])));
          if (level == 0 || key >> (level == 1 ? 21 : 10) == prefix) add(width - 1 - static_cast<int>((key >> shift) & (width - 1)), w);
        }
      }
      g = find([&](bool& mass) { mass = by_mass; return lim; }, g.mass_before, g.count_before);
      prefix = (prefix << (level == 2 ? 10 : 11)) | static_cast<uint32_t>(width - 1 - g.bin);
    }
    // all keys here are equal, and so are their weights
    const u64 each = weight_of_bits(__float_as_uint(expf(below(__uint_as_float(prefix & 0x80000000u ? prefix & 0x7fffffffu : ~prefix), m, q.inv))));
    const u64 ties = by_mass ? (lim - g.mass_before + each - 1) / each : lim - g.count_before;
    return Cut{prefix, g.count_before, ties, g.mass_before + ties * each};
  };

  // kept: keys above the cut's, and the first `ties` of those equal to it
  Cut cut{0, 0, ~0ull, 0};
  uint32_t e_cut = 0;
  if (limited) {
    u64 lim = 0;
    bool by_mass = true;
    Found f = find([&](bool& mass) {
      by_mass = !(q.k && total_c > static_cast<unsigned>(q.k));
      mass = by_mass;
      lim = by_mass ? (q.p < 1.0 ? mass_limit(q.p, total_m) : 0) : static_cast<u64>(q.k);
      return lim;
    }, 0, 0);
    if (lim) {
      cut = refine(by_mass, lim, f);
      if (!by_mass && q.p < 1.0) {
        lim = mass_limit(q.p, cut.mass_upto);
        if (!intact) rebuild();
        f = find([&](bool& mass) { mass = true; return lim; }, 0, 0);
        cut = refine(true, lim, f);
      }
      e_cut = __float_as_uint(expf(below(__uint_as_float(cut.key & 0x80000000u ? cut.key & 0x7fffffffu : ~cut.key), m, q.inv)));
    }
  }

  // the draw: every warp owns a run of the slice, so sums are in index order
  const int run = (total_slots + kThreads - 1) / kThreads * 32;
  const int w_lo = min(total_slots, warp * run), w_hi = min(total_slots, w_lo + run);
  // 0: dropped, 1: above the cut, 2: equal to it
  auto side = [&](uint32_t bits, int i) {
    if (!cut.key || bits > e_cut) return 1;
    if (bits < e_cut) return 0;
    const uint32_t key = key_of(clean(to_f(row[i - off])));
    return key > cut.key ? 1 : key == cut.key ? 2 : 0;
  };
  u64 above = 0;
  unsigned equal = 0;
#pragma unroll 4
  for (int i = w_lo + lane; i < w_hi; i += 32) {
    const uint32_t bits = __float_as_uint(zs[i]);
    const u64 w = weight_of_bits(bits);
    if (w) {
      const int s = side(bits, i);
      if (s == 1) above += w;
      else equal += s == 2;
    }
  }
  above = warp_sum(above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  const u64 tie_w = cut.key ? weight_of_bits(e_cut) : 0;
  __syncthreads();
  if (lane == 0) {
    sm.warp_m[warp] = above;
    sm.warp_c[warp] = equal;
  }
  __syncthreads();
  if (threadIdx.x < CS) {
    u64 s = 0;
    unsigned c = 0;
    for (int w = 0; w < kWarps; ++w) {
      s += sm.warp_m[w];
      c += sm.warp_c[w];
    }
    peer(sm.x_m, threadIdx.x)[rank] = s;
    peer(sm.x_c, threadIdx.x)[rank] = c;
  }
  sync();                                    // the last: nobody looks into another block after it
  u64 total = 0, mass_at = 0, ties_at = 0, all_ties = 0;
#pragma unroll
  for (int c = 0; c < CS; ++c) {
    if (c < rank) {
      mass_at += sm.x_m[c];
      ties_at += sm.x_c[c];
    }
    total += sm.x_m[c];
    all_ties += sm.x_c[c];
  }
  total += min(all_ties, cut.ties) * tie_w;
  mass_at += min(ties_at, cut.ties) * tie_w;
  const u64 at = draw_at(a.u[id], total);
  // this warp's start
  for (int w = 0; w < warp; ++w) {
    const u64 c = sm.warp_c[w];
    mass_at += sm.warp_m[w] + (min(ties_at + c, cut.ties) - min(ties_at, cut.ties)) * tie_w;
    ties_at += c;
  }
  const u64 mine = sm.warp_m[warp] + (min(ties_at + sm.warp_c[warp], cut.ties) - min(ties_at, cut.ties)) * tie_w;
  if (at >= mass_at && at < mass_at + mine) {
    for (int i0 = w_lo; i0 < w_hi; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t bits = i < w_hi ? __float_as_uint(zs[i]) : 0;
      u64 w = weight_of_bits(bits);
      const int s = w ? side(bits, i) : 0;
      const unsigned eq = __ballot_sync(0xffffffffu, s == 2);
      if (s == 0 || (s == 2 && ties_at + __popc(eq & ((1u << lane) - 1u)) >= cut.ties)) w = 0;
      ties_at += __popc(eq);
      const u64 upto = mass_at + warp_scan(w, lane);
      if (w && upto > at && upto - w <= at) {
        a.token[id] = lo + i - off;
        a.logp[id] = log_share(w, total);
      }
      mass_at = __shfl_sync(0xffffffffu, upto, 31);
      if (mass_at > at) break;
    }
  }
}

template <typename T, int CS> int launch_large(const TokenArgs& a, int slice, cudaStream_t s) {
  constexpr size_t kFixed = (sizeof(TokenSmem) + 15) / 16 * 16 + 16 * sizeof(float);   // a slice is shifted by up to 7
  const size_t smem = kFixed + static_cast<size_t>(slice) * sizeof(float);
  const int64_t blocks = static_cast<int64_t>(a.rows) * a.heads * CS;
  if (blocks > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
  if (const int rc = allow_smem<large_kernel<T, CS>>(kFixed + kMaxSlice * sizeof(float))) return rc;
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
