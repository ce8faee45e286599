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
static_assert(sizeof(TokenArgs) == 9 * 8 + 6 * 4 + 2 * kMaxHeads * 4, "as the caller packs it");

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
// Ranks and the weight before a candidate by looking at every other lane in turn: 2 sizes'
// shuffles a head, all in registers (2048 rows of six heads 9.4 us, 410 KB: the two
// loops' chains of shuffles, in warps most of whose lanes are idle).
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
// an e; only there the logits are looked at again). That rests on an expf that never falls as
// its argument rises: so it is here, every argument from -0 to -104 looked at.
//
// With enough rows to fill the GPU a row is one block's (kStream): no barriers between
// blocks; the row is read again from the L2 cache and its exponentials made again instead
// of being kept (a slice of the whole row would not fit).
//
// Measured on a B200: 256 rows of 131072 under top_p 155 us in bf16 (67 MB), 160 us in f32 (134
// MB; bf16 without a limit 56 us), as clusters 325 us; at a temperature of 0.7 133 us, as
// clusters 215 us; one row of 32768 under top_k and top_p 18 us in both types, 64 rows of them in
// f32 24 us. What bounds many rows is instructions, 106 for a candidate under top_p (two
// exponentials, two weights in whole numbers, one place in the histogram) at 0.7 a cycle; what
// bounds a few rows is the cluster's barriers, thirteen of them under top_k with top_p, five of
// these for the second limit.
constexpr int kMaxCluster = 16, kMaxSlice = 16384, kMaxStream = kMaxCluster * kMaxSlice;
constexpr int kList = 512;
template <bool kStream> struct Large {
  static constexpr int kThreads = kStream ? 512 : 256, kWarps = kThreads / 32;
  static constexpr int kBinShift = kStream ? 16 : 18;          // 128 or 32 bins an octave of e, 40 octaves
  static constexpr int kBins = kStream ? 5136 : 1312;          // > 40 octaves, whole shares for 1 .. 16 blocks
  static constexpr int kNoWeight = 40 * (1 << (23 - kBinShift)) + 1;   // the first bin of e < 2^-40 alone
};
constexpr int kAllKept = 1 << 30, kNoBin = -1;

struct Found { u64 mass_before; unsigned count_before; int bin; };
struct Cut { u64 ties, mass_upto; uint32_t key; unsigned pad; };     // kept: keys above, `ties` equal ones

template <int kBins, int kWarps> struct TokenSmem {
  unsigned hist_lo[kBins + 32], hist_hi[kBins + 32], hist_c[kBins + 32];      // weight in two words, count
  uint32_t list_key[kList], list_e[kList];           // of the bin where the limit falls
  int list_at[kList];
  u64 warp_m[kWarps], share_m[kMaxCluster], x_m[kMaxCluster];
  unsigned warp_c[kWarps], share_c[kMaxCluster], x_c[kMaxCluster];
  float x_max[kMaxCluster], red[kWarps];
  Found found;
  Cut cut;
  unsigned list_n;
};

// w = floor(e * 2^40), e in [0, 1], as w1 * 2^23 + w0: the additions of 2^23 that round down
// leave the whole part in the low bits of a float (what is left is exact in between). Both
// come with the bits of 2^23 on top (kTop), which sums take off at their end.
constexpr uint32_t kTop = 0x4b000000u;
__device__ __forceinline__ void split_weight(float e, uint32_t& w1, uint32_t& w0) {
  const float t = __fmaf_rd(e, 131072.0f, 8388608.0f);
  const float rest = __fmaf_rn(e, 131072.0f, -__fsub_rn(t, 8388608.0f));
  w1 = __float_as_uint(t);
  w0 = __float_as_uint(__fmaf_rd(rest, 8388608.0f, 8388608.0f));
}
__device__ __forceinline__ u64 whole_weight(float e) {
  uint32_t w1, w0;
  split_weight(e, w1, w0);
  return (static_cast<u64>(w1 - kTop) << 23) + (w0 - kTop);
}
// *p += v in shared memory where v is not zero, without a branch
__device__ __forceinline__ void add_some(unsigned* p, unsigned v) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  asm volatile("{\n.reg .pred some;\nsetp.ne.u32 some, %1, 0;\n@some red.shared.add.u32 [%0], %1;\n}" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

template <typename T, int CS, bool kStream>
__global__ void __launch_bounds__(Large<kStream>::kThreads, 1024 / Large<kStream>::kThreads) large_kernel(TokenArgs a, int slice) {
  constexpr int kThreads = Large<kStream>::kThreads, kWarps = Large<kStream>::kWarps, kBins = Large<kStream>::kBins;
  constexpr int kNoWeight = Large<kStream>::kNoWeight;
  using Smem = TokenSmem<kBins, kWarps>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  float* zs = reinterpret_cast<float*>(smem_raw + (sizeof(Smem) + 15) / 16 * 16);
  auto bin_of_bits = [](uint32_t e) { return static_cast<int>((0x3f800000u - e) >> Large<kStream>::kBinShift); };
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
  const int slots = (off + n + 3) / 4 * 4;
  float mx = -INFINITY;
  if (!kStream && threadIdx.x < off) zs[threadIdx.x] = -INFINITY;
  if (!kStream && threadIdx.x < slots - off - n) zs[off + n + threadIdx.x] = -INFINITY;
  if (threadIdx.x < min(head, n)) {
    const float z = to_f(row[threadIdx.x]);
    if (!kStream) zs[off + threadIdx.x] = z;
    mx = fmaxf(mx, z);                               // passes NaN over
  }
  const int whole = n > head ? (n - head) / W * W : 0;
#pragma unroll 4
  for (int i = threadIdx.x * W; i < whole; i += kThreads * W) {
    float v[W];
    load_vec<T, W>(row + head + i, v);
#pragma unroll
    for (int j = 0; j < W; ++j) mx = fmaxf(mx, v[j]);
    if (!kStream) {
#pragma unroll
      for (int j = 0; j < W; j += 4)
        *reinterpret_cast<float4*>(zs + off + head + i + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    }
  }
  if (const int i = head + whole + threadIdx.x; i < n) {
    const float z = to_f(row[i]);
    if (!kStream) zs[off + i] = z;
    mx = fmaxf(mx, z);
  }
  auto clear = [&] {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sm.hist_lo[i] = sm.hist_hi[i] = sm.hist_c[i] = 0;
    __syncthreads();
  };
  mx = warp_max(mx);
  if (lane == 0) sm.red[warp] = mx;
  if (threadIdx.x == 0) sm.list_n = 0;
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

  // every warp owns a run of the slice, so that sums over warps are in index order
  const int run = (slots + kWarps * 128 - 1) / (kWarps * 128) * 128;
  const int w_lo = min(slots, warp * run), w_hi = min(slots, w_lo + run);
  const bool limited = q.k || q.p < 1.0;
  auto add = [&](int bin, u64 w) {           // two 32-bit additions: shared memory has no 64-bit one
    const unsigned x = static_cast<unsigned>(w), old = atomicAdd(&sm.hist_lo[bin], x);
    const unsigned up = static_cast<unsigned>(w >> 32) + (old + x < old ? 1u : 0u);
    if (up) atomicAdd(&sm.hist_hi[bin], up);
    if (q.k) atomicAdd(&sm.hist_c[bin], 1u);
  };
  // logit -> e (0 for NaN and what min_p drops)
  const bool plain = m < INFINITY && q.inv < INFINITY;   // else equal logits need below()
  auto exp_of = [&](float z) {
    const float e = expf(plain ? __fmul_rn(__fsub_rn(z, m), q.inv) : below(z, m, q.inv));
    return e >= q.min_p ? e : 0.0f;
  };
  auto args_of_four = [&](float (&z)[4]) {
    if (plain) {
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = __fmul_rn(__fsub_rn(z[j], m), q.inv);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = below(z[j], m, q.inv);
    }
  };
  auto exp_of_args = [&](float (&d)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = fmaxf(expf(d[j]), 0.0f);          // NaN: 0
    if (q.min_p > 0.0f) {
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = d[j] >= q.min_p ? d[j] : 0.0f;
    }
  };
  auto exp_of_four = [&](float (&z)[4]) {
    args_of_four(z);
    exp_of_args(z);
  };
  // the logits of candidates i .. i + 3 (slots; i a multiple of 4) again from the row
  auto logits_of_four = [&](int i, float (&z)[4]) {
    if (i >= off && i + 4 <= off + n) {
      load_vec<T, 4>(row + i - off, z);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = i + j >= off && i + j < off + n ? to_f(row[i + j - off]) : -INFINITY;
    }
  };
  // their e, and the e of one
  auto four = [&](int i, float (&e)[4]) {
    if constexpr (kStream) {
      logits_of_four(i, e);
      exp_of_four(e);
    } else {
      const float4 v = *reinterpret_cast<const float4*>(zs + i);
      e[0] = v.x; e[1] = v.y; e[2] = v.z; e[3] = v.w;
    }
  };
  auto one = [&](int i) {
    if constexpr (kStream) return i >= off && i < off + n ? exp_of(to_f(row[i - off])) : 0.0f;
    else return zs[i];
  };
  // weights into the histogram, or summed; sums of a thread stay within 2^32 for 256 slots
  uint32_t s1 = 0, s0 = 0;
  u64 above = 0;
  uint32_t added = 0;                        // candidates in s1 and s0
  auto flush = [&] {
    above += (static_cast<u64>(s1 - added * kTop) << 23) + (s0 - added * kTop);
    s1 = s0 = added = 0;
  };
  const int no_bin = kNoWeight + lane;       // bins that nobody reads take what has no weight
#pragma unroll 2
  for (int i = w_lo + lane * 4; i < w_hi; i += 128) {
    float e[4];
    four(i, e);
    if constexpr (!kStream) {
      exp_of_four(e);
      *reinterpret_cast<float4*>(zs + i) = make_float4(e[0], e[1], e[2], e[3]);
    }
    uint32_t w1[4], w0[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) split_weight(e[j], w1[j], w0[j]);
    if (limited) {
      // four additions in flight
      unsigned old[4];
      int bin[4];
      uint32_t x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bin[j] = min(bin_of_bits(__float_as_uint(e[j])), no_bin);
        x[j] = (w1[j] << 23) + (w0[j] - kTop);             // the low word: kTop << 23 is gone
        old[j] = atomicAdd(&sm.hist_lo[bin[j]], x[j]);
      }
      if (q.k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) atomicAdd(&sm.hist_c[bin[j]], w1[j] != kTop || w0[j] != kTop ? 1u : 0u);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        add_some(&sm.hist_hi[bin[j]], ((w1[j] & 0x7fffffu) >> 9) + (old[j] + x[j] < old[j] ? 1u : 0u));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s1 += w1[j];
        s0 += w0[j];
      }
      added += 4;
      if (kStream && ((i - w_lo) & 8191) >= 8064) flush();
    }
  }
  flush();
  __syncthreads();

  // Kept: everything in bins below `edge`; in bin `edge`, keys above the cut's and the first
  // `ties` of those equal to it.
  Cut cut{~0ull, 0, 0, 0};
  int edge = kAllKept;
  u64 tie_w = 0;
  unsigned listed = 0;
  bool by_list = true;
  if (limited) {
    u64 lim = 0;                             // 0: from the totals
    bool by_mass = true, intact = true, got;
    int level = -1;                          // of the key's digits, where the list is too short
    uint32_t prefix = 0;
    Found f{0, 0, 0};
    constexpr int kShare = kBins / CS, kEach = (kShare + kThreads - 1) / kThreads;
    for (;;) {
      // The first bin at which the running weight (or count) reaches the limit, over the
      // cluster's histograms: a block sums its share of the bins over the cluster, the block
      // whose share holds the bin tells the others.
      sync();
      {
        u64 bm[kEach], tm = 0;
        unsigned bc[kEach], tc = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          bm[j] = 0;
          bc[j] = 0;
          const int bin = threadIdx.x * kEach + j;
          if (bin < kShare) {
#pragma unroll 8
            for (int c = 0; c < CS; ++c) {
              bm[j] += (static_cast<u64>(peer(sm.hist_hi, c)[rank * kShare + bin]) << 32) + peer(sm.hist_lo, c)[rank * kShare + bin];
              if (q.k) bc[j] += peer(sm.hist_c, c)[rank * kShare + bin];
            }
          }
          tm += bm[j];
          tc += bc[j];
        }
        const u64 scan_m = warp_scan(tm, lane);
        const unsigned scan_c = warp_scan(tc, lane);
        if (lane == 31) {
          sm.warp_m[warp] = scan_m;
          sm.warp_c[warp] = scan_c;
        }
        __syncthreads();
        u64 all_m = 0, cm = scan_m - tm;
        unsigned all_c = 0, cc = scan_c - tc;
#pragma unroll
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
        if (threadIdx.x == 0) sm.found.bin = kNoBin;
        sync();
        u64 total_m = f.mass_before;
        unsigned total_c = f.count_before;
        for (int c = 0; c < CS; ++c) {
          if (c == rank) {
            cm += total_m;
            cc += total_c;
          }
          total_m += sm.share_m[c];
          total_c += sm.share_c[c];
        }
        if (!lim) {
          by_mass = !(q.k && total_c > static_cast<unsigned>(q.k));
          lim = by_mass ? (q.p < 1.0 ? mass_limit(q.p, total_m) : 0) : static_cast<u64>(q.k);
        }
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          const u64 before = by_mass ? cm : cc, upto = by_mass ? cm + bm[j] : cc + bc[j];
          if (before < lim && lim <= upto) {
            const Found at{cm, cc, rank * kShare + static_cast<int>(threadIdx.x) * kEach + j};
            for (int c = 0; c < CS; ++c) *peer(&sm.found, c) = at;
          }
          cm += bm[j];
          cc += bc[j];
        }
        sync();
        f = sm.found;
      }
      if (level < 0) {
        // the sums of what is surely kept, and the candidates of the bin where the limit falls
        // (bins by the e above which they lie: all bits of smaller bins are larger)
        edge = lim ? f.bin : kAllKept;
        const float e_sure = lim ? __uint_as_float(0x3f800000u - (static_cast<uint32_t>(edge) << Large<kStream>::kBinShift)) : -1.0f;
        const float e_edge = lim ? __uint_as_float(0x3f800000u - (static_cast<uint32_t>(edge + 1) << Large<kStream>::kBinShift)) : -1.0f;
        above = 0;
        auto add_four = [&](int i, const float (&e)[4]) {
          bool in_edge = false;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t w1, w0;
            split_weight(e[j], w1, w0);
            const bool sure = e[j] > e_sure;
            s1 += sure ? w1 : kTop;
            s0 += sure ? w0 : kTop;
            in_edge |= !sure && e[j] > e_edge;
          }
          added += 4;
          if (in_edge) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t bits = __float_as_uint(e[j]);
              if (bin_of_bits(bits) != edge || !whole_weight(__uint_as_float(bits))) continue;
              const unsigned at = atomicAdd(peer(&sm.list_n, 0), 1u);
              if (at < kList) {
                peer(sm.list_e, 0)[at] = bits;
                peer(sm.list_key, 0)[at] = key_of(clean(to_f(row[i + j - off])));
                peer(sm.list_at, 0)[at] = lo + i + j - off;
              }
            }
          }
        };
        // Under top_k most warps' 128 candidates lie below the edge's bin altogether; in a
        // stream their exponentials are spared by the arguments (0.001 below the edge's: a
        // thousand times the exponential's error). 256 rows of 131072 bf16 of normal logits:
        // top_k 50 134 -> 114 us, with top_p 182 -> 141. Under top_p alone it is not taken: it
        // costs a wide set 155 -> 164 us (top_p 0.95 at a temperature of 1), where it would spare a
        // narrow one 126 -> 106 us (at 0.3). A rule on where the limit lies has not been built.
        if (kStream && q.k) {
          const float d_edge = lim ? logf(e_edge) - 0.001f : -INFINITY;
#pragma unroll 2
          for (int i0 = w_lo; i0 < w_hi; i0 += 128) {
            const int i = i0 + lane * 4;
            float e[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (i < w_hi) {
              logits_of_four(i, e);
              args_of_four(e);
            }
            if (!__any_sync(0xffffffffu, fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])) > d_edge)) continue;
            exp_of_args(e);
            add_four(i, e);
            if (added >= 256) flush();
          }
        } else {
#pragma unroll 2
          for (int i = w_lo + lane * 4; i < w_hi; i += 128) {
            float e[4];
            four(i, e);
            add_four(i, e);
            if (kStream && ((i - w_lo) & 8191) >= 8064) flush();
          }
        }
        flush();
        if (!lim) break;
        sync();
        listed = *peer(&sm.list_n, 0);
        got = listed <= kList;
        if (got) {
          // their order by counting: a warp for each, all blocks with a copy of the list
          if (rank != 0) {
            for (unsigned i = threadIdx.x; i < listed; i += kThreads) {
              sm.list_key[i] = peer(sm.list_key, 0)[i];
              sm.list_e[i] = peer(sm.list_e, 0)[i];
              sm.list_at[i] = peer(sm.list_at, 0)[i];
            }
          }
          __syncthreads();
          for (unsigned i = rank * kWarps + warp; i < listed; i += CS * kWarps) {
            const uint32_t key = sm.list_key[i];
            const int at = sm.list_at[i];
            u64 before = 0;
            unsigned count = 0, same = 0;
            for (unsigned j = lane; j < listed; j += 32) {
              const uint32_t kj = sm.list_key[j];
              const bool equal_before = kj == key && sm.list_at[j] < at;
              if (kj > key || equal_before) {
                before += whole_weight(__uint_as_float(sm.list_e[j]));
                ++count;
              }
              same += equal_before;
            }
            before = f.mass_before + warp_sum(before);
            count = f.count_before + __reduce_add_sync(0xffffffffu, count);
            same = __reduce_add_sync(0xffffffffu, same);
            const u64 w = whole_weight(__uint_as_float(sm.list_e[i]));
            if ((by_mass ? before < lim && lim <= before + w : count + 1 == lim) && lane < CS)
              *peer(&sm.cut, lane) = Cut{static_cast<u64>(same) + 1, before + w, key, 0};
          }
          sync();
          cut = sm.cut;
        } else {
          level = 0;                         // many equal or nearly equal logits: by the bytes of their keys
          prefix = 0;
          intact = false;
        }
      } else {
        prefix = prefix << 8 | static_cast<uint32_t>(255 - f.bin);
        got = ++level == 4;
        if (got) {                           // all keys left are equal, and so are their weights
          const u64 each = whole_weight(expf(below(logit_of(prefix), m, q.inv)));
          const u64 ties = by_mass ? (lim - f.mass_before + each - 1) / each : lim - f.count_before;
          cut = Cut{ties, f.mass_before + ties * each, prefix, 0};
          level = -1;
        }
      }
      if (got) {
        if (by_mass || q.p >= 1.0) break;
        by_mass = true;                      // top_p of what top_k has left
        lim = mass_limit(q.p, cut.mass_upto);
        f = Found{0, 0, 0};
        if (rank == 0 && threadIdx.x == 0) sm.list_n = 0;
        if (!intact) {
          clear();
          for (int i = threadIdx.x; i < slots; i += kThreads) {
            const float e = one(i);
            if (const u64 w = whole_weight(e)) add(bin_of_bits(__float_as_uint(e)), w);
          }
        }
      } else {
        clear();
        for (int i = threadIdx.x; i < slots; i += kThreads) {
          const float e = one(i);
          if (bin_of_bits(__float_as_uint(e)) != edge) continue;
          const u64 w = whole_weight(e);
          if (!w) continue;
          const uint32_t key = key_of(clean(to_f(row[i - off])));
          if (level == 0 || key >> (32 - 8 * level) == prefix) add(255 - static_cast<int>(key >> (24 - 8 * level) & 255u), w);
        }
      }
    }
    by_list = listed <= kList;
  }
  // 0: dropped, 1: kept, 2: equal to the cut
  auto side = [&](uint32_t e, int i) {
    const int bin = bin_of_bits(e);
    if (bin != edge) return bin < edge ? 1 : 0;
    const uint32_t key = key_of(clean(to_f(row[i - off])));
    return key > cut.key ? 1 : key == cut.key ? 2 : 0;
  };

  // the runs' sums: what is surely kept, and the shares of the bin with the cut
  above = warp_sum(above);
  __syncthreads();
  if (lane == 0) {
    sm.warp_m[warp] = above;
    sm.warp_c[warp] = 0;
  }
  __syncthreads();
  if (edge != kAllKept) {
    tie_w = whole_weight(expf(below(logit_of(cut.key), m, q.inv)));
    if (by_list) {
      for (unsigned j = threadIdx.x; j < listed; j += kThreads) {
        const int i = sm.list_at[j] - lo;
        const uint32_t key = sm.list_key[j];
        if (i < 0 || i >= n || key < cut.key) continue;
        if (key > cut.key) atomicAdd(&sm.warp_m[(off + i) / run], whole_weight(__uint_as_float(sm.list_e[j])));
        else atomicAdd(&sm.warp_c[(off + i) / run], 1u);
      }
    } else {
      u64 more = 0;
      unsigned equal = 0;
      for (int i = w_lo + lane; i < w_hi; i += 32) {
        const float e = one(i);
        if (bin_of_bits(__float_as_uint(e)) != edge) continue;
        const u64 w = whole_weight(e);
        const int s = w ? side(__float_as_uint(e), i) : 0;
        if (s == 1) more += w;
        equal += s == 2;
      }
      more = warp_sum(more);
      equal = __reduce_add_sync(0xffffffffu, equal);
      if (lane == 0) {
        sm.warp_m[warp] += more;
        sm.warp_c[warp] = equal;
      }
    }
    __syncthreads();
  }
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
  // the run that holds it, again in parts, one for each warp, and the part walked 32 at a time
  if (threadIdx.x == 0) sm.found.bin = -1;
  __syncthreads();
  if (at >= mass_at && at < mass_at + mine && lane == 0) sm.found = Found{mass_at, static_cast<unsigned>(ties_at), warp};
  __syncthreads();
  if (sm.found.bin < 0) return;
  mass_at = sm.found.mass_before;
  ties_at = sm.found.count_before;
  const int r_lo = min(slots, sm.found.bin * run), r_hi = min(slots, r_lo + run);
  const int part = run / kWarps;             // run is a multiple of 128
  const int p_lo = min(r_hi, r_lo + warp * part), p_hi = warp == kWarps - 1 ? r_hi : min(r_hi, p_lo + part);
  u64 sure = 0;
  unsigned equal = 0;
#pragma unroll 4
  for (int i = p_lo + lane; i < p_hi; i += 32) {
    const float e = one(i);
    const u64 w = whole_weight(e);
    const int s = w ? side(__float_as_uint(e), i) : 0;
    if (s == 1) sure += w;
    equal += s == 2;
  }
  sure = warp_sum(sure);
  equal = __reduce_add_sync(0xffffffffu, equal);
  __syncthreads();
  if (lane == 0) {
    sm.warp_m[warp] = sure;
    sm.warp_c[warp] = equal;
  }
  __syncthreads();
  for (int w = 0; w < warp; ++w) {
    const u64 c = sm.warp_c[w];
    mass_at += sm.warp_m[w] + (min(ties_at + c, cut.ties) - min(ties_at, cut.ties)) * tie_w;
    ties_at += c;
  }
  if (at < mass_at || at >= mass_at + sure + (min(ties_at + equal, cut.ties) - min(ties_at, cut.ties)) * tie_w) return;
  for (int i0 = p_lo; i0 < p_hi; i0 += 32) {
    const int i = i0 + lane;
    const float e = i < p_hi ? one(i) : 0.0f;
    u64 w = whole_weight(e);
    const int s = w ? side(__float_as_uint(e), i) : 0;
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

template <typename T, int CS, bool kStream> int launch_large(const TokenArgs& a, int slice, cudaStream_t s) {
  using L = Large<kStream>;
  constexpr size_t kFixed = (sizeof(TokenSmem<L::kBins, L::kWarps>) + 15) / 16 * 16 + 16 * sizeof(float);   // a slice is shifted by up to 7
  const size_t smem = kFixed + (kStream ? 0 : static_cast<size_t>(slice) * sizeof(float));
  const int64_t blocks = static_cast<int64_t>(a.rows) * a.heads * CS;
  if (blocks > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
  if (const int rc = allow_smem<large_kernel<T, CS, kStream>, (CS > 8)>(kFixed + (kStream ? 0 : kMaxSlice * sizeof(float)))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(L::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CS > 1 ? 1 : 0;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, large_kernel<T, CS, kStream>, a, slice));
}

template <typename T> int launch_tokens(const TokenArgs& a, int widest, cudaStream_t s) {
  const int64_t answers = static_cast<int64_t>(a.rows) * a.heads;
  if (widest <= 32) {
    const int64_t blocks = surfk::ceil_div(answers, 4);
    if (blocks > 0x7fffffffLL) return static_cast<int>(cudaErrorInvalidValue);
    small_kernel<T><<<static_cast<unsigned>(blocks), 128, 0, s>>>(a);
    SURF_RETURN_LAUNCH();
  }
  if (answers >= 148 && widest > 8192 && widest <= kMaxStream) return launch_large<T, 1, true>(a, widest, s);
  // slices of at most 8192 candidates (32 a thread, 4 blocks on an SM), of 16384 once the
  // blocks fill the GPU. Wider clusters cost more at their barriers than their blocks save:
  // 64 rows of 32768 take 24 us in clusters of 4, 32 us in clusters of 8; 64 of 131072 57 us
  // in clusters of 8, 65 us in clusters of 16; one of 32768 18.5 us in 4 blocks, 18.1 in 16.
  int cs = 1;
  while (cs < kMaxCluster && widest > cs * (answers * cs >= 148 ? kMaxSlice : 8192)) cs *= 2;
  const int slice = static_cast<int>(surfk::ceil_div(widest, cs));
  if (slice > kMaxSlice) return static_cast<int>(cudaErrorInvalidValue);
  switch (cs) {
    case 1: return launch_large<T, 1, false>(a, slice, s);
    case 2: return launch_large<T, 2, false>(a, slice, s);
    case 4: return launch_large<T, 4, false>(a, slice, s);
    case 8: return launch_large<T, 8, false>(a, slice, s);
    default: return launch_large<T, 16, false>(a, slice, s);
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
