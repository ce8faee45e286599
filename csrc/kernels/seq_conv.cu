// seq_conv.cu — short causal depthwise convolution over the tokens of a row,
// SiLU behind it: whole sequences, their gradient, single tokens (sm_100a).
//
//   pre[t, d] = bias[d] + sum_{k < W} w[d, k] * x[t - (W - 1) + k, d]
//   y = pre * sigmoid(pre)            (or pre itself)
//
// The tokens before the row are the W - 1 rows of `state` (oldest first, zeros
// without one); reset[b, t] drops everything before token t, and tokens from
// lengths[b] on are not there: they give zeros and are never read. Everything is
// one pass over memory (2 W + 4 flops per element against 4 to 8 bytes): the
// window slides through registers, a thread owning neighbouring channels over a
// stretch of tokens, so each x is read once (plus W - 1 of every stretch).
//
// Measured on a B200, W = 4, with resets, back to back: forward 256 x 128 x 1024 bf16 33 us (134
// MB, 4.1 TB/s), f32 50 us (268 MB, 5.3 TB/s), gradient 76 us (201 MB, 2.6 TB/s) and 97 us (403
// MB, 4.2 TB/s), a prompt of 16385 x 1024 18 us (67 MB, 3.7 TB/s) and 23 us (134 MB, 5.8 TB/s);
// one token of 64 envs 2.9 us. In bf16 neither the issue slots (0.49 and 0.59 of a cycle and
// scheduler in forward and gradient) nor DRAM is full: the 16 warps of an SM wait, most of all
// for results of their own arithmetic. Of the 14 instructions an element of the forward and 36
// of the gradient a sigmoid takes 5 and its derivative 10, an exponential and a reciprocal in a
// row; the SiLU takes 10 and 28 us. The wait and the copies of every token keep a thread's tokens
// apart, so that these chains do not overlap; fewer waits have not been tried.
#include <type_traits>

#include "seq_common.cuh"

namespace {

using namespace seqk;

struct ConvArgs {
  const void* x;
  const void* dy;
  const void* state;          // [B, W-1, D] or null
  const void* dfinal;         // [B, W-1, D] or null
  const float* w;             // [D, W]
  const float* bias;          // [D] or null
  const uint8_t* reset;       // [B, T] or null
  const int* lengths;         // [B] or null
  void* y;                    // forward: [B, T, D]; gradient: dx
  void* final_state;          // forward: [B, W-1, D] or null; gradient: dstate or null
  float* part;                // gradient: [rows][W + 1][D] partial sums of dw and dbias
  int64_t x_b, x_t, dy_b, dy_t, y_b, y_t, r_b;
  int B, T, D, silu;
  int tt, chunks;             // tokens of a stretch, stretches of a row
};
static_assert(sizeof(ConvArgs) == 18 * 8 + 6 * 4, "as the caller packs it");

// Channels of a thread: in whole sequences 16 bytes of them in the forward, 8 in the
// gradient (its weights, sums and pending dx fill the registers otherwise), 4 bytes where
// rows are only aligned to that, else one. All the arithmetic is on pairs of channels
// (f32x2), a lone channel being half a pair.
//
// Tokens come through a ring in shared memory, kU of them on their way to every thread by
// asynchronous copies. A thread reads only what it has copied itself, so there are no
// barriers; held in registers, the 8 tokens of 4 channels cost the warps that hide the
// latency (256 x 128 x 1024: forward 67 us, gradient 186 us; with the ring 41 and 110 us).
constexpr int kThreads = 256, kU = 8;
template <int V> constexpr int kPairs = (V + 1) / 2;
template <int V> struct Pairs { f2 p[kPairs<V>]; };

template <int V> __device__ __forceinline__ Pairs<V> zeros() {
  Pairs<V> r;
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) r.p[i].v = 0;
  return r;
}
template <int V> __device__ __forceinline__ Pairs<V> to_pairs(const float (&v)[V]) {
  Pairs<V> r;
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) r.p[i] = pack2(v[2 * i], 2 * i + 1 < V ? v[(2 * i + 1) % V] : 0.0f);
  return r;
}
template <int V> __device__ __forceinline__ void from_pairs(const Pairs<V>& r, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) {
    float lo, hi;
    unpack2(r.p[i], lo, hi);
    v[2 * i] = lo;
    if (2 * i + 1 < V) v[(2 * i + 1) % V] = hi;
  }
}
template <int V> __device__ __forceinline__ void madd(Pairs<V>& c, const Pairs<V>& x, const Pairs<V>& y) {
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) c.p[i] = fma2(x.p[i], y.p[i], c.p[i]);
}

// V channels of a row as they are in memory
template <typename T, int V> struct Raw {
  static constexpr int kBytes = V * static_cast<int>(sizeof(T));
  using Word = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, uint32_t, uint16_t>>>;
  Word w;
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const Word*>(p); }
  __device__ __forceinline__ void clear() { w = Word{}; }
  static __device__ __forceinline__ void copy_async(Word* dst, const T* src) {
    const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
    if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else if constexpr (kBytes >= 4) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(kBytes) : "memory");
  }
  __device__ __forceinline__ Pairs<V> pairs() const {
    float v[V];
    if constexpr (sizeof(T) == 4) {
      const float* q = reinterpret_cast<const float*>(&w);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = q[i];
    } else if constexpr (V == 1) {
      v[0] = __uint_as_float(static_cast<uint32_t>(w) << 16);
    } else {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        v[2 * i] = __uint_as_float(q[i] << 16);
        v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
      }
    }
    return to_pairs<V>(v);
  }
};
template <typename T, int V> __device__ __forceinline__ Pairs<V> load_pairs_of(const T* p) {
  Raw<T, V> r;
  r.load(p);
  return r.pairs();
}
template <typename T, int V> __device__ __forceinline__ void store_pairs_of(T* p, const Pairs<V>& r) {
  float v[V];
  from_pairs<V>(r, v);
  store_vec<T, V>(p, v);
}

// The channels' weights, tap by tap
template <int W, int V> __device__ __forceinline__ void load_weights(const float* p, Pairs<V> (&w)[W]) {
  float flat[V * W];
  if constexpr (V * W % 4 == 0 && V > 1) {
#pragma unroll
    for (int q = 0; q < V * W / 4; ++q) {
      const float4 v = reinterpret_cast<const float4*>(p)[q];
      flat[4 * q] = v.x; flat[4 * q + 1] = v.y; flat[4 * q + 2] = v.z; flat[4 * q + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int q = 0; q < V * W; ++q) flat[q] = p[q];
  }
#pragma unroll
  for (int k = 0; k < W; ++k) {
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = flat[i * W + k];
    w[k] = to_pairs<V>(v);
  }
}

// One stretch of tokens of one row, as a thread sees it.
template <typename T> struct Stretch {
  const T* x;
  const T* state;             // [W - 1] rows before the first token, or null
  const uint8_t* reset;
  int b, chunk, t0, t1, len;
  __device__ __forceinline__ Stretch(const ConvArgs& a, int item, int d, int W) {
    b = item / a.chunks;
    chunk = item - b * a.chunks;
    len = a.lengths ? max(0, min(a.T, a.lengths[b])) : a.T;
    t0 = chunk * a.tt;
    t1 = min(a.T, t0 + a.tt);
    x = static_cast<const T*>(a.x) + b * a.x_b + d;
    state = a.state ? static_cast<const T*>(a.state) + static_cast<int64_t>(b) * (W - 1) * a.D + d : nullptr;
    reset = a.reset ? a.reset + b * a.r_b : nullptr;
  }
  __device__ __forceinline__ bool cut(int t) const { return reset && t >= 0 && t < len && reset[t]; }
};

// Bit u: token t + u starts an episode, for the 8 tokens from t on.
template <typename T> __device__ __forceinline__ unsigned cuts_of(const Stretch<T>& s, int t) {
  static_assert(kU == 8, "the flags of 8 tokens are one word");
  if (!s.reset) return 0;
  const uint8_t* p = s.reset + t;
  if ((reinterpret_cast<uintptr_t>(p) & 7) == 0 && t + 8 <= s.len && *reinterpret_cast<const unsigned long long*>(p) == 0) return 0;
  unsigned m = 0;
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (t + u < s.len && p[u]) m |= 1u << u;
  return m;
}

// The tokens of a row on their way to one thread: slot u of kU holds token t0 + u, then
// t0 + u + kU, ... (kAsync), or the kU tokens of a step are loaded at its start.
template <typename T, int V> struct Ring {
  static constexpr bool kAsync = Raw<T, V>::kBytes >= 4;
  typename Raw<T, V>::Word* slot;              // of this thread
  const T* src;
  int64_t stride;
  int stop;                                    // first token that is not there
  Raw<T, V> held[kAsync ? 1 : kU];
  __device__ __forceinline__ void issue(int u, int t) {
    if constexpr (kAsync)
      if (t < stop) Raw<T, V>::copy_async(slot + u * kThreads, src + t * stride);
  }
  __device__ __forceinline__ void batch(int t) {
    if constexpr (!kAsync) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        held[u].clear();
        if (t + u < stop) held[u].load(src + (t + u) * stride);
      }
    }
  }
  // token t in slot u (anything if it is not there)
  __device__ __forceinline__ Pairs<V> get(int u) {
    if constexpr (kAsync) {
      Raw<T, V> r;
      r.w = slot[u * kThreads];
      return r.pairs();
    } else {
      return held[u].pairs();
    }
  }
};

// The W - 1 tokens before the stretch as its first token finds them (before its own reset).
template <typename T, int W, int V>
__device__ __forceinline__ void window_of(const ConvArgs& a, const Stretch<T>& s, Pairs<V> (&h)[W - 1]) {
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const int t = s.t0 - (W - 1) + j;
    h[j] = zeros<V>();
    if (t >= 0 && t < s.len) {
      if (s.cut(t)) {
#pragma unroll
        for (int q = 0; q < j; ++q) h[q] = zeros<V>();
      }
      h[j] = load_pairs_of<T, V>(s.x + t * a.x_t);
    } else if (t < 0 && s.state) {
      h[j] = load_pairs_of<T, V>(s.state + static_cast<int64_t>(W - 1 + t) * a.D);
    }
  }
}

// ---- whole sequences ----------------------------------------------------------------
// A thread keeps its channels' weights and takes one stretch after the other.
template <typename T, int W, int V>
__global__ void __launch_bounds__(kThreads, 2) conv_kernel(ConvArgs a, int items) {
  extern __shared__ __align__(16) unsigned char smem[];
  using Word = typename Raw<T, V>::Word;
  const int cg = blockIdx.x * blockDim.x + threadIdx.x, d = cg * V;
  if (cg >= a.D / V) return;
  Pairs<V> w[W], bias = zeros<V>();
  load_weights<W, V>(a.w + static_cast<int64_t>(d) * W, w);
  if (a.bias) {
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = a.bias[d + i];
    bias = to_pairs<V>(v);
  }
  for (int item = blockIdx.y * blockDim.y + threadIdx.y; item < items; item += gridDim.y * blockDim.y) {
    const Stretch<T> s(a, item, d, W);
    T* y = static_cast<T*>(a.y) + s.b * a.y_b + d;
    Pairs<V> h[W - 1];
    window_of<T, W, V>(a, s, h);
    const int live = min(s.t1, s.len);
    Ring<T, V> in{reinterpret_cast<Word*>(smem) + threadIdx.y * blockDim.x + threadIdx.x, s.x, a.x_t, live};
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      in.issue(u, s.t0 + u);
      cp_async_commit();
    }
    // whole: kU tokens are there; resets: one of them starts an episode
    auto step = [&](int t, unsigned cuts, auto whole, auto resets) {
      constexpr bool kWhole = decltype(whole)::value, kResets = decltype(resets)::value;
      in.batch(t);
#pragma unroll (kWhole || !Ring<T, V>::kAsync ? kU : 1)
      for (int u = 0; u < kU; ++u) {
        if (kWhole || t + u < live) {
          cp_async_wait<kU - 1>();
          if (kResets && (cuts >> u & 1u)) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j) h[j] = zeros<V>();
          }
          const Pairs<V> now = in.get(u);
          Pairs<V> acc = bias;
#pragma unroll
          for (int j = 0; j < W - 1; ++j) madd<V>(acc, w[j], h[j]);
          madd<V>(acc, w[W - 1], now);
#pragma unroll
          for (int j = 0; j + 1 < W - 1; ++j) h[j] = h[j + 1];
          h[W - 2] = now;
          float o[V];
          from_pairs<V>(acc, o);
          if (a.silu) {
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] *= sigmoid(o[i]);
          }
          store_vec<T, V>(y + (t + u) * a.y_t, o);
          in.issue(u, t + u + kU);
          cp_async_commit();
        }
      }
    };
    for (int t = s.t0; t < live; t += kU) {
      const unsigned cuts = cuts_of<T>(s, t);
      if (t + kU > live) step(t, cuts, std::false_type{}, std::true_type{});
      else if (cuts) step(t, cuts, std::true_type{}, std::true_type{});
      else step(t, 0, std::true_type{}, std::false_type{});
    }
    cp_async_wait<0>();
    for (int t = max(s.t0, live); t < s.t1; ++t) store_pairs_of<T, V>(y + t * a.y_t, zeros<V>());
    // what the next token finds behind it: by the stretch of the last token
    if (a.final_state && (s.len > 0 ? (s.len - 1 >= s.t0 && s.len - 1 < s.t0 + a.tt) : s.chunk == 0)) {
      T* f = static_cast<T*>(a.final_state) + static_cast<int64_t>(s.b) * (W - 1) * a.D + d;
#pragma unroll
      for (int j = 0; j < W - 1; ++j) store_pairs_of<T, V>(f + static_cast<int64_t>(j) * a.D, h[j]);
    }
  }
}

// ---- gradient -------------------------------------------------------------------------
// One sweep in token order: with the window at hand pre[t] is recomputed, dpre[t] =
// dy[t] * silu'(pre[t]) is spread onto the W pending dx of the tokens that it sees,
// and dx[t - (W - 1)] is then complete. A stretch runs W - 1 tokens on into the next
// one for its own last tokens; only its own tokens count for dw and dbias, whose
// sums a block joins in shared memory and leaves as one row of `part`, summed in
// row order by conv_reduce_kernel: no atomics, so a rerun gives the same bits.
template <typename T, int W, int V>
__global__ void __launch_bounds__(kThreads, 2) conv_grad_kernel(ConvArgs a, int items) {
  extern __shared__ __align__(16) unsigned char smem[];
  using Word = typename Raw<T, V>::Word;
  float* red = reinterpret_cast<float*>(smem);                  // at the end: [blockDim.y][W + 1][blockDim.x * V]
  const int cg = blockIdx.x * blockDim.x + threadIdx.x;
  const int d = cg * V;
  const bool on = cg < a.D / V;
  Pairs<V> w[W], dw[W], bias = zeros<V>(), db = zeros<V>();
#pragma unroll
  for (int k = 0; k < W; ++k) dw[k] = w[k] = zeros<V>();
  if (on) {
    load_weights<W, V>(a.w + static_cast<int64_t>(d) * W, w);
    if (a.bias) {
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = a.bias[d + i];
      bias = to_pairs<V>(v);
    }
    for (int item = blockIdx.y * blockDim.y + threadIdx.y; item < items; item += gridDim.y * blockDim.y) {
      const Stretch<T> s(a, item, d, W);
      const T* dy = static_cast<const T*>(a.dy) + s.b * a.dy_b + d;
      T* dx = static_cast<T*>(a.y) + s.b * a.y_b + d;
      const int64_t ends = static_cast<int64_t>(s.b) * (W - 1) * a.D + d;
      const T* df = a.dfinal ? static_cast<const T*>(a.dfinal) + ends : nullptr;
      T* ds = a.final_state ? static_cast<T*>(a.final_state) + ends : nullptr;
      Pairs<V> h[W - 1], pend[W];                    // pend[j]: dx of token t - j so far
      window_of<T, W, V>(a, s, h);
#pragma unroll
      for (int j = 0; j < W; ++j) pend[j] = zeros<V>();
      if (s.len == 0 && s.chunk == 0 && df) {        // an empty row hands its state on
#pragma unroll
        for (int j = 0; j < W - 1; ++j) pend[j + 1] = load_pairs_of<T, V>(df + static_cast<int64_t>(W - 2 - j) * a.D);
      }
      // Tokens from `from` on still wait for their dx. A reset at token t ends the wait of all
      // before it: theirs is written there and then, and what is added to them later is not.
      int from = s.chunk == 0 && ds ? -(W - 1) : s.t0;
      auto emit = [&](int t, const Pairs<V>& v) {
        if (t >= 0) store_pairs_of<T, V>(dx + t * a.y_t, v);
        else store_pairs_of<T, V>(ds + static_cast<int64_t>(W - 1 + t) * a.D, v);
      };
      const int end = s.t1 + W - 1;
      Word* const slots = reinterpret_cast<Word*>(smem) + threadIdx.y * blockDim.x + threadIdx.x;
      const int stop = min(end, s.len);
      Ring<T, V> xin{slots, s.x, a.x_t, stop}, gin{slots + kU * kThreads, dy, a.dy_t, stop};
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        xin.issue(u, s.t0 + u);
        gin.issue(u, s.t0 + u);
        cp_async_commit();
      }
      // whole: kU tokens of the stretch's own, the row goes on behind them; resets: one of them
      // starts an episode
      auto step = [&](int tb, unsigned cuts, auto whole, auto resets) {
        constexpr bool kWhole = decltype(whole)::value, kResets = decltype(resets)::value;
        xin.batch(tb);
        gin.batch(tb);
#pragma unroll (kWhole || !Ring<T, V>::kAsync ? kU : 1)
        for (int u = 0; u < kU; ++u) {
          const int t = tb + u;
          if (kWhole || t < end) {
            cp_async_wait<kU - 1>();
            const Pairs<V> now = kWhole || t < s.len ? xin.get(u) : zeros<V>();
            if (kWhole || t < s.len) {
              if (kResets && (cuts >> u & 1u)) {
#pragma unroll
                for (int j = 0; j < W - 1; ++j) h[j] = zeros<V>();
#pragma unroll
                for (int j = W - 1; j > 0; --j)
                  if (t - j >= from && t - j < s.t1) emit(t - j, pend[j]);
                from = max(from, t);
              }
              Pairs<V> g = gin.get(u);
              if (a.silu) {
                Pairs<V> pre = bias;
#pragma unroll
                for (int j = 0; j < W - 1; ++j) madd<V>(pre, w[j], h[j]);
                madd<V>(pre, w[W - 1], now);
                float p[V], q[V];
                from_pairs<V>(pre, p);
                from_pairs<V>(g, q);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                  const float sg = sigmoid(p[i]);
                  q[i] *= sg * fmaf(p[i], 1.0f - sg, 1.0f);
                }
                g = to_pairs<V>(q);
              }
              madd<V>(pend[0], w[W - 1], g);
#pragma unroll
              for (int j = 1; j < W; ++j) madd<V>(pend[j], w[W - 1 - j], g);
              if (kWhole || t < s.t1) {
#pragma unroll
                for (int i = 0; i < kPairs<V>; ++i) db.p[i] = add2(db.p[i], g.p[i]);
#pragma unroll
                for (int k = 0; k < W - 1; ++k) madd<V>(dw[k], h[k], g);
                madd<V>(dw[W - 1], now, g);
              }
              if (!kWhole && t == s.len - 1 && df) {             // the state behind the last token
#pragma unroll
                for (int j = 0; j < W - 1; ++j) {
                  const Pairs<V> e = load_pairs_of<T, V>(df + static_cast<int64_t>(W - 2 - j) * a.D);
#pragma unroll
                  for (int i = 0; i < kPairs<V>; ++i) pend[j].p[i] = add2(pend[j].p[i], e.p[i]);
                }
              }
            }
            const int done = t - (W - 1);
            if (done >= from && (kWhole || done < s.t1)) emit(done, pend[W - 1]);
#pragma unroll
            for (int j = W - 1; j > 0; --j) pend[j] = pend[j - 1];
            pend[0] = zeros<V>();
#pragma unroll
            for (int j = 0; j + 1 < W - 1; ++j) h[j] = h[j + 1];
            h[W - 2] = now;
            xin.issue(u, t + kU);
            gin.issue(u, t + kU);
            cp_async_commit();
          }
        }
      };
      for (int tb = s.t0; tb < end; tb += kU) {
        const unsigned cuts = cuts_of<T>(s, tb);
        if (tb + kU > s.t1 || tb + kU >= s.len) step(tb, cuts, std::false_type{}, std::true_type{});
        else if (cuts) step(tb, cuts, std::true_type{}, std::true_type{});
        else step(tb, 0, std::true_type{}, std::false_type{});
      }
      cp_async_wait<0>();
    }
  }
  __syncthreads();                             // the rings are done with
  // join the block's rows of sums
  const int cols = blockDim.x * V;
  float* mine = red + threadIdx.y * (W + 1) * cols + threadIdx.x * V;
#pragma unroll
  for (int k = 0; k <= W; ++k) {
    float v[V];
    from_pairs<V>(k < W ? dw[k % W] : db, v);
#pragma unroll
    for (int i = 0; i < V; ++i) mine[k * cols + i] = v[i];
  }
  __syncthreads();
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  for (int e = tid; e < (W + 1) * cols; e += blockDim.x * blockDim.y) {
    float s = 0.0f;
    for (int r = 0; r < static_cast<int>(blockDim.y); ++r) s += red[r * (W + 1) * cols + e];
    const int k = e / cols, c = blockIdx.x * cols + (e - k * cols);
    if (c < a.D) a.part[(static_cast<int64_t>(blockIdx.y) * (W + 1) + k) * a.D + c] = s;
  }
}

// dw[d, k] and dbias[d] from the rows of `part`, 8 row sums side by side, joined in order
template <int W>
__global__ void __launch_bounds__(256) conv_reduce_kernel(const float* part, int rows, int D, float* dw, float* dbias) {
  __shared__ float red[8][33];
  const int e = blockIdx.x * 32 + threadIdx.x;
  const int total = (W + 1) * D;
  float s = 0.0f;
  if (e < total)
    for (int r = threadIdx.y; r < rows; r += 8) s += part[static_cast<int64_t>(r) * total + e];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && e < total) {
#pragma unroll
    for (int r = 1; r < 8; ++r) s += red[r][threadIdx.x];
    const int k = e / D, d = e - k * D;
    if (k < W) dw[static_cast<int64_t>(d) * W + k] = s;
    else if (dbias) dbias[d] = s;
  }
}

// ---- single tokens -----------------------------------------------------------------------
// Row r is the next token of the env in slot slots[r] of the state pool (-1: none, its
// output is zero); the slot's window is moved on in place.
template <typename T, int W, int V>
__global__ void __launch_bounds__(128) conv_step_kernel(const T* x, int64_t ldx, const float* w, const float* bias, T* pool,
                                                        const uint8_t* reset, const int* slots, int n_slots, T* y, int64_t ldy,
                                                        int D, int silu, int* err) {
  const int r = blockIdx.x, d = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (d >= D) return;
  const int slot = slots ? slots[r] : r;
  float o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.0f;
  if (slot >= n_slots) {
    surfk::report_error(err, surfk::kErrSlotIndex);
  } else if (slot >= 0) {
    T* st = pool + static_cast<int64_t>(slot) * (W - 1) * D + d;
    float h[W][V];
    load_vec<T, V>(x + r * ldx + d, h[W - 1]);
    const bool cut = reset && reset[r];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      if (cut) {
#pragma unroll
        for (int i = 0; i < V; ++i) h[j][i] = 0.0f;
      } else {
        load_vec<T, V>(st + static_cast<int64_t>(j) * D, h[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float acc = bias ? bias[d + i] : 0.0f;
#pragma unroll
      for (int k = 0; k < W; ++k) acc = fmaf(w[static_cast<int64_t>(d + i) * W + k], h[k][i], acc);
      o[i] = silu ? acc * sigmoid(acc) : acc;
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_vec<T, V>(st + static_cast<int64_t>(j) * D, h[j + 1]);
  }
  store_vec<T, V>(y + r * ldy + d, o);
}

// ---- launches -------------------------------------------------------------------------------
// width -> template argument; several channels a thread where `vec`, else one
template <typename F> int by_width(int W, F f) {
  switch (W) {
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
  }
  return static_cast<int>(cudaErrorInvalidValue);
}

template <typename T, int W, int V> int launch_conv(ConvArgs a, int rows, cudaStream_t s) {
  const int groups = a.D / V;
  int bx = 1;
  while (bx < 32 && bx < groups) bx *= 2;
  const dim3 grid(static_cast<unsigned>(surfk::ceil_div(groups, bx)), static_cast<unsigned>(rows));
  constexpr size_t smem = kU * kThreads * sizeof(typename Raw<T, V>::Word);
  conv_kernel<T, W, V><<<grid, dim3(bx, kThreads / bx), smem, s>>>(a, a.B * a.chunks);
  SURF_RETURN_LAUNCH();
}

template <typename T, int W, int V>
int launch_grad(ConvArgs a, int rows, float* dw, float* dbias, cudaStream_t s) {
  const int groups = a.D / V;
  int bx = 1;
  while (bx < 32 && bx < groups) bx *= 2;
  const int by = kThreads / bx;
  const dim3 grid(static_cast<unsigned>(surfk::ceil_div(groups, bx)), static_cast<unsigned>(rows));
  constexpr size_t kRings = 2 * kU * kThreads * sizeof(typename Raw<T, V>::Word), kSums = kThreads * (W + 1) * V * sizeof(float);
  constexpr size_t smem = kRings > kSums ? kRings : kSums;
  if (const int rc = allow_smem<conv_grad_kernel<T, W, V>>(smem)) return rc;
  conv_grad_kernel<T, W, V><<<grid, dim3(bx, by), smem, s>>>(a, a.B * a.chunks);
  const int rc = static_cast<int>(cudaGetLastError());
  if (rc) return rc;
  conv_reduce_kernel<W><<<static_cast<unsigned>(surfk::ceil_div((W + 1) * static_cast<int64_t>(a.D), 32)), dim3(32, 8), 0, s>>>(
      a.part, rows, a.D, dw, dbias);
  SURF_RETURN_LAUNCH();
}

}  // namespace

// bytes: what a thread's channels take in a row; a multiple of it are D, every base and every stride
SURF_EXPORT int surf_seq_conv(const void* args, int dtype, int W, int bytes, int rows, void* stream) {
  const ConvArgs a = *static_cast<const ConvArgs*>(args);
  if (a.D <= 0 || rows <= 0 || rows > 65535) return static_cast<int>(cudaErrorInvalidValue);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_width(W, [&](auto w) {
    constexpr int kW = decltype(w)::value;
    if (dtype == kBf16) {
      if (bytes == 16) return launch_conv<bf16, kW, 8>(a, rows, s);
      return bytes == 4 ? launch_conv<bf16, kW, 2>(a, rows, s) : launch_conv<bf16, kW, 1>(a, rows, s);
    }
    return bytes == 16 ? launch_conv<float, kW, 4>(a, rows, s) : launch_conv<float, kW, 1>(a, rows, s);
  });
}

SURF_EXPORT int surf_seq_conv_grad(const void* args, int dtype, int W, int bytes, int rows, float* dw, float* dbias,
                                   void* stream) {
  const ConvArgs a = *static_cast<const ConvArgs*>(args);
  if (a.D <= 0 || rows <= 0 || rows > 65535) return static_cast<int>(cudaErrorInvalidValue);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_width(W, [&](auto w) {
    constexpr int kW = decltype(w)::value;
    if (dtype == kBf16) {
      if (bytes == 8) return launch_grad<bf16, kW, 4>(a, rows, dw, dbias, s);
      return bytes == 4 ? launch_grad<bf16, kW, 2>(a, rows, dw, dbias, s) : launch_grad<bf16, kW, 1>(a, rows, dw, dbias, s);
    }
    return bytes == 8 ? launch_grad<float, kW, 2>(a, rows, dw, dbias, s) : launch_grad<float, kW, 1>(a, rows, dw, dbias, s);
  });
}

SURF_EXPORT int surf_seq_conv_step(const void* x, int64_t ldx, const float* w, const float* bias, void* pool,
                                   const uint8_t* reset, const int* slots, int n_slots, void* y, int64_t ldy, int rows, int D,
                                   int W, int silu, int dtype, int vec, int* err, void* stream) {
  if (rows <= 0 || D <= 0) return 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_width(W, [&](auto wc) {
    constexpr int kW = decltype(wc)::value;
    auto go = [&](auto t, auto v) {
      using T = decltype(t);
      constexpr int V = decltype(v)::value;
      const int threads = D / V < 128 ? (D / V + 31) / 32 * 32 : 128;
      const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(surfk::ceil_div(D / V, threads)));
      conv_step_kernel<T, kW, V><<<grid, threads, 0, s>>>(static_cast<const T*>(x), ldx, w, bias, static_cast<T*>(pool), reset,
                                                          slots, n_slots, static_cast<T*>(y), ldy, D, silu, err);
      SURF_RETURN_LAUNCH();
    };
    if (dtype == kBf16) return vec ? go(bf16{}, std::integral_constant<int, 4>{}) : go(bf16{}, std::integral_constant<int, 1>{});
    return vec ? go(float{}, std::integral_constant<int, 4>{}) : go(float{}, std::integral_constant<int, 1>{});
  });
}
