// delta.cu — the gated delta rule over sequences and for single tokens (sm_100a). The formulas
// of a chunk are in delta.cuh.
#include "delta.cuh"

namespace {

using namespace delta;

// ---- sequences --------------------------------------------------------------------------
constexpr int kMain = 4;                               // warps that carry chunks out at most
constexpr int kPrep = 2;                               // warps that make chunks ready

template <typename T, int DK> struct Forward {
  // chunks ready, in the making or on their way
  static constexpr int kStages = (sizeof(T) == 4 && DK == 128 ? 2 : 3) * kPrep;
  using Keys = Tile<T, DK>;
  static_assert(kStages % kPrep == 0 && kStages >= 2 * kPrep, "a stage is one warp's, and its next one another");
  struct Stage {
    Chunk<T, Planes<T>::kShort> c;
    int t0, n, more;                                   // more: the tile's next episode follows in this stage
    unsigned marks;
    alignas(16) bf16 tk[Keys::kSize], tq[Keys::kSize];
  };
  struct Shared {
    Stage stage[kStages];
    alignas(16) Scratch scratch[kPrep];
  };
  static constexpr int kRow = 16 + 16 / static_cast<int>(sizeof(T));     // pitch of a warp's outputs
  // behind them: the values' rows of each stage, the outputs of each warp
  static __host__ __device__ constexpr int pitch_v(int warps) { return warps * 16 + 16 / static_cast<int>(sizeof(T)); }
  static __host__ __device__ constexpr size_t bytes(int warps) {
    return sizeof(Shared) + (static_cast<size_t>(kStages) * kTile * pitch_v(warps) + static_cast<size_t>(warps) * kTile * kRow) * sizeof(T);
  }
  // and, where the state goes out by bulk copies, each warp's rows of it and of W
  static __host__ __device__ constexpr size_t kept_bytes(int warps, int keys) { return static_cast<size_t>(warps) * 16 * (keys + kTile) * sizeof(float); }
};

// A block for up to 64 values of a sequence's value head. Two warps make the chunks ready in turn
// (tiles, decays, P, the inverse: nothing of it waits for the state), the others hold 16 values'
// rows of the state each, as accumulators from the first token to the last. They meet at
// numbered barriers: stage s is ready (1 + s), stage s is free (1 + kStages + s). With few blocks the chain
// from state to state bounds it (64 keys: 1.8 thousand cycles a chunk of one warp's products, each
// waiting for the one before, against 0.1 of memory), with many the same warps' waits and instructions
// (256x128x8x64x64: 0.38 a cycle and scheduler, tensor pipe 26%, 0.41 of the copy rate).
// kKeep: for the gradient. Calls that keep nothing are kernels of their own (1x8191x8x128x128 1054 -> 745 us,
// 2x4096x16x64x64 313 -> 248 us).
template <typename T, int DK, int kBlocks, bool kKeep>
__global__ void __launch_bounds__((kPrep + kMain) * 32, kBlocks) delta_forward(DeltaArgs a, int bulk) {
  constexpr int NT = Planes<T>::kToken, NI = Planes<T>::kInner, NS = Planes<T>::kShort, kSteps = DK / 16;
  using F = Forward<T, DK>;
  using Keys = Tile<T, DK>;
  constexpr int kStages = F::kStages;
  extern __shared__ __align__(16) char smem[];
  typename F::Shared& sh = *reinterpret_cast<typename F::Shared*>(smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32 - kPrep;
  const int pitch_v = F::pitch_v(warps), threads = (warps + 1) * 32;
  T* values = reinterpret_cast<T*>(smem + sizeof(typename F::Shared));
  const int bi = blockIdx.x / a.heads, h = blockIdx.x % a.heads, gr = h / (a.heads / a.groups);
  const int vb = blockIdx.y * warps * 16, mine = min(warps * 16, a.values - vb);
  const int length = a.lengths ? max(0, min(a.lengths[bi], a.length)) : a.length;

  if (warp >= warps) {
    const int w = warp - warps;
    const T* q = static_cast<const T*>(a.q) + bi * a.q_b + gr * a.q_g;
    const T* k = static_cast<const T*>(a.k) + bi * a.k_b + gr * a.k_g;
    const T* v = static_cast<const T*>(a.v) + bi * a.v_b + h * a.v_h + vb;
    const T* dt = static_cast<const T*>(a.dt) + bi * a.dt_b + h;
    const T* gb = static_cast<const T*>(a.b) + bi * a.b_b + h;
    const float rate = rate_at(a.A, h), bias = a.bias ? a.bias[h] : 0.0f;
    const int tiles = (length + kTile - 1) / kTile;
    Marks look{a.reset ? a.reset + static_cast<int64_t>(bi) * a.length : nullptr, length, 0u};
    // Tokens [t0, t0 + n) on their way to a stage; their decays are made meanwhile, from this lane's token.
    auto fetch = [&](typename F::Stage& st, T* tv, int t0, int n, unsigned marks, float raw_dt, float raw_b) {
      Keys::load(st.tk, k + t0 * a.k_t, a.k_t, n, a.keys, a.piece_k == 16);
      Keys::load(st.tq, q + t0 * a.q_t, a.q_t, n, a.keys, a.piece_k == 16);
      load_rows(tv, pitch_v, kTile, warps * 16, v + t0 * a.v_t, a.v_t, n, mine, a.piece_v == 16);
      cp_async_commit();
      Gate e{};
      if (lane < n) e = gate_of(raw_dt, raw_b, bias, rate);
      decays(st.c, e.g, e.beta, marks);
      if (lane == 0) {
        st.t0 = t0;
        st.n = n;
        st.marks = marks;
        st.more = 0;
      }
      return __any_sync(0xffffffffu, fmaf(e.g, 0.0f, e.beta * 0.0f) != 0.0f);
    };
    // resets and gates a tile of this warp's ahead of the rest
    T raw_dt = from_f<T>(0.0f), raw_b = raw_dt;
    auto ahead = [&](int i) {
      look.look(i * kTile);
      if (lane < kTile && i * kTile + lane < length) {
        raw_dt = dt[(i * kTile + lane) * a.dt_t];
        raw_b = gb[(i * kTile + lane) * a.b_t];
      }
    };
    bool bad_here = false, bad_next = false;
    unsigned marks_here = 0, marks_next = 0;
    auto begin = [&](int i) {
      const int at = i % kStages;
      if (i >= kStages) bar_sync(1 + kStages + at, threads);
      marks_next = look.get();
      const float x = to_f(raw_dt), y = to_f(raw_b);
      ahead(i + kPrep);
      bad_next = fetch(sh.stage[at], values + at * kTile * pitch_v, i * kTile, min(kTile, length - i * kTile), marks_next, x, y);
    };
    ahead(w);
    if (w < tiles) begin(w);
    for (int i = w; i < tiles; i += kPrep) {
      const int at = i % kStages, t0 = i * kTile, n = min(kTile, length - t0);
      typename F::Stage& st = sh.stage[at];
      T* tv = values + at * kTile * pitch_v;
      marks_here = marks_next;
      bad_here = bad_next;
      if (i + kPrep < tiles) begin(i + kPrep);
      else cp_async_commit();
      cp_async_wait<1>();
      __syncwarp();
      auto ready = [&](unsigned marks) {
        prepare<T, DK, false>(st.c, sh.scratch[w], nullptr, st.tk, st.tq, marks, a.scale, a.unit);
        bar_arrive(1 + at, threads);
      };
      const bool split = (marks_here & ~1u) && (bad_here || not_finite(st.tk, Keys::kPitch, DK, n) || not_finite(st.tq, Keys::kPitch, DK, n) ||
                                                not_finite(tv, pitch_v, warps * 16, n));
      if (!split) {
        ready(marks_here);
        continue;
      }
      for (unsigned left = marks_here | 1u; left;) {
        const int from = __ffs(left) - 1;
        left &= left - 1;
        const unsigned mark = (marks_here >> from) & 1u;
        if (from > 0) bar_sync(1 + kStages + at, threads);
        const int to = left ? __ffs(left) - 1 : n;
        const bool on = from + lane < to;
        fetch(st, tv, t0 + from, to - from, mark, on ? to_f(dt[(t0 + from + lane) * a.dt_t]) : 0.0f,
              on ? to_f(gb[(t0 + from + lane) * a.b_t]) : 0.0f);
        if (lane == 0) st.more = left != 0;
        cp_async_wait<0>();
        __syncwarp();
        ready(mark);
      }
    }
    return;
  }

  const int row = lane >> 2, col = (lane & 3) * 2, vl = warp * 16, v0 = vb + vl;
  T* out = static_cast<T*>(a.out) + bi * a.o_b + h * a.o_h;
  T* out_row = out + lane / (16 / kVec16<T>) * a.o_t + v0 + lane % (16 / kVec16<T>) * kVec16<T>;       // this lane's first piece
  T* so = values + kStages * kTile * pitch_v + warp * kTile * F::kRow;
  const int64_t head_size = static_cast<int64_t>(a.values) * a.keys;
  const int64_t head_at = (static_cast<int64_t>(bi) * a.heads + h) * head_size;
  const bool pairs = (a.keys & 1) == 0, even = (reinterpret_cast<uintptr_t>(a.state) & 7) == 0;

  // s[n]: rows v0 + row, + 8; keys 8 n + col, + 1
  float s[DK / 8][4];
  auto each = [&](auto f) {
#pragma unroll
    for (int n = 0; n < DK / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) f(s[n][2 * e], s[n][2 * e + 1], v0 + row + 8 * e, 8 * n + col);
  };
  auto store = [&](float* to, int pitch) {
    each([&](float x, float y, int r, int kc) {
      if (r >= a.values || kc >= a.keys) return;
      float* p = to + r * pitch + kc;
      if (pairs) {
        *reinterpret_cast<float2*>(p) = make_float2(x, y);
      } else {
        p[0] = x;
        if (kc + 1 < a.keys) p[1] = y;
      }
    });
  };
  each([&](float& x, float& y, int r, int kc) {
    const bool on = a.state && r < a.values && kc < a.keys;
    const float* p = a.state + head_at + r * a.keys + kc;
    if (pairs && even) {
      const float2 v = on ? *reinterpret_cast<const float2*>(p) : make_float2(0.0f, 0.0f);
      x = v.x;
      y = v.y;
    } else {
      x = on ? p[0] : 0.0f;
      y = on && kc + 1 < a.keys ? p[1] : 0.0f;
    }
  });

  const int tiles = (a.length + kTile - 1) / kTile, pitch_s = a.keys + kTile;
  float* kept = reinterpret_cast<float*>(smem + F::bytes(warps)) + warp * 16 * pitch_s;
  for (int i = 0, more = 0; i < (length + kTile - 1) / kTile; i += more ? 0 : 1) {
    const int at = i % kStages;
    typename F::Stage& st = sh.stage[at];
    bar_sync(1 + at, threads);
    const int t0 = st.t0, n = st.n;
    const unsigned marks = st.marks;
    more = st.more;
    const Chunk<T, NS>& c = st.c;
    // The state before the tile and W, for the gradient: rows of both side by side, as one bulk copy from
    // shared memory where that is allowed (stored lane by lane they held the chain up: 2x4096x16x64x64
    // 449 us). A warp behind the last value (a head's values need not divide among its blocks' warps) has none: its
    // copy's size would be 0 or below.
    float* saved = kKeep && v0 < a.values
                       ? a.saved + ((static_cast<int64_t>(bi) * tiles + t0 / kTile) * a.heads + h) * a.values * pitch_s : nullptr;
    const bool copied = saved && bulk && t0 % kTile == 0 && !more;
    if (copied) {
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      __syncwarp();
      each([&](float x, float y, int r, int kc) {
        if (kc < a.keys) *reinterpret_cast<float2*>(kept + (r - v0) * pitch_s + kc) = make_float2(x, y);
      });
    } else if (saved && t0 % kTile == 0) {
      store(saved, pitch_s);
    }
    if (marks & 1u) each([&](float& x, float& y, int, int) { x = y = 0.0f; });
    const T* tv = values + at * kTile * pitch_v;

    // per-token numbers of this lane's columns
    auto pair = [&](const float (&x)[kTile], int t) { return *reinterpret_cast<const float2*>(&x[8 * t + col]); };
    // whether the state before the chunk reaches a token
    auto seen = [&](int tok) { return !(marks & ((2u << tok) - 1u)); };
    // K S^T and Q S^T, transposed: rows values, columns tokens
    float sk[2][4] = {}, sq[2][4] = {}, w[2][4] = {};
    const uint32_t ka = smem_of(st.tk) + at_rows(lane, Keys::kPitch), qa = smem_of(st.tq) + at_rows(lane, Keys::kPitch);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      Frag<NI> f;
      f.from(s[2 * i], s[2 * i + 1]);
      uint32_t bk[NT][4], bq[NT][4];
      load_planes<NT, false>(bk, ka + i * 32, Keys::kPlane * 2);
      load_planes<NT, false>(bq, qa + i * 32, Keys::kPlane * 2);
      mma_planes2<NI, NS>(sk[0], sk[1], sq[0], sq[1], f.r, bk, bq);
    }
    if (marks)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!seen(8 * t + col + (e & 1))) sk[t][e] = sq[t][e] = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float2 hk = pair(c.head_k, t), hq = pair(c.head_q, t);
      const T* from = tv + (8 * t + col) * pitch_v + vl + row;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sk[t][e] = fmaf(-(e & 1 ? hk.y : hk.x), sk[t][e], to_f(from[(e & 1) * pitch_v + (e >> 1) * 8]));
        sq[t][e] *= e & 1 ? hq.y : hq.x;
      }
    }
    // W and P U. A state that is not finite reaches the first episode's tokens alone: with others in
    // the chunk, theirs are sums without them.
    bool apart = false;
    if (marks & ~1u) {
      float bad = 0.0f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) bad = fmaf(sk[t][e], 0.0f, bad);
      apart = __any_sync(0xffffffffu, bad != 0.0f);
    }
#pragma unroll 1
    for (int part = 0; part < (apart ? 2 : 1); ++part) {
      auto ours = [&](int tok) { return seen(tok) == (part != 0); };
      float r[2][4], x[2][4] = {}, y[2][4] = {};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) r[t][e] = apart && !ours(8 * t + col + (e & 1)) ? 0.0f : sk[t][e];
      Frag<NI> f;
      f.from(r[0], r[1]);
      uint32_t b[NI][4];
      load_planes<NI, false>(b, smem_of(c.inv) + at_rows(lane, kSide), kTile * kSide * 2);
      mma_planes<NI, NI>(x[0], x[1], f.r, b);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float2 beta = pair(c.beta, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[t][e] = x[t][e] * (e & 1 ? beta.y : beta.x);
      }
      Frag<NS> g;
      g.from(r[0], r[1]);
      uint32_t p[NS][4];
      load_planes<NS, false>(p, smem_of(c.p) + at_rows(lane, kSide), kTile * kSide * 2);
      mma_planes<NS, NS>(y[0], y[1], g.r, p);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!apart || ours(8 * t + col + (e & 1))) {
            w[t][e] = x[t][e];
            sq[t][e] += y[t][e];
          }
    }
    if (copied) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float2*>(kept + (row + 8 * e) * pitch_s + a.keys + 8 * t + col) = make_float2(w[t][2 * e], w[t][2 * e + 1]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(saved + static_cast<int64_t>(v0) * pitch_s),
                     "r"(smem_of(kept)), "r"(min(16, a.values - v0) * pitch_s * 4) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    } else if (saved) {
      float* p = saved + a.keys + t0 % kTile;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = t * 8 + col + (e & 1), r = v0 + row + (e >> 1) * 8;
          if (tok < n && r < a.values) p[r * pitch_s + tok] = w[t][e];
        }
    }
    // the state
    if (marks) {                                       // of it the tokens behind the last reset alone are left
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (marks >> (8 * t + col + (e & 1) + 1)) w[t][e] = 0.0f;
      each([&](float& x, float& y, int, int) { x = y = 0.0f; });
    } else {
      const float end = c.head[kTile - 1];
      each([&](float& x, float& y, int, int) {
        x *= end;
        y *= end;
      });
    }
    {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float2 tail = pair(c.tail_k, t), beta = pair(c.beta, t);
        const float fx = tail.x * beta.x, fy = tail.y * beta.y;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[t][e] *= e & 1 ? fy : fx;
      }
      Frag<NI> f;
      f.from(w[0], w[1]);
      const uint32_t kt = smem_of(st.tk) + at_cols(lane, Keys::kPitch);
      // two steps at a time, so that four sums take turns
#pragma unroll
      for (int i = 0; i < kSteps; i += 2) {
        uint32_t b[NT][4], d[NT][4];
        load_planes<NT, true>(b, kt + i * 32, Keys::kPlane * 2);
        load_planes<NT, true>(d, kt + i * 32 + 32, Keys::kPlane * 2);
        mma_planes2<NI, NI>(s[2 * i], s[2 * i + 1], s[2 * i + 2], s[2 * i + 3], f.r, b, d);
      }
    }
    bar_arrive(1 + kStages + at, threads);
    // the outputs, by tokens
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) so[(t * 8 + col + (e & 1)) * F::kRow + row + (e >> 1) * 8] = from_f<T>(sq[t][e]);
    __syncwarp();
    T* to = out_row + t0 * a.o_t;
    if (a.piece_v == 16) {
      constexpr int V = kVec16<T>, kPer = 16 / V, kRows = 32 / kPer;
#pragma unroll
      for (int r = 0; r < kTile; r += kRows)
        if (r + lane / kPer < n && lane % kPer * V < a.values - v0)
          *reinterpret_cast<uint4*>(to + r * a.o_t) = *reinterpret_cast<const uint4*>(so + (r + lane / kPer) * F::kRow + lane % kPer * V);
    } else {
      for (int j = lane; j < n * 16; j += 32) {
        const int r = j / 16, cc = j % 16;
        if (v0 + cc < a.values) out[(t0 + r) * a.o_t + v0 + cc] = so[r * F::kRow + cc];
      }
    }
    __syncwarp();
  }
  store(a.final_ + head_at, a.keys);
  if (kKeep && bulk && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  // tokens that are not there give zeros
  for (int t = length + warp; t < a.length; t += warps)
    for (int j = lane; j < mine; j += 32) out[t * a.o_t + vb + j] = from_f<T>(0.0f);
}

template <typename T, int DK> int forward(const DeltaArgs& a, cudaStream_t s) {
  using F = Forward<T, DK>;
  constexpr int kBlocks = sizeof(T) == 4 && DK == 128 ? 1 : 2;
  // values of a block: as many as it takes, or fewer where that leaves SMs without one (2x4096x16x64x64,
  // states kept: 361 us; with 64 a block 385)
  const int all = (a.values + 15) / 16;
  int warps = all < kMain ? all : kMain;
  while (warps > 1 && static_cast<int64_t>(a.batch) * a.heads * ((all + warps - 1) / warps) < 148) warps = (warps + 1) / 2;
  const int64_t blocks = static_cast<int64_t>(a.batch) * a.heads * ((all + warps - 1) / warps);
  // bulk copies of what is kept want rows of whole 16 bytes, and no shared memory that would cost many
  // blocks their neighbour on the SM (lane by lane 2x4096x16x64x64 takes 428 us, 361 so; 256x128x8x64x64 167, 158)
  const size_t kept = F::kept_bytes(warps, a.keys);
  const bool bulk = a.saved && a.keys % 4 == 0 && F::bytes(warps) + kept <= (blocks > 148 && kBlocks > 1 ? 113 : 227) * 1024;
  constexpr size_t kMost = F::bytes(kMain) + F::kept_bytes(kMain, DK);
  auto go = [&](auto keep) {
    constexpr auto kernel = delta_forward<T, DK, kBlocks, decltype(keep)::value>;
    if (const int e = allow_smem<kernel>(kMost < 227 * 1024 ? kMost : 227 * 1024)) return e;
    kernel<<<dim3(a.batch * a.heads, (all + warps - 1) / warps), (warps + kPrep) * 32, F::bytes(warps) + (bulk ? kept : 0), s>>>(a, bulk);
    return static_cast<int>(cudaGetLastError());
  };
  return a.saved ? go(std::true_type()) : go(std::false_type());
}
template <typename T> int forward_by(const DeltaArgs& a, cudaStream_t s) {
  if (a.keys <= 32) return forward<T, 32>(a, s);
  if (a.keys <= 64) return forward<T, 64>(a, s);
  return forward<T, 128>(a, s);
}

// ---- single tokens ------------------------------------------------------------------------
struct StepArgs {
  const void *q, *k, *v, *dt, *b;
  const float *A, *bias;
  float* state;
  const uint8_t* reset;
  const int* slots;
  void* out;
  int* err;
  int64_t q_r, q_g, k_r, k_g, v_r, v_h, dt_r, b_r, o_r, o_h;
  float scale;
  int rows, groups, heads, keys, values, unit, pools;
};
static_assert(sizeof(StepArgs) == 12 * 8 + 10 * 8 + 8 * 4, "as the caller packs it");

// A warp for `per` values of a head of a row (blockIdx.y): its lanes hold the key and the query, LK
// lanes a value's row of the state. S k and S q come from one look at the state:
//   u = beta (v - e^g S k),  S <- e^g S + u k^T,  o = scale (e^g S q + u k.q).
// Bound by the state's bytes: 2048x8x64x64 97 us, 0.86 of the copy rate, with four rows a lane on their way
// (one: 119 us).
template <typename T, int LK> __global__ void __launch_bounds__(256) delta_step(StepArgs a, int per) {
  constexpr int kRows = 32 / LK;                       // values that a warp takes at once
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5);
  if (item >= static_cast<int64_t>(a.rows) * a.heads) return;
  const int r = static_cast<int>(item / a.heads), h = static_cast<int>(item % a.heads), gr = h / (a.heads / a.groups);
  T* out = static_cast<T*>(a.out) + r * a.o_r + h * a.o_h;
  const int first = blockIdx.y * per, last = min(first + per, a.values);
  const int slot = a.slots ? a.slots[r] : r;
  if (slot < 0 || slot >= a.pools) {
    if (slot >= a.pools && h == 0 && first == 0 && lane == 0) surfk::report_error(a.err, surfk::kErrSlotIndex);
    for (int i = first + lane; i < last; i += 32) out[i] = from_f<T>(0.0f);
    return;
  }
  const int l = lane % LK, k0 = l * 4;
  float k[4], q[4], kk = 0.0f, qq = 0.0f, kq = 0.0f;
  const T* pk = static_cast<const T*>(a.k) + r * a.k_r + gr * a.k_g;
  const T* pq = static_cast<const T*>(a.q) + r * a.q_r + gr * a.q_g;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool on = k0 + j < a.keys;
    k[j] = on ? to_f(pk[k0 + j]) : 0.0f;
    q[j] = on ? to_f(pq[k0 + j]) : 0.0f;
    kk = fmaf(k[j], k[j], kk);
    qq = fmaf(q[j], q[j], qq);
  }
#pragma unroll
  for (int o = LK / 2; o; o >>= 1) {
    kk += __shfl_xor_sync(0xffffffffu, kk, o);
    qq += __shfl_xor_sync(0xffffffffu, qq, o);
  }
  if (a.unit) {
    const float rk = rsqrtf(kk + kNormEps), rq = rsqrtf(qq + kNormEps);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      k[j] *= rk;
      q[j] *= rq;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) kq = fmaf(k[j], q[j], kq);
#pragma unroll
  for (int o = LK / 2; o; o >>= 1) kq += __shfl_xor_sync(0xffffffffu, kq, o);
  const float pre = to_f(static_cast<const T*>(a.dt)[r * a.dt_r + h]) + (a.bias ? a.bias[h] : 0.0f);
  const bool fresh = a.reset && a.reset[r];
  const float decay = exp2_hw(fmaf(rate_at(a.A, h) * softplus(pre), kLog2e, kExp2Shift));
  const float beta = sigmoid(to_f(static_cast<const T*>(a.b)[r * a.b_r + h]));
  const T* pv = static_cast<const T*>(a.v) + r * a.v_r + h * a.v_h;
  float* state = a.state + (static_cast<int64_t>(slot) * a.heads + h) * a.values * a.keys;
  const bool whole = a.keys % 4 == 0;
  // several rows of the state are on their way before the first is used
  constexpr int kAhead = 4;
  for (int v0 = first + lane / LK; v0 < last + lane / LK; v0 += kAhead * kRows) {
    float s[kAhead][4];
    float v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int vr = v0 + i * kRows;
      const float* p = state + vr * a.keys + k0;
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
      v[i] = 0.0f;
      if (vr >= last) continue;
      v[i] = to_f(pv[vr]);
      if (fresh) continue;
      if (whole) {
        if (k0 < a.keys) *reinterpret_cast<float4*>(s[i]) = *reinterpret_cast<const float4*>(p);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k0 + j < a.keys) s[i][j] = p[j];
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int vr = v0 + i * kRows;
      float* p = state + vr * a.keys + k0;
      float sk = 0.0f, sq = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] *= decay;
        sk = fmaf(s[i][j], k[j], sk);
        sq = fmaf(s[i][j], q[j], sq);
      }
#pragma unroll
      for (int o = LK / 2; o; o >>= 1) {
        sk += __shfl_xor_sync(0xffffffffu, sk, o);
        sq += __shfl_xor_sync(0xffffffffu, sq, o);
      }
      if (vr >= last) continue;
      const float u = beta * (v[i] - sk);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = fmaf(u, k[j], s[i][j]);
      if (whole) {
        if (k0 < a.keys) *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(s[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k0 + j < a.keys) p[j] = s[i][j];
      }
      if (l == 0) out[vr] = from_f<T>(a.scale * fmaf(u, kq, sq));
    }
  }
}

template <typename T> int step(const StepArgs& a, cudaStream_t s) {
  const int64_t heads = static_cast<int64_t>(a.rows) * a.heads;
  auto go = [&](auto lanes) {
    constexpr int LK = decltype(lanes)::value;
    // a head's values in as many warps as give every SM 32, of at least the rows that are on their way
    // at once: 64 rows of 8 heads of 64 x 64 take 11.9 us in one warp a head and 5.5 in four
    const int least = 4 * (32 / LK), most = (a.values + least - 1) / least;
    int parts = static_cast<int>(heads >= 148 * 32 ? 1 : (148 * 32 + heads - 1) / heads);
    parts = parts < most ? parts : most;
    const int per = ((a.values + parts - 1) / parts + least - 1) / least * least;
    delta_step<T, LK><<<dim3(static_cast<unsigned>((heads + 7) / 8), (a.values + per - 1) / per), 256, 0, s>>>(a, per);
    return static_cast<int>(cudaGetLastError());
  };
  if (a.keys <= 16) return go(std::integral_constant<int, 4>());
  if (a.keys <= 32) return go(std::integral_constant<int, 8>());
  if (a.keys <= 64) return go(std::integral_constant<int, 16>());
  return go(std::integral_constant<int, 32>());
}

}  // namespace

SURF_EXPORT int surf_delta(const void* args, int dtype, void* stream) {
  const DeltaArgs& a = *static_cast<const DeltaArgs*>(args);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == kBf16 ? forward_by<bf16>(a, s) : forward_by<float>(a, s);
}

SURF_EXPORT int surf_delta_step(const void* args, int dtype, void* stream) {
  const StepArgs& a = *static_cast<const StepArgs*>(args);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == kBf16 ? step<bf16>(a, s) : step<float>(a, s);
}
