// Log probabilities of given tokens with entropy and the k most likely
// alternatives, and their gradient.
//
// A row holds the logits x_v of one prediction.  With c = scale, m = max x,
//   S = sum e^{c(x_v - m)},  T = sum c(x_v - m) e^{c(x_v - m)}
// everything the forward call returns follows from (m, S, T):
//   lse = c m + ln S,  logprob = c(x_t - m) - ln S,  entropy = ln S - T / S.
// The gradient is one expression a logit (see k_logprob_grad).
#include <cooperative_groups.h>

#include "lm_rows.cuh"

namespace cg = cooperative_groups;

namespace acd {

__device__ __forceinline__ float lp_log(float x) { return logf(x); }
__device__ __forceinline__ double lp_log(double x) { return log(x); }

struct LogprobArgs {
  Rows x;
  RowShape s;
  double scale;
  const void *tokens;
  void *logprob, *entropy, *lse;  // accumulator type, one a row
  void *top_index, *top_logprob;  // [L, k, O]
  int k;
  bool wide_token, wide_index, one_based;
};

constexpr int kMaxTop = 32;

// ---------------------------------------------------------------------------
// sums of a part of a row: m, S and T with respect to m
// ---------------------------------------------------------------------------
// float32 works with powers of two, z = c log2(e) (x - m), which is what the
// special function unit evaluates (ex2.approx: 2 ulp); T is then in bits.
template <typename A>
struct LpMath;
template <>
struct LpMath<float> {
  static constexpr float kUnit = 0.693147180559945309f;  // ln 2: T in bits -> nats
  static constexpr float kFloor = -200.0f;                // 2^-200 = 0 in float32
  static __device__ __forceinline__ float factor(double scale) { return (float)(scale * 1.4426950408889634074); }
  static __device__ __forceinline__ float ex(float z) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(z));
    return r;
  }
  // max that keeps a NaN of z
  static __device__ __forceinline__ float floor_z(float z) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(kFloor));
    return r;
  }
  static __device__ __forceinline__ float lowest() { return -FLT_MAX; }
  static __device__ __forceinline__ float max2(float a, float b) { return fmaxf(a, b); }
};
template <>
struct LpMath<double> {
  static constexpr double kUnit = 1.0;
  static __device__ __forceinline__ double factor(double scale) { return scale; }
  static __device__ __forceinline__ double ex(double z) { return exp(z); }
  static __device__ __forceinline__ double floor_z(double z) { return z < -1000.0 ? -1000.0 : z; }  // e^-1000 = 0
  static __device__ __forceinline__ double lowest() { return -DBL_MAX; }
  static __device__ __forceinline__ double max2(double a, double b) { return fmax(a, b); }
};

// m starts at the lowest finite value, so that -Inf - m is -Inf and never NaN:
// a part of -Inf only keeps S = 0.  floor_z keeps T free of 0 * Inf.  A NaN
// logit, and +Inf (Inf - Inf), make S NaN; the maximum passes over NaN.
template <typename A>
struct Part {
  A m, s, t;
  __device__ __forceinline__ void init() {
    m = LpMath<A>::lowest();
    s = t = A(0);
  }
  __device__ __forceinline__ void rescale(A mn, A c) {
    const A z = LpMath<A>::floor_z((m - mn) * c);
    const A f = LpMath<A>::ex(z);
    t = f * fma_a(s, z, t);
    s *= f;
    m = mn;
  }
  // N logits whose maximum is bm: one rescaling for all of them.
  template <int N>
  __device__ __forceinline__ void add(const A (&x)[N], A bm, A c) {
    rescale(LpMath<A>::max2(m, bm), c);
    A ls = 0, lt = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const A z = LpMath<A>::floor_z((x[j] - m) * c);
      const A e = LpMath<A>::ex(z);
      ls += e;
      lt = fma_a(e, z, lt);
    }
    s += ls;
    t += lt;
  }
  __device__ __forceinline__ void merge(Part o, A c) {
    const A mn = LpMath<A>::max2(m, o.m);
    rescale(mn, c);
    o.rescale(mn, c);
    s += o.s;
    t += o.t;
  }
  // Over the warp, in every lane; the order is fixed.
  __device__ __forceinline__ void warp_merge(A c) {
#pragma unroll
    for (int q = 16; q; q >>= 1) {
      Part o;
      o.m = __shfl_xor_sync(~0u, m, q);
      o.s = __shfl_xor_sync(~0u, s, q);
      o.t = __shfl_xor_sync(~0u, t, q);
      merge(o, c);
    }
  }
};

// ---------------------------------------------------------------------------
// the best logits of a part of a row: a warp's sorted list, one entry a lane
// ---------------------------------------------------------------------------
constexpr int kNone = INT_MAX;  // the index of an empty entry (value -Inf)

template <typename A>
__device__ __forceinline__ bool better(A v, int i, A w, int j) {
  return v > w || (v == w && i < j);
}

template <typename A>
struct TopList {
  A v;   // this lane's entry, falling over the lanes
  int i;
  A kv;  // entry k - 1, in every lane
  int ki;
  __device__ __forceinline__ void init() {
    v = kv = A(-INFINITY);
    i = ki = kNone;
  }
  __device__ __forceinline__ void refresh(int k) {
    kv = __shfl_sync(~0u, v, k - 1);
    ki = __shfl_sync(~0u, i, k - 1);
  }
  // One logit, the same in every lane, better than entry k - 1.
  __device__ __forceinline__ void insert(A x, int xi, int k) {
    const int lane = threadIdx.x & 31;
    const int pos = __popc(__ballot_sync(~0u, better(v, i, x, xi)));
    const A pv = __shfl_up_sync(~0u, v, 1);
    const int pi = __shfl_up_sync(~0u, i, 1);
    if (lane > pos) {
      v = pv;
      i = pi;
    } else if (lane == pos) {
      v = x;
      i = xi;
    }
    refresh(k);
  }
  // Every lane offers one logit (index `none` to offer nothing).
  __device__ __forceinline__ void offer(A x, int xi, bool valid, A floor, int k) {
    unsigned mask = __ballot_sync(~0u, valid && x >= floor && better(x, xi, kv, ki));
    while (mask) {
      const int src = __ffs(mask) - 1;
      insert(__shfl_sync(~0u, x, src), __shfl_sync(~0u, xi, src), k);
      mask &= mask - 1;
      mask &= __ballot_sync(~0u, better(x, xi, kv, ki));
    }
  }
  // Another sorted list, lane q holding its entry 31 - q: the better of each
  // pair is a bitonic sequence of the 32 best; five exchanges sort it.
  __device__ __forceinline__ void merge_reversed(A ov, int oi) {
    if (better(ov, oi, v, i)) {
      v = ov;
      i = oi;
    }
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int q = 16; q; q >>= 1) {
      const A pv = __shfl_xor_sync(~0u, v, q);
      const int pi = __shfl_xor_sync(~0u, i, q);
      if (((lane & q) == 0) == better(pv, pi, v, i)) {
        v = pv;
        i = pi;
      }
    }
  }
};

// The k-th largest of the lanes' values (bitonic sort, falling).
template <typename A>
__device__ __forceinline__ A kth_of_lanes(A x, int k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int q = size >> 1; q; q >>= 1) {
      const A o = __shfl_xor_sync(~0u, x, q);
      const bool up = ((lane & size) == 0) == ((lane & q) == 0);
      x = up ? (o > x ? o : x) : (o < x ? o : x);
    }
  return __shfl_sync(~0u, x, k - 1);
}

// What one warp knows of the part of a row that it has read.  A batch is N =
// U * V logits a lane: lane l holds elements base + u*32*V + l*V + j.  Batches
// come with rising base, so a later logit that equals entry k - 1 never wins.
// `floor`: some k logits of the row are at least this large.
template <typename A, int U, int V, bool TOP>
struct RowState {
  Part<A> p;
  TopList<A> top;
  __device__ __forceinline__ void init() {
    p.init();
    if (TOP) top.init();
  }
  __device__ __forceinline__ void batch(const A (&x)[U * V], int base, int D, A c, int k, A floor) {
    A vm[U], bm;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      vm[u] = x[u * V];
#pragma unroll
      for (int j = 1; j < V; ++j) vm[u] = LpMath<A>::max2(vm[u], x[u * V + j]);
      bm = u ? LpMath<A>::max2(bm, vm[u]) : LpMath<A>::max2(vm[0], A(-INFINITY));
    }
    p.add(x, bm, c);
    if (TOP) {
      const bool first = top.ki == kNone;
      if (!first && !__any_sync(~0u, bm > top.kv && bm >= floor)) return;
      // k lanes' maxima are at least as large as the k-th of them
      if (first) floor = LpMath<A>::max2(floor, kth_of_lanes(bm, k));
      const int lane = threadIdx.x & 31;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!__any_sync(~0u, vm[u] >= floor && vm[u] >= top.kv)) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int xi = base + (u * 32 + lane) * V + j;
          top.offer(x[u * V + j], xi, xi >= 0 && xi < D, floor, k);
        }
      }
    }
  }
};

// The row's results from what is known of all of it; called by a whole warp.
template <typename A, bool TOP>
__device__ __forceinline__ void finish_row(const LogprobArgs &a, int64_t r, const Part<A> &p, A v, int i, int64_t t,
                                           A xt) {
  const int lane = threadIdx.x & 31;
  const bool empty = p.s == A(0);  // every logit -Inf
  const A c = (A)a.scale;
  const A log_s = empty ? A(0) : lp_log(p.s);
  if (lane == 0) {
    if (a.lse) static_cast<A *>(a.lse)[r] = empty ? A(-INFINITY) : fma_a(c, p.m, log_s);
    if (a.entropy) static_cast<A *>(a.entropy)[r] = empty ? A(0) : log_s - LpMath<A>::kUnit * (p.t / p.s);
    if (a.logprob) {
      A lp = A(NAN);
      if (t == -1)
        lp = A(0);
      else if (t >= 0 && t < a.s.D)
        lp = empty ? A(-INFINITY) : c * (xt - p.m) - log_s;
      static_cast<A *>(a.logprob)[r] = lp;
    }
  }
  if (TOP && lane < a.k) {
    const int64_t o = r / a.s.L, l = r - o * a.s.L;
    const int64_t at = l + a.s.L * (lane + a.k * o);
    const bool none = i == kNone;
    store_index(a.top_index, a.wide_index, at,
                none ? (a.wide_index ? INT64_MIN : (int64_t)INT32_MIN) : (int64_t)i + (a.one_based ? 1 : 0));
    static_cast<A *>(a.top_logprob)[at] = none ? A(NAN) : c * (v - p.m) - log_s;
  }
}

// The token asked for (0-based; -1 none; others outside the row) and its logit.
template <typename T, typename A>
__device__ __forceinline__ void asked_token(const LogprobArgs &a, int64_t r, const T *x, int64_t &t, A &xt) {
  t = -1;
  xt = A(0);
  if (a.logprob) {
    t = load_index(a.tokens, a.wide_token, r) - (a.one_based ? 1 : 0);
    if (t >= 0 && t < a.s.D) xt = to_acc(x[t * a.x.sd]);
  }
}

// ---------------------------------------------------------------------------
// rows along the axis
// ---------------------------------------------------------------------------
// How many pieces of V logits a lane holds at once.
template <typename T, int V>
struct BatchU { static constexpr int value = V == 1 ? 8 : 4; };

// A warp reads batches `from`, `from + step`, ... of the row up to `to`.
template <typename T, int V, bool TOP, typename State>
__device__ __forceinline__ void read_batches(const T *x, int64_t sd, int D, int shift, int from, int step, int to,
                                             typename AccOf<T>::type c, int k, State &st,
                                             volatile typename AccOf<T>::type *floor) {
  using A = typename AccOf<T>::type;
  constexpr int U = BatchU<T, V>::value;
  const int lane = threadIdx.x & 31;
  for (int b = from; b < to; b += step) {
    const int base = b * (U * V * 32) - shift;
    A xs[U * V];
#pragma unroll
    for (int u = 0; u < U; ++u) load_piece<T, A, V>(x, sd, base + (u * 32 + lane) * V, D, A(-INFINITY), xs + u * V);
    st.batch(xs, base, D, c, k, TOP && floor ? *floor : A(-INFINITY));
    // any warp's entry k - 1 will do as floor: the value decides how much is
    // looked at, never the result
    if (TOP && floor && lane == 0 && st.top.ki != kNone && st.top.kv > *floor) *floor = st.top.kv;
  }
}

// One warp a row.
template <typename T, int V, bool TOP>
__global__ void __launch_bounds__(256) k_logprob_warp(LogprobArgs a) {
  using A = typename AccOf<T>::type;
  constexpr int U = BatchU<T, V>::value;
  const A c = LpMath<A>::factor(a.scale);
  const int D = (int)a.s.D;
  const int64_t rows = a.s.rows();
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    const T *x = row_ptr<T>(a.x, r, a.s.L);
    int64_t t;
    A xt;
    asked_token<T, A>(a, r, x, t, xt);
    const int shift = row_shift<T, V>(x);
    const int batches = (int)(((int64_t)shift + D + U * V * 32 - 1) / (U * V * 32));
    RowState<A, U, V, TOP> st;
    st.init();
    read_batches<T, V, TOP>(x, a.x.sd, D, shift, 0, 1, batches, c, a.k, st,
                            static_cast<volatile A *>(nullptr));
    st.p.warp_merge(c);
    finish_row<A, TOP>(a, r, st.p, st.top.v, st.top.i, t, xt);
  }
}

// A cluster of blocks a row: its batches go round the warps of all blocks; the
// warps' sums and lists are joined in each block, the blocks' in the first one
// through distributed shared memory, always in the same order.
template <typename T, int V, bool TOP, int NW>
__global__ void __launch_bounds__(NW * 32) k_logprob_cta(LogprobArgs a) {
  using A = typename AccOf<T>::type;
  constexpr int U = BatchU<T, V>::value;
  __shared__ Part<A> sh_p[NW];
  __shared__ A sh_v[NW][32];
  __shared__ int sh_i[NW][32];
  __shared__ A sh_floor;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const A c = LpMath<A>::factor(a.scale);
  const int D = (int)a.s.D;
  const int64_t r = blockIdx.x / C;
  const T *x = row_ptr<T>(a.x, r, a.s.L);
  int64_t t;
  A xt;
  asked_token<T, A>(a, r, x, t, xt);
  if (threadIdx.x == 0) sh_floor = A(-INFINITY);
  if (TOP) __syncthreads();
  const int shift = row_shift<T, V>(x);
  const int batches = (int)(((int64_t)shift + D + U * V * 32 - 1) / (U * V * 32));
  RowState<A, U, V, TOP> st;
  st.init();
  read_batches<T, V, TOP>(x, a.x.sd, D, shift, rank * NW + warp, C * NW, batches, c, a.k, st,
                          static_cast<volatile A *>(&sh_floor));
  st.p.warp_merge(c);
  if (lane == 0) sh_p[warp] = st.p;
  if (TOP) {
    sh_v[warp][lane] = st.top.v;
    sh_i[warp][lane] = st.top.i;
  }
  __syncthreads();
  // lists: halve the number of warps until one is left
  if (TOP) {
#pragma unroll
    for (int n = NW / 2; n; n >>= 1) {
      if (warp < n) {
        st.top.merge_reversed(sh_v[warp + n][31 - lane], sh_i[warp + n][31 - lane]);
        sh_v[warp][lane] = st.top.v;
        sh_i[warp][lane] = st.top.i;
      }
      __syncthreads();
    }
  }
  if (warp == 0) {
    st.p.init();
    if (lane < NW) st.p = sh_p[lane];
    st.p.warp_merge(c);
    if (lane == 0) sh_p[0] = st.p;
  }
  if (C > 1) {
    cluster.sync();
    if (rank == 0 && warp == 0) {
      st.p.init();
      if (lane < C) st.p = cluster.map_shared_rank(sh_p, lane)[0];
      st.p.warp_merge(c);
      if (TOP)
        for (int q = 1; q < C; ++q)
          st.top.merge_reversed(cluster.map_shared_rank(&sh_v[0][0], q)[31 - lane],
                                cluster.map_shared_rank(&sh_i[0][0], q)[31 - lane]);
    }
    cluster.sync();  // no block leaves while its shared memory is read
  }
  if (rank == 0 && warp == 0) finish_row<A, TOP>(a, r, st.p, st.top.v, st.top.i, t, xt);
}

// ---------------------------------------------------------------------------
// rows across the lanes
// ---------------------------------------------------------------------------
// Column-major logits [tokens, vocabulary]: a row's logits are `sd` apart,
// neighbouring rows lie side by side.  A block takes LT neighbouring rows
// (lanes), reads S steps of them along the lanes (full 128-byte lines), turns
// the tile round in shared memory and has each warp read its four rows along
// the steps, as the kernels above do.  A word holds PAIR steps of one lane.
template <typename T>
struct LaneTile {  // float32, float64
  static constexpr int LT = 32, NW = 8, PAIR = 1, W = sizeof(T) == 4 ? 128 : 64;
  using Word = T;
};
template <>
struct LaneTile<__half> {  // lane pairs are read as one word
  static constexpr int LT = 64, NW = 16, PAIR = 2, W = 128;
  using Word = uint32_t;
};

struct LaneArgs {
  LogprobArgs a;
  int64_t lblocks;  // blocks of LT lanes
  int chunk;        // steps a block of the cluster takes, a multiple of the tile's
  bool pairs;       // float16: lane pairs are 4-byte aligned in every step
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(LaneTile<T>::NW * 32, LaneTile<T>::NW == 16 ? 2 : 3) k_logprob_lanes(LaneArgs la) {
  using A = typename AccOf<T>::type;
  using Tile = LaneTile<T>;
  using Word = typename Tile::Word;
  constexpr int LT = Tile::LT, NW = Tile::NW, PAIR = Tile::PAIR, W = Tile::W, S = W * PAIR;
  constexpr int ITER = W / NW, R = LT / NW, U = W / 32;
  static_assert(R == 4, "four rows a warp");
  constexpr size_t kTile = sizeof(Word) * LT * (W + 1);
  constexpr size_t kJoin = (sizeof(Part<A>) + 32 * (sizeof(A) + sizeof(int))) * LT;
  __shared__ __align__(16) unsigned char raw[kTile > kJoin ? kTile : kJoin];
  Word(*tile)[W + 1] = reinterpret_cast<Word(*)[W + 1]>(raw);
  const LogprobArgs &a = la.a;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t group = blockIdx.x / C, o = group / la.lblocks, l0 = (group - o * la.lblocks) * LT;
  const int64_t L = a.s.L, sd = a.x.sd;
  const int D = (int)a.s.D;
  const T *x = static_cast<const T *>(a.x.p) + o * a.x.so + l0;
  const int left = L - l0 < LT ? (int)(L - l0) : LT;  // lanes of this block
  const A c = LpMath<A>::factor(a.scale);
  const int s0 = rank * la.chunk, s1 = D < s0 + la.chunk ? D : s0 + la.chunk;
  // row q of the tile is lane q (float16: even lanes, then odd ones)
  auto lane_of = [](int q) { return PAIR == 1 ? q : (q < 32 ? 2 * q : 2 * (q - 32) + 1); };
  // the tokens asked for: lane q of a warp holds its row q's
  int64_t tok = -1;
  A tok_x = A(0);
  if (lane < R && lane_of(warp * R + lane) < left)
    asked_token<T, A>(a, o * L + l0 + lane_of(warp * R + lane), x + lane_of(warp * R + lane), tok, tok_x);

  Word reg[ITER * PAIR];
  auto load = [&](int s) {
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int step = s + (i * NW + warp) * PAIR;
      if constexpr (PAIR == 1) {
        reg[i] = lane < left && step < s1 ? x[step * sd + lane] : (T)(-INFINITY);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t w = 0xFC00FC00u;  // -Inf, -Inf
          if (step + j < s1) {
            const T *p = x + (step + j) * sd + 2 * lane;
            if (la.pairs && 2 * lane + 1 < left)
              w = *reinterpret_cast<const uint32_t *>(p);
            else {
              const unsigned short *h = reinterpret_cast<const unsigned short *>(p);
              if (2 * lane < left) w = (w & 0xFFFF0000u) | h[0];
              if (2 * lane + 1 < left) w = (w & 0xFFFFu) | ((uint32_t)h[1] << 16);
            }
          }
          reg[2 * i + j] = w;
        }
      }
    }
  };

  RowState<A, U, PAIR, TOP> st[R];
#pragma unroll
  for (int q = 0; q < R; ++q) st[q].init();
  if (s0 < s1) load(s0);
  for (int s = s0; s < s1; s += S) {
    __syncthreads();  // the tile before has been read
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      if constexpr (PAIR == 1) {
        tile[lane][i * NW + warp] = reg[i];
      } else {
        tile[lane][i * NW + warp] = __byte_perm(reg[2 * i], reg[2 * i + 1], 0x5410);
        tile[32 + lane][i * NW + warp] = __byte_perm(reg[2 * i], reg[2 * i + 1], 0x7632);
      }
    }
    __syncthreads();
    if (s + S < s1) load(s + S);  // in flight while this tile is worked on
#pragma unroll
    for (int q = 0; q < R; ++q) {
      A xs[U * PAIR];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Word w = tile[warp * R + q][u * 32 + lane];
        if constexpr (PAIR == 1) {
          xs[u] = w;
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
          xs[2 * u] = f.x;
          xs[2 * u + 1] = f.y;
        }
      }
      st[q].batch(xs, s, D, c, a.k, A(-INFINITY));
    }
  }
#pragma unroll
  for (int q = 0; q < R; ++q) st[q].p.warp_merge(c);

  if (C == 1) {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int l = lane_of(warp * R + q);
      const int64_t t = __shfl_sync(~0u, tok, q);
      const A xt = __shfl_sync(~0u, tok_x, q);
      if (l < left) finish_row<A, TOP>(a, o * L + l0 + l, st[q].p, st[q].top.v, st[q].top.i, t, xt);
    }
    return;
  }
  // the blocks' sums and lists: row q of the tile is joined by block q / (LT / C)
  A *jv = reinterpret_cast<A *>(raw);                       // [LT][32]
  Part<A> *jp = reinterpret_cast<Part<A> *>(jv + LT * 32);  // [LT]
  int *ji = reinterpret_cast<int *>(jp + LT);               // [LT][32]
  __syncthreads();
#pragma unroll
  for (int q = 0; q < R; ++q) {
    const int row = warp * R + q;
    if (lane == 0) jp[row] = st[q].p;
    if (TOP) {
      jv[row * 32 + lane] = st[q].top.v;
      ji[row * 32 + lane] = st[q].top.i;
    }
  }
  cluster.sync();
  const int per = LT / C;
  for (int row = rank * per + warp; row < (rank + 1) * per; row += NW) {
    const int l = lane_of(row);
    if (l >= left) continue;
    RowState<A, U, PAIR, TOP> z;
    z.init();
    if (lane < C) z.p = cluster.map_shared_rank(jp, lane)[row];
    z.p.warp_merge(c);
    if (TOP)
      for (int q = 0; q < C; ++q)
        z.top.merge_reversed(cluster.map_shared_rank(jv, q)[row * 32 + 31 - lane],
                             cluster.map_shared_rank(ji, q)[row * 32 + 31 - lane]);
    int64_t t;
    A xt;
    asked_token<T, A>(a, o * L + l0 + l, x + l, t, xt);
    finish_row<A, TOP>(a, o * L + l0 + l, z.p, z.top.v, z.top.i, t, xt);
  }
  cluster.sync();  // no block leaves while its shared memory is read
}

struct LogprobGradArgs {
  Rows x, g;
  RowShape s;
  double scale;
  const void *tokens, *lse, *entropy, *d_logprob, *d_entropy, *d_lse;
  bool wide_token, one_based;
};

// A row's coefficients, scale included.  With d = c x_v - lse = log p_v:
//   grad_v = p_v (a0 - a1 d) + [v = t] gt,  a0 = c (g_lse - g - g_H H), a1 = c g_H.
// d is rounded once (fma) before the exponential, so its error is that of its
// own size and not of the logit's.
template <typename A>
struct GradRow {
  A lse, a0, a1, gt;
  int t;
};

template <typename A>
__device__ __forceinline__ GradRow<A> grad_row(const LogprobGradArgs &a, int64_t r) {
  GradRow<A> g;
  const A c = (A)a.scale;
  g.lse = static_cast<const A *>(a.lse)[r];
  g.t = -1;
  g.gt = A(0);
  if (a.d_logprob) {
    const int64_t t = load_index(a.tokens, a.wide_token, r) - (a.one_based ? 1 : 0);
    if (t >= 0 && t < a.s.D) {
      g.t = (int)t;
      g.gt = c * static_cast<const A *>(a.d_logprob)[r];
    }
  }
  g.a0 = (a.d_lse ? c * static_cast<const A *>(a.d_lse)[r] : A(0)) - g.gt;
  g.a1 = A(0);
  if (a.d_entropy) {
    g.a1 = c * static_cast<const A *>(a.d_entropy)[r];
    g.a0 = fma_a(-g.a1, static_cast<const A *>(a.entropy)[r], g.a0);
  }
  // a row without mass: p = 0 everywhere and no token term.  So is one masked
  // throughout by the type's lowest value: its lse has no digits left for ln S.
  if (g.lse <= (std::is_same<A, double>::value ? (A)(-DBL_MAX / 4) : (A)(-FLT_MAX / 4))) {
    g.lse = A(INFINITY);
    g.a0 = g.a1 = g.gt = A(0);
  }
  return g;
}

template <typename A>
__device__ __forceinline__ A grad_value(const GradRow<A> &g, A x, A c);
template <>
__device__ __forceinline__ float grad_value<float>(const GradRow<float> &g, float x, float c) {
  using M = LpMath<float>;
  const float d = M::floor_z(fmaf(c, x, -g.lse));  // p = 0 where d is below the floor: 0 log 0 = 0
  return M::ex(d * 1.44269504088896341f) * fmaf(-g.a1, d, g.a0);
}
template <>
__device__ __forceinline__ double grad_value<double>(const GradRow<double> &g, double x, double c) {
  const double d = LpMath<double>::floor_z(fma(c, x, -g.lse));
  return exp(d) * fma(-g.a1, d, g.a0);
}

// Rows along the axis: a warp takes U pieces a lane of one row, 16 bytes each
// (V logits; the row may start and end inside a piece), reads them all and
// then writes.  V = 1: any strides.
template <typename T, int V>
__global__ void __launch_bounds__(256) k_logprob_grad_rows(LogprobGradArgs a, uint32_t segs, uint32_t tasks) {
  using A = typename AccOf<T>::type;
  constexpr int U = BatchU<T, V>::value;
  const int lane = threadIdx.x & 31;
  const A c = (A)a.scale;
  const int D = (int)a.s.D;
  for (uint32_t task = blockIdx.x * 8 + (threadIdx.x >> 5); task < tasks; task += gridDim.x * 8) {
    const uint32_t r = task / segs, seg = task - r * segs;
    const T *x = row_ptr<T>(a.x, r, a.s.L);
    T *out = row_ptr<T>(a.g, r, a.s.L);
    const int base = (int)seg * (U * V * 32) - row_shift<T, V>(x);
    A xs[U * V];
#pragma unroll
    for (int u = 0; u < U; ++u) load_piece<T, A, V>(x, a.x.sd, base + (u * 32 + lane) * V, D, A(-INFINITY), xs + u * V);
    const GradRow<A> g = grad_row<A>(a, r);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int first = base + (u * 32 + lane) * V;
      A v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = grad_value<A>(g, xs[u * V + j], c);
      if (g.t >= first && g.t < first + V) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (first + j == g.t) v[j] += g.gt;
      }
      store_piece<T, A, V>(out, a.g.sd, first, D, v);
    }
  }
}

// Rows across the lanes: a thread keeps the coefficients of V neighbouring
// rows and walks along the steps, so that a warp reads and writes 32 * V
// neighbouring logits at a time.  A block is bx threads along the lanes by
// 256 / bx along the steps, and takes `chunk` steps.
template <typename T, int V>
__global__ void __launch_bounds__(256) k_logprob_grad_lanes(LogprobGradArgs a, int bx_log2, int64_t lblocks,
                                                            int64_t chunk) {
  using A = typename AccOf<T>::type;
  constexpr int UN = 4;
  const int bx = 1 << bx_log2, by = 256 >> bx_log2;
  const int64_t lb = blockIdx.x % lblocks, o = blockIdx.x / lblocks;
  const int64_t l = (lb * bx + (threadIdx.x & (bx - 1))) * V;
  if (l >= a.s.L) return;
  const A c = (A)a.scale;
  GradRow<A> g[V];
#pragma unroll
  for (int j = 0; j < V; ++j) g[j] = grad_row<A>(a, o * a.s.L + l + j);
  const T *x = static_cast<const T *>(a.x.p) + o * a.x.so + l;
  T *out = static_cast<T *>(a.g.p) + o * a.g.so + l;
  int64_t s = blockIdx.y * chunk;
  const int64_t s1 = s + chunk < a.s.D ? s + chunk : a.s.D;
  for (s += threadIdx.x >> bx_log2; s < s1; s += UN * by) {
    Vec<T, V> w[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (s + u * by < s1) w[u] = *reinterpret_cast<const Vec<T, V> *>(x + (s + u * by) * a.x.sd);
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (s + u * by >= s1) break;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        A v = grad_value<A>(g[j], to_acc(w[u].v[j]), c);
        if (g[j].t == (int)(s + u * by)) v += g[j].gt;
        w[u].v[j] = from_acc<T, A>(v);
      }
      *reinterpret_cast<Vec<T, V> *>(out + (s + u * by) * a.g.sd) = w[u];
    }
  }
}

static bool row_dtype(int32_t dt) { return dt == ACD_FLOAT32 || dt == ACD_FLOAT64 || dt == ACD_FLOAT16; }
static int32_t stat_dtype(int32_t dt) { return dt == ACD_FLOAT64 ? ACD_FLOAT64 : ACD_FLOAT32; }

static acd_status check_logits(const char *op, const acd_desc *logits, int32_t axis, double scale) {
  ACD_TRY(check_desc(logits, "logits"));
  if (!row_dtype(logits->dtype)) return fail(ACD_ERR_DTYPE, "%s: float32, float64 or float16 logits required", op);
  if (axis < 0 || axis >= logits->ndim) return fail(ACD_ERR_AXIS, "%s: axis %d out of range", op, axis);
  if (!(scale > 0.0) || !std::isfinite(scale)) return fail(ACD_ERR_INVALID, "%s: scale must be positive and finite", op);
  // positions are ints, with room for the last batch
  if (logits->shape[axis] > INT32_MAX - 65536) return fail(ACD_ERR_UNSUPPORTED, "%s: more than 2^31 - 65537 tokens", op);
  return ACD_OK;
}

static acd_status check_stat(const char *op, const char *name, const acd_desc *d, const acd_desc *logits, int axis) {
  if (!d) return ACD_OK;
  ACD_TRY(check_row_tensor(op, name, d, logits, axis));
  if (d->dtype != stat_dtype(logits->dtype))
    return fail(ACD_ERR_DTYPE, "%s: %s must be %s", op, name, logits->dtype == ACD_FLOAT64 ? "float64" : "float32");
  return ACD_OK;
}

static acd_status check_tokens(const char *op, const acd_desc *tokens, const acd_desc *logits, int axis) {
  ACD_TRY(check_row_tensor(op, "tokens", tokens, logits, axis));
  if (tokens->dtype != ACD_INT32 && tokens->dtype != ACD_INT64)
    return fail(ACD_ERR_DTYPE, "%s: tokens must be int32 or int64", op);
  return ACD_OK;
}

static void *ptr_or_null(const acd_desc *d) { return d ? desc_ptr(d) : nullptr; }

template <typename K, typename Args>
static acd_status launch_clusters(K kernel, const Args &a, int64_t blocks, int threads, int cluster, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ACD_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  return ACD_OK;
}

template <typename T, bool TOP>
static acd_status launch_lanes(acd_ctx *ctx, const LogprobArgs &a, cudaStream_t s) {
  using Tile = LaneTile<T>;
  constexpr int S = Tile::W * Tile::PAIR;
  LaneArgs la{};
  la.a = a;
  la.lblocks = (a.s.L + Tile::LT - 1) / Tile::LT;
  const int64_t groups = la.lblocks * a.s.O, tiles = (a.s.D + S - 1) / S;
  int C = 1;
  while (C < 8 && groups * C < ctx->sm_count && tiles >= C * 2) C *= 2;
  la.chunk = (int)((tiles + C - 1) / C * S);
  la.pairs = sizeof(T) == 2 && aligned_to<char>(a.x.p, 4) && a.x.sd % 2 == 0 && a.x.so % 2 == 0;
  if (groups * C > INT32_MAX) return fail(ACD_ERR_UNSUPPORTED, "acd_token_logprob: too many rows");
  return launch_clusters(k_logprob_lanes<T, TOP>, la, groups * C, Tile::NW * 32, C, s);
}

template <typename T, int V, bool TOP>
static acd_status launch_rows(acd_ctx *ctx, const LogprobArgs &a, cudaStream_t s) {
  const int64_t rows = a.s.rows(), batch = (int64_t)BatchU<T, V>::value * V * 32;
  const int64_t batches = (a.s.D + batch - 1) / batch;
  if (rows >= (int64_t)ctx->sm_count * 16 && batches <= 16) {
    const int grid = persistent_grid(ctx, k_logprob_warp<T, V, TOP>, 256, 0, (rows + 7) / 8);
    k_logprob_warp<T, V, TOP><<<grid, 256, 0, s>>>(a);
    return ACD_OK;
  }
  // blocks a row: as long as there are SMs without one and batches for their warps
  int C = 1;
  while (C < 8 && rows * C * 2 <= ctx->sm_count && batches > C * 8) C *= 2;
  if (rows * C > INT32_MAX) return fail(ACD_ERR_UNSUPPORTED, "acd_token_logprob: too many rows");
  return launch_clusters(k_logprob_cta<T, V, TOP, 8>, a, rows * C, 256, C, s);
}

template <typename T>
static acd_status launch_logprob(acd_ctx *ctx, const LogprobArgs &a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  // eight lanes fill a 32-byte sector of float32 (half of one of float16)
  if (a.x.sd != 1 && a.x.sl == 1 && a.s.L >= 8)
    return a.k ? launch_lanes<T, true>(ctx, a, s) : launch_lanes<T, false>(ctx, a, s);
  if (a.x.sd == 1) return a.k ? launch_rows<T, V, true>(ctx, a, s) : launch_rows<T, V, false>(ctx, a, s);
  return a.k ? launch_rows<T, 1, true>(ctx, a, s) : launch_rows<T, 1, false>(ctx, a, s);
}

template <typename T, int V>
static acd_status launch_grad_rows(acd_ctx *ctx, const LogprobGradArgs &a, cudaStream_t s) {
  constexpr int64_t batch = (int64_t)BatchU<T, V>::value * V * 32;
  const int64_t segs = (a.s.D + (V - 1) + batch - 1) / batch, tasks = segs * a.s.rows();
  // tasks are counted in 32 bits, with room for the last stride of the grid
  if (tasks > (int64_t)UINT32_MAX - (1 << 20))
    return fail(ACD_ERR_UNSUPPORTED, "acd_token_logprob_grad: too many rows");
  const int grid = persistent_grid(ctx, k_logprob_grad_rows<T, V>, 256, 0, (tasks + 7) / 8);
  k_logprob_grad_rows<T, V><<<grid, 256, 0, s>>>(a, (uint32_t)segs, (uint32_t)tasks);
  return ACD_OK;
}

template <typename T, int V>
static acd_status launch_grad_lanes(acd_ctx *ctx, const LogprobGradArgs &a, cudaStream_t s) {
  const int64_t nl = (a.s.L + V - 1) / V;
  int bx_log2 = 0;
  while (bx_log2 < 5 && (1 << bx_log2) < nl) ++bx_log2;
  const int64_t bx = 1 << bx_log2, by = 256 >> bx_log2, lblocks = (nl + bx - 1) / bx, blocks = lblocks * a.s.O;
  // 64 steps a thread pay for its coefficients; fewer where blocks are wanted
  int64_t chunk = by * 64;
  while (chunk > by * 8 && blocks * ((a.s.D + chunk - 1) / chunk) < (int64_t)ctx->sm_count * 16) chunk /= 2;
  while ((a.s.D + chunk - 1) / chunk > 65535) chunk *= 2;
  if (blocks > INT32_MAX) return fail(ACD_ERR_UNSUPPORTED, "acd_token_logprob_grad: too many rows");
  const dim3 grid((unsigned)blocks, (unsigned)((a.s.D + chunk - 1) / chunk));
  k_logprob_grad_lanes<T, V><<<grid, 256, 0, s>>>(a, bx_log2, lblocks, chunk);
  return ACD_OK;
}

template <typename T>
static acd_status launch_logprob_grad(acd_ctx *ctx, const LogprobGradArgs &a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int size = sizeof(T);
  if (a.x.sd != 1 && a.x.sl == 1 && a.g.sl == 1 && a.s.L >= 8) {
    auto wide = [&](int v) {  // every step starts on a boundary of v elements
      return a.s.L % v == 0 && aligned_to<char>(a.x.p, v * size) && a.x.sd % v == 0 && a.x.so % v == 0 &&
             pieces_match(a.x, a.g, a.x.sd, a.g.sd, v, size);
    };
    if (wide(V)) return launch_grad_lanes<T, V>(ctx, a, s);
    if constexpr (sizeof(T) == 2) {
      if (wide(2)) return launch_grad_lanes<T, 2>(ctx, a, s);
    }
    return launch_grad_lanes<T, 1>(ctx, a, s);
  }
  if (a.x.sd == 1 && a.g.sd == 1 && pieces_match(a.x, a.g, a.x.sl, a.g.sl, V, size))
    return launch_grad_rows<T, V>(ctx, a, s);
  return launch_grad_rows<T, 1>(ctx, a, s);
}

}  // namespace acd

using namespace acd;

extern "C" {

acd_status acd_token_logprob(acd_ctx *ctx, const acd_desc *logprob, const acd_desc *entropy, const acd_desc *lse,
                             const acd_desc *top_index, const acd_desc *top_logprob, const acd_desc *logits,
                             const acd_desc *tokens, int32_t axis, double scale, int32_t one_based,
                             acd_stream stream) {
  const char *op = "acd_token_logprob";
  if (!ctx) return fail(ACD_ERR_INVALID, "%s: null context", op);
  ACD_TRY(check_logits(op, logits, axis, scale));
  if ((tokens == nullptr) != (logprob == nullptr))
    return fail(ACD_ERR_INVALID, "%s: tokens and logprob must both be given or both be NULL", op);
  if ((top_index == nullptr) != (top_logprob == nullptr))
    return fail(ACD_ERR_INVALID, "%s: top_index and top_logprob must both be given or both be NULL", op);
  if (tokens) ACD_TRY(check_tokens(op, tokens, logits, axis));
  ACD_TRY(check_stat(op, "logprob", logprob, logits, axis));
  ACD_TRY(check_stat(op, "entropy", entropy, logits, axis));
  ACD_TRY(check_stat(op, "lse", lse, logits, axis));
  LogprobArgs a{};
  if (top_index) {
    ACD_TRY(check_desc(top_index, "top_index"));
    if (top_index->ndim != logits->ndim)
      return fail(ACD_ERR_SHAPE, "%s: top_index must have the logits' rank", op);
    const int64_t k = top_index->shape[axis];
    if (k < 1 || k > kMaxTop) return fail(ACD_ERR_UNSUPPORTED, "%s: 1 to %d alternatives", op, kMaxTop);
    if (k > logits->shape[axis]) return fail(ACD_ERR_SHAPE, "%s: more alternatives than tokens", op);
    ACD_TRY(check_row_tensor(op, "top_index", top_index, logits, axis, k));
    ACD_TRY(check_row_tensor(op, "top_logprob", top_logprob, logits, axis, k));
    if (!same_shape(top_index, top_logprob))
      return fail(ACD_ERR_SHAPE, "%s: top_index and top_logprob differ in shape", op);
    if (top_index->dtype != ACD_INT32 && top_index->dtype != ACD_INT64)
      return fail(ACD_ERR_DTYPE, "%s: top_index must be int32 or int64", op);
    if (top_logprob->dtype != stat_dtype(logits->dtype))
      return fail(ACD_ERR_DTYPE, "%s: top_logprob must have the statistics' dtype", op);
    a.k = (int)k;
    a.wide_index = top_index->dtype == ACD_INT64;
  }
  if (!split_rows(logits, axis, a.s, a.x))
    return fail(ACD_ERR_UNSUPPORTED, "%s: view not collapsible around the axis; make it contiguous first", op);
  if (a.s.rows() == 0) return ACD_OK;
  if (a.s.D == 0) return fail(ACD_ERR_SHAPE, "%s: rows without tokens", op);
  if (a.s.rows() > INT32_MAX) return fail(ACD_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows", op);
  a.scale = scale;
  a.tokens = ptr_or_null(tokens);
  a.wide_token = tokens && tokens->dtype == ACD_INT64;
  a.one_based = one_based != 0;
  a.logprob = ptr_or_null(logprob);
  a.entropy = ptr_or_null(entropy);
  a.lse = ptr_or_null(lse);
  a.top_index = ptr_or_null(top_index);
  a.top_logprob = ptr_or_null(top_logprob);
  DeviceGuard g(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logits->dtype == ACD_FLOAT32)
    ACD_TRY(launch_logprob<float>(ctx, a, s));
  else if (logits->dtype == ACD_FLOAT64)
    ACD_TRY(launch_logprob<double>(ctx, a, s));
  else
    ACD_TRY(launch_logprob<__half>(ctx, a, s));
  ACD_CUDA(cudaGetLastError());
  return ACD_OK;
}

acd_status acd_token_logprob_grad(acd_ctx *ctx, const acd_desc *grad, const acd_desc *logits, const acd_desc *tokens,
                                  int32_t axis, double scale, const acd_desc *lse, const acd_desc *entropy,
                                  const acd_desc *d_logprob, const acd_desc *d_entropy, const acd_desc *d_lse,
                                  int32_t one_based, acd_stream stream) {
  const char *op = "acd_token_logprob_grad";
  if (!ctx) return fail(ACD_ERR_INVALID, "%s: null context", op);
  ACD_TRY(check_logits(op, logits, axis, scale));
  ACD_TRY(check_desc(grad, "grad"));
  if (grad->dtype != logits->dtype) return fail(ACD_ERR_DTYPE, "%s: grad must have the logits' dtype", op);
  if (!same_shape(grad, logits)) return fail(ACD_ERR_SHAPE, "%s: grad must have the logits' shape", op);
  if (!d_logprob && !d_entropy && !d_lse) return fail(ACD_ERR_INVALID, "%s: no gradient given", op);
  if (!lse) return fail(ACD_ERR_INVALID, "%s: null lse", op);
  if (d_logprob && !tokens) return fail(ACD_ERR_INVALID, "%s: d_logprob needs tokens", op);
  if (d_entropy && !entropy) return fail(ACD_ERR_INVALID, "%s: d_entropy needs entropy", op);
  if (d_logprob) ACD_TRY(check_tokens(op, tokens, logits, axis));
  ACD_TRY(check_stat(op, "lse", lse, logits, axis));
  if (d_entropy) ACD_TRY(check_stat(op, "entropy", entropy, logits, axis));
  ACD_TRY(check_stat(op, "d_logprob", d_logprob, logits, axis));
  ACD_TRY(check_stat(op, "d_entropy", d_entropy, logits, axis));
  ACD_TRY(check_stat(op, "d_lse", d_lse, logits, axis));
  LogprobGradArgs a{};
  RowShape sg;
  if (!split_rows(logits, axis, a.s, a.x) || !split_rows(grad, axis, sg, a.g))
    return fail(ACD_ERR_UNSUPPORTED, "%s: view not collapsible around the axis; make it contiguous first", op);
  if (a.s.rows() == 0 || a.s.D == 0) return ACD_OK;
  if (a.s.rows() > INT32_MAX) return fail(ACD_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows", op);
  a.scale = scale;
  a.tokens = d_logprob ? desc_ptr(tokens) : nullptr;
  a.wide_token = d_logprob && tokens->dtype == ACD_INT64;
  a.one_based = one_based != 0;
  a.lse = desc_ptr(lse);
  a.entropy = d_entropy ? desc_ptr(entropy) : nullptr;
  a.d_logprob = ptr_or_null(d_logprob);
  a.d_entropy = ptr_or_null(d_entropy);
  a.d_lse = ptr_or_null(d_lse);
  DeviceGuard g(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (logits->dtype == ACD_FLOAT32)
    ACD_TRY(launch_logprob_grad<float>(ctx, a, s));
  else if (logits->dtype == ACD_FLOAT64)
    ACD_TRY(launch_logprob_grad<double>(ctx, a, s));
  else
    ACD_TRY(launch_logprob_grad<__half>(ctx, a, s));
  ACD_CUDA(cudaGetLastError());
  return ACD_OK;
}

}  // extern "C"
