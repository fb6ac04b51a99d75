// Log probabilities of given tokens with entropy and the k most likely
// alternatives, and their gradient.
//
// A row holds the logits x_v of one prediction.  With c = scale, m = max x,
//   S = sum e^{c(x_v - m)},  T = sum c(x_v - m) e^{c(x_v - m)}
// everything the forward call returns follows from (m, S, T):
//   lse = c m + ln S,  logprob = c(x_t - m) - ln S,  entropy = ln S - T / S.
// The gradient is one expression a logit (see grad_values).
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
  // A log probability: floor_z, and never above 0.
  static __device__ __forceinline__ float limit_lp(float z) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(floor_z(z)), "f"(0.0f));
    return r;
  }
  static constexpr float kFar = -1048576.0f, kNear = 512.0f;  // -2^20, 2^9
  static __device__ __forceinline__ float lowest() { return -FLT_MAX; }
  static __device__ __forceinline__ float max2(float a, float b) { return fmaxf(a, b); }
  static __device__ __forceinline__ float min2(float a, float b) { return fminf(a, b); }
};
template <>
struct LpMath<double> {
  static constexpr double kUnit = 1.0;
  static __device__ __forceinline__ double factor(double scale) { return scale; }
  static __device__ __forceinline__ double ex(double z) { return exp(z); }
  static __device__ __forceinline__ double floor_z(double z) { return z < -1000.0 ? -1000.0 : z; }  // e^-1000 = 0
  static __device__ __forceinline__ double limit_lp(double z) { return z > 0.0 ? 0.0 : floor_z(z); }
  static constexpr double kFar = -562949953421312.0, kNear = 512.0;  // -2^49
  static __device__ __forceinline__ double lowest() { return -DBL_MAX; }
  static __device__ __forceinline__ double max2(double a, double b) { return fmax(a, b); }
  static __device__ __forceinline__ double min2(double a, double b) { return fmin(a, b); }
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
  // N logits against the present m.
  template <int N>
  __device__ __forceinline__ void sum(const A (&x)[N], A c) {
    if constexpr (std::is_same<A, float>::value && N % 2 == 0) {
      const uint64_t nm = pack2(-m, -m), cc = pack2(c, c);
      uint64_t s2 = pack2(0.0f, 0.0f), t2 = s2;
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float z0, z1;
        unpack2(mul2(add2(pack2(x[j], x[j + 1]), nm), cc), z0, z1);
        z0 = LpMath<A>::floor_z(z0);
        z1 = LpMath<A>::floor_z(z1);
        const uint64_t e = pack2(LpMath<A>::ex(z0), LpMath<A>::ex(z1));
        s2 = add2(s2, e);
        t2 = fma2(e, pack2(z0, z1), t2);
      }
      float a0, a1;
      unpack2(s2, a0, a1);
      s += a0 + a1;
      unpack2(t2, a0, a1);
      t += a0 + a1;
    } else {
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
  // Every lane offers one logit, or nothing (not `valid`).
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

// Looks through a batch of U * V values a lane for what belongs to the list:
// lane l holds elements base + u*32*V + l*V + j, bm is its largest.  Batches
// come with rising base, so a later value that equals entry k - 1 never wins.
// `floor`: some k values are at least this large.  Only lanes whose largest
// value can enter the list are looked at, one after the other, the warp reading
// such a lane's values together from `spread` in shared memory.
template <typename A, int U, int V>
__device__ __forceinline__ void search_batch(TopList<A> &top, const A (&x)[U * V], A bm, int base, int D, int k, A floor,
                                             A *spread) {
  const bool first = top.ki == kNone;
  if (!first && !__any_sync(~0u, bm > top.kv && bm >= floor)) return;
  // k lanes' maxima are at least as large as the k-th of them
  if (first) floor = LpMath<A>::max2(floor, kth_of_lanes(bm, k));
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < V; ++j) spread[(u * 32 + lane) * V + j] = x[u * V + j];
  __syncwarp();
  unsigned mask = __ballot_sync(~0u, bm >= floor && (first || bm > top.kv));
#pragma unroll 1
  while (mask) {
    const int src = __ffs(mask) - 1, at = (lane / V * 32 + src) * V + lane % V, xi = base + at;
    const bool mine = lane < U * V && xi >= 0 && xi < D;
    top.offer(mine ? spread[at] : A(0), xi, mine, floor, k);
    mask &= mask - 1;
    mask &= __ballot_sync(~0u, bm >= top.kv);
  }
  __syncwarp();
}

template <typename A, int N>
__device__ __forceinline__ A largest(const A (&x)[N]) {
  A m = LpMath<A>::max2(x[0], A(-INFINITY));
#pragma unroll
  for (int j = 1; j < N; ++j) m = LpMath<A>::max2(m, x[j]);
  return m;
}

// What one warp knows of the part of a row that it has read.
template <typename T, int U, int V, bool TOP>
struct RowState {
  using A = typename AccOf<T>::type;
  Part<A> p;
  TopList<A> top;
  __device__ __forceinline__ void init() {
    p.init();
    if (TOP) top.init();
  }
  __device__ __forceinline__ void batch(const Piece<T, V> (&raw)[U], int base, int D, A c, int k, A floor, A *spread) {
    A x[U * V];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u].widen(x + u * V);
    const A bm = largest(x);
    p.rescale(LpMath<A>::max2(p.m, bm), c);  // once for all of them
    p.sum(x, c);
    if (TOP) search_batch<A, U, V>(top, x, bm, base, D, k, floor, spread);
  }
};

// A row's results from what is known of all of it: statistics by one thread,
// alternatives one by one.
template <typename A>
struct RowResult {
  A m, log_s;
  __device__ __forceinline__ RowResult(const LogprobArgs &a, const Part<A> &p)
      : m(p.m), log_s(p.s == A(0) ? A(0) : lp_log(p.s)) {}
  __device__ __forceinline__ void stats(const LogprobArgs &a, int64_t r, const Part<A> &p, int64_t t, A xt) const {
    const bool empty = p.s == A(0);  // every logit -Inf
    const A c = (A)a.scale;
    if (a.lse) static_cast<A *>(a.lse)[r] = empty ? A(-INFINITY) : fma_a(c, m, log_s);
    if (a.entropy) static_cast<A *>(a.entropy)[r] = empty ? A(0) : log_s - LpMath<A>::kUnit * (p.t / p.s);
    if (a.logprob) {
      A lp = A(NAN);
      if (t == -1)
        lp = A(0);
      else if (t >= 0 && t < a.s.D)
        lp = empty ? A(-INFINITY) : c * (xt - m) - log_s;
      static_cast<A *>(a.logprob)[r] = lp;
    }
  }
  __device__ __forceinline__ void alternative(const LogprobArgs &a, int64_t r, int j, A v, int i) const {
    const int64_t o = (uint32_t)r / (uint32_t)a.s.L, l = r - o * a.s.L;
    const int64_t at = l + a.s.L * (j + a.k * o);
    const bool none = i == kNone;
    store_index(a.top_index, a.wide_index, at,
                none ? (a.wide_index ? INT64_MIN : (int64_t)INT32_MIN) : (int64_t)i + (a.one_based ? 1 : 0));
    static_cast<A *>(a.top_logprob)[at] = none ? A(NAN) : (A)a.scale * (v - m) - log_s;
  }
};

template <typename A, bool TOP>
__device__ __forceinline__ void finish_row(const LogprobArgs &a, int64_t r, const Part<A> &p, A v, int i, int64_t t,
                                           A xt) {
  const int lane = threadIdx.x & 31;
  const RowResult<A> res(a, p);
  if (lane == 0) res.stats(a, r, p, t, xt);
  if (TOP && lane < a.k) res.alternative(a, r, lane, v, i);
}

// The token asked for (0-based; -1 none; others outside the row) and its logit.
__device__ __forceinline__ int64_t asked_token(const LogprobArgs &a, int64_t r) {
  return a.logprob ? load_index(a.tokens, a.wide_token, r) - (a.one_based ? 1 : 0) : -1;
}
template <typename T, typename A>
__device__ __forceinline__ A asked_logit(const LogprobArgs &a, int64_t t, const T *x) {
  return t >= 0 && t < a.s.D ? to_acc(x[t * a.x.sd]) : A(0);
}

// ---------------------------------------------------------------------------
// rows along the axis
// ---------------------------------------------------------------------------
// How many pieces of V logits a lane holds at once.
template <typename T, int V>
struct BatchU { static constexpr int value = V == 1 ? 8 : 4; };

// A lane's pieces of batch b, -Inf beyond the row's ends.
template <typename T, int V, int U>
__device__ __forceinline__ void load_batch(const T *x, int64_t sd, int D, int shift, int b, Piece<T, V> (&out)[U]) {
  const int lane = threadIdx.x & 31, base = b * (U * V * 32) - shift;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int first = base + (u * 32 + lane) * V;
    if (V == 1) {
      out[u].set(0, first < D ? x[first * sd] : (T)(-INFINITY));
    } else if (first >= 0 && first + V <= D) {
      out[u] = *reinterpret_cast<const Piece<T, V> *>(x + first);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) out[u].set(j, first + j >= 0 && first + j < D ? x[first + j] : (T)(-INFINITY));
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ int row_batches(int D, int shift) {
  constexpr int N = BatchU<T, V>::value * V * 32;
  return (int)(((int64_t)shift + D + N - 1) / N);
}

// One warp a row.  The next batch, of this row or of the next one, is on its
// way while one is worked on; so is the next row's token.  Bound by the reads:
// 65536 x 4096 float32 in 156 us, 1.05 of a copy's rate (reads alone run faster
// than a copy); with five alternatives 65536 x 1024 in 130 us, bound by the
// insertions into the lists.
template <typename T, int V, bool TOP>
__global__ void __launch_bounds__(256, sizeof(T) == 8 ? 2 : TOP ? 3 : 4) k_logprob_warp(LogprobArgs a) {
  using A = typename AccOf<T>::type;
  constexpr int U = BatchU<T, V>::value;
  __shared__ __align__(16) A sh_spread[TOP ? 8 : 1][TOP ? U * V * 32 : 1];
  A *spread = sh_spread[TOP ? threadIdx.x >> 5 : 0];
  const A c = LpMath<A>::factor(a.scale);
  const int D = (int)a.s.D;
  const int64_t rows = a.s.rows(), step = (int64_t)gridDim.x * 8;
  int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= rows) return;
  const T *x = row_ptr<T>(a.x, r, a.s.L);
  Piece<T, V> cur[U], next[U];
  load_batch<T, V, U>(x, a.x.sd, D, row_shift<T, V>(x), 0, cur);
  int64_t t = asked_token(a, r);
  while (true) {
    const bool more = r + step < rows;
    const T *xn = more ? row_ptr<T>(a.x, r + step, a.s.L) : x;
    const int64_t tn = more ? asked_token(a, r + step) : -1;
    const A xt = asked_logit<T, A>(a, t, x);
    const int shift = row_shift<T, V>(x), batches = row_batches<T, V>(D, shift);
    RowState<T, U, V, TOP> st;
    st.init();
    for (int b = 0; b < batches; ++b) {
      if (b + 1 < batches)
        load_batch<T, V, U>(x, a.x.sd, D, shift, b + 1, next);
      else if (more)
        load_batch<T, V, U>(xn, a.x.sd, D, row_shift<T, V>(xn), 0, next);
      st.batch(cur, b * (U * V * 32) - shift, D, c, a.k, A(-INFINITY), spread);
#pragma unroll
      for (int u = 0; u < U; ++u) cur[u] = next[u];
    }
    st.p.warp_merge(c);
    finish_row<A, TOP>(a, r, st.p, st.top.v, st.top.i, t, xt);
    if (!more) return;
    r += step;
    x = xn;
    t = tn;
  }
}

// A cluster of blocks a row: its batches go round the warps of all blocks; the
// warps' sums and lists are joined in each block, the blocks' in the first one
// through distributed shared memory, always in the same order.  Bound by the
// reads where there are many rows (4096 x 50001 float32 in 123 us, 1.02 of a
// copy's rate).  One row of 131072 float16 takes 3.8 us without alternatives, 6.8
// with one, 9.3 with five and 17.5 with twenty: the lists take their candidates
// one after the other.  (Twenty with one block a row 36 us, with two 28, with four
// 22.)
template <typename T, int V, bool TOP, int NW>
__global__ void __launch_bounds__(NW * 32, sizeof(T) == 8 ? 2 : TOP ? 3 : 4) k_logprob_cta(LogprobArgs a) {
  using A = typename AccOf<T>::type;
  constexpr int U = BatchU<T, V>::value;
  __shared__ Part<A> sh_p[NW];
  __shared__ A sh_v[NW][32];
  __shared__ int sh_i[NW][32];
  __shared__ A sh_floor;
  __shared__ __align__(16) A sh_spread[TOP ? NW : 1][TOP ? U * V * 32 : 1];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const A c = LpMath<A>::factor(a.scale);
  const int D = (int)a.s.D;
  const int64_t r = blockIdx.x / C;
  const T *x = row_ptr<T>(a.x, r, a.s.L);
  const int shift = row_shift<T, V>(x), batches = row_batches<T, V>(D, shift), step = C * NW;
  Piece<T, V> cur[U], next[U];
  int b = rank * NW + warp;
  if (b < batches) load_batch<T, V, U>(x, a.x.sd, D, shift, b, cur);
  int64_t t = asked_token(a, r);
  if (threadIdx.x == 0) sh_floor = A(-INFINITY);
  if (TOP) __syncthreads();
  RowState<T, U, V, TOP> st;
  st.init();
  volatile A *floor = &sh_floor;
  for (; b < batches; b += step) {
    if (b + step < batches) load_batch<T, V, U>(x, a.x.sd, D, shift, b + step, next);
    st.batch(cur, b * (U * V * 32) - shift, D, c, a.k, TOP ? *floor : A(0), sh_spread[TOP ? warp : 0]);
    // any warp's entry k - 1 will do as floor: the value decides how much is
    // looked at, never the result
    if (TOP && lane == 0 && st.top.ki != kNone && st.top.kv > *floor) *floor = st.top.kv;
#pragma unroll
    for (int u = 0; u < U; ++u) cur[u] = next[u];
  }
  const A xt = asked_logit<T, A>(a, t, x);
  st.p.warp_merge(c);
  if (lane == 0) sh_p[warp] = st.p;
  if (TOP) {
    sh_v[warp][lane] = st.top.v;
    sh_i[warp][lane] = st.top.i;
  }
  __syncthreads();
  // lists: halve the number of warps until one is left
  auto join_lists = [&](int n) {
    for (n >>= 1; n; n >>= 1) {
      if (warp < n) {
        st.top.merge_reversed(sh_v[warp + n][31 - lane], sh_i[warp + n][31 - lane]);
        sh_v[warp][lane] = st.top.v;
        sh_i[warp][lane] = st.top.i;
      }
      __syncthreads();
    }
  };
  if (TOP) join_lists(NW);
  if (warp == 0) {
    st.p.init();
    if (lane < NW) st.p = sh_p[lane];
    st.p.warp_merge(c);
    if (lane == 0) sh_p[0] = st.p;
  }
  if (C > 1) {
    cluster.sync();
    if (rank == 0) {
      // a warp fetches a block's list
      A v = A(-INFINITY);
      int i = kNone;
      if (TOP && warp < C) {
        v = cluster.map_shared_rank(&sh_v[0][0], warp)[lane];
        i = cluster.map_shared_rank(&sh_i[0][0], warp)[lane];
      }
      if (warp == 0) {
        st.p.init();
        if (lane < C) st.p = cluster.map_shared_rank(sh_p, lane)[0];
        st.p.warp_merge(c);
      }
      if (TOP) {
        __syncthreads();
        st.top.v = sh_v[warp][lane] = v;
        st.top.i = sh_i[warp][lane] = i;
        __syncthreads();
        join_lists(NW);
      }
    }
    cluster.sync();  // no block leaves while its shared memory is read
  }
  if (rank == 0 && warp == 0) finish_row<A, TOP>(a, r, st.p, st.top.v, st.top.i, t, xt);
}

// ---------------------------------------------------------------------------
// rows across the lanes
// ---------------------------------------------------------------------------
// Column-major logits [tokens, vocabulary]: a row's logits are `sd` apart,
// neighbouring rows lie side by side.  A thread keeps the sums of V neighbouring
// rows and walks along the steps: a warp reads 32 * V neighbouring logits at a
// time and nothing is exchanged but at the end.
//   m is a reference here, not the maximum: sums are scaled anew only when a
// logit is 8 bits above it, which after the first steps it hardly ever is.
//   For the alternatives a thread takes the maximum of every four of its logits
// (a unit), and for each segment of its steps leaves the two largest of these
// and where the largest is (9 bytes a segment).  k segments' largest logits set
// a bound that the k best logits reach, so each of these stands in the best unit
// of a segment, or in a segment whose second value reaches the bound too: of
// those, a few in a hundred, all logits are read again.
//   (Lists kept while reading cost far more: 65536 x 4096 float32 with five
// alternatives took 462 us with tiles turned round in shared memory, 643 us with
// candidates gathered by atomics; reading the best segments again without
// knowing where in them took 336 us, tracking single logits 311 us; 264 us now.)
constexpr int kUnit = 4;  // logits of which one maximum is taken

template <typename A, int V>
struct LaneShape {
  static constexpr int UN = (sizeof(A) == 8 ? 8 : 16) / V;  // steps a thread and tile
  static constexpr int ROWS = 32 * V, STEPS = 8 * UN;
};

struct LaneArgs {
  LogprobArgs a;
  int64_t lblocks;  // blocks of 32 * V rows
  int chunk;        // steps a block takes, a multiple of a segment's tiles
  int chunks;       // blocks a row
  void *parts;      // [chunk][row], null: the block writes the results
  void *segs;       // [tile group][warp][row]: largest logit of `group` tiles' steps of a thread,
  void *seconds;    //   the largest outside its unit,
  uint8_t *places;  //   and which unit that is
  int nsegs;        // segments a row
  int group;        // tiles a segment
  int un_log2, group_log2, len_log2;  // steps a thread and tile, tiles and logits a segment
};
constexpr int kSegList = 128;  // segments of a row that are looked into one by one

template <typename T, int V, bool TOP>
__global__ void __launch_bounds__(256, 4) k_logprob_lanes(LaneArgs la) {
  using A = typename AccOf<T>::type;
  using S = LaneShape<A, V>;
  constexpr int UN = S::UN, ROWS = S::ROWS, STEPS = S::STEPS;
  __shared__ Part<A> parts[8][ROWS];
  const LogprobArgs &a = la.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t blk = blockIdx.x / la.chunks, o = blk / la.lblocks, l0 = (blk - o * la.lblocks) * ROWS;
  const int chunk = (int)(blockIdx.x - blk * la.chunks);
  const int64_t L = a.s.L, sd = a.x.sd, l = l0 + lane * V;
  const bool active = l < L;  // V divides L
  const int D = (int)a.s.D;
  const T *x = static_cast<const T *>(a.x.p) + o * a.x.so + (active ? l : 0);
  const A c = LpMath<A>::factor(a.scale);
  const int s0 = chunk * la.chunk, s1 = D - s0 < la.chunk ? D : s0 + la.chunk;
  Piece<T, V> cur[UN], next[UN];
  auto load = [&](int s, Piece<T, V> (&out)[UN]) {
    if (active && s + STEPS <= s1) {
      const T *p = x + (int64_t)(s + warp) * sd;
#pragma unroll
      for (int u = 0; u < UN; ++u, p += 8 * sd) out[u] = *reinterpret_cast<const Piece<T, V> *>(p);
    } else {
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int step = s + u * 8 + warp;
        if (active && step < s1) {
          out[u] = *reinterpret_cast<const Piece<T, V> *>(x + step * sd);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) out[u].set(j, (T)(-INFINITY));
        }
      }
    }
  };
  Part<A> p[V];
  A limit[V], s1st[V], s2nd[V];  // scale anew above `limit`; the segment's two largest
  int place[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    p[j].init();
    limit[j] = LpMath<A>::lowest();
    s1st[j] = s2nd[j] = A(-INFINITY);
    place[j] = 0;
  }
  int unit = 0;  // units of the segment so far
  int64_t seg = ((int64_t)(s0 / (STEPS * la.group)) * 8 + warp) * a.s.rows() + o * L + l;
  if (s0 < s1) load(s0, cur);
  for (int s = s0; s < s1; s += STEPS) {
    // the next tile is under way meanwhile; with the segments' values there are
    // no registers for it at four blocks an SM, which are worth more
    if (TOP) {
      if (s > s0) load(s, cur);
    } else if (s + STEPS < s1) {
      load(s + STEPS, next);
    }
    A f[UN][V];
#pragma unroll
    for (int u = 0; u < UN; ++u) cur[u].widen(f[u]);
    bool grown = false;
    A bm[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      bm[j] = A(-INFINITY);
#pragma unroll
      for (int q = 0; q < UN / kUnit; ++q) {
        A um = f[q * kUnit][j];
#pragma unroll
        for (int u = 1; u < kUnit; ++u) um = LpMath<A>::max2(um, f[q * kUnit + u][j]);
        if (TOP) {
          place[j] = um > s1st[j] ? unit + q : place[j];
          s2nd[j] = LpMath<A>::max2(s2nd[j], LpMath<A>::min2(um, s1st[j]));
          s1st[j] = LpMath<A>::max2(s1st[j], um);
        }
        bm[j] = LpMath<A>::max2(bm[j], um);
      }
      grown |= bm[j] > limit[j];
    }
    unit += UN / kUnit;
    if (__any_sync(~0u, grown)) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (bm[j] > limit[j]) {
          p[j].rescale(bm[j], c);
          limit[j] = bm[j] + A(8) / c;
        }
    }
    if constexpr (std::is_same<A, float>::value && V % 2 == 0) {
      const uint64_t cc = pack2(c, c);
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const uint64_t nm = pack2(-p[j].m, -p[j + 1].m);
        uint64_t s2 = pack2(p[j].s, p[j + 1].s), t2 = pack2(p[j].t, p[j + 1].t);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          float z0, z1;
          unpack2(mul2(add2(pack2(f[u][j], f[u][j + 1]), nm), cc), z0, z1);
          z0 = LpMath<A>::floor_z(z0);
          z1 = LpMath<A>::floor_z(z1);
          const uint64_t e = pack2(LpMath<A>::ex(z0), LpMath<A>::ex(z1));
          s2 = add2(s2, e);
          t2 = fma2(e, pack2(z0, z1), t2);
        }
        unpack2(s2, p[j].s, p[j + 1].s);
        unpack2(t2, p[j].t, p[j + 1].t);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        A col[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) col[u] = f[u][j];
        p[j].sum(col, c);
      }
    }
    if (TOP && (unit * kUnit == 1 << la.len_log2 || s + STEPS >= s1)) {
      Vec<A, V> w1, w2;
      Vec<uint8_t, V> wp;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        w1.v[j] = s1st[j];
        w2.v[j] = s2nd[j];
        wp.v[j] = (uint8_t)place[j];
        s1st[j] = s2nd[j] = A(-INFINITY);
        place[j] = 0;
      }
      unit = 0;
      if (active) {
        *reinterpret_cast<Vec<A, V> *>(static_cast<A *>(la.segs) + seg) = w1;
        *reinterpret_cast<Vec<A, V> *>(static_cast<A *>(la.seconds) + seg) = w2;
        *reinterpret_cast<Vec<uint8_t, V> *>(la.places + seg) = wp;
      }
      seg += 8 * a.s.rows();
    }
    if (!TOP) {
#pragma unroll
      for (int u = 0; u < UN; ++u) cur[u] = next[u];
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) parts[warp][lane * V + j] = p[j];
  __syncthreads();
  const int row = threadIdx.x;
  if (row >= ROWS || l0 + row >= L) return;
  Part<A> q = parts[0][row];
  for (int w = 1; w < 8; ++w) q.merge(parts[w][row], c);
  const int64_t r = o * L + l0 + row;
  if (la.parts) {
    static_cast<Part<A> *>(la.parts)[chunk * a.s.rows() + r] = q;
    return;
  }
  const int64_t t = asked_token(a, r);
  RowResult<A>(a, q).stats(a, r, q, t, asked_logit<T, A>(a, t, static_cast<const T *>(a.x.p) + o * a.x.so + l0 + row));
}

// Where logit i of segment g lies in the row: tile g / 8 of groups, step within it.
__device__ __forceinline__ int segment_step(const LaneArgs &la, int g, int i) {
  return ((((g >> 3) << la.group_log2) + (i >> la.un_log2)) << (la.un_log2 + 3)) +
         ((i & ((1 << la.un_log2) - 1)) << 3) + (g & 7);
}

// The k best logits of row r, found by a warp.
template <typename T>
__device__ __forceinline__ TopList<typename AccOf<T>::type> row_alternatives(const LaneArgs &la, int64_t r, int *list) {
  using A = typename AccOf<T>::type;
  constexpr int U = 8;
  const LogprobArgs &a = la.a;
  const int lane = threadIdx.x & 31, k = a.k;
  const int64_t rows = a.s.rows();
  const T *x = row_ptr<T>(a.x, r, a.s.L);
  TopList<A> top;
  top.init();
  const A *segs = static_cast<const A *>(la.segs) + r;
  const int n = la.nsegs, D = (int)a.s.D;
  A kept[U], lm = A(-INFINITY);  // the first segments' maxima, and the largest of this lane's
#pragma unroll
  for (int u = 0; u < U; ++u) kept[u] = u * 32 + lane < n ? segs[(int64_t)(u * 32 + lane) * rows] : A(NAN);
#pragma unroll
  for (int u = 0; u < U; ++u) lm = LpMath<A>::max2(lm, kept[u]);
  for (int g = U * 32 + lane; g < n; g += 32) lm = LpMath<A>::max2(lm, segs[(int64_t)g * rows]);
  const A floor = kth_of_lanes(lm, k);  // k segments, so k logits, are at least this large
  // the segments that reach the floor; with `above` those over it
  auto gather = [&](bool above) {
    int count = 0;
    auto add = [&](int g, A v) {
      const bool in = above ? v > floor : v >= floor;
      const unsigned mask = __ballot_sync(~0u, in);
      const int at = count + __popc(mask & ((1u << lane) - 1));
      if (in && at < kSegList) list[at] = g;
      count += __popc(mask);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) add(u * 32 + lane, kept[u]);
    for (int b = U * 32; b < n; b += 32) add(b + lane, b + lane < n ? segs[(int64_t)(b + lane) * rows] : A(NAN));
    __syncwarp();
    return count;
  };
  auto look = [&](int to, bool above) {
    constexpr int M = 4;  // batches in flight
    for (int e = 0; e < to; e += 32 * M) {
      A v[M];
      int step[M];
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const int at = e + m * 32 + lane;
        step[m] = D;
        if (at < to) {
          const int g = list[at >> la.len_log2], i = at & ((1 << la.len_log2) - 1);
          step[m] = segment_step(la, g, i);
        }
        v[m] = step[m] < D ? to_acc(x[step[m] * a.x.sd]) : A(NAN);
      }
#pragma unroll
      for (int m = 0; m < M; ++m) top.offer(v[m], step[m], above ? v[m] > floor : v[m] >= floor, floor, k);
    }
  };
  int count = gather(false);
  if (count <= kSegList && floor > A(-INFINITY)) {
    for (int e = 0; e < count * kUnit; e += 32) {
      const int at = e + lane;
      int step = D;
      if (at < count * kUnit) {
        const int g = list[at / kUnit];
        step = segment_step(la, g, la.places[(int64_t)g * rows + r] * kUnit + at % kUnit);
      }
      const A v = step < D ? to_acc(x[step * a.x.sd]) : A(NAN);
      top.offer(v, step, v >= floor, floor, k);
    }
    const A bound = top.kv;  // no less than the floor
    for (int e = 0; e < count; e += 32) {
      const int64_t g = e + lane < count ? list[e + lane] : 0;
      unsigned mask = __ballot_sync(~0u, e + lane < count && static_cast<const A *>(la.seconds)[g * rows + r] >= bound);
      while (mask) {
        const int64_t gs = __shfl_sync(~0u, g, __ffs(mask) - 1);
        mask &= mask - 1;
        const int place = la.places[gs * rows + r];
        for (int i = 0; i < 1 << la.len_log2; i += 32) {
          const int step = segment_step(la, (int)gs, i + lane);
          const bool ok = i + lane < 1 << la.len_log2 && (i + lane) / kUnit != place && step < D;
          top.offer(ok ? to_acc(x[step * a.x.sd]) : A(0), step, ok, bound, k);
        }
      }
    }
  } else {
    // Many logits equal to the floor: those over it from their segments (less
    // than k lanes have one), the others from the row's beginning, where
    // enough of them are soon found.
    count = gather(true);
    if (count <= kSegList) {
      look(count << la.len_log2, true);
    } else {
      for (int s = 0; s < D; s += 32) {
        const A v = s + lane < D ? to_acc(x[(s + lane) * a.x.sd]) : A(NAN);
        top.offer(v, s + lane, v > floor, floor, k);
      }
    }
    for (int s = 0; s < D && top.ki == kNone; s += 32) {
      const A v = s + lane < D ? to_acc(x[(s + lane) * a.x.sd]) : A(NAN);
      top.offer(v, s + lane, v == floor, floor, k);
    }
  }
  return top;
}

// A warp a row: joins the parts of blocks and finds the alternatives.
template <typename T, bool TOP>
__global__ void __launch_bounds__(256, sizeof(T) == 8 ? 3 : 5) k_logprob_join(const __grid_constant__ LaneArgs la) {
  using A = typename AccOf<T>::type;
  __shared__ int sh_list[TOP ? 8 : 1][TOP ? kSegList : 1];
  const LogprobArgs &a = la.a;
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.s.rows(), r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= rows) return;
  const T *x = row_ptr<T>(a.x, r, a.s.L);
  const int64_t t = asked_token(a, r);
  const A c = LpMath<A>::factor(a.scale);
  Part<A> p;
  p.init();
  for (int q = lane; q < la.chunks; q += 32) p.merge(static_cast<const Part<A> *>(la.parts)[q * rows + r], c);
  p.warp_merge(c);
  const A xt = asked_logit<T, A>(a, t, x);
  TopList<A> top;
  top.init();
  if constexpr (TOP) top = row_alternatives<T>(la, r, sh_list[threadIdx.x >> 5]);
  finish_row<A, TOP>(a, r, p, top.v, top.i, t, xt);
}

template <typename T>
__device__ __noinline__ TopList<typename AccOf<T>::type> row_alternatives_apart(const LaneArgs &la, int64_t r, int *list) {
  return row_alternatives<T>(la, r, list);
}

// Few alternatives of many rows: a thread a row, its lists in registers, so that
// the segments are read along the rows and a row costs a tenth of a warp's
// instructions.  Three segments more than K are kept for those that tie with
// the K-th; a row with more ties, or with fewer than K logits above -Inf, and a
// segment that has to be read again are looked at by the whole warp.  It costs 68
// of the 264 us of 65536 x 4096 float32 with five alternatives, spent on scattered
// reads of the units that hold them (a warp a row: 190 us).
template <typename T, int K>
__global__ void __launch_bounds__(128) k_logprob_pick(const __grid_constant__ LaneArgs la) {
  using A = typename AccOf<T>::type;
  constexpr int U = 8, N = K + 3;
  __shared__ int sh_list[4][kSegList];
  const LogprobArgs &a = la.a;
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.s.rows(), row = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const bool active = row < rows;
  const int64_t r = active ? row : rows - 1;
  const T *x = row_ptr<T>(a.x, r, a.s.L);
  const int64_t t = asked_token(a, r);
  const A *segs = static_cast<const A *>(la.segs) + r, *seconds = static_cast<const A *>(la.seconds) + r;
  const uint8_t *places = la.places + r;
  const int n = la.nsegs, D = (int)a.s.D, len = 1 << la.len_log2;
  A v[N], lost = A(-INFINITY);  // segments by their largest logit; the largest left out
  int g[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    v[j] = A(-INFINITY);
    g[j] = 0;
  }
  for (int b = 0; b < n; b += U) {
    A s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = b + u < n ? segs[(int64_t)(b + u) * rows] : A(-INFINITY);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      lost = LpMath<A>::max2(lost, LpMath<A>::min2(s[u], v[N - 1]));
      if (s[u] > v[N - 1]) {
#pragma unroll
        for (int j = N - 1; j >= 0; --j) {
          const int q = j > 0 ? j - 1 : 0;
          const bool here = s[u] > v[j], above = j > 0 && s[u] > v[q];
          if (here) {
            v[j] = above ? v[q] : s[u];
            g[j] = above ? g[q] : b + u;
          }
        }
      }
    }
  }
  const A bound = v[K - 1];
  const bool plain = bound > A(-INFINITY) && lost < bound;
  A w[K];  // the logits
  int at[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    w[j] = A(-INFINITY);
    at[j] = kNone;
  }
  auto insert = [&](A y, int i) {
#pragma unroll
    for (int j = K - 1; j >= 0; --j) {
      const int q = j > 0 ? j - 1 : 0;
      const bool here = better(y, i, w[j], at[j]), above = j > 0 && better(y, i, w[q], at[q]);
      if (here) {
        w[j] = above ? w[q] : y;
        at[j] = above ? at[q] : i;
      }
    }
  };
  int place[N];
  bool again[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const bool in = active && plain && v[j] >= bound;
    place[j] = in ? places[(int64_t)g[j] * rows] : -1;
    again[j] = in && seconds[(int64_t)g[j] * rows] >= bound;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    A y[kUnit];
    int step[kUnit];
#pragma unroll
    for (int u = 0; u < kUnit; ++u) {
      step[u] = segment_step(la, g[j], place[j] * kUnit + u);
      y[u] = place[j] >= 0 && step[u] < D ? to_acc(x[step[u] * a.x.sd]) : A(NAN);
    }
#pragma unroll
    for (int u = 0; u < kUnit; ++u)
      if (y[u] >= bound) insert(y[u], step[u]);
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    for (unsigned mask = __ballot_sync(~0u, again[j]); mask; mask &= mask - 1) {
      const int src = __ffs(mask) - 1, gs = __shfl_sync(~0u, g[j], src), ps = __shfl_sync(~0u, place[j], src);
      const A lim = __shfl_sync(~0u, bound, src);
      const T *xs = row_ptr<T>(a.x, __shfl_sync(~0u, r, src), a.s.L);
      for (int i = 0; i < len; i += 32) {
        const int step = segment_step(la, gs, i + lane);
        const bool ok = i + lane < len && step < D && (i + lane) / kUnit != ps;
        const A y = ok ? to_acc(xs[step * a.x.sd]) : A(0);
        for (unsigned in = __ballot_sync(~0u, ok && y >= lim); in; in &= in - 1) {
          const A z = __shfl_sync(~0u, y, __ffs(in) - 1);
          const int zi = __shfl_sync(~0u, step, __ffs(in) - 1);
          if (lane == src) insert(z, zi);
        }
      }
    }
  for (unsigned mask = __ballot_sync(~0u, active && !plain); mask; mask &= mask - 1) {
    const int src = __ffs(mask) - 1;
    const TopList<A> top = row_alternatives_apart<T>(la, __shfl_sync(~0u, r, src), sh_list[threadIdx.x >> 5]);
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const A tv = __shfl_sync(~0u, top.v, j);
      const int ti = __shfl_sync(~0u, top.i, j);
      if (lane == src) {
        w[j] = tv;
        at[j] = ti;
      }
    }
  }
  if (!active) return;
  const A c = LpMath<A>::factor(a.scale);
  Part<A> p = static_cast<const Part<A> *>(la.parts)[r];
  for (int q = 1; q < la.chunks; ++q) p.merge(static_cast<const Part<A> *>(la.parts)[q * rows + r], c);
  const RowResult<A> res(a, p);
  res.stats(a, r, p, t, asked_logit<T, A>(a, t, x));
#pragma unroll
  for (int j = 0; j < K; ++j) res.alternative(a, r, j, w[j], at[j]);
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
// d is rounded once (fma) before the exponential, so that rounding is of its own
// size and not of the logit's.  lse was rounded when it was stored: p is off by up
// to |lse| u of itself, and far from 0 d, the log of a probability, has to be kept
// from being above 0, which the rounded lse alone would allow by any amount.
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
  // throughout by a large finite value: at -2^20 (float64: -2^49) lse has three
  // binary digits left after the point, at -2^24 (-2^53) none for ln S.  (A scale
  // above 1 takes ordinary logits that far: then it is the logits that count.)
  if (g.lse <= LpMath<A>::kFar * LpMath<A>::max2(c, A(1))) {
    g.lse = A(INFINITY);
    g.a0 = g.a1 = g.gt = A(0);
  }
  return g;
}

// N logits of one row (or, with G = N, of N rows side by side).  NEAR: |lse| is at
// most kNear, where its rounding (2^-15 of p in float32) can stay.
template <typename A, int N, int G, bool NEAR>
__device__ __forceinline__ void grad_values(const GradRow<A> (&g)[G], A (&x)[N], A c) {
  using M = LpMath<A>;
  // p = 0 where d is below the floor: 0 log 0 = 0
  auto limit = [](A d) { return NEAR ? M::floor_z(d) : M::limit_lp(d); };
  if constexpr (std::is_same<A, float>::value && N % 2 == 0) {
    const uint64_t cc = pack2(c, c), l2e = pack2(1.44269504088896341f, 1.44269504088896341f);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const GradRow<A> &p = g[G == 1 ? 0 : j], &q = g[G == 1 ? 0 : j + 1];
      float d0, d1, z0, z1;
      unpack2(fma2(cc, pack2(x[j], x[j + 1]), pack2(-p.lse, -q.lse)), d0, d1);
      d0 = limit(d0);
      d1 = limit(d1);
      const uint64_t d = pack2(d0, d1);
      unpack2(mul2(d, l2e), z0, z1);
      unpack2(mul2(pack2(M::ex(z0), M::ex(z1)), fma2(pack2(-p.a1, -q.a1), d, pack2(p.a0, q.a0))), x[j], x[j + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const GradRow<A> &p = g[G == 1 ? 0 : j];
      const A d = limit(fma_a(c, x[j], -p.lse));
      const A e = std::is_same<A, float>::value ? M::ex(d * A(1.44269504088896341)) : M::ex(d);
      x[j] = e * fma_a(-p.a1, d, p.a0);
    }
  }
}

// Rows along the axis: a warp takes U pieces a lane of one row, 16 bytes each
// (V logits; the row may start and end inside a piece), reads them all and
// then writes.  V = 1: any strides.  Bound by reads and writes: 4096 x 32768
// float16 with the entropy's term in 85 us, 0.96 of a copy's rate (124 us with the
// pieces widened as they came in: twice the registers, fewer blocks).
template <typename T, int V>
__global__ void __launch_bounds__(256, sizeof(T) == 8 ? 2 : 5) k_logprob_grad_rows(LogprobGradArgs a, uint32_t segs, uint32_t tasks) {
  using A = typename AccOf<T>::type;
  constexpr int U = BatchU<T, V>::value;
  const int lane = threadIdx.x & 31;
  const A c = (A)a.scale;
  const int D = (int)a.s.D;
  for (uint32_t task = blockIdx.x * 8 + (threadIdx.x >> 5); task < tasks; task += gridDim.x * 8) {
    const uint32_t r = task / segs, seg = task - r * segs;
    const T *x = row_ptr<T>(a.x, r, a.s.L);
    T *out = row_ptr<T>(a.g, r, a.s.L);
    const int shift = row_shift<T, V>(x), base = (int)seg * (U * V * 32) - shift;
    Piece<T, V> raw[U];
    load_batch<T, V, U>(x, a.x.sd, D, shift, (int)seg, raw);
    const GradRow<A> g[1] = {grad_row<A>(a, r)};
    auto finish = [&](auto near) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int first = base + (u * 32 + lane) * V;
        A v[V];
        raw[u].widen(v);
        grad_values<A, V, 1, decltype(near)::value>(g, v, c);
        if (g[0].t >= first && g[0].t < first + V) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (first + j == g[0].t) v[j] += g[0].gt;
        }
        store_piece<T, A, V>(out, a.g.sd, first, D, v);
      }
    };
    if (fabs(g[0].lse) <= LpMath<A>::kNear)
      finish(std::true_type());
    else
      finish(std::false_type());
  }
}

// Rows across the lanes: a thread keeps the coefficients of V neighbouring
// rows and walks along the steps, so that a warp reads and writes 32 * V
// neighbouring logits at a time.  A block is bx threads along the lanes by
// 256 / bx along the steps, and takes `chunk` steps.  Bound by reads and writes:
// 65536 x 4096 float32 in 338 us, 0.97 of a copy's rate.
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
    Piece<T, V> w[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (s + u * by < s1) w[u] = *reinterpret_cast<const Piece<T, V> *>(x + (s + u * by) * a.x.sd);
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (s + u * by >= s1) break;
      A v[V];
      w[u].widen(v);
      grad_values<A, V, V, false>(g, v, c);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (g[j].t == (int)(s + u * by)) v[j] += g[j].gt;
      w[u].round(v);
      *reinterpret_cast<Piece<T, V> *>(out + (s + u * by) * a.g.sd) = w[u];
    }
  }
}

static bool row_dtype(int32_t dt) { return dt == ACD_FLOAT32 || dt == ACD_FLOAT64 || dt == ACD_FLOAT16; }
static int32_t stat_dtype(int32_t dt) { return dt == ACD_FLOAT64 ? ACD_FLOAT64 : ACD_FLOAT32; }

// What float32 statistics work with: c log2(e) is a finite float32, and c not
// below the smallest one (0 would make 0 * Inf of masked logits; 2^-149 moves no
// scaled logit by more than 2^-21).
constexpr double kMaxScale32 = 2.3e38, kMinScale32 = 0x1p-149;
static double stat_scale(const acd_desc *logits, double scale) {
  return logits->dtype != ACD_FLOAT64 && scale < kMinScale32 ? kMinScale32 : scale;
}

static acd_status check_logits(const char *op, const acd_desc *logits, int32_t axis, double scale) {
  ACD_TRY(check_desc(logits, "logits"));
  if (!row_dtype(logits->dtype)) return fail(ACD_ERR_DTYPE, "%s: float32, float64 or float16 logits required", op);
  if (axis < 0 || axis >= logits->ndim) return fail(ACD_ERR_AXIS, "%s: axis %d out of range", op, axis);
  if (!(scale > 0.0) || !std::isfinite(scale)) return fail(ACD_ERR_INVALID, "%s: scale must be positive and finite", op);
  if (logits->dtype != ACD_FLOAT64 && scale > kMaxScale32)
    return fail(ACD_ERR_INVALID, "%s: scale is beyond float32's range", op);
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

template <typename T, int V, bool TOP>
static acd_status launch_lanes(acd_ctx *ctx, const LogprobArgs &a, cudaStream_t s) {
  using A = typename AccOf<T>::type;
  using S = LaneShape<A, V>;
  LaneArgs la{};
  la.a = a;
  la.lblocks = (a.s.L + S::ROWS - 1) / S::ROWS;
  const int64_t blocks = la.lblocks * a.s.O, tiles = (a.s.D + S::STEPS - 1) / S::STEPS;
  la.group = 1;
  while (1 << la.un_log2 < S::UN) ++la.un_log2;
  if (TOP) {
    // a segment of n logits costs 18 bytes written and read, and k^2 / 2 in the
    // row's V / n segments are read again, 64 bytes a logit: least at n^3 = 0.28
    // (V / k)^2 (places are bytes: at most 256)
    auto enough = [&](double m) { return m * m * m * a.k * a.k > 0.28 * (double)a.s.D * (double)a.s.D; };
    while (la.group * S::UN < 256 && !enough(1.5 * la.group * S::UN)) {
      la.group *= 2;
      ++la.group_log2;
    }
  }
  la.len_log2 = la.un_log2 + la.group_log2;
  // rows are divided while there is room for blocks, eight tiles each at least
  int64_t chunks = (int64_t)ctx->sm_count * 3 / blocks;
  if (chunks > tiles / 8) chunks = tiles / 8;
  if (chunks < 1) chunks = 1;
  const int64_t groups = (tiles + la.group - 1) / la.group, per = (groups + chunks - 1) / chunks;
  la.chunk = (int)(per * la.group * S::STEPS);
  la.chunks = (int)((groups + per - 1) / per);
  la.nsegs = (int)(groups * 8);
  if (blocks * la.chunks > INT32_MAX) return fail(ACD_ERR_UNSUPPORTED, "acd_token_logprob: too many rows");
  const bool join = TOP || la.chunks > 1;
  if (join) {
    const size_t np = (size_t)la.chunks * a.s.rows(), ns = TOP ? (size_t)la.nsegs * a.s.rows() : 0;
    void *scratch;
    ACD_TRY(get_scratch(ctx, ns * (2 * sizeof(A) + 1) + np * sizeof(Part<A>), s, &scratch));
    la.segs = scratch;  // written V rows at a time: rows are a multiple of V
    la.seconds = static_cast<A *>(scratch) + ns;
    la.parts = static_cast<A *>(scratch) + 2 * ns;
    la.places = reinterpret_cast<uint8_t *>(static_cast<Part<A> *>(la.parts) + np);
  }
  k_logprob_lanes<T, V, TOP><<<(unsigned)(blocks * la.chunks), 256, 0, s>>>(la);
  if (!join) return ACD_OK;
  if constexpr (TOP && sizeof(T) < 8) {
    // A thread a row where there are rows to hide its scattered reads: more of them
    // the more alternatives there are.  Rows of 4096 float32, a thread or a warp a
    // row, 1, 3, 5 and 8 alternatives: 9472 rows 46, 63, 79, 91 or 49, 53, 57, 58 us;
    // 18944 rows 80, 93, 106, 128 or 93, 91, 96, 105 us; 37888 rows 151, 176, 196,
    // 219 or 178, 191, 201, 216 us; 65536 rows 202, 235, 264, 294 or 252, 273, 289,
    // 315 us.
    if (a.k <= 8 && a.s.rows() >= (int64_t)ctx->sm_count * 32 * (a.k + 1)) {
      const unsigned grid = (unsigned)((a.s.rows() + 127) / 128);
      switch (a.k) {
        case 1: k_logprob_pick<T, 1><<<grid, 128, 0, s>>>(la); break;
        case 2: k_logprob_pick<T, 2><<<grid, 128, 0, s>>>(la); break;
        case 3: k_logprob_pick<T, 3><<<grid, 128, 0, s>>>(la); break;
        case 4: k_logprob_pick<T, 4><<<grid, 128, 0, s>>>(la); break;
        case 5: k_logprob_pick<T, 5><<<grid, 128, 0, s>>>(la); break;
        case 6: k_logprob_pick<T, 6><<<grid, 128, 0, s>>>(la); break;
        case 7: k_logprob_pick<T, 7><<<grid, 128, 0, s>>>(la); break;
        default: k_logprob_pick<T, 8><<<grid, 128, 0, s>>>(la); break;
      }
      return ACD_OK;
    }
  }
  k_logprob_join<T, TOP><<<(unsigned)((a.s.rows() + 7) / 8), 256, 0, s>>>(la);
  return ACD_OK;
}

// Rows a thread: as many as a 16-byte (float16: 8-byte) load holds, if they are
// aligned alike in every step and there are rows for more than half a warp.
template <typename T, bool TOP>
static acd_status launch_lanes_any(acd_ctx *ctx, const LogprobArgs &a, cudaStream_t s) {
  auto fits = [&](int v) {
    return a.s.L % v == 0 && a.s.L > 16 * v && aligned_to<char>(a.x.p, v * (int)sizeof(T)) && a.x.sd % v == 0 &&
           a.x.so % v == 0;
  };
  if constexpr (sizeof(T) < 8) {
    if (fits(4)) return launch_lanes<T, 4, TOP>(ctx, a, s);
  }
  if (fits(2)) return launch_lanes<T, 2, TOP>(ctx, a, s);
  return launch_lanes<T, 1, TOP>(ctx, a, s);
}

template <typename T, int V, bool TOP>
static acd_status launch_rows(acd_ctx *ctx, const LogprobArgs &a, cudaStream_t s) {
  const int64_t rows = a.s.rows(), batch = (int64_t)BatchU<T, V>::value * V * 32;
  const int64_t batches = (a.s.D + batch - 1) / batch;
  // Warps a row need no join, blocks a row have more of a long row under way.
  // float32 rows of 512 logits a batch, a warp or a block a row: 65536 rows of 2
  // batches 52 or 230 us, of 8 156 or 276 us, 16384 rows of 16 83 or 100 us, of 32
  // 177 or 165 us; with five alternatives 65536 rows of 2 batches 130 or 683 us.
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
  // (fewer rows are read an element at a time: 2, 4 and 7 rows of 131072 float16 in
  // 6.4, 6.7 and 9.0 us, 8 rows across the lanes in 10.6)
  if (a.x.sd != 1 && a.x.sl == 1 && a.s.L >= 8)
    return a.k ? launch_lanes_any<T, true>(ctx, a, s) : launch_lanes_any<T, false>(ctx, a, s);
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
  a.scale = stat_scale(logits, scale);
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
  a.scale = stat_scale(logits, scale);
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
