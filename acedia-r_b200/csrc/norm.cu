// A residual update with the norms around it, and its gradients.
//
//   b' = b rs_b w_post,  h = alpha r + gate b',  y = h rs_h w_pre,
//   rs_v = 1 / sqrt(mean(v^2) + eps)
// The gradients, with hn = h rs_h and bn = b rs_b:
//   t = dh + rs_h (dy w_pre - hn mean(dy w_pre hn)),  dr = alpha t,
//   u = t gate,  db = rs_b (u w_post - bn mean(u w_post bn)),
//   dw_pre = sum dy hn,  dw_post = sum u bn,  dgate = sum t b'.
#include <cooperative_groups.h>

#include "lm_rows.cuh"
#include "tma.cuh"

namespace cg = cooperative_groups;

namespace acd {

struct NormArgs {
  RowShape s;
  double alpha, eps;
  Rows r, b, h, y;
  const void *w_pre, *w_post, *gate;
  int64_t gate_sd, gate_sg;  // strides of the gate along the row and over its groups
  int64_t per;               // consecutive rows that share a gate row
  void *rstd_h, *rstd_b;
};

struct NormGradArgs {
  RowShape s;
  double alpha;
  Rows dr, db, dh, dy, h, b;  // dh.p may be null
  const void *w_pre, *w_post, *gate;
  int64_t gate_sd, gate_sg, per;
  const void *rstd_h, *rstd_b;
  void *d_w_pre, *d_w_post, *d_gate;
};

__device__ __forceinline__ float rsqrt_a(float x) { return 1.0f / sqrtf(x); }
__device__ __forceinline__ double rsqrt_a(double x) { return 1.0 / sqrt(x); }

// Sum over the block, in every thread.
template <typename A>
__device__ __forceinline__ A block_sum(A v, A *sh) {
  for (int q = 16; q; q >>= 1) v += __shfl_xor_sync(~0u, v, q);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  A t = 0;
  for (int q = 0; q < (int)(blockDim.x >> 5); ++q) t += sh[q];
  return t;
}

// One block a row, any strides.
template <typename T>
__global__ void __launch_bounds__(256) k_norm_rows(NormArgs a) {
  using A = typename AccOf<T>::type;
  __shared__ A sh[8];
  const A alpha = (A)a.alpha, eps = (A)a.eps, D = (A)a.s.D;
  const T *w_pre = static_cast<const T *>(a.w_pre), *w_post = static_cast<const T *>(a.w_post);
  for (int64_t row = blockIdx.x; row < a.s.rows(); row += gridDim.x) {
    const T *r = row_ptr<T>(a.r, row, a.s.L), *b = row_ptr<T>(a.b, row, a.s.L);
    T *h = row_ptr<T>(a.h, row, a.s.L), *y = row_ptr<T>(a.y, row, a.s.L);
    const T *gate = a.gate ? static_cast<const T *>(a.gate) + (int64_t)((uint32_t)row / (uint32_t)a.per) * a.gate_sg : nullptr;
    A rb = 1;
    if (w_post) {
      A q = 0;
      for (int64_t d = threadIdx.x; d < a.s.D; d += 256) {
        const A v = to_acc(b[d * a.b.sd]);
        q = fma_a(v, v, q);
      }
      rb = rsqrt_a(block_sum(q, sh) / D + eps);
    }
    auto update = [&](int64_t d) {
      A v = to_acc(b[d * a.b.sd]);
      if (w_post) v = v * rb * to_acc(w_post[d]);
      if (gate) v *= to_acc(gate[d * a.gate_sd]);
      return fma_a(alpha, to_acc(r[d * a.r.sd]), v);
    };
    A q = 0;
    for (int64_t d = threadIdx.x; d < a.s.D; d += 256) {
      const A v = update(d);
      q = fma_a(v, v, q);
    }
    const A rh = rsqrt_a(block_sum(q, sh) / D + eps);
    // computed again rather than read back: h may lie over r, y over b
    for (int64_t d = threadIdx.x; d < a.s.D; d += 256) {
      const A v = update(d);
      h[d * a.h.sd] = from_acc<T, A>(v);
      y[d * a.y.sd] = from_acc<T, A>(v * rh * to_acc(w_pre[d]));
    }
    if (threadIdx.x == 0) {
      if (a.rstd_h) static_cast<A *>(a.rstd_h)[row] = rh;
      if (a.rstd_b) static_cast<A *>(a.rstd_b)[row] = rb;
    }
  }
}

// One block a row, any strides: the two means, then both row gradients.
template <typename T>
__global__ void __launch_bounds__(256) k_norm_grad_rows(NormGradArgs a) {
  using A = typename AccOf<T>::type;
  __shared__ A sh[8];
  const A alpha = (A)a.alpha, D = (A)a.s.D;
  const T *w_pre = static_cast<const T *>(a.w_pre), *w_post = static_cast<const T *>(a.w_post);
  for (int64_t row = blockIdx.x; row < a.s.rows(); row += gridDim.x) {
    T *dr = row_ptr<T>(a.dr, row, a.s.L), *db = row_ptr<T>(a.db, row, a.s.L);
    const T *dh = a.dh.p ? row_ptr<T>(a.dh, row, a.s.L) : nullptr, *dy = row_ptr<T>(a.dy, row, a.s.L);
    const T *h = row_ptr<T>(a.h, row, a.s.L), *b = row_ptr<T>(a.b, row, a.s.L);
    const T *gate = a.gate ? static_cast<const T *>(a.gate) + (int64_t)((uint32_t)row / (uint32_t)a.per) * a.gate_sg : nullptr;
    const A rh = static_cast<const A *>(a.rstd_h)[row];
    const A rb = w_post ? static_cast<const A *>(a.rstd_b)[row] : A(1);
    A m1 = 0, m2 = 0;
    for (int64_t d = threadIdx.x; d < a.s.D; d += 256)
      m1 = fma_a(to_acc(dy[d * a.dy.sd]) * to_acc(w_pre[d]), to_acc(h[d * a.h.sd]) * rh, m1);
    m1 = block_sum(m1, sh) / D;
    auto total = [&](int64_t d) {
      A t = rh * (to_acc(dy[d * a.dy.sd]) * to_acc(w_pre[d]) - to_acc(h[d * a.h.sd]) * rh * m1);
      return dh ? t + to_acc(dh[d * a.dh.sd]) : t;
    };
    if (w_post) {
      for (int64_t d = threadIdx.x; d < a.s.D; d += 256) {
        A u = total(d) * to_acc(w_post[d]);
        if (gate) u *= to_acc(gate[d * a.gate_sd]);
        m2 = fma_a(u, to_acc(b[d * a.b.sd]) * rb, m2);
      }
      m2 = block_sum(m2, sh) / D;
    }
    // dr may lie over dh and db over dy: each element is read before it is written
    for (int64_t d = threadIdx.x; d < a.s.D; d += 256) {
      const A t = total(d);
      A u = gate ? t * to_acc(gate[d * a.gate_sd]) : t;
      if (w_post) u = rb * (u * to_acc(w_post[d]) - to_acc(b[d * a.b.sd]) * rb * m2);
      dr[d * a.dr.sd] = from_acc<T, A>(alpha * t);
      db[d * a.db.sd] = from_acc<T, A>(u);
    }
  }
}

// The mean of dy w_pre hn of each row, for the column sums (which read dh and
// dy before k_norm_grad_rows may write over them).
template <typename T>
__global__ void __launch_bounds__(256) k_norm_grad_means(NormGradArgs a, typename AccOf<T>::type *means) {
  using A = typename AccOf<T>::type;
  __shared__ A sh[8];
  const T *w_pre = static_cast<const T *>(a.w_pre);
  for (int64_t row = blockIdx.x; row < a.s.rows(); row += gridDim.x) {
    const T *dy = row_ptr<T>(a.dy, row, a.s.L), *h = row_ptr<T>(a.h, row, a.s.L);
    const A rh = static_cast<const A *>(a.rstd_h)[row];
    A m = 0;
    for (int64_t d = threadIdx.x; d < a.s.D; d += 256)
      m = fma_a(to_acc(dy[d * a.dy.sd]) * to_acc(w_pre[d]), to_acc(h[d * a.h.sd]) * rh, m);
    m = block_sum(m, sh);
    if (threadIdx.x == 0) means[row] = m / (A)a.s.D;
  }
}

// Column sums: block (32, 8) takes 32 columns of one gate group; the 8 rows of
// threads split its rows and are added in order.  The weights' sums of the
// groups are added by one block walking over all groups in order.
template <typename T>
__global__ void __launch_bounds__(256) k_norm_grad_cols(NormGradArgs a, const typename AccOf<T>::type *means) {
  using A = typename AccOf<T>::type;
  __shared__ A sh[3][8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t d = (int64_t)blockIdx.x * 32 + lane;
  const bool ok = d < a.s.D;
  const T *w_pre = static_cast<const T *>(a.w_pre), *w_post = static_cast<const T *>(a.w_post);
  const int64_t groups = a.s.rows() / a.per;
  A p = 0, q = 0;  // dw_pre, dw_post
  for (int64_t g = 0; g < groups; ++g) {
    A e = 0;  // dgate
    const A gv = a.gate && ok ? to_acc(static_cast<const T *>(a.gate)[g * a.gate_sg + d * a.gate_sd]) : A(1);
    if (ok) {
      const A wp = to_acc(w_pre[d]), wo = w_post ? to_acc(w_post[d]) : A(1);
      for (int64_t row = g * a.per + warp; row < (g + 1) * a.per; row += 8) {
        const A rh = static_cast<const A *>(a.rstd_h)[row];
        const A rb = w_post ? static_cast<const A *>(a.rstd_b)[row] : A(1);
        const A dy = to_acc(row_ptr<T>(a.dy, row, a.s.L)[d * a.dy.sd]);
        const A hn = to_acc(row_ptr<T>(a.h, row, a.s.L)[d * a.h.sd]) * rh;
        const A bn = to_acc(row_ptr<T>(a.b, row, a.s.L)[d * a.b.sd]) * rb;
        A t = rh * (dy * wp - hn * means[row]);
        if (a.dh.p) t += to_acc(row_ptr<T>(a.dh, row, a.s.L)[d * a.dh.sd]);
        p = fma_a(dy, hn, p);
        q = fma_a(t * gv, bn, q);
        e = fma_a(t, bn * wo, e);
      }
    }
    if (a.d_gate) {
      __syncthreads();
      sh[2][warp][lane] = e;
      __syncthreads();
      if (warp == 0 && ok) {
        e = 0;
        for (int k = 0; k < 8; ++k) e += sh[2][k][lane];
        static_cast<A *>(a.d_gate)[g * a.gate_sg + d * a.gate_sd] = e;
      }
    }
  }
  sh[0][warp][lane] = p;
  sh[1][warp][lane] = q;
  __syncthreads();
  if (warp == 0 && ok) {
    p = q = 0;
    for (int k = 0; k < 8; ++k) {
      p += sh[0][k][lane];
      q += sh[1][k][lane];
    }
    if (a.d_w_pre) static_cast<A *>(a.d_w_pre)[d] = p;
    if (a.d_w_post) static_cast<A *>(a.d_w_post)[d] = q;
  }
}

// ---------------------------------------------------------------------------
// contiguous rows
// ---------------------------------------------------------------------------
// The V columns of a row that thread `tid` of TPR has in its n-th piece.
// They come in groups of G that are read at once, and start on a boundary of as
// many elements in every row, weight and gate row; the threads' groups lie side by
// side, so that a warp reads neighbouring elements.  G = V: whole pieces.  G = 2:
// rows of even width (16384 x 1634 float16, the gradient: 88 us, 216 with G = 1).
// G = 1: any alignment, width and stride.  (A thread's columns are the same in
// every row; a piece moved by each row's misalignment would not be, and its
// weights would be read 16 bytes apart.)
template <int V, int TPR, int G>
__device__ __forceinline__ int column(int tid, int n, int j) {
  return ((n * (V / G) + j / G) * TPR + tid) * G + j % G;
}

template <typename T, int V, int TPR, int G>
__device__ __forceinline__ Piece<T, V> fetch_cols(const T *x, int64_t sd, int tid, int n, int D) {
  Piece<T, V> p;
  if (G == V && column<V, TPR, V>(tid, n, 0) < D) {
    p = *reinterpret_cast<const Piece<T, V> *>(x + column<V, TPR, V>(tid, n, 0));
    return p;
  }
#pragma unroll
  for (int j = 0; j < V; j += G == V ? 1 : G) {
    const int d = column<V, TPR, G>(tid, n, j);
    if (G == 2 && G < V) {
      Vec<T, 2> w = {};
      if (d < D) w = *reinterpret_cast<const Vec<T, 2> *>(x + d);
      p.set(j, w.v[0]);
      p.set(j + 1, w.v[1]);
    } else {
      p.set(j, G < V && d < D ? x[d * sd] : (T)0.0f);
    }
  }
  return p;
}

template <typename T, typename A, int V, int TPR, int G>
__device__ __forceinline__ void load_cols(const T *x, int64_t sd, int tid, int n, int D, A *out) {
  fetch_cols<T, V, TPR, G>(x, sd, tid, n, D).widen(out);
}

template <typename T, typename A, int V, int TPR, int G>
__device__ __forceinline__ void store_cols(T *x, int64_t sd, int tid, int n, int D, const A *v) {
  if (G == V) {
    const int first = column<V, TPR, V>(tid, n, 0);
    if (first < D) {
      Piece<T, V> w;
      w.round(v);
      *reinterpret_cast<Piece<T, V> *>(x + first) = w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; j += G) {
      const int d = column<V, TPR, G>(tid, n, j);
      if (d >= D) continue;
      if (G == 2) {
        Vec<T, 2> w = {from_acc<T, A>(v[j]), from_acc<T, A>(v[j + G - 1])};
        *reinterpret_cast<Vec<T, 2> *>(x + d) = w;
      } else {
        x[d * sd] = from_acc<T, A>(v[j]);
      }
    }
  }
}

// Sums of N values over the TPR threads of a row, in every one of them.  sh
// holds one set for each warp; two sets alternate, so that one barrier a sum
// is enough.
template <typename A, int N, int TPR>
__device__ __forceinline__ void row_sum(A (&v)[N], A *sh) {
#pragma unroll
  for (int q = 16; q; q >>= 1)
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] += __shfl_xor_sync(~0u, v[j], q);
  if (TPR > 32) {
    constexpr int NW = TPR / 32;
    const int warp = threadIdx.x >> 5, first = warp / NW * NW, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int j = 0; j < N; ++j) sh[warp * N + j] = v[j];
    __syncthreads();
    // the lanes take a warp's sum each
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = lane < NW ? sh[(first + lane) * N + j] : A(0);
#pragma unroll
    for (int q = 16; q; q >>= 1)
      if (q < NW)
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += __shfl_xor_sync(~0u, v[j], q);
    if (NW < 32)
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = __shfl_sync(~0u, v[j], 0);
  }
}

// TPR threads a row, NV pieces of V columns a thread; the row stays in registers
// between the two sums.  Bound by its reads and writes (16384 x 4096 float16 with
// 16 gate rows: 101 us, 0.81 of a copy's rate); what is left is the two
// reductions a row, during which the block waits.
template <typename T, int TPR, int NV, int G>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_norm_vec(NormArgs a) {
  using A = typename AccOf<T>::type;
  using P = Pk<A>;
  constexpr int V = 16 / sizeof(T), BLOCK = TPR < 256 ? 256 : TPR, M = V / P::N;
  __shared__ A sh[2][BLOCK / 32];
  const int64_t row = (int64_t)blockIdx.x * (BLOCK / TPR) + threadIdx.x / TPR;
  const bool ok = row < a.s.rows();  // whole warps: a row has at least one
  const int64_t rr = ok ? row : 0;
  const int tid = threadIdx.x % TPR;
  const int D = ok ? (int)a.s.D : 0;
  const T *r = row_ptr<T>(a.r, rr, a.s.L), *b = row_ptr<T>(a.b, rr, a.s.L);
  const T *w_pre = static_cast<const T *>(a.w_pre), *w_post = static_cast<const T *>(a.w_post);
  const A eps = (A)a.eps, inv = A(1) / (A)a.s.D;
  Piece<T, V> br[NV], rr_[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    br[n] = fetch_cols<T, V, TPR, G>(b, a.b.sd, tid, n, D);
    rr_[n] = fetch_cols<T, V, TPR, G>(r, a.r.sd, tid, n, D);
  }
  P h[NV][M];
  A f[V];
  auto sum_of_squares = [&]() {
    P q = P::all(A(0));
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int j = 0; j < M; ++j) q = pfma(h[n][j], h[n][j], q);
    return q.sum();
  };
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    br[n].widen(f);
#pragma unroll
    for (int j = 0; j < M; ++j) h[n][j] = P::from(f + j * P::N);
  }
  A rb = 1;
  if (w_post) {
    A q[1] = {sum_of_squares()};
    row_sum<A, 1, TPR>(q, sh[0]);
    rb = rsqrt_a(q[0] * inv + eps);
    const P prb = P::all(rb);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      load_cols<T, A, V, TPR, G>(w_post, 1, tid, n, D, f);
#pragma unroll
      for (int j = 0; j < M; ++j) h[n][j] = pmul(pmul(h[n][j], prb), P::from(f + j * P::N));
    }
  }
  const P alpha = P::all((A)a.alpha);
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    if (a.gate) {
      load_cols<T, A, V, TPR, G>(static_cast<const T *>(a.gate) + (int64_t)((uint32_t)rr / (uint32_t)a.per) * a.gate_sg, a.gate_sd, tid, n, D, f);
#pragma unroll
      for (int j = 0; j < M; ++j) h[n][j] = pmul(h[n][j], P::from(f + j * P::N));
    }
    rr_[n].widen(f);
#pragma unroll
    for (int j = 0; j < M; ++j) h[n][j] = pfma(alpha, P::from(f + j * P::N), h[n][j]);
  }
  A q[1] = {sum_of_squares()};
  row_sum<A, 1, TPR>(q, sh[1]);
  const A rh = rsqrt_a(q[0] * inv + eps);
  if (!ok) return;
  const P prh = P::all(rh);
  T *ho = row_ptr<T>(a.h, rr, a.s.L), *yo = row_ptr<T>(a.y, rr, a.s.L);
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    A y[V];
    load_cols<T, A, V, TPR, G>(w_pre, 1, tid, n, D, f);
#pragma unroll
    for (int j = 0; j < M; ++j) pmul(pmul(h[n][j], prh), P::from(f + j * P::N)).to(y + j * P::N);
    store_cols<T, A, V, TPR, G>(yo, a.y.sd, tid, n, D, y);
#pragma unroll
    for (int j = 0; j < M; ++j) h[n][j].to(f + j * P::N);
    store_cols<T, A, V, TPR, G>(ho, a.h.sd, tid, n, D, f);
  }
  if (tid == 0) {
    if (a.rstd_h) static_cast<A *>(a.rstd_h)[row] = rh;
    if (a.rstd_b) static_cast<A *>(a.rstd_b)[row] = rb;
  }
}

// How the rows of a gradient call are dealt out: `parts` units a gate row,
// unit u = (group u / parts, part u % parts); a block takes units u, u + grid,
// ...  The column sums of a block's rows go to its own row of the partial
// arrays, a unit's gate sums to the unit's row, and k_norm_grad_join adds them
// in order.
struct GradPlan {
  int64_t groups, parts, per;
  void *pre, *post;  // [grid][D]
  void *gate;        // [groups * parts][D], or d_gate itself where parts = 1
  int64_t gate_sd, gate_su;
};

// Which rows a unit has.
__device__ __forceinline__ void unit_rows(const GradPlan &p, int64_t u, int64_t &r0, int64_t &r1) {
  const int64_t g = u / p.parts, part = u - g * p.parts;
  r0 = g * p.per + part * p.per / p.parts;
  r1 = g * p.per + (part + 1) * p.per / p.parts;
}

// V columns of a row's gradient, in two steps around the row's sums.  With
//   u = d_y w_pre,  q = d_h + rs_h u,  f = gate w_post,  e = f b
// and the sums s0 = sum u h, s1 = sum q e, s2 = sum h e over the row,
//   m1 = rs_h mean(d_y w_pre hn) = rs_h^2 s0 / D,  t = q - m1 hn,
//   mean(u w_post bn) = rs_b (s1 - m1 rs_h s2) / D:
// one reduction a row.  sum t bn is what the gradients of the gate (times
// w_post) and of w_post (times gate) have in common while the gate row stays.
template <typename A, int V>
struct GradCols {
  using P = Pk<A>;
  static constexpr int M = V / P::N;
  P q[M], h[M], b[M], dy[M];
  __device__ __forceinline__ void take(const A (&dhv)[V], const A (&dyv)[V], const A (&hv)[V], const A (&bv)[V],
                                       const P (&wp)[M], A rh) {
    const P prh = P::all(rh);
#pragma unroll
    for (int j = 0; j < M; ++j) {
      dy[j] = P::from(dyv + j * P::N);
      h[j] = P::from(hv + j * P::N);
      b[j] = P::from(bv + j * P::N);
      q[j] = pfma(prh, pmul(dy[j], wp[j]), P::from(dhv + j * P::N));
    }
  }
  __device__ __forceinline__ void sums(const P (&wp)[M], const P (&f)[M], A (&s)[3]) const {
    P s0 = P::all(A(0)), s1 = s0, s2 = s0;
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const P e = pmul(f[j], b[j]);
      s0 = pfma(pmul(dy[j], wp[j]), h[j], s0);
      s1 = pfma(q[j], e, s1);
      s2 = pfma(h[j], e, s2);
    }
    s[0] = s0.sum();
    s[1] = s1.sum();
    s[2] = s2.sum();
  }
  // s: the row's sums; adds to pre and tb, leaves the gradients in dr and db.
  __device__ __forceinline__ void finish(const A (&s)[3], A inv, A rh, A rb, A alpha, bool post, const P (&f)[M],
                                         P (&pre)[M], P (&tb)[M], A (&dr)[V], A (&db)[V]) const {
    // (rs_h is put to h before the mean, and to s2: rs_h^3 alone may be beyond the type)
    const A m1 = rh * (s[0] * inv) * rh;
    const P nm1 = P::all(-m1), prh = P::all(rh), prb = P::all(rb), pal = P::all(alpha);
    const P nm2 = P::all(post ? -(rb * inv) * (s[1] - m1 * (rh * s[2])) : A(0));
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const P hn = pmul(h[j], prh), t = pfma(hn, nm1, q[j]), bn = pmul(b[j], prb);
      pre[j] = pfma(dy[j], hn, pre[j]);
      tb[j] = pfma(t, bn, tb[j]);
      pmul(pal, t).to(dr + j * P::N);
      P x = pmul(t, f[j]);
      if (post) x = pmul(pfma(bn, nm2, x), prb);
      x.to(db + j * P::N);
    }
  }
};

// The operands that stay while the gate row does: w_pre, and f = gate w_post.
template <typename T, typename A, int V, int TPR, int G>
__device__ __forceinline__ void load_operands(const NormGradArgs &a, int64_t row, int tid, int n, int D, A (&wo)[V], A (&g)[V],
                                              Pk<A> (&f)[V / Pk<A>::N]) {
#pragma unroll
  for (int j = 0; j < V; ++j) wo[j] = g[j] = A(1);
  if (a.w_post) load_cols<T, A, V, TPR, G>(static_cast<const T *>(a.w_post), 1, tid, n, D, wo);
  if (a.gate)
    load_cols<T, A, V, TPR, G>(static_cast<const T *>(a.gate) + (int64_t)((uint32_t)row / (uint32_t)a.per) * a.gate_sg, a.gate_sd, tid, n, D, g);
#pragma unroll
  for (int j = 0; j < V / Pk<A>::N; ++j)
    f[j] = pmul(Pk<A>::from(wo + j * Pk<A>::N), Pk<A>::from(g + j * Pk<A>::N));
}

// Adds the RPB sub-blocks' columns into the first one's, in order.
template <typename A, int V, int TPR, int RPB>
__device__ __forceinline__ void add_subs(A (&acc)[V], A (*join)[V]) {
  if (RPB == 1) return;
  const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) join[threadIdx.x][j] = acc[j];
  __syncthreads();
  if (sub == 0)
    for (int q = 1; q < RPB; ++q)
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += join[q * TPR + tid][j];
}

template <typename A, int V, int TPR, int G>
__device__ __forceinline__ void store_sums(A *dst, int64_t sd, int tid, int n, int D, const A (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int d = column<V, TPR, G>(tid, n, j);
    if (d < D) dst[d * sd] = v[j];
  }
}

// V columns a thread, TPR threads a row; the column sums stay in registers.  The
// next row is under way while one is worked on.  Both means of a row come from
// one reduction of three sums: the mean of the post norm's gradient splits into
// two that do not wait for the other mean.  16384 x 4096 float16 with 16 gate rows
// in 186 us, 0.66 of a copy's rate: its registers leave one block of 512 threads
// an SM, which waits at the reduction's barrier.  Rows of odd width are
// read an element at a time: 5000 x 1001 float32 in 36.5 us, 0.50.  (1024 threads,
// for rows that the ring cannot take, have 64 registers each and spill up to 488
// bytes.)
template <typename T, int TPR, int G>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, TPR > 512 ? 1 : TPR > 256 || sizeof(T) == 8 ? 1 : 2)
    k_norm_grad_vec(NormGradArgs a, GradPlan plan) {
  using A = typename AccOf<T>::type;
  using P = Pk<A>;
  constexpr int V = 16 / sizeof(T), BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR, M = V / P::N;
  __shared__ A sh[2][BLOCK / 32 * 3];
  __shared__ A join[RPB > 1 ? BLOCK : 1][V];
  const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int D = (int)a.s.D;
  const bool post = a.w_post != nullptr;
  const A alpha = (A)a.alpha, inv = A(1) / (A)a.s.D;
  P wp[M], f[M], pre[M], pst[M];
  A wo[V], g[V], c[V];
  load_cols<T, A, V, TPR, G>(static_cast<const T *>(a.w_pre), 1, tid, 0, D, c);
#pragma unroll
  for (int j = 0; j < M; ++j) {
    wp[j] = P::from(c + j * P::N);
    pre[j] = pst[j] = P::all(A(0));
  }
  int flip = 0;
  for (int64_t u = blockIdx.x; u < plan.groups * plan.parts; u += gridDim.x) {
    int64_t r0, r1;
    unit_rows(plan, u, r0, r1);
    load_operands<T, A, V, TPR, G>(a, r0, tid, 0, D, wo, g, f);
    P tb[M];
#pragma unroll
    for (int j = 0; j < M; ++j) tb[j] = P::all(A(0));
    struct {
      Piece<T, V> dh, dy, h, b;
      A rh, rb;
    } cur, next;
    auto fetch = [&](int64_t rr, auto &x) {
      const bool ok = rr + sub < r1;
      const int64_t row = ok ? rr + sub : r0;
      const int n = ok ? D : 0;
      if (a.dh.p) x.dh = fetch_cols<T, V, TPR, G>(row_ptr<T>(a.dh, row, a.s.L), a.dh.sd, tid, 0, n);
      x.dy = fetch_cols<T, V, TPR, G>(row_ptr<T>(a.dy, row, a.s.L), a.dy.sd, tid, 0, n);
      x.h = fetch_cols<T, V, TPR, G>(row_ptr<T>(a.h, row, a.s.L), a.h.sd, tid, 0, n);
      x.b = fetch_cols<T, V, TPR, G>(row_ptr<T>(a.b, row, a.s.L), a.b.sd, tid, 0, n);
      x.rh = ok ? static_cast<const A *>(a.rstd_h)[row] : A(0);
      x.rb = post && ok ? static_cast<const A *>(a.rstd_b)[row] : A(1);
    };
    if (r0 < r1) fetch(r0, cur);
    for (int64_t rr = r0; rr < r1; rr += RPB) {
      if (rr + RPB < r1) fetch(rr + RPB, next);
      A dh[V], dy[V], h[V], b[V], s[3];
#pragma unroll
      for (int j = 0; j < V; ++j) dh[j] = A(0);
      if (a.dh.p) cur.dh.widen(dh);
      cur.dy.widen(dy);
      cur.h.widen(h);
      cur.b.widen(b);
      GradCols<A, V> p;
      p.take(dh, dy, h, b, wp, cur.rh);
      p.sums(wp, f, s);
      row_sum<A, 3, TPR>(s, sh[flip]);
      flip ^= 1;
      p.finish(s, inv, cur.rh, cur.rb, alpha, post, f, pre, tb, dh, dy);
      if (rr + sub < r1) {
        store_cols<T, A, V, TPR, G>(row_ptr<T>(a.dr, rr + sub, a.s.L), a.dr.sd, tid, 0, D, dh);
        store_cols<T, A, V, TPR, G>(row_ptr<T>(a.db, rr + sub, a.s.L), a.db.sd, tid, 0, D, dy);
      }
      cur = next;
    }
    // (read again: they are wanted once a unit only)
    load_operands<T, A, V, TPR, G>(a, r0, tid, 0, D, wo, g, f);
#pragma unroll
    for (int j = 0; j < M; ++j) {
      pst[j] = pfma(P::from(g + j * P::N), tb[j], pst[j]);
      pmul(P::from(wo + j * P::N), tb[j]).to(c + j * P::N);
    }
    if (plan.gate) {
      add_subs<A, V, TPR, RPB>(c, join);
      if (sub == 0) store_sums<A, V, TPR, G>(static_cast<A *>(plan.gate) + u * plan.gate_su, plan.gate_sd, tid, 0, D, c);
    }
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    A *dst = static_cast<A *>(w ? plan.post : plan.pre);
    if (!dst) continue;
#pragma unroll
    for (int j = 0; j < M; ++j) (w ? pst[j] : pre[j]).to(c + j * P::N);
    add_subs<A, V, TPR, RPB>(c, join);
    if (sub == 0) store_sums<A, V, TPR, G>(dst + (int64_t)blockIdx.x * D, 1, tid, 0, D, c);
  }
}

// The same for wider rows: a cluster of CL blocks divides the columns, and the
// rows come in by bulk copies through a ring of stages, so that several rows are
// under way while one is worked on.  A row stays in shared memory: it is read
// once for its sums and once more for its gradients, which leaves the registers
// to the column sums of NV pieces a thread and allows two blocks on an SM, whose
// barriers then overlap.  The rows' sums go to the other blocks by asynchronous
// stores that count on a barrier there.
//   A block takes 512 pieces, the last one what is left, so the time is that of a
// row of full blocks: 16384 rows of 4160, 5120, 6144 and 8192 float16 columns take
// 434, 430, 427 and 429 us (0.29 to 0.57 of a copy's rate), of 4096 float32 251 us
// (0.98), without gate rows.  8192 float16 and 4096 float32 columns have the same
// bytes and the same number of exchanges: what the first wait for is its
// instructions.  They are 1.63 times as many (an element is widened and
// multiplied twice, and 72 bytes a thread are spilled), issued at the same rate,
// 41% and 43% of the slots, with 16 warps an SM to hide their latency.  One piece
// a thread and twice the blocks took 1.4 times as long for 4096 float32, 1.2 for
// 8192 and 1.3 for 5120 float16; k_norm_grad_vec with 1024 threads 1.45, 1.2 and
// 1.06.
constexpr uint64_t kRingWaitNs = 1000000000ull;  // 1 s
constexpr int kRingWaitCode = 6;
constexpr int kRingStages = 3;
constexpr int kRingCluster = 8;
constexpr int kRingPieces = 2;  // of 16 bytes a thread

template <typename A>
struct RingShared {
  uint64_t full[kRingStages], joined[2];
  A part[2][32][4];                             // the warps' sums
  alignas(16) A other[2][kRingCluster][4];      // the blocks' sums, sent 16 bytes at a time
  int abort;
};

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_addr(dst)),
               "l"(src), "r"(bytes), "r"(smem_addr(bar))
               : "memory");
}

// 16 bytes to the same place of block `rank` of the cluster, counted on its barrier.
__device__ __forceinline__ void send16(const void *at, const uint64_t *bar, int rank, uint64_t lo, uint64_t hi) {
  uint32_t d, m;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_addr(at)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(smem_addr(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(d), "l"(lo),
               "l"(hi), "r"(m)
               : "memory");
}

constexpr int kRingThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kRingThreads, 2) k_norm_grad_ring(NormGradArgs a, GradPlan plan, Control *control) {
  constexpr int TPR = kRingThreads, NV = kRingPieces;
  using A = typename AccOf<T>::type;
  using P = Pk<A>;
  constexpr int V = 16 / sizeof(T), M = V / P::N, NW = TPR / 32, N = kRingStages;
  extern __shared__ __align__(128) unsigned char ring[];  // [stage][dy, h, b, dh][NV * TPR * 16 bytes]
  __shared__ RingShared<A> sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int CL = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t cid = blockIdx.x / CL, nclusters = gridDim.x / CL, units = plan.groups * plan.parts;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tid = threadIdx.x;
  constexpr int W = NV * TPR * V, ROW = NV * TPR * 16;  // columns of a block, bytes of its part of a row
  const int c0 = rank * W;
  const int D = (int)a.s.D - c0 < W ? (int)a.s.D - c0 : W;
  const bool post = a.w_post != nullptr;
  if (tid == 0) {
    for (int i = 0; i < N; ++i) mbar_init(&sh.full[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&sh.joined[i], 1);
    sh.abort = 0;
    mbar_init_fence();
  }
  // what no copy writes
  for (int i = tid; i < N * 4 * NV * TPR; i += TPR)
    if (i % (NV * TPR) * V >= D) reinterpret_cast<uint4 *>(ring)[i] = make_uint4(0, 0, 0, 0);
  cluster.sync();
  // thread 0 walks ahead over the rows of this block's units and issues their copies
  int64_t fu = cid, frow = 0, fend = 0;
  int issued = 0;
  if (fu < units) unit_rows(plan, fu, frow, fend);
  auto issue = [&]() {
    while (frow >= fend) {
      fu += nclusters;
      if (fu >= units) return;
      unit_rows(plan, fu, frow, fend);
    }
    uint64_t *bar = &sh.full[issued % N];
    unsigned char *st = ring + (size_t)(issued % N) * 4 * ROW;
    const uint32_t bytes = D * (uint32_t)sizeof(T);
    mbar_arrive_expect_tx(bar, bytes * (a.dh.p ? 4 : 3));
    bulk_load(st, row_ptr<T>(a.dy, frow, a.s.L) + c0, bytes, bar);
    bulk_load(st + ROW, row_ptr<T>(a.h, frow, a.s.L) + c0, bytes, bar);
    bulk_load(st + 2 * ROW, row_ptr<T>(a.b, frow, a.s.L) + c0, bytes, bar);
    if (a.dh.p) bulk_load(st + 3 * ROW, row_ptr<T>(a.dh, frow, a.s.L) + c0, bytes, bar);
    ++frow;
    ++issued;
  };
  if (tid == 0)
    for (int i = 0; i < N && fu < units; ++i) issue();

  const A alpha = (A)a.alpha, inv = A(1) / (A)a.s.D;
  NormGradArgs slice = a;  // operands from this block's first column on
  slice.w_pre = static_cast<const T *>(a.w_pre) + c0;
  if (a.w_post) slice.w_post = static_cast<const T *>(a.w_post) + c0;
  if (a.gate) slice.gate = static_cast<const T *>(a.gate) + c0;
  Piece<T, V> wraw[NV];
  P f[NV][M], pre[NV][M], tb[NV][M];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    wraw[v] = fetch_cols<T, V, TPR, V>(static_cast<const T *>(slice.w_pre), 1, tid, v, D);
#pragma unroll
    for (int j = 0; j < M; ++j) pre[v][j] = P::all(A(0));
  }
  int n = 0, slot = 0, flip = 0;
  uint32_t phase = 0, joined = 0;
  bool dead = false, first = true;
  for (int64_t u = cid; u < units; u += nclusters) {
    int64_t r0, r1;
    unit_rows(plan, u, r0, r1);
    A wo[V], g[V], c[V];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      load_operands<T, A, V, TPR, V>(slice, r0, tid, v, D, wo, g, f[v]);
#pragma unroll
      for (int j = 0; j < M; ++j) tb[v][j] = P::all(A(0));
    }
    A rh_next = r0 < r1 ? static_cast<const A *>(a.rstd_h)[r0] : A(0);
    A rb_next = r0 < r1 && post ? static_cast<const A *>(a.rstd_b)[r0] : A(1);
    for (int64_t row = r0; row < r1; ++row, ++n) {
      const A rh = rh_next, rb = rb_next;
      if (row + 1 < r1) {
        rh_next = static_cast<const A *>(a.rstd_h)[row + 1];
        if (post) rb_next = static_cast<const A *>(a.rstd_b)[row + 1];
      }
      // once given up, the warps go on without waiting: all of them reach the barriers
      dead = dead || !mbar_wait_warp(&sh.full[slot], phase, &sh.abort, control, kRingWaitCode, kRingWaitNs);
      const unsigned char *st = ring + (size_t)slot * 4 * ROW;
      A s[3] = {A(0), A(0), A(0)};
      GradCols<A, V> p;
      P wp[M];
      auto read = [&](int v) {
        A dh[V], dy[V], h[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) dh[j] = A(0);
        wraw[v].widen(dy);
#pragma unroll
        for (int j = 0; j < M; ++j) wp[j] = P::from(dy + j * P::N);
        // (beyond the row's end a stage holds zeros)
        const Piece<T, V> *at = reinterpret_cast<const Piece<T, V> *>(st) + v * TPR + tid;
        at[0].widen(dy);
        at[NV * TPR].widen(h);
        at[2 * NV * TPR].widen(b);
        if (a.dh.p) at[3 * NV * TPR].widen(dh);
        p.take(dh, dy, h, b, wp, rh);
      };
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        A part[3];
        read(v);
        p.sums(wp, f[v], part);
#pragma unroll
        for (int j = 0; j < 3; ++j) s[j] += part[j];
      }
#pragma unroll
      for (int q = 16; q; q >>= 1)
#pragma unroll
        for (int j = 0; j < 3; ++j) s[j] += __shfl_xor_sync(~0u, s[j], q);
      if (lane == 0)
#pragma unroll
        for (int j = 0; j < 3; ++j) sh.part[flip][warp][j] = s[j];
      __syncthreads();
      // the row before has been read to the end by everyone: its stage is free
      if (tid == 0 && n > 0 && fu < units && !dead) issue();
#pragma unroll
      for (int j = 0; j < 3; ++j) s[j] = lane < NW ? sh.part[flip][lane][j] : A(0);
#pragma unroll
      for (int q = NW / 2; q; q >>= 1)
#pragma unroll
        for (int j = 0; j < 3; ++j) s[j] += __shfl_xor_sync(~0u, s[j], q);
#pragma unroll
      for (int j = 0; j < 3; ++j) s[j] = __shfl_sync(~0u, s[j], 0);
      if (warp == 0 && lane < CL) {
        if (lane == 0) mbar_arrive_expect_tx(&sh.joined[flip], CL * 4 * (uint32_t)sizeof(A));
        // the block's sums to every block, its own included
        if constexpr (sizeof(A) == 4) {
          send16(&sh.other[flip][rank][0], &sh.joined[flip], lane, pack2(s[0], s[1]), pack2(s[2], 0.0f));
        } else {
          send16(&sh.other[flip][rank][0], &sh.joined[flip], lane, __double_as_longlong(s[0]),
                 __double_as_longlong(s[1]));
          send16(&sh.other[flip][rank][2], &sh.joined[flip], lane, __double_as_longlong(s[2]), 0);
        }
      }
      __syncwarp();
      dead = dead || !mbar_wait_warp(&sh.joined[flip], joined, &sh.abort, control, kRingWaitCode, kRingWaitNs);
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        s[j] = A(0);
        for (int q = 0; q < CL; ++q) s[j] += sh.other[flip][q][j];
      }
      joined ^= (uint32_t)flip;  // both barriers have had a phase
      flip ^= 1;
      asm volatile("" ::: "memory");  // read again, not kept
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        A dr[V], db[V];
        read(v);
        p.finish(s, inv, rh, rb, alpha, post, f[v], pre[v], tb[v], dr, db);
        store_cols<T, A, V, TPR, V>(row_ptr<T>(a.dr, row, a.s.L) + c0, 1, tid, v, D, dr);
        store_cols<T, A, V, TPR, V>(row_ptr<T>(a.db, row, a.s.L) + c0, 1, tid, v, D, db);
      }
      if (++slot == N) {
        slot = 0;
        phase ^= 1u;
      }
    }
    // (wo and g read again rather than kept over the rows; the sums of w_post go
    // straight to this block's row of the partial sums)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      load_operands<T, A, V, TPR, V>(slice, r0, tid, v, D, wo, g, f[v]);
      if (plan.post && column<V, TPR, V>(tid, v, 0) < D) {
        A *dst = static_cast<A *>(plan.post) + cid * a.s.D + c0 + column<V, TPR, V>(tid, v, 0);
#pragma unroll
        for (int j = 0; j < M; ++j) pmul(P::from(g + j * P::N), tb[v][j]).to(c + j * P::N);
#pragma unroll
        for (int j = 0; j < V; ++j) dst[j] = first ? c[j] : dst[j] + c[j];
      }
      if (plan.gate) {
#pragma unroll
        for (int j = 0; j < M; ++j) pmul(P::from(wo + j * P::N), tb[v][j]).to(c + j * P::N);
        store_sums<A, V, TPR, V>(static_cast<A *>(plan.gate) + u * plan.gate_su + c0 * plan.gate_sd, plan.gate_sd, tid, v,
                                    D, c);
      }
    }
    first = false;
  }
  if (plan.pre) {
    A c[V];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int j = 0; j < M; ++j) pre[v][j].to(c + j * P::N);
      store_sums<A, V, TPR, V>(static_cast<A *>(plan.pre) + cid * a.s.D + c0, 1, tid, v, D, c);
    }
  }
  // given up: the copies in flight land before the block may end
  if (dead && tid == 0)
    for (int q = issued > N ? issued - N : 0; q < issued; ++q)
      mbar_wait_bounded(&sh.full[q % N], (uint32_t)(q / N) & 1u, kRingWaitNs);
  __syncwarp();
  cluster.sync();  // no block leaves while another may still write to it
}

// Column sums of `n` partial rows: a block takes 32 W columns, its 8 warps split
// the rows and are added in order.
template <typename A>
struct JoinArgs {
  const A *src[3];
  A *dst[3];
  int64_t n[3], sd[3], sg[3];  // rows a sum, strides of dst along the row and over its groups
  int64_t D;
};

template <typename A, int W>
__global__ void __launch_bounds__(256) k_norm_grad_join(JoinArgs<A> a) {
  __shared__ Vec<A, W> sh[8][32];
  // blockIdx.y: 0 pre, 1 post, 2 + g gate row g
  const int w = blockIdx.y < 2 ? blockIdx.y : 2;
  const int64_t g = w == 2 ? blockIdx.y - 2 : 0;
  if (!a.dst[w]) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t d = ((int64_t)blockIdx.x * 32 + lane) * W, n = a.n[w];
  Vec<A, W> s;
#pragma unroll
  for (int j = 0; j < W; ++j) s.v[j] = A(0);
  if (d < a.D) {  // W divides D
    const A *p = a.src[w] + g * n * a.D + d;
    constexpr int U = 12;  // rows in flight
    for (int64_t i = warp; i < n; i += 8 * U) {
      Vec<A, W> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + 8 * u < n) x[u] = *reinterpret_cast<const Vec<A, W> *>(p + (i + 8 * u) * a.D);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + 8 * u < n)
#pragma unroll
          for (int j = 0; j < W; ++j) s.v[j] += x[u].v[j];
    }
  }
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && d < a.D)
#pragma unroll
    for (int j = 0; j < W; ++j) {
      for (int q = 1; q < 8; ++q) s.v[j] += sh[q][lane].v[j];
      a.dst[w][(d + j) * a.sd[w] + g * a.sg[w]] = s.v[j];
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Whether the rows of `v` are contiguous and start on boundaries of g elements
// (the width is checked once, for all of them).
template <typename T>
static bool whole_rows(const Rows &v, int g) {
  return v.sd == 1 && aligned_to<char>(v.p, g * (int)sizeof(T)) && v.sl % g == 0 && v.so % g == 0;
}
// Weights and gate rows too.
template <typename T>
static bool whole_weights(const void *w_pre, const void *w_post, const void *gate, int64_t sd, int64_t sg, int g) {
  const int bytes = g * (int)sizeof(T);
  return aligned_to<char>(w_pre, bytes) && (!w_post || aligned_to<char>(w_post, bytes)) &&
         (!gate || (aligned_to<char>(gate, bytes) && sd == 1 && sg % g == 0));
}
// Elements that are read at once: a piece, two, or one.
template <typename T, typename Fits>
static int granule(int64_t D, Fits fits) {
  constexpr int V = 16 / sizeof(T);
  return D % V == 0 && fits(V) ? V : D % 2 == 0 && fits(2) ? 2 : 1;
}

template <typename T, int TPR, int NV>
static acd_status launch_norm_vec(const NormArgs &a, int g, cudaStream_t s) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR, V = 16 / sizeof(T);
  const int64_t grid = (a.s.rows() + RPB - 1) / RPB;
  auto kern = k_norm_vec<T, TPR, NV, 1>;
  if (g == V)
    kern = k_norm_vec<T, TPR, NV, V>;
  else if (g == 2)
    kern = k_norm_vec<T, TPR, NV, 2>;
  kern<<<(unsigned)grid, BLOCK, 0, s>>>(a);
  return ACD_OK;
}

template <typename T>
static acd_status launch_norm(acd_ctx *ctx, const NormArgs &a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int g = granule<T>(a.s.D, [&](int n) {
    return whole_rows<T>(a.r, n) && whole_rows<T>(a.b, n) && whole_rows<T>(a.h, n) && whole_rows<T>(a.y, n) &&
           whole_weights<T>(a.w_pre, a.w_post, a.gate, a.gate_sd, a.gate_sg, n);
  });
  const int64_t pieces = (a.s.D + V - 1) / V;
  // (Rows across the lanes come here too, G = 1: each element of a warp's lies in
  // a sector of its own.  16384 x 4096 float16 with axis = 2 takes 1653 us, the
  // gradient 11250 us, against 101 and 186 us along the first axis.)
  if (pieces <= 4096) {
    // A warp a row up to three pieces a lane, whose sums need no barrier, then
    // one to four pieces a thread.  16384 rows of float16 with a warp or 128
    // threads: 64 pieces 16.4 or 24.1 us, 128 pieces 33.5 or 29.0 us; 512 pieces
    // with 128 threads 128 us, with 256 101 us, with 512 113 us.
    if (pieces <= 32) return launch_norm_vec<T, 32, 1>(a, g, s);
    if (pieces <= 64) return launch_norm_vec<T, 32, 2>(a, g, s);
    if (pieces <= 96) return launch_norm_vec<T, 32, 3>(a, g, s);
    if (pieces <= 128) return launch_norm_vec<T, 128, 1>(a, g, s);
    if (pieces <= 256) return launch_norm_vec<T, 128, 2>(a, g, s);
    if (pieces <= 384) return launch_norm_vec<T, 128, 3>(a, g, s);
    if (pieces <= 512) return launch_norm_vec<T, 256, 2>(a, g, s);
    if (pieces <= 768) return launch_norm_vec<T, 256, 3>(a, g, s);
    if (pieces <= 1024) return launch_norm_vec<T, 512, 2>(a, g, s);
    if (pieces <= 1536) return launch_norm_vec<T, 512, 3>(a, g, s);
    if (pieces <= 2048) return launch_norm_vec<T, 512, 4>(a, g, s);
    return launch_norm_vec<T, 1024, 4>(a, g, s);
  }
  const int grid = persistent_grid(ctx, k_norm_rows<T>, 256, 0, a.s.rows());
  k_norm_rows<T><<<grid, 256, 0, s>>>(a);
  return ACD_OK;
}

// Deals the rows out to `grid` blocks (or clusters) that take `sub` rows at a
// time, runs `go` with the plan and joins the column sums.
template <typename A, typename Go>
static acd_status run_norm_grad(acd_ctx *ctx, const NormGradArgs &a, int64_t grid, int sub, cudaStream_t s, Go go) {
  const int64_t rows = a.s.rows(), D = a.s.D;
  GradPlan p{};
  p.per = a.per;
  p.groups = rows / a.per;
  p.parts = grid / p.groups;
  if (p.parts > (p.per + sub - 1) / sub) p.parts = (p.per + sub - 1) / sub;
  if (p.parts < 1) p.parts = 1;
  if (grid > p.groups * p.parts) grid = p.groups * p.parts;
  const bool gate_part = a.d_gate && p.parts > 1;
  const size_t cols = sizeof(A) * (size_t)D;
  void *scratch;
  ACD_TRY(get_scratch(ctx, cols * (2 * grid + (gate_part ? p.groups * p.parts : 0)), s, &scratch));
  A *pre = static_cast<A *>(scratch), *post = pre + grid * D, *gate = post + grid * D;
  p.pre = a.d_w_pre ? pre : nullptr;
  p.post = a.d_w_post ? post : nullptr;
  p.gate = a.d_gate ? (gate_part ? gate : a.d_gate) : nullptr;
  p.gate_sd = gate_part ? 1 : a.gate_sd;
  p.gate_su = gate_part ? D : a.gate_sg;
  ACD_TRY(go(grid, p));
  JoinArgs<A> j{};
  j.D = D;
  j.src[0] = pre;
  j.src[1] = post;
  j.src[2] = gate;
  j.dst[0] = static_cast<A *>(a.d_w_pre);
  j.dst[1] = static_cast<A *>(a.d_w_post);
  j.dst[2] = gate_part ? static_cast<A *>(a.d_gate) : nullptr;
  j.n[0] = j.n[1] = grid;
  j.n[2] = p.parts;
  j.sd[0] = j.sd[1] = 1;
  j.sd[2] = a.gate_sd;
  j.sg[2] = a.gate_sg;
  if (j.dst[0] || j.dst[1] || j.dst[2]) {
    const unsigned rows_y = (unsigned)(2 + (gate_part ? p.groups : 0));
    if (D % 2 == 0)
      k_norm_grad_join<A, 2><<<dim3((unsigned)((D / 2 + 31) / 32), rows_y), 256, 0, s>>>(j);
    else
      k_norm_grad_join<A, 1><<<dim3((unsigned)((D + 31) / 32), rows_y), 256, 0, s>>>(j);
  }
  return ACD_OK;
}

template <typename T, int TPR>
static acd_status launch_norm_grad_vec(acd_ctx *ctx, const NormGradArgs &a, int g, cudaStream_t s) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR, V = 16 / sizeof(T);
  auto kern = k_norm_grad_vec<T, TPR, 1>;
  if constexpr (TPR <= 512)  // wider whole rows go through the ring
    if (g == V) kern = k_norm_grad_vec<T, TPR, V>;
  if constexpr (V > 2)
    if (g == 2) kern = k_norm_grad_vec<T, TPR, 2>;
  const int64_t grid = (int64_t)ctx->sm_count * resident_blocks(reinterpret_cast<const void *>(kern), BLOCK, 0);
  return run_norm_grad<typename AccOf<T>::type>(ctx, a, grid, BLOCK / TPR, s, [&](int64_t blocks, const GradPlan &p) {
    kern<<<(unsigned)blocks, BLOCK, 0, s>>>(a, p);
    return ACD_OK;
  });
}

template <typename T>
static acd_status launch_norm_grad_ring(acd_ctx *ctx, const NormGradArgs &a, int CL, cudaStream_t s) {
  auto kern = k_norm_grad_ring<T>;
  const int dyn = kRingStages * 4 * kRingPieces * kRingThreads * 16;
  ACD_TRY(allow_smem(ctx, reinterpret_cast<const void *>(kern), dyn));
  return run_norm_grad<typename AccOf<T>::type>(
      ctx, a, (int64_t)ctx->sm_count * 2 / CL, 1, s, [&](int64_t clusters, const GradPlan &p) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(clusters * CL), 1, 1);
        cfg.blockDim = dim3(kRingThreads, 1, 1);
        cfg.dynamicSmemBytes = dyn;
        cfg.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = CL;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        ACD_CUDA(cudaLaunchKernelEx(&cfg, kern, a, p, ctx->control));
        return ACD_OK;
      });
}

template <typename T>
static acd_status launch_norm_grad(acd_ctx *ctx, const NormGradArgs &a, cudaStream_t s) {
  using A = typename AccOf<T>::type;
  constexpr int V = 16 / sizeof(T);
  const int g = granule<T>(a.s.D, [&](int n) {
    return whole_rows<T>(a.dr, n) && whole_rows<T>(a.db, n) && (!a.dh.p || whole_rows<T>(a.dh, n)) &&
           whole_rows<T>(a.dy, n) && whole_rows<T>(a.h, n) && whole_rows<T>(a.b, n) &&
           whole_weights<T>(a.w_pre, a.w_post, a.gate, a.gate_sd, a.gate_sg, n);
  });
  const int64_t pieces = (a.s.D + V - 1) / V;
  // Up to 512 pieces of 16 bytes a row a block keeps the row in registers, one
  // piece a thread (16384 rows of float16: 256 pieces 94 us, 512 pieces 186 us; a
  // single block of the ring 113 and 207 us); see k_norm_grad_ring for wider rows.
  constexpr int block = kRingPieces * kRingThreads;
  if (g == V && pieces > block && pieces <= block * kRingCluster)
    return launch_norm_grad_ring<T>(ctx, a, (int)((pieces + block - 1) / block), s);
  if (pieces <= 1024) {
    if (pieces <= 32) return launch_norm_grad_vec<T, 32>(ctx, a, g, s);
    if (pieces <= 64) return launch_norm_grad_vec<T, 64>(ctx, a, g, s);
    if (pieces <= 128) return launch_norm_grad_vec<T, 128>(ctx, a, g, s);
    if (pieces <= 256) return launch_norm_grad_vec<T, 256>(ctx, a, g, s);
    if (pieces <= 512) return launch_norm_grad_vec<T, 512>(ctx, a, g, s);
    return launch_norm_grad_vec<T, 1024>(ctx, a, g, s);
  }
  // Wider rows that are not on 16 bytes throughout (or longer than 64 KB): a
  // kernel for the means, one for the column sums, one for the rows, which read
  // their tensors ten times in all.  Far from the floor: 8192 x 8194 float16 1741 us
  // (123), 8192 x 4099 float32 1436 us (123).
  void *scratch;
  ACD_TRY(get_scratch(ctx, sizeof(A) * (size_t)a.s.rows(), s, &scratch));
  A *means = static_cast<A *>(scratch);
  if (a.d_w_pre || a.d_w_post || a.d_gate) {
    const int grid = persistent_grid(ctx, k_norm_grad_means<T>, 256, 0, a.s.rows());
    k_norm_grad_means<T><<<grid, 256, 0, s>>>(a, means);
    k_norm_grad_cols<T><<<(unsigned)((a.s.D + 31) / 32), 256, 0, s>>>(a, means);
  }
  const int grid = persistent_grid(ctx, k_norm_grad_rows<T>, 256, 0, a.s.rows());
  k_norm_grad_rows<T><<<grid, 256, 0, s>>>(a);
  return ACD_OK;
}

// ---------------------------------------------------------------------------
// argument checks
// ---------------------------------------------------------------------------
// A tensor of the call's row shape and dtype.
static acd_status check_rows(const char *op, const char *name, const acd_desc *d, const acd_desc *like, int axis,
                             RowShape &s, Rows &v) {
  ACD_TRY(check_desc(d, name));
  if (d->dtype != like->dtype) return fail(ACD_ERR_DTYPE, "%s: %s has another dtype than the block", op, name);
  if (!same_shape(d, like)) return fail(ACD_ERR_SHAPE, "%s: %s has another shape than the block", op, name);
  if (!split_rows(d, axis, s, v))
    return fail(ACD_ERR_UNSUPPORTED, "%s: %s not collapsible around the axis; make it contiguous first", op, name);
  return ACD_OK;
}

static acd_status check_block(const char *op, const acd_desc *block, int32_t axis) {
  ACD_TRY(check_desc(block, "block"));
  if (block->dtype != ACD_FLOAT32 && block->dtype != ACD_FLOAT64 && block->dtype != ACD_FLOAT16)
    return fail(ACD_ERR_DTYPE, "%s: float32, float64 or float16 rows required", op);
  if (axis < 0 || axis >= block->ndim) return fail(ACD_ERR_AXIS, "%s: axis %d out of range", op, axis);
  if (block->shape[axis] > INT32_MAX) return fail(ACD_ERR_UNSUPPORTED, "%s: rows of more than 2^31 - 1 elements", op);
  if (desc_numel(block) > 0 && desc_numel(block) / block->shape[axis] > INT32_MAX)
    return fail(ACD_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows", op);
  return ACD_OK;
}

// D elements, contiguous; `dtype` differs between operands and gradients.
static acd_status check_weight(const char *op, const char *name, const acd_desc *w, int64_t D, int32_t dtype) {
  ACD_TRY(check_desc(w, name));
  if (w->dtype != dtype) return fail(ACD_ERR_DTYPE, "%s: %s has the wrong dtype", op, name);
  if (w->ndim < 1 || desc_numel(w) != D) return fail(ACD_ERR_SHAPE, "%s: %s must have one element for each of a row", op, name);
  if (!desc_is_contiguous(w)) return fail(ACD_ERR_UNSUPPORTED, "%s: %s must be contiguous", op, name);
  return ACD_OK;
}

// The gate's strides and how many consecutive rows share one of its rows.
static acd_status check_gate(const char *op, const char *name, const acd_desc *g, const acd_desc *like, int axis,
                             int32_t dtype, int64_t *sd, int64_t *sg, int64_t *per) {
  ACD_TRY(check_desc(g, name));
  if (g->dtype != dtype) return fail(ACD_ERR_DTYPE, "%s: %s has the wrong dtype", op, name);
  const int64_t D = like->shape[axis];
  int64_t rows = 1;
  for (int k = 0; k < like->ndim; ++k)
    if (k != axis) rows *= like->shape[k];
  *sg = 0;
  *per = rows;
  if (!desc_is_contiguous(g)) return fail(ACD_ERR_UNSUPPORTED, "%s: %s must be contiguous", op, name);
  if (g->ndim == 1 && g->shape[0] == D) {
    *sd = g->stride[0];
    return ACD_OK;
  }
  bool ok = g->ndim == like->ndim && g->shape[axis] == D;
  int64_t groups = 1, next = 0;
  bool begun = false;
  for (int k = 0; ok && k < like->ndim; ++k) {
    if (k == axis) continue;
    if (g->shape[k] != like->shape[k]) {
      ok = g->shape[k] == 1 && !begun;
      continue;
    }
    if (g->shape[k] == 1) continue;
    if (begun && g->stride[k] != next)
      return fail(ACD_ERR_UNSUPPORTED, "%s: %s not collapsible around the axis", op, name);
    if (!begun) *sg = g->stride[k];
    next = g->stride[k] * g->shape[k];
    groups *= g->shape[k];
    begun = true;
  }
  if (!ok)
    return fail(ACD_ERR_SHAPE, "%s: %s must have one row, or one for each of the last axes' entries", op, name);
  *sd = g->stride[axis];
  *per = groups ? rows / groups : rows;
  return ACD_OK;
}

static acd_status check_rstd(const char *op, const char *name, const acd_desc *d, const acd_desc *block, int axis) {
  ACD_TRY(check_row_tensor(op, name, d, block, axis));
  if (d->dtype != (block->dtype == ACD_FLOAT64 ? ACD_FLOAT64 : ACD_FLOAT32))
    return fail(ACD_ERR_DTYPE, "%s: %s has the wrong dtype", op, name);
  return ACD_OK;
}

}  // namespace acd

using namespace acd;

extern "C" {

acd_status acd_residual_norm(acd_ctx *ctx, const acd_desc *h, const acd_desc *y, const acd_desc *rstd_h,
                             const acd_desc *rstd_block, const acd_desc *residual, const acd_desc *block,
                             const acd_desc *w_pre, const acd_desc *w_post, const acd_desc *gate, int32_t axis,
                             double alpha, double eps, acd_stream stream) {
  const char *op = "acd_residual_norm";
  if (!ctx) return fail(ACD_ERR_INVALID, "%s: null context", op);
  ACD_TRY(check_block(op, block, axis));
  if (!std::isfinite(alpha)) return fail(ACD_ERR_INVALID, "%s: alpha must be finite", op);
  if (!(eps >= 0.0) || !std::isfinite(eps)) return fail(ACD_ERR_INVALID, "%s: eps must be finite and not negative", op);
  NormArgs a{};
  ACD_TRY(check_rows(op, "block", block, block, axis, a.s, a.b));
  ACD_TRY(check_rows(op, "residual", residual, block, axis, a.s, a.r));
  ACD_TRY(check_rows(op, "h", h, block, axis, a.s, a.h));
  ACD_TRY(check_rows(op, "y", y, block, axis, a.s, a.y));
  ACD_TRY(check_weight(op, "w_pre", w_pre, a.s.D, block->dtype));
  if (w_post) ACD_TRY(check_weight(op, "w_post", w_post, a.s.D, block->dtype));
  if (rstd_block && !w_post) return fail(ACD_ERR_INVALID, "%s: rstd_block without w_post", op);
  a.per = a.s.rows();
  if (gate) ACD_TRY(check_gate(op, "gate", gate, block, axis, block->dtype, &a.gate_sd, &a.gate_sg, &a.per));
  if (rstd_h) ACD_TRY(check_rstd(op, "rstd_h", rstd_h, block, axis));
  if (rstd_block) ACD_TRY(check_rstd(op, "rstd_block", rstd_block, block, axis));
  if (a.s.rows() == 0) return ACD_OK;
  if (a.s.D == 0) return fail(ACD_ERR_SHAPE, "%s: rows without elements", op);
  a.alpha = alpha;
  a.eps = eps;
  a.w_pre = desc_ptr(w_pre);
  a.w_post = w_post ? desc_ptr(w_post) : nullptr;
  a.gate = gate ? desc_ptr(gate) : nullptr;
  a.rstd_h = rstd_h ? desc_ptr(rstd_h) : nullptr;
  a.rstd_b = rstd_block ? desc_ptr(rstd_block) : nullptr;
  DeviceGuard g(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (block->dtype == ACD_FLOAT32)
    ACD_TRY(launch_norm<float>(ctx, a, s));
  else if (block->dtype == ACD_FLOAT64)
    ACD_TRY(launch_norm<double>(ctx, a, s));
  else
    ACD_TRY(launch_norm<__half>(ctx, a, s));
  ACD_CUDA(cudaGetLastError());
  return ACD_OK;
}

acd_status acd_residual_norm_grad(acd_ctx *ctx, const acd_desc *d_residual, const acd_desc *d_block,
                                  const acd_desc *d_w_pre, const acd_desc *d_w_post, const acd_desc *d_gate,
                                  const acd_desc *d_h, const acd_desc *d_y, const acd_desc *h, const acd_desc *block,
                                  const acd_desc *rstd_h, const acd_desc *rstd_block, const acd_desc *w_pre,
                                  const acd_desc *w_post, const acd_desc *gate, int32_t axis, double alpha,
                                  acd_stream stream) {
  const char *op = "acd_residual_norm_grad";
  if (!ctx) return fail(ACD_ERR_INVALID, "%s: null context", op);
  ACD_TRY(check_block(op, block, axis));
  if (!std::isfinite(alpha)) return fail(ACD_ERR_INVALID, "%s: alpha must be finite", op);
  NormGradArgs a{};
  ACD_TRY(check_rows(op, "block", block, block, axis, a.s, a.b));
  ACD_TRY(check_rows(op, "d_residual", d_residual, block, axis, a.s, a.dr));
  ACD_TRY(check_rows(op, "d_block", d_block, block, axis, a.s, a.db));
  if (d_h) ACD_TRY(check_rows(op, "d_h", d_h, block, axis, a.s, a.dh));
  ACD_TRY(check_rows(op, "d_y", d_y, block, axis, a.s, a.dy));
  ACD_TRY(check_rows(op, "h", h, block, axis, a.s, a.h));
  const int32_t st = block->dtype == ACD_FLOAT64 ? ACD_FLOAT64 : ACD_FLOAT32;
  ACD_TRY(check_weight(op, "w_pre", w_pre, a.s.D, block->dtype));
  if (w_post) ACD_TRY(check_weight(op, "w_post", w_post, a.s.D, block->dtype));
  if ((w_post == nullptr) != (rstd_block == nullptr))
    return fail(ACD_ERR_INVALID, "%s: w_post and rstd_block must both be given or both be NULL", op);
  if (d_w_post && !w_post) return fail(ACD_ERR_INVALID, "%s: d_w_post without w_post", op);
  if (d_gate && !gate) return fail(ACD_ERR_INVALID, "%s: d_gate without gate", op);
  if (!rstd_h) return fail(ACD_ERR_INVALID, "%s: null rstd_h", op);
  if (d_w_pre) ACD_TRY(check_weight(op, "d_w_pre", d_w_pre, a.s.D, st));
  if (d_w_post) ACD_TRY(check_weight(op, "d_w_post", d_w_post, a.s.D, st));
  a.per = a.s.rows();
  if (gate) ACD_TRY(check_gate(op, "gate", gate, block, axis, block->dtype, &a.gate_sd, &a.gate_sg, &a.per));
  if (d_gate) {
    int64_t sd, sg, per;
    ACD_TRY(check_gate(op, "d_gate", d_gate, block, axis, st, &sd, &sg, &per));
    if (sd != a.gate_sd || sg != a.gate_sg || per != a.per)
      return fail(ACD_ERR_SHAPE, "%s: d_gate has another shape than gate", op);
  }
  ACD_TRY(check_rstd(op, "rstd_h", rstd_h, block, axis));
  if (rstd_block) ACD_TRY(check_rstd(op, "rstd_block", rstd_block, block, axis));
  DeviceGuard g(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.s.rows() == 0) {  // no rows: the sums are empty
    const size_t es = dtype_size(st);
    if (d_w_pre && a.s.D) ACD_CUDA(cudaMemsetAsync(desc_ptr(d_w_pre), 0, es * a.s.D, s));
    if (d_w_post && a.s.D) ACD_CUDA(cudaMemsetAsync(desc_ptr(d_w_post), 0, es * a.s.D, s));
    if (d_gate && desc_numel(d_gate)) ACD_CUDA(cudaMemsetAsync(desc_ptr(d_gate), 0, es * desc_numel(d_gate), s));
    return ACD_OK;
  }
  if (a.s.D == 0) return fail(ACD_ERR_SHAPE, "%s: rows without elements", op);
  a.alpha = alpha;
  a.w_pre = desc_ptr(w_pre);
  a.w_post = w_post ? desc_ptr(w_post) : nullptr;
  a.gate = gate ? desc_ptr(gate) : nullptr;
  a.rstd_h = desc_ptr(rstd_h);
  a.rstd_b = rstd_block ? desc_ptr(rstd_block) : nullptr;
  a.d_w_pre = d_w_pre ? desc_ptr(d_w_pre) : nullptr;
  a.d_w_post = d_w_post ? desc_ptr(d_w_post) : nullptr;
  a.d_gate = d_gate ? desc_ptr(d_gate) : nullptr;
  if (block->dtype == ACD_FLOAT32)
    ACD_TRY(launch_norm_grad<float>(ctx, a, s));
  else if (block->dtype == ACD_FLOAT64)
    ACD_TRY(launch_norm_grad<double>(ctx, a, s));
  else
    ACD_TRY(launch_norm_grad<__half>(ctx, a, s));
  ACD_CUDA(cudaGetLastError());
  return ACD_OK;
}

}  // extern "C"
