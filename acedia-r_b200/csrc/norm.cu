// A residual update with the norms around it, and its gradients.
//
//   b' = b rs_b w_post,  h = alpha r + gate b',  y = h rs_h w_pre,
//   rs_v = 1 / sqrt(mean(v^2) + eps)
// The gradients, with hn = h rs_h and bn = b rs_b:
//   t = dh + rs_h (dy w_pre - hn mean(dy w_pre hn)),  dr = alpha t,
//   u = t gate,  db = rs_b (u w_post - bn mean(u w_post bn)),
//   dw_pre = sum dy hn,  dw_post = sum u bn,  dgate = sum t b'.
#include "lm_rows.cuh"

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
    const T *gate = a.gate ? static_cast<const T *>(a.gate) + row / a.per * a.gate_sg : nullptr;
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
    const T *gate = a.gate ? static_cast<const T *>(a.gate) + row / a.per * a.gate_sg : nullptr;
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
// WHOLE: 16 consecutive bytes; every row, weight and gate row starts on a
// 16-byte boundary and D is a multiple of V.  Otherwise TPR apart, so that a
// warp still reads neighbouring elements: any alignment, width and stride, and
// a thread's columns are the same in every row (a piece moved by each row's
// misalignment would not be, and its weights would be read 16 bytes apart).
template <int V, int TPR, bool WHOLE>
__device__ __forceinline__ int column(int tid, int n, int j) {
  return WHOLE ? (n * TPR + tid) * V + j : (n * V + j) * TPR + tid;
}

template <typename T, typename A, int V, int TPR, bool WHOLE>
__device__ __forceinline__ void load_cols(const T *x, int64_t sd, int tid, int n, int D, A *out) {
  if (WHOLE) {
    const int first = column<V, TPR, true>(tid, n, 0);
    if (first < D) {
      const Vec<T, V> v = *reinterpret_cast<const Vec<T, V> *>(x + first);
#pragma unroll
      for (int j = 0; j < V; ++j) out[j] = to_acc(v.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) out[j] = A(0);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int d = column<V, TPR, false>(tid, n, j);
      out[j] = d < D ? to_acc(x[d * sd]) : A(0);
    }
  }
}

template <typename T, typename A, int V, int TPR, bool WHOLE>
__device__ __forceinline__ void store_cols(T *x, int64_t sd, int tid, int n, int D, const A *v) {
  if (WHOLE) {
    const int first = column<V, TPR, true>(tid, n, 0);
    if (first < D) {
      Vec<T, V> w;
#pragma unroll
      for (int j = 0; j < V; ++j) w.v[j] = from_acc<T, A>(v[j]);
      *reinterpret_cast<Vec<T, V> *>(x + first) = w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int d = column<V, TPR, false>(tid, n, j);
      if (d < D) x[d * sd] = from_acc<T, A>(v[j]);
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

// TPR threads a row, NV pieces of V columns a thread; the row stays in registers between
// the two sums.
template <typename T, int TPR, int NV, bool WHOLE>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_norm_vec(NormArgs a) {
  using A = typename AccOf<T>::type;
  constexpr int V = 16 / sizeof(T), BLOCK = TPR < 256 ? 256 : TPR;
  __shared__ A sh[2][BLOCK / 32];
  const int64_t row = (int64_t)blockIdx.x * (BLOCK / TPR) + threadIdx.x / TPR;
  const bool ok = row < a.s.rows();  // whole warps: a row has at least one
  const int64_t rr = ok ? row : 0;
  const int tid = threadIdx.x % TPR;
  const int D = ok ? (int)a.s.D : 0;
  const T *r = row_ptr<T>(a.r, rr, a.s.L), *b = row_ptr<T>(a.b, rr, a.s.L);
  const T *w_pre = static_cast<const T *>(a.w_pre), *w_post = static_cast<const T *>(a.w_post);
  const A alpha = (A)a.alpha, eps = (A)a.eps, inv = A(1) / (A)a.s.D;
  A bv[NV][V], rv[NV][V];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    load_cols<T, A, V, TPR, WHOLE>(b, a.b.sd, tid, n, D, bv[n]);
    load_cols<T, A, V, TPR, WHOLE>(r, a.r.sd, tid, n, D, rv[n]);
  }
  A rb = 1;
  if (w_post) {
    A q[1] = {A(0)};
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int j = 0; j < V; ++j) q[0] = fma_a(bv[n][j], bv[n][j], q[0]);
    row_sum<A, 1, TPR>(q, sh[0]);
    rb = rsqrt_a(q[0] * inv + eps);
  }
  A q[1] = {A(0)};
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    A w[V];
    if (w_post) {
      load_cols<T, A, V, TPR, WHOLE>(w_post, 1, tid, n, D, w);
#pragma unroll
      for (int j = 0; j < V; ++j) bv[n][j] *= rb * w[j];
    }
    if (a.gate) {
      load_cols<T, A, V, TPR, WHOLE>(static_cast<const T *>(a.gate) + rr / a.per * a.gate_sg, a.gate_sd, tid, n, D, w);
#pragma unroll
      for (int j = 0; j < V; ++j) bv[n][j] *= w[j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      bv[n][j] = fma_a(alpha, rv[n][j], bv[n][j]);
      q[0] = fma_a(bv[n][j], bv[n][j], q[0]);
    }
  }
  row_sum<A, 1, TPR>(q, sh[1]);
  const A rh = rsqrt_a(q[0] * inv + eps);
  if (!ok) return;
  T *h = row_ptr<T>(a.h, rr, a.s.L), *y = row_ptr<T>(a.y, rr, a.s.L);
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    A w[V];
    load_cols<T, A, V, TPR, WHOLE>(w_pre, 1, tid, n, D, w);
    store_cols<T, A, V, TPR, WHOLE>(h, a.h.sd, tid, n, D, bv[n]);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] *= bv[n][j] * rh;
    store_cols<T, A, V, TPR, WHOLE>(y, a.y.sd, tid, n, D, w);
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

// One piece of a row's gradient, in two steps around the row's sums.  With
//   q = d_h + rs_h d_y w_pre,  hn = h rs_h,  bn = b rs_b,  e = gate w_post bn
// t = q - rs_h hn m1, so that mean(u w_post bn) = mean(q e) - m1 mean(rs_h hn e)
// comes from the same pass as m1 = mean(d_y w_pre hn): one reduction a row.
template <typename T, typename A, int V, int TPR, bool WHOLE>
struct GradPiece {
  A dh[V], dy[V], h[V], b[V];
  __device__ __forceinline__ void load(const NormGradArgs &a, int64_t row, int tid, int D) {
    if (a.dh.p) {
      load_cols<T, A, V, TPR, WHOLE>(row_ptr<T>(a.dh, row, a.s.L), a.dh.sd, tid, 0, D, dh);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) dh[j] = A(0);
    }
    load_cols<T, A, V, TPR, WHOLE>(row_ptr<T>(a.dy, row, a.s.L), a.dy.sd, tid, 0, D, dy);
    load_cols<T, A, V, TPR, WHOLE>(row_ptr<T>(a.h, row, a.s.L), a.h.sd, tid, 0, D, h);
    load_cols<T, A, V, TPR, WHOLE>(row_ptr<T>(a.b, row, a.s.L), a.b.sd, tid, 0, D, b);
  }
  __device__ __forceinline__ void sums(const A *wp, const A *wo, const A *g, A rh, A rb, A (&s)[3]) const {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const A hn = h[j] * rh, u = dy[j] * wp[j], e = g[j] * wo[j] * (b[j] * rb);
      s[0] = fma_a(u, hn, s[0]);
      s[1] = fma_a(fma_a(rh, u, dh[j]), e, s[1]);
      s[2] = fma_a(rh * hn, e, s[2]);
    }
  }
  // Leaves alpha t in dh and the block's gradient in dy; adds to the sums.
  __device__ __forceinline__ void finish(const A *wp, const A *wo, const A *g, A rh, A rb, A m1, A m2, A alpha,
                                         bool post, A *pre, A *pst, A *gte) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const A hn = h[j] * rh, bn = b[j] * rb;
      const A t = fma_a(rh, fma_a(dy[j], wp[j], -(hn * m1)), dh[j]);
      const A u = t * g[j];
      pre[j] = fma_a(dy[j], hn, pre[j]);
      pst[j] = fma_a(u, bn, pst[j]);
      gte[j] = fma_a(t, bn * wo[j], gte[j]);
      dh[j] = alpha * t;
      dy[j] = post ? rb * fma_a(u, wo[j], -(bn * m2)) : u;
    }
  }
};

template <typename A, int V>
__device__ __forceinline__ void ones(A *v) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = A(1);
}

// One piece a thread, TPR threads a row; the column sums stay in registers.
template <typename T, int TPR, bool WHOLE>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_norm_grad_vec(NormGradArgs a, GradPlan plan) {
  using A = typename AccOf<T>::type;
  constexpr int V = 16 / sizeof(T), BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR;
  __shared__ A sh[2][BLOCK / 32 * 3];
  __shared__ A join[RPB > 1 ? BLOCK : 1][V];
  const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int D = (int)a.s.D;
  const T *w_pre = static_cast<const T *>(a.w_pre), *w_post = static_cast<const T *>(a.w_post);
  const A alpha = (A)a.alpha, inv = A(1) / (A)a.s.D;
  A pre[V] = {}, pst[V] = {};
  int flip = 0;
  for (int64_t u = blockIdx.x; u < plan.groups * plan.parts; u += gridDim.x) {
    int64_t r0, r1;
    unit_rows(plan, u, r0, r1);
    A gte[V] = {};
    for (int64_t rr = r0; rr < r1; rr += RPB) {
      const int64_t row = rr + sub;
      const bool ok = row < r1;
      GradPiece<T, A, V, TPR, WHOLE> p;
      p.load(a, ok ? row : r0, tid, ok ? D : 0);
      A wp[V], wo[V], g[V];
      load_cols<T, A, V, TPR, WHOLE>(w_pre, 1, tid, 0, D, wp);
      if (w_post)
        load_cols<T, A, V, TPR, WHOLE>(w_post, 1, tid, 0, D, wo);
      else
        ones<A, V>(wo);
      if (a.gate)
        load_cols<T, A, V, TPR, WHOLE>(static_cast<const T *>(a.gate) + r0 / a.per * a.gate_sg, a.gate_sd, tid, 0, D, g);
      else
        ones<A, V>(g);
      const A rh = ok ? static_cast<const A *>(a.rstd_h)[row] : A(0);
      const A rb = w_post && ok ? static_cast<const A *>(a.rstd_b)[row] : A(1);
      A s[3] = {};
      p.sums(wp, wo, g, rh, rb, s);
      row_sum<A, 3, TPR>(s, sh[flip]);
      flip ^= 1;
      const A m1 = s[0] * inv, m2 = (s[1] - m1 * s[2]) * inv;
      p.finish(wp, wo, g, rh, rb, m1, m2, alpha, w_post != nullptr, pre, pst, gte);
      if (ok) {
        store_cols<T, A, V, TPR, WHOLE>(row_ptr<T>(a.dr, row, a.s.L), a.dr.sd, tid, 0, D, p.dh);
        store_cols<T, A, V, TPR, WHOLE>(row_ptr<T>(a.db, row, a.s.L), a.db.sd, tid, 0, D, p.dy);
      }
    }
    if (plan.gate) {
      if (RPB > 1) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) join[threadIdx.x][j] = gte[j];
        __syncthreads();
        if (sub == 0)
          for (int q = 1; q < RPB; ++q)
#pragma unroll
            for (int j = 0; j < V; ++j) gte[j] += join[q * TPR + tid][j];
      }
      if (sub == 0)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (column<V, TPR, WHOLE>(tid, 0, j) < D)
            static_cast<A *>(plan.gate)[u * plan.gate_su + column<V, TPR, WHOLE>(tid, 0, j) * plan.gate_sd] = gte[j];
    }
  }
  for (int w = 0; w < 2; ++w) {
    A *dst = static_cast<A *>(w ? plan.post : plan.pre);
    A *acc = w ? pst : pre;
    if (!dst) continue;
    if (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j) join[threadIdx.x][j] = acc[j];
      __syncthreads();
      if (sub == 0)
        for (int q = 1; q < RPB; ++q)
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] += join[q * TPR + tid][j];
    }
    if (sub == 0)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (column<V, TPR, WHOLE>(tid, 0, j) < D)
          dst[(int64_t)blockIdx.x * D + column<V, TPR, WHOLE>(tid, 0, j)] = acc[j];
  }
}

// Column sums of `n` partial rows: 32 columns a block, its 8 warps split the
// rows and are added in order.
template <typename A>
struct JoinArgs {
  const A *src[3];
  A *dst[3];
  int64_t n[3], sd[3], sg[3];  // rows a sum, strides of dst along the row and over its groups
  int64_t D;
};

template <typename A>
__global__ void __launch_bounds__(256) k_norm_grad_join(JoinArgs<A> a) {
  __shared__ A sh[8][32];
  // blockIdx.y: 0 pre, 1 post, 2 + g gate row g
  const int w = blockIdx.y < 2 ? blockIdx.y : 2;
  const int64_t g = w == 2 ? blockIdx.y - 2 : 0;
  if (!a.dst[w]) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t d = (int64_t)blockIdx.x * 32 + lane, n = a.n[w];
  A s = 0;
  if (d < a.D) {
    const A *p = a.src[w] + g * n * a.D + d;
#pragma unroll 8
    for (int64_t i = warp; i < n; i += 8) s += p[i * a.D];
  }
  sh[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && d < a.D) {
    for (int q = 1; q < 8; ++q) s += sh[q][lane];
    a.dst[w][d * a.sd[w] + g * a.sg[w]] = s;
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Whether the rows of `v` are contiguous and start on 16-byte boundaries (the
// width is checked once, for all of them).
static bool whole_rows(const Rows &v, int V) {
  return v.sd == 1 && aligned_to<char>(v.p, 16) && v.sl % V == 0 && v.so % V == 0;
}
// Weights and gate rows too.
static bool whole_weights(const void *w_pre, const void *w_post, const void *gate, int64_t sd, int64_t sg, int V) {
  return aligned_to<char>(w_pre, 16) && (!w_post || aligned_to<char>(w_post, 16)) &&
         (!gate || (aligned_to<char>(gate, 16) && sd == 1 && sg % V == 0));
}

template <typename T, int TPR, int NV>
static acd_status launch_norm_vec(const NormArgs &a, bool whole, cudaStream_t s) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR, RPB = BLOCK / TPR;
  const int64_t grid = (a.s.rows() + RPB - 1) / RPB;
  if (whole)
    k_norm_vec<T, TPR, NV, true><<<(unsigned)grid, BLOCK, 0, s>>>(a);
  else
    k_norm_vec<T, TPR, NV, false><<<(unsigned)grid, BLOCK, 0, s>>>(a);
  return ACD_OK;
}

template <typename T>
static acd_status launch_norm(acd_ctx *ctx, const NormArgs &a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool whole = a.s.D % V == 0 && whole_rows(a.r, V) && whole_rows(a.b, V) && whole_rows(a.h, V) &&
                     whole_rows(a.y, V) && whole_weights(a.w_pre, a.w_post, a.gate, a.gate_sd, a.gate_sg, V);
  const int64_t pieces = (a.s.D + V - 1) / V;
  if (pieces <= 4096) {
    if (pieces <= 32) return launch_norm_vec<T, 32, 1>(a, whole, s);
    if (pieces <= 64) return launch_norm_vec<T, 32, 2>(a, whole, s);
    if (pieces <= 256) return launch_norm_vec<T, 128, 2>(a, whole, s);
    if (pieces <= 512) return launch_norm_vec<T, 256, 2>(a, whole, s);
    if (pieces <= 1024) return launch_norm_vec<T, 512, 2>(a, whole, s);
    if (pieces <= 2048) return launch_norm_vec<T, 1024, 2>(a, whole, s);
    return launch_norm_vec<T, 1024, 4>(a, whole, s);
  }
  const int grid = persistent_grid(ctx, k_norm_rows<T>, 256, 0, a.s.rows());
  k_norm_rows<T><<<grid, 256, 0, s>>>(a);
  return ACD_OK;
}

template <typename T, int TPR>
static acd_status launch_norm_grad_vec(acd_ctx *ctx, const NormGradArgs &a, bool whole, cudaStream_t s) {
  using A = typename AccOf<T>::type;
  constexpr int BLOCK = TPR < 256 ? 256 : TPR;
  auto kern = whole ? k_norm_grad_vec<T, TPR, true> : k_norm_grad_vec<T, TPR, false>;
  const int64_t rows = a.s.rows(), D = a.s.D;
  int64_t grid = (int64_t)ctx->sm_count * resident_blocks(reinterpret_cast<const void *>(kern), BLOCK, 0);
  GradPlan p{};
  p.per = a.per;
  p.groups = rows / a.per;
  p.parts = grid / p.groups;
  if (p.parts > (p.per + BLOCK / TPR - 1) / (BLOCK / TPR)) p.parts = (p.per + BLOCK / TPR - 1) / (BLOCK / TPR);
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
  kern<<<(unsigned)grid, BLOCK, 0, s>>>(a, p);
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
  if (j.dst[0] || j.dst[1] || j.dst[2])
    k_norm_grad_join<A><<<dim3((unsigned)((D + 31) / 32), (unsigned)(2 + (gate_part ? p.groups : 0))), 256, 0, s>>>(j);
  return ACD_OK;
}

template <typename T>
static acd_status launch_norm_grad(acd_ctx *ctx, const NormGradArgs &a, cudaStream_t s) {
  using A = typename AccOf<T>::type;
  constexpr int V = 16 / sizeof(T);
  const bool whole = a.s.D % V == 0 && whole_rows(a.dr, V) && whole_rows(a.db, V) &&
                     (!a.dh.p || whole_rows(a.dh, V)) && whole_rows(a.dy, V) && whole_rows(a.h, V) &&
                     whole_rows(a.b, V) && whole_weights(a.w_pre, a.w_post, a.gate, a.gate_sd, a.gate_sg, V);
  const int64_t pieces = (a.s.D + V - 1) / V;
  if (pieces <= 1024) {
    if (pieces <= 32) return launch_norm_grad_vec<T, 32>(ctx, a, whole, s);
    if (pieces <= 128) return launch_norm_grad_vec<T, 128>(ctx, a, whole, s);
    if (pieces <= 256) return launch_norm_grad_vec<T, 256>(ctx, a, whole, s);
    if (pieces <= 512) return launch_norm_grad_vec<T, 512>(ctx, a, whole, s);
    return launch_norm_grad_vec<T, 1024>(ctx, a, whole, s);
  }
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
