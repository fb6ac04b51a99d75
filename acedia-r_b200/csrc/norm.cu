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

template <typename T>
static acd_status launch_norm(acd_ctx *ctx, const NormArgs &a, cudaStream_t s) {
  const int grid = persistent_grid(ctx, k_norm_rows<T>, 256, 0, a.s.rows());
  k_norm_rows<T><<<grid, 256, 0, s>>>(a);
  return ACD_OK;
}

template <typename T>
static acd_status launch_norm_grad(acd_ctx *ctx, const NormGradArgs &a, cudaStream_t s) {
  using A = typename AccOf<T>::type;
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
