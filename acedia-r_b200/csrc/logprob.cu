// Log probabilities of given tokens with entropy and the k most likely
// alternatives, and their gradient.
//
// A row holds the logits x_v of one prediction.  With c = scale, m = max x,
//   S = sum e^{c(x_v - m)},  T = sum c(x_v - m) e^{c(x_v - m)}
// everything the forward call returns follows from (m, S, T):
//   lse = c m + ln S,  logprob = c(x_t - m) - ln S,  entropy = ln S - T / S.
// The gradient is one expression a logit (see k_logprob_grad).
#include "lm_rows.cuh"

namespace acd {

__device__ __forceinline__ float lp_exp(float x) { return expf(x); }
__device__ __forceinline__ double lp_exp(double x) { return exp(x); }
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

// (value, index): the better one has the larger value, then the lower index.
template <typename A>
struct Cand {
  A v;
  int64_t i;
  __device__ __forceinline__ bool better(const Cand &o) const { return v > o.v || (v == o.v && i < o.i); }
};

// Row results from (m, S, T).
template <typename T, typename A>
__device__ __forceinline__ void write_row(const LogprobArgs &a, int64_t r, A m, A S, A Tm, A &log_s) {
  const bool empty = S == A(0);  // every logit -Inf (a NaN leaves S = NaN)
  const A c = (A)a.scale;
  log_s = empty ? A(0) : lp_log(S);
  if (a.lse) static_cast<A *>(a.lse)[r] = empty ? A(-INFINITY) : c * m + log_s;
  if (a.entropy) static_cast<A *>(a.entropy)[r] = empty ? A(0) : log_s - Tm / S;
  if (a.logprob) {
    const int64_t t = load_index(a.tokens, a.wide_token, r) - (a.one_based ? 1 : 0);
    A lp = A(NAN);
    if (t == -1)
      lp = A(0);
    else if (t >= 0 && t < a.s.D)
      lp = empty ? A(-INFINITY) : c * (to_acc(row_ptr<T>(a.x, r, a.s.L)[t * a.x.sd]) - m) - log_s;
    static_cast<A *>(a.logprob)[r] = lp;
  }
}

// One block a row, any strides: maximum, then sums, then k searches for the
// best logit behind the last one found.
template <typename T>
__global__ void __launch_bounds__(256) k_logprob_rows(LogprobArgs a) {
  using A = typename AccOf<T>::type;
  __shared__ A sh[3][8];
  __shared__ Cand<A> shc[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const A c = (A)a.scale;
  for (int64_t r = blockIdx.x; r < a.s.rows(); r += gridDim.x) {
    const T *x = row_ptr<T>(a.x, r, a.s.L);
    A m = A(-INFINITY);
    bool nan = false;
    for (int64_t d = threadIdx.x; d < a.s.D; d += 256) {
      const A v = to_acc(x[d * a.x.sd]);
      nan |= v != v;
      m = v > m ? v : m;
    }
    for (int q = 16; q; q >>= 1) {
      const A o = __shfl_xor_sync(~0u, m, q);
      m = o > m ? o : m;
    }
    nan = __syncthreads_or(nan);
    if (lane == 0) sh[0][warp] = m;
    __syncthreads();
    for (int q = 0; q < 8; ++q) m = sh[0][q] > m ? sh[0][q] : m;
    if (nan) m = A(NAN);
    A S = 0, Tm = 0;
    if (m != A(-INFINITY))
      for (int64_t d = threadIdx.x; d < a.s.D; d += 256) {
        const A z = c * (to_acc(x[d * a.x.sd]) - m);
        const A e = lp_exp(z);
        S += e;
        if (e != A(0)) Tm = fma_a(z, e, Tm);
      }
    for (int q = 16; q; q >>= 1) {
      S += __shfl_xor_sync(~0u, S, q);
      Tm += __shfl_xor_sync(~0u, Tm, q);
    }
    if (lane == 0) {
      sh[1][warp] = S;
      sh[2][warp] = Tm;
    }
    __syncthreads();
    S = Tm = 0;
    for (int q = 0; q < 8; ++q) {
      S += sh[1][q];
      Tm += sh[2][q];
    }
    A log_s = 0;
    if (threadIdx.x == 0) write_row<T, A>(a, r, m, S, Tm, log_s);
    Cand<A> last{A(INFINITY), -1};
    const int64_t o = r / a.s.L, l = r - o * a.s.L;
    for (int j = 0; j < a.k; ++j) {
      Cand<A> best{A(-INFINITY), INT64_MAX};
      for (int64_t d = threadIdx.x; d < a.s.D; d += 256) {
        const Cand<A> q{to_acc(x[d * a.x.sd]), d};
        if (last.better(q) && q.better(best)) best = q;
      }
      for (int q = 16; q; q >>= 1) {
        const Cand<A> b{__shfl_xor_sync(~0u, best.v, q), __shfl_xor_sync(~0u, best.i, q)};
        if (b.better(best)) best = b;
      }
      __syncthreads();
      if (lane == 0) shc[warp] = best;
      __syncthreads();
      for (int q = 0; q < 8; ++q)
        if (shc[q].better(best)) best = shc[q];
      last = best;
      if (threadIdx.x == 0) {
        const int64_t at = l + a.s.L * (j + a.k * o);
        const bool none = best.i == INT64_MAX;
        store_index(a.top_index, a.wide_index, at,
                    none ? (a.wide_index ? INT64_MIN : (int64_t)INT32_MIN) : best.i + (a.one_based ? 1 : 0));
        A lp = c * (best.v - m) - log_s;
        if (m == A(-INFINITY)) lp = A(-INFINITY);
        static_cast<A *>(a.top_logprob)[at] = none ? A(NAN) : lp;
      }
    }
    __syncthreads();
  }
}

struct LogprobGradArgs {
  Rows x, g;
  RowShape s;
  double scale;
  const void *tokens, *lse, *entropy, *d_logprob, *d_entropy, *d_lse;
  bool wide_token, one_based;
};

// Coefficients of a row: grad_v = p_v (a0 - a1 (lp_v + H)) + [v = token] gt.
template <typename A>
struct GradRow {
  A lse, H, a0, a1, gt;
  int64_t t;
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
      g.t = t;
      g.gt = c * static_cast<const A *>(a.d_logprob)[r];
    }
  }
  g.a1 = a.d_entropy ? c * static_cast<const A *>(a.d_entropy)[r] : A(0);
  g.H = a.d_entropy ? static_cast<const A *>(a.entropy)[r] : A(0);
  g.a0 = (a.d_lse ? c * static_cast<const A *>(a.d_lse)[r] : A(0)) - g.gt;
  // a row without mass: p = 0 everywhere and no token term.  So is one masked
  // throughout by the type's lowest value: its lse has no digits left for ln S.
  if (g.lse <= (std::is_same<A, double>::value ? (A)(-DBL_MAX / 4) : (A)(-FLT_MAX / 4))) {
    g.lse = A(INFINITY);
    g.t = -1;
  }
  return g;
}

template <typename A>
__device__ __forceinline__ A grad_value(const GradRow<A> &g, A x, A c, bool is_token) {
  const A lp = fma_a(c, x, -g.lse);
  const A p = lp_exp(lp);
  // p = 0 (a logit of -Inf, or far below the maximum): 0 log 0 = 0
  A v = p == A(0) ? A(0) : p * fma_a(-g.a1, lp + g.H, g.a0);
  return is_token ? v + g.gt : v;
}

// One element a thread, along the lanes first: any strides.
template <typename T>
__global__ void __launch_bounds__(256) k_logprob_grad(LogprobGradArgs a) {
  using A = typename AccOf<T>::type;
  for (int64_t r = blockIdx.x; r < a.s.rows(); r += gridDim.x) {
    const GradRow<A> g = grad_row<A>(a, r);
    const T *x = row_ptr<T>(a.x, r, a.s.L);
    T *out = row_ptr<T>(a.g, r, a.s.L);
    for (int64_t d = threadIdx.x; d < a.s.D; d += 256)
      out[d * a.g.sd] = from_acc<T, A>(grad_value<A>(g, to_acc(x[d * a.x.sd]), (A)a.scale, d == g.t));
  }
}

static bool row_dtype(int32_t dt) { return dt == ACD_FLOAT32 || dt == ACD_FLOAT64 || dt == ACD_FLOAT16; }
static int32_t stat_dtype(int32_t dt) { return dt == ACD_FLOAT64 ? ACD_FLOAT64 : ACD_FLOAT32; }

static acd_status check_logits(const char *op, const acd_desc *logits, int32_t axis, double scale) {
  ACD_TRY(check_desc(logits, "logits"));
  if (!row_dtype(logits->dtype)) return fail(ACD_ERR_DTYPE, "%s: float32, float64 or float16 logits required", op);
  if (axis < 0 || axis >= logits->ndim) return fail(ACD_ERR_AXIS, "%s: axis %d out of range", op, axis);
  if (!(scale > 0.0) || !std::isfinite(scale)) return fail(ACD_ERR_INVALID, "%s: scale must be positive and finite", op);
  if (logits->shape[axis] > INT32_MAX) return fail(ACD_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens", op);
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

template <typename T>
static acd_status launch_logprob(acd_ctx *ctx, const LogprobArgs &a, cudaStream_t s) {
  const int grid = persistent_grid(ctx, k_logprob_rows<T>, 256, 0, a.s.rows());
  k_logprob_rows<T><<<grid, 256, 0, s>>>(a);
  return ACD_OK;
}

template <typename T>
static acd_status launch_logprob_grad(acd_ctx *ctx, const LogprobGradArgs &a, cudaStream_t s) {
  const int grid = persistent_grid(ctx, k_logprob_grad<T>, 256, 0, a.s.rows());
  k_logprob_grad<T><<<grid, 256, 0, s>>>(a);
  return ACD_OK;
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
