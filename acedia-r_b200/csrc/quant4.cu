// Products with weights held in 4 bits, one scale (and zero point) for each
// group of a row:
//   y[o, j] = sum_k s[k/G, o] (q[o, k] - z[k/G, o]) x[k, j]
// The weights of output o are 16 * ceil(in/32) consecutive bytes, two weights
// a byte, the even one low.
#include "common.cuh"

namespace acd {

struct Quant4Args {
  const uint8_t *w;
  const void *scales, *zeros;
  const void *x;
  void *out;
  int64_t M, K, N;       // outputs, inputs, columns of x
  int64_t pitch, ngroups;
  int64_t xs, xc, os, oc;  // strides of x and out along the vector and over its columns
  int group;
  bool scale16, x16, out16;
};

__device__ __forceinline__ float load_f(const void *p, bool half, int64_t i) {
  return half ? __half2float(static_cast<const __half *>(p)[i]) : static_cast<const float *>(p)[i];
}
__device__ __forceinline__ void store_f(void *p, bool half, int64_t i, float v) {
  if (half)
    static_cast<__half *>(p)[i] = __float2half_rn(v);
  else
    static_cast<float *>(p)[i] = v;
}

// One warp an output and column; a lane takes one byte (two weights) in 32.
__global__ void __launch_bounds__(256) k_quant4_warp(Quant4Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t total = a.M * a.N;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < total; i += (int64_t)gridDim.x * 8) {
    const int64_t o = i % a.M, j = i / a.M;
    float acc = 0;
    for (int64_t b = lane; 2 * b < a.K; b += 32) {
      const int q = a.w[o * a.pitch + b];
      const int64_t k = 2 * b, g = o * a.ngroups + k / a.group;
      const float z = a.zeros ? load_f(a.zeros, a.scale16, g) : 8.0f;
      float v = ((float)(q & 15) - z) * load_f(a.x, a.x16, k * a.xs + j * a.xc);
      if (k + 1 < a.K) v += ((float)(q >> 4) - z) * load_f(a.x, a.x16, (k + 1) * a.xs + j * a.xc);
      acc = fmaf(v, load_f(a.scales, a.scale16, g), acc);
    }
    for (int q = 16; q; q >>= 1) acc += __shfl_xor_sync(~0u, acc, q);
    if (lane == 0) store_f(a.out, a.out16, o * a.os + j * a.oc, acc);
  }
}

struct Encode4Args {
  const void *w;
  int dtype;
  int64_t M, K, ws, wc;  // strides of w over outputs and inputs
  uint8_t *q;
  int64_t pitch, ngroups;
  void *scales, *zeros;
  bool scale16;
  int group;
};

__device__ __forceinline__ float load_w(const Encode4Args &a, int64_t o, int64_t k) {
  const int64_t i = o * a.ws + k * a.wc;
  if (a.dtype == ACD_FLOAT64) return (float)static_cast<const double *>(a.w)[i];
  return load_f(a.w, a.dtype == ACD_FLOAT16, i);
}

// One thread a group (of 16-byte multiples): its range, its scale, its bytes.
// Neighbouring threads take neighbouring outputs, so that an [out, in] matrix
// in column-major order is read along its contiguous axis.  Run once for a
// weight matrix.
__global__ void __launch_bounds__(128) k_quant4_encode(Encode4Args a) {
  const int64_t total = a.M * a.ngroups;
  for (int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 128) {
    const int64_t g = i / a.M, o = i - g * a.M;
    const int64_t k0 = g * a.group;
    const int64_t k1 = k0 + a.group < a.K ? k0 + a.group : a.K;
    float lo = 0, hi = 0;
    bool bad = false;
    for (int64_t k = k0; k < k1; ++k) {
      const float v = load_w(a, o, k);
      bad |= !(fabsf(v) <= 3.402823466e38f);
      lo = fminf(lo, v);
      hi = fmaxf(hi, v);
    }
    float s = a.zeros ? (hi * (1.0f / 15) - lo * (1.0f / 15)) : fmaxf(hi, -lo) / 7.0f;
    if (bad) s = NAN;
    if (a.scale16) s = __half2float(__float2half_rn(s));
    const bool none = !(s > 0);  // 0 or NaN
    float z = 8;
    if (a.zeros) z = none ? 0.0f : fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f);
    const int64_t at = o * a.ngroups + g;
    store_f(a.scales, a.scale16, at, s);
    if (a.zeros) store_f(a.zeros, a.scale16, at, z);
    // bytes up to the next group, or to the column's end
    const int64_t b1 = g + 1 == a.ngroups ? a.pitch : k0 / 2 + a.group / 2;
    for (int64_t b = k0 / 2; b < b1; ++b) {
      int byte = 0;
      for (int h = 0; h < 2; ++h) {
        const int64_t k = 2 * b + h;
        float q = z;
        if (k < k1 && !none) q = fminf(fmaxf(rintf(load_w(a, o, k) / s) + z, 0.0f), 15.0f);
        byte |= (int)q << (4 * h);
      }
      a.q[o * a.pitch + b] = (uint8_t)byte;
    }
  }
}

static bool half_or_float(int32_t dt) { return dt == ACD_FLOAT32 || dt == ACD_FLOAT16; }

// The tensors that hold a quantised matrix of M outputs and K inputs.
static acd_status check_quantised(const char *op, const acd_desc *weights, const acd_desc *scales,
                                  const acd_desc *zeros, int32_t group, int64_t M, int64_t K, int64_t *pitch,
                                  int64_t *ngroups) {
  if (group <= 0 || group % 32) return fail(ACD_ERR_INVALID, "%s: group must be a positive multiple of 32", op);
  ACD_TRY(check_desc(weights, "weights"));
  ACD_TRY(check_desc(scales, "scales"));
  if (zeros) ACD_TRY(check_desc(zeros, "zeros"));
  if (weights->dtype != ACD_INT8) return fail(ACD_ERR_DTYPE, "%s: weights must be int8", op);
  if (!half_or_float(scales->dtype)) return fail(ACD_ERR_DTYPE, "%s: scales must be float16 or float32", op);
  if (zeros && zeros->dtype != scales->dtype)
    return fail(ACD_ERR_DTYPE, "%s: zeros must have the scales' dtype", op);
  *pitch = 16 * ((K + 31) / 32);
  *ngroups = (K + group - 1) / group;
  if (weights->ndim != 2 || weights->shape[0] != *pitch || weights->shape[1] != M)
    return fail(ACD_ERR_SHAPE, "%s: weights must have shape [16 * ceil(in / 32), out] = [%lld, %lld]", op,
                (long long)*pitch, (long long)M);
  for (const acd_desc *d : {scales, zeros})
    if (d && (d->ndim != 2 || d->shape[0] != *ngroups || d->shape[1] != M))
      return fail(ACD_ERR_SHAPE, "%s: scales and zeros must have shape [ceil(in / group), out] = [%lld, %lld]", op,
                  (long long)*ngroups, (long long)M);
  if (!desc_is_contiguous(weights) || !desc_is_contiguous(scales) || (zeros && !desc_is_contiguous(zeros)))
    return fail(ACD_ERR_UNSUPPORTED, "%s: weights, scales and zeros must be contiguous", op);
  if (M > 0 && K > 0 && !aligned_to<char>(desc_ptr(weights), 16))
    return fail(ACD_ERR_UNSUPPORTED, "%s: weights must start on a 16-byte boundary", op);
  if (M > INT32_MAX || K > INT32_MAX) return fail(ACD_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows or columns", op);
  return ACD_OK;
}

}  // namespace acd

using namespace acd;

extern "C" {

acd_status acd_quant4_matvec(acd_ctx *ctx, const acd_desc *out, const acd_desc *weights, const acd_desc *scales,
                             const acd_desc *zeros, const acd_desc *x, int32_t group, acd_stream stream) {
  const char *op = "acd_quant4_matvec";
  if (!ctx) return fail(ACD_ERR_INVALID, "%s: null context", op);
  ACD_TRY(check_desc(x, "x"));
  ACD_TRY(check_desc(out, "out"));
  if (!half_or_float(x->dtype) || !half_or_float(out->dtype))
    return fail(ACD_ERR_DTYPE, "%s: x and out must be float16 or float32", op);
  if (x->ndim < 1 || x->ndim > 2 || out->ndim != x->ndim)
    return fail(ACD_ERR_SHAPE, "%s: x must be [in] or [in, n] and out [out] or [out, n]", op);
  Quant4Args a{};
  a.K = x->shape[0];
  a.M = out->shape[0];
  a.N = x->ndim == 2 ? x->shape[1] : 1;
  if (x->ndim == 2 && out->shape[1] != a.N) return fail(ACD_ERR_SHAPE, "%s: x and out differ in columns", op);
  ACD_TRY(check_quantised(op, weights, scales, zeros, group, a.M, a.K, &a.pitch, &a.ngroups));
  if (a.M == 0 || a.N == 0) return ACD_OK;
  if (a.K == 0) return fail(ACD_ERR_SHAPE, "%s: a matrix without columns", op);
  a.w = reinterpret_cast<const uint8_t *>(desc_ptr(weights));
  a.scales = desc_ptr(scales);
  a.zeros = zeros ? desc_ptr(zeros) : nullptr;
  a.x = desc_ptr(x);
  a.out = desc_ptr(out);
  a.xs = x->stride[0];
  a.xc = x->ndim == 2 ? x->stride[1] : 0;
  a.os = out->stride[0];
  a.oc = out->ndim == 2 ? out->stride[1] : 0;
  a.group = group;
  a.scale16 = scales->dtype == ACD_FLOAT16;
  a.x16 = x->dtype == ACD_FLOAT16;
  a.out16 = out->dtype == ACD_FLOAT16;
  DeviceGuard g(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = persistent_grid(ctx, k_quant4_warp, 256, 0, (a.M * a.N + 7) / 8);
  k_quant4_warp<<<grid, 256, 0, s>>>(a);
  ACD_CUDA(cudaGetLastError());
  return ACD_OK;
}

acd_status acd_quant4_encode(acd_ctx *ctx, const acd_desc *weights, const acd_desc *scales, const acd_desc *zeros,
                             const acd_desc *w, int32_t group, acd_stream stream) {
  const char *op = "acd_quant4_encode";
  if (!ctx) return fail(ACD_ERR_INVALID, "%s: null context", op);
  ACD_TRY(check_desc(w, "w"));
  if (w->dtype != ACD_FLOAT16 && w->dtype != ACD_FLOAT32 && w->dtype != ACD_FLOAT64)
    return fail(ACD_ERR_DTYPE, "%s: w must be float16, float32 or float64", op);
  if (w->ndim != 2) return fail(ACD_ERR_SHAPE, "%s: w must be an [out, in] matrix", op);
  Encode4Args a{};
  a.M = w->shape[0];
  a.K = w->shape[1];
  ACD_TRY(check_quantised(op, weights, scales, zeros, group, a.M, a.K, &a.pitch, &a.ngroups));
  if (a.M == 0 || a.K == 0) return ACD_OK;
  a.w = desc_ptr(w);
  a.dtype = w->dtype;
  a.ws = w->stride[0];
  a.wc = w->stride[1];
  a.q = reinterpret_cast<uint8_t *>(desc_ptr(weights));
  a.scales = desc_ptr(scales);
  a.zeros = zeros ? desc_ptr(zeros) : nullptr;
  a.scale16 = scales->dtype == ACD_FLOAT16;
  a.group = group;
  DeviceGuard g(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = persistent_grid(ctx, k_quant4_encode, 128, 0, (a.M * a.ngroups + 127) / 128);
  k_quant4_encode<<<grid, 128, 0, s>>>(a);
  ACD_CUDA(cudaGetLastError());
  return ACD_OK;
}

}  // extern "C"
