// Shared by the language-model row operators (logprob.cu, norm.cu): the view
// of a tensor as rows along one axis, the accumulator type of an element type
// and the checks of their small tensors.
#pragma once

#include <cfloat>
#include <climits>

#include "common.cuh"

namespace acd {

// Element type -> the type its sums and statistics are held in.
template <typename T>
struct AccOf { using type = float; };
template <>
struct AccOf<double> { using type = double; };

__device__ __forceinline__ float to_acc(float x) { return x; }
__device__ __forceinline__ float to_acc(__half x) { return __half2float(x); }
__device__ __forceinline__ double to_acc(double x) { return x; }
// One rounding to the storage type.
template <typename T, typename A>
__device__ __forceinline__ T from_acc(A x) { return (T)x; }
template <>
__device__ __forceinline__ __half from_acc<__half, float>(float x) { return __float2half_rn(x); }

// Fused multiply-add and exponentials of the accumulator type.  (The library
// is compiled without contraction, so a fused product is asked for by name.)
__device__ __forceinline__ float fma_a(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_a(double a, double b, double c) { return fma(a, b, c); }

// Two float32 values in one register pair: one instruction for both.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// As many accumulator values as one instruction takes: two float32, one float64.
template <typename A>
struct Pk;
template <>
struct Pk<float> {
  static constexpr int N = 2;
  uint64_t v;
  static __device__ __forceinline__ Pk from(const float *f) { return {pack2(f[0], f[1])}; }
  static __device__ __forceinline__ Pk all(float x) { return {pack2(x, x)}; }
  __device__ __forceinline__ void to(float *f) const { unpack2(v, f[0], f[1]); }
  __device__ __forceinline__ float sum() const {
    float a, b;
    unpack2(v, a, b);
    return a + b;
  }
};
__device__ __forceinline__ Pk<float> pmul(Pk<float> a, Pk<float> b) { return {mul2(a.v, b.v)}; }
__device__ __forceinline__ Pk<float> pfma(Pk<float> a, Pk<float> b, Pk<float> c) { return {fma2(a.v, b.v, c.v)}; }
template <>
struct Pk<double> {
  static constexpr int N = 1;
  double v;
  static __device__ __forceinline__ Pk from(const double *f) { return {f[0]}; }
  static __device__ __forceinline__ Pk all(double x) { return {x}; }
  __device__ __forceinline__ void to(double *f) const { f[0] = v; }
  __device__ __forceinline__ double sum() const { return v; }
};
__device__ __forceinline__ Pk<double> pmul(Pk<double> a, Pk<double> b) { return {a.v * b.v}; }
__device__ __forceinline__ Pk<double> pfma(Pk<double> a, Pk<double> b, Pk<double> c) { return {fma(a.v, b.v, c.v)}; }

// V elements as they lie in memory; float16 pairs as words, so that
// they take no more registers than bytes until they are widened.
template <typename T, int V>
struct Piece {
  Vec<T, V> d;
  template <typename A>
  __device__ __forceinline__ void widen(A *f) const {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = to_acc(d.v[j]);
  }
  __device__ __forceinline__ void set(int j, T x) { d.v[j] = x; }
  template <typename A>
  __device__ __forceinline__ void round(const A *f) {
#pragma unroll
    for (int j = 0; j < V; ++j) d.v[j] = from_acc<T, A>(f[j]);
  }
};
template <int V>
struct Half2Piece {
  Vec<uint32_t, V / 2> d;
  __device__ __forceinline__ void widen(float *f) const {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&d.v[j / 2]));
      f[j] = p.x;
      f[j + 1] = p.y;
    }
  }
  __device__ __forceinline__ void round(const float *f) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const __half2 h = __floats2half2_rn(f[j], f[j + 1]);
      d.v[j / 2] = *reinterpret_cast<const uint32_t *>(&h);
    }
  }
  __device__ __forceinline__ void set(int j, __half x) {
    const uint32_t h = __half_as_ushort(x);
    d.v[j / 2] = j % 2 ? (d.v[j / 2] & 0xFFFFu) | h << 16 : (d.v[j / 2] & 0xFFFF0000u) | h;
  }
};
template <>
struct Piece<__half, 2> : Half2Piece<2> {};
template <>
struct Piece<__half, 4> : Half2Piece<4> {};
template <>
struct Piece<__half, 8> : Half2Piece<8> {};

// A tensor as rows: element d of row r = l + L*o lies at p + l*sl + d*sd + o*so.
struct Rows {
  void *p = nullptr;
  int64_t sl = 0, sd = 0, so = 0;
};

// Geometry shared by the tensors of one call.
struct RowShape {
  int64_t L = 1, D = 1, O = 1;
  __host__ __device__ int64_t rows() const { return L * O; }
};

// (Rows are counted in 31 bits: a 64-bit division is many times a 32-bit one.  The
// branch keeps the division, some 100 cycles, away from rows that need none.)
template <typename T>
__device__ __forceinline__ T *row_ptr(const Rows &v, int64_t r, int64_t L) {
  int64_t at = r * v.so;
  if (L != 1) {
    asm volatile("" ::: "memory");  // not turned into a selection of both results
    const uint32_t o = (uint32_t)r / (uint32_t)L, l = (uint32_t)r - o * (uint32_t)L;
    at = l * v.sl + o * v.so;
  }
  return static_cast<T *>(v.p) + at;
}

// Views `d` around `axis`; the axes before it, and those after it, must each
// merge into one (extents of 1 aside).  False when they do not.
inline bool split_rows(const acd_desc *d, int axis, RowShape &s, Rows &v) {
  auto merge = [&](int d0, int d1, int64_t &n, int64_t &st) {
    n = 1;
    st = 0;
    int64_t next = 0;
    bool first = true;
    for (int k = d0; k < d1; ++k) {
      if (d->shape[k] == 1) continue;
      if (first) st = d->stride[k];
      if (!first && d->stride[k] != next) return false;
      next = d->stride[k] * d->shape[k];
      n *= d->shape[k];
      first = false;
    }
    return true;
  };
  if (!merge(0, axis, s.L, v.sl) || !merge(axis + 1, d->ndim, s.O, v.so)) return false;
  s.D = d->shape[axis];
  v.sd = d->stride[axis];
  v.p = desc_ptr(d);
  return true;
}

// A row tensor of `like` along `axis`: extents of `like` without the axis, or
// with `k` on it; contiguous.
inline acd_status check_row_tensor(const char *op, const char *name, const acd_desc *d, const acd_desc *like, int axis,
                                   int64_t k = 1) {
  ACD_TRY(check_desc(d, name));
  bool ok = false;
  if (d->ndim == like->ndim) {
    ok = true;
    for (int i = 0; i < like->ndim; ++i) ok = ok && d->shape[i] == (i == axis ? k : like->shape[i]);
  }
  if (!ok && k == 1 && d->ndim == like->ndim - 1) {
    ok = true;
    for (int i = 0; i < d->ndim; ++i) ok = ok && d->shape[i] == like->shape[i < axis ? i : i + 1];
  }
  // one row: a one-element tensor of any rank, as the reductions return it
  if (!ok && k == 1 && like->ndim == 1) ok = desc_numel(d) == 1;
  if (!ok) return fail(ACD_ERR_SHAPE, "%s: %s does not have one entry a row", op, name);
  if (!desc_is_contiguous(d)) return fail(ACD_ERR_UNSUPPORTED, "%s: %s must be contiguous", op, name);
  return ACD_OK;
}

inline bool same_shape(const acd_desc *a, const acd_desc *b) {
  if (a->ndim != b->ndim) return false;
  for (int k = 0; k < a->ndim; ++k)
    if (a->shape[k] != b->shape[k]) return false;
  return true;
}

// INT32 or INT64 values read and written as int64.
__device__ __forceinline__ int64_t load_index(const void *p, bool wide, int64_t i) {
  return wide ? static_cast<const int64_t *>(p)[i] : (int64_t) static_cast<const int32_t *>(p)[i];
}
__device__ __forceinline__ void store_index(void *p, bool wide, int64_t i, int64_t v) {
  if (wide)
    static_cast<int64_t *>(p)[i] = v;
  else
    static_cast<int32_t *>(p)[i] = (int32_t)v;
}

// A row is read in pieces of V elements that start on 16-byte boundaries; it may
// itself start (by `row_shift` elements) and end inside a piece.
template <typename T, int V>
__device__ __forceinline__ int row_shift(const T *x) {
  return V == 1 ? 0 : (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % V);
}

// Elements first .. first + V - 1 of a row of D, as far as the row has them.
// V = 1: any stride.
template <typename T, typename A, int V>
__device__ __forceinline__ void store_piece(T *x, int64_t sd, int first, int D, const A *v) {
  if (V > 1 && first >= 0 && first + V <= D) {
    Piece<T, V> w;
    w.round(v);
    *reinterpret_cast<Piece<T, V> *>(x + first) = w;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (first + j >= 0 && first + j < D) x[(first + j) * sd] = from_acc<T, A>(v[j]);
  }
}

// Whether the pieces of V elements of `size` bytes of x and g coincide in every
// row: same offset in 16 bytes, strides sx, sg that differ by whole pieces.
inline bool pieces_match(const Rows &x, const Rows &g, int64_t sx, int64_t sg, int V, int size) {
  const uintptr_t px = reinterpret_cast<uintptr_t>(x.p), pg = reinterpret_cast<uintptr_t>(g.p);
  return (px - pg) % (uintptr_t)(V * size) == 0 && (sx - sg) % V == 0 && (x.so - g.so) % V == 0;
}

}  // namespace acd
