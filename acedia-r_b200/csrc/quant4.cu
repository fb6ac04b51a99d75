// Products with weights held in 4 bits, one scale (and zero point) for each
// group of a row:
//   y[o, j] = sum_k s[k/G, o] (q[o, k] - z[k/G, o]) x[k, j]
// The weights of output o are 16 * ceil(in/32) consecutive bytes, two weights
// a byte, the even one low.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "tma.cuh"

namespace cg = cooperative_groups;

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

// ---------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------
// A block takes 128 outputs and a range of the inputs. One thread brings the
// weights in by TMA, 128 outputs x 128 bytes (256 inputs) at a time through a
// ring of stages; eight warps of 16 outputs each multiply them with the legacy
// matrix instruction m16n8k16 (a product with a few columns is bound by the
// bytes of its weights: a tcgen05 tile of 128 columns would be empty but for
// these).  The order of the inputs inside the instruction is free as long as
// weights and activations agree, so the four threads of a row take 8
// consecutive inputs each, one 4-byte word, of every 32: a group's inputs never
// share an instruction with another group's.
//   Weights become exact small integers n - 8 in float16 (bfloat16 for float32
// activations) by putting the four bits into the mantissa of 1024 (128) and
// subtracting; scales are applied to the float32 sums of 32 inputs:
//   y += s (sum (n - 8) x + (8 - z) sum x).
//   float32 activations are split into three bfloat16 parts that hold all 24
// bits, which go in as three columns.
constexpr int kRowsPerBlock = 128;
constexpr int kTileBytes = 128;               // of one output: 256 inputs, 8 chunks of 32
constexpr int kStageBytes = kRowsPerBlock * kTileBytes;
constexpr int kStages = 4;
constexpr int kXBytes = 44 * 1024;            // activations of a segment, and their sums
constexpr uint64_t kQWaitNs = 1000000000ull;  // 1 s
constexpr int kQWaitCode = 5;

struct Quant4Plan {
  int ktiles, tper;    // tiles of 256 inputs: in all, a block
  int seg;             // tiles whose activations are in shared memory at once
  int vectors;         // columns of x a block (gridDim.y blocks of them)
  int cols;            // matrix columns: vectors, or three for each
  FastDiv chunks;      // chunks of 32 inputs a group
};

template <bool X16>
struct Q4Type { using H2 = __half2; };
template <>
struct Q4Type<false> { using H2 = __nv_bfloat162; };

__device__ __forceinline__ uint32_t and_or(uint32_t q, uint32_t m, uint32_t o) { return (q & m) | o; }

// Eight weights of a word: w[i] holds inputs i and i + 4 as n - 8.
template <bool X16>
__device__ __forceinline__ void unpack8(uint32_t q, uint32_t (&w)[4]) {
  if constexpr (X16) {
    // 1024 + n, and 1024 + 16 n where the bits lie four places up
    const __half2 bias = __float2half2_rn(1032.0f), sixteenth = __float2half2_rn(0.0625f), bias16 = __float2half2_rn(-72.0f);
    uint32_t r[4] = {and_or(q, 0x000F000Fu, 0x64006400u), and_or(q, 0x00F000F0u, 0x64006400u),
                     and_or(q >> 8, 0x000F000Fu, 0x64006400u), and_or(q >> 8, 0x00F000F0u, 0x64006400u)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h = *reinterpret_cast<__half2 *>(&r[i]);
      h = i & 1 ? __hfma2(h, sixteenth, bias16) : __hsub2(h, bias);
      w[i] = *reinterpret_cast<uint32_t *>(&h);
    }
  } else {
    const __nv_bfloat162 bias = __float2bfloat162_rn(136.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t r = and_or(q >> (4 * i), 0x000F000Fu, 0x43004300u);  // 128 + n
      __nv_bfloat162 h = *reinterpret_cast<__nv_bfloat162 *>(&r);
      h = __hsub2(h, bias);
      w[i] = *reinterpret_cast<uint32_t *>(&h);
    }
  }
}

template <bool X16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (X16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Inputs i and i + 4 of eight side by side, as unpack8 leaves the weights.
__device__ __forceinline__ uint4 interleave8(const uint16_t (&h)[8]) {
  return make_uint4(h[0] | (uint32_t)h[4] << 16, h[1] | (uint32_t)h[5] << 16, h[2] | (uint32_t)h[6] << 16,
                    h[3] | (uint32_t)h[7] << 16);
}

// Truncates to bfloat16; what is cut off is exact in float32.  Infinities and
// NaN are whole in the first part.
__device__ __forceinline__ uint16_t take_bf16(float &x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7F800000u) == 0x7F800000u) {
    x = 0.0f;
    return (uint16_t)((u >> 16) | ((u & 0x7FFFFFu) ? 0x40u : 0u));
  }
  x -= __uint_as_float(u & 0xFFFF0000u);
  return (uint16_t)(u >> 16);
}

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

struct Quant4Shared {
  uint64_t full[kStages], empty[kStages];
  int abort;
};

// Activations of the chunks of tiles [tile, tile + n) in the order of the
// instruction's operand, [chunk][thread of a row][column] of 16 bytes, and
// their sums, [chunk][8 NT].
template <bool X16, int NT>
__device__ __forceinline__ void stage_x(const Quant4Args &a, const Quant4Plan &p, int tile, int n, int v0, uint4 *xf,
                                        float *sx) {
  const int vectors = a.N - v0 < p.vectors ? (int)(a.N - v0) : p.vectors;
  const int per = n * 32, items = per * vectors;  // 8 inputs an item, four items a chunk
  for (int i = threadIdx.x; i < ((items + 31) & ~31); i += 256) {
    float sum = 0;
    const int v = i < items ? i / per : 0, it = i < items ? i - v * per : 0;
    if (i < items) {
      const int64_t k = (int64_t)tile * 256 + it * 8;
      const int64_t at = k * a.xs + (v0 + v) * a.xc;
      if constexpr (X16) {
        const __half *x = static_cast<const __half *>(a.x) + at;
        uint16_t h[8];
        if (a.xs == 1 && k + 8 <= a.K && aligned_to<char>(x, 16)) {
          const Vec<uint16_t, 8> w = *reinterpret_cast<const Vec<uint16_t, 8> *>(x);
#pragma unroll
          for (int j = 0; j < 8; ++j) h[j] = w.v[j];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            h[j] = k + j < a.K ? reinterpret_cast<const uint16_t *>(x)[j * a.xs] : (uint16_t)0;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += __half2float(__ushort_as_half(h[j]));
        xf[it * p.cols + v] = interleave8(h);
      } else {
        const float *x = static_cast<const float *>(a.x) + at;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          f[j] = k + j < a.K ? x[j * a.xs] : 0.0f;
          sum += f[j];
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          uint16_t h[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) h[j] = take_bf16(f[j]);
          xf[it * p.cols + 3 * v + q] = interleave8(h);
        }
      }
    }
    sum += __shfl_xor_sync(~0u, sum, 1);
    sum += __shfl_xor_sync(~0u, sum, 2);
    if (i < items && (it & 3) == 0) {
      float *s = sx + (it >> 2) * (8 * NT) + (X16 ? v : 3 * v);
      s[0] = sum;
      if (!X16) s[1] = s[2] = 0.0f;
    }
  }
}

template <bool X16, int NT, bool ZEROS>
__global__ void __launch_bounds__(288, 2) k_quant4_mma(const __grid_constant__ CUtensorMap map, Quant4Args a,
                                                       Quant4Plan p, Control *control) {
  extern __shared__ unsigned char smem[];
  __shared__ Quant4Shared sh;
  // the swizzle goes by the address: stages start on 1024 bytes
  unsigned char *stages = smem + ((1024u - (smem_addr(smem) & 1023u)) & 1023u);
  uint4 *xf = reinterpret_cast<uint4 *>(stages + kStages * kStageBytes);
  float *sx = reinterpret_cast<float *>(xf + p.seg * 32 * p.cols);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t o0 = (int64_t)(blockIdx.x / C) * kRowsPerBlock;
  const int v0 = blockIdx.y * p.vectors;
  const int t0 = rank * p.tper;
  int nt = p.ktiles - t0;
  nt = nt > p.tper ? p.tper : nt < 0 ? 0 : nt;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 8);
    }
    sh.abort = 0;
    mbar_init_fence();
  }
  __syncthreads();
  float tot[NT][4] = {};
  if (warp == 8) {
    if (lane == 0) {
      int i = 0;
      for (; i < nt; ++i) {
        const int slot = i % kStages;
        if (i >= kStages && !mbar_wait_thread(&sh.empty[slot], (uint32_t)(i / kStages - 1) & 1u, &sh.abort, control,
                                              kQWaitCode, kQWaitNs))
          break;
        mbar_arrive_expect_tx(&sh.full[slot], kStageBytes);
        tma_load_2d(stages + slot * kStageBytes, &map, &sh.full[slot], (t0 + i) * kTileBytes, (int)o0);
      }
      // given up: the copies in flight land before the block may end
      if (*reinterpret_cast<volatile int *>(&sh.abort))
        for (int q = i > kStages ? i - kStages : 0; q < i; ++q)
          mbar_wait_bounded(&sh.full[q % kStages], (uint32_t)(q / kStages) & 1u, kQWaitNs);
    }
  } else {
    const int g = lane >> 2, t = lane & 3;
    // Scales of a tile: lane 2 r + h holds row r's chunks 4 h .. 4 h + 3.
    float sc[4], zc[4];
    const int64_t srow = o0 + warp * 16 + (lane >> 1);
    auto load_scales = [&](int tile) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t gi = p.chunks.div((uint32_t)(tile * 8 + (lane & 1) * 4 + q));
        const bool ok = srow < a.M && gi < a.ngroups;
        const int64_t at = srow * a.ngroups + gi;
        sc[q] = ok ? load_f(a.scales, a.scale16, at) : 0.0f;
        if (ZEROS) zc[q] = ok ? sc[q] * (8.0f - load_f(a.zeros, a.scale16, at)) : 0.0f;
      }
    };
    bool dead = false;
    for (int i = 0; i < nt; ++i) {
      if (i % p.seg == 0) {
        if (i) consumer_sync();  // the segment before has been read
        stage_x<X16, NT>(a, p, t0 + i, nt - i < p.seg ? nt - i : p.seg, v0, xf, sx);
        consumer_sync();
      }
      load_scales(t0 + i);
      const int slot = i % kStages;
      // once given up, the warps go on without waiting: all of them reach the barriers
      dead = dead || !mbar_wait_warp(&sh.full[slot], (uint32_t)(i / kStages) & 1u, &sh.abort, control, kQWaitCode,
                                     kQWaitNs);
      const unsigned char *st = stages + slot * kStageBytes + (warp * 16 + g) * kTileBytes + t * 4;
      const uint4 *xc = xf + (i % p.seg) * 32 * p.cols + t * p.cols;
      const float *sc_x = sx + (i % p.seg) * 8 * (8 * NT) + 2 * t;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint32_t q0 = *reinterpret_cast<const uint32_t *>(st + ((c ^ g) << 4));
        const uint32_t q1 = *reinterpret_cast<const uint32_t *>(st + 8 * kTileBytes + ((c ^ g) << 4));
        uint32_t w0[4], w1[4];
        unpack8<X16>(q0, w0);
        unpack8<X16>(q1, w1);
        const float s0 = __shfl_sync(~0u, sc[c & 3], 2 * g + (c >> 2)), s1 = __shfl_sync(~0u, sc[c & 3], 2 * g + 16 + (c >> 2));
        float z0 = 0, z1 = 0;
        if (ZEROS) {
          z0 = __shfl_sync(~0u, zc[c & 3], 2 * g + (c >> 2));
          z1 = __shfl_sync(~0u, zc[c & 3], 2 * g + 16 + (c >> 2));
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint4 b = make_uint4(0, 0, 0, 0);
          if (n * 8 + g < p.cols) b = xc[c * 4 * p.cols + n * 8 + g];
          float part[4] = {};
          mma16816<X16>(part, w0[0], w1[0], w0[1], w1[1], b.x, b.y);
          mma16816<X16>(part, w0[2], w1[2], w0[3], w1[3], b.z, b.w);
          tot[n][0] = fmaf(s0, part[0], tot[n][0]);
          tot[n][1] = fmaf(s0, part[1], tot[n][1]);
          tot[n][2] = fmaf(s1, part[2], tot[n][2]);
          tot[n][3] = fmaf(s1, part[3], tot[n][3]);
          if (ZEROS) {
            const float2 x = *reinterpret_cast<const float2 *>(sc_x + c * (8 * NT) + n * 8);
            tot[n][0] = fmaf(z0, x.x, tot[n][0]);
            tot[n][1] = fmaf(z0, x.y, tot[n][1]);
            tot[n][2] = fmaf(z1, x.x, tot[n][2]);
            tot[n][3] = fmaf(z1, x.y, tot[n][3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[slot]);
    }
  }
  // the blocks of a cluster hold sums of different inputs of the same outputs
  __syncthreads();
  float *red = reinterpret_cast<float *>(stages);  // [128][8 NT], over the stages
  if (warp < 8) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        red[(warp * 16 + g + 8 * (q >> 1)) * (8 * NT) + n * 8 + 2 * t + (q & 1)] = tot[n][q];
  }
  if (C > 1)
    cluster.sync();
  else
    __syncthreads();
  const int rows = kRowsPerBlock / C;
  const int vectors = a.N - v0 < p.vectors ? (int)(a.N - v0) : p.vectors;
  for (int i = threadIdx.x; i < rows * vectors; i += 288) {
    const int v = i / rows, r = rank * rows + i - v * rows;
    const int64_t o = o0 + r;
    if (o >= a.M) continue;
    float y = 0;
    for (int q = 0; q < C; ++q) {
      const float *other = C > 1 ? cluster.map_shared_rank(red, q) : red;
      if (X16) {
        y += other[r * (8 * NT) + v];
      } else {
#pragma unroll
        for (int w = 2; w >= 0; --w) y += other[r * (8 * NT) + 3 * v + w];
      }
    }
    store_f(a.out, a.out16, o * a.os + (v0 + v) * a.oc, y);
  }
  if (C > 1) cluster.sync();  // no block leaves while its shared memory is read
}

template <bool X16, int NT, bool ZEROS>
static acd_status launch_mma(acd_ctx *ctx, const Quant4Args &a, Quant4Plan &p, int cluster, const CUtensorMap &map,
                             cudaStream_t s) {
  // a tile of x: 32 pieces of 16 bytes a column, 8 sums a column
  const int per = 32 * 16 * p.cols + 8 * 4 * 8 * NT;
  p.seg = kXBytes / per;
  if (p.seg > p.tper) p.seg = p.tper;
  const int dyn = 1024 + kStages * kStageBytes + p.seg * per;
  auto kern = k_quant4_mma<X16, NT, ZEROS>;
  ACD_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, dyn));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.M + kRowsPerBlock - 1) / kRowsPerBlock * cluster),
                     (unsigned)((a.N + p.vectors - 1) / p.vectors), 1);
  cfg.blockDim = dim3(288, 1, 1);
  cfg.dynamicSmemBytes = dyn;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ACD_CUDA(cudaLaunchKernelEx(&cfg, kern, map, a, p, ctx->control));
  return ACD_OK;
}

static acd_status launch_quant4(acd_ctx *ctx, const Quant4Args &a, cudaStream_t s) {
  Quant4Plan p{};
  p.ktiles = (int)((a.K + 255) / 256);
  p.chunks = FastDiv((uint32_t)(a.group / 32));
  // blocks along the inputs: while two blocks an SM are not reached
  const int64_t mblocks = (a.M + kRowsPerBlock - 1) / kRowsPerBlock;
  int C = 1;
  while (C < 8 && mblocks * C * 2 <= ctx->sm_count * 2 && p.ktiles >= C * 2) C *= 2;
  p.tper = (p.ktiles + C - 1) / C;
  const int most = a.x16 ? 32 : 10;  // columns of four instructions
  p.vectors = a.N < most ? (int)a.N : most;
  p.cols = a.x16 ? p.vectors : 3 * p.vectors;
  if ((a.N + most - 1) / most > 65535) return fail(ACD_ERR_UNSUPPORTED, "acd_quant4_matvec: too many columns");
  CUtensorMap map;
  if (!encode_tensor_map_bytes(&map, a.w, a.pitch, a.M, a.pitch, kRowsPerBlock))
    return fail(ACD_ERR_CUDA, "acd_quant4_matvec: the driver rejects the weights' tensor map");
  auto go = [&](auto x16, auto n) {
    return a.zeros ? launch_mma<decltype(x16)::value, decltype(n)::value, true>(ctx, a, p, C, map, s)
                   : launch_mma<decltype(x16)::value, decltype(n)::value, false>(ctx, a, p, C, map, s);
  };
  auto width = [&](auto x16) {
    if (p.cols <= 8) return go(x16, std::integral_constant<int, 1>());
    if (p.cols <= 16) return go(x16, std::integral_constant<int, 2>());
    if (p.cols <= 24) return go(x16, std::integral_constant<int, 3>());
    return go(x16, std::integral_constant<int, 4>());
  };
  return a.x16 ? width(std::true_type()) : width(std::false_type());
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
  ACD_TRY(launch_quant4(ctx, a, s));
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
