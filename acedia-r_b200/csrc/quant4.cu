// Products with weights held in 4 bits, one scale (and zero point) for each
// group of a row:
//   y[o, j] = sum_k s[k/G, o] (q[o, k] - z[k/G, o]) x[k, j]
// The weights of output o are 16 * ceil(in/32) consecutive bytes, two weights
// a byte, the even one low.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <cfloat>

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
// A block takes 64 outputs at a time and a range of the inputs.  One thread
// brings the weights in by TMA through a ring of stages of 64 outputs x 256
// bytes (two tiles of 256 inputs); eight warps multiply them, 16 outputs a warp,
// every second stage each, with the legacy matrix instruction m16n8k16 (a product
// with a few columns is bound by the bytes of its weights: a tcgen05 tile of
// 128 columns would be empty but for these).  The order of the inputs inside
// the instruction is free as long as weights and activations agree, so the four
// threads of a row take 8 consecutive inputs each, one 4-byte word, of every
// 32: a group's inputs never share an instruction with another group's.
//   Weights become exact small integers n - 8 in float16 (bfloat16 for float32
// activations) by putting the four bits into the mantissa of 1024 (128) and
// subtracting; scales are applied to the float32 sums of SUB * 32 inputs:
//   y = sum_groups s sum (n - 8) x  +  sum_groups s (8 - z) sum x,
// the second term from sums of x that are made once.  float32 activations are
// split into three bfloat16 parts that hold all 24 bits, which go in as three
// columns.  The blocks prepare activations for themselves where all of them fit
// into shared memory, or where they are one instruction's columns (NT = 1; then
// a segment of the inputs at a time).  More would cost the blocks more than
// their weights do (64 us on 10007 x 8200 with six float32 columns, 53 us now):
// a kernel of its own prepares them once and they come in with the weights.
//   One float16 column: 4096 x 4096 in 7.0 us (latency: 64 blocks of outputs in
// clusters of two), 131072 x 4096 with a scale and zero point for 64 inputs in
// 76 us, 0.61 of a copy's rate: the schedulers issue in 60% of the cycles, most of
// it the unpacking.  10007 x 8200 with six float32 columns and groups of 32 in
// 54 us, 0.15: 16 warps an SM, 96 registers each, cannot hide the latency of
// eighteen matrix columns' loads, and 157 blocks of outputs fill 296 places
// unevenly.  One block a cluster took 57 us there, two 61, three (the rule's) 54,
// four 65, eight 89.  Scales through shared memory, by the lanes or by
// asynchronous copies of aligned pieces, made the first two slower (82 us).
//   Made for some tens of columns: each set of 32 (float32: 10) reads and unpacks all
// weights again.  4096 x 4096 float16 takes 12.3 us for 8 columns, 33 for 32, 39
// for 128 and 902 for 4096.  Three and four instructions' columns (17 to 32
// float16, 6 to 10 float32) spill, with groups of 32 and zero points up to 1090
// bytes a thread.
constexpr int kRowsPerBlock = 64;
constexpr int kTileBytes = 128;                       // of one output: 256 inputs, 8 chunks of 32
constexpr int kBoxBytes = kRowsPerBlock * kTileBytes;
constexpr int kStageBytes = 2 * kBoxBytes;
constexpr uint64_t kQWaitNs = 1000000000ull;  // 1 s
constexpr int kQWaitCode = 5;

struct Quant4Plan {
  int mblocks;         // blocks of 64 outputs
  int ktiles, tper;    // tiles of 256 inputs: in all, a block of a cluster (even, or all)
  int stages;          // of the ring
  int seg;             // tiles whose activations are in shared memory at once
  int xtile;           // bytes of a tile's activations and sums where k_quant4_x has prepared them
  int vectors;         // columns of x a block (gridDim.y blocks of them)
  int cols;            // matrix columns: vectors, or three for each
  int xcols;           // places for them: 2 more than a multiple of 4, whose 16-byte reads meet no bank twice
  int group;           // chunks of 32 inputs a group
  FastDiv chunks;      // the same, to divide by
  bool wide;           // a tile's scales are one aligned load
};

constexpr int kMaxStages = 4;

// Columns of x that 8 NT matrix columns hold.
template <bool X16, int NT>
struct Q4Vectors { static constexpr int value = X16 ? 8 * NT : 8 * NT / 3; };

// (q & m) | o in one instruction (the truth table of a lop3).
__device__ __forceinline__ uint32_t and_or(uint32_t q, uint32_t m, uint32_t o) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(q), "r"(m), "r"(o));
  return r;
}

// Eight weights of a word: w[i] holds inputs i and i + 4 as n - 8.  (The usual way
// to make floating-point values of small integers: as the last bits of a mantissa
// whose unit is 1.)
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
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The first product of a sum.
template <bool X16>
__device__ __forceinline__ void mma16816_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  if constexpr (X16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// Inputs i and i + 4 of eight side by side, as unpack8 leaves the weights.
__device__ __forceinline__ uint4 interleave8(const uint16_t (&h)[8]) {
  return make_uint4(h[0] | (uint32_t)h[4] << 16, h[1] | (uint32_t)h[5] << 16, h[2] | (uint32_t)h[6] << 16,
                    h[3] | (uint32_t)h[7] << 16);
}

// Eight float32 activations as a bfloat16 part each, side by side like
// interleave8; f is left with what the part cuts off, exact in float32.
__device__ __forceinline__ uint4 take_bf16(float (&f)[8]) {
  uint32_t u[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    u[j] = __float_as_uint(f[j]);
    f[j] -= __uint_as_float(u[j] & 0xFFFF0000u);
  }
  return make_uint4(__byte_perm(u[0], u[4], 0x7632), __byte_perm(u[1], u[5], 0x7632), __byte_perm(u[2], u[6], 0x7632),
                    __byte_perm(u[3], u[7], 0x7632));
}

// The two warps of 16 outputs.
__device__ __forceinline__ void pair_sync(int pair) { asm volatile("bar.sync %0, 64;" ::"r"(2 + pair) : "memory"); }
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Shared memory by its 32-bit address, so that the compiler neither widens it
// nor adds a base to every access.  volatile: not moved over the waits.
template <int OFFSET>
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(r) : "r"(at), "n"(OFFSET) : "memory");
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
  return r;
}

struct Quant4Shared {
  uint64_t full[kMaxStages], empty[kMaxStages];
  int abort;
};

// Activations of the chunks of tiles [tile, tile + n) in the order of the
// instruction's operand, [chunk][thread of a row][column] of 16 bytes, and the
// sums of SUB chunks each, [.][VS].
template <bool X16, int SUB, int VS, bool ZEROS>
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
        xf[it * p.xcols + v] = interleave8(h);
      } else {
        const float *x = static_cast<const float *>(a.x) + at;
        float f[8];
        if (a.xs == 1 && k + 8 <= a.K && aligned_to<char>(x, 16)) {
          const float4 lo = reinterpret_cast<const float4 *>(x)[0], hi = reinterpret_cast<const float4 *>(x)[1];
          f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w;
          f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = k + j < a.K ? x[j * a.xs] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += f[j];
        const bool fine = fabsf(sum) <= FLT_MAX;  // else an infinity or NaN may be among them
        uint4 *to = xf + it * p.xcols + 3 * v;
        if (!fine) {  // a NaN whose set bits would be cut off
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = f[j] != f[j] ? NAN : f[j];
        }
        to[0] = take_bf16(f);
        if (!fine) {  // whole in the first part: Inf - Inf is not to be added
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = f[j] != f[j] ? 0.0f : f[j];
        }
        to[1] = take_bf16(f);
        to[2] = take_bf16(f);
      }
    }
    if (ZEROS) {
      // four items a chunk, side by side; 4 SUB of them divide a warp
#pragma unroll
      for (int q = 1; q < 4 * SUB; q <<= 1) sum += __shfl_xor_sync(~0u, sum, q);
      if (i < items && it % (4 * SUB) == 0) sx[it / (4 * SUB) * VS + v] = sum;
    }
  }
}

// Floats between two outputs' sums in shared memory: 8 more than a multiple of
// 32, so that the 8 rows and 4 column pairs that a warp writes at once lie in
// different banks.
template <int N>
struct SumsStride { static constexpr int value = N <= 8 ? 8 : (N - 8 + 31) / 32 * 32 + 8; };

// The value of an output's column v from its sums.
template <bool X16, int NT, bool ZEROS>
__device__ __forceinline__ float row_value(const float *red, int v) {
  const float y = X16 ? red[v] : red[3 * v] + (red[3 * v + 1] + red[3 * v + 2]);
  return ZEROS ? y + red[8 * NT + v] : y;
}

// The activations of a tile and of a block's columns, as stage_x lays them out.
template <bool X16, int NT, int SUB, bool ZEROS>
__global__ void __launch_bounds__(256) k_quant4_x(Quant4Args a, Quant4Plan p, unsigned char *out) {
  unsigned char *at = out + ((int64_t)blockIdx.y * p.ktiles + blockIdx.x) * p.xtile;
  stage_x<X16, SUB, Q4Vectors<X16, NT>::value, ZEROS>(a, p, blockIdx.x, 1, blockIdx.y * p.vectors,
                                                      reinterpret_cast<uint4 *>(at),
                                                      reinterpret_cast<float *>(at + 512 * p.xcols));
}

template <bool X16, int NT, int SUB, bool ZEROS>
__global__ void __launch_bounds__(288, 2) k_quant4_mma(const __grid_constant__ CUtensorMap map, Quant4Args a,
                                                       Quant4Plan p, const unsigned char *xpre, Control *control) {
  constexpr int VS = Q4Vectors<X16, NT>::value, RED = SumsStride<8 * NT + (ZEROS ? VS : 0)>::value, SLOTS = 8 / SUB;
  const bool prepared = NT > 1 && xpre != nullptr;
  extern __shared__ unsigned char smem[];
  __shared__ Quant4Shared sh;
  // the swizzle goes by the address: stages start on 1024 bytes
  unsigned char *stages = smem + ((1024u - (smem_addr(smem) & 1023u)) & 1023u);
  const int kStages = p.stages;
  const uint32_t stride = prepared ? (uint32_t)(kStageBytes + 2 * p.xtile + 1023) & ~1023u : (uint32_t)kStageBytes;
  float *red = reinterpret_cast<float *>(stages + kStages * stride);  // [64][RED]
  uint4 *xf = reinterpret_cast<uint4 *>(red + kRowsPerBlock * RED);
  float *sx = reinterpret_cast<float *>(xf + p.seg * 32 * p.xcols);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mstep = gridDim.x / C;
  const int v0 = blockIdx.y * p.vectors;
  const int vectors = a.N - v0 < p.vectors ? (int)(a.N - v0) : p.vectors;
  const int t0 = rank * p.tper;
  int nt = p.ktiles - t0;
  nt = nt > p.tper ? p.tper : nt < 0 ? 0 : nt;
  const int ns = (nt + 1) / 2;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 4);
    }
    sh.abort = 0;
    mbar_init_fence();
  }
  __syncthreads();
  if (warp == 8) {
    if (lane == 0) {
      int n = 0, slot = 0;  // stages filled so far, and the next one's place
      uint32_t phase = 1;
      bool go = true;
      for (int mb = blockIdx.x / C; go && mb < p.mblocks; mb += mstep)
        for (int i = 0; i < ns; ++i, ++n) {
          if (n >= kStages &&
              !mbar_wait_thread(&sh.empty[slot], phase, &sh.abort, control, kQWaitCode, kQWaitNs)) {
            go = false;
            break;
          }
          const bool two = 2 * i + 1 < nt;  // a tile past the range is not loaded
          unsigned char *st = stages + slot * stride;
          const uint32_t xbytes = prepared ? (two ? 2 : 1) * p.xtile : 0;
          mbar_arrive_expect_tx(&sh.full[slot], (two ? kStageBytes : kBoxBytes) + xbytes);
          if (prepared)
            asm volatile(
                "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                    smem_addr(st + kStageBytes)),
                "l"(xpre + ((int64_t)blockIdx.y * p.ktiles + t0 + 2 * i) * p.xtile), "r"(xbytes),
                "r"(smem_addr(&sh.full[slot]))
                : "memory");
          tma_load_2d(st, &map, &sh.full[slot], (t0 + 2 * i) * kTileBytes, mb * kRowsPerBlock);
          if (two) tma_load_2d(st + kBoxBytes, &map, &sh.full[slot], (t0 + 2 * i + 1) * kTileBytes, mb * kRowsPerBlock);
          if (++slot == kStages) {
            slot = 0;
            phase ^= 1u;
          }
        }
      // given up: the copies in flight land before the block may end
      if (*reinterpret_cast<volatile int *>(&sh.abort))
        for (int q = n > kStages ? n - kStages : 0; q < n; ++q)
          mbar_wait_bounded(&sh.full[q % kStages], (uint32_t)(q / kStages) & 1u, kQWaitNs);
    }
  } else {
    const int g = lane >> 2, t = lane & 3, odd = warp >> 2, row0 = (warp & 3) * 16;
    // activation columns of this lane; beyond the last one any finite address
    // does, their results are not stored
    uint32_t xcol[NT];
    const uint32_t xstep = 4 * 16 * p.xcols;  // bytes of a chunk
#pragma unroll
    for (int n = 0; n < NT; ++n)
      xcol[n] = (prepared ? smem_addr(stages) + kStageBytes : smem_addr(xf)) + 16 * (t * p.xcols + (n * 8 + g < p.cols ? n * 8 + g : p.cols - 1));
    // scales of a stage: lane 2 r + h holds row r's of its tile h (the next
    // stage's as loaded: converting them would wait for the load)
    float sc[SLOTS], zc[SLOTS];
    uint32_t sn[SLOTS], zn[SLOTS];
    auto load_raw = [&](const void *x, int64_t i) -> uint32_t {
      return a.scale16 ? static_cast<const uint16_t *>(x)[i] : static_cast<const uint32_t *>(x)[i];
    };
    auto value = [&](uint32_t raw) {
      return a.scale16 ? __half2float(__ushort_as_half((uint16_t)raw)) : __uint_as_float(raw);
    };
    const uint32_t ng = (uint32_t)a.ngroups;
    int64_t srow = 0;  // this lane's row of scales
    bool sok = false;
    auto scale_row = [&](int mb) {
      const int64_t o = (int64_t)mb * kRowsPerBlock + row0 + (lane >> 1);
      srow = o * a.ngroups;
      sok = o < a.M;
    };
    auto load_scales = [&](int tile) {
      const uint32_t chunk = (tile + (lane & 1)) * 8;
#pragma unroll
      for (int q = 0; q < SLOTS; ++q) sn[q] = zn[q] = 0;
      if (p.wide) {  // groups of SUB chunks, their number a multiple of a tile's
        const uint32_t gi = chunk / SUB;
        if (sok && gi < ng) {
          using S = Vec<uint16_t, SLOTS>;
          const S s = *reinterpret_cast<const S *>(static_cast<const uint16_t *>(a.scales) + srow + gi);
#pragma unroll
          for (int q = 0; q < SLOTS; ++q) sn[q] = s.v[q];
          if (ZEROS) {
            const S z = *reinterpret_cast<const S *>(static_cast<const uint16_t *>(a.zeros) + srow + gi);
#pragma unroll
            for (int q = 0; q < SLOTS; ++q) zn[q] = z.v[q];
          }
        }
        return;
      }
#pragma unroll
      for (int q = 0; q < SLOTS; ++q) {
        const uint32_t gi = p.chunks.div(chunk + q * SUB);
        if (sok && gi < ng) {
          sn[q] = load_raw(a.scales, srow + gi);
          if (ZEROS) zn[q] = load_raw(a.zeros, srow + gi);
        }
      }
    };
    const uint32_t lane_addr = smem_addr(stages) + (row0 + g) * kTileBytes + (g << 4) + t * 4;
    bool dead = false;
    int staged = -1;     // first tile of the activations in shared memory
    // place and phase of the ring at a block's first stage; stages further on
    const int turn = ns % kStages;
    const uint32_t turns = (uint32_t)(ns / kStages) & 1u;
    int slot0 = 0;
    uint32_t phase0 = 0;
    scale_row(blockIdx.x / C);
    if (odd < ns) load_scales(t0 + 2 * odd);
    for (int mb = blockIdx.x / C; mb < p.mblocks; mb += mstep) {
      float tot[NT][4] = {};
      float corr[ZEROS ? VS : 1] = {};
      int seg0 = 0, slot = slot0 + odd;
      uint32_t phase = phase0;
      if (slot >= kStages) {
        slot -= kStages;
        phase ^= 1u;
      }
      for (int j = 0; j < ns; j += 2) {
        const int i = j + odd, tile = 2 * i;  // this warp's stage, and its tiles of this block's range
        if (!prepared && 2 * j >= seg0 + p.seg) seg0 += p.seg;
        if (!prepared && seg0 != staged) {
          if (staged >= 0) consumer_sync();  // the segment before has been read
          stage_x<X16, SUB, VS, ZEROS>(a, p, t0 + seg0, nt - seg0 < p.seg ? nt - seg0 : p.seg, v0, xf, sx);
          consumer_sync();
          staged = seg0;
        }
        if (i >= ns) continue;
#pragma unroll
        for (int q = 0; q < SLOTS; ++q) {
          sc[q] = value(sn[q]);
          zc[q] = sc[q] * (8.0f - value(zn[q]));
        }
        // the next stage's scales are on their way while this one is worked on
        if (i + 2 < ns) {
          load_scales(t0 + tile + 4);
        } else if (mb + mstep < p.mblocks) {
          scale_row(mb + mstep);
          load_scales(t0 + 2 * odd);
        }
        // once given up, the warps go on without waiting: all of them reach the barriers
        dead = dead || !mbar_wait_warp(&sh.full[slot], phase, &sh.abort, control, kQWaitCode, kQWaitNs);
        uint32_t xt[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) xt[n] = xcol[n] + (prepared ? slot * stride : (tile - seg0) * 8 * xstep);
#pragma unroll 1
        for (int h = 0; h < 2 && tile + h < nt; ++h) {
          if (prepared && h)
#pragma unroll
            for (int n = 0; n < NT; ++n) xt[n] = xcol[n] + slot * stride + p.xtile;
          const uint32_t st = lane_addr + slot * stride + h * kBoxBytes;
          float part[NT][4];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t w0[4], w1[4];
            const uint32_t q0 = lds32<0>(st ^ (c << 4)), q1 = lds32<8 * kTileBytes>(st ^ (c << 4));
            unpack8<X16>(q0, w0);
            unpack8<X16>(q1, w1);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint4 b = lds128(xt[n]);
              xt[n] += xstep;
              if (c % SUB == 0)
                mma16816_zero<X16>(part[n], w0[0], w1[0], w0[1], w1[1], b.x, b.y);
              else
                mma16816<X16>(part[n], w0[0], w1[0], w0[1], w1[1], b.x, b.y);
              mma16816<X16>(part[n], w0[2], w1[2], w0[3], w1[3], b.z, b.w);
            }
            if (c % SUB == SUB - 1) {
              const float s0 = __shfl_sync(~0u, sc[c / SUB], 2 * g + h), s1 = __shfl_sync(~0u, sc[c / SUB], 2 * g + 16 + h);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                tot[n][0] = fmaf(s0, part[n][0], tot[n][0]);
                tot[n][1] = fmaf(s0, part[n][1], tot[n][1]);
                tot[n][2] = fmaf(s1, part[n][2], tot[n][2]);
                tot[n][3] = fmaf(s1, part[n][3], tot[n][3]);
              }
            }
          }
        }
        if (ZEROS && tile + (lane & 1) < nt) {
          const float *s = prepared ? reinterpret_cast<const float *>(stages + slot * stride + kStageBytes +
                                                                 (lane & 1) * p.xtile + 512 * p.xcols)
                               : sx + (tile + (lane & 1) - seg0) * SLOTS * VS;
#pragma unroll
          for (int v = 0; v < VS; ++v) {
            if (v >= vectors) break;
#pragma unroll
            for (int q = 0; q < SLOTS; ++q) corr[v] = fmaf(zc[q], s[q * VS + v], corr[v]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[slot]);
        slot += 2;
        if (slot >= kStages) {
          slot -= kStages;
          phase ^= 1u;
        }
      }
      slot0 += turn;
      phase0 ^= turns;
      if (slot0 >= kStages) {
        slot0 -= kStages;
        phase0 ^= 1u;
      }
      // the odd stages' sums join the even ones'
      auto exchange = [&](auto f) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            f(red[(row0 + g + 8 * (q >> 1)) * RED + n * 8 + 2 * t + (q & 1)], tot[n][q]);
        if (ZEROS && (lane & 1) == 0)
#pragma unroll
          for (int v = 0; v < VS; ++v) f(red[(row0 + (lane >> 1)) * RED + 8 * NT + v], corr[v]);
      };
      if (ZEROS)
#pragma unroll
        for (int v = 0; v < VS; ++v) corr[v] += __shfl_xor_sync(~0u, corr[v], 1);
      if (odd) exchange([](float &r, float x) { r = x; });
      pair_sync(warp & 3);
      if (!odd) {
        exchange([](float &r, float x) { r += x; });
        __syncwarp();
        if (C == 1)
          for (int i = lane; i < 16 * vectors; i += 32) {
            const int r = row0 + (i & 15), v = i >> 4;
            const int64_t o = (int64_t)mb * kRowsPerBlock + r;
            if (o < a.M) store_f(a.out, a.out16, o * a.os + (v0 + v) * a.oc, row_value<X16, NT, ZEROS>(red + r * RED, v));
          }
      }
      if (mb + mstep < p.mblocks) pair_sync(warp & 3);  // red is written again
    }
  }
  if (C == 1) return;
  __syncwarp();
  // the blocks of a cluster hold sums over different inputs of the same outputs
  cluster.sync();
  const int mb = blockIdx.x / C, r0 = rank * kRowsPerBlock / C, rows = (rank + 1) * kRowsPerBlock / C - r0;
  for (int i = threadIdx.x; i < rows * vectors; i += 288) {
    const int v = i / rows, r = r0 + i - v * rows;
    const int64_t o = (int64_t)mb * kRowsPerBlock + r;
    if (o >= a.M) continue;
    float y = 0;
    for (int q = 0; q < C; ++q) y += row_value<X16, NT, ZEROS>(cluster.map_shared_rank(red, q) + r * RED, v);
    store_f(a.out, a.out16, o * a.os + (v0 + v) * a.oc, y);
  }
  cluster.sync();  // no block leaves while its shared memory is read
}

constexpr int kBlockSmem = 112 * 1024;   // two blocks an SM
constexpr int kWholeSmem = 226 * 1024;   // one

template <bool X16, int NT, int SUB, bool ZEROS>
static acd_status launch_mma(acd_ctx *ctx, const Quant4Args &a, Quant4Plan &p, int C, const CUtensorMap &map,
                             cudaStream_t s) {
  constexpr int VS = Q4Vectors<X16, NT>::value, RED = SumsStride<8 * NT + (ZEROS ? VS : 0)>::value;
  // a tile of x: 32 pieces of 16 bytes a column, 8 / SUB sums
  const int per = 32 * 16 * p.xcols + (ZEROS ? 8 / SUB * 4 * VS : 0);
  const int64_t blocks = (int64_t)p.mblocks * C, columns = (a.N + p.vectors - 1) / p.vectors;
  const int fixed = 1024 + kRowsPerBlock * RED * 4;
  int dyn;
  unsigned char *xpre = nullptr;
  // the stages of the ring, and with them the tiles of activations there is room
  // for: all of a block's range, or whole pairs of stages (a warp takes one each)
  auto room = [&](int stages, int smem) {
    const int tiles = (smem - fixed - stages * kStageBytes) / per;
    return tiles >= p.tper ? p.tper : tiles & ~3;
  };
  p.stages = kMaxStages;
  p.seg = room(p.stages, blocks * columns <= ctx->sm_count ? kWholeSmem : kBlockSmem);
  if (NT > 1 && p.seg < p.tper) p.seg = room(p.stages = 3, kBlockSmem);
  // all inputs at once are prepared by the blocks, which mostly have several
  // blocks of outputs to use them for
  if (NT > 1 && p.seg < p.tper) {
    p.seg = 0;
    p.xtile = (per + 15) & ~15;
    const int stage = (kStageBytes + 2 * p.xtile + 1023) & ~1023;
    p.stages = (kBlockSmem - fixed) / stage;
    if (p.stages < 2) p.stages = (kWholeSmem - fixed) / stage;  // one block an SM
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    dyn = fixed + p.stages * stage;
    void *scratch;
    ACD_TRY(get_scratch(ctx, (size_t)columns * p.ktiles * p.xtile, s, &scratch));
    xpre = static_cast<unsigned char *>(scratch);
    k_quant4_x<X16, NT, SUB, ZEROS><<<dim3((unsigned)p.ktiles, (unsigned)columns), 256, 0, s>>>(a, p, xpre);
  } else {
    dyn = fixed + p.stages * kStageBytes + p.seg * per;
  }
  auto kern = k_quant4_mma<X16, NT, SUB, ZEROS>;
  ACD_TRY(allow_smem(ctx, reinterpret_cast<const void *>(kern), dyn));
  int64_t grid = blocks;
  const int64_t resident = (int64_t)ctx->sm_count * (dyn > kBlockSmem ? 1 : 2);
  if (C == 1 && grid > resident) grid = resident;  // persistent
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, (unsigned)columns, 1);
  cfg.blockDim = dim3(288, 1, 1);
  cfg.dynamicSmemBytes = dyn;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ACD_CUDA(cudaLaunchKernelEx(&cfg, kern, map, a, p, (const unsigned char *)xpre, ctx->control));
  return ACD_OK;
}

static acd_status launch_quant4(acd_ctx *ctx, const Quant4Args &a, cudaStream_t s) {
  Quant4Plan p{};
  p.ktiles = (int)((a.K + 255) / 256);
  p.mblocks = (int)((a.M + kRowsPerBlock - 1) / kRowsPerBlock);
  p.group = a.group / 32;
  p.chunks = FastDiv((uint32_t)p.group);
  const int sub = p.group % 4 == 0 ? 4 : p.group % 2 == 0 ? 2 : 1;
  const int slots = 8 / sub;
  p.wide = p.group == sub && a.scale16 && a.ngroups % slots == 0 && aligned_to<char>(a.scales, 2 * slots) &&
           (!a.zeros || aligned_to<char>(a.zeros, 2 * slots));
  // blocks a cluster, along the inputs: an SM works through its blocks' stages
  // and about two stages' time of starting and joining each
  int C = 1;
  int64_t best = INT64_MAX;
  for (int c = 1; c <= 8 && c <= (p.ktiles + 1) / 2; ++c) {
    const int64_t stages = ((p.ktiles + 1) / 2 + c - 1) / c;
    const int64_t cost = ((int64_t)p.mblocks * c + ctx->sm_count - 1) / ctx->sm_count * (stages + 2);
    if (cost < best) {
      best = cost;
      C = c;
    }
  }
  p.tper = C == 1 ? p.ktiles : ((p.ktiles + 1) / 2 + C - 1) / C * 2;
  const int most = a.x16 ? 32 : 10;  // columns of four instructions
  p.vectors = a.N < most ? (int)a.N : most;
  p.cols = a.x16 ? p.vectors : 3 * p.vectors;
  p.xcols = p.cols == 1 ? 1 : (p.cols + 1) / 4 * 4 + 2;
  if ((a.N + most - 1) / most > 65535) return fail(ACD_ERR_UNSUPPORTED, "acd_quant4_matvec: too many columns");
  CUtensorMap map;
  if (!encode_tensor_map_bytes(&map, a.w, a.pitch, a.M, a.pitch, kRowsPerBlock))
    return fail(ACD_ERR_CUDA, "acd_quant4_matvec: the driver rejects the weights' tensor map");
  auto go = [&](auto x16, auto n, auto sb) {
    constexpr bool X = decltype(x16)::value;
    constexpr int NT = decltype(n)::value, SUB = decltype(sb)::value;
    return a.zeros ? launch_mma<X, NT, SUB, true>(ctx, a, p, C, map, s)
                   : launch_mma<X, NT, SUB, false>(ctx, a, p, C, map, s);
  };
  auto grouped = [&](auto x16, auto n) {
    if (sub == 4) return go(x16, n, std::integral_constant<int, 4>());
    if (sub == 2) return go(x16, n, std::integral_constant<int, 2>());
    return go(x16, n, std::integral_constant<int, 1>());
  };
  auto width = [&](auto x16) {
    if (p.cols <= 8) return grouped(x16, std::integral_constant<int, 1>());
    if (p.cols <= 16) return grouped(x16, std::integral_constant<int, 2>());
    if (p.cols <= 24) return grouped(x16, std::integral_constant<int, 3>());
    return grouped(x16, std::integral_constant<int, 4>());
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

// One thread a group (of 16-byte multiples): its range, its scale, its bytes.
// Neighbouring threads take neighbouring outputs, so that an [out, in] matrix
// in column-major order is read along its contiguous axis.  Run once for a
// weight matrix.  W: float32 for float16 and float32 weights, or float64.  The
// scale is worked out in float64 and rounded once; a quotient next to a tie is
// taken in float64, where the quotient of float32 values cannot be rounded onto
// the tie.  (All of it in float64: 2.68 ms for 131072 x 4096 float32, 2.41 ms
// this way, most of it the bytes' strided stores.)
template <typename W>
__global__ void __launch_bounds__(128) k_quant4_encode(Encode4Args a) {
  const int64_t total = a.M * a.ngroups;
  const W largest = sizeof(W) == 8 ? (W)DBL_MAX : (W)FLT_MAX;
  auto load = [&](int64_t o, int64_t k) -> W {
    const int64_t i = o * a.ws + k * a.wc;
    if constexpr (sizeof(W) == 8)
      return static_cast<const double *>(a.w)[i];
    else
      return load_f(a.w, a.dtype == ACD_FLOAT16, i);
  };
  for (int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 128) {
    const int64_t g = i / a.M, o = i - g * a.M;
    const int64_t k0 = g * a.group;
    const int64_t k1 = k0 + a.group < a.K ? k0 + a.group : a.K;
    W lo = 0, hi = 0;
    bool bad = false;
    for (int64_t k = k0; k < k1; ++k) {
      const W v = load(o, k);
      bad |= !(v <= largest && v >= -largest);
      lo = v < lo ? v : lo;
      hi = v > hi ? v : hi;
    }
    // (divided apart: the difference of two finite values may not be finite)
    const double range = a.zeros ? (double)hi / 15 - (double)lo / 15 : (double)(hi > -lo ? hi : -lo) / 7;
    const double most = a.scale16 ? 65504.0 : (double)FLT_MAX;
    double s = a.scale16 ? (double)__half2float(__double2half(range)) : (double)(float)range;
    const bool cut = s > most;  // beyond the type: the weights are cut off
    if (cut) s = most;
    if (bad) s = NAN;
    const bool none = !(s > 0);  // 0 or NaN
    float z = 8;
    if (a.zeros) z = none ? 0.0f : (float)fmin(fmax(rint(-(double)lo / (cut ? range : s)), 0.0), 15.0);
    const int64_t at = o * a.ngroups + g;
    store_f(a.scales, a.scale16, at, (float)s);
    if (a.zeros) store_f(a.zeros, a.scale16, at, z);
    // round(w / s): by a product where that is away from a tie, which it is off by
    // 16 * 2^-22 at most for the quotients that count (a scale below the normal
    // range, or a product above it, compares false)
    const float inv = s >= FLT_MIN ? 1.0f / (float)s : NAN;
    auto quotient = [&](W v) -> float {
      if constexpr (sizeof(W) == 4) {
        const float t = v * inv, n = rintf(t);
        if (fabsf(t - n) < 0.4999f) return n;
      }
      return (float)rint((double)v / s);
    };
    // bytes up to the next group, or to the column's end
    const int64_t b1 = g + 1 == a.ngroups ? a.pitch : k0 / 2 + a.group / 2;
    for (int64_t b = k0 / 2; b < b1; ++b) {
      int byte = 0;
      for (int h = 0; h < 2; ++h) {
        const int64_t k = 2 * b + h;
        float q = z;
        if (k < k1 && !none) q = fminf(fmaxf(quotient(load(o, k)) + z, 0.0f), 15.0f);
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
  auto kern = w->dtype == ACD_FLOAT64 ? k_quant4_encode<double> : k_quant4_encode<float>;
  const int grid = persistent_grid(ctx, kern, 128, 0, (a.M * a.ngroups + 127) / 128);
  kern<<<grid, 128, 0, s>>>(a);
  ACD_CUDA(cudaGetLastError());
  return ACD_OK;
}

}  // extern "C"
