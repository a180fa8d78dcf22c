// cwg_fp8.cu -- e4m3 quantiser and matrix product with fp32 scales per block of 128
// (cwg_fp8_quantize, cwg_fp8_matmul).
//
//   y[i][j] = act(bias[j] + sum_kb as[i][kb] ws[j / 128][kb] sum_{k in kb} a[i][k] w[j][k])
//
// The inner sum over one block of 128 runs on the tensor cores (kind::f8f6f4, e4m3,
// fp32 accumulators in tensor memory); as soon as a block is done, the promoting
// warps read it back, scale it and add it to fp32 registers, while the next block's
// MMAs fill another accumulator.  The scales differ from block to block, so no sum
// can run across blocks inside the tensor core.
#include <cstdint>

#include <cuda.h>
#include <cuda_fp8.h>

#include "../../include/cwg.h"
#include "cwg_seq.cuh"
#include "cwg_tcgen05.cuh"

namespace cwg {
namespace fp8 {

using namespace tc;
using seq::pack1;

__device__ unsigned int g_fp8_status;

__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *abort) {
  return tc::mbar_wait(bar, parity, abort, &g_fp8_status);
}

// ---- quantiser ---------------------------------------------------------------------
constexpr float kE4m3Max = 448.f;
constexpr float kScaleMin = 1.17549435e-38f;  // 2^-126

__device__ __forceinline__ float scale_of(uint32_t amax) {
  const float s = __fdiv_rn(__uint_as_float(amax), kE4m3Max);
  return s < kScaleMin ? kScaleMin : s;  // NaN stays
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const __nv_fp8x2_storage_t lo =
      __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi =
      __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)lo | (uint32_t)hi << 16;
}
// Codes of v / s, the quotients rounded to fp32 first.  With r = 1 / s correctly rounded
// and q = v r, one correction q + (v - q s) r gives the correctly rounded quotient
// (Markstein 1990) as long as v - q s is exact: 1.5 two-wide instructions per element
// instead of a division.  It is computed with the opposite sign, whose rounding is the same,
// so that a zero keeps its own: v - q s of an exact quotient is +0, which would turn q = -0
// into +0, but -0 = +0 (-r) leaves either -q.  A test of the interval around v r, with the
// division only where two codes are possible, does not pay for bf16 data: its quotients are
// often exactly between two codes (30.5 against 16.9 us for 8192 x 4096).
__device__ __forceinline__ uint32_t codes4(const float *v, float s, float r) {
  using namespace seq;
  const F2 minus_r = f2(-r, -r), ss = f2(s, s);
  float2 c[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const F2 x = f2(v[2 * i], v[2 * i + 1]), q = mul2(x, minus_r);
    c[i] = halves(fma2(fma2(q, ss, x), minus_r, q));
  }
  return e4m3x4(c[0].x, c[0].y, c[1].x, c[1].y) ^ 0x80808080u;
}
__device__ __noinline__ uint32_t divided4(float a, float b, float c, float d, float s) {
  return e4m3x4(__fdiv_rn(a, s), __fdiv_rn(b, s), __fdiv_rn(c, s), __fdiv_rn(d, s));
}

struct QuantArgs {
  const void *x;
  uint8_t *q;
  float *scale;
  size_t ldx, ldq, lds;
  int rows, cols, kblocks;
  long long groups;
};

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// 8 consecutive elements of a row, zeros past the end, as they are in memory: whole 16-byte
// vectors, of which a row has a whole number.
template <typename T>
struct Eight {
  static constexpr int E = 16 / (int)sizeof(T);
  uint4 raw[8 / E];
  __device__ __forceinline__ void load(const T *p, int n) {
#pragma unroll
    for (int i = 0; i < 8; i += E)
      raw[i / E] = i < n ? seq::load_raw<T, E>(p + i) : seq::zero_raw<T, E>();
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; i += E) {
      float f[E];
      seq::unpack(raw[i / E], f);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i + e] = f[e];
    }
  }
  // Largest magnitude, by its bits: NaN is above infinity, infinity above any number.
  __device__ __forceinline__ uint32_t amax() const {
    if constexpr (sizeof(T) == 2) {
      const uint32_t k = 0x7fff7fffu;
      const uint32_t m = __vmaxu2(__vmaxu2(raw[0].x & k, raw[0].y & k),
                                  __vmaxu2(raw[0].z & k, raw[0].w & k));
      return max(m << 16, m & 0xffff0000u);
    } else {
      float v[8];
      get(v);
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
      return m;
    }
  }
};
// Codes of N values.  Scales near the end of the range, where the correction's remainder
// would underflow, and infinite or NaN ones take the division.
template <int N>
__device__ __forceinline__ void codes_of(const float (&v)[N], float s, uint32_t (&w)[N / 4]) {
  if (s > 0x1p-90f && s < 0x1p127f) {
    const float r = __frcp_rn(s);
#pragma unroll
    for (int k = 0; k < N; k += 4) w[k / 4] = codes4(v + k, s, r);
  } else {
#pragma unroll
    for (int k = 0; k < N; k += 4) w[k / 4] = divided4(v[k], v[k + 1], v[k + 2], v[k + 3], s);
  }
}
// The same of four pieces, which are unpacked one at a time (all at once they take 60
// registers a thread instead of 40: 18.8 against 16.8 us for 8192 x 4096 bf16).
template <typename T>
__device__ __forceinline__ void codes_of(const Eight<T> (&v)[4], float s, uint32_t (&w)[8]) {
  if (s > 0x1p-90f && s < 0x1p127f) {
    const float r = __frcp_rn(s);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float f[8];
      v[k].get(f);
      w[2 * k] = codes4(f, s, r);
      w[2 * k + 1] = codes4(f + 4, s, r);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float f[8];
      v[k].get(f);
      w[2 * k] = divided4(f[0], f[1], f[2], f[3], s);
      w[2 * k + 1] = divided4(f[4], f[5], f[6], f[7], s);
    }
  }
}
// The codes of 8 elements of a row, of which n are the matrix's.
__device__ __forceinline__ void store8(uint8_t *q, uint32_t a, uint32_t b, int n) {
  if (n >= 8) {
    *reinterpret_cast<uint2 *>(q) = make_uint2(a, b);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) q[i] = (uint8_t)((i < 4 ? a >> 8 * i : b >> 8 * (i - 4)) & 0xff);
  }
}

// Groups of 1 x 128.  VEC: four lanes per group, 32 elements a lane, all loaded before the
// first is used; per group one division, one reciprocal and one index division then serve
// 32 elements of each lane.  Else a warp per group, neighbouring lanes on neighbouring
// elements.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows(const QuantArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kLanes = VEC ? 4 : 32;
  const unsigned g = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool ok = g < (unsigned)a.groups;
  const int row = ok ? (int)(g / (unsigned)a.kblocks) : 0;
  const int kb = ok ? (int)g - row * a.kblocks : 0;
  const T *x = static_cast<const T *>(a.x) + (size_t)row * a.ldx + kb * 128;
  uint8_t *q = a.q + (size_t)row * a.ldq + kb * 128;
  const int n = ok ? a.cols - kb * 128 : 0;  // the group's elements, and those behind it
  uint32_t m = 0;
  auto scale_group = [&]() {  // from the lanes' largest magnitudes
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float s = scale_of(m);
    if (ok && lane == 0) a.scale[(size_t)row * a.lds + kb] = s;
    return m ? s : 1.f;  // zeros, and lanes without a group, need no slow division
  };
  if constexpr (VEC) {
    Eight<T> v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k].load(x + k * 32 + lane * 8, n - k * 32 - lane * 8);
#pragma unroll
    for (int k = 0; k < 4; ++k) m = max(m, v[k].amax());
    uint32_t w[8];
    codes_of(v, scale_group(), w);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = k * 32 + lane * 8;
      if (c < n) store8(q + c, w[2 * k], w[2 * k + 1], n - c);
    }
  } else {
    float f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[k] = k * 32 + lane < n ? to_f32(x[k * 32 + lane]) : 0.f;
      m = max(m, abs_bits(f[k]));
    }
    uint32_t w[1];
    codes_of(f, scale_group(), w);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k * 32 + lane < n) q[k * 32 + lane] = (uint8_t)(w[0] >> 8 * k);
  }
}

// One CTA per block of 128 x 128, 32 elements a thread held in registers: four pieces of 8
// columns (VEC), or one column of 32 rows, so that neighbouring threads read and write
// neighbouring elements (1000 x 1543 fp32: 7.4 us with pieces of 8 there too, 5.2 so).
template <typename T, bool VEC>
__global__ void __launch_bounds__(512) quantize_blocks(const QuantArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ uint32_t s_max[16];
  const int kb = blockIdx.x % a.kblocks, rb = blockIdx.x / a.kblocks;
  const int tid = threadIdx.x;
  const int c = kb * 128 + (VEC ? tid % 16 * 8 : tid % 128);
  const int r0 = rb * 128 + (VEC ? tid / 16 : tid / 128);
  const int n = a.cols - c;
  const T *x = static_cast<const T *>(a.x) + c;
  uint8_t *q = a.q + c;
  uint32_t m = 0, w[8];
  auto scale_block = [&]() {  // from the threads' largest magnitudes
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) s_max[tid >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, s_max[i]);
    const float s = scale_of(m);
    if (tid == 0) a.scale[(size_t)rb * a.lds + kb] = s;
    return m ? s : 1.f;  // zeros need no slow division
  };
  if constexpr (VEC) {
    Eight<T> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + i * 32;
      v[i].load(x + (size_t)(r < a.rows ? r : 0) * a.ldx, r < a.rows ? n : 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, v[i].amax());
    codes_of(v, scale_block(), w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + i * 32;
      if (r < a.rows && n > 0) store8(q + (size_t)r * a.ldq, w[2 * i], w[2 * i + 1], n);
    }
  } else {
    float f[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int r = r0 + i * 4;
      f[i] = r < a.rows && n > 0 ? to_f32(x[(size_t)r * a.ldx]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) m = max(m, abs_bits(f[i]));
    codes_of(f, scale_block(), w);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int r = r0 + i * 4;
      if (r < a.rows && n > 0) q[(size_t)r * a.ldq] = (uint8_t)(w[i / 4] >> 8 * (i % 4));
    }
  }
}

template <typename T>
static int quantize(QuantArgs a, int block_rows, int pdl, cudaStream_t s) {
  constexpr int E = 16 / (int)sizeof(T);
  const bool one = a.rows <= 1;
  const bool vec = ((uintptr_t)a.x & 15) == 0 && ((uintptr_t)a.q & 7) == 0 &&
                   a.cols % E == 0 && (one || (a.ldx % E == 0 && a.ldq % 8 == 0));
  const long long blocks =
      block_rows != 1 ? a.groups : vec ? (a.groups + 63) / 64 : (a.groups + 7) / 8;
  if (a.groups > 0x7fffffffLL - 64) return -2;  // 32-bit group numbers
  const bool one_row = block_rows == 1;
  const auto kernel = one_row ? (vec ? quantize_rows<T, true> : quantize_rows<T, false>)
                              : (vec ? quantize_blocks<T, true> : quantize_blocks<T, false>);
  const cudaError_t e = launch_dependent(kernel, dim3((unsigned)blocks), one_row ? 256 : 512, 0, s,
                                         pdl, 1, a);
  cwgk_count_launch();
  if (e != cudaSuccess) {
    cwgk_set_cuda_error((int)e);
    return -3;
  }
  return 0;
}

// ---- matrix product -----------------------------------------------------------------
// The weights are the MMA's M side: a CTA owns 128 outputs x TN rows of a, so that
// few rows (decoding) waste no MMA rows and the weight stream is read once.  Operand
// tiles of 128 k (128 bytes a row) come by TMA with the 128-byte swizzle; four MMAs of
// k = 32 make a block.  TMEM lane = output, column = row of a.  Promoting warps hold
// 32 outputs x TN (or TN / 2) sums each; the block's scales as * ws, one per column,
// are a broadcast read from shared memory that one warp keeps filled ahead.
// When the tiles leave SMs idle, the k blocks are cut among the CTAs of a cluster,
// which add their sums through distributed shared memory in rank order: the result
// does not depend on timing, and no workspace is needed.
constexpr int kTileK = 128;
constexpr int kGroupK = 8;  // blocks whose scales are staged together

template <int TN>
struct Cfg {
  static constexpr int kPromote = TN > 32 ? 8 : 4;       // promoting warps
  static constexpr int kCols = TN * 4 / kPromote;        // columns per promoting thread
  static constexpr int kThreads = (kPromote + 3) * 32;
  static constexpr int kMinBlocks = TN > 64 ? 1 : 2;
  static constexpr int kAcc = TN > 64 ? 2 : 4;           // accumulators in flight
  static constexpr int kTmem = kAcc * TN;
  static constexpr int kStageBytes = 128 * kTileK + TN * kTileK;
  static constexpr int kStages = TN > 64 ? 6 : 4;
  static constexpr int kScaleOff = kStages * kStageBytes;
  static constexpr int kScaleBytes = 2 * kGroupK * TN * 4;
  static constexpr int kBarOff = kScaleOff + kScaleBytes;
  // full[], empty[], acc_full[], acc_empty[], s_full[2], s_empty[2], drain
  static constexpr int kBars = 2 * kStages + 2 * kAcc + 5;
  static constexpr int kSmem = kBarOff + 8 * kBars + 16 + 1024;  // + slack to align to 1024
  static_assert(128 * TN * 4 <= kStages * kStageBytes, "partial sums reuse the stages");
};

struct MatArgs {
  const float *a_scale, *w_scale, *bias;
  void *y;
  size_t lda_scale, ldw_scale, ldy;
  int m, n, kblocks, per;  // per: k blocks of one cluster rank
  int splits, relu, bf16;
  int vec_y, vec_scale;    // rows of y and of a_scale are 16-byte aligned
  int pair_y;              // rows of y are 4-byte aligned
};

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, int x, int y,
                                       uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma_fp8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// K-major operand of 128-byte rows in the 128-byte swizzle: 8-row groups 1024 B apart.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f8f6f4: D fp32, A and B e4m3, both K-major.
__host__ __device__ constexpr uint32_t idesc_fp8(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// 16 columns of one lane, and 32; valid after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ void store_out(const MatArgs &a, int row, int col, float v,
                                          float bias) {
  v += bias;
  if (a.relu && v < 0.f) v = 0.f;  // NaN stays
  const size_t at = (size_t)row * a.ldy + col;
  if (a.bf16)
    static_cast<__nv_bfloat16 *>(a.y)[at] = pack1<__nv_bfloat16>(v);
  else
    static_cast<float *>(a.y)[at] = v;
}
// Adds the S ranks' sums of a tile's rows (columns of `part`) rank, rank + S, ... in rank
// order and stores them: a warp takes a row, a lane four outputs.  All S loads from the
// other CTAs' shared memory are issued before the first is used.
template <int S, int TN, int WARPS>
__device__ __forceinline__ void join_ranks(const MatArgs &p, uint32_t part, int rank, int warp,
                                           int lane, int m0, int n0, const float (&bias)[4]) {
  const int col = n0 + lane * 4;
  uint32_t from[S];
#pragma unroll
  for (int r = 0; r < S; ++r) from[r] = mapa_shared(part + lane * 16, (uint32_t)r);
  for (int j = rank + warp * S; j < TN && m0 + j < p.m; j += WARPS * S) {
    float4 f[S];
#pragma unroll
    for (int r = 0; r < S; ++r) f[r] = ld_cluster4(from[r] + j * 512);
    float v[4] = {f[0].x, f[0].y, f[0].z, f[0].w};
#pragma unroll
    for (int r = 1; r < S; ++r) v[0] += f[r].x, v[1] += f[r].y, v[2] += f[r].z, v[3] += f[r].w;
    if (p.vec_y && col + 4 <= p.n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] += bias[e];
        if (p.relu && v[e] < 0.f) v[e] = 0.f;  // NaN stays
      }
      const size_t at = (size_t)(m0 + j) * p.ldy + col;
      if (p.bf16)
        seq::store_raw<__nv_bfloat16, 4>(static_cast<__nv_bfloat16 *>(p.y) + at,
                                         seq::pack<__nv_bfloat16, 4>(v));
      else
        seq::store_raw<float, 4>(static_cast<float *>(p.y) + at, seq::pack<float, 4>(v));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < p.n) store_out(p, m0 + j, col + e, v[e], bias[e]);
    }
  }
}

template <int TN>
__global__ void __launch_bounds__(Cfg<TN>::kThreads, Cfg<TN>::kMinBlocks)
    fp8_matmul(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
               const MatArgs p) {
  using C = Cfg<TN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t *smem = smem_raw + (sbase - smem_u32(smem_raw));
  const uint32_t full = sbase + C::kBarOff, empty = full + 8 * C::kStages;
  const uint32_t acc_full = empty + 8 * C::kStages, acc_empty = acc_full + 8 * C::kAcc;
  const uint32_t s_full = acc_empty + 8 * C::kAcc, s_empty = s_full + 16, drain = s_empty + 16;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::kBarOff + 8 * C::kBars);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int rank = p.splits > 1 ? (int)cluster_rank() : 0;
  const int tile = blockIdx.x / p.splits;
  const int ntiles = (p.n + 127) / 128;
  const int n0 = (tile % ntiles) * 128, m0 = (tile / ntiles) * TN;
  const int kb0 = min(rank * p.per, p.kblocks), kb1 = min(kb0 + p.per, p.kblocks);
  const int nkb = kb1 - kb0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < C::kAcc; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, C::kPromote);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(s_empty + 8 * i, C::kPromote);
    }
    mbar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Nothing above touched global memory.  Tensor memory is taken only now: the previous
  // kernel's CTAs may still have to allocate theirs, and this one waits for them.
  griddep_wait();
  if (warp == C::kPromote) {  // the MMA warp owns the tensor memory
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(C::kTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();
  const uint32_t tmem = *tmem_slot;

  float acc[C::kCols];
#pragma unroll
  for (int j = 0; j < C::kCols; ++j) acc[j] = 0.f;

  if (warp == C::kPromote) {
    // ---- MMAs
    constexpr uint32_t idesc = idesc_fp8(128, TN);
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      const int st = i % C::kStages, ac = i % C::kAcc;
      ok = __all_sync(0xffffffffu,
                      mbar_wait(acc_empty + 8 * ac, ((i / C::kAcc) & 1) ^ 1, abort) &&
                          mbar_wait(full + 8 * st, (i / C::kStages) & 1, abort));
      if (!ok) break;
      tc_fence_after();
      const uint64_t w = desc_sw128(sbase + st * C::kStageBytes);
      const uint64_t a = desc_sw128(sbase + st * C::kStageBytes + 128 * kTileK);
#pragma unroll
      for (int k = 0; k < 4; ++k)  // 32 bytes along k = 2 descriptor units
        if (elect_one()) mma_fp8(tmem + ac * TN, w + 2 * k, a + 2 * k, idesc, k > 0);
      __syncwarp();
      if (elect_one()) tc_commit(empty + 8 * st);
      if (elect_one()) tc_commit(acc_full + 8 * ac);
      __syncwarp();
    }
    if (!ok) {  // let what was issued finish before the tensor memory is freed
      if (elect_one()) tc_commit(drain);
      __syncwarp();
      const unsigned long long t0 = globaltimer();
      while (!mbar_try(drain, 0) && globaltimer() - t0 < kTimeoutNs) {
      }
    }
  } else if (warp == C::kPromote + 1) {
    // ---- operand tiles
    int issued = 0;
    for (int i = 0; i < nkb; ++i) {
      const int st = i % C::kStages;
      if (!__all_sync(0xffffffffu,
                      mbar_wait(empty + 8 * st, ((i / C::kStages) & 1) ^ 1, abort)))
        break;
      if (elect_one()) {
        const uint32_t dst = sbase + st * C::kStageBytes;
        mbar_expect_tx(full + 8 * st, C::kStageBytes);
        tma_2d(dst, &map_w, (kb0 + i) * kTileK, n0, full + 8 * st);
        tma_2d(dst + 128 * kTileK, &map_a, (kb0 + i) * kTileK, m0, full + 8 * st);
      }
      __syncwarp();
      issued = i + 1;
    }
    // never leave the CTA with a copy still writing shared memory
    for (int i = issued - C::kStages > 0 ? issued - C::kStages : 0; i < issued; ++i) {
      const unsigned long long t0 = globaltimer();
      while (!mbar_try(full + 8 * (i % C::kStages), (i / C::kStages) & 1) &&
             globaltimer() - t0 < kTimeoutNs) {
      }
    }
  } else if (warp == C::kPromote + 2) {
    // ---- scales: as[row][kb] * ws[kb] of kGroupK blocks at a time, one group ahead in
    // registers
    float *s_scale = reinterpret_cast<float *>(smem + C::kScaleOff);
    constexpr int R = (TN + 31) / 32;
    const float *ws = p.w_scale + (size_t)(n0 / 128) * p.ldw_scale;
    float v[R][kGroupK];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int row = m0 + r * 32 + lane;
        const bool ok = r * 32 + lane < TN && row < p.m;
        const float *as = p.a_scale + (size_t)(ok ? row : 0) * p.lda_scale;
#pragma unroll
        for (int k = 0; k < kGroupK; ++k)
          v[r][k] = ok && i0 + k < nkb ? as[kb0 + i0 + k] * ws[kb0 + i0 + k] : 0.f;
      }
    };
    fetch(0);
    for (int i = 0, g = 0; i < nkb; i += kGroupK, ++g) {
      if (!__all_sync(0xffffffffu, mbar_wait(s_empty + 8 * (g & 1), ((g >> 1) & 1) ^ 1, abort)))
        break;
      float *dst = s_scale + (g & 1) * kGroupK * TN;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < kGroupK; ++k)
          if (r * 32 + lane < TN) dst[k * TN + r * 32 + lane] = v[r][k];
      __syncwarp();
      if (lane == 0) mbar_arrive(s_full + 8 * (g & 1));
      if (i + kGroupK < nkb) fetch(i + kGroupK);
    }
  } else {
    // ---- promotion
    const int quad = warp & 3, half = warp >> 2;
    const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16) + half * C::kCols;
    const float *s_scale = reinterpret_cast<const float *>(smem + C::kScaleOff) + half * C::kCols;
    for (int i = 0; i < nkb; ++i) {
      const int ac = i % C::kAcc, g = i / kGroupK, k = i % kGroupK;
      bool ok = true;
      if (k == 0) ok = mbar_wait(s_full + 8 * (g & 1), (g >> 1) & 1, abort);
      ok = ok && mbar_wait(acc_full + 8 * ac, (i / C::kAcc) & 1, abort);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const float *sc = s_scale + ((g & 1) * kGroupK + k) * TN;
      uint32_t v[C::kCols];
      if constexpr (C::kCols == 16) {
        tmem_ld16(trow + ac * TN, v);
      } else {
#pragma unroll
        for (int j = 0; j < C::kCols; j += 32) tmem_ld32(trow + ac * TN + j, v + j);
      }
      tmem_wait_ld();
      tc_fence_before();  // all read: the accumulator may be filled again
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty + 8 * ac);
#pragma unroll
      for (int j = 0; j < C::kCols; j += 4) {
        const float4 f = *reinterpret_cast<const float4 *>(sc + j);
        acc[j] = fmaf(__uint_as_float(v[j]), f.x, acc[j]);
        acc[j + 1] = fmaf(__uint_as_float(v[j + 1]), f.y, acc[j + 1]);
        acc[j + 2] = fmaf(__uint_as_float(v[j + 2]), f.z, acc[j + 2]);
        acc[j + 3] = fmaf(__uint_as_float(v[j + 3]), f.w, acc[j + 3]);
      }
      if (k == kGroupK - 1) {
        __syncwarp();
        if (lane == 0) mbar_arrive(s_empty + 8 * (g & 1));
      }
    }
    const int row = quad * 32 + lane, col = n0 + row;
    if (p.splits == 1) {
      if (col < p.n) {
        const float bias = p.bias ? p.bias[col] : 0.f;
#pragma unroll
        for (int j = 0; j < C::kCols; ++j)
          if (m0 + half * C::kCols + j < p.m)
            store_out(p, m0 + half * C::kCols + j, col, acc[j], bias);
      }
    }
  }
  if (p.splits > 1) {
    // all copies have landed and all MMAs have read them once every role is here
    __syncthreads();
    float *part = reinterpret_cast<float *>(smem);  // [column][output]
    if (warp < C::kPromote) {
      const int row = (warp & 3) * 32 + lane;
#pragma unroll
      for (int j = 0; j < C::kCols; ++j) part[((warp >> 2) * C::kCols + j) * 128 + row] = acc[j];
    }
    float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int col = n0 + lane * 4 + e;
      bias[e] = p.bias && col < p.n ? p.bias[col] : 0.f;
    }
    cluster_sync_all();
    constexpr int kWarps = C::kThreads / 32;
    if (p.splits == 2)
      join_ranks<2, TN, kWarps>(p, sbase, rank, warp, lane, m0, n0, bias);
    else if (p.splits == 4)
      join_ranks<4, TN, kWarps>(p, sbase, rank, warp, lane, m0, n0, bias);
    else
      join_ranks<8, TN, kWarps>(p, sbase, rank, warp, lane, m0, n0, bias);
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while another reads its sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kPromote) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(C::kTmem));
  }
}

// ---- many rows: two SMs on one tile ---------------------------------------------------
// A CTA pair computes 256 rows of a x 256 outputs with tcgen05.mma.cta_group::2: each CTA
// loads its 128 rows of a and 128 of the 256 rows of w per block of 128 k (32 KB for the
// 512 cycles of its MMAs; one CTA with a 128 x 256 tile would need 48 KB).  A block's
// products fill one of two accumulators of 128 rows x 256 columns; the eight promoting
// warps of each CTA, 32 rows x 128 columns each, read it back, multiply by the row's
// as[kb] and the 128 columns' ws[kb], and add it to 128 fp32 registers a thread while the
// other accumulator is being filled.
//
// What bounds it is the promoting warps' chain of latencies per block (barrier, tensor
// memory, hand-over), not their arithmetic, so that chain is what the code shortens: a
// chunk of 32 columns is always on its way from tensor memory while the one before it is
// added, the next block's first chunk too; that takes 64 more registers a thread, which
// the warps that only issue give up.
//
// Persistent: a pair walks over tiles, and the rings run on.  Rank 0 issues all MMAs; rank
// 1's MMA warp relays its landed stages to it.  One warp per CTA keeps the scales of its
// 128 rows, those of the tile's two blocks of w, and the biases in shared memory, a group
// of eight blocks ahead.
struct PairCfg {
  static constexpr int kN = 256;
  static constexpr int kPromote = 8;               // warps 4 .. 11
  static constexpr int kCols = 4 * kN / kPromote;  // columns per promoting thread
  static constexpr int kThreads = 4 * 32 + kPromote * 32;
  // registers: 168 a thread at launch, 384 threads; 72 x 128 + 216 x 256 are as many
  static constexpr int kRegsFew = 72, kRegsMany = 216;
  static constexpr int kAcc = 2;
  static constexpr int kTmem = 512;
  static constexpr int kStageBytes = (128 + kN / 2) * kTileK;
  static constexpr int kStages = 6;
  static constexpr int kPatchOff = kStages * kStageBytes;  // 32 rows x 64 bytes per warp
  // scales of kGroupK blocks, twice: [block][128 rows], then [block] of two w blocks
  static constexpr int kScaleOff = kPatchOff + kPromote * 32 * 64;
  static constexpr int kScaleBytes = kGroupK * (128 + 2) * 4;
  // biases of three tiles: the scale warp may be two tiles ahead of a promoting warp's stores
  static constexpr int kBiasOff = kScaleOff + 2 * kScaleBytes;
  static constexpr int kBarOff = kBiasOff + 3 * kN * 4;
  // full[], peer[], empty[], acc_full[], acc_empty[], s_full[2], s_empty[2], drain
  static constexpr int kBars = 3 * kStages + 2 * kAcc + 5;
  static constexpr int kSmem = kBarOff + 8 * kBars + 16 + 1024;
  static_assert(kAcc == 2, "the promoting warps take the accumulators in turn");
  static_assert(kRegsFew * 128 + kRegsMany * 256 <= 168 * kThreads, "registers at launch");
};

__device__ __forceinline__ void mma_fp8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                             uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// Tiles in the order a pair's neighbours take them: bands of 8 tile rows, column by
// column, so that pairs that run together share rows of a and of w in L2.
__device__ __forceinline__ void pair_tile(const MatArgs &p, int t, int &m0, int &n0) {
  const int mt = (p.m + 255) / 256, nt = (p.n + PairCfg::kN - 1) / PairCfg::kN;
  const int band = t / (8 * nt), rows = min(8, mt - band * 8), r = t - band * 8 * nt;
  m0 = (band * 8 + r % rows) * 256;
  n0 = r / rows * PairCfg::kN;
}

// W bytes, as one access.
template <int W>
struct Bytes {
  typedef uint4 type;
};
template <>
struct Bytes<4> {
  typedef uint32_t type;
};
template <>
struct Bytes<2> {
  typedef uint16_t type;
};

// A warp's 32 rows x COLS columns, 64 bytes of each row at a time through a patch of its
// own, whose 16-byte pieces are turned by the row so that neither side has bank conflicts:
// a store instruction then writes 64 bytes of 8 rows instead of 16 bytes of 32.  W: bytes
// that y's rows are aligned to; 64 bytes of one or two rows at a time where that is an
// element (3424 x 844 x 120 bf16: 49 us without the patch, 11).
template <typename T, int COLS, int W>
__device__ __forceinline__ void store_rows(uint8_t *patch, const seq::F2 (&acc)[COLS / 2],
                                           const MatArgs &p, int row, int col, int lane) {
  constexpr int E = 16 / (int)sizeof(T), kRound = 4 * E;  // columns per 64 bytes
  constexpr int kLanes = 64 / W, kRows = 32 / kLanes;     // of one store instruction
  constexpr int EW = W / (int)sizeof(T);
  typedef typename Bytes<W>::type Word;
  row -= lane;
#pragma unroll
  for (int c0 = 0; c0 < COLS; c0 += kRound) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float v[E];
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 f = seq::halves(acc[(c0 + k * E + e) / 2]);
        v[e] = f.x, v[e + 1] = f.y;
      }
      *reinterpret_cast<uint4 *>(patch + lane * 64 + ((k ^ (lane >> 1)) & 3) * 16) =
          seq::pack<T, E>(v);
    }
    __syncwarp();
    const int b = lane % kLanes * W, c = col + c0 + b / (int)sizeof(T);
#pragma unroll(W == 16 ? 4 : 2)
    for (int g = 0; g < 32 / kRows; ++g) {
      const int r = g * kRows + lane / kLanes;
      const uint8_t *from = patch + r * 64 + ((b / 16 ^ (r >> 1)) & 3) * 16 + b % 16;
      if (row + r >= p.m) continue;
      T *to = static_cast<T *>(p.y) + (size_t)(row + r) * p.ldy + c;
      if (c + EW <= p.n) {
        *reinterpret_cast<Word *>(to) = *reinterpret_cast<const Word *>(from);
      } else {
        for (int e = 0; e < EW; ++e)
          if (c + e < p.n) to[e] = reinterpret_cast<const T *>(from)[e];
      }
    }
    __syncwarp();
  }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg::kThreads, 1)
    fp8_matmul_pair(const __grid_constant__ CUtensorMap map_a,
                    const __grid_constant__ CUtensorMap map_w, const MatArgs p, int tiles) {
  using C = PairCfg;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t *smem = smem_raw + (sbase - smem_u32(smem_raw));
  const uint32_t full = sbase + C::kBarOff, peer = full + 8 * C::kStages;
  const uint32_t empty = peer + 8 * C::kStages, acc_full = empty + 8 * C::kStages;
  const uint32_t acc_empty = acc_full + 8 * C::kAcc, s_full = acc_empty + 8 * C::kAcc;
  const uint32_t s_empty = s_full + 16, drain = s_empty + 16;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::kBarOff + 8 * C::kBars);
  volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int mine = pair < tiles ? (tiles - 1 - pair) / pairs + 1 : 0;  // tiles of this pair

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(peer + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < C::kAcc; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, 2 * C::kPromote);  // both CTAs' warps, at rank 0
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(s_empty + 8 * i, C::kPromote);
    }
    mbar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  griddep_wait();  // before tensor memory is taken, as above
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(C::kTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any remote arrival
  tc_fence_after();
  griddep_launch_dependents();
  const uint32_t tmem = *tmem_slot;
  const int total = mine * p.kblocks;  // blocks this pair works through

  if (warp < 4) {
  regs_dec<C::kRegsFew>();
  if (warp == 0) {
    if (rank == 0) {
      // ---- MMAs of the pair
      constexpr uint32_t idesc = idesc_fp8(256, C::kN);
      bool ok = true;
      for (int i = 0; i < total; ++i) {
        const int st = i % C::kStages, ac = i % C::kAcc;
        const uint32_t ph = (i / C::kStages) & 1;
        // the lanes wait for the three barriers side by side: a look at one takes about 100
        // cycles
        const uint32_t bar = lane % 3 == 0   ? acc_empty + 8 * ac
                             : lane % 3 == 1 ? full + 8 * st
                                             : peer + 8 * st;
        const uint32_t par = lane % 3 == 0 ? ((i / C::kAcc) & 1) ^ 1 : ph;
        ok = __all_sync(0xffffffffu, mbar_wait(bar, par, abort));
        if (!ok) break;
        tc_fence_after();
        const uint64_t a = desc_sw128(sbase + st * C::kStageBytes);
        const uint64_t w = desc_sw128(sbase + st * C::kStageBytes + 128 * kTileK);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (elect_one()) mma_fp8_pair(tmem + ac * C::kN, a + 2 * k, w + 2 * k, idesc, k > 0);
        __syncwarp();
        if (elect_one()) tc_commit_pair(empty + 8 * st, 3);
        if (elect_one()) tc_commit_pair(acc_full + 8 * ac, 3);
        __syncwarp();
      }
      if (!ok) {  // what was issued finishes before anything is freed
        if (elect_one()) tc_commit_pair(drain, 1);
        __syncwarp();
        const unsigned long long t0 = globaltimer();
        while (!mbar_try(drain, 0) && globaltimer() - t0 < kTimeoutNs) {
        }
      }
    } else {
      const uint32_t peer0 = mapa_shared(peer, 0);
      for (int i = 0; i < total; ++i) {
        const int st = i % C::kStages;
        if (!__all_sync(0xffffffffu, mbar_wait(full + 8 * st, (i / C::kStages) & 1, abort)))
          break;
        if (elect_one()) mbar_arrive_cluster(peer0 + 8 * st);
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // ---- this CTA's rows of a and of w
    int i = 0;
    bool ok = true;
    for (int j = 0; ok && j < mine; ++j) {
      int m0, n0;
      pair_tile(p, pair + j * pairs, m0, n0);
      for (int kb = 0; kb < p.kblocks; ++kb, ++i) {
        const int st = i % C::kStages;
        ok = __all_sync(0xffffffffu,
                        mbar_wait(empty + 8 * st, ((i / C::kStages) & 1) ^ 1, abort));
        if (!ok) break;
        if (elect_one()) {
          const uint32_t dst = sbase + st * C::kStageBytes;
          mbar_expect_tx(full + 8 * st, C::kStageBytes);
          tma_2d(dst, &map_a, kb * kTileK, m0 + (int)rank * 128, full + 8 * st);
          tma_2d(dst + 128 * kTileK, &map_w, kb * kTileK, n0 + (int)rank * (C::kN / 2),
                 full + 8 * st);
        }
        __syncwarp();
      }
    }
    // never leave the CTA with a copy still writing shared memory
    for (int q = i - C::kStages > 0 ? i - C::kStages : 0; q < i; ++q) {
      const unsigned long long t0 = globaltimer();
      while (!mbar_try(full + 8 * (q % C::kStages), (q / C::kStages) & 1) &&
             globaltimer() - t0 < kTimeoutNs) {
      }
    }
  } else if (warp == 2) {
    // ---- scales, the next group's in registers while the ring is full
    float as[4][kGroupK], ws = 0.f, bias[C::kN / 32] = {};
    auto fetch = [&](int j, int kb) {
      int m0, n0;
      pair_tile(p, pair + j * pairs, m0, n0);
      m0 += (int)rank * 128;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = m0 + r * 32 + lane;
        const float *from = p.a_scale + (size_t)(row < p.m ? row : 0) * p.lda_scale + kb;
#pragma unroll
        for (int k = 0; k < kGroupK; k += 4) {
          if (p.vec_scale && kb + k + 4 <= p.kblocks) {
            const float4 v = *reinterpret_cast<const float4 *>(from + k);
            as[r][k] = v.x, as[r][k + 1] = v.y, as[r][k + 2] = v.z, as[r][k + 3] = v.w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) as[r][k + e] = kb + k + e < p.kblocks ? from[k + e] : 0.f;
          }
        }
      }
      // lanes 0 .. 7: the first block of w, 8 .. 15: the second
      const int nb = n0 / 128 + lane / kGroupK, b = kb + lane % kGroupK;
      ws = lane < 2 * kGroupK && nb < (p.n + 127) / 128 && b < p.kblocks
               ? p.w_scale[(size_t)nb * p.ldw_scale + b]
               : 0.f;
      if (kb == 0 && p.bias) {
#pragma unroll
        for (int e = 0; e < C::kN / 32; ++e)
          bias[e] = n0 + e * 32 + lane < p.n ? p.bias[n0 + e * 32 + lane] : 0.f;
      }
    };
    if (mine > 0) fetch(0, 0);
    bool ok = true;
    for (int j = 0, g = 0; ok && j < mine; ++j)
      for (int kb = 0; kb < p.kblocks; kb += kGroupK, ++g) {
        ok = __all_sync(0xffffffffu, mbar_wait(s_empty + 8 * (g & 1), ((g >> 1) & 1) ^ 1, abort));
        if (!ok) break;
        float *dst = reinterpret_cast<float *>(smem + C::kScaleOff + (g & 1) * C::kScaleBytes);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int k = 0; k < kGroupK; ++k) dst[k * 128 + r * 32 + lane] = as[r][k];
        if (lane < 2 * kGroupK) dst[kGroupK * 128 + lane] = ws;
        if (kb == 0) {
          float *to = reinterpret_cast<float *>(smem + C::kBiasOff) + j % 3 * C::kN;
#pragma unroll
          for (int e = 0; e < C::kN / 32; ++e) to[e * 32 + lane] = bias[e];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(s_full + 8 * (g & 1));
        if (kb + kGroupK < p.kblocks)
          fetch(j, kb + kGroupK);
        else if (j + 1 < mine)
          fetch(j + 1, 0);
      }
  }
  } else {
    // ---- promotion
    regs_inc<C::kRegsMany>();
    using seq::F2;
    const int quad = warp & 3, half = (warp - 4) >> 2;
    const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16) + half * C::kCols;
    const uint32_t free_at = mapa_shared(acc_empty, 0);  // rank 0 waits for both CTAs' warps
    uint8_t *patch = smem + C::kPatchOff + (warp - 4) * (32 * 64);
    constexpr int kChunks = C::kCols / 32;
    static_assert(kChunks % 2 == 0, "a block begins with the first buffer");
    uint32_t buf[2][32];
    bool ok = true;
    int ac = 0, par = 0, g = 0;  // accumulator, parity of its round, group of scales
    for (int j = 0; ok && j < mine; ++j) {
      int m0, n0;
      pair_tile(p, pair + j * pairs, m0, n0);
      F2 acc[C::kCols / 2];
#pragma unroll
      for (int q = 0; q < C::kCols / 2; ++q) acc[q] = seq::f2(0.f, 0.f);
      bool begun = false;  // the block's first chunk is on its way already
      for (int kb = 0; kb < p.kblocks; ++kb) {
        const int k = kb % kGroupK;
        // a wait may have given up for some lanes only, and all have to leave together: where a
        // chunk is on its way already, at the next block that is waited for, or behind the tile
        if (k == 0)
          ok = __all_sync(0xffffffffu,
                          ok && mbar_wait(s_full + 8 * (g & 1), (g >> 1) & 1, abort));
        const float *sc =
            reinterpret_cast<const float *>(smem + C::kScaleOff + (g & 1) * C::kScaleBytes);
        const float scale =
            sc[k * 128 + quad * 32 + lane] * sc[kGroupK * 128 + half * kGroupK + k];
        if (!begun) {
          ok = __all_sync(0xffffffffu, ok && mbar_wait(acc_full + 8 * ac, par, abort));
          if (!ok) break;
          tc_fence_after();
          tmem_ld32(trow + ac * C::kN, buf[0]);
        }
        const F2 s2 = seq::f2(scale, scale);
        const int next = ac ^ 1, next_par = par ^ ac;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          bool ready = false;  // a look at the next block, while this one's last chunk comes
          if (c + 1 == kChunks && kb + 1 < p.kblocks)
            ready = mbar_test(acc_full + 8 * next, next_par);
          tmem_wait_ld();
          if (c + 1 < kChunks) {
            tmem_ld32(trow + ac * C::kN + (c + 1) * 32, buf[(c + 1) & 1]);
          } else {
            tc_fence_before();  // all read: the accumulator may be filled again
            begun = __all_sync(0xffffffffu, ready);
            if (elect_one()) mbar_arrive_cluster(free_at + 8 * ac);
            if (begun) {
              tc_fence_after();
              tmem_ld32(trow + next * C::kN, buf[0]);
            }
          }
#pragma unroll
          for (int q = 0; q < 16; ++q)
            acc[c * 16 + q] = seq::fma2(seq::f2(__uint_as_float(buf[c & 1][2 * q]),
                                                __uint_as_float(buf[c & 1][2 * q + 1])),
                                        s2, acc[c * 16 + q]);
        }
        if (k == kGroupK - 1 || kb == p.kblocks - 1) {  // the group's last block
          __syncwarp();
          if (lane == 0) mbar_arrive(s_empty + 8 * (g & 1));
          ++g;
        }
        par = next_par;
        ac = next;
      }
      const int row = m0 + (int)rank * 128 + quad * 32 + lane, col = n0 + half * C::kCols;
      if (!ok || col >= p.n) continue;  // whole warps
      if (p.bias) {
        const float *bias = reinterpret_cast<const float *>(smem + C::kBiasOff) +
                            j % 3 * C::kN + half * C::kCols;
#pragma unroll
        for (int c = 0; c < C::kCols; c += 4) {
          const float4 f = *reinterpret_cast<const float4 *>(bias + c);
          acc[c / 2] = seq::add2(acc[c / 2], seq::f2(f.x, f.y));
          acc[c / 2 + 1] = seq::add2(acc[c / 2 + 1], seq::f2(f.z, f.w));
        }
      }
      if (p.relu) {
#pragma unroll
        for (int c = 0; c < C::kCols / 2; ++c) {
          const float2 f = seq::halves(acc[c]);
          acc[c] = seq::f2(f.x < 0.f ? 0.f : f.x, f.y < 0.f ? 0.f : f.y);  // NaN stays
        }
      }
      if (p.bf16 && p.vec_y)
        store_rows<__nv_bfloat16, C::kCols, 16>(patch, acc, p, row, col, lane);
      else if (p.bf16 && p.pair_y)
        store_rows<__nv_bfloat16, C::kCols, 4>(patch, acc, p, row, col, lane);
      else if (p.bf16)
        store_rows<__nv_bfloat16, C::kCols, 2>(patch, acc, p, row, col, lane);
      else if (p.vec_y)
        store_rows<float, C::kCols, 16>(patch, acc, p, row, col, lane);
      else
        store_rows<float, C::kCols, 4>(patch, acc, p, row, col, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // rank 0's MMAs read both CTAs' shared memory and tensor memory
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(C::kTmem));
  }
}

// Row-major e4m3 matrix [rows][k], rows ld bytes apart, as tiles of box_rows x 128.
// Reads outside [rows][k] give zeros.
static int make_map(CUtensorMap *map, const void *base, long long ld, int rows, int k,
                    int box_rows) {
  typedef CUresult (*encode_fn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<encode_fn> found_fn{nullptr};  // the same pointer for every thread
  encode_fn encode = found_fn.load(std::memory_order_acquire);
  if (!encode) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000,
                                                           cudaEnableDefault, &found);
    if (e != cudaSuccess || found != cudaDriverEntryPointSuccess || !fn) {
      cwgk_set_cuda_error((int)(e != cudaSuccess ? e : cudaErrorNotSupported));
      return -3;
    }
    encode = (encode_fn)fn;
    found_fn.store(encode, std::memory_order_release);
  }
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? ld : ((long long)k + 15) / 16 * 16)};
  const cuuint32_t box[2] = {kTileK, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  const CUresult r =
      encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box,
             ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    cwgk_set_cuda_error((int)cudaErrorInvalidValue);
    return -3;
  }
  return 0;
}

static MatArgs make_args(const cwgk_fp8 *op) {
  MatArgs p;
  p.a_scale = op->a_scale;
  p.w_scale = op->w_scale;
  p.bias = op->bias;
  p.y = op->y;
  p.lda_scale = (size_t)op->lda_scale;
  p.ldw_scale = (size_t)op->ldw_scale;
  p.ldy = (size_t)op->ldy;
  p.m = op->m;
  p.n = op->n;
  p.kblocks = (op->k + kTileK - 1) / kTileK;
  p.per = p.kblocks;
  p.splits = 1;
  p.relu = op->relu;
  p.bf16 = op->bf16;
  const long long esz = op->bf16 ? 2 : 4;
  p.vec_scale = ((uintptr_t)op->a_scale & 15) == 0 && (op->m <= 1 || op->lda_scale % 4 == 0);
  p.vec_y = ((uintptr_t)op->y & 15) == 0 && (op->m <= 1 || op->ldy * esz % 16 == 0);
  p.pair_y = ((uintptr_t)op->y & 3) == 0 && (op->m <= 1 || op->ldy * esz % 4 == 0);
  return p;
}

// Co-resident pairs of the current device (one CTA per SM; a cluster needs two SMs that
// can form one), asked once per device.
static int resident_pairs() {
  static std::atomic<int> cache[64];
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = cache[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(sms / 2 * 2));
  cfg.blockDim = dim3(PairCfg::kThreads);
  cfg.dynamicSmemBytes = PairCfg::kSmem;
  if (cudaOccupancyMaxActiveClusters(&n, (const void *)fp8_matmul_pair, &cfg) != cudaSuccess ||
      n <= 0) {
    (void)cudaGetLastError();
    n = sms / 2;
  }
  cache[dev].store(n, std::memory_order_relaxed);
  return n;
}

static long long pair_tiles(const cwgk_fp8 *op) {
  return (long long)((op->m + 255) / 256) * ((op->n + PairCfg::kN - 1) / PairCfg::kN);
}

static int launch_pair(const cwgk_fp8 *op, cudaStream_t s) {
  CUtensorMap map_a, map_w;
  int rc = make_map(&map_a, op->a, op->lda, op->m, op->k, 128);
  if (!rc) rc = make_map(&map_w, op->w, op->ldw, op->n, op->k, PairCfg::kN / 2);
  if (rc) return rc;
  const MatArgs p = make_args(op);
  const long long tiles = pair_tiles(op);
  if (tiles * p.kblocks > 0x7fffffffLL) return -2;
  cudaError_t e = smem_attr_once<fp8_matmul_pair>(PairCfg::kSmem);
  if (e == cudaSuccess) {
    const int most = resident_pairs(), pairs = (int)(tiles < most ? tiles : most);
    if (pairs <= 0) return -3;
    e = launch_dependent(fp8_matmul_pair, dim3((unsigned)(2 * pairs)), PairCfg::kThreads,
                         PairCfg::kSmem, s, op->pdl, 1, map_a, map_w, p, (int)tiles);
    cwgk_count_launch();
  }
  if (e != cudaSuccess) {
    cwgk_set_cuda_error((int)e);
    return -3;
  }
  return 0;
}

static long long out_tiles(const cwgk_fp8 *op, int tn) {
  return (long long)((op->n + 127) / 128) * ((op->m + tn - 1) / tn);
}

template <int TN>
static int launch(const cwgk_fp8 *op, cudaStream_t s) {
  using C = Cfg<TN>;
  CUtensorMap map_a, map_w;
  int rc = make_map(&map_a, op->a, op->lda, op->m, op->k, TN);
  if (!rc) rc = make_map(&map_w, op->w, op->ldw, op->n, op->k, 128);
  if (rc) return rc;
  MatArgs p = make_args(op);
  const long long tiles = out_tiles(op, TN);
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= 148 * C::kMinBlocks &&
         p.kblocks >= splits * 4)
    splits *= 2;
  p.splits = splits;
  p.per = (p.kblocks + splits - 1) / splits;
  if (tiles * splits > 0x7fffffffLL) return -2;
  cudaError_t e = smem_attr_once<fp8_matmul<TN>>(C::kSmem);
  if (e == cudaSuccess) {
    e = launch_dependent(fp8_matmul<TN>, dim3((unsigned)(tiles * splits)), C::kThreads, C::kSmem,
                         s, op->pdl, (unsigned)splits, map_a, map_w, p);
    cwgk_count_launch();
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    cwgk_set_cuda_error((int)e);
    return -3;
  }
  return 0;
}

}  // namespace fp8
}  // namespace cwg

extern "C" {

int cwgk_fp8_quantize(const void *x, long long ldx, void *q, long long ldq, float *scale,
                      long long lds, int rows, int cols, int block_rows, int bf16, int pdl,
                      void *stream) {
  cwg::fp8::QuantArgs a;
  a.x = x;
  a.q = static_cast<uint8_t *>(q);
  a.scale = scale;
  a.ldx = (size_t)ldx;
  a.ldq = (size_t)ldq;
  a.lds = (size_t)lds;
  a.rows = rows;
  a.cols = cols;
  a.kblocks = (cols + 127) / 128;
  a.groups = (long long)((rows + block_rows - 1) / block_rows) * a.kblocks;
  return bf16 ? cwg::fp8::quantize<__nv_bfloat16>(a, block_rows, pdl, (cudaStream_t)stream)
              : cwg::fp8::quantize<float>(a, block_rows, pdl, (cudaStream_t)stream);
}

int cwgk_fp8_matmul(const cwgk_fp8 *op, void *stream) {
  cudaStream_t s = (cudaStream_t)stream;
  // Rows per tile.  Small tiles make more CTAs of work that is bound by latencies, as long
  // as those run at once, two per SM (72 rows x 2048 x 8192: 10.0 us with tiles of 32 rows,
  // 11.1 with 64, 18.9 with 128; x 11008 x 4096, 258 tiles of 32: 16.1, 21.8, 20.6; 128 rows,
  // 344 tiles: 26.3, 23.8, 22.1).  With more rows the weights, which every tile of rows reads
  // again, count too: 512 x 1024 x 4096, 128 tiles of 32: 10.1, 10.9, 11.3; 768 rows, 192 tiles:
  // 15.4, 14.6, 14.1; 1024 x 2048 x 512, 256 tiles of 64: 11.0, 7.6, 9.2; 768 x 4096 x 512, 384
  // tiles of 64: 16.1, 12.2, 17.7, 8.6 with pairs.  Along a long k the larger tiles win (512 x
  // 4096 x 4096: 24.0 with 64, 21.5 with 128, 22.8 with pairs; 512 x 2048 x 8192: 24.0, 20.0,
  // 38.8; 512 x 600 x 3600: 10.8, 11.7, 20.5), and pairs once they fill half of the GPU (192 x
  // 11008 x 4096, 43 tiles: 37.9 with 128, 24.4).
  using namespace cwg::fp8;
  if (op->m <= 16) return launch<16>(op, s);
  if (op->m <= 32 || out_tiles(op, 32) <= (op->m <= 128 ? 2 * 148 : 148)) return launch<32>(op, s);
  const bool long_k = op->k > 31 * kTileK;
  if (op->m <= 64 || (op->m > 128 && !long_k && out_tiles(op, 64) <= 2 * 148))
    return launch<64>(op, s);
  if (op->m > 128 && (!long_k || pair_tiles(op) >= 37)) return launch_pair(op, s);
  return launch<128>(op, s);
}

int cwgk_fp8_read_clear_status(unsigned *status) {
  return cwg::read_clear_status(cwg::fp8::g_fp8_status, status);
}

}  // extern "C"
