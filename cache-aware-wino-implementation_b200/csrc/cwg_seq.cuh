// cwg_seq.cuh -- device helpers shared by the sequence layers: rows of mixed
// types as fp32 vectors, packed sequences and their cache lines.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cwg_common.cuh"
#include "cwg_tcgen05.cuh"

namespace cwg {
namespace seq {

using tc::griddep_launch_dependents;
using tc::griddep_wait;

// V elements of T, moved as one 16-byte vector (or 8 bytes, or one element, V = 1).
template <typename T, int V>
struct Raw {
  static_assert(V * sizeof(T) == 16, "one element, 8 bytes or 16 bytes");
  using type = uint4;
};
template <>
struct Raw<__nv_bfloat16, 4> {
  using type = uint2;
};
template <>
struct Raw<float, 1> {
  using type = float;
};
template <>
struct Raw<__nv_bfloat16, 1> {
  using type = __nv_bfloat16;
};

template <typename T, int V>
__device__ __forceinline__ typename Raw<T, V>::type load_raw(const T *p) {
  return *reinterpret_cast<const typename Raw<T, V>::type *>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_raw(T *p, typename Raw<T, V>::type v) {
  *reinterpret_cast<typename Raw<T, V>::type *>(p) = v;
}
template <typename T, int V>
__device__ __forceinline__ typename Raw<T, V>::type zero_raw() {
  if constexpr (V == 1)
    return from_f32<T>(0.f);
  else if constexpr (V * sizeof(T) == 8)
    return make_uint2(0, 0);
  else
    return make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ void unpack(float v, float (&f)[1]) { f[0] = v; }
__device__ __forceinline__ void unpack(__nv_bfloat16 v, float (&f)[1]) { f[0] = to_f32(v); }
__device__ __forceinline__ void unpack(uint4 v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x);
  f[1] = __uint_as_float(v.y);
  f[2] = __uint_as_float(v.z);
  f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(uint2 v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x << 16);
  f[1] = __uint_as_float(v.x & 0xFFFF0000u);
  f[2] = __uint_as_float(v.y << 16);
  f[3] = __uint_as_float(v.y & 0xFFFF0000u);
}
__device__ __forceinline__ void unpack(uint4 v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
// One rounding, to nearest even (none for fp32).
template <typename T>
__device__ __forceinline__ T pack1(float v) {
  return from_f32<T>(v);
}
template <typename T, int V>
__device__ __forceinline__ typename Raw<T, V>::type pack(const float (&f)[V]) {
  if constexpr (V == 1) {
    return from_f32<T>(f[0]);
  } else if constexpr (V * sizeof(T) == 8) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]);
    const __nv_bfloat162 b = __floats2bfloat162_rn(f[2], f[3]);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&a),
                      *reinterpret_cast<const uint32_t *>(&b));
  } else if constexpr (V == 4) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Two fp32 values in one 64-bit register: one instruction works on both, each half
// rounded as the scalar instruction rounds.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(F2 p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// v / (1 + exp(-v)).  fp32 results take expf and a rounded division; below -88.7 expf is
// infinite and the result zero (3e-37 at most is lost).  For bf16 results, whose half step is
// 2^-8 of the value, ex2 and a reciprocal (2 ulp each) with the exponent's two roundings, which
// add 2 |v| u, stay within (8 + 2 |v|) u, u = 2^-24: 2^-16 at v = -87; 5 instructions instead of
// about 30.  Results below 1.1e-36 in magnitude (v under -87.3) come out as zero.  Both give NaN
// for v = -infinity, as the formula does.
template <typename T>
__device__ __forceinline__ float silu(float v) {
  if constexpr (sizeof(T) == 4)
    return v / (1.f + expf(-v));
  else
    return v * rcp(1.f + ex2(-kLog2e * v));
}

__device__ __forceinline__ F2 silu_bf16x2(F2 v) {
  const float2 t = halves(mul2(v, f2(-kLog2e, -kLog2e)));
  const float2 e = halves(add2(f2(ex2(t.x), ex2(t.y)), f2(1.f, 1.f)));
  return mul2(v, f2(rcp(e.x), rcp(e.y)));
}

// log(1 + exp(v)) = max(v, 0) + log1p(e) with e = exp(-|v|) <= 1, and the series
//   log1p(e) = 2 (s + s^3/3 + s^5/5 + ...),  s = e / (2 + e) <= 1/3,
// which has no cancellation for small e (a step's relative error goes into the decay of
// every state).  Cut after s^17: the rest is below (1/9)^9 / 19 = 1.4e-10 of the first
// term.  Relative error: ex2 4 u, its argument 2 |v| u, the reciprocal 2 u, about 6 u for
// the sums (u = 2^-24).
__device__ __forceinline__ float softplus(float v) {
  const float e = ex2(-kLog2e * fabsf(v));
  const float s = e * rcp(2.f + e);
  const float q = s * s;
  float p = 1.f / 17;
  p = fmaf(p, q, 1.f / 15);
  p = fmaf(p, q, 1.f / 13);
  p = fmaf(p, q, 1.f / 11);
  p = fmaf(p, q, 1.f / 9);
  p = fmaf(p, q, 1.f / 7);
  p = fmaf(p, q, 1.f / 5);
  p = fmaf(p, q, 1.f / 3);
  p = fmaf(p, q, 1.f);
  const float r = fmaf(2.f * s, p, fmaxf(v, 0.f));
  return v != v ? v : r;  // fmaxf would drop a NaN
}

// First b in [0, n) with s[b] >= v (n if none); ends for any contents of s.
__device__ __forceinline__ int lower_bound(const int *s, int n, int v) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// Whether slots[b] occurs among slots[0 .. b-1]: the calling warp's lanes search
// together, and all of them get the answer.
__device__ __forceinline__ bool taken_before(const int *slots, int b, int slot) {
  bool hit = false;
  for (int i0 = (int)(threadIdx.x & 31); i0 < b; i0 += 128) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // four loads in flight
      const int i = i0 + 32 * k;
      hit |= i < b && slots[i] == slot;
    }
  }
  return __any_sync(0xffffffffu, hit) != 0;
}

// Cache line of sequence b, or -1: no line (a negative slot), or an index that
// cannot be served (outside the lines, or an earlier sequence's), which `bad`
// reports.  Called by whole warps with a warp-uniform b.  The first 128 lines of earlier
// sequences are read along with b's own.
__device__ __forceinline__ int line_of(const int *slots, int b, int n_slots, bool &bad) {
  if (!slots) {
    if (b < n_slots) return b;
    bad = true;
    return -1;
  }
  const int lane = (int)(threadIdx.x & 31);
  int other[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) other[k] = lane + 32 * k < b ? slots[lane + 32 * k] : -1;
  const int slot = slots[b];
  if (slot < 0) return -1;
  const bool hit = other[0] == slot || other[1] == slot || other[2] == slot || other[3] == slot;
  if (slot >= n_slots || __any_sync(0xffffffffu, hit) ||
      (b > 128 && taken_before(slots + 128, b - 128, slot))) {
    bad = true;
    return -1;
  }
  return slot;
}

}  // namespace seq
}  // namespace cwg
