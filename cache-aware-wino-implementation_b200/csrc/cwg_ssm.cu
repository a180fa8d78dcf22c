// cwg_ssm.cu -- selective state space scan (cwg_ssm_scan, cwg_ssm_step).
//
// For every channel c with states i = 0 .. N-1, step d = softplus(dt + dt_bias):
//   h_i <- exp(d A_i) h_i + d u B_i,   y = (sum_i C_i h_i + D u) z / (1 + exp(-z))
//
// A channel's N states are spread over L lanes, four per lane (N padded to 4 L
// with A = B = C = 0, whose states stay zero), so a warp holds 32 / L channels.
// exp(d A) is computed as 2^(d (A log2 e)) with ex2.approx (2 ulp); state, decay
// and sums are fp32.
#include <cstdint>

#include "../../include/cwg.h"
#include "cwg_seq.cuh"

namespace cwg {
namespace ssm {

using namespace seq;

__device__ unsigned int g_ssm_status;

constexpr int kS = 4;    // states per lane
constexpr int kTT = 32;  // tokens per tile of the prompt kernel

struct Args {
  cwg_ssm p;
  int per;      // channels per group
  int cblocks;  // CTAs along one group's channels
  bool vec_state, vec_a;  // the state's and A's rows are whole 16-byte vectors
  bool vec_bc;            // B and C can be read four states at a time
};

// A lane's four states of one cache line, or zeros.
__device__ __forceinline__ void load_states(const float *line, int i0, int n, bool vec,
                                            float (&h)[kS]) {
  if (vec) {
    const float4 f = *reinterpret_cast<const float4 *>(line + i0);
    h[0] = f.x, h[1] = f.y, h[2] = f.z, h[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < kS; ++i) h[i] = i0 + i < n ? line[i0 + i] : 0.f;
  }
}
__device__ __forceinline__ void store_states(float *line, int i0, int n, bool vec,
                                             const float (&h)[kS]) {
  if (vec) {
    *reinterpret_cast<float4 *>(line + i0) = make_float4(h[0], h[1], h[2], h[3]);
  } else {
#pragma unroll
    for (int i = 0; i < kS; ++i)
      if (i0 + i < n) line[i0 + i] = h[i];
  }
}

// ---- prompts --------------------------------------------------------------------
// One CTA per (sequence, block of CH channels of one group): it walks the sequence
// in tiles of kTT tokens.  Per tile the CTA turns dt and u into (d, d u) pairs and
// B, C into fp32 in shared memory, the lanes run the recurrence over the tile, and
// the CTA finishes y with full-width row accesses.  The next tile's operands are
// loaded into registers while the recurrence runs.
template <int L>
struct Geo {
  static constexpr int kCH = L <= 4 ? 64 : 256 / L;
  static constexpr int kThreads = kCH * L;
  static constexpr int kNP = kS * L;
  static constexpr int kTasks = kTT * kCH / 8;  // 8-channel pieces of a tile
  static constexpr int kPer = (kTasks + kThreads - 1) / kThreads;
  static constexpr int kPerB = kTT * kNP / kThreads;
};

// 8 consecutive channels of one row as fp32; channels past `n` read as zero.
template <typename T, bool VEC>
struct Piece {
  static constexpr int kRaw = VEC ? (int)sizeof(T) * 8 / 16 : 8;
  using R = typename Raw<T, VEC ? 16 / (int)sizeof(T) : 1>::type;
  R raw[kRaw];
  __device__ __forceinline__ void load(const T *p, int n) {
#pragma unroll
    for (int i = 0; i < kRaw; ++i) {
      constexpr int E = 8 / kRaw;
      raw[i] = i * E < n ? load_raw<T, E>(p + i * E) : zero_raw<T, E>();
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    constexpr int E = 8 / kRaw;
#pragma unroll
    for (int i = 0; i < kRaw; ++i) {
      float g[E];
      unpack(raw[i], g);
#pragma unroll
      for (int e = 0; e < E; ++e) f[i * E + e] = g[e];
    }
  }
  __device__ static __forceinline__ void store(T *p, const float (&f)[8], int n) {
    constexpr int E = 8 / kRaw;
#pragma unroll
    for (int i = 0; i < kRaw; ++i) {
      float g[E];
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] = f[i * E + e];
      if (i * E < n) store_raw<T, E>(p + i * E, pack<T, E>(g));
    }
  }
};

template <typename T, int L, bool VEC>
__global__ void __launch_bounds__(Geo<L>::kThreads) ssm_prompt(const Args a) {
  using G = Geo<L>;
  constexpr int CH = G::kCH, NT = G::kThreads, NP = G::kNP, PER = G::kPer, PERB = G::kPerB;
  __shared__ __align__(16) float2 s_dx[kTT][CH];
  __shared__ __align__(16) float s_b[kTT][NP], s_c[kTT][NP];
  __shared__ __align__(16) float s_y[kTT][CH];
  const cwg_ssm &p = a.p;
  const int tid = threadIdx.x;
  const int cblk = blockIdx.x % a.cblocks;
  const int group = (blockIdx.x / a.cblocks) % p.groups;
  const int b = blockIdx.x / (a.cblocks * p.groups);
  const int in0 = cblk * CH;                // first channel within the group
  const int c0 = group * a.per + in0;       // first channel
  const int nch = min(CH, a.per - in0);
  const int begin = p.starts[b], end = p.starts[b + 1];
  const bool report = tid == 0 && cblk == 0 && group == 0;
  if (begin < 0 || end < begin || end > p.tokens) {
    if (report) atomicOr(&g_ssm_status, CWGK_STATUS_INDEX);
    return;
  }
  bool bad = false;
  const int slot = p.state ? line_of(p.slots, b, p.n_slots, bad) : -1;
  if (bad && report) atomicOr(&g_ssm_status, CWGK_STATUS_INDEX);
  const bool carry = slot >= 0 && p.resume && p.resume[b];

  // the recurrence's view: lane `l` of channel `ch`, states i0 .. i0 + 3
  const int ch = tid / L, l = tid % L, i0 = l * kS;
  const bool mine = ch < nch;
  float A2[kS], h[kS];
  float *line = p.state + ((size_t)(slot < 0 ? 0 : slot) * p.channels + c0 + ch) * p.states;
#pragma unroll
  for (int i = 0; i < kS; ++i) {
    A2[i] = mine && i0 + i < p.states ? p.A[(size_t)(c0 + ch) * p.states + i0 + i] * kLog2e : 0.f;
    h[i] = 0.f;
  }
  if (carry && mine) load_states(line, i0, p.states, a.vec_state, h);

  // the tile's view: 8-channel pieces
  Piece<T, VEC> ru[PER], rd[PER], rz[PER], cu[PER], cz[PER];
  float rb[PERB], rc[PERB];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int task = tid + i * NT;
      const int t = t0 + task / (CH / 8), c = (task % (CH / 8)) * 8;
      const int n = task < G::kTasks && t < end ? nch - c : 0;
      const size_t at = (size_t)t;
      ru[i].load(static_cast<const T *>(p.u) + at * p.ldu + c0 + c, n);
      rd[i].load(static_cast<const T *>(p.dt) + at * p.lddt + c0 + c, n);
      rz[i].load(static_cast<const T *>(p.z) + at * p.ldz + c0 + c, p.z ? n : 0);
    }
#pragma unroll
    for (int i = 0; i < PERB; ++i) {
      const int e = tid + i * NT;
      const int t = t0 + e / NP, s = e % NP;
      const bool ok = t < end && s < p.states;
      const size_t col = (size_t)group * p.states + s;
      rb[i] = ok ? to_f32(static_cast<const T *>(p.B)[(size_t)t * p.ldb + col]) : 0.f;
      rc[i] = ok ? to_f32(static_cast<const T *>(p.C)[(size_t)t * p.ldc + col]) : 0.f;
    }
  };

  fetch(begin);
  for (int t0 = begin; t0 < end; t0 += kTT) {
    // (d, d u) of every (token, channel); rows past the end have d = 0, which
    // leaves the states as they are
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int task = tid + i * NT;
      const int t = task / (CH / 8), c = (task % (CH / 8)) * 8;
      if (task < G::kTasks) {
        float u[8], d[8];
        ru[i].get(u);
        rd[i].get(d);
        const bool row = t0 + t < end;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool ok = row && c + e < nch;
          float v = d[e] + (ok && p.dt_bias ? p.dt_bias[c0 + c + e] : 0.f);
          if (p.flags & CWG_SOFTPLUS) v = softplus(v);
          s_dx[t][c + e] = ok ? make_float2(v, v * u[e]) : make_float2(0.f, 0.f);
        }
      }
      cu[i] = ru[i];
      cz[i] = rz[i];
    }
#pragma unroll
    for (int i = 0; i < PERB; ++i) {
      const int e = tid + i * NT;
      s_b[e / NP][e % NP] = rb[i];
      s_c[e / NP][e % NP] = rc[i];
    }
    __syncthreads();
    if (t0 + kTT < end) fetch(t0 + kTT);
#pragma unroll 4
    for (int t = 0; t < kTT; ++t) {
      const float2 dx = s_dx[t][ch];
      const float4 bv = *reinterpret_cast<const float4 *>(&s_b[t][i0]);
      const float4 cv = *reinterpret_cast<const float4 *>(&s_c[t][i0]);
      h[0] = fmaf(ex2(dx.x * A2[0]), h[0], dx.y * bv.x);
      h[1] = fmaf(ex2(dx.x * A2[1]), h[1], dx.y * bv.y);
      h[2] = fmaf(ex2(dx.x * A2[2]), h[2], dx.y * bv.z);
      h[3] = fmaf(ex2(dx.x * A2[3]), h[3], dx.y * bv.w);
      float y = fmaf(h[0], cv.x, h[1] * cv.y) + fmaf(h[2], cv.z, h[3] * cv.w);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
      if (l == 0) s_y[t][ch] = y;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int task = tid + i * NT;
      const int t = task / (CH / 8), c = (task % (CH / 8)) * 8;
      if (task < G::kTasks && t0 + t < end && c < nch) {
        float u[8], z[8], y[8];
        cu[i].get(u);
        cz[i].get(z);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = fmaf(p.D && c + e < nch ? p.D[c0 + c + e] : 0.f, u[e], s_y[t][c + e]);
          if (p.z) y[e] *= silu<T>(z[e]);
        }
        Piece<T, VEC>::store(static_cast<T *>(p.y) + (size_t)(t0 + t) * p.ldy + c0 + c, y,
                             nch - c);
      }
    }
  }
  if (slot >= 0 && mine) store_states(line, i0, p.states, a.vec_state, h);
}

// ---- one token of each sequence ----------------------------------------------------
// Bound by the states, 8 N bytes per channel in and out.  A CTA takes RR rows of one
// channel block: the rows share A, and all their states are loaded before the first is
// used.  Meanwhile the CTA's threads look together for lines that an earlier row has too.
template <typename T>
__device__ __forceinline__ void load4(const T *p, int i0, int n, bool vec, float (&f)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      unpack(*reinterpret_cast<const uint4 *>(p + i0), f);
    } else {
      const uint2 v = *reinterpret_cast<const uint2 *>(p + i0);
      f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xFFFF0000u);
      f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = i0 + i < n ? to_f32(p[i0 + i]) : 0.f;
  }
}

template <typename T, int L, int RR>
__global__ void __launch_bounds__(Geo<L>::kThreads) ssm_token(const Args a) {
  constexpr int CH = Geo<L>::kCH, NT = Geo<L>::kThreads;
  const cwg_ssm &p = a.p;
  const int tid = threadIdx.x;
  const int cblk = blockIdx.x % a.cblocks;
  const int group = (blockIdx.x / a.cblocks) % p.groups;
  const int r0 = blockIdx.x / (a.cblocks * p.groups) * RR;
  const int ch = tid / L, l = tid % L, i0 = l * kS;
  const int in = cblk * CH + ch, c = group * a.per + in;
  const bool mine = in < a.per;
  const size_t width = (size_t)p.channels * p.states, at = (size_t)c * p.states;
  // Rows r0 + l, r0 + l + L, ... of the channel are lane l's: it computes their steps and
  // finishes their outputs (with more lanes than rows, lane l takes row l % RR too, which
  // only lane l = row stores).
  constexpr int E = L < RR ? RR / L : 1;
  float h[RR][kS], u[E], d[E], z[E];
  int slot[RR];
  bool bad = false;
#pragma unroll
  for (int k = 0; k < RR; ++k) {
    const int r = r0 + k;
    slot[k] = r >= p.tokens ? -1 : p.slots ? p.slots[r] : r;
    if (slot[k] >= p.n_slots) slot[k] = -1, bad = true;
  }
#pragma unroll
  for (int k = 0; k < RR; ++k) {
#pragma unroll
    for (int i = 0; i < kS; ++i) h[k][i] = 0.f;
    if (mine && slot[k] >= 0)
      load_states(p.state + (size_t)slot[k] * width + at, i0, p.states, a.vec_state, h[k]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int r = r0 + (L < RR ? e * L + l : l % RR);
    const size_t rr = (size_t)(r < p.tokens ? r : 0);
    u[e] = d[e] = z[e] = 0.f;
    if (mine) {
      u[e] = to_f32(static_cast<const T *>(p.u)[rr * p.ldu + c]);
      d[e] = to_f32(static_cast<const T *>(p.dt)[rr * p.lddt + c]);
      if (p.z) z[e] = to_f32(static_cast<const T *>(p.z)[rr * p.ldz + c]);
    }
  }
  float A2[kS] = {0.f, 0.f, 0.f, 0.f};
  if (mine) load_states(p.A + at, i0, p.states, a.vec_a, A2);
#pragma unroll
  for (int i = 0; i < kS; ++i) A2[i] *= kLog2e;
  const float bias = mine && p.dt_bias ? p.dt_bias[c] : 0.f;
  const float skip = mine && p.D ? p.D[c] : 0.f;
  if (p.slots) {
    int taken = 0;
    for (int i = tid; i < r0 + RR - 1 && i < p.tokens; i += NT) {
      const int other = p.slots[i];
#pragma unroll
      for (int k = 0; k < RR; ++k) taken |= (i < r0 + k && other == slot[k]) << k;
    }
    if (__syncthreads_or(taken)) {
#pragma unroll
      for (int k = 0; k < RR; ++k)
        if (__syncthreads_or(taken & (1 << k)) && slot[k] >= 0) {
          slot[k] = -1;
          bad = true;
#pragma unroll
          for (int i = 0; i < kS; ++i) h[k][i] = 0.f;
        }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    d[e] += bias;
    if (p.flags & CWG_SOFTPLUS) d[e] = softplus(d[e]);
    z[e] = p.z ? silu<T>(z[e]) : 1.f;
  }
  const T *Brow = static_cast<const T *>(p.B) + (size_t)r0 * p.ldb + (size_t)group * p.states;
  const T *Crow = static_cast<const T *>(p.C) + (size_t)r0 * p.ldc + (size_t)group * p.states;
  float out[E] = {};
#pragma unroll
  for (int k = 0; k < RR; ++k) {
    if (RR > 1 && r0 + k >= p.tokens) break;
    // lane and piece that hold row k's step
    constexpr unsigned kAll = 0xffffffffu;
    const int from = L < RR ? k % L : k, e = L < RR ? k / L : 0;
    const float step = L > 1 && RR > 1 ? __shfl_sync(kAll, d[e], from, L) : d[e];
    const float uk = L > 1 && RR > 1 ? __shfl_sync(kAll, u[e], from, L) : u[e];
    float bv[4], cv[4];
    load4(Brow + (size_t)k * p.ldb, i0, p.states, a.vec_bc, bv);
    load4(Crow + (size_t)k * p.ldc, i0, p.states, a.vec_bc, cv);
    const float du = step * uk;
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < kS; ++i) {
      h[k][i] = fmaf(ex2(step * A2[i]), h[k][i], du * bv[i]);
      y = fmaf(h[k][i], cv[i], y);
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) y += __shfl_xor_sync(kAll, y, o);
    if (mine && slot[k] >= 0)
      store_states(p.state + (size_t)slot[k] * width + at, i0, p.states, a.vec_state, h[k]);
    if (l == from || RR == 1) out[e] = y;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int k = L < RR ? e * L + l : l;
    if (mine && k < RR && r0 + k < p.tokens) {
      const float y = fmaf(skip, u[e], out[e]) * z[e];
      static_cast<T *>(p.y)[(size_t)(r0 + k) * p.ldy + c] = pack1<T>(y);
    }
  }
  if (bad && tid == 0 && cblk == 0 && group == 0) atomicOr(&g_ssm_status, CWGK_STATUS_INDEX);
}

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

static int done() {
  cwgk_count_launch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    cwgk_set_cuda_error((int)e);
    return -3;
  }
  return 0;
}

template <typename T, int L>
static int launch(const cwg_ssm *op, bool step, cudaStream_t s) {
  using G = Geo<L>;
  Args a;
  a.p = *op;
  if (op->tokens <= 1) a.p.ldu = a.p.lddt = a.p.ldz = a.p.ldy = 0, a.p.ldb = a.p.ldc = 0;
  a.per = op->channels / op->groups;
  a.cblocks = (a.per + G::kCH - 1) / G::kCH;
  a.vec_state = op->states == G::kNP && aligned16(op->state);
  a.vec_a = op->states == G::kNP && aligned16(op->A);
  a.vec_bc = op->states == G::kNP && ((uintptr_t)op->B % (4 * sizeof(T))) == 0 &&
             ((uintptr_t)op->C % (4 * sizeof(T))) == 0 && a.p.ldb % 4 == 0 && a.p.ldc % 4 == 0;
  const long long blocks = (long long)op->n_seq * a.cblocks * op->groups;
  const long long step_blocks = (long long)op->tokens * a.cblocks * op->groups;
  if ((step ? step_blocks : blocks) > 0x7fffffffLL) return -2;
  if (step) {
    // rows that share A as soon as every SM has work all the same
    if (step_blocks >= 4 * 4 * 148)
      ssm_token<T, L, 4><<<(unsigned)((long long)((op->tokens + 3) / 4) * a.cblocks * op->groups),
                           G::kThreads, 0, s>>>(a);
    else
      ssm_token<T, L, 1><<<(unsigned)step_blocks, G::kThreads, 0, s>>>(a);
    return done();
  }
  constexpr int E = 16 / (int)sizeof(T);
  const bool vec = a.per % 8 == 0 && aligned16(op->u) && aligned16(op->dt) && aligned16(op->z) &&
                   aligned16(op->y) && a.p.ldu % E == 0 && a.p.lddt % E == 0 &&
                   a.p.ldy % E == 0 && (!op->z || a.p.ldz % E == 0);
  if (vec)
    ssm_prompt<T, L, true><<<(unsigned)blocks, G::kThreads, 0, s>>>(a);
  else
    ssm_prompt<T, L, false><<<(unsigned)blocks, G::kThreads, 0, s>>>(a);
  return done();
}

template <typename T>
static int by_states(const cwg_ssm *op, bool step, cudaStream_t s) {
  if (op->states <= 4) return launch<T, 1>(op, step, s);
  if (op->states <= 8) return launch<T, 2>(op, step, s);
  if (op->states <= 16) return launch<T, 4>(op, step, s);
  if (op->states <= 32) return launch<T, 8>(op, step, s);
  return launch<T, 16>(op, step, s);
}

static int any(const cwg_ssm *op, bool step, cudaStream_t s) {
  return op->flags & CWG_BF16 ? by_states<__nv_bfloat16>(op, step, s) : by_states<float>(op, step, s);
}

}  // namespace ssm
}  // namespace cwg

extern "C" {

size_t cwgk_ssm_workspace_bytes(int tokens, int n_seq, int channels, int states) { return 256; }

int cwgk_ssm_scan(const cwg_ssm *op, void *workspace, size_t workspace_bytes, void *stream) {
  return cwg::ssm::any(op, false, (cudaStream_t)stream);
}

int cwgk_ssm_step(const cwg_ssm *op, void *stream) {
  return cwg::ssm::any(op, true, (cudaStream_t)stream);
}

int cwgk_ssm_read_clear_status(unsigned *status) {
  return cwg::read_clear_status(cwg::ssm::g_ssm_status, status);
}

}  // extern "C"
