// cwg_ssm.cu -- selective state space scan (cwg_ssm_scan, cwg_ssm_step).
//
// For every channel c with states i = 0 .. N-1, step d = softplus(dt + dt_bias):
//   h_i <- exp(d A_i) h_i + d u B_i,   y = (sum_i C_i h_i + D u) z / (1 + exp(-z))
//
// A channel's N states are spread over L lanes, four per lane (steps: eight where there are
// that many), N padded with A = B = C = 0, whose states stay zero; so a warp holds 32 / L
// channels.
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
  int chunk;    // prompts: tokens per chunk of a cut sequence, 0: not cut
  float *ends, *sums;  // cut sequences: see ssm_prompt
  bool vec_state, vec_a;  // the state's and A's rows are whole 16-byte vectors
  bool vec_bc;            // B and C can be read four states at a time
};

// A lane's four states of one cache line (or four values of A's row).
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

// A log2(e), kept finite: rows behind a sequence's last token have a step of zero, which has to
// leave the states as they are, and zero times an infinity would not.
__device__ __forceinline__ float decay_rate(float A) {
  constexpr float kMost = 3.402823466e38f;
  const float v = A * kLog2e;
  return fabsf(v) > kMost ? copysignf(kMost, v) : v;  // NaN stays
}

// ---- prompts --------------------------------------------------------------------
// One CTA per (sequence, block of kCH channels of one group) walks the sequence in tiles
// of kTT tokens, its warps in two roles that work on neighbouring tiles at the same time:
//   * scan warps hold the states and run the recurrence over tile i, reading the pairs
//     (d, d u) and B, C from shared memory; a channel's L lanes reduce L tokens' sums
//     together, so that each lane ends up with one token's (L - 1 shuffles per L tokens);
//   * element warps finish tile i - 1 (skip, gate, full-width row stores), prepare tile
//     i + 1 (step, d u) and start the asynchronous copies of tile i + 3.
// One barrier per tile.  Bound by the exponentials: N per token and channel at 16 a clock
// and SM; the elementwise part adds 4 more, and the shared-memory reads of B and C (kept
// in the input's type) come next.
template <int L>
struct Prompt {
  static constexpr int kCH = L <= 4 ? 32 : 128 / L;
  static constexpr int kScan = kCH * L;             // scan threads
  static constexpr int kTasks = kTT * kCH / 4;      // 4-channel pieces of a tile
  static constexpr int kElem = kTasks < 128 ? 128 : kTasks;  // element threads
  static constexpr int kThreads = kScan + kElem;
  // y rows: the L tokens x 32 / L channels of one store fall in (nearly) all banks
  static constexpr int kPitch = kCH + (L <= 8 ? 32 / L : 4);
  static_assert(kPitch % 4 == 0 && kCH % 8 == 0, "rows of whole vectors");
};

// Asynchronous copy of B bytes into shared memory; zeros where !ok.
template <int B>
__device__ __forceinline__ void copy_async(void *dst, const void *src, bool ok) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (B == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src),
                 "r"(ok ? 16 : 0)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(src), "n"(B),
                 "r"(ok ? B : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_wait() {  // all but the N newest groups have landed
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// Part of a tile that the element threads copy: W elements at a time of rows of `width`,
// of which n exist and `rows` hold tokens; consecutive threads take neighbouring
// pieces.  VEC: pieces of 16 bytes (or W elements if that is less), all aligned and n
// whole pieces.  Two-byte elements that are not aligned cannot be copied asynchronously.
template <typename T, int NT, int WIDTH, int W, bool VEC, typename Dst>
__device__ __forceinline__ void copy_rows(int e, const T *src, size_t ld, int n, int rows,
                                          Dst dst) {
  constexpr int B = W * (int)sizeof(T) < 16 ? W * (int)sizeof(T) : 16;
  constexpr int E = VEC ? B / (int)sizeof(T) : 1, per = WIDTH / E;
#pragma unroll
  for (int q0 = 0; q0 < kTT * per; q0 += NT) {
    const int q = q0 + e, t = q / per, c = q % per * E;
    if (kTT * per % NT && q >= kTT * per) break;
    const bool ok = t < rows && c < n;
    const T *from = ok ? src + (size_t)t * ld + c : src;
    if constexpr (E * sizeof(T) >= 4)
      copy_async<E * (int)sizeof(T)>(dst(t, c), from, ok);
    else
      *dst(t, c) = ok ? *from : from_f32<T>(0.f);
  }
}
// Barrier of the element warps alone.
template <int N>
__device__ __forceinline__ void named_bar() {
  asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
}
template <typename T>
__device__ __forceinline__ void read4(const T *p, float (&f)[4]) {
  unpack(load_raw<T, 4>(p), f);
}
template <typename T, bool VEC>
__device__ __forceinline__ void write4(T *p, const float (&f)[4], int n) {
  if constexpr (VEC) {
    store_raw<T, 4>(p, pack<T, 4>(f));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = pack1<T>(f[i]);
  }
}

__device__ __forceinline__ void unpack_word(uint2 v, float (&f)[2]) {
  f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y);
}
__device__ __forceinline__ void unpack_word(uint2 v, float (&f)[4]) { unpack(v, f); }
// A lane's four states' B and C of one token, in the input's type.
template <typename T>
struct alignas(16) LaneBC {
  static constexpr int kWords = 2 * kS * (int)sizeof(T) / 8;
  uint2 raw[kWords];
  __device__ __forceinline__ T *at(int i) { return reinterpret_cast<T *>(raw) + i; }
  __device__ __forceinline__ void read(const LaneBC &from) {  // in 16-byte vectors
#pragma unroll
    for (int i = 0; i < kWords; i += 2) {
      const uint4 q = *reinterpret_cast<const uint4 *>(from.raw + i);
      raw[i] = make_uint2(q.x, q.y);
      raw[i + 1] = make_uint2(q.z, q.w);
    }
  }
  __device__ __forceinline__ void get(F2 (&b)[kS / 2], F2 (&c)[kS / 2]) const {
    constexpr int E = 8 / (int)sizeof(T);  // values per word
    float f[2 * kS];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      float g[E];
      unpack_word(raw[i], g);
#pragma unroll
      for (int e = 0; e < E; ++e) f[i * E + e] = g[e];
    }
#pragma unroll
    for (int i = 0; i < kS / 2; ++i) {
      b[i] = f2(f[2 * i], f[2 * i + 1]);
      c[i] = f2(f[kS + 2 * i], f[kS + 2 * i + 1]);
    }
  }
};

// Where the pairs (d, d u) of channels 2 j, 2 j + 1 of an 8-channel piece are kept in
// their row: turned so that 8 threads' 16-byte stores fall in all banks.
__device__ __forceinline__ int turned(int t, int c8, int j) {
  return c8 * 4 + ((j + (c8 >> 1) + 2 * (t & 1)) & 3);
}

// Shared memory of a CTA: the rows of five tiles (three ahead of the one in work, one
// behind it; of three tiles, with one ahead, in kShort), the pairs and sums of two.
template <typename T, int L, int STAGES>
struct PromptSmem {
  using G = Prompt<L>;
  static constexpr int kStages = STAGES;
  float4 dx[2][kTT][G::kCH / 2];
  float y[2][kTT][G::kPitch];
  LaneBC<T> bc[kStages][kTT][L];
  T u[kStages][kTT][G::kCH], d[kStages][kTT][G::kCH], z[kStages][kTT][G::kCH];
};

// Cut sequences.  A recurrence is serial, so one sequence alone keeps n_seq x channels / 32
// CTAs busy; when that is few, sequences are cut into chunks of a.chunk tokens.  A first
// launch (SUMMARY) runs the recurrence of every chunk but a sequence's last, from zeros
// (the first chunk: from the sequence's state), without outputs, and keeps each chunk's
// end states and sum of steps.  In the second launch a chunk finds its initial state
// from those of the chunks before it,
//   h = end_0;  h = exp(A sum_j d) h + end_j,  j = 1 .. k - 1,
// and runs as a whole sequence does.  Exponentials are computed about 1.8 times.
//
// Chunk k of sequence b has index starts[b] / chunk + b + k: ascending offsets give every
// chunk an index of its own below tokens / chunk + n_seq.  `ends` and `sums` are kept by
// that index; the entry of a sequence's last chunk, which has no summary, keeps the state
// that the sequence begins with, since the last chunk may replace the cache line before the
// first one of the second launch has started.
//
// kRoomy is the whole kernel compiled for one CTA per SM: with 100 to 150 registers the scan
// warps' operands are read further ahead, which shortens a tile when a CTA has its SM for
// itself (nine fp32 sequences, 288 CTAs: 30 us, 40 dense; one of 4096 tokens x 2048 channels
// x 64 states: 233, 324), and costs occupancy when there are many CTAs (eight sequences of
// 1024 x 4096: 272 us, 232 dense).
//
// kShort keeps three tiles instead of five, so that more CTAs fit an SM when there are many
// sequences of about one tile, whose CTAs last as long as their latencies (18 sequences, 161
// tokens, 4 groups of 768 channels, 4 states, fp32: 30 us, 34 dense; 19 of 108
// tokens, 246 channels, 23 states, bf16: 6.4, 8.8).  The host knows the mean length only; one
// long sequence among many of one token does not lose by it either (4096 of one and one of 4096
// tokens, 256 channels, bf16: 359 us, 399 dense; 1024 and 8192, 1024 channels: 415, 440; fp32
// 466, 447).
enum { kDense = 0, kRoomy = 1, kSummary = 2, kShort = 3 };
template <int MODE>
constexpr int kStagesOf = MODE == kShort ? 3 : 5;
template <typename T, int L, bool VEC, bool VBC, int MODE>
__global__ void __launch_bounds__(Prompt<L>::kThreads, MODE == kRoomy ? 1 : 0)
    ssm_prompt(const Args a) {
  constexpr bool SUMMARY = MODE == kSummary;
  griddep_wait();
  griddep_launch_dependents();
  using G = Prompt<L>;
  constexpr int CH = G::kCH;
  using Smem = PromptSmem<T, L, kStagesOf<MODE>>;
  constexpr int NS = Smem::kStages;
  extern __shared__ __align__(16) unsigned char smem[];
  Smem &sh = *reinterpret_cast<Smem *>(smem);
  const cwg_ssm &p = a.p;
  const int tid = threadIdx.x;
  const int cblk = blockIdx.x % a.cblocks;
  const int group = (blockIdx.x / a.cblocks) % p.groups;
  const int index = blockIdx.x / (a.cblocks * p.groups);
  const int in0 = cblk * CH;            // first channel within the group
  const int c0 = group * a.per + in0;   // first channel
  const int nch = min(CH, a.per - in0);
  const bool report = tid == 0 && cblk == 0 && group == 0;
  int b = index, part = 0, parts = 1, head = index;  // sequence, its chunks, its first index
  if (a.chunk) {
    auto base = [&](int q) { return min(max(p.starts[q], 0), p.tokens) / a.chunk + q; };
    int hi = p.n_seq;
    b = 0;  // after the search: the first sequence with a base above `index`
    while (b < hi) {
      const int mid = (b + hi) >> 1;
      if (base(mid) <= index)
        b = mid + 1;
      else
        hi = mid;
    }
    if (blockIdx.x == 0 && !SUMMARY) {  // a sequence with bad offsets may have no index
      bool wrong = false;
      for (int q = tid; q < p.n_seq; q += G::kThreads)
        wrong |= p.starts[q] < 0 || p.starts[q + 1] < p.starts[q] || p.starts[q + 1] > p.tokens;
      if (wrong) atomicOr(&g_ssm_status, CWGK_STATUS_INDEX);
    }
    if (--b < 0) return;
    head = base(b);
    part = index - head;
  }
  int begin = p.starts[b], end = p.starts[b + 1];
  if (begin < 0 || end < begin || end > p.tokens) {
    if (report) atomicOr(&g_ssm_status, CWGK_STATUS_INDEX);
    return;
  }
  if (a.chunk) {
    parts = max(1, (end - begin + a.chunk - 1) / a.chunk);
    if (part >= parts || (SUMMARY && part == parts - 1)) return;
    begin += part * a.chunk;
    end = min(end, begin + a.chunk);
  }
  bool bad = false;
  const unsigned char resume = p.resume ? p.resume[b] : 0;
  const int slot = p.state ? line_of(p.slots, b, p.n_slots, bad) : -1;
  if (bad && report) atomicOr(&g_ssm_status, CWGK_STATUS_INDEX);
  const bool carry = slot >= 0 && resume;
  const int tiles = (end - begin + kTT - 1) / kTT;

  if (tid < G::kScan) {
    // ---- lane l of channel ch, states i0 .. i0 + 3
    const int ch = tid / L, l = tid % L, i0 = l * kS;
    const bool mine = ch < nch;
    float A2[kS] = {}, h[kS] = {};
    const size_t at = (size_t)(c0 + ch) * p.states;
    const size_t width = (size_t)p.channels * p.states;
    float *line = p.state + (size_t)(slot < 0 ? 0 : slot) * width + at;
    if (mine) {
      load_states(p.A + at, i0, p.states, a.vec_a, A2);
#pragma unroll
      for (int k = 0; k < kS; ++k) A2[k] = decay_rate(A2[k]);
      float *ends = a.ends + (size_t)head * width + at;  // of the sequence's first chunk
      const bool vec = p.states == kS * L;
      if (part == 0 && (SUMMARY || parts == 1)) {
        if (carry) load_states(line, i0, p.states, a.vec_state, h);
        if (SUMMARY) store_states(ends + (size_t)(parts - 1) * width, i0, p.states, vec, h);
      } else if (part == 0) {
        load_states(ends + (size_t)(parts - 1) * width, i0, p.states, vec, h);
      } else if (!SUMMARY) {
        load_states(ends, i0, p.states, vec, h);
#pragma unroll 4
        for (int j = 1; j < part; ++j) {
          float e[kS];
          load_states(ends + (size_t)j * width, i0, p.states, vec, e);
          const float d = a.sums[(size_t)(head + j) * p.channels + c0 + ch];
#pragma unroll
          for (int k = 0; k < kS; ++k) h[k] = fmaf(ex2(d * A2[k]), h[k], e[k]);
        }
      }
    }
    float sum_d = 0.f, lost_d = 0.f;  // of the steps, with what its additions lost
    F2 a2[kS / 2], hh[kS / 2];
#pragma unroll
    for (int k = 0; k < kS / 2; ++k) {
      a2[k] = f2(A2[2 * k], A2[2 * k + 1]);
      hh[k] = f2(h[2 * k], h[2 * k + 1]);
    }
    const int at0 = turned(0, ch >> 3, (ch & 7) >> 1) * 4 + (ch & 1) * 2;
    const int at1 = turned(1, ch >> 3, (ch & 7) >> 1) * 4 + (ch & 1) * 2;
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      const float *dx = reinterpret_cast<const float *>(sh.dx[i & 1]);
      const LaneBC<T>(*bc)[L] = sh.bc[i % NS];
      float(*ys)[G::kPitch] = sh.y[i & 1];
      // TG tokens at a time, their sums reduced together; the next ones' operands are read
      // while these are worked on
      constexpr int TG = L > 8 ? L : 8;
      float2 v[TG];
      LaneBC<T> w[TG];
      auto fetch = [&](int t0) {
#pragma unroll
        for (int t = 0; t < TG; ++t) {
          v[t] = *reinterpret_cast<const float2 *>(dx + (t0 + t) * (CH * 2) + (t & 1 ? at1 : at0));
          w[t].read(bc[t0 + t][l]);
        }
      };
      fetch(0);
#pragma unroll
      for (int t0 = 0; t0 < kTT; t0 += TG) {
        float y[TG];
        float2 dv[TG];
        LaneBC<T> sv[TG];
#pragma unroll
        for (int t = 0; t < TG; ++t) dv[t] = v[t], sv[t] = w[t];
        if (t0 + TG < kTT) fetch(t0 + TG);
#pragma unroll
        for (int t = 0; t < TG; ++t) {
          F2 bv[kS / 2], cv[kS / 2], sum;
          sv[t].get(bv, cv);
          const F2 dd = f2(dv[t].x, dv[t].x), uu = f2(dv[t].y, dv[t].y);
#pragma unroll
          for (int k = 0; k < kS / 2; ++k) {
            const float2 x = halves(mul2(dd, a2[k]));
            hh[k] = fma2(f2(ex2(x.x), ex2(x.y)), hh[k], mul2(uu, bv[k]));
            if (!SUMMARY) sum = k ? fma2(hh[k], cv[k], sum) : mul2(hh[k], cv[k]);
          }
          if (SUMMARY) {
            y[t] = dv[t].x;
          } else {
            const float2 s = halves(sum);
            y[t] = s.x + s.y;
          }
        }
        // a chunk's steps are added pairwise, then with compensation: their sum's rounding
        // enters the decay of everything before the chunk
        if constexpr (SUMMARY) {
#pragma unroll
          for (int o = 1; o < TG; o *= 2)
#pragma unroll
            for (int t = 0; t < TG; t += 2 * o) y[t] += y[t + o];
          const float to = sum_d + y[0], back = to - sum_d;
          lost_d += (sum_d - (to - back)) + (y[0] - back);
          sum_d = to;
        } else {
#pragma unroll
          for (int o = L / 2; o > 0; o >>= 1) {  // L tokens' sums over the channel's L lanes
            const bool up = l & o;
#pragma unroll
            for (int g = 0; g < TG; g += L)
#pragma unroll
              for (int k = 0; k < o; ++k) {
                const float give = up ? y[g + k] : y[g + k + o];
                const float keep = up ? y[g + k + o] : y[g + k];
                y[g + k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
              }
          }
#pragma unroll
          for (int g = 0; g < TG; g += L) ys[t0 + g + l][ch] = y[g];
        }
      }
      __syncthreads();
    }
    float out[kS];
#pragma unroll
    for (int k = 0; k < kS / 2; ++k) {
      const float2 x = halves(hh[k]);
      out[2 * k] = x.x, out[2 * k + 1] = x.y;
    }
    if (SUMMARY && mine) {
      store_states(a.ends + (size_t)index * width + at, i0, p.states, p.states == kS * L, out);
      if (l == 0) a.sums[(size_t)index * p.channels + c0 + ch] = sum_d + lost_d;
    }
    if (!SUMMARY && slot >= 0 && mine && part == parts - 1)
      store_states(line, i0, p.states, a.vec_state, out);
  } else {
    // ---- 4-channel pieces of the tiles' rows
    const int e = tid - G::kScan;
    const int tt = e / (CH / 4), c4 = e % (CH / 4), c = c4 * 4;
    const bool task = e < G::kTasks && c < nch;
    float bias[4], skip[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool ok = task && c + k < nch;
      bias[k] = ok && p.dt_bias ? p.dt_bias[c0 + c + k] : 0.f;
      skip[k] = ok && p.D ? p.D[c0 + c + k] : 0.f;
    }
    auto load = [&](int i) {
      const int st = i % NS, t0 = begin + i * kTT, rows = end - t0;
      const size_t at = (size_t)(rows > 0 ? t0 : begin), col = (size_t)group * p.states;
      auto rows_of = [&](const void *src, long long ld, T(*to)[CH]) {
        copy_rows<T, G::kElem, CH, 8, VEC>(e, static_cast<const T *>(src) + at * ld + c0,
                                           (size_t)ld, nch, rows,
                                           [&](int t, int k) { return &to[t][k]; });
      };
      rows_of(p.u, p.ldu, sh.u[st]);
      rows_of(p.dt, p.lddt, sh.d[st]);
      if (p.z && !SUMMARY) rows_of(p.z, p.ldz, sh.z[st]);
      copy_rows<T, G::kElem, kS * L, kS, VBC>(
          e, static_cast<const T *>(p.B) + at * p.ldb + col, (size_t)p.ldb, p.states, rows,
          [&](int t, int k) { return sh.bc[st][t][k / kS].at(k % kS); });
      if (!SUMMARY)
        copy_rows<T, G::kElem, kS * L, kS, VBC>(
            e, static_cast<const T *>(p.C) + at * p.ldc + col, (size_t)p.ldc, p.states, rows,
            [&](int t, int k) { return sh.bc[st][t][k / kS].at(kS + k % kS); });
      copy_commit();
    };
    // pairs (d, d u); rows past the end have d = 0, which leaves the states as they are
    auto prepare = [&](int i) {
      const bool row = begin + i * kTT + tt < end;
      if (e < G::kTasks) {
        float u[4], d[4];
        read4(&sh.u[i % NS][tt][c], u);
        read4(&sh.d[i % NS][tt][c], d);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float v = d[k] + bias[k];
          if (p.flags & CWG_SOFTPLUS) v = softplus(v);
          d[k] = row && c + k < nch ? v : 0.f;
          u[k] = row && c + k < nch ? v * u[k] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
          sh.dx[i & 1][tt][turned(tt, c4 >> 1, (c4 & 1) * 2 + k)] =
              make_float4(d[2 * k], u[2 * k], d[2 * k + 1], u[2 * k + 1]);
      }
    };
    auto finish = [&](int i) {
      const int t = begin + i * kTT + tt;
      if (!task || t >= end) return;
      float u[4], z[4], y[4];
      read4(&sh.u[i % NS][tt][c], u);
      read4(&sh.y[i & 1][tt][c], y);
      if (p.z) read4(&sh.z[i % NS][tt][c], z);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        y[k] = fmaf(skip[k], u[k], y[k]);
        if (p.z) y[k] *= silu<T>(z[k]);
      }
      write4<T, VEC>(static_cast<T *>(p.y) + (size_t)t * p.ldy + c0 + c, y, nch - c);
    };
    // All element threads' copies of a tile have landed when the barrier behind their
    // waits is passed; the scan warps need B and C, the element threads each other's rows.
    if (tiles > 0) {
      load(0);
      if constexpr (NS == 5) {
        load(1);
        load(2);
      }
      copy_wait<NS == 5 ? 1 : 0>();
    }
    named_bar<G::kElem>();
    if (tiles > 0) prepare(0);
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      if (i > 0 && !SUMMARY) finish(i - 1);
      if (i + 1 < tiles) {
        load(i + NS - 2);  // where tile i - 2 was
        if constexpr (NS == 5) {
          prepare(i + 1);
          copy_wait<1>();  // tile i + 2
        } else {
          copy_wait<0>();
          named_bar<G::kElem>();
          prepare(i + 1);
        }
      }
      __syncthreads();
    }
    if (tiles > 0 && !SUMMARY) finish(tiles - 1);
    copy_wait<0>();
  }
}

template <int V, int L>
struct Geo {
  static constexpr int kCH = V * L <= 4 ? 64 : 256 / (V * L);
  static constexpr int kThreads = kCH * L;
  static constexpr int kNP = 4 * V * L;
};

// How a step's states, A, B and C are read: one at a time; four at a time, where there are
// whole fours of them; states == 4 V L, in the widest vectors.
enum { kSingle = 0, kFours = 1, kWhole = 2 };

// One row's B or C of a lane: 4 V values, as they are in memory.
template <typename T, int V, int VEC>
struct Row4 {
  static constexpr int E =
      !VEC ? 1 : VEC == kWhole && V * 4 * (int)sizeof(T) >= 16 ? 16 / (int)sizeof(T) : 4;
  typename Raw<T, E>::type raw[4 * V / E];
  __device__ __forceinline__ void load(const T *p, int n) {  // n of them exist
#pragma unroll
    for (int i = 0; i < 4 * V; i += E) raw[i / E] = i < n ? load_raw<T, E>(p + i) : zero_raw<T, E>();
  }
  __device__ __forceinline__ void get(F2 (&v)[2 * V]) const {
    float f[4 * V];
#pragma unroll
    for (int i = 0; i < 4 * V; i += E) {
      float g[E];
      unpack(raw[i / E], g);
#pragma unroll
      for (int e = 0; e < E; ++e) f[i + e] = g[e];
    }
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
  }
};

// 4 V states per lane: 8 where there are that many, since what a row costs besides its
// states (step, shuffles, addresses) is then paid by half as many threads.
template <typename T, int V, int L, int RR, int VEC>
__global__ void __launch_bounds__(Geo<V, L>::kThreads) ssm_token(const Args a) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int CH = Geo<V, L>::kCH, NT = Geo<V, L>::kThreads;
  const cwg_ssm &p = a.p;
  const int tid = threadIdx.x;
  const int cblk = blockIdx.x, group = blockIdx.y, r0 = (int)blockIdx.z * RR;
  const int ch = tid / L, l = tid % L, i0 = l * 4 * V;
  const int in = cblk * CH + ch, c = group * a.per + in;
  const bool mine = in < a.per;
  auto exists = [&](int v) { return VEC != kFours || i0 + 4 * v < p.states; };
  const int rows = min(RR, p.tokens - r0);
  const size_t width = (size_t)p.channels * p.states;
  float *state = p.state + (size_t)c * p.states;
  // Rows r0 + l, r0 + l + L, ... of the channel are lane l's: it computes their steps and
  // finishes their outputs (with more lanes than rows, lane l takes row l % RR too, which
  // only lane l = row stores).
  constexpr int E = L < RR ? RR / L : 1;
  int slot[RR];
  bool bad = false;
#pragma unroll
  for (int k = 0; k < RR; ++k) {
    slot[k] = k >= rows ? -1 : p.slots ? p.slots[r0 + k] : r0 + k;
    if (slot[k] >= p.n_slots) slot[k] = -1, bad = true;
  }
  float h[RR][V][kS], u[E], d[E], z[E];
  Row4<T, V, VEC> bv[RR], cv[RR];
#pragma unroll
  for (int k = 0; k < RR; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int i = 0; i < kS; ++i) h[k][v][i] = 0.f;
      if (mine && slot[k] >= 0 && exists(v))
        load_states(state + (size_t)slot[k] * width, i0 + 4 * v, p.states, VEC, h[k][v]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int k = L < RR ? e * L + l : l % RR;
    const size_t r = (size_t)(r0 + (k < rows ? k : 0));
    u[e] = d[e] = z[e] = 0.f;
    if (mine) {
      u[e] = to_f32(static_cast<const T *>(p.u)[r * p.ldu + c]);
      d[e] = to_f32(static_cast<const T *>(p.dt)[r * p.lddt + c]);
      if (p.z) z[e] = to_f32(static_cast<const T *>(p.z)[r * p.ldz + c]);
    }
  }
  const T *Brow =
      static_cast<const T *>(p.B) + (size_t)r0 * p.ldb + (size_t)group * p.states + i0;
  const T *Crow =
      static_cast<const T *>(p.C) + (size_t)r0 * p.ldc + (size_t)group * p.states + i0;
#pragma unroll
  for (int k = 0; k < RR; ++k) {
    bv[k].load(Brow + (size_t)k * p.ldb, k < rows ? p.states - i0 : 0);
    cv[k].load(Crow + (size_t)k * p.ldc, k < rows ? p.states - i0 : 0);
  }
  F2 a2[2 * V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float f[kS] = {0.f, 0.f, 0.f, 0.f};
    if (mine && exists(v))
      load_states(p.A + (size_t)c * p.states, i0 + 4 * v, p.states, VEC, f);
    a2[2 * v] = f2(f[0] * kLog2e, f[1] * kLog2e);
    a2[2 * v + 1] = f2(f[2] * kLog2e, f[3] * kLog2e);
  }
  const float bias = mine && p.dt_bias ? p.dt_bias[c] : 0.f;
  const float skip = mine && p.D ? p.D[c] : 0.f;
  if (p.slots) {
    int taken = 0;
    const int upto = min(r0 + RR - 1, p.tokens);
    for (int i = tid; i < upto; i += NT) {
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
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < kS; ++i) h[k][v][i] = 0.f;
        }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    d[e] += bias;
    if (p.flags & CWG_SOFTPLUS) d[e] = softplus(d[e]);
    z[e] = p.z ? silu<T>(z[e]) : 1.f;
  }
  float out[E] = {};
#pragma unroll
  for (int k = 0; k < RR; ++k) {
    // lane and piece that hold row k's step
    constexpr unsigned kAll = 0xffffffffu;
    const int from = L < RR ? k % L : k, e = L < RR ? k / L : 0;
    const float step = L > 1 && RR > 1 ? __shfl_sync(kAll, d[e], from, L) : d[e];
    const float uk = L > 1 && RR > 1 ? __shfl_sync(kAll, u[e], from, L) : u[e];
    const float du = step * uk;
    F2 b[2 * V], q[2 * V], sum;
    bv[k].get(b);
    cv[k].get(q);
    const F2 ss = f2(step, step), dd = f2(du, du);
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) {
      float *hh = h[k][i / 2] + i % 2 * 2;
      const float2 x = halves(mul2(ss, a2[i]));
      const F2 w = fma2(f2(ex2(x.x), ex2(x.y)), f2(hh[0], hh[1]), mul2(dd, b[i]));
      sum = i ? fma2(w, q[i], sum) : mul2(w, q[i]);
      const float2 f = halves(w);
      hh[0] = f.x, hh[1] = f.y;
    }
    const float2 s = halves(sum);
    float y = s.x + s.y;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) y += __shfl_xor_sync(kAll, y, o);
    if (mine && slot[k] >= 0) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (exists(v))
          store_states(state + (size_t)slot[k] * width, i0 + 4 * v, p.states, VEC, h[k][v]);
    }
    if (l == from || RR == 1) out[e] = y;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int k = L < RR ? e * L + l : l;
    if (mine && k < rows) {
      const float y = fmaf(skip, u[e], out[e]) * z[e];
      static_cast<T *>(p.y)[(size_t)(r0 + k) * p.ldy + c] = pack1<T>(y);
    }
  }
  if (bad && tid == 0 && cblk == 0 && group == 0) atomicOr(&g_ssm_status, CWGK_STATUS_INDEX);
}

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <typename K>
static int start(K kernel, dim3 grid, unsigned threads, size_t smem, cudaStream_t s,
                 const Args &a) {
  const cudaError_t e =
      launch_dependent(kernel, grid, threads, smem, s, !(a.p.flags & CWG_NO_PDL), 1, a);
  cwgk_count_launch();
  if (e != cudaSuccess) {
    cwgk_set_cuda_error((int)e);
    return -3;
  }
  return 0;
}

template <typename T, int L, bool VEC, bool VBC>
static int launch_prompt(const Args &a, unsigned blocks, cudaStream_t s) {
  constexpr int bytes = (int)sizeof(PromptSmem<T, L, 5>), threads = Prompt<L>::kThreads;
  constexpr int short_bytes = (int)sizeof(PromptSmem<T, L, 3>);
  cudaError_t e = smem_attr_once<ssm_prompt<T, L, VEC, VBC, kDense>>(bytes);
  if (e == cudaSuccess) e = smem_attr_once<ssm_prompt<T, L, VEC, VBC, kRoomy>>(bytes);
  if (e == cudaSuccess) e = smem_attr_once<ssm_prompt<T, L, VEC, VBC, kSummary>>(bytes);
  if (e == cudaSuccess) e = smem_attr_once<ssm_prompt<T, L, VEC, VBC, kShort>>(short_bytes);
  if (e != cudaSuccess) {
    cwgk_set_cuda_error((int)e);
    return -3;
  }
  if (a.chunk) {
    const int rc = start(ssm_prompt<T, L, VEC, VBC, kSummary>, dim3(blocks), threads, bytes, s, a);
    if (rc) return rc;
  }
  if (blocks > 2 * 148 && a.p.tokens / a.p.n_seq <= kTT)
    return start(ssm_prompt<T, L, VEC, VBC, kShort>, dim3(blocks), threads, short_bytes, s, a);
  const auto kernel = blocks <= 2 * 148 ? ssm_prompt<T, L, VEC, VBC, kRoomy>
                                        : ssm_prompt<T, L, VEC, VBC, kDense>;
  return start(kernel, dim3(blocks), threads, bytes, s, a);
}

// Tokens per chunk when a call's sequences are cut, else 0.  `ctas`: CTAs along the
// channels.  Cut where at most half of the SMs would have a CTA.  Chunks of 128 to 256 tokens if
// all their CTAs then have an SM each (1024 tokens, 256 channels: 16 us, 23 in chunks of 256;
// 1024 channels: 24 us in four chunks, 29 in eight), else of 256 or more, as many as make three
// CTAs per SM (8192 tokens and 256, 1024, 2048 channels: 52, 130, 254 us, 300 uncut).  One
// sequence is cut from three chunks on (512 tokens, 1024 channels: 16 us, 22 uncut), several
// from two chunks on average, since the longest one's length decides uncut (4096 tokens in two
// sequences, 1024 channels: 75 us cut; uncut 76 if they are equally long, 100 if one has two
// thirds; in eight, 256 channels: 27 to 30, uncut 22 and 36).
static int chunk_of(int tokens, int n_seq, long long ctas) {
  if (n_seq <= 0 || ctas * n_seq > 74) return 0;
  const long long parts = 148 / ctas - (n_seq - 1);  // each sequence but one: a last, short one
  auto tiles_of = [](long long n) { return (n + kTT - 1) / kTT * kTT; };
  long long chunk = tiles_of((tokens + parts - 1) / parts);
  if (chunk < 128) chunk = 128;
  if (chunk > 256) chunk = tiles_of((tokens * ctas + 3 * 148 - 1) / (3 * 148));
  if (chunk < 256 && tokens > parts * chunk) chunk = 256;
  return tokens / n_seq >= (n_seq > 1 ? 2 : 3) * chunk ? (int)chunk : 0;
}
static size_t al256(size_t n) { return (n + 255) / 256 * 256; }
static size_t ends_bytes(long long slots, int channels, int states) {
  return al256((size_t)slots * channels * states * 4);
}

static size_t workspace_bytes(long long slots, int channels, int states) {
  return ends_bytes(slots, channels, states) + al256((size_t)slots * channels * 4);
}

// lane: values of B and C that are read at a time.
static Args make_args(const cwg_ssm *op, int np, int lane, size_t esz) {
  Args a;
  a.p = *op;
  if (op->tokens <= 1) a.p.ldu = a.p.lddt = a.p.ldz = a.p.ldy = 0, a.p.ldb = a.p.ldc = 0;
  a.per = op->channels / op->groups;
  a.cblocks = a.chunk = 0;
  a.ends = a.sums = nullptr;
  a.vec_state = op->states == np && aligned16(op->state);
  a.vec_a = op->states == np && aligned16(op->A);
  a.vec_bc = op->states % lane == 0 && ((uintptr_t)op->B % (lane * esz)) == 0 &&
             ((uintptr_t)op->C % (lane * esz)) == 0 && a.p.ldb % lane == 0 &&
             a.p.ldc % lane == 0;
  return a;
}

template <typename T, int L>
static int prompts(const cwg_ssm *op, void *workspace, cudaStream_t s) {
  Args a = make_args(op, kS * L, 4, sizeof(T));
  a.cblocks = (a.per + Prompt<L>::kCH - 1) / Prompt<L>::kCH;
  const long long ctas = (long long)a.cblocks * op->groups;
  a.chunk = workspace ? chunk_of(op->tokens, op->n_seq, ctas) : 0;
  const long long slots = a.chunk ? op->tokens / a.chunk + op->n_seq : op->n_seq;
  if (a.chunk) {
    a.ends = static_cast<float *>(workspace);
    a.sums = a.ends + ends_bytes(slots, op->channels, op->states) / 4;
  }
  const long long blocks = slots * ctas;
  if (blocks > 0x7fffffffLL) return -2;
  constexpr int E = 16 / (int)sizeof(T);
  const bool vec = a.per % 8 == 0 && aligned16(op->u) && aligned16(op->dt) && aligned16(op->z) &&
                   aligned16(op->y) && a.p.ldu % E == 0 && a.p.lddt % E == 0 &&
                   a.p.ldy % E == 0 && (!op->z || a.p.ldz % E == 0);
  if (vec && a.vec_bc) return launch_prompt<T, L, true, true>(a, (unsigned)blocks, s);
  if (vec) return launch_prompt<T, L, true, false>(a, (unsigned)blocks, s);
  if (a.vec_bc) return launch_prompt<T, L, false, true>(a, (unsigned)blocks, s);
  return launch_prompt<T, L, false, false>(a, (unsigned)blocks, s);
}

template <typename T, int V, int L>
static int steps(const cwg_ssm *op, cudaStream_t s) {
  using G = Geo<V, L>;
  Args a = make_args(op, G::kNP, V * 4 * sizeof(T) >= 16 ? 16 / (int)sizeof(T) : 4, sizeof(T));
  a.cblocks = (a.per + G::kCH - 1) / G::kCH;
  if (op->groups > 65535 || op->tokens > 65535) return -2;
  // two rows that share A as soon as every SM has work all the same (256 rows of 4096 x 16:
  // 38.4 us with four)
  const long long blocks = (long long)op->tokens * a.cblocks * op->groups;
  const bool two = blocks >= 4 * 2 * 148, whole = a.vec_state && a.vec_a && a.vec_bc;
  const bool fours = op->states % 4 == 0 && aligned16(op->state) && aligned16(op->A) &&
                     make_args(op, G::kNP, 4, sizeof(T)).vec_bc;
  const dim3 grid((unsigned)a.cblocks, (unsigned)op->groups,
                  (unsigned)(two ? (op->tokens + 1) / 2 : op->tokens));
  // 318 rows of 3456 x 12 bf16: 45 us one at a time, 29 in fours
  const auto kernel = two     ? (whole   ? ssm_token<T, V, L, 2, kWhole>
                                 : fours ? ssm_token<T, V, L, 2, kFours>
                                         : ssm_token<T, V, L, 2, kSingle>)
                      : whole ? ssm_token<T, V, L, 1, kWhole>
                      : fours ? ssm_token<T, V, L, 1, kFours>
                              : ssm_token<T, V, L, 1, kSingle>;
  return start(kernel, grid, G::kThreads, 0, s, a);
}

template <typename T, int L>
static int launch(const cwg_ssm *op, bool step, void *workspace, cudaStream_t s) {
  constexpr int V = L > 1 ? 2 : 1;
  return step ? steps<T, V, L / V>(op, s) : prompts<T, L>(op, workspace, s);
}

template <typename T>
static int by_states(const cwg_ssm *op, bool step, void *workspace, cudaStream_t s) {
  if (op->states <= 4) return launch<T, 1>(op, step, workspace, s);
  if (op->states <= 8) return launch<T, 2>(op, step, workspace, s);
  if (op->states <= 16) return launch<T, 4>(op, step, workspace, s);
  if (op->states <= 32) return launch<T, 8>(op, step, workspace, s);
  return launch<T, 16>(op, step, workspace, s);
}

static int any(const cwg_ssm *op, bool step, void *workspace, cudaStream_t s) {
  return op->flags & CWG_BF16 ? by_states<__nv_bfloat16>(op, step, workspace, s)
                              : by_states<float>(op, step, workspace, s);
}

static int channels_per_cta(int states) {
  return states <= 16 ? 32 : states <= 32 ? Prompt<8>::kCH : Prompt<16>::kCH;
}

}  // namespace ssm
}  // namespace cwg

extern "C" {

// An upper bound over all calls of at most so many tokens and sequences, and any groups.  A
// cut call has n_seq <= 74 / ctas, chunks of at least 128 tokens, and of at least tokens x ctas /
// 444 (see chunk_of: else all of its CTAs have an SM, ctas chunks <= 148); more groups make more
// CTAs along the channels than one.
size_t cwgk_ssm_workspace_bytes(int tokens, int n_seq, int channels, int states) {
  using namespace cwg::ssm;
  const int ch = channels_per_cta(states);
  const long long ctas = (channels + ch - 1) / ch;
  if (ctas > 74 || n_seq < 1 || tokens < 3 * 128) return 256;
  const long long chunks = tokens / 128 < 444 / ctas ? tokens / 128 : 444 / ctas;
  return workspace_bytes(chunks + (n_seq < 74 / ctas ? n_seq : 74 / ctas), channels, states);
}

size_t cwgk_ssm_call_bytes(const cwg_ssm *op) {
  using namespace cwg::ssm;
  const int ch = channels_per_cta(op->states), per = op->channels / op->groups;
  const int chunk = chunk_of(op->tokens, op->n_seq, (long long)((per + ch - 1) / ch) * op->groups);
  return chunk ? workspace_bytes(op->tokens / chunk + op->n_seq, op->channels, op->states) : 256;
}

int cwgk_ssm_scan(const cwg_ssm *op, void *workspace, void *stream) {
  return cwg::ssm::any(op, false, workspace, (cudaStream_t)stream);
}

int cwgk_ssm_step(const cwg_ssm *op, void *stream) {
  return cwg::ssm::any(op, true, nullptr, (cudaStream_t)stream);
}

int cwgk_ssm_read_clear_status(unsigned *status) {
  return cwg::read_clear_status(cwg::ssm::g_ssm_status, status);
}

}  // extern "C"
