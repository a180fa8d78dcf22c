// cwg_conv1d.cu -- short causal convolution over time, one filter per channel
// (cwg_conv1d_causal, cwg_conv1d_causal_step).
//
//   y[t][c] = act(bias[c] + sum_{j < K} w[c][j] x[t - K + 1 + j][c]),  K = 2 .. 4
//
// 2K flops and one exponential per element against 4 bytes (bf16) or 8 (fp32) in
// and out: bound by memory.
//
// Prompts: a thread owns one 16-byte vector of channels and a run of consecutive
// rows, so that a row is read once (plus K - 1 rows of halo per run) and the
// window slides through registers while the next four rows are loaded.
// The K - 1 first rows of a sequence, which need the cache line, are all computed
// by the thread whose run holds the sequence's first row, and that thread stores
// the new line after it: no other thread reads a line, so the old line can be
// replaced within the same launch.  All other rows are plain windows.
#include <cstdint>

#include "../../include/cwg.h"
#include "cwg_seq.cuh"

namespace cwg {
namespace seq {

__device__ unsigned int g_seq_status;

constexpr int kConvThreads = 128;
constexpr int kAhead = 4;          // rows per step; the next step's are loaded meanwhile
constexpr int kStartsInSmem = 1024;

template <typename T, int ACT>
__device__ __forceinline__ float activate(float v) {
  if (ACT == CWGK_ACT_RELU) return v < 0.f ? 0.f : v;  // NaN stays
  if (ACT == CWGK_ACT_SILU) return silu<T>(v);
  return v;
}

struct ConvArgs {
  const void *x;
  const float *w, *bias;
  void *y, *state;
  const int *starts, *slots;
  const unsigned char *resume;
  size_t ldx, ldy;
  int tokens, n_seq, n_slots, channels;
  int cblocks;  // CTAs along the channels
  int wc;       // warps along the channels; the CTA's other warps take further runs
  int run;      // rows per run (prompts) or per thread (steps), a multiple of kAhead
  int runs;
};

template <int V, int K>
__device__ __forceinline__ void load_weights(const ConvArgs &a, int c, bool active,
                                             float (&w)[V][K], float (&b)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    b[v] = active && a.bias ? a.bias[c + v] : 0.f;
    if (V > 1 && K == 4) {  // 16-byte aligned: the host checked w for the vector path
      const float4 f = active ? *reinterpret_cast<const float4 *>(a.w + (size_t)(c + v) * K)
                              : make_float4(0, 0, 0, 0);
      w[v][0] = f.x;
      w[v][1] = f.y;
      w[v][K > 2 ? 2 : 0] = f.z;
      w[v][K - 1] = f.w;
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j) w[v][j] = active ? a.w[(size_t)(c + v) * K + j] : 0.f;
    }
  }
}

// act(b + sum_j w[j] h[j]) with h the window's rows, oldest first, x the newest.
template <typename T, int V, int K, int ACT>
__device__ __forceinline__ void window_row(const float (&w)[V][K], const float (&b)[V],
                                           const float (&h)[K - 1][V], const float (&x)[V],
                                           float (&y)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float s = b[v];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) s = fmaf(w[v][j], h[j][v], s);
    y[v] = activate<T, ACT>(fmaf(w[v][K - 1], x[v], s));
  }
}
template <int V, int K>
__device__ __forceinline__ void slide(float (&h)[K - 1][V], const float (&x)[V]) {
#pragma unroll
  for (int j = 0; j < K - 2; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) h[j][v] = h[j + 1][v];
#pragma unroll
  for (int v = 0; v < V; ++v) h[K - 2][v] = x[v];
}

template <typename T, int V, int K, int ACT>
__global__ void __launch_bounds__(kConvThreads, 4) conv1d_prompt(const ConvArgs a) {
  __shared__ int s_starts[kStartsInSmem + 1];
  const T *x = static_cast<const T *>(a.x);
  T *y = static_cast<T *>(a.y);
  T *state = static_cast<T *>(a.state);
  const int *starts = a.starts;
  if (a.n_seq <= kStartsInSmem) {
    for (int i = threadIdx.x; i <= a.n_seq; i += kConvThreads) s_starts[i] = a.starts[i];
    __syncthreads();
    starts = s_starts;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cb = blockIdx.x % a.cblocks;
  const int run = (blockIdx.x / a.cblocks) * (4 / a.wc) + warp / a.wc;
  if (run >= a.runs) return;  // a whole warp
  const int c = ((cb * a.wc + warp % a.wc) * 32 + lane) * V;
  const bool active = c < a.channels;
  const int t0 = run * a.run;
  const int t1 = min(t0 + a.run, a.tokens);

  float w[V][K], b[V], h[K - 1][V];
  load_weights<V, K>(a, c, active, w, b);

  // Sequences that begin in this run (the first run also has those that begin
  // before row 0 by a bad offset, the last one those that begin at the end).
  const int first = run == 0 ? 0 : lower_bound(starts, a.n_seq, t0);
  const int last = run == a.runs - 1 ? a.n_seq : lower_bound(starts, a.n_seq, t0 + a.run);
  bool bad = false;
  for (int s = first; s < last; ++s) {
    const int begin = starts[s], end = starts[s + 1];
    if (begin < 0 || end < begin || end > a.tokens) {
      bad = true;
      continue;
    }
    const int slot = state ? line_of(a.slots, s, a.n_slots, bad) : -1;
    const bool carry = slot >= 0 && a.resume && a.resume[s];
    if (!active) continue;
    T *line = state + ((size_t)(slot < 0 ? 0 : slot) * (K - 1)) * a.channels + c;
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
      unpack(carry ? load_raw<T, V>(line + (size_t)j * a.channels) : zero_raw<T, V>(), h[j]);
    const int len = end - begin;
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      if (i < len) {
        float xv[V], yv[V];
        unpack(load_raw<T, V>(x + (size_t)(begin + i) * a.ldx + c), xv);
        window_row<T, V, K, ACT>(w, b, h, xv, yv);
        store_raw<T, V>(y + (size_t)(begin + i) * a.ldy + c, pack<T, V>(yv));
        slide<V, K>(h, xv);
      }
    }
    if (slot >= 0) {
#pragma unroll
      for (int j = 0; j < K - 1; ++j)
        store_raw<T, V>(line + (size_t)j * a.channels,
                        len >= K - 1 ? load_raw<T, V>(x + (size_t)(end - (K - 1) + j) * a.ldx + c)
                                     : pack<T, V>(h[j]));
    }
  }
  if (bad && lane == 0 && c == 0) atomicOr(&g_seq_status, CWGK_STATUS_INDEX);
  if (!active) return;

  // The rows with a whole window inside their sequence.
  int s = lower_bound(starts, a.n_seq, t0 + 1) - 1;  // the last one that begins by row t0
  int begin = 0, end = 0;                            // empty: nothing before the first
  if (s >= 0) begin = starts[s], end = starts[s + 1];
  if (begin < 0 || end > a.tokens) end = begin = 0;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const int t = t0 - (K - 1) + j;
    unpack(t >= 0 && t < a.tokens ? load_raw<T, V>(x + (size_t)t * a.ldx + c) : zero_raw<T, V>(),
           h[j]);
  }
  typename Raw<T, V>::type raw[kAhead], next[kAhead];
  auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      next[i] = t + i < t1 ? load_raw<T, V>(x + (size_t)(t + i) * a.ldx + c) : zero_raw<T, V>();
  };
  fetch(t0);
  for (int t = t0; t < t1; t += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) raw[i] = next[i];
    fetch(t + kAhead);
    if (t - begin >= K - 1 && t + kAhead <= end) {  // all of one sequence, as nearly always
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        float xv[V], yv[V];
        unpack(raw[i], xv);
        window_row<T, V, K, ACT>(w, b, h, xv, yv);
        store_raw<T, V>(y + (size_t)(t + i) * a.ldy + c, pack<T, V>(yv));
        slide<V, K>(h, xv);
      }
      continue;
    }
#pragma unroll 1
    for (int i = 0; i < kAhead; ++i) {
      if (t + i >= t1) break;
      while (s + 1 < a.n_seq && starts[s + 1] <= t + i) {
        ++s;
        begin = starts[s];
        end = starts[s + 1];
        if (begin < 0 || end > a.tokens) end = begin = 0;
      }
      float xv[V];
      unpack(i == 0 ? raw[0] : i == 1 ? raw[1] : i == 2 ? raw[2] : raw[3], xv);
      if (t + i < end && t + i - begin >= K - 1) {
        float yv[V];
        window_row<T, V, K, ACT>(w, b, h, xv, yv);
        store_raw<T, V>(y + (size_t)(t + i) * a.ldy + c, pack<T, V>(yv));
      }
      slide<V, K>(h, xv);
    }
  }
}

// One token of each sequence: a thread owns a vector of channels and `run` rows,
// which share the weights; per row K vectors in and K out (x and the line, y and
// the line moved by one).
template <typename T, int V, int K, int ACT>
__global__ void __launch_bounds__(kConvThreads) conv1d_step(const ConvArgs a) {
  const T *x = static_cast<const T *>(a.x);
  T *y = static_cast<T *>(a.y);
  T *state = static_cast<T *>(a.state);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cb = blockIdx.x % a.cblocks;
  const int run = (blockIdx.x / a.cblocks) * (4 / a.wc) + warp / a.wc;
  if (run >= a.runs) return;
  const int c = ((cb * a.wc + warp % a.wc) * 32 + lane) * V;
  const bool active = c < a.channels;
  float w[V][K], b[V];
  load_weights<V, K>(a, c, active, w, b);
  bool bad = false;
  const int r1 = min((run + 1) * a.run, a.n_seq);
  for (int r = run * a.run; r < r1; ++r) {
    const int slot = line_of(a.slots, r, a.n_slots, bad);
    if (!active) continue;
    T *line = state + ((size_t)(slot < 0 ? 0 : slot) * (K - 1)) * a.channels + c;
    typename Raw<T, V>::type raw[K];
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
      raw[j] = slot >= 0 ? load_raw<T, V>(line + (size_t)j * a.channels) : zero_raw<T, V>();
    raw[K - 1] = load_raw<T, V>(x + (size_t)r * a.ldx + c);
    float h[K - 1][V], xv[V], yv[V];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) unpack(raw[j], h[j]);
    unpack(raw[K - 1], xv);
    window_row<T, V, K, ACT>(w, b, h, xv, yv);
    store_raw<T, V>(y + (size_t)r * a.ldy + c, pack<T, V>(yv));
    if (slot >= 0) {
#pragma unroll
      for (int j = 0; j < K - 1; ++j)
        store_raw<T, V>(line + (size_t)j * a.channels, raw[j + 1]);
    }
  }
  if (bad && lane == 0 && c == 0) atomicOr(&g_seq_status, CWGK_STATUS_INDEX);
}

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <typename T, int V, int K, int ACT>
static int launch_conv1d(const cwgk_conv1d *op, bool step, cudaStream_t stream) {
  ConvArgs a;
  a.x = op->x;
  a.w = op->w;
  a.bias = op->bias;
  a.y = op->y;
  a.state = op->state;
  a.starts = op->starts;
  a.slots = op->slots;
  a.resume = op->resume;
  a.ldx = (size_t)op->ldx;
  a.ldy = (size_t)op->ldy;
  a.tokens = op->tokens;
  a.n_seq = op->n_seq;
  a.n_slots = op->n_slots;
  a.channels = op->channels;
  const int warps = (op->channels + 32 * V - 1) / (32 * V);
  a.wc = warps >= 3 ? 4 : warps;
  a.cblocks = (warps + a.wc - 1) / a.wc;
  const int rows = step ? op->n_seq : op->tokens;
  a.run = step ? 1 : 32;
  a.runs = rows > 0 ? (rows + a.run - 1) / a.run : 1;
  const int per = 4 / a.wc;
  const long long blocks = (long long)a.cblocks * ((a.runs + per - 1) / per);
  if (blocks > 0x7fffffffLL) return -2;
  if (step)
    conv1d_step<T, V, K, ACT><<<(unsigned)blocks, kConvThreads, 0, stream>>>(a);
  else
    conv1d_prompt<T, V, K, ACT><<<(unsigned)blocks, kConvThreads, 0, stream>>>(a);
  cwgk_count_launch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    cwgk_set_cuda_error((int)e);
    return -3;
  }
  return 0;
}

template <typename T, int V, int K>
static int conv1d_act(const cwgk_conv1d *op, bool step, cudaStream_t s) {
  switch (op->act) {
    case CWGK_ACT_SILU: return launch_conv1d<T, V, K, CWGK_ACT_SILU>(op, step, s);
    case CWGK_ACT_RELU: return launch_conv1d<T, V, K, CWGK_ACT_RELU>(op, step, s);
    default: return launch_conv1d<T, V, K, CWGK_ACT_NONE>(op, step, s);
  }
}
template <typename T, int V>
static int conv1d_width(const cwgk_conv1d *op, bool step, cudaStream_t s) {
  switch (op->width) {
    case 2: return conv1d_act<T, V, 2>(op, step, s);
    case 3: return conv1d_act<T, V, 3>(op, step, s);
    default: return conv1d_act<T, V, 4>(op, step, s);
  }
}
template <typename T>
static int conv1d(const cwgk_conv1d *op, bool step, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool one = (step ? op->n_seq : op->tokens) <= 1;  // no second row: ld says nothing
  const bool vec = op->channels % V == 0 && aligned16(op->x) && aligned16(op->y) &&
                   aligned16(op->state) && aligned16(op->w) &&
                   (one || (op->ldx % V == 0 && op->ldy % V == 0));
  return vec ? conv1d_width<T, V>(op, step, s) : conv1d_width<T, 1>(op, step, s);
}

}  // namespace seq
}  // namespace cwg

extern "C" {

int cwgk_conv1d_prompt(const cwgk_conv1d *op, void *stream) {
  return op->bf16 ? cwg::seq::conv1d<__nv_bfloat16>(op, false, (cudaStream_t)stream)
                  : cwg::seq::conv1d<float>(op, false, (cudaStream_t)stream);
}
int cwgk_conv1d_step(const cwgk_conv1d *op, void *stream) {
  return op->bf16 ? cwg::seq::conv1d<__nv_bfloat16>(op, true, (cudaStream_t)stream)
                  : cwg::seq::conv1d<float>(op, true, (cudaStream_t)stream);
}

int cwgk_conv1d_read_clear_status(unsigned *status) {
  return cwg::read_clear_status(cwg::seq::g_seq_status, status);
}

}  // extern "C"
