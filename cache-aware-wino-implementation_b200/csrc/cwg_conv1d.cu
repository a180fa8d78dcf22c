// cwg_conv1d.cu -- short causal convolution over time, one filter per channel
// (cwg_conv1d_causal, cwg_conv1d_causal_step).
//
//   y[t][c] = act(bias[c] + sum_{j < K} w[c][j] x[t - K + 1 + j][c]),  K = 2 .. 4
//
// 2K flops and one exponential per element against 4 bytes (bf16) or 8 (fp32) in
// and out: bound by memory.
//
// Prompts: a thread owns four channels and a run of consecutive
// rows, so that a row is read once (plus K - 1 rows of halo per run) and the
// window slides through registers while the next eight rows are loaded.
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
constexpr int kAhead = 8;          // rows per step; the next step's are loaded meanwhile
constexpr int kStartsInSmem = 1024;

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

// V channels as pairs (one channel: the second half of its pair is idle).
template <int V>
struct Chan {
  static constexpr int N = (V + 1) / 2;
  F2 p[N];
  __device__ __forceinline__ void set(const float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = f2(f[2 * i], V > 1 ? f[(2 * i + 1) % V] : 0.f);
  }
  __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float2 h = halves(p[i]);
      f[2 * i] = h.x;
      if (V > 1) f[(2 * i + 1) % V] = h.y;
    }
  }
  template <typename R>
  __device__ __forceinline__ void from(R raw) {
    float f[V];
    unpack(raw, f);
    set(f);
  }
};

template <int V, int K>
__device__ __forceinline__ void load_weights(const ConvArgs &a, int c, bool active,
                                             Chan<V> (&w)[K], Chan<V> &b) {
  float f[K][V], g[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    g[v] = active && a.bias ? a.bias[c + v] : 0.f;
    if (V > 1 && K == 4) {  // 16-byte aligned: the host checked w for the vector path
      const float4 q = active ? *reinterpret_cast<const float4 *>(a.w + (size_t)(c + v) * K)
                              : make_float4(0, 0, 0, 0);
      f[0][v] = q.x;
      f[1][v] = q.y;
      f[K > 2 ? 2 : 0][v] = q.z;
      f[K - 1][v] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j) f[j][v] = active ? a.w[(size_t)(c + v) * K + j] : 0.f;
    }
  }
  b.set(g);
#pragma unroll
  for (int j = 0; j < K; ++j) w[j].set(f[j]);
}

// act(b + sum_j w[j] h[j]) with h the window's rows, oldest first, x the newest.
template <typename T, int V, int K, int ACT>
__device__ __forceinline__ typename Raw<T, V>::type window_row(const Chan<V> (&w)[K],
                                                               const Chan<V> &b,
                                                               const Chan<V> (&h)[K - 1],
                                                               const Chan<V> &x) {
  Chan<V> s = b;
#pragma unroll
  for (int i = 0; i < Chan<V>::N; ++i) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) s.p[i] = fma2(w[j].p[i], h[j].p[i], s.p[i]);
    s.p[i] = fma2(w[K - 1].p[i], x.p[i], s.p[i]);
    if (ACT == CWGK_ACT_SILU && sizeof(T) == 2) s.p[i] = silu_bf16x2(s.p[i]);
  }
  float y[V];
  s.get(y);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (ACT == CWGK_ACT_RELU && y[v] < 0.f) y[v] = 0.f;  // NaN stays
    if (ACT == CWGK_ACT_SILU && sizeof(T) == 4) y[v] = silu<float>(y[v]);
  }
  return pack<T, V>(y);
}
template <int V, int K>
__device__ __forceinline__ void slide(Chan<V> (&h)[K - 1], const Chan<V> &x) {
#pragma unroll
  for (int j = 0; j < K - 2; ++j) h[j] = h[j + 1];
  h[K - 2] = x;
}

template <typename T, int V, int K, int ACT>
__global__ void __launch_bounds__(kConvThreads) conv1d_prompt(const ConvArgs a) {
  __shared__ int s_starts[kStartsInSmem + 1];
  griddep_wait();
  griddep_launch_dependents();
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

  Chan<V> w[K], b, h[K - 1];
  load_weights<V, K>(a, c, active, w, b);

  // The run's first rows, and those before it, are on their way while the sequences that begin
  // in it are looked at.
  const T *px = x + (size_t)t0 * a.ldx + c;  // of row t
  T *py = y + (size_t)t0 * a.ldy + c;
  typename Raw<T, V>::type raw[kAhead], next[kAhead];
  auto fetch = [&](const T *from, int left) {  // kAhead rows, of which `left` are the run's
    if (left >= kAhead) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) next[i] = load_raw<T, V>(from + i * a.ldx);
    } else {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        next[i] = i < left ? load_raw<T, V>(from + i * a.ldx) : zero_raw<T, V>();
    }
  };
  fetch(px, active ? t1 - t0 : 0);
  typename Raw<T, V>::type before[K - 1];
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const int t = t0 - (K - 1) + j;
    before[j] = active && t >= 0 && t < a.tokens ? load_raw<T, V>(x + (size_t)t * a.ldx + c)
                                                 : zero_raw<T, V>();
  }

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
    const int len = end - begin;
    typename Raw<T, V>::type xs[K - 1];
#pragma unroll
    for (int i = 0; i < K - 1; ++i)
      xs[i] = active && i < len ? load_raw<T, V>(x + (size_t)(begin + i) * a.ldx + c)
                                : zero_raw<T, V>();
    const unsigned char resume = a.resume ? a.resume[s] : 0;
    const int slot = state ? line_of(a.slots, s, a.n_slots, bad) : -1;
    const bool carry = slot >= 0 && resume;
    if (!active) continue;
    T *line = state + ((size_t)(slot < 0 ? 0 : slot) * (K - 1)) * a.channels + c;
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
      h[j].from(carry ? load_raw<T, V>(line + (size_t)j * a.channels) : zero_raw<T, V>());
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      if (i < len) {
        Chan<V> xv;
        xv.from(xs[i]);
        store_raw<T, V>(y + (size_t)(begin + i) * a.ldy + c,
                        window_row<T, V, K, ACT>(w, b, h, xv));
        slide<V, K>(h, xv);
      }
    }
    if (slot >= 0) {
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        float f[V];
        h[j].get(f);
        store_raw<T, V>(line + (size_t)j * a.channels,
                        len >= K - 1 ? load_raw<T, V>(x + (size_t)(end - (K - 1) + j) * a.ldx + c)
                                     : pack<T, V>(f));
      }
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
  for (int j = 0; j < K - 1; ++j) h[j].from(before[j]);
  for (int t = t0; t < t1; t += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) raw[i] = next[i];
    px += kAhead * a.ldx;
    fetch(px, t1 - t - kAhead);
    if (t - begin >= K - 1 && t + kAhead <= end && t + kAhead <= t1) {
      // all of one sequence, as nearly always
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        Chan<V> xv;
        xv.from(raw[i]);
        store_raw<T, V>(py + i * a.ldy, window_row<T, V, K, ACT>(w, b, h, xv));
        slide<V, K>(h, xv);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (t + i < t1) {
          while (s + 1 < a.n_seq && starts[s + 1] <= t + i) {
            ++s;
            begin = starts[s];
            end = starts[s + 1];
            if (begin < 0 || end > a.tokens) end = begin = 0;
          }
          Chan<V> xv;
          xv.from(raw[i]);
          if (t + i < end && t + i - begin >= K - 1)
            store_raw<T, V>(py + i * a.ldy, window_row<T, V, K, ACT>(w, b, h, xv));
          slide<V, K>(h, xv);
        }
      }
    }
    py += kAhead * a.ldy;
  }
}

// One token of each sequence: a thread owns a vector of channels of one row; K vectors
// in (x and the line) and K out (y and the line moved by one).  The loads are issued
// before the search for an earlier row with the same line.
template <typename T, int V, int K, int ACT>
__global__ void __launch_bounds__(kConvThreads) conv1d_step(const ConvArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const T *x = static_cast<const T *>(a.x);
  T *y = static_cast<T *>(a.y);
  T *state = static_cast<T *>(a.state);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cb = blockIdx.x % a.cblocks;
  const int r = (blockIdx.x / a.cblocks) * (4 / a.wc) + warp / a.wc;
  if (r >= a.runs) return;
  const int c = ((cb * a.wc + warp % a.wc) * 32 + lane) * V;
  const bool active = c < a.channels;
  int slot = a.slots ? a.slots[r] : r;
  bool bad = slot >= a.n_slots;
  if (bad) slot = -1;
  T *line = state + ((size_t)(slot < 0 ? 0 : slot) * (K - 1)) * a.channels + c;
  typename Raw<T, V>::type raw[K];
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
    raw[j] = slot >= 0 && active ? load_raw<T, V>(line + (size_t)j * a.channels)
                                 : zero_raw<T, V>();
  raw[K - 1] = active ? load_raw<T, V>(x + (size_t)r * a.ldx + c) : zero_raw<T, V>();
  Chan<V> w[K], b, h[K - 1], xv;
  load_weights<V, K>(a, c, active, w, b);
  if (slot >= 0 && a.slots && taken_before(a.slots, r, slot)) {
    slot = -1;
    bad = true;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) raw[j] = zero_raw<T, V>();
  }
  if (bad && lane == 0 && c == 0) atomicOr(&g_seq_status, CWGK_STATUS_INDEX);
  if (!active) return;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) h[j].from(raw[j]);
  xv.from(raw[K - 1]);
  store_raw<T, V>(y + (size_t)r * a.ldy + c, window_row<T, V, K, ACT>(w, b, h, xv));
  if (slot >= 0) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
      store_raw<T, V>(line + (size_t)j * a.channels, raw[j + 1]);
  }
}

static bool aligned(const void *p, size_t n) { return (uintptr_t)p % n == 0; }

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
  const int rows = step ? op->n_seq : op->tokens;
  a.wc = warps >= 3 ? 4 : warps;
  a.cblocks = (warps + a.wc - 1) / a.wc;
  // Long runs share the weights and the first rows' halo; the run is halved until every SM
  // has 16 warps (16384 x 4096 bf16: 58 us with 128 or 64 rows, 61 with 32; 1237 x 1001
  // fp32: 17, 11.5, 9.3 us with 128, 64, 32).
  a.run = step ? 1 : 128;
  while (!step && a.run > kAhead && (long long)warps * ((rows + a.run - 1) / a.run) < 148 * 16)
    a.run /= 2;
  a.runs = rows > 0 ? (rows + a.run - 1) / a.run : 1;
  const int per = 4 / a.wc;
  const long long blocks = (long long)a.cblocks * ((a.runs + per - 1) / per);
  if (blocks > 0x7fffffffLL) return -2;
  const auto kernel = step ? conv1d_step<T, V, K, ACT> : conv1d_prompt<T, V, K, ACT>;
  const cudaError_t e = launch_dependent(kernel, dim3((unsigned)blocks), kConvThreads, 0, stream,
                                         op->pdl, 1, a);
  cwgk_count_launch();
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
  constexpr int V = 4;  // 8 or 16 bytes: with 8 bf16 channels a thread needs 128 registers
  const bool one = (step ? op->n_seq : op->tokens) <= 1;  // no second row: ld says nothing
  constexpr size_t B = V * sizeof(T);
  const bool vec = op->channels % V == 0 && aligned(op->x, B) && aligned(op->y, B) &&
                   aligned(op->state, B) && aligned(op->w, 16) &&
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
