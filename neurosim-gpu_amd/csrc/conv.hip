// Short causal convolution per channel (gfx950): forward, one tick, backward.
//
// One thread takes V neighbouring channels of one column (16 bytes of a row) and a
// chunk of ticks, and keeps the last W inputs in registers, so every input is read
// once (plus W-1 ticks per chunk) and every output written once: the kernels are
// bound by HBM.  T=4096, B=4, N=4096, W=4 in bf16: 66 us for 268 MB, 4.1 TB/s of the 5.1 a
// large copy reaches.  The last vector of a row starts at N - V: neighbours then compute
// the same outputs twice and store equal values, which needs no tail code.
#include "ns_signal.h"

namespace ns {

struct ConvShape {
  int64_t ticks, batch, channels;
  int64_t vectors, chunks, chunk;   // vectors per row, chunks of `chunk` ticks
  int32_t silu;
};

// A thread's place: channels n0 .., column b, ticks [t0, t0 + chunk).
struct ConvPlace {
  int64_t n0, b, c, t0;
};

template <int V>
__device__ __forceinline__ bool conv_place(const ConvShape& s, ConvPlace& p) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= s.vectors * s.batch * s.chunks) return false;
  const int64_t line = id / s.vectors;
  p.n0 = (id - line * s.vectors) * V;
  if (p.n0 > s.channels - V) p.n0 = s.channels - V;
  p.c = line / s.batch;
  p.b = line - p.c * s.batch;
  p.t0 = p.c * s.chunk;
  return true;
}

// Input row of column b at tick t >= -(W-1): the signal, or the history (absent: zeros).
template <class T, int V, int W>
__device__ __forceinline__ void conv_input(const Signal<T>& x, const Signal<T>& history,
                                           const ConvPlace& p, int64_t t, int64_t end, float* out) {
  if (t >= 0 ? t < end : history.data != nullptr) {
    const Pack<T, V> v =
        load_pack<T, V>((t >= 0 ? x.row(t, p.b) : history.row(t + W - 1, p.b)) + p.n0);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = static_cast<float>(v.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = 0.0f;
  }
}

template <int V, int W>
__device__ __forceinline__ void conv_weights(const float* weight, const float* bias, int64_t n0,
                                             float (&w)[V][W], float (&c)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k < W; ++k) w[i][k] = weight[(n0 + i) * W + k];
    c[i] = bias ? bias[n0 + i] : 0.0f;
  }
}

constexpr int kConvAhead = 4;   // ticks whose rows are requested before any is used

template <class T, int V, int W>
__global__ __launch_bounds__(kThreads) void conv_forward(ConvShape s, Signal<T> x,
                                                         const float* weight, const float* bias,
                                                         Signal<T> history, const int32_t* lengths,
                                                         Signal<T> y, Signal<T> out_history) {
  ConvPlace p;
  if (!conv_place<V>(s, p)) return;
  const int64_t end = column_ticks(lengths, p.b, s.ticks);
  float w[V][W], c[V];
  conv_weights<V, W>(weight, bias, p.n0, w, c);
  float win[W][V];                                  // inputs t-W+1 .. t
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) conv_input<T, V, W>(x, history, p, p.t0 - W + 1 + k, end, win[k]);
  const int64_t stop = p.t0 + s.chunk < s.ticks ? p.t0 + s.chunk : s.ticks;
  for (int64_t t = p.t0; t < stop; t += kConvAhead) {
    float next[kConvAhead][V];
#pragma unroll
    for (int u = 0; u < kConvAhead; ++u) conv_input<T, V, W>(x, history, p, t + u, end, next[u]);
#pragma unroll
    for (int u = 0; u < kConvAhead; ++u) {
      if (t + u < stop) {
        Pack<T, V> out;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          win[W - 1][i] = next[u][i];
          float pre = c[i];
#pragma unroll
          for (int k = 0; k < W; ++k) pre = fmaf(w[i][k], win[k][i], pre);
          const float value = s.silu ? pre * sigmoid(pre) : pre;
          out.v[i] = static_cast<T>(t + u < end ? value : 0.0f);
        }
        store_pack<T, V>(y.row(t + u, p.b) + p.n0, out);
#pragma unroll
        for (int k = 0; k + 1 < W; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
      }
    }
  }
  if (out_history.data && p.c == s.chunks - 1) {    // the column's last W-1 inputs
#pragma unroll
    for (int k = 0; k + 1 < W; ++k) {
      float last[V];
      conv_input<T, V, W>(x, history, p, end - W + 1 + k, end, last);
      Pack<T, V> out;
#pragma unroll
      for (int i = 0; i < V; ++i) out.v[i] = static_cast<T>(last[i]);
      store_pack<T, V>(out_history.row(k, p.b) + p.n0, out);
    }
  }
}

// One tick; a thread owns one (column, channel), so its history can move on in place.  A
// launch is all it takes: 2.2 us at B=1, N=1024.
template <class T, int W>
__global__ __launch_bounds__(kThreads) void conv_step(int64_t batch, int64_t channels, int32_t silu,
                                                      const T* x, int64_t x_sb, const float* weight,
                                                      const float* bias, Signal<T> history, T* y,
                                                      int64_t y_sb) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= batch * channels) return;
  const int64_t b = id / channels, n = id - b * channels;
  float pre = bias ? bias[n] : 0.0f;
  const T now = x[b * x_sb + n];
  T old[W];
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) old[k] = history.row(k, b)[n];
  old[W - 1] = now;
#pragma unroll
  for (int k = 0; k < W; ++k) pre = fmaf(weight[n * W + k], static_cast<float>(old[k]), pre);
  y[b * y_sb + n] = static_cast<T>(silu ? pre * sigmoid(pre) : pre);
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) history.row(k, b)[n] = old[k + 1];
}

// Backward.  With q[t] = dy[t] y'(p[t]) (0 outside the column's ticks),
//   dx[t] = sum_k w[k] q[t + W-1-k],  dw[k] = sum_t q[t] x[t-W+1+k],  dbias = sum_t q[t].
// A thread walks its chunk and W-1 ticks more, recomputing p from the inputs, and gives
// dx of tick t - W+1 when q[t] is known; chunk 0 gives the history's gradient as well.
// Its sums for dw and dbias cover its own ticks; a second launch adds the threads' sums, in
// order.  T=1500, B=7, N=1031, W=3 in float32 (130 MB, in the caches): 24 us, and 5.4 for the
// sums; forward 14.
template <class T, int V, int W>
__global__ __launch_bounds__(kThreads) void conv_backward(ConvShape s, Signal<T> x,
                                                          const float* weight, const float* bias,
                                                          Signal<T> history, const int32_t* lengths,
                                                          Signal<T> dy, Signal<T> dout_history,
                                                          Signal<T> dx, Signal<T> dhistory,
                                                          float* partials) {
  ConvPlace p;
  if (!conv_place<V>(s, p)) return;
  const int64_t end = column_ticks(lengths, p.b, s.ticks);
  float w[V][W], c[V], dw[V][W] = {}, dc[V] = {};
  conv_weights<V, W>(weight, bias, p.n0, w, c);
  float win[W][V], q[W][V] = {};                    // inputs and q of ticks t-W+1 .. t
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) conv_input<T, V, W>(x, history, p, p.t0 - W + 1 + k, end, win[k]);
  const int64_t own = p.t0 + s.chunk < s.ticks ? p.t0 + s.chunk : s.ticks;
  const int64_t from = p.c == 0 ? 1 - W : p.t0;     // first tick whose dx this thread gives
  const int64_t stop = own + W - 1;
  for (int64_t t = p.t0; t < stop; t += kConvAhead) {
    float next[kConvAhead][V], up[kConvAhead][V];
#pragma unroll
    for (int u = 0; u < kConvAhead; ++u) {
      conv_input<T, V, W>(x, history, p, t + u, end, next[u]);
      conv_input<T, V, W>(dy, Signal<T>{}, p, t + u, end, up[u]);
    }
#pragma unroll
    for (int u = 0; u < kConvAhead; ++u) {
      const int64_t now = t + u, back = now - W + 1;
      if (now < stop) {
        float g[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          win[W - 1][i] = next[u][i];
          float slope = 1.0f;
          if (s.silu) {
            float pre = c[i];
#pragma unroll
            for (int k = 0; k < W; ++k) pre = fmaf(w[i][k], win[k][i], pre);
            const float gate = sigmoid(pre);
            slope = gate * (1.0f + pre * (1.0f - gate));
          }
          const float now_q = now < end ? up[u][i] * slope : 0.0f;
          q[W - 1][i] = now_q;
          if (now < own) {
            dc[i] += now_q;
#pragma unroll
            for (int k = 0; k < W; ++k)
              dw[i][k] = now < end ? fmaf(now_q, win[k][i], dw[i][k]) : dw[i][k];
          }
          g[i] = 0.0f;
#pragma unroll
          for (int k = 0; k < W; ++k) g[i] = fmaf(w[i][W - 1 - k], q[k][i], g[i]);
        }
        if (back >= from) {
          // The input of tick `back` is row k of the column's last W-1 inputs.
          const int64_t k = back - (end - W + 1);
          if (dout_history.data && k >= 0 && k < W - 1) {
            const Pack<T, V> more = load_pack<T, V>(dout_history.row(k, p.b) + p.n0);
#pragma unroll
            for (int i = 0; i < V; ++i) g[i] += static_cast<float>(more.v[i]);
          }
          Pack<T, V> out;
#pragma unroll
          for (int i = 0; i < V; ++i) out.v[i] = static_cast<T>(g[i]);
          if (back >= 0) {
            if (dx.data && back < own) store_pack<T, V>(dx.row(back, p.b) + p.n0, out);
          } else if (dhistory.data) {
            store_pack<T, V>(dhistory.row(back + W - 1, p.b) + p.n0, out);
          }
        }
#pragma unroll
        for (int k = 0; k + 1 < W; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            win[k][i] = win[k + 1][i];
            q[k][i] = q[k + 1][i];
          }
      }
    }
  }
  // One part per (chunk, column): [N][W], then [N].
  float* part = partials + (p.c * s.batch + p.b) * s.channels * (W + 1);
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k < W; ++k) part[(p.n0 + i) * W + k] = dw[i][k];
    part[s.channels * W + p.n0 + i] = dc[i];
  }
}

// out[m] = sum over parts, 64 neighbouring m per workgroup, its wavefronts taking every
// kWaves-th part and adding up through LDS, in order.
template <int kWaves>
__global__ __launch_bounds__(64 * kWaves) void add_parts(const float* __restrict__ partials,
                                                         int64_t parts, int64_t m_total,
                                                         float* __restrict__ out) {
  __shared__ float sums[kWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float sum = 0.0f;
  if (m < m_total) {
    float four[4] = {};
    int64_t p = wave;
    for (; p + 3 * kWaves < parts; p += 4 * kWaves)
#pragma unroll
      for (int u = 0; u < 4; ++u) four[u] += partials[(p + kWaves * u) * m_total + m];
    for (; p < parts; p += kWaves) four[0] += partials[p * m_total + m];
    sum = (four[0] + four[1]) + (four[2] + four[3]);
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && m < m_total) {
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w += 4)
      total += (sums[w][lane] + sums[w + 1][lane]) + (sums[w + 2][lane] + sums[w + 3][lane]);
    out[m] = total;
  }
}

// Many parts go to sixteen wavefronts: 658 parts of 4124 sums take 13.2 us with four, 5.4 with
// sixteen.  Few leave them nothing to do: 8 parts of 73,728 sums take 4.7 with four.
int sum_partials(const float* partials, int64_t parts, int64_t m_total, float* out, void* stream) {
  if (m_total <= 0) return NS_OK;
  const dim3 grid(static_cast<unsigned>((m_total + 63) / 64));
  auto queue = static_cast<hipStream_t>(stream);
  if (parts >= 64)
    add_parts<16><<<grid, dim3(64 * 16), 0, queue>>>(partials, parts, m_total, out);
  else
    add_parts<4><<<grid, dim3(64 * 4), 0, queue>>>(partials, parts, m_total, out);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch("partial sums", err);
}

namespace {

int64_t type_bytes(int32_t type) { return type == NS_TYPE_F32 ? 4 : 2; }

int64_t vector_width(int64_t channels, int32_t type) {
  const int64_t wide = 16 / type_bytes(type);
  return channels >= wide ? wide : 1;
}

int check_conv(const ns_conv_args* a) {
  if (!a) return fail("convolution arguments are required");
  if (a->ticks < 0 || a->batch < 0 || a->channels <= 0)
    return fail("a signal is [T, B, N] with N > 0");
  if (a->taps < 1 || a->taps > NS_CONV_MAX_TAPS)
    return fail("a convolution has 1 to %d taps", NS_CONV_MAX_TAPS);
  if (a->type != NS_TYPE_F32 && a->type != NS_TYPE_BF16 && a->type != NS_TYPE_F16)
    return fail("unknown element type");
  if (a->chunk < 0) return fail("ticks per thread must not be negative");
  if (!a->weight) return fail("the convolution's weights are required");
  if (a->batch && a->ticks && !a->x.data) return fail("the input signal is required");
  return NS_OK;
}

int64_t chunk_of(const ns_conv_args* a, bool backward) {
  return a->chunk > 0 ? a->chunk
                      : ns_conv_chunk(a->ticks, a->batch, a->channels, a->type, backward);
}

ConvShape shape_of(const ns_conv_args* a, bool backward) {
  ConvShape s{};
  s.ticks = a->ticks;
  s.batch = a->batch;
  s.channels = a->channels;
  const int64_t v = vector_width(a->channels, a->type);
  s.vectors = (a->channels + v - 1) / v;
  s.chunk = chunk_of(a, backward);
  s.chunks = a->ticks > 0 ? (a->ticks + s.chunk - 1) / s.chunk : 1;
  s.silu = a->silu;
  return s;
}

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

int grid_of(int64_t threads, dim3* grid) {
  const int64_t groups = (threads + kThreads - 1) / kThreads;
  if (groups > INT32_MAX) return fail("the signal is too large for one launch");
  *grid = dim3(static_cast<unsigned>(groups));
  return NS_OK;
}

template <class T, int V, int W>
int run_forward(const ns_conv_args* a, hipStream_t stream) {
  const ConvShape s = shape_of(a, false);
  dim3 grid;
  if (int rc = grid_of(s.vectors * s.batch * s.chunks, &grid)) return rc;
  conv_forward<T, V, W><<<grid, dim3(kThreads), 0, stream>>>(
      s, signal<T>(a->x), a->weight, a->bias, signal<T>(a->history), a->lengths, signal<T>(a->y),
      signal<T>(a->out_history));
  return launched("convolution");
}

template <class T, int V, int W>
int run_backward(const ns_conv_args* a, hipStream_t stream) {
  const ConvShape s = shape_of(a, true);
  dim3 grid;
  if (int rc = grid_of(s.vectors * s.batch * s.chunks, &grid)) return rc;
  conv_backward<T, V, W><<<grid, dim3(kThreads), 0, stream>>>(
      s, signal<T>(a->x), a->weight, a->bias, signal<T>(a->history), a->lengths,
      signal<T>(a->dy), signal<T>(a->dout_history), signal<T>(a->dx), signal<T>(a->dhistory),
      a->partials);
  if (int rc = launched("convolution backward")) return rc;
  return sum_partials(a->partials, s.chunks * s.batch, s.channels * (W + 1), a->dweight, stream);
}

template <class T, int W>
int run_step(const ns_conv_args* a, hipStream_t stream) {
  dim3 grid;
  if (int rc = grid_of(a->batch * a->channels, &grid)) return rc;
  conv_step<T, W><<<grid, dim3(kThreads), 0, stream>>>(
      a->batch, a->channels, a->silu, static_cast<const T*>(a->x.data), a->x.stride_b, a->weight,
      a->bias, signal<T>(a->history), static_cast<T*>(a->y.data), a->y.stride_b);
  return launched("convolution step");
}

enum class ConvPass { kForward, kStep, kBackward };

template <class T, int W>
int run_taps(const ns_conv_args* a, ConvPass pass, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  if (pass == ConvPass::kStep) return run_step<T, W>(a, stream);
  if (vector_width(a->channels, a->type) == V)
    return pass == ConvPass::kForward ? run_forward<T, V, W>(a, stream)
                                      : run_backward<T, V, W>(a, stream);
  return pass == ConvPass::kForward ? run_forward<T, 1, W>(a, stream)
                                    : run_backward<T, 1, W>(a, stream);
}

template <class T>
int run_type(const ns_conv_args* a, ConvPass pass, hipStream_t stream) {
  switch (a->taps) {
    case 1: return run_taps<T, 1>(a, pass, stream);
    case 2: return run_taps<T, 2>(a, pass, stream);
    case 3: return run_taps<T, 3>(a, pass, stream);
    case 4: return run_taps<T, 4>(a, pass, stream);
    case 5: return run_taps<T, 5>(a, pass, stream);
    case 6: return run_taps<T, 6>(a, pass, stream);
    case 7: return run_taps<T, 7>(a, pass, stream);
    default: return run_taps<T, 8>(a, pass, stream);
  }
}

int run(const ns_conv_args* a, ConvPass pass, void* stream) {
  auto queue = static_cast<hipStream_t>(stream);
  if (a->type == NS_TYPE_F32) return run_type<float>(a, pass, queue);
  if (a->type == NS_TYPE_BF16) return run_type<__bf16>(a, pass, queue);
  return run_type<_Float16>(a, pass, queue);
}

}  // namespace
}  // namespace ns

extern "C" {

int64_t ns_conv_chunk(int64_t ticks, int64_t batch, int64_t channels, int32_t type,
                      int32_t backward) {
  const int64_t lanes = (channels + ns::vector_width(channels, type) - 1) /
                        ns::vector_width(channels, type) * (batch > 0 ? batch : 1);
  // Three workgroups per compute unit: all of them run at once, in chunks long enough that
  // the weights and the W-1 ticks read again cost little.  T=4096, B=4, N=4096 in bf16 takes
  // 107 us in chunks of 8, 92 of 16, 82 of 28, 71 of 44, 82 of 64, 124 of 128; T=1500, B=7,
  // N=1031 in float32 17.6 of 16, 17 of 24, 24.5 of 64.
  const int64_t most = backward ? 128 : 64, least = backward ? 16 : 4;
  int64_t chunk = ticks * lanes / (3 * 256 * ns::kThreads);
  chunk = (chunk + 3) / 4 * 4;
  return chunk < least ? least : (chunk > most ? most : chunk);
}

int64_t ns_conv_backward_floats(int64_t ticks, int64_t batch, int64_t channels, int32_t taps,
                                int32_t type) {
  if (ticks <= 0 || batch <= 0 || channels <= 0) return batch > 0 ? batch * channels * (taps + 1) : 0;
  const int64_t chunk = ns_conv_chunk(ticks, batch, channels, type, 1);
  return (ticks + chunk - 1) / chunk * batch * channels * (taps + 1);
}

int ns_conv_forward(const ns_conv_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_conv(a)) return rc;
  if (a->batch == 0) return NS_OK;
  if (a->ticks && !a->y.data) return ns::fail("the output signal is required");
  return ns::run(a, ns::ConvPass::kForward, stream);
}

int ns_conv_step(const ns_conv_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_conv(a)) return rc;
  if (a->ticks != 1 || a->lengths) return ns::fail("a step is one tick of every column");
  if (a->batch == 0) return NS_OK;
  if (!a->y.data) return ns::fail("the output signal is required");
  if (a->taps > 1 && (!a->history.data || a->out_history.data != a->history.data))
    return ns::fail("a step moves its history on in place");
  return ns::run(a, ns::ConvPass::kStep, stream);
}

int ns_conv_backward(const ns_conv_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_conv(a)) return rc;
  if (!a->dweight) return ns::fail("the weight gradient is required");
  if (a->batch && (!a->partials || (a->ticks && !a->dy.data)))
    return ns::fail("the backward needs a workspace and the gradient of y");
  if (a->batch == 0)
    return ns::sum_partials(a->partials, 0, a->channels * (a->taps + 1), a->dweight, stream);
  return ns::run(a, ns::ConvPass::kBackward, stream);
}

}  // extern "C"
