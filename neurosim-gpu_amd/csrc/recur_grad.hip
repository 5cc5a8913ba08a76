// Backward of the gated linear recurrence (gfx950).
//
// With gy = dy silu(z), g the adjoint of h, and the names of ns_recur.h:
//   g[t] = gy[t] + a[t+1] g[t+1]
//   dx = g m i,  dwrite = g m i x (1 - i),  dz = dy h silu'(z),  dstate = a[0] g[0]
//   k = g (a^2/m i x - a h[t-1])  (the derivative by u: da = -a du, dm = a^2/m du)
//   dforget = k u (1 - s),  drates = sum of k s
// The states are walked again from those kept at each tile's start; the adjoint's stretch of
// ticks has the same decay as the state's, so both meet in LDS at once: one barrier a tile.
// At u = 0 the term a^2/m, which grows without bound there, is left out.  A rate below zero counts
// as zero, and its gradient is zero.
//
// Bound as the forward is: 2048 ticks of 8 x 4096 in bf16 with a gate (1208 MB) 316 us in passes back to
// back (the average of 40; 385 in the first ones), 3.8 TB/s, the vector ALU 77% busy.
#include "ns_recur.h"

namespace ns {
namespace {

constexpr int kWaves = 8, kRun = kRecurTile / kWaves;
constexpr int kGradThreads = 64 * kWaves;

template <class T, int V>
struct GradRaw {
  Pack<T, V> x[kRun], forget[kRun], write[kRun], z[kRun], dy[kRun];
};

template <class T, int V, bool kGate>
__device__ __forceinline__ void request(const RecurIn<T>& in, const Signal<T>& dy, const RecurPlace& p,
                                        int t, GradRaw<T, V>& raw) {
  load_run<T, V>(in.x, p, t, raw.x);
  load_run<T, V>(in.forget, p, t, raw.forget);
  load_run<T, V>(in.write, p, t, raw.write);
  load_run<T, V>(dy, p, t, raw.dy);
  if (kGate) load_run<T, V>(in.z, p, t, raw.z);
}

template <class T>
struct RecurGrads {
  Signal<T> dx, dforget, dwrite, dz;
};

template <int V>
struct TwoWays {
  float decay[V], state[V], adjoint[V];
};

// Chunks' stretches of the adjoint: g before the chunk = decay g behind it + add.  The
// wavefronts take runs of ticks from the chunk's start to its end.
template <class T, int V, bool kGate>
__global__ __launch_bounds__(kGradThreads) void adjoint_ends(RecurShape s, RecurIn<T> in, Signal<T> dy,
                                                             float* ends) {
  __shared__ TwoWays<V> meet[kWaves][64];
  const RecurPlace p = recur_place<V>(s, in.lengths);
  const int wave = uniform(threadIdx.x >> 6);
  float rate[V];
  load_floats<V>(in.rates, p, rate);
  TwoWays<V> own;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    rate[j] = fade_rate(rate[j]);
    own.decay[j] = 1.0f;
    own.adjoint[j] = 0.0f;
  }
  const int run = static_cast<int>(s.chunk) / kWaves;
  const int from = p.t0 + wave * run, stop = from + run < p.end ? from + run : p.end;
  Pack<T, V> forget[kRun], z[kRun], up[kRun];
  const auto ask = [&](int t) __attribute__((always_inline)) {
    load_run<T, V>(in.forget, p, t, forget);
    load_run<T, V>(dy, p, t, up);
    if (kGate) load_run<T, V>(in.z, p, t, z);
  };
  if (from < stop) ask(from);
  for (int t = from; t < stop; t += kRun) {
    float decay[kRun][V], add[kRun][V];
#pragma unroll
    for (int k = 0; k < kRun; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float u = rate[j] * sigmoid(static_cast<float>(forget[k].v[j]));
        const float gated = kGate ? static_cast<float>(z[k].v[j]) : 0.0f;
        const float gy = static_cast<float>(up[k].v[j]) * (kGate ? gated * sigmoid(gated) : 1.0f);
        decay[k][j] = t + k < stop ? __builtin_amdgcn_exp2f(-kLog2e * u) : 1.0f;
        add[k][j] = t + k < stop ? gy : 0.0f;
      }
    ask(t + kRun);
    // own: what a unit behind the run, and the run's own gy, bring before it.
#pragma unroll
    for (int k = 0; k < kRun; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        own.decay[j] *= decay[k][j];
        own.adjoint[j] = fmaf(own.decay[j], add[k][j], own.adjoint[j]);
      }
  }
  meet[wave][threadIdx.x & 63] = own;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    const TwoWays<V> other = meet[w][threadIdx.x];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      own.adjoint[j] = fmaf(own.decay[j], other.adjoint[j], own.adjoint[j]);
      own.decay[j] *= other.decay[j];
    }
  }
  float* row = ends + p.c * 2 * (s.batch * s.channels) + p.b * s.channels;
  store_floats<V>(row, p, own.decay);
  store_floats<V>(row + s.batch * s.channels, p, own.adjoint);
}

// The adjoint that arrives from behind chunk c: the later chunks' stretches, composed by the
// wavefronts in runs.
template <int V>
__device__ __forceinline__ void chunk_behind(const RecurShape& s, const RecurPlace& p,
                                             const float* ends, int wave, TwoWays<V> (*meet)[64],
                                             float (&g)[V]) {
  const int first = static_cast<int>(p.c) + 1, later = static_cast<int>(s.chunks) - first;
  const int per = (later + kWaves - 1) / kWaves;
  const int from = wave * per < later ? wave * per : later;
  const int stop = from + per < later ? from + per : later;
  const int64_t lines = s.batch * s.channels;
  TwoWays<V> own;
#pragma unroll
  for (int j = 0; j < V; ++j) own.decay[j] = 1.0f, own.adjoint[j] = 0.0f;
#pragma unroll 4
  for (int c = from; c < stop; ++c) {
    const float* row = ends + (first + c) * 2 * lines + p.b * s.channels;
    float decay[V], add[V];
    load_floats<V>(row, p, decay);
    load_floats<V>(row + lines, p, add);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      own.adjoint[j] = fmaf(own.decay[j], add[j], own.adjoint[j]);
      own.decay[j] *= decay[j];
    }
  }
  meet[wave][threadIdx.x & 63] = own;
  __syncthreads();
  for (int w = kWaves - 1; w >= 0; --w) {
    const TwoWays<V> other = meet[w][threadIdx.x & 63];
#pragma unroll
    for (int j = 0; j < V; ++j) g[j] = fmaf(other.decay[j], g[j], other.adjoint[j]);
  }
  __syncthreads();
}

template <class T, int V, bool kGate>
__global__ __launch_bounds__(kGradThreads) void recur_backward(RecurShape s, RecurIn<T> in,
                                                               Signal<T> dy, const float* dout_state,
                                                               const float* checkpoints,
                                                               const float* ends, RecurGrads<T> to,
                                                               float* dstate, float* partials) {
  __shared__ TwoWays<V> meet[2][kWaves][64];
  const RecurPlace p = recur_place<V>(s, in.lengths);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t row = p.b * s.channels, lines = s.batch * s.channels;
  float rate[V], g[V] = {}, sum[V] = {};
  load_floats<V>(in.rates, p, rate);
#pragma unroll
  for (int j = 0; j < V; ++j) rate[j] = fade_rate(rate[j]);
  if (dout_state) load_floats<V>(dout_state + row, p, g);
  const int last = p.t0 + (p.t1 - p.t0 - 1) / kRecurTile * kRecurTile;
  GradRaw<T, V> raw;
  float kept[V] = {};
  if (last < p.end) {
    request<T, V, kGate>(in, dy, p, last + wave * kRun, raw);
    load_floats<V>(checkpoints + last / kRecurTile * lines + row, p, kept);
  }
  if (p.c + 1 < s.chunks) chunk_behind<V>(s, p, ends, wave, meet[0], g);
  int turn = 0;
  for (int t = last; t >= p.t0; t -= kRecurTile) {
    const int own = t + wave * kRun;
    if (t >= p.end) {
#pragma unroll
      for (int k = 0; k < kRun; ++k) {
        const float zero[V] = {};
        if (own + k < p.t1) {
          store_tick<T, V>(to.dx, p, own + k, zero);
          store_tick<T, V>(to.dforget, p, own + k, zero);
          store_tick<T, V>(to.dwrite, p, own + k, zero);
          if (kGate) store_tick<T, V>(to.dz, p, own + k, zero);
        }
      }
      // The next tile may be the first with ticks of the column.
      if (t - kRecurTile >= p.t0 && t - kRecurTile < p.end) {
        request<T, V, kGate>(in, dy, p, own - kRecurTile, raw);
        load_floats<V>(checkpoints + (t / kRecurTile - 1) * lines + row, p, kept);
      }
      continue;
    }
    // Per tick: the decay, m, x, both gates and what is off of them, and gy; dy and z as read.
    float decay[kRun][V], room[kRun][V], x[kRun][V], gy[kRun][V];
    Sigmoid forget[kRun][V], write[kRun][V];
    Pack<T, V> up[kRun], gate[kRun];
    TwoWays<V> mine;
#pragma unroll
    for (int j = 0; j < V; ++j) mine.decay[j] = 1.0f, mine.state[j] = mine.adjoint[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      up[k] = raw.dy[k];
      if (kGate) gate[k] = raw.z[k];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool live = own + k < p.end;
        forget[k][j] = both_sigmoids(static_cast<float>(raw.forget[k].v[j]));
        write[k][j] = both_sigmoids(static_cast<float>(raw.write[k].v[j]));
        const float u = rate[j] * forget[k][j].on, a = __builtin_amdgcn_exp2f(-kLog2e * u);
        room[k][j] = __builtin_amdgcn_sqrtf(room_squared(u, a));
        x[k][j] = static_cast<float>(raw.x[k].v[j]);
        const float z = kGate ? static_cast<float>(gate[k].v[j]) : 0.0f;
        const float passed = static_cast<float>(up[k].v[j]) * (kGate ? z * sigmoid(z) : 1.0f);
        decay[k][j] = live ? a : 1.0f;
        gy[k][j] = live ? passed : 0.0f;
        const float add = live ? room[k][j] * write[k][j].on * x[k][j] : 0.0f;
        mine.state[j] = fmaf(decay[k][j], mine.state[j], add);
        mine.decay[j] *= decay[k][j];
        mine.adjoint[j] = fmaf(mine.decay[j], gy[k][j], mine.adjoint[j]);
      }
    }
    float h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = kept[j];
    if (t - kRecurTile >= p.t0) {
      request<T, V, kGate>(in, dy, p, own - kRecurTile, raw);
      load_floats<V>(checkpoints + (t / kRecurTile - 1) * lines + row, p, kept);
    }
    meet[turn][wave][lane] = mine;
    __syncthreads();
    float behind[V];
#pragma unroll 4
    for (int w = kWaves - 1; w >= 0; --w) {
      const TwoWays<V> other = meet[turn][w][lane];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (w == wave) behind[j] = g[j];
        g[j] = fmaf(other.decay[j], g[j], other.adjoint[j]);
      }
    }
    for (int w = 0; w < wave; ++w) {
      const TwoWays<V> other = meet[turn][w][lane];
#pragma unroll
      for (int j = 0; j < V; ++j) h[j] = fmaf(other.decay[j], h[j], other.state[j]);
    }
    turn ^= 1;
    float before[kRun][V];
#pragma unroll
    for (int k = 0; k < kRun; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        before[k][j] = h[j];
        const float add = own + k < p.end ? room[k][j] * write[k][j].on * x[k][j] : 0.0f;
        h[j] = fmaf(decay[k][j], h[j], add);
      }
#pragma unroll
    for (int k = kRun - 1; k >= 0; --k) {
      const bool live = own + k < p.end;
      float dx[V], dforget[V], dwrite[V], dz[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float a = decay[k][j], at = gy[k][j] + behind[j];     // the adjoint of h[t]
        behind[j] = a * at;
        const float input = write[k][j].on * x[k][j];
        const float slope = room[k][j] > 0.0f ? a * a * __builtin_amdgcn_rcpf(room[k][j]) : 0.0f;
        const float by_u = at * (slope * input - a * before[k][j]);
        const float open = at * room[k][j] * write[k][j].on;
        dx[j] = live ? open : 0.0f;
        dwrite[j] = live ? open * x[k][j] * write[k][j].off : 0.0f;
        dforget[j] = live ? by_u * (rate[j] * forget[k][j].on) * forget[k][j].off : 0.0f;
        sum[j] += live ? by_u * forget[k][j].on : 0.0f;
        if (kGate) {
          const float z = static_cast<float>(gate[k].v[j]);
          const Sigmoid both = both_sigmoids(z);
          const float after = fmaf(a, before[k][j], room[k][j] * input);
          dz[j] = live ? static_cast<float>(up[k].v[j]) * after * (both.on * fmaf(z, both.off, 1.0f))
                       : 0.0f;
        }
      }
      if (own + k < p.t1) {
        store_tick<T, V>(to.dx, p, own + k, dx);
        store_tick<T, V>(to.dforget, p, own + k, dforget);
        store_tick<T, V>(to.dwrite, p, own + k, dwrite);
        if (kGate) store_tick<T, V>(to.dz, p, own + k, dz);
      }
    }
  }
  if (p.c == 0 && wave == 0 && dstate) store_floats<V>(dstate + row, p, g);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) meet[0][wave][lane].decay[j] = sum[j];
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w)
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] += meet[0][w][lane].decay[j];
  // What is computed with a rate below zero does not depend on it.
  load_floats<V>(in.rates, p, rate);
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = rate[j] < 0.0f ? 0.0f : sum[j];
  store_floats<V>(partials + p.c * lines + row, p, sum);
}

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

template <class T, int V, bool kGate>
int run_backward(const ns_recurrence_args* a, hipStream_t stream) {
  const RecurShape s = recur_shape(a, V);
  dim3 grid;
  if (int rc = recur_grid(s, &grid)) return rc;
  const RecurIn<T> in = recur_in<T>(a);
  const Signal<T> dy = signal<T>(a->dy);
  if (s.chunks > 1) {
    adjoint_ends<T, V, kGate><<<grid, dim3(kGradThreads), 0, stream>>>(s, in, dy, a->ends);
    if (int rc = launched("recurrence chunks")) return rc;
  }
  const RecurGrads<T> to{signal<T>(a->dx), signal<T>(a->dforget), signal<T>(a->dwrite),
                         signal<T>(a->dz)};
  recur_backward<T, V, kGate><<<grid, dim3(kGradThreads), 0, stream>>>(
      s, in, dy, a->dout_state, a->checkpoints, a->ends, to, a->dstate, a->partials);
  if (int rc = launched("recurrence backward")) return rc;
  return sum_partials(a->partials, s.chunks * s.batch, s.channels, a->drates, stream);
}

// One channel a lane: two of them do not fit the 128 registers that leave a compute unit two
// workgroups (2048 x 8 x 4096 in bf16 with its forward, on 16 wavefronts, 1632 us against 495).
template <class T>
int run(const ns_recurrence_args* a, hipStream_t stream) {
  return a->z.data ? run_backward<T, 1, true>(a, stream) : run_backward<T, 1, false>(a, stream);
}

}  // namespace
}  // namespace ns

extern "C" int ns_recurrence_backward(const ns_recurrence_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_recurrence(a)) return rc;
  if (a->batch == 0 || a->ticks == 0) return ns::fail("a backward has at least one tick and column");
  if (!a->checkpoints) return ns::fail("a backward needs the forward's states");
  if (!a->dy.data || !a->dx.data || !a->dforget.data || !a->dwrite.data || !a->drates || !a->partials)
    return ns::fail("dy, the gradients and the workspace are required");
  if (!a->z.data != !a->dz.data) return ns::fail("dz is given exactly where z is");
  if (ns::recur_shape(a, 1).chunks > 1 && !a->ends)
    return ns::fail("a chunked recurrence needs its workspace");
  auto queue = static_cast<hipStream_t>(stream);
  if (a->type == NS_TYPE_F32) return ns::run<float>(a, queue);
  if (a->type == NS_TYPE_BF16) return ns::run<__bf16>(a, queue);
  return ns::run<_Float16>(a, queue);
}
