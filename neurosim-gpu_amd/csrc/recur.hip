// Gated linear recurrence (gfx950): forward over whole signals, and one tick.  The formulas
// and the split of the work are in ns_recur.h.
//
// Bound by memory and, nearly as much, by the elementwise part: two sigmoids, an exp2, a root and the
// series are some 40 slots of the vector ALU a tick and channel, which it is 72 to 76% busy with.
// 2048 ticks of 8 x 4096 in bf16 with a gate (671 MB) take 148 us in passes back to back (the average
// of 40; 174 in the first ones), 4.5 TB/s; 16,384 of 2048 channels (335 MB) 114: the chunks' ends 48, at
// 4.2 TB/s, and the outputs 70, at 4.8.
#include "ns_recur.h"

namespace ns {
namespace {

constexpr int kWaves = 8, kRun = kRecurTile / kWaves;    // wavefronts; ticks of a tile each
constexpr int kRecurThreads = 64 * kWaves;

template <class T, int V>
struct RecurRaw {
  Pack<T, V> x[kRun], forget[kRun], write[kRun], z[kRun];
};

template <class T, int V, bool kGate>
__device__ __forceinline__ void request(const RecurIn<T>& in, const RecurPlace& p, int t,
                                        RecurRaw<T, V>& raw) {
  load_run<T, V>(in.x, p, t, raw.x);
  load_run<T, V>(in.forget, p, t, raw.forget);
  load_run<T, V>(in.write, p, t, raw.write);
  if (kGate) load_run<T, V>(in.z, p, t, raw.z);
}

// A tick's decay and what it adds.
struct Tick {
  float decay, add;
};
__device__ __forceinline__ Tick recur_tick(float x, float forget, float write, float rate, bool live) {
  const float u = rate * sigmoid(forget), a = __builtin_amdgcn_exp2f(-kLog2e * u);
  const float add = __builtin_amdgcn_sqrtf(room_squared(u, a)) * sigmoid(write) * x;
  return Tick{live ? a : 1.0f, live ? add : 0.0f};
}

// A stretch of ticks, h -> decay h + add.
template <int V>
struct Stretch {
  float decay[V], add[V];
};

// The state that chunk c starts from: the stretches of the chunks before it, composed by the
// wavefronts in runs, which meet in LDS.
template <int V>
__device__ __forceinline__ void chunk_start(const RecurShape& s, const RecurPlace& p, const float* ends,
                                            int wave, Stretch<V> (*meet)[64], float (&h)[V]) {
  const int before = static_cast<int>(p.c), per = (before + kWaves - 1) / kWaves;
  const int first = wave * per < before ? wave * per : before;
  const int last = first + per < before ? first + per : before;
  const int64_t lines = s.batch * s.channels;
  Stretch<V> own;
#pragma unroll
  for (int j = 0; j < V; ++j) own.decay[j] = 1.0f, own.add[j] = 0.0f;
#pragma unroll 4
  for (int c = first; c < last; ++c) {
    const float* row = ends + c * 2 * lines + p.b * s.channels;
    float decay[V], add[V];
    load_floats<V>(row, p, decay);
    load_floats<V>(row + lines, p, add);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      own.add[j] = fmaf(decay[j], own.add[j], add[j]);
      own.decay[j] *= decay[j];
    }
  }
  meet[wave][threadIdx.x & 63] = own;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) {
    const Stretch<V> other = meet[w][threadIdx.x & 63];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = fmaf(other.decay[j], h[j], other.add[j]);
  }
  __syncthreads();
}

// Chunks' stretches, for chunked calls: the wavefronts take neighbouring runs of whole tiles'
// ticks and meet once at the end.
template <class T, int V>
__global__ __launch_bounds__(kRecurThreads) void recur_ends(RecurShape s, RecurIn<T> in, float* ends) {
  __shared__ Stretch<V> meet[kWaves][64];
  const RecurPlace p = recur_place<V>(s, in.lengths);
  const int wave = uniform(threadIdx.x >> 6);
  float rate[V];
  load_floats<V>(in.rates, p, rate);
#pragma unroll
  for (int j = 0; j < V; ++j) rate[j] = fade_rate(rate[j]);
  Stretch<V> own;
#pragma unroll
  for (int j = 0; j < V; ++j) own.decay[j] = 1.0f, own.add[j] = 0.0f;
  const int run = static_cast<int>(s.chunk) / kWaves;     // whole runs of kRun ticks
  const int from = p.t0 + wave * run, stop = from + run < p.end ? from + run : p.end;
  RecurRaw<T, V> raw;
  if (from < stop) request<T, V, false>(in, p, from, raw);
  for (int t = from; t < stop; t += kRun) {
    float decay[kRun][V], add[kRun][V];
#pragma unroll
    for (int k = 0; k < kRun; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const Tick tick = recur_tick(static_cast<float>(raw.x[k].v[j]),
                                     static_cast<float>(raw.forget[k].v[j]),
                                     static_cast<float>(raw.write[k].v[j]), rate[j], t + k < stop);
        decay[k][j] = tick.decay;
        add[k][j] = tick.add;
      }
    request<T, V, false>(in, p, t + kRun, raw);
#pragma unroll
    for (int k = 0; k < kRun; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        own.add[j] = fmaf(decay[k][j], own.add[j], add[k][j]);
        own.decay[j] *= decay[k][j];
      }
  }
  meet[wave][threadIdx.x & 63] = own;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    const Stretch<V> other = meet[w][threadIdx.x];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      own.add[j] = fmaf(other.decay[j], own.add[j], other.add[j]);
      own.decay[j] *= other.decay[j];
    }
  }
  float* row = ends + p.c * 2 * (s.batch * s.channels) + p.b * s.channels;
  store_floats<V>(row, p, own.decay);
  store_floats<V>(row + s.batch * s.channels, p, own.add);
}

template <class T, int V, bool kGate>
__global__ __launch_bounds__(kRecurThreads) void recur_forward(RecurShape s, RecurIn<T> in, Signal<T> y,
                                                               const float* start, float* out_state,
                                                               float* checkpoints, const float* ends) {
  __shared__ Stretch<V> meet[2][kWaves][64];
  const RecurPlace p = recur_place<V>(s, in.lengths);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t row = p.b * s.channels, lines = s.batch * s.channels;
  float rate[V], h[V] = {};
  load_floats<V>(in.rates, p, rate);
#pragma unroll
  for (int j = 0; j < V; ++j) rate[j] = fade_rate(rate[j]);
  if (start) load_floats<V>(start + row, p, h);
  RecurRaw<T, V> raw;
  if (p.t0 < p.end) request<T, V, kGate>(in, p, p.t0 + wave * kRun, raw);
  if (p.c > 0) chunk_start<V>(s, p, ends, wave, meet[0], h);
  int turn = 0;
  for (int t = p.t0; t < p.t1; t += kRecurTile, turn ^= 1) {
    if (checkpoints && wave == 0) store_floats<V>(checkpoints + t / kRecurTile * lines + row, p, h);
    const int own = t + wave * kRun;
    if (t >= p.end) {
#pragma unroll
      for (int k = 0; k < kRun; ++k) {
        const float zero[V] = {};
        if (own + k < p.t1) store_tick<T, V>(y, p, own + k, zero);
      }
      continue;
    }
    float decay[kRun][V], add[kRun][V], gate[kRun][V];
    Stretch<V> mine;
#pragma unroll
    for (int j = 0; j < V; ++j) mine.decay[j] = 1.0f, mine.add[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < kRun; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const Tick tick = recur_tick(static_cast<float>(raw.x[k].v[j]),
                                     static_cast<float>(raw.forget[k].v[j]),
                                     static_cast<float>(raw.write[k].v[j]), rate[j], own + k < p.end);
        decay[k][j] = tick.decay;
        add[k][j] = tick.add;
        mine.add[j] = fmaf(tick.decay, mine.add[j], tick.add);
        mine.decay[j] *= tick.decay;
        const float z = kGate ? static_cast<float>(raw.z[k].v[j]) : 0.0f;
        gate[k][j] = kGate ? z * sigmoid(z) : 1.0f;
      }
    request<T, V, kGate>(in, p, own + kRecurTile, raw);
    // Two places to meet in turn: a wavefront that is a tile ahead leaves this one alone.
    meet[turn][wave][lane] = mine;
    __syncthreads();
    float from[V];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const Stretch<V> other = meet[turn][w][lane];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (w == wave) from[j] = h[j];
        h[j] = fmaf(other.decay[j], h[j], other.add[j]);
      }
    }
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      float out[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        from[j] = fmaf(decay[k][j], from[j], add[k][j]);
        out[j] = own + k < p.end ? from[j] * gate[k][j] : 0.0f;
      }
      if (own + k < p.t1) store_tick<T, V>(y, p, own + k, out);
    }
  }
  if (p.c == s.chunks - 1 && wave == 0 && out_state) store_floats<V>(out_state + row, p, h);
}

// One tick, the states updated in place; a lane per state.
template <class T>
__global__ __launch_bounds__(kThreads) void recur_step(RecurShape s, RecurIn<T> in, Signal<T> y,
                                                       float* state) {
  const int64_t line = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (line >= s.batch * s.channels) return;
  const uint32_t channels = static_cast<uint32_t>(s.channels);   // line: below 2^31
  const uint32_t b = static_cast<uint32_t>(line) / channels;
  const uint32_t n = static_cast<uint32_t>(line) - b * channels;
  const Tick tick = recur_tick(static_cast<float>(in.x.row(0, b)[n]),
                               static_cast<float>(in.forget.row(0, b)[n]),
                               static_cast<float>(in.write.row(0, b)[n]), fade_rate(in.rates[n]), true);
  const float z = in.z.data ? static_cast<float>(in.z.row(0, b)[n]) : 0.0f;
  const float h = fmaf(tick.decay, state[line], tick.add);
  state[line] = h;
  y.row(0, b)[n] = static_cast<T>(in.z.data ? h * (z * sigmoid(z)) : h);
}

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

template <class T, int V>
int run_forward(const ns_recurrence_args* a, hipStream_t stream) {
  const RecurShape s = recur_shape(a, V);
  dim3 grid;
  if (int rc = recur_grid(s, &grid)) return rc;
  const RecurIn<T> in = recur_in<T>(a);
  if (s.chunks > 1) {
    recur_ends<T, V><<<grid, dim3(kRecurThreads), 0, stream>>>(s, in, a->ends);
    if (int rc = launched("recurrence chunks")) return rc;
  }
  if (a->z.data)
    recur_forward<T, V, true><<<grid, dim3(kRecurThreads), 0, stream>>>(
        s, in, signal<T>(a->y), a->state, a->out_state, a->checkpoints, a->ends);
  else
    recur_forward<T, V, false><<<grid, dim3(kRecurThreads), 0, stream>>>(
        s, in, signal<T>(a->y), a->state, a->out_state, a->checkpoints, a->ends);
  return launched("recurrence");
}

template <class T>
int run_step(const ns_recurrence_args* a, hipStream_t stream) {
  if (a->batch * a->channels > INT32_MAX) return fail("the signal is too large for one launch");
  const int64_t groups = (a->batch * a->channels + kThreads - 1) / kThreads;
  recur_step<T><<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, stream>>>(
      recur_shape(a, 1), recur_in<T>(a), signal<T>(a->y), a->out_state);
  return launched("recurrence step");
}

template <class T>
int run(const ns_recurrence_args* a, bool step, hipStream_t stream) {
  if (step) return run_step<T>(a, stream);
  return recur_lane_channels(a) == 2 ? run_forward<T, 2>(a, stream) : run_forward<T, 1>(a, stream);
}

int run_types(const ns_recurrence_args* a, bool step, void* stream) {
  auto queue = static_cast<hipStream_t>(stream);
  if (a->type == NS_TYPE_F32) return run<float>(a, step, queue);
  if (a->type == NS_TYPE_BF16) return run<__bf16>(a, step, queue);
  return run<_Float16>(a, step, queue);
}

int64_t recur_blocks(const ns_recurrence_args* a, int lane_channels) {
  return (a->channels + 64 * lane_channels - 1) / (64 * lane_channels);
}

// Time chunks worth walking side by side: enough to fill the card twice, four tiles each at least.
// Bf16, us, in one chunk and in chunks: T=2000, B=4, N=4096 (256 workgroups) 89 / 122; T=200, B=4,
// N=600 (40 workgroups) 13.6 / 20.6 (both with tiles of 64 ticks).  With 256, 512 and 1024 workgroups:
// T=16384, B=1, N=2048 132 / 114 / 117, T=65536, B=1, N=512 132 / 117 / 122, T=8192, B=2, N=2048 133 / 118 / 116.
int64_t worth_recur_chunks(const ns_recurrence_args* a) {
  if (a->ticks <= 0 || a->batch <= 0) return 1;
  const int64_t blocks = recur_blocks(a, recur_lane_channels(a)) * a->batch;
  const int64_t tiles = (a->ticks + kRecurTile - 1) / kRecurTile;
  if (blocks >= 192 || tiles < 24) return 1;
  const int64_t chunks = 512 / blocks < tiles / 4 ? 512 / blocks : tiles / 4;
  return chunks < 2 ? 1 : chunks;
}

}  // namespace

// Two channels of 16 bits to a lane where workgroups are many all the same, or where time is cut
// into chunks and there is enough of it for the wider loads to count.  Us, with one and with two:
// T=16384, B=1, N=2048 150 / 126; T=4096, B=4, N=1024 81 / 70; but T=2000, B=1, N=600 16.6 / 22.4, T=16000,
// B=1, N=100 18.4 / 24.5, T=2000, B=4, N=4096 in one chunk 89 and in chunks of two 122.
int recur_lane_channels(const ns_recurrence_args* a) {
  if (a->type == NS_TYPE_F32 || a->channels < 2) return 1;
  if (recur_blocks(a, 2) * a->batch >= 256) return 2;
  if (recur_blocks(a, 1) * a->batch >= 192) return 1;
  constexpr int64_t kMany = 1 << 23;
  return a->batch > 0 && a->ticks * a->channels >= (kMany + a->batch - 1) / a->batch ? 2 : 1;
}

RecurShape recur_shape(const ns_recurrence_args* a, int lane_channels) {
  RecurShape s{};
  s.ticks = a->ticks;
  s.batch = a->batch;
  s.channels = a->channels;
  s.blocks = recur_blocks(a, lane_channels);
  const int64_t tiles = (a->ticks + kRecurTile - 1) / kRecurTile;
  const int64_t wanted = a->chunks > 1 ? a->chunks : 1;
  const int64_t per = tiles > 0 ? (tiles + wanted - 1) / wanted : 1;
  s.chunk = per * kRecurTile;
  s.chunks = tiles > 0 ? (tiles + per - 1) / per : 1;
  return s;
}

int check_recurrence(const ns_recurrence_args* a) {
  if (!a) return fail("recurrence arguments are required");
  if (a->ticks < 0 || a->batch < 0 || a->channels <= 0)
    return fail("a signal is [T, B, N] with N > 0");
  if (a->ticks > INT32_MAX / 2) return fail("a recurrence takes fewer than 2^30 ticks");
  if (a->batch > INT32_MAX) return fail("the signal is too large for one launch");
  if (a->type != NS_TYPE_F32 && a->type != NS_TYPE_BF16 && a->type != NS_TYPE_F16)
    return fail("unknown element type");
  if (a->chunks < 1) return fail("a recurrence has at least one chunk");
  if (!a->rates) return fail("the rates are required");
  if (a->batch && a->ticks && (!a->x.data || !a->forget.data || !a->write.data))
    return fail("x, forget and write are required");
  return NS_OK;
}

int recur_grid(const RecurShape& s, dim3* grid) {
  const int64_t groups = s.blocks * s.batch * s.chunks;
  if (s.blocks > INT32_MAX / s.batch / s.chunks)
    return fail("the signal is too large for one launch");
  *grid = dim3(static_cast<unsigned>(groups));
  return NS_OK;
}

}  // namespace ns

extern "C" {

int ns_recurrence_plan(int64_t ticks, int64_t batch, int64_t channels, int32_t type,
                       int64_t* sizes) {
  ns::clear_error();
  static const float present = 0.0f;
  ns_recurrence_args a{};
  a.ticks = ticks;
  a.batch = batch;
  a.channels = channels;
  a.type = type;
  a.chunks = 1;
  a.rates = &present;
  a.x.data = a.forget.data = a.write.data = const_cast<float*>(&present);
  if (!sizes) return ns::fail("the sizes' place is required");
  if (int rc = ns::check_recurrence(&a)) return rc;
  a.chunks = static_cast<int32_t>(ns::worth_recur_chunks(&a));
  const ns::RecurShape s = ns::recur_shape(&a, ns::recur_lane_channels(&a));
  const int64_t lines = batch * channels;
  sizes[0] = s.chunks;
  sizes[1] = s.chunks > 1 ? s.chunks * 2 * lines : 0;
  sizes[2] = (ticks + ns::kRecurTile - 1) / ns::kRecurTile * lines;
  sizes[3] = s.chunks * lines;
  return NS_OK;
}

int ns_recurrence_forward(const ns_recurrence_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_recurrence(a)) return rc;
  if (a->batch == 0) return NS_OK;
  if (a->ticks && !a->y.data) return ns::fail("the output signal is required");
  if (ns::recur_shape(a, 1).chunks > 1 && !a->ends)
    return ns::fail("a chunked recurrence needs its workspace");
  return ns::run_types(a, false, stream);
}

int ns_recurrence_step(const ns_recurrence_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_recurrence(a)) return rc;
  if (a->ticks != 1 || a->lengths) return ns::fail("a step is one tick of every column");
  if (a->batch == 0) return NS_OK;
  if (!a->y.data) return ns::fail("the output signal is required");
  if (!a->out_state || a->state != a->out_state)
    return ns::fail("a step updates its state in place");
  return ns::run_types(a, true, stream);
}

}  // extern "C"
