// What the forward and the backward of the gated linear recurrence share: the split of the
// work over workgroups and wavefronts, and the elementwise part of a tick.
//
//   s = sigmoid(forget), i = sigmoid(write), u = rate s, a = exp(-u), m = sqrt(1 - a^2)
//   h[t] = a h[t-1] + m i x,   y[t] = h silu(z)
//
// A workgroup takes 64 V neighbouring channels of one column, a lane V of them, and walks
// the ticks in tiles of kRecurTile.  A tile's ticks are dealt to the wavefronts in runs: each
// composes its run, h -> P h + E, the wavefronts meet once in LDS, and each then replays its
// run from its true start.  So the whole of time is walked once, with as many wavefronts a
// channel as hide the memory's latency.
#pragma once

#include "ns_scan.h"

namespace ns {

// Ticks a tile, and between two kept states: eight wavefronts' runs of four.  (Twice as many, us
// against these: the training pass of 2048 x 8 x 4096 in bf16 494 / 461, 16384 ticks of 2048 channels
// 125 / 117, but 2000 x 4 x 4096 89 / 99; runs of eight by four wavefronts 516 and 128.)
constexpr int kRecurTile = 32;

struct RecurShape {
  int64_t ticks, batch, channels;   // ticks below 2^31
  int64_t blocks;                   // workgroups per column and chunk
  int64_t chunks, chunk;            // chunks of `chunk` ticks (whole tiles)
};

template <class T>
struct RecurIn {
  Signal<T> x, forget, write, z;
  const float* rates;
  const int32_t* lengths;
};

// A lane's place: channels n .. n + V - 1 of column b, ticks [t0, t1) of chunk c, of which
// [t0, end) belong to the column.  Past the last channel a lane takes the last V again, as
// another does, and computes and stores what that one does.
struct RecurPlace {
  int64_t base;                     // the workgroup's first channel
  uint32_t lane;                    // the lane's first one from there
  uint32_t b, c;
  int t0, t1, end;
};

template <int V>
__device__ __forceinline__ RecurPlace recur_place(const RecurShape& s, const int32_t* lengths) {
  RecurPlace p;
  const uint32_t blocks = static_cast<uint32_t>(s.blocks), batch = static_cast<uint32_t>(s.batch);
  const uint32_t line = uniform(blockIdx.x / blocks), block = blockIdx.x - line * blocks;
  p.c = uniform(line / batch);
  p.b = line - p.c * batch;
  const int64_t first = static_cast<int64_t>(block) * (64 * V), last = s.channels - V;
  p.base = first < last ? first : last;
  const int64_t own = first + (threadIdx.x & 63) * V;
  p.lane = static_cast<uint32_t>((own < last ? own : last) - p.base);
  const int ticks = static_cast<int>(s.ticks), chunk = static_cast<int>(s.chunk);
  p.t0 = static_cast<int>(p.c) * chunk;
  p.t1 = ticks - p.t0 < chunk ? ticks : p.t0 + chunk;
  const int length = static_cast<int>(uniform(static_cast<uint32_t>(column_ticks(lengths, p.b, ticks))));
  p.end = length < p.t1 ? length : p.t1;
  return p;
}

// Ticks t .. t + K - 1 of a signal at a lane's channels.  Ticks outside [t0, end) read a
// neighbour's value, which is never used: no branches between the loads.
template <class T, int V, int K>
__device__ __forceinline__ void load_run(const Signal<T>& from, const RecurPlace& p, int t,
                                         Pack<T, V> (&to)[K]) {
  const T* base = from.data + p.b * from.sb + p.base;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    int tick = t + k;
    tick = tick < p.end ? tick : p.end - 1;
    tick = tick > p.t0 ? tick : p.t0;
    to[k] = load_pack<T, V>(&at_lane(base + tick * from.st, p.lane * sizeof(T)));
  }
}

template <class T, int V>
__device__ __forceinline__ void store_tick(const Signal<T>& to, const RecurPlace& p, int t,
                                           const float (&v)[V]) {
  Pack<T, V> out;
#pragma unroll
  for (int j = 0; j < V; ++j) out.v[j] = static_cast<T>(v[j]);
  store_pack<T, V>(&at_lane(to.data + t * to.st + p.b * to.sb + p.base, p.lane * sizeof(T)), out);
}

// A lane's V floats of a [.., B, N] workspace or state whose row starts at `row`.
template <int V>
__device__ __forceinline__ void load_floats(const float* row, const RecurPlace& p, float (&v)[V]) {
  const Pack<float, V> in = load_pack<float, V>(row + p.base + p.lane);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = in.v[j];
}
template <int V>
__device__ __forceinline__ void store_floats(float* row, const RecurPlace& p, const float (&v)[V]) {
  Pack<float, V> out;
#pragma unroll
  for (int j = 0; j < V; ++j) out.v[j] = v[j];
  store_pack<float, V>(row + p.base + p.lane, out);
}

// sigmoid(x) and 1 - sigmoid(x), each to its own relative accuracy.
struct Sigmoid {
  float on, off;
};
__device__ __forceinline__ Sigmoid both_sigmoids(float x) {
  const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(x));
  const float large = __builtin_amdgcn_rcpf(1.0f + e), small = e * large;
  return x >= 0.0f ? Sigmoid{large, small} : Sigmoid{small, large};
}

// A rate as it is used: negative ones count as none, and infinity (a channel that forgets at
// once) as the largest number, which times a gate of zero is zero, and not NaN.
__device__ __forceinline__ float fade_rate(float rate) {
  constexpr float kHighest = 3.402823466e38f;
  return rate < 0.0f ? 0.0f : rate > kHighest ? kHighest : rate;
}

// 1 - exp(-2u) given a = exp(-u): for small u by its series (the first term left out is below
// 2^-25 of it), where 1 - a^2 would cancel.
__device__ __forceinline__ float room_squared(float u, float a) {
  const float w = 2.0f * u;
  float s = fmaf(w, -1.0f / 7.0f, 1.0f);
  s = fmaf(w * (-1.0f / 6.0f), s, 1.0f);
  s = fmaf(w * (-1.0f / 5.0f), s, 1.0f);
  s = fmaf(w * (-1.0f / 4.0f), s, 1.0f);
  s = fmaf(w * (-1.0f / 3.0f), s, 1.0f);
  s = fmaf(w * (-1.0f / 2.0f), s, 1.0f);
  return w < 0.25f ? w * s : fmaf(-a, a, 1.0f);
}

template <class T>
inline RecurIn<T> recur_in(const ns_recurrence_args* a) {
  return RecurIn<T>{signal<T>(a->x), signal<T>(a->forget), signal<T>(a->write), signal<T>(a->z),
                    a->rates, a->lengths};
}

// Host: channels per lane, shape of a call (validated), and the checks both directions share.
int recur_lane_channels(const ns_recurrence_args* a);
RecurShape recur_shape(const ns_recurrence_args* a, int lane_channels);
int check_recurrence(const ns_recurrence_args* a);
int recur_grid(const RecurShape& s, dim3* grid);

}  // namespace ns
