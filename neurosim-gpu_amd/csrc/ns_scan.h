// What the forward and the backward of the selective scan share: the split of the work
// over workgroups and lanes, and the elementwise part of a tick.
//
// A workgroup takes 64 neighbouring channels of one group and column, and a chunk of
// ticks; four neighbouring lanes share a channel, lane q of them holding the R states
// q*R .. q*R + R-1 (S padded to 4R with rates, B and C of zero: such states stay zero).
// Four lanes per channel rather than one give four times the wavefronts without a
// second pass over time, and leave a lane few enough states that the backward keeps a
// whole tile of them in registers; the price is two DPP adds per tick to join y.  The lanes of
// channels that a group lacks idle: T=512, B=8, N=1024, S=16 in bf16 takes 53 us in one group,
// 51 in 16 (of 64 channels), 97 in 64 (of 16), 980 in 1024 (of one).
//
// Time goes in tiles of kTile<R> ticks.  All threads first do a tile's elementwise work,
// each (tick, channel) once, and leave dt, dt*x (and what else the ticks need) in LDS as
// float32, with the tile's B and C; then the lanes walk the ticks.
#pragma once

#include "ns_signal.h"

namespace ns {

constexpr int kScanChannels = 64;   // channels per workgroup of kThreads lanes

// Ticks per tile: the backward keeps R states and R decays per tick and lane in registers.
template <int R>
constexpr int kTile = R <= 4 ? 16 : 64 / R;

constexpr int tile_of(int64_t r) { return r <= 4 ? 16 : static_cast<int>(64 / r); }

// States per lane for S states.
constexpr int64_t lane_states(int64_t s) {
  return s <= 4 ? 1 : s <= 8 ? 2 : s <= 16 ? 4 : s <= 32 ? 8 : 16;
}

struct ScanShape {
  int64_t ticks, batch, channels, groups;
  int64_t group_channels, group_blocks;   // N/G; workgroups per group
  int64_t chunks, chunk;                  // chunks of `chunk` ticks (whole tiles)
  int32_t states, softplus;
};   // below 2^31: ticks (the scalar unit compares 32 bits), and batch times groups times
     // group_blocks times chunks (scan_grid)

template <class T>
struct ScanIn {
  Signal<T> x, delta, z, write, read;
  const float* rates;
  const float* skip;
  const float* delta_bias;
  const int32_t* lengths;
};

// A value that is the same in every lane of a wavefront, known as such to the compiler:
// what is addressed by it alone is then computed once, on the scalar unit.
__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return __builtin_amdgcn_readfirstlane(v);
}

// A workgroup's place: channels n0 .. n0 + own - 1 of a group, column, chunk.
struct ScanPlace {
  int64_t n0;
  int own, t0, t1, end;        // ticks [t0, t1), of which [t0, end) belong to the column
  uint32_t group, block, b, c;
};

__device__ __forceinline__ ScanPlace scan_place(const ScanShape& s, const int32_t* lengths) {
  ScanPlace p;
  const uint32_t group_blocks = static_cast<uint32_t>(s.group_blocks);
  const uint32_t blocks = static_cast<uint32_t>(s.groups) * group_blocks;
  const uint32_t line = uniform(blockIdx.x / blocks), block = blockIdx.x - line * blocks;
  p.c = uniform(line / static_cast<uint32_t>(s.batch));
  p.b = line - p.c * static_cast<uint32_t>(s.batch);
  p.group = uniform(block / group_blocks);
  p.block = block - p.group * group_blocks;
  const int64_t first = static_cast<int64_t>(p.block) * kScanChannels;
  p.n0 = p.group * s.group_channels + first;
  const int64_t left = s.group_channels - first;
  p.own = static_cast<int>(left < kScanChannels ? left : kScanChannels);
  const int ticks = static_cast<int>(s.ticks), chunk = static_cast<int>(s.chunk);
  p.t0 = static_cast<int>(p.c) * chunk;
  p.t1 = ticks - p.t0 < chunk ? ticks : p.t0 + chunk;
  const int length = static_cast<int>(uniform(static_cast<uint32_t>(column_ticks(lengths, p.b, ticks))));
  p.end = length < p.t1 ? length : p.t1;
  return p;
}

// Element `lane_bytes` bytes past an address that is the same in every lane: the address
// stays in scalar registers and the lane's part is one 32-bit offset, shared by all signals.
template <class T>
__device__ __forceinline__ const T& at_lane(const T* uniform_base, uint32_t lane_bytes) {
  return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(uniform_base) + lane_bytes);
}
template <class T>
__device__ __forceinline__ T& at_lane(T* uniform_base, uint32_t lane_bytes) {
  return *reinterpret_cast<T*>(reinterpret_cast<char*>(uniform_base) + lane_bytes);
}

// One tile of a signal at a workgroup's channels: wavefront w, lane l has ticks w, w+4, ...
// of channel l.  Ticks outside [t0, end) and channels not owned read a neighbour's value,
// which is never used: no branches between the loads.
template <class T, int kItems>
__device__ __forceinline__ void load_items(const Signal<T>& from, const ScanPlace& p, int t, int wave,
                                           uint32_t lane_bytes, T (&to)[kItems]) {
  const T* base = from.data + p.b * from.sb + p.n0;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    int tick = t + wave + 4 * i;
    tick = tick < p.end ? tick : p.end - 1;
    tick = tick > p.t0 ? tick : p.t0;
    to[i] = at_lane(base + tick * from.st, lane_bytes);
  }
}

// The lane part of a channel's address (a channel not owned: the last one's).
template <class T>
__device__ __forceinline__ uint32_t lane_bytes(const ScanPlace& p, int lane) {
  return static_cast<uint32_t>(lane < p.own ? lane : p.own - 1) * sizeof(T);
}

// The thread's number, computed anew: what depends on it (places in LDS and in rows) is
// then not kept in registers across a tile's ticks.
__device__ __forceinline__ int fresh_thread() {
  int thread = static_cast<int>(threadIdx.x);
  asm volatile("" : "+v"(thread));
  return thread;
}

// Sum over the four lanes of a channel, in every one of them (quad permutations 1032, 2301).
__device__ __forceinline__ float quad_sum(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
  return v;
}

// Has `v` computed here: the compiler otherwise moves such work to its later use, and keeps
// its several inputs in registers across a tile's ticks instead of this one value.
__device__ __forceinline__ void settle(float& v) { asm volatile("" : "+v"(v)); }

// A channel's time step.  Computed both ways: a branch between a thread's items would keep
// their chains of dependent operations from overlapping.
__device__ __forceinline__ float time_step(float raw, bool soft) {
  float smooth = softplus(raw);
  settle(smooth);
  return soft ? smooth : raw;
}

// A tile's B or C rows, one value per thread: requested with the tile's other inputs, and
// put into LDS (padded with zeros past S and past the column's end) when the tile begins.
template <class T, int R>
__device__ __forceinline__ T load_shared(const Signal<T>& from, const ScanShape& s,
                                         const ScanPlace& p, int t, int thread) {
  static_assert(kTile<R> * 4 * R <= kThreads, "one value per thread");
  const int tick = thread / (4 * R), state = thread % (4 * R);
  const int start = t < p.t0 ? p.t0 : t < p.end ? t : p.end - 1;
  const T* base = from.data + p.b * from.sb + start * from.st + p.group * s.states;
  const bool inside = state < s.states && start + tick < p.end;
  return base[inside ? tick * from.st + state : 0];
}

template <class T, int R>
__device__ __forceinline__ void place_shared(T value, const ScanShape& s, const ScanPlace& p, int t,
                                             int thread, float (*to)[4 * R]) {
  const int tick = thread / (4 * R), state = thread % (4 * R);
  if (kTile<R> * 4 * R == kThreads || tick < kTile<R>)
    to[tick][state] = state < s.states && t + tick < p.end ? static_cast<float>(value) : 0.0f;
}

// A lane's R values of row n of a [N][S] table, zero past S and for channels not owned: one
// wide load where the lanes' parts are whole.
template <int R, class T = float>
__device__ __forceinline__ void lane_row(const T* table, int64_t n, int q, int32_t states, bool own,
                                         float (&out)[R]) {
  if (table && states == 4 * R) {
    const Pack<T, R> v = load_pack<T, R>(table + n * (4 * R) + q * R);
#pragma unroll
    for (int r = 0; r < R; ++r) out[r] = own ? static_cast<float>(v.v[r]) : 0.0f;
    return;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int s = q * R + r;
    out[r] = own && table && s < states ? static_cast<float>(table[n * states + s]) : 0.0f;
  }
}

// A rate A as the exponent of two that a unit of time brings.  What lies below float32 then,
// minus infinity for one (a state that forgets at once), is its lowest value: a time step of
// zero, as ticks past a column's end have, times that is zero, and not NaN.
__device__ __forceinline__ float exponent_rate(float rate) {
  constexpr float kLowest = -3.402823466e38f;
  const float exponent = rate * kLog2e;
  return exponent < kLowest ? kLowest : exponent;
}

// A lane's R floats of a padded [line][N][4R] workspace at a workgroup's channels.
template <int R>
struct LaneStates {
  float v[R];
};
template <int R>
__device__ __forceinline__ uint32_t lane_states_bytes(int channel, int q) {
  return static_cast<uint32_t>((channel * 4 + q) * R) * 4;
}
template <int R>
__device__ __forceinline__ void load_lane(const float* uniform_base, uint32_t bytes, float (&out)[R]) {
  LaneStates<R> v;
  __builtin_memcpy(&v, &at_lane(uniform_base, bytes), sizeof(v));
#pragma unroll
  for (int r = 0; r < R; ++r) out[r] = v.v[r];
}
template <int R>
__device__ __forceinline__ void store_lane(float* uniform_base, uint32_t bytes, const float (&v)[R]) {
  LaneStates<R> out;
#pragma unroll
  for (int r = 0; r < R; ++r) out.v[r] = v[r];
  __builtin_memcpy(&at_lane(uniform_base, bytes), &out, sizeof(out));
}

template <class T>
inline ScanIn<T> scan_in(const ns_scan_args* a) {
  return ScanIn<T>{signal<T>(a->x), signal<T>(a->delta), signal<T>(a->z), signal<T>(a->write),
                   signal<T>(a->read), a->rates, a->skip, a->delta_bias, a->lengths};
}

// Host: shape of a call (validated), and the checks both directions share.
ScanShape scan_shape(const ns_scan_args* a);
int check_shape(const ns_scan_args* a);
int check_scan(const ns_scan_args* a);
int64_t scan_part_floats(const ns_scan_args* a);   // of ns_scan_backward's partials
int scan_grid(const ScanShape& s, dim3* grid);
// Turns each chunk's own end state (from zero) and decay into the state it starts from, or,
// `reverse`, the adjoint it starts from at its last tick.  Layout: see scan.hip.
int join_chunks(const ns_scan_args* a, float* ends, const float* start, bool reverse, void* stream);

}  // namespace ns
