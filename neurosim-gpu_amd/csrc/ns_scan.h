// What the forward and the backward of the selective scan share: the split of the work
// over workgroups and lanes, and the elementwise part of a tick.
//
// A workgroup takes 64 neighbouring channels of one group and column, and a chunk of
// ticks; four neighbouring lanes share a channel, lane q of them holding the R states
// q*R .. q*R + R-1 (S padded to 4R with rates, B and C of zero: such states stay zero).
// Four lanes per channel rather than one give four times the wavefronts without a
// second pass over time, and leave a lane few enough states that the backward keeps a
// whole tile of them in registers; the price is two DPP adds per tick to join y.
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
};

template <class T>
struct ScanIn {
  Signal<T> x, delta, z, write, read;
  const float* rates;
  const float* skip;
  const float* delta_bias;
  const int32_t* lengths;
};

// A workgroup's place: channels n0 .. n0 + own - 1 of a group, column, chunk.
struct ScanPlace {
  int64_t n0, own, group, b, c, t0, t1;
};

__device__ __forceinline__ ScanPlace scan_place(const ScanShape& s) {
  ScanPlace p;
  const int64_t blocks = s.groups * s.group_blocks;
  const int64_t line = blockIdx.x / blocks, block = blockIdx.x - line * blocks;
  p.c = line / s.batch;
  p.b = line - p.c * s.batch;
  p.group = block / s.group_blocks;
  const int64_t first = (block - p.group * s.group_blocks) * kScanChannels;
  p.n0 = p.group * s.group_channels + first;
  const int64_t left = s.group_channels - first;
  p.own = left < kScanChannels ? left : kScanChannels;
  p.t0 = p.c * s.chunk;
  p.t1 = p.t0 + s.chunk < s.ticks ? p.t0 + s.chunk : s.ticks;
  return p;
}

// Sum over the four lanes of a channel, in every one of them (quad permutations 1032, 2301).
__device__ __forceinline__ float quad_sum(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
  return v;
}

// A channel's time step and its slope in delta.
__device__ __forceinline__ float time_step(float raw, bool soft) { return soft ? softplus(raw) : raw; }

// The tile's B or C rows (padded with zeros past S and past the column's end) into LDS.
template <class T, int R, int kTicks>
__device__ __forceinline__ void stage_shared(const Signal<T>& from, const ScanShape& s,
                                             const ScanPlace& p, int64_t t, int64_t end,
                                             float (*to)[4 * R]) {
#pragma unroll
  for (int i = threadIdx.x; i < kTicks * 4 * R; i += kThreads) {
    const int tick = i / (4 * R), state = i % (4 * R);
    float v = 0.0f;
    if (state < s.states && t + tick < end)
      v = static_cast<float>(from.row(t + tick, p.b)[p.group * s.states + state]);
    to[tick][state] = v;
  }
}

// A lane's R values of row n of a [N][S] table, zero past S and for channels not owned.
template <int R>
__device__ __forceinline__ void lane_row(const float* table, int64_t n, int q, int32_t states,
                                         bool own, float (&out)[R]) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int s = q * R + r;
    out[r] = own && table && s < states ? table[n * states + s] : 0.0f;
  }
}

// Places of a lane's R floats in the padded [line][N][4R] workspaces.
template <int R>
__device__ __forceinline__ void load_lane(const float* from, float (&out)[R]) {
#pragma unroll
  for (int r = 0; r < R; ++r) out[r] = from[r];
}
template <int R>
__device__ __forceinline__ void store_lane(float* to, const float (&v)[R]) {
#pragma unroll
  for (int r = 0; r < R; ++r) to[r] = v[r];
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
int64_t worth_chunks(const ns_scan_args* a, bool backward);
int64_t scan_part_floats(const ns_scan_args* a);   // of ns_scan_backward's partials
int scan_grid(const ScanShape& s, dim3* grid);
// Turns each chunk's own end state (from zero) and decay into the state it starts from, or,
// `reverse`, the adjoint it starts from at its last tick.  Layout: see scan.hip.
int join_chunks(const ns_scan_args* a, float* ends, const float* start, bool reverse, void* stream);

}  // namespace ns
