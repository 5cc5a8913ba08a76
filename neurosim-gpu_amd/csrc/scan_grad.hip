// Backward of the selective scan (gfx950).
//
// With gy = dy silu(z), a[t] = exp(dt[t] A) and the adjoint
//   g[t] = C[t] gy[t] + a[t+1] g[t+1]      (after the last tick: the final state's gradient)
// the gradients are, per tick,
//   dC = sum_n gy h[t],  dB = sum_n g dt x,  dx = dt sum_s g B + D gy,
//   d(dt) = sum_s (g B x + g h[t-1] a A),  d(delta) = d(dt) softplus',
//   dz = dy (sum_s C h + D x) silu'(z),
// and dA = sum_{t,b} g h[t-1] a dt, dD = sum gy x, the state's gradient a[0] g[0].
//
// Tiles run from the last to the first.  The forward left h before every tile, so a tile's
// states are scanned again from there and kept with their decays in registers (no exp in
// the way back), then the adjoint runs down the tile.  Bound by the vector ALU, 74% busy:
// T=2048, B=8, N=4096, S=16 in bf16 takes 1050 us, and 25 for the sums of dB and dC.
//
// dB and dC are sums over a group's channels.  A wavefront holds 16 channels: per four ticks
// its 8R products per lane are summed over them by two rounds of half exchanges
// (permlane32_swap, permlane16_swap: after them row k of 16 lanes holds tick k's values,
// half the adds of a full butterfly) and two rotations within rows.  The workgroup's four
// wavefronts are added through LDS, its sums stored, and a last launch adds the workgroups:
// no atomics, so results do not change from run to run.
#include "ns_scan.h"

namespace ns {

template <class T>
struct ScanUp {
  Signal<T> dy;
  const float* dout_state;
};

template <class T>
struct ScanOut {
  Signal<T> dx, ddelta, dz;
  float* dstate;
  float* parts;         // [chunks*B] of dA [N][S], dD [N], d(delta_bias) [N]
  float* shared_parts;  // [group_blocks][B][G][T][2][4R]: dC, dB
};

template <class T, int kItems>
struct GradRaw {
  T x[kItems], delta[kItems], z[kItems], dy[kItems], write, read;
};

template <class T, int R, int kItems, bool kEnds>
__device__ __forceinline__ void request(const ScanIn<T>& in, const ScanShape& s, const Signal<T>& dy,
                                        const ScanPlace& p, int t, int wave, int thread,
                                        GradRaw<T, kItems>& raw) {
  const uint32_t bytes = lane_bytes<T>(p, thread & 63);
  if (!kEnds) load_items<T, kItems>(in.x, p, t, wave, bytes, raw.x);
  load_items<T, kItems>(in.delta, p, t, wave, bytes, raw.delta);
  load_items<T, kItems>(dy, p, t, wave, bytes, raw.dy);
  if (in.z.data) load_items<T, kItems>(in.z, p, t, wave, bytes, raw.z);
  if (!kEnds) raw.write = load_shared<T, R>(in.write, s, p, t, thread);
  raw.read = load_shared<T, R>(in.read, s, p, t, thread);
}

// A chunk's own adjoint at its start from zero at its end, and its summed time step.
template <class T, int R>
__global__ __launch_bounds__(kThreads) void scan_adjoint_ends(ScanShape s, ScanIn<T> in,
                                                              Signal<T> dy, float* ends,
                                                              float* steps) {
  constexpr int CT = kTile<R>, kItems = CT / 4;
  __shared__ float2 step_of[CT][kScanChannels];          // dt, gy
  __shared__ float read[CT][4 * R];
  const ScanPlace p = scan_place(s, in.lengths);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int q = threadIdx.x & 3, channel = threadIdx.x >> 2;
  const bool own = channel < p.own;
  const int64_t n = p.n0 + (own ? channel : 0), line = p.b * s.channels + n;
  const int64_t first_line = p.b * s.channels + p.n0, lines = s.batch * s.channels;
  const uint32_t state_bytes = lane_states_bytes<R>(channel, q);
  float rate[R], g[R];
  lane_row<R>(in.rates, n, q, s.states, own, rate);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    rate[r] = exponent_rate(rate[r]);
    g[r] = 0.0f;
  }
  const float bias = in.delta_bias && lane < p.own ? in.delta_bias[p.n0 + lane] : 0.0f;
  float total = 0.0f;
  if (p.end > p.t0) {
    const int last = p.t0 + (p.end - 1 - p.t0) / CT * CT;
    GradRaw<T, kItems> even{}, odd{};
    request<T, R, kItems, true>(in, s, dy, p, last, wave, threadIdx.x, even);
    request<T, R, kItems, true>(in, s, dy, p, last - CT, wave, threadIdx.x, odd);
    const auto tile = [&](int t, GradRaw<T, kItems>& raw) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int tick = wave + 4 * i;
        const bool live = t + tick < p.end && lane < p.own;
        const float z = static_cast<float>(raw.z[i]);
        const float dt = time_step(static_cast<float>(raw.delta[i]) + bias, s.softplus);
        float gate = z * sigmoid(z);
        settle(gate);
        const float gy = static_cast<float>(raw.dy[i]) * (in.z.data ? gate : 1.0f);
        step_of[tick][lane] = make_float2(live ? dt : 0.0f, live ? gy : 0.0f);
      }
      place_shared<T, R>(raw.read, s, p, t, threadIdx.x, read);
      request<T, R, kItems, true>(in, s, dy, p, t - 2 * CT, wave, threadIdx.x, raw);
      __syncthreads();
#pragma unroll
      for (int tick = CT - 1; tick >= 0; --tick) {
        const float2 d = step_of[tick][channel];
        total += d.x;
#pragma unroll
        for (int r = 0; r < R; ++r)
          g[r] = __builtin_amdgcn_exp2f(d.x * rate[r]) * fmaf(read[tick][q * R + r], d.y, g[r]);
      }
      __syncthreads();
    };
    for (int t = last; t >= p.t0; t -= 2 * CT) {
      tile(t, even);
      if (t - CT >= p.t0) tile(t - CT, odd);
    }
  }
  if (own) {
    store_lane<R>(ends + (p.c * lines + first_line) * (4 * R), state_bytes, g);
    if (q == 0) steps[p.c * lines + line] = total;
  }
}

// u over the low 32 lanes' side and v over the high side, each summed with its partner half.
__device__ __forceinline__ float join32(float u, float v) {
  const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, u),
                                                     __builtin_bit_cast(unsigned, v), false, false);
  const unsigned first = both[0], second = both[1];   // a bit_cast of both[1] itself reads both[0]
  return __builtin_bit_cast(float, first) + __builtin_bit_cast(float, second);
}
// The same for even and odd rows of 16 lanes.
__device__ __forceinline__ float join16(float u, float v) {
  const auto both = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, u),
                                                     __builtin_bit_cast(unsigned, v), false, false);
  const unsigned first = both[0], second = both[1];   // a bit_cast of both[1] itself reads both[0]
  return __builtin_bit_cast(float, first) + __builtin_bit_cast(float, second);
}
// Sum over the four quads of a row (rotations by 4 and 8 lanes).
__device__ __forceinline__ float row_quads(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xF, 0xF, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xF, 0xF, true));
  return v;
}

template <class T, int R>
__global__ __launch_bounds__(kThreads, 2) void scan_backward(ScanShape s, ScanIn<T> in, ScanUp<T> up,
                                                          ScanOut<T> out, const float* checkpoints,
                                                          const float* ends) {
  constexpr int CT = kTile<R>, kItems = CT / 4, SP = 4 * R;
  __shared__ float4 step_of[CT][kScanChannels];          // dt, dt * x, gy, x
  __shared__ float write[CT][SP], read[CT][SP];
  __shared__ float sum_y[CT][kScanChannels], sum_w[CT][kScanChannels], sum_f[CT][kScanChannels];
  __shared__ float parts[4][CT][2 * SP];                 // per wavefront: dC, dB
  const ScanPlace p = scan_place(s, in.lengths);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int q = threadIdx.x & 3, channel = threadIdx.x >> 2;
  const bool own = channel < p.own;
  const int64_t n = p.n0 + (own ? channel : 0), line = p.b * s.channels + n;
  const int64_t first_line = p.b * s.channels + p.n0, lines = s.batch * s.channels;
  const uint32_t state_bytes = lane_states_bytes<R>(channel, q);
  // The workgroup's sums for dC and dB: [T][2][4R] of its block, column and group.
  float* shared = out.shared_parts +
                  ((p.block * s.batch + p.b) * s.groups + p.group) * s.ticks * (2 * SP);

  float rate[R], g[R], drate[R];
  lane_row<R>(in.rates, n, q, s.states, own, rate);
  if (p.c < s.chunks - 1) {
    load_lane<R>(ends + (p.c * lines + first_line) * SP, own ? state_bytes : 0, g);
  } else {
    lane_row<R>(up.dout_state, line, q, s.states, own, g);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    rate[r] = exponent_rate(rate[r]);
    drate[r] = 0.0f;
    if (!own) g[r] = 0.0f;
  }
  const float bias = in.delta_bias && lane < p.own ? in.delta_bias[p.n0 + lane] : 0.0f;
  const float skip = in.skip && lane < p.own ? in.skip[p.n0 + lane] : 0.0f;
  float dskip = 0.0f, dbias = 0.0f;

  const int last = p.t0 + (p.t1 - 1 - p.t0) / CT * CT;
  const int64_t tile_floats = lines * SP;
  const float* checkpoint = checkpoints + last / CT * tile_floats + first_line * SP;
  GradRaw<T, kItems> raw{};
  if (p.t0 < p.end) request<T, R, kItems, false>(in, s, up.dy, p, last, wave, threadIdx.x, raw);
  for (int t = last; t >= p.t0; t -= CT, checkpoint -= tile_floats) {
    const int thread = fresh_thread(), lane = thread & 63;
    const uint32_t bytes = lane_bytes<T>(p, lane);
    if (t >= p.end) {                       // past the column's end: zeros
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int tick = t + wave + 4 * i;
        if (tick < p.t1 && lane < p.own) {
          const T zero = static_cast<T>(0.0f);
          at_lane(out.dx.row(tick, p.b) + p.n0, bytes) = zero;
          at_lane(out.ddelta.row(tick, p.b) + p.n0, bytes) = zero;
          if (in.z.data) at_lane(out.dz.row(tick, p.b) + p.n0, bytes) = zero;
        }
      }
      for (int i = thread; i < CT * 2 * SP; i += kThreads)
        if (t + i / (2 * SP) < p.t1) (shared + static_cast<int64_t>(t) * (2 * SP))[i] = 0.0f;
      if (p.t0 < p.end)
        request<T, R, kItems, false>(in, s, up.dy, p, t - CT, wave, thread, raw);
      continue;
    }
    float item_sig[kItems], item_slope[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int tick = wave + 4 * i;
      const bool live = t + tick < p.end && lane < p.own;
      const float x = live ? static_cast<float>(raw.x[i]) : 0.0f, z = static_cast<float>(raw.z[i]);
      const float dy = live ? static_cast<float>(raw.dy[i]) : 0.0f;
      const float soft = static_cast<float>(raw.delta[i]) + bias;
      const float step = time_step(soft, s.softplus), dt = live ? step : 0.0f;
      const float gate = sigmoid(z);
      float gated = dy * (z * gate), slope = sigmoid(soft);
      settle(gated);
      settle(slope);
      const float gy = in.z.data ? gated : dy;
      item_sig[i] = s.softplus ? slope : 1.0f;
      item_slope[i] = dy * (gate * (1.0f + z * (1.0f - gate)));
      settle(item_sig[i]);
      settle(item_slope[i]);
      step_of[tick][lane] = make_float4(dt, dt * x, gy, x);
    }
    place_shared<T, R>(raw.write, s, p, t, thread, write);
    place_shared<T, R>(raw.read, s, p, t, thread, read);
    float start[R], h[CT][R], a[CT][R];
#pragma unroll
    for (int r = 0; r < R; ++r) start[r] = 0.0f;
    if (own) load_lane<R>(checkpoint, state_bytes, start);
    __syncthreads();
#pragma unroll
    for (int tick = 0; tick < CT; ++tick) {
      const float4 d = step_of[tick][channel];
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        a[tick][r] = __builtin_amdgcn_exp2f(d.x * rate[r]);
        h[tick][r] = fmaf(a[tick][r], tick ? h[tick - 1][r] : start[r], d.y * write[tick][q * R + r]);
        sum = fmaf(read[tick][q * R + r], h[tick][r], sum);
      }
      sum_y[tick][channel] = quad_sum(sum);
      if (tick % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int four = CT - 4; four >= 0; four -= 4) {
      // Half the tile's registers are free by now: the next tile's inputs fit.
      if (four == (CT > 4 ? 4 : 0))
        request<T, R, kItems, false>(in, s, up.dy, p, t - CT, wave, fresh_thread(), raw);
      constexpr int RG = R < 2 ? R : 2;   // states whose B and C of four ticks are held
      float4 d[4];
      float through[4] = {}, flow[4] = {};
#pragma unroll
      for (int k = 0; k < 4; ++k) d[k] = step_of[four + k][channel];
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += RG) {
        float w[4][RG], c[4][RG], sum_c[RG], sum_b[RG];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          __builtin_memcpy(w[k], &write[four + k][q * R + r0], sizeof(w[k]));
          __builtin_memcpy(c[k], &read[four + k][q * R + r0], sizeof(c[k]));
        }
#pragma unroll
        for (int r = 0; r < RG; ++r) {
          const int rr = r0 + r;
          float dc[4], db[4];
#pragma unroll
          for (int k = 3; k >= 0; --k) {
            const int tick = four + k;
            g[rr] = fmaf(c[k][r], d[k].z, g[rr]);
            dc[k] = d[k].z * h[tick][rr];
            db[k] = g[rr] * d[k].y;
            through[k] = fmaf(g[rr], w[k][r], through[k]);
            g[rr] *= a[tick][rr];
            const float f = g[rr] * (tick ? h[tick - 1][rr] : start[rr]);
            flow[k] = fmaf(f, rate[rr], flow[k]);
            drate[rr] = fmaf(f, d[k].x, drate[rr]);
          }
          // Row k of the wavefront gets tick four + k, summed over the 16 channels.
          sum_c[r] = row_quads(join16(join32(dc[0], dc[2]), join32(dc[1], dc[3])));
          sum_b[r] = row_quads(join16(join32(db[0], db[2]), join32(db[1], db[3])));
        }
        float* part = &parts[wave][four + (lane >> 4)][q * R + r0];
        __builtin_memcpy(part, sum_c, sizeof(sum_c));
        __builtin_memcpy(part + SP, sum_b, sizeof(sum_b));
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        sum_w[four + k][channel] = quad_sum(through[k]);
        sum_f[four + k][channel] = quad_sum(flow[k]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    const int later = fresh_thread(), out_lane = later & 63;
    const uint32_t out_bytes = lane_bytes<T>(p, out_lane);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int tick = wave + 4 * i;
      if (t + tick < p.t1 && out_lane < p.own) {
        const float4 d = step_of[tick][out_lane];
        const float through = sum_w[tick][out_lane], inner = sum_y[tick][out_lane] + skip * d.w;
        const float dx = fmaf(d.x, through, skip * d.z);
        const float dd = fmaf(sum_f[tick][out_lane], kLn2, d.w * through) * item_sig[i];
        const bool live = t + tick < p.end;
        at_lane(out.dx.row(t + tick, p.b) + p.n0, out_bytes) = static_cast<T>(live ? dx : 0.0f);
        at_lane(out.ddelta.row(t + tick, p.b) + p.n0, out_bytes) = static_cast<T>(live ? dd : 0.0f);
        if (in.z.data)
          at_lane(out.dz.row(t + tick, p.b) + p.n0, out_bytes) = static_cast<T>(live ? item_slope[i] * inner : 0.0f);
        dskip += live ? d.z * d.w : 0.0f;
        dbias += live ? dd : 0.0f;
      }
    }
#pragma unroll
    for (int first = 0; first < CT * 2 * SP; first += kThreads) {
      const uint32_t i = first + later;
      const float* sums = &parts[0][0][0];
      if (i < CT * 2 * SP && t + static_cast<int>(i / (2 * SP)) < p.t1)
        at_lane(shared + static_cast<int64_t>(t) * (2 * SP), 4 * i) =
            (sums[i] + sums[i + CT * 2 * SP]) + (sums[i + 2 * CT * 2 * SP] + sums[i + 3 * CT * 2 * SP]);
    }
    __syncthreads();                      // before the next tile overwrites LDS
  }
  float* const own_parts = out.parts + (p.c * s.batch + p.b) * s.channels * (s.states + 2);
  if (own) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int state = q * R + r;
      if (state < s.states) {
        own_parts[n * s.states + state] = drate[r];
        if (p.c == 0 && out.dstate) out.dstate[line * s.states + state] = g[r];
      }
    }
  }
  sum_y[wave][lane] = dskip;
  sum_w[wave][lane] = dbias;
  __syncthreads();
  if (wave == 0 && lane < p.own) {
    own_parts[s.channels * s.states + p.n0 + lane] =
        (sum_y[0][lane] + sum_y[1][lane]) + (sum_y[2][lane] + sum_y[3][lane]);
    own_parts[s.channels * (s.states + 1) + p.n0 + lane] =
        (sum_w[0][lane] + sum_w[1][lane]) + (sum_w[2][lane] + sum_w[3][lane]);
  }
}

// dC and dB: the workgroups' sums added in order, one lane per (column, group, tick, state).
template <class T>
__global__ __launch_bounds__(kThreads) void add_shared(ScanShape s, int32_t padded,
                                                       const float* __restrict__ parts,
                                                       Signal<T> dread, Signal<T> dwrite) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t total = s.ticks * s.batch * s.groups * 2 * padded;
  if (id >= total) return;
  float four[4] = {};
  int64_t block = 0;
  for (; block + 4 <= s.group_blocks; block += 4)
#pragma unroll
    for (int u = 0; u < 4; ++u) four[u] += parts[(block + u) * total + id];
  for (; block < s.group_blocks; ++block) four[0] += parts[block * total + id];
  const int64_t tick = id / (2 * padded), state = id - tick * (2 * padded);
  const int64_t line = tick / s.ticks, t = tick - line * s.ticks;
  const int64_t b = line / s.groups, group = line - b * s.groups;
  const int64_t own = state < padded ? state : state - padded;
  if (own < s.states)
    (state < padded ? dread : dwrite).row(t, b)[group * s.states + own] =
        static_cast<T>((four[0] + four[1]) + (four[2] + four[3]));
}

namespace {

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

struct PartSizes {
  int64_t parameters, shared;
};

PartSizes part_sizes(const ns_scan_args* a) {
  const ScanShape s = scan_shape(a);
  return PartSizes{s.chunks * s.batch * s.channels * (s.states + 2),
                   s.group_blocks * s.ticks * s.batch * s.groups * 8 * lane_states(s.states)};
}

template <class T, int R>
int run_backward(const ns_scan_args* a, hipStream_t stream) {
  const ScanShape s = scan_shape(a);
  dim3 grid;
  if (int rc = scan_grid(s, &grid)) return rc;
  const ScanIn<T> in = scan_in<T>(a);
  const PartSizes sizes = part_sizes(a);
  ScanOut<T> out{signal<T>(a->dx), signal<T>(a->ddelta), signal<T>(a->dz), a->dstate, a->partials,
                 a->partials + sizes.parameters};
  const Signal<T> dy = signal<T>(a->dy);
  if (s.chunks > 1) {
    scan_adjoint_ends<T, R><<<grid, dim3(kThreads), 0, stream>>>(
        s, in, dy, a->ends, a->ends + s.chunks * s.batch * s.channels * (4 * R));
    if (int rc = launched("scan adjoint chunks")) return rc;
    if (int rc = join_chunks(a, a->ends, a->dout_state, true, stream)) return rc;
  }
  scan_backward<T, R><<<grid, dim3(kThreads), 0, stream>>>(
      s, in, ScanUp<T>{dy, a->dout_state}, out, a->checkpoints, a->ends);
  if (int rc = launched("scan backward")) return rc;
  if (int rc = sum_partials(out.parts, s.chunks * s.batch, s.channels * (s.states + 2),
                            a->dparameters, stream))
    return rc;
  const int64_t values = s.ticks * s.batch * s.groups * 8 * R;
  const int64_t groups = (values + kThreads - 1) / kThreads;
  if (groups > INT32_MAX) return fail("the signal is too large for one launch");
  if (groups == 0) return NS_OK;
  add_shared<T><<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, stream>>>(
      s, 4 * R, out.shared_parts, signal<T>(a->dread), signal<T>(a->dwrite));
  return launched("scan shared gradients");
}

template <class T>
int run(const ns_scan_args* a, hipStream_t stream) {
  switch (lane_states(a->states)) {
    case 1: return run_backward<T, 1>(a, stream);
    case 2: return run_backward<T, 2>(a, stream);
    case 4: return run_backward<T, 4>(a, stream);
    case 8: return run_backward<T, 8>(a, stream);
    default: return run_backward<T, 16>(a, stream);
  }
}

}  // namespace

int64_t scan_part_floats(const ns_scan_args* a) {
  const PartSizes sizes = part_sizes(a);
  return sizes.parameters + sizes.shared;
}

}  // namespace ns

extern "C" {

int ns_scan_backward(const ns_scan_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_scan(a)) return rc;
  if (!a->dparameters)
    return ns::fail("the gradients of the rates, skips and biases are required");
  if (a->batch && a->ticks) {
    if (!a->partials || !a->checkpoints) return ns::fail("the backward needs its workspaces");
    if (!a->dy.data || !a->dx.data || !a->ddelta.data || !a->dwrite.data || !a->dread.data)
      return ns::fail("the gradients of y, x, delta, B and C are required");
    if ((a->z.data != nullptr) != (a->dz.data != nullptr))
      return ns::fail("z and its gradient go together");
    if (ns::scan_shape(a).chunks > 1 && !a->ends)
      return ns::fail("a chunked scan needs its workspace");
  } else {
    return ns::fail("the backward needs at least one tick and column");
  }
  auto queue = static_cast<hipStream_t>(stream);
  if (a->type == NS_TYPE_F32) return ns::run<float>(a, queue);
  if (a->type == NS_TYPE_BF16) return ns::run<__bf16>(a, queue);
  return ns::run<_Float16>(a, queue);
}

}  // extern "C"
