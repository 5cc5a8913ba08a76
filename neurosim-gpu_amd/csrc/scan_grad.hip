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
// the way back), then the adjoint runs down the tile.  Bound by the vector ALU.
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
  float* rate_parts;    // [chunks*B][N][S]
  float* skip_parts;    // [chunks*B][N]
  float* bias_parts;    // [chunks*B][N]
  float* shared_parts;  // [group_blocks][T][B][G][2][4R]: dC, dB
};

template <class T, int kItems>
struct GradRaw {
  T x[kItems], delta[kItems], z[kItems], dy[kItems];
};

template <class T, int kItems, bool kEnds>
__device__ __forceinline__ void request(const ScanIn<T>& in, const Signal<T>& dy,
                                        const ScanPlace& p, int64_t t, int64_t end,
                                        GradRaw<T, kItems>& raw) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int64_t tick = t + wave + 4 * i;
    raw.x[i] = raw.delta[i] = raw.z[i] = raw.dy[i] = static_cast<T>(0.0f);
    if (t >= p.t0 && tick < end && lane < p.own) {
      const int64_t n = p.n0 + lane;
      if (!kEnds) raw.x[i] = in.x.row(tick, p.b)[n];
      raw.delta[i] = in.delta.row(tick, p.b)[n];
      raw.dy[i] = dy.row(tick, p.b)[n];
      if (in.z.data) raw.z[i] = in.z.row(tick, p.b)[n];
    }
  }
}

// A chunk's own adjoint at its start from zero at its end, and its summed time step.
template <class T, int R>
__global__ __launch_bounds__(kThreads) void scan_adjoint_ends(ScanShape s, ScanIn<T> in,
                                                              Signal<T> dy, float* ends,
                                                              float* steps) {
  constexpr int CT = kTile<R>, kItems = CT / 4;
  __shared__ float2 step_of[CT][kScanChannels];          // dt, gy
  __shared__ float read[CT][4 * R];
  const ScanPlace p = scan_place(s);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int q = threadIdx.x & 3, channel = threadIdx.x >> 2;
  const bool own = channel < p.own;
  const int64_t n = p.n0 + (own ? channel : 0), line = p.b * s.channels + n;
  const int64_t length = column_ticks(in.lengths, p.b, s.ticks);
  const int64_t end = length < p.t1 ? length : p.t1;
  float rate[R], g[R];
  lane_row<R>(in.rates, n, q, s.states, own, rate);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    rate[r] *= kLog2e;
    g[r] = 0.0f;
  }
  const float bias = in.delta_bias && lane < p.own ? in.delta_bias[p.n0 + lane] : 0.0f;
  float total = 0.0f;
  if (end > p.t0) {
    const int64_t last = p.t0 + (end - 1 - p.t0) / CT * CT;
    GradRaw<T, kItems> raw;
    request<T, kItems, true>(in, dy, p, last, end, raw);
    for (int64_t t = last; t >= p.t0; t -= CT) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int tick = wave + 4 * i;
        const float z = static_cast<float>(raw.z[i]);
        float dt = time_step(static_cast<float>(raw.delta[i]) + bias, s.softplus);
        dt = t + tick < end && lane < p.own ? dt : 0.0f;
        const float gate = in.z.data ? z * sigmoid(z) : 1.0f;
        step_of[tick][lane] = make_float2(dt, static_cast<float>(raw.dy[i]) * gate);
      }
      stage_shared<T, R, CT>(in.read, s, p, t, end, read);
      request<T, kItems, true>(in, dy, p, t - CT, end, raw);
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
    }
  }
  if (own) {
    store_lane<R>(ends + (p.c * s.batch * s.channels + line) * (4 * R) + q * R, g);
    if (q == 0) steps[p.c * s.batch * s.channels + line] = total;
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
__global__ __launch_bounds__(kThreads) void scan_backward(ScanShape s, ScanIn<T> in, ScanUp<T> up,
                                                          ScanOut<T> out, const float* checkpoints,
                                                          const float* ends) {
  constexpr int CT = kTile<R>, kItems = CT / 4, SP = 4 * R;
  __shared__ float4 step_of[CT][kScanChannels];          // dt, dt * x, gy
  __shared__ float write[CT][SP], read[CT][SP];
  __shared__ float sum_y[CT][kScanChannels], sum_w[CT][kScanChannels], sum_f[CT][kScanChannels];
  __shared__ float parts[4][CT][2 * SP];                 // per wavefront: dC, dB
  const ScanPlace p = scan_place(s);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int q = threadIdx.x & 3, channel = threadIdx.x >> 2;
  const bool own = channel < p.own;
  const int64_t n = p.n0 + (own ? channel : 0), line = p.b * s.channels + n;
  const int64_t length = column_ticks(in.lengths, p.b, s.ticks);
  const int64_t end = length < p.t1 ? length : p.t1;
  const int64_t block = (p.n0 - p.group * s.group_channels) / kScanChannels;
  float* shared = out.shared_parts +
                  (block * s.ticks * s.batch * s.groups + p.b * s.groups + p.group) * (2 * SP);
  const int64_t shared_t = s.batch * s.groups * (2 * SP);

  float rate[R], g[R], drate[R];
  lane_row<R>(in.rates, n, q, s.states, own, rate);
  if (p.c < s.chunks - 1) {
    load_lane<R>(ends + (p.c * s.batch * s.channels + line) * SP + q * R, g);
  } else {
    lane_row<R>(up.dout_state, line, q, s.states, own, g);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    rate[r] *= kLog2e;
    drate[r] = 0.0f;
    if (!own) g[r] = 0.0f;
  }
  const float bias = in.delta_bias && lane < p.own ? in.delta_bias[p.n0 + lane] : 0.0f;
  const float skip = in.skip && lane < p.own ? in.skip[p.n0 + lane] : 0.0f;
  float dskip = 0.0f, dbias = 0.0f;

  const int64_t last = p.t0 + (p.t1 - 1 - p.t0) / CT * CT;
  GradRaw<T, kItems> raw;
  request<T, kItems, false>(in, up.dy, p, last, end, raw);
  for (int64_t t = last; t >= p.t0; t -= CT) {
    if (t >= end) {                       // past the column's end: zeros
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int64_t tick = t + wave + 4 * i;
        if (tick < p.t1 && lane < p.own) {
          const T zero = static_cast<T>(0.0f);
          out.dx.row(tick, p.b)[p.n0 + lane] = zero;
          out.ddelta.row(tick, p.b)[p.n0 + lane] = zero;
          if (in.z.data) out.dz.row(tick, p.b)[p.n0 + lane] = zero;
        }
      }
      for (int i = threadIdx.x; i < CT * 2 * SP; i += kThreads)
        if (t + i / (2 * SP) < p.t1) shared[(t + i / (2 * SP)) * shared_t + i % (2 * SP)] = 0.0f;
      request<T, kItems, false>(in, up.dy, p, t - CT, end, raw);
      continue;
    }
    float item_x[kItems], item_sig[kItems], item_slope[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int tick = wave + 4 * i;
      const bool live = t + tick < end && lane < p.own;
      const float x = static_cast<float>(raw.x[i]), z = static_cast<float>(raw.z[i]);
      const float dy = static_cast<float>(raw.dy[i]);
      const float soft = static_cast<float>(raw.delta[i]) + bias;
      const float dt = live ? time_step(soft, s.softplus) : 0.0f;
      const float gate = sigmoid(z);
      const float gy = in.z.data ? dy * (z * gate) : dy;
      item_x[i] = x;
      item_sig[i] = s.softplus ? sigmoid(soft) : 1.0f;
      item_slope[i] = dy * (gate * (1.0f + z * (1.0f - gate)));
      step_of[tick][lane] = make_float4(dt, dt * x, gy, 0.0f);
    }
    stage_shared<T, R, CT>(in.write, s, p, t, end, write);
    stage_shared<T, R, CT>(in.read, s, p, t, end, read);
    request<T, kItems, false>(in, up.dy, p, t - CT, end, raw);
    float start[R], h[CT][R], a[CT][R];
#pragma unroll
    for (int r = 0; r < R; ++r) start[r] = 0.0f;
    if (own)
      load_lane<R>(checkpoints + (t / CT * s.batch * s.channels + line) * SP + q * R, start);
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
    }
#pragma unroll
    for (int four = CT - 4; four >= 0; four -= 4) {
      float value[4][2 * R];              // of ticks four .. four+3: dC and dB products
#pragma unroll
      for (int k = 3; k >= 0; --k) {
        const int tick = four + k;
        const float4 d = step_of[tick][channel];
        float through = 0.0f, flow = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          g[r] = fmaf(read[tick][q * R + r], d.z, g[r]);
          value[k][r] = d.z * h[tick][r];
          value[k][R + r] = g[r] * d.y;
          through = fmaf(g[r], write[tick][q * R + r], through);
          g[r] *= a[tick][r];
          const float f = g[r] * (tick ? h[tick - 1][r] : start[r]);
          flow = fmaf(f, rate[r], flow);
          drate[r] = fmaf(f, d.x, drate[r]);
        }
        sum_w[tick][channel] = quad_sum(through);
        sum_f[tick][channel] = quad_sum(flow);
      }
      // Row k of the wavefront gets tick four + k, summed over the 16 channels.
#pragma unroll
      for (int v = 0; v < 2 * R; ++v) {
        const float low = join16(join32(value[0][v], value[2][v]), join32(value[1][v], value[3][v]));
        parts[wave][four + (lane >> 4)][v < R ? q * R + v : SP + q * R + v - R] = row_quads(low);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int tick = wave + 4 * i;
      if (t + tick < p.t1 && lane < p.own) {
        const float4 d = step_of[tick][lane];
        const float through = sum_w[tick][lane], inner = sum_y[tick][lane] + skip * item_x[i];
        const float dx = fmaf(d.x, through, skip * d.z);
        const float dd = fmaf(sum_f[tick][lane], kLn2, item_x[i] * through) * item_sig[i];
        const bool live = t + tick < end;
        out.dx.row(t + tick, p.b)[p.n0 + lane] = static_cast<T>(live ? dx : 0.0f);
        out.ddelta.row(t + tick, p.b)[p.n0 + lane] = static_cast<T>(live ? dd : 0.0f);
        if (in.z.data)
          out.dz.row(t + tick, p.b)[p.n0 + lane] = static_cast<T>(live ? item_slope[i] * inner : 0.0f);
        dskip += live ? d.z * item_x[i] : 0.0f;
        dbias += live ? dd : 0.0f;
      }
    }
    for (int i = threadIdx.x; i < CT * 2 * SP; i += kThreads) {
      const int tick = i / (2 * SP), v = i % (2 * SP);
      if (t + tick < p.t1)
        shared[(t + tick) * shared_t + v] = (parts[0][tick][v] + parts[1][tick][v]) +
                                            (parts[2][tick][v] + parts[3][tick][v]);
    }
    __syncthreads();                      // before the next tile overwrites LDS
  }
  const int64_t part = p.c * s.batch + p.b;
  if (own) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int state = q * R + r;
      if (state < s.states) {
        out.rate_parts[(part * s.channels + n) * s.states + state] = drate[r];
        if (p.c == 0 && out.dstate) out.dstate[line * s.states + state] = g[r];
      }
    }
  }
  sum_y[wave][lane] = dskip;
  sum_w[wave][lane] = dbias;
  __syncthreads();
  if (wave == 0 && lane < p.own) {
    out.skip_parts[part * s.channels + p.n0 + lane] =
        (sum_y[0][lane] + sum_y[1][lane]) + (sum_y[2][lane] + sum_y[3][lane]);
    out.bias_parts[part * s.channels + p.n0 + lane] =
        (sum_w[0][lane] + sum_w[1][lane]) + (sum_w[2][lane] + sum_w[3][lane]);
  }
}

// dC and dB: the workgroups' sums added in order, one lane per (tick, column, group, state).
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
  const int64_t pair = id / (2 * padded), state = id - pair * (2 * padded);
  const int64_t line = pair / s.groups, group = pair - line * s.groups;
  const int64_t t = line / s.batch, b = line - t * s.batch;
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
  int64_t rates, lines, shared;
};

PartSizes part_sizes(const ns_scan_args* a) {
  const ScanShape s = scan_shape(a);
  const int64_t parts = s.chunks * s.batch;
  return PartSizes{parts * s.channels * s.states, parts * s.channels,
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
                 a->partials + sizes.rates, a->partials + sizes.rates + sizes.lines,
                 a->partials + sizes.rates + 2 * sizes.lines};
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
  const int64_t parts = s.chunks * s.batch;
  if (int rc = sum_partials(out.rate_parts, parts, s.channels * s.states, a->drates, stream)) return rc;
  if (int rc = sum_partials(out.skip_parts, parts, s.channels, a->dskip, stream)) return rc;
  if (int rc = sum_partials(out.bias_parts, parts, s.channels, a->ddelta_bias, stream)) return rc;
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
  return sizes.rates + 2 * sizes.lines + sizes.shared;
}

}  // namespace ns

extern "C" {

int ns_scan_backward(const ns_scan_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_scan(a)) return rc;
  if (!a->drates || !a->dskip || !a->ddelta_bias)
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
