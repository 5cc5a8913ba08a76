// Selective state space scan (gfx950): forward over whole signals, and one tick.
//
//   dt = softplus(delta + bias);  h[t] = exp(dt A) h[t-1] + dt x B[t]
//   y[t] = (sum_s C[t] h[t] + D x) silu(z)
//
// Per (tick, channel, state) one exp2 (two issue slots), three multiplies or adds of the update
// and one of the sum, against 8 bytes (bf16) per (tick, channel): the vector ALU bounds it, at
// 16 states by about two to one over HBM.  T=2048, B=8, N=4096, S=16 in bf16: 377 us, of which
// those six slots alone take 192 at the card's 33.5e12 lanes/s and the elementwise part (two
// exp, a log, a reciprocal and their like per tick and channel) about 80: the ALU is 67% busy,
// with two wavefronts a SIMD (512 workgroups); the chunked scan below, with eight, keeps it
// 89-96% busy, but walks twice.  (With inputs two tiles ahead 412, with the elementwise part of
// a thread's items overlapping 377; a tile's ticks beside the next one's elementwise part, in
// two halves of LDS, 375 and so left out.)
//
// Few columns and channels leave most of the card idle, so time is then cut into chunks
// scanned side by side: a first pass gives every chunk's end state from zero and its
// summed time step, whose exponential is the chunk's decay exp(A sum dt); the chunks are
// joined in order; a second pass runs them from their true start.  It costs the update
// twice, so it is taken only where workgroups are few (worth_chunks).  T=16384, B=1, N=2048,
// S=16 in bf16, 64 chunks: 107 us for the ends, 13 for the join, 160 for the outputs; in one
// chunk the 32 workgroups would take 40 us per 256 ticks.
#include "ns_scan.h"

namespace ns {

// What a thread keeps of its (tick, channel) items from the elementwise work to the output.
template <int kItems>
struct ScanItems {
  float skip[kItems], gate[kItems];
};

template <class T, int kItems>
struct ScanRaw {
  T x[kItems], delta[kItems], z[kItems], write, read;
};

template <class T, int R, int kItems, bool kEnds>
__device__ __forceinline__ void request(const ScanIn<T>& in, const ScanShape& s, const ScanPlace& p,
                                        int t, int wave, uint32_t bytes, ScanRaw<T, kItems>& raw) {
  load_items<T, kItems>(in.x, p, t, wave, bytes, raw.x);
  load_items<T, kItems>(in.delta, p, t, wave, bytes, raw.delta);
  if (!kEnds && in.z.data) load_items<T, kItems>(in.z, p, t, wave, bytes, raw.z);
  raw.write = load_shared<T, R>(in.write, s, p, t, threadIdx.x);
  if (!kEnds) raw.read = load_shared<T, R>(in.read, s, p, t, threadIdx.x);
}

// kEnds: the first pass of a chunked scan, which keeps only end states and summed steps.
template <class T, int R, bool kEnds>
__global__ __launch_bounds__(kThreads) void scan_forward(ScanShape s, ScanIn<T> in, Signal<T> y,
                                                         const float* start, float* out_state,
                                                         float* checkpoints, float* ends,
                                                         float* steps) {
  constexpr int CT = kTile<R>, kItems = CT / 4;
  __shared__ float2 step_of[CT][kScanChannels];          // dt, dt * x
  __shared__ float write[CT][4 * R], read[CT][4 * R];
  __shared__ float sums[CT][kScanChannels];
  const ScanPlace p = scan_place(s, in.lengths);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int q = threadIdx.x & 3, channel = threadIdx.x >> 2;
  const bool own = channel < p.own;
  const int64_t n = p.n0 + (own ? channel : 0), line = p.b * s.channels + n;
  const int64_t first_line = p.b * s.channels + p.n0, lines = s.batch * s.channels;
  const uint32_t bytes = lane_bytes<T>(p, lane), state_bytes = lane_states_bytes<R>(channel, q);

  float rate[R], h[R];
  lane_row<R>(in.rates, n, q, s.states, own, rate);
#pragma unroll
  for (int r = 0; r < R; ++r) rate[r] = exponent_rate(rate[r]);
  if (kEnds) {
#pragma unroll
    for (int r = 0; r < R; ++r) h[r] = 0.0f;
  } else if (p.c > 0) {
    load_lane<R>(ends + (p.c * lines + first_line) * (4 * R), own ? state_bytes : 0, h);
  } else {
    lane_row<R>(start, line, q, s.states, own, h);
  }
  const float bias = in.delta_bias && lane < p.own ? in.delta_bias[p.n0 + lane] : 0.0f;
  const float skip = in.skip && lane < p.own ? in.skip[p.n0 + lane] : 0.0f;
  float total = 0.0f;

  // Two tiles of inputs are on their way: a tile's ticks take about as long as one request.
  ScanRaw<T, kItems> even{}, odd{};
  if (p.t0 < p.end) {
    request<T, R, kItems, kEnds>(in, s, p, p.t0, wave, bytes, even);
    request<T, R, kItems, kEnds>(in, s, p, p.t0 + CT, wave, bytes, odd);
  }
  const int64_t tile_floats = lines * (4 * R);
  float* checkpoint = checkpoints ? checkpoints + p.t0 / CT * tile_floats + first_line * (4 * R)
                                  : nullptr;
  const auto tile = [&](int t, ScanRaw<T, kItems>& raw) __attribute__((always_inline)) {
    if (!kEnds && checkpoints) {
      if (own) store_lane<R>(checkpoint, state_bytes, h);
      checkpoint += tile_floats;
    }
    ScanItems<kItems> items;
    if (t < p.end) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int tick = wave + 4 * i;
        const bool live = t + tick < p.end && lane < p.own;
        const float x = live ? static_cast<float>(raw.x[i]) : 0.0f;
        float dt = time_step(static_cast<float>(raw.delta[i]) + bias, s.softplus);
        dt = live ? dt : 0.0f;
        step_of[tick][lane] = make_float2(dt, dt * x);
        if (!kEnds) {
          const float z = static_cast<float>(raw.z[i]);
          float gate = z * sigmoid(z);
          settle(gate);
          items.skip[i] = skip * x;
          items.gate[i] = in.z.data ? gate : 1.0f;
          settle(items.skip[i]);
          settle(items.gate[i]);
        }
      }
      place_shared<T, R>(raw.write, s, p, t, threadIdx.x, write);
      if (!kEnds) place_shared<T, R>(raw.read, s, p, t, threadIdx.x, read);
      request<T, R, kItems, kEnds>(in, s, p, t + 2 * CT, wave, bytes, raw);
      __syncthreads();
#pragma unroll
      for (int tick = 0; tick < CT; ++tick) {
        const float2 d = step_of[tick][channel];
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float decay = __builtin_amdgcn_exp2f(d.x * rate[r]);
          h[r] = fmaf(decay, h[r], d.y * write[tick][q * R + r]);
          if (!kEnds) sum = fmaf(read[tick][q * R + r], h[r], sum);
        }
        if (kEnds) total += d.x;
        else sums[tick][channel] = quad_sum(sum);
      }
      __syncthreads();
    }
    if (!kEnds) {
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int tick = wave + 4 * i;
        if (t + tick < p.t1 && lane < p.own)
          at_lane(y.row(t + tick, p.b) + p.n0, bytes) = static_cast<T>(
              t + tick < p.end ? (sums[tick][lane] + items.skip[i]) * items.gate[i] : 0.0f);
      }
    }
  };
  for (int t = p.t0; t < p.t1; t += 2 * CT) {
    tile(t, even);
    if (t + CT < p.t1) tile(t + CT, odd);
  }
  if (kEnds) {
    if (own) {
      store_lane<R>(ends + (p.c * lines + first_line) * (4 * R), state_bytes, h);
      if (q == 0) steps[p.c * lines + line] = total;
    }
  } else if (p.c == s.chunks - 1 && own && out_state) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (q * R + r < s.states) out_state[line * s.states + q * R + r] = h[r];
  }
}

// 2^exponent carry, also where 2^exponent alone has no float32: growing states (positive
// rates) multiply by more than that over a chunk, which a carry of zero or a tiny one bears as
// it does tick by tick.  Beyond 2^+-1000 any carry but zero is past float32's range.
__device__ __forceinline__ float over_chunk(float carry, float exponent) {
  const float bounded = fminf(fmaxf(exponent, -1000.0f), 1000.0f), whole = rintf(bounded);
  return __builtin_ldexpf(__builtin_amdgcn_exp2f(bounded - whole) * carry, static_cast<int>(whole));
}

// One lane per (column, channel, padded state): walks the chunks in order, leaving in
// place of each chunk's own end the state (or adjoint) it starts from.  `blocks` workgroups
// to a column.  Reads past the last chunk are the last one's again, so that all of a round
// are requested without a branch between them.  64 chunks of 2048 channels with 16 states (17
// MB that another XCD has just written): 13 us, all 64 requested at once 11.
__global__ __launch_bounds__(kThreads) void join_kernel(ScanShape s, uint32_t blocks,
                                                        uint32_t padded, const float* rates,
                                                        const float* start, float* ends,
                                                        const float* steps, bool reverse) {
  const uint32_t b = uniform(blockIdx.x / blocks);
  const int64_t at = static_cast<int64_t>(blockIdx.x - b * blocks) * kThreads + threadIdx.x;
  if (at >= s.channels * padded) return;
  const uint32_t state = static_cast<uint32_t>(at) & (padded - 1);   // a power of two
  const int64_t channel = at >> (31 - __builtin_clz(padded)), lines = s.batch * s.channels;
  const int64_t line = b * s.channels + channel;
  const bool real = state < static_cast<uint32_t>(s.states);
  const float rate = real ? exponent_rate(rates[channel * s.states + state]) : 0.0f;
  float carry = real && start ? start[line * s.states + state] : 0.0f;
  const int chunks = static_cast<int>(s.chunks);
  constexpr int kAhead = 16;
  for (int first = 0; first < chunks; first += kAhead) {
    float own[kAhead], step[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int k = first + u < chunks ? first + u : chunks - 1;
      const int64_t c = reverse ? chunks - 1 - k : k;
      own[u] = ends[(c * lines + line) * padded + state];
      step[u] = steps[c * lines + line];
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (first + u < chunks) {
        const int64_t c = reverse ? chunks - 1 - first - u : first + u;
        ends[(c * lines + line) * padded + state] = carry;
        carry = over_chunk(carry, step[u] * rate) + own[u];
      }
    }
  }
}

// One tick, the states updated in place.  Bound by the states' bytes, each read and
// written once; a channel's four lanes read neighbouring floats.  B=32, N=4096, S=16: 6.4 us
// for 18 MB, of which a launch takes 2.
template <class T, int R>
__global__ __launch_bounds__(kThreads) void scan_step(ScanShape s, ScanIn<T> in, Signal<T> y,
                                                      float* state) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t line = id >> 2;
  const int q = threadIdx.x & 3;
  if (line >= s.batch * s.channels) return;
  const uint32_t channels = static_cast<uint32_t>(s.channels);   // line: below 2^31
  const uint32_t b = static_cast<uint32_t>(line) / channels;
  const uint32_t n = static_cast<uint32_t>(line) - b * channels;
  const uint32_t group = n / static_cast<uint32_t>(s.group_channels);
  float rate[R], h[R], write[R], read[R];
  lane_row<R>(state, line, q, s.states, true, h);
  lane_row<R>(in.rates, n, q, s.states, true, rate);
  lane_row<R, T>(in.write.row(0, b), group, q, s.states, true, write);
  lane_row<R, T>(in.read.row(0, b), group, q, s.states, true, read);
  const float x = static_cast<float>(in.x.row(0, b)[n]);
  const float raw = static_cast<float>(in.delta.row(0, b)[n]);
  const float z = in.z.data ? static_cast<float>(in.z.row(0, b)[n]) : 0.0f;
  const float bias = in.delta_bias ? in.delta_bias[n] : 0.0f;
  const float skip = in.skip ? in.skip[n] : 0.0f;
  const float dt = time_step(raw + bias, s.softplus);
  float sum = 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    h[r] = fmaf(__builtin_amdgcn_exp2f(dt * exponent_rate(rate[r])), h[r], dt * x * write[r]);
    sum = fmaf(read[r], h[r], sum);
  }
  if (s.states == 4 * R) {
    Pack<float, R> out;
#pragma unroll
    for (int r = 0; r < R; ++r) out.v[r] = h[r];
    store_pack<float, R>(state + line * (4 * R) + q * R, out);
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (q * R + r < s.states) state[line * s.states + q * R + r] = h[r];
  }
  sum = quad_sum(sum) + skip * x;
  if (q == 0) y.row(0, b)[n] = static_cast<T>(in.z.data ? sum * (z * sigmoid(z)) : sum);
}

// Time chunks worth scanning side by side: enough to fill the card, at least two tiles each.
// Forward / backward, us, at 16 states in bf16:
//   blocks (T, B, N)            1 chunk      8          16         32         64
//   256  (2048, 8, 2048)        293 / 801    244 / 631  238 / 636
//   64   (4096, 1, 4096)                                136 / 340  134 / 341
//   32   (16384, 1, 2048)                                          262 / 651  249 / 642
//   32   (256, 1, 2048)         40           18.7
// Few tiles over many blocks do not pay: 256 blocks, forward with 1 and 4 chunks, 400 ticks
// 64 and 60, 128 ticks 23 and 31.  With 512 blocks one chunk is faster than two, 369 / 1039
// against 499 / 1254: every further pass costs the update again.
static int64_t worth_chunks(const ns_scan_args* a) {
  if (a->ticks <= 0 || a->batch <= 0) return 1;
  const int64_t per = a->channels / a->groups;
  const int64_t blocks = a->groups * ((per + kScanChannels - 1) / kScanChannels) * a->batch;
  const int64_t tile = tile_of(lane_states(a->states)), tiles = (a->ticks + tile - 1) / tile;
  if (blocks >= 512 || tiles < 8 + blocks / 16) return 1;
  const int64_t chunks = 2048 / blocks < tiles / 2 ? 2048 / blocks : tiles / 2;
  return chunks < 2 ? 1 : chunks;
}

ScanShape scan_shape(const ns_scan_args* a) {
  ScanShape s{};
  s.ticks = a->ticks;
  s.batch = a->batch;
  s.channels = a->channels;
  s.groups = a->groups;
  s.group_channels = a->channels / a->groups;
  s.group_blocks = (s.group_channels + kScanChannels - 1) / kScanChannels;
  const int64_t tile = tile_of(lane_states(a->states));
  const int64_t tiles = (a->ticks + tile - 1) / tile;
  const int64_t wanted = a->chunks > 1 ? a->chunks : 1;
  const int64_t per = tiles > 0 ? (tiles + wanted - 1) / wanted : 1;
  s.chunk = per * tile;
  s.chunks = tiles > 0 ? (tiles + per - 1) / per : 1;
  s.states = a->states;
  s.softplus = a->softplus;
  return s;
}

int check_shape(const ns_scan_args* a) {
  if (a->ticks < 0 || a->batch < 0 || a->channels <= 0)
    return fail("a signal is [T, B, N] with N > 0");
  if (a->ticks > INT32_MAX - 64) return fail("a scan takes fewer than 2^31 ticks");
  if (a->groups < 1 || a->channels % a->groups)
    return fail("the groups must divide the channels");
  if (a->states < 1 || a->states > NS_SCAN_MAX_STATES)
    return fail("a channel has 1 to %d states", NS_SCAN_MAX_STATES);
  return NS_OK;
}

int check_scan(const ns_scan_args* a) {
  if (!a) return fail("scan arguments are required");
  if (int rc = check_shape(a)) return rc;
  if (a->type != NS_TYPE_F32 && a->type != NS_TYPE_BF16 && a->type != NS_TYPE_F16)
    return fail("unknown element type");
  if (a->chunks < 1) return fail("a scan has at least one chunk");
  if (!a->rates) return fail("the decay rates are required");
  if (a->batch && a->ticks &&
      (!a->x.data || !a->delta.data || !a->write.data || !a->read.data))
    return fail("x, delta, B and C are required");
  return NS_OK;
}

int scan_grid(const ScanShape& s, dim3* grid) {
  const int64_t groups = s.groups * s.group_blocks * s.batch * s.chunks;
  if (groups > INT32_MAX) return fail("the signal is too large for one launch");
  *grid = dim3(static_cast<unsigned>(groups));
  return NS_OK;
}

namespace {

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

template <class T, int R>
int run_forward(const ns_scan_args* a, hipStream_t stream) {
  const ScanShape s = scan_shape(a);
  dim3 grid;
  if (int rc = scan_grid(s, &grid)) return rc;
  const ScanIn<T> in = scan_in<T>(a);
  const Signal<T> y = signal<T>(a->y);
  float* steps = a->ends ? a->ends + s.chunks * s.batch * s.channels * (4 * R) : nullptr;
  if (s.chunks > 1) {
    scan_forward<T, R, true><<<grid, dim3(kThreads), 0, stream>>>(s, in, y, nullptr, nullptr,
                                                                  nullptr, a->ends, steps);
    if (int rc = launched("scan chunks")) return rc;
    if (int rc = join_chunks(a, a->ends, a->state, false, stream)) return rc;
  }
  scan_forward<T, R, false><<<grid, dim3(kThreads), 0, stream>>>(
      s, in, y, a->state, a->out_state, a->checkpoints, a->ends, nullptr);
  return launched("scan");
}

template <class T, int R>
int run_step(const ns_scan_args* a, hipStream_t stream) {
  const ScanShape s = scan_shape(a);
  if (s.batch * s.channels > INT32_MAX) return fail("the signal is too large for one launch");
  const int64_t groups = (s.batch * s.channels * 4 + kThreads - 1) / kThreads;
  scan_step<T, R><<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, stream>>>(
      s, scan_in<T>(a), signal<T>(a->y), a->out_state);
  return launched("scan step");
}

template <class T>
int run(const ns_scan_args* a, bool step, hipStream_t stream) {
  switch (lane_states(a->states)) {
    case 1: return step ? run_step<T, 1>(a, stream) : run_forward<T, 1>(a, stream);
    case 2: return step ? run_step<T, 2>(a, stream) : run_forward<T, 2>(a, stream);
    case 4: return step ? run_step<T, 4>(a, stream) : run_forward<T, 4>(a, stream);
    case 8: return step ? run_step<T, 8>(a, stream) : run_forward<T, 8>(a, stream);
    default: return step ? run_step<T, 16>(a, stream) : run_forward<T, 16>(a, stream);
  }
}

int run_types(const ns_scan_args* a, bool step, void* stream) {
  auto queue = static_cast<hipStream_t>(stream);
  if (a->type == NS_TYPE_F32) return run<float>(a, step, queue);
  if (a->type == NS_TYPE_BF16) return run<__bf16>(a, step, queue);
  return run<_Float16>(a, step, queue);
}

}  // namespace

int join_chunks(const ns_scan_args* a, float* ends, const float* start, bool reverse, void* stream) {
  const ScanShape s = scan_shape(a);
  const int64_t padded = 4 * lane_states(a->states), lines = s.batch * s.channels;
  const int64_t blocks = (s.channels * padded + kThreads - 1) / kThreads;
  if (s.batch * blocks > INT32_MAX) return fail("the signal is too large for one launch");
  join_kernel<<<dim3(static_cast<unsigned>(s.batch * blocks)), dim3(kThreads), 0,
                static_cast<hipStream_t>(stream)>>>(
      s, static_cast<uint32_t>(blocks), static_cast<uint32_t>(padded), a->rates, start, ends,
      ends + s.chunks * lines * padded, reverse);
  return launched("scan join");
}

}  // namespace ns

extern "C" {

int ns_scan_plan(int64_t ticks, int64_t batch, int64_t channels, int64_t groups, int32_t states,
                 int32_t backward, int64_t* sizes) {
  ns::clear_error();
  static const float present = 0.0f;
  ns_scan_args a{};
  a.ticks = ticks;
  a.batch = batch;
  a.channels = channels;
  a.groups = groups;
  a.states = states;
  a.chunks = 1;
  a.rates = &present;
  if (!sizes) return ns::fail("the sizes' place is required");
  if (int rc = ns::check_shape(&a)) return rc;
  a.chunks = static_cast<int32_t>(ns::worth_chunks(&a));
  const ns::ScanShape s = ns::scan_shape(&a);
  const int64_t r = ns::lane_states(states), tile = ns::tile_of(r), lines = batch * channels;
  sizes[0] = s.chunks;
  sizes[1] = s.chunks > 1 ? s.chunks * lines * (4 * r + 1) : 0;
  sizes[2] = (ticks + tile - 1) / tile * lines * 4 * r;
  sizes[3] = backward ? ns::scan_part_floats(&a) : 0;
  return NS_OK;
}

int ns_scan_forward(const ns_scan_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_scan(a)) return rc;
  if (a->batch == 0) return NS_OK;
  if (a->ticks && !a->y.data) return ns::fail("the output signal is required");
  if (ns::scan_shape(a).chunks > 1 && !a->ends)
    return ns::fail("a chunked scan needs its workspace");
  return ns::run_types(a, false, stream);
}

int ns_scan_step(const ns_scan_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_scan(a)) return rc;
  if (a->ticks != 1 || a->lengths) return ns::fail("a step is one tick of every column");
  if (a->batch == 0) return NS_OK;
  if (!a->y.data) return ns::fail("the output signal is required");
  if (!a->out_state || a->state != a->out_state)
    return ns::fail("a step updates its state in place");
  return ns::run_types(a, true, stream);
}

}  // extern "C"
