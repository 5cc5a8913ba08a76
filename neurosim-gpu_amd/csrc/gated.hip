// Gated projection (gfx950): y = f(x gate^T) * (x up^T), both products and what joins them in
// one kernel, for rows of float32, bfloat16 and float16.
//
// Tiles take as many rows of `gate` as of `up`, for the same columns of y, and deal them to the
// wavefronts so that a lane ends with both sums of its results: the activation and the
// product are its own affair, and the two M x F products never reach memory (but for a
// training pass, which keeps them in float32: rounded to 16 bits they would cost the gradients
// as much again as the rounding of their own operands).
//
// 8192 x 4096 to 8192 in bf16 with both products kept (0.5 GB of them) takes 890 to 940 us, 1.2
// PFLOP/s, the matrix cores 60% busy: a stage's way into LDS and the stores at a tile's end are what
// they wait for.  One row of 4096 to 8192 (134 MB) takes 23.7 us, 5.7 TB/s.
#include "ns_gated.h"

namespace ns {
namespace {

// Half of a wavefront's strips: those of y.
template <class G>
struct HalfTile {
  static constexpr int MI = G::MI, NJ = G::NJ / 2;
};

// A wavefront's results from row m, column f on, of `rows` x `width`: both products where they are
// kept, and y.  The two strips may be one place: a wavefront uses them one after the other.
template <class G, class T>
__device__ __forceinline__ void store_gated(const v4f (&sum)[G::MI][G::NJ], int activation, T* y,
                                            int64_t stride, float* pre, int64_t m, int64_t f, int64_t rows,
                                            int64_t width, int lane, Strip<HalfTile<G>, T>& strip,
                                            Strip<HalfTile<G>, float>& kept) {
  using H = HalfTile<G>;
  v4f part[H::MI][H::NJ];
  if (pre) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < H::MI; ++i)
#pragma unroll
        for (int j = 0; j < H::NJ; ++j) part[i][j] = sum[i][j + half * H::NJ];
      store_tiles<H, float, false>(pre + half * rows * width + m * width + f, width, part, nullptr, rows - m,
                                   width - f, lane, kept);
    }
  }
#pragma unroll
  for (int i = 0; i < H::MI; ++i)
#pragma unroll
    for (int j = 0; j < H::NJ; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        part[i][j][r] = activated(sum[i][j][r], activation) * sum[i][j + H::NJ][r];
  store_tiles<H, T, false>(y + m * stride + f, stride, part, nullptr, rows - m, width - f, lane, strip);
}

template <class G, class T>
__global__ __launch_bounds__(G::threads, 512 / G::threads) void gated_tiles(Rows x, Rows gate, Rows up, uint32_t pieces,
                                                          int activation, T* y, int64_t stride,
                                                          float* pre, uint32_t tiles_m,
                                                          uint32_t tiles_n) {
  using H = HalfTile<G>;
  // Both kinds of strips of a wavefront lie in its own place: another one may be behind.
  union OwnStrips {
    Strip<H, T> y;
    Strip<H, float> kept;
  };
  __shared__ union {
    v4i stages[G::stages * G::rows * 8];
    OwnStrips strips[G::WM * G::WN];
  } lds;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const TilePlace tile = tile_place(tiles_m, tiles_n);
  const int64_t m0 = static_cast<int64_t>(tile.m) * G::rows_m;
  const int64_t f0 = static_cast<int64_t>(tile.n) * (G::rows_n / 2);
  GemmPlace p;
  p.lane = lane;
  p.wave = wave;
  p.stride_a = static_cast<uint32_t>(x.stride);
  p.stride_b = static_cast<uint32_t>(gate.stride);
  p.pieces = pieces;
  p.a = rows_buffer(x, m0, G::rows_m, pieces);
  const Second<true> b = second_pair<G>(rows_buffer(gate, f0, G::rows_n / 2, pieces),
                                        rows_buffer(up, f0, G::rows_n / 2, pieces), wave);
  v4f sum[G::MI][G::NJ] = {};
  gemm_tile<G, T, true>(p, b, lds.stages, sum);

  const int64_t m = m0 + 16 * (wave / G::WN) * G::MI, f = f0 + 16 * (wave % G::WN) * H::NJ;
  store_gated<G, T>(sum, activation, y, stride, pre, m, f, x.rows, gate.rows, lane, lds.strips[wave].y,
                    lds.strips[wave].kept);
}

// The same for float32 rows in thirds.
template <class G>
__global__ __launch_bounds__(G::threads) void gated_split(Rows x, Rows gate, Rows up, uint32_t blocks,
                                                          int activation, float* y, int64_t stride,
                                                          float* pre, uint32_t tiles_m, uint32_t tiles_n) {
  using H = HalfTile<G>;
  __shared__ union {
    uint8_t stages[G::stages * G::stage_bytes];
    Strip<H, float> strips[G::waves];
    v4i aligned;
  } lds;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const TilePlace tile = tile_place(tiles_m, tiles_n);
  const int64_t m0 = static_cast<int64_t>(tile.m) * G::rows_m;
  const int64_t f0 = static_cast<int64_t>(tile.n) * (G::rows_n / 2);
  const uint32_t pieces = blocks * (kThirds / 16);
  const SplitPlace<G> p = split_place<G, true>(
      lane, wave, blocks, rows_buffer(x, m0, G::rows_m, pieces), static_cast<uint32_t>(x.stride),
      rows_buffer(gate, f0, G::rows_n / 2, pieces), rows_buffer(up, f0, G::rows_n / 2, pieces),
      static_cast<uint32_t>(gate.stride));
  v4f sum[G::MI][G::NJ] = {};
  split_tile<G>(p, lds.stages, sum);
  const int64_t m = m0 + 16 * (wave / G::WN) * G::MI, f = f0 + 16 * (wave % G::WN) * H::NJ;
  store_gated<G, float>(sum, activation, y, stride, pre, m, f, x.rows, gate.rows, lane, lds.strips[wave],
                        lds.strips[wave]);
}

// Up to 16 rows of x: bound by the weights' bytes, each read once.  A workgroup takes 16
// columns of y, 16 rows of both weights, straight from memory to registers, kAhead stages (128
// bytes of a row) requested ahead; its wavefronts take a part of K each and meet in LDS.  Rows
// may start at any element; a row's last, partial stage is read element by element.
constexpr int kFewRows = 16, kAhead = 3, kRowWaves = 8;

template <class T>
__device__ __forceinline__ void load_pieces(const T* from, int64_t stage, v4i (&to)[2]) {
  __builtin_memcpy(to, from + stage * (128 / sizeof(T)), 32);
}

template <class T>
__device__ __forceinline__ void load_last(const T* row, int64_t first, int64_t columns, v4i (&to)[2]) {
  constexpr int kValues = 32 / sizeof(T);
  Pack<T, kValues> v;
#pragma unroll
  for (int k = 0; k < kValues; ++k) v.v[k] = first + k < columns ? row[first + k] : T{};
  __builtin_memcpy(to, &v, sizeof(v));
}

template <class T>
__global__ __launch_bounds__(64 * kRowWaves) void gated_rows(const T* x, int64_t x_stride, const T* gate,
                                                             int64_t gate_stride, const T* up,
                                                             int64_t up_stride, int64_t rows,
                                                             int64_t columns, int64_t width,
                                                             int activation, T* y, int64_t stride,
                                                             float* pre) {
  __shared__ v4f sums[2][kRowWaves][64];
  constexpr int kValues = 128 / sizeof(T);                 // of a row in a stage
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t f0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int64_t own = f0 + (lane & 15) < width ? f0 + (lane & 15) : width - 1;
  const int64_t m = (lane & 15) < rows ? lane & 15 : rows - 1;
  // A quarter of the wavefront takes two neighbouring pieces of a row's eight.
  const int64_t first = (lane >> 4) * (kValues / 4);
  const T* const gate_row = gate + own * gate_stride;
  const T* const up_row = up + own * up_stride;
  const T* const x_row = x + m * x_stride;
  const int64_t whole = columns / kValues, per = (whole + kRowWaves - 1) / kRowWaves;
  const int64_t begin = wave * per, stop = begin + per < whole ? begin + per : whole;
  v4f gated = {}, raised = {};
  v4i g[kAhead][2], u[kAhead][2], v[kAhead][2];
  const auto load = [&](int64_t stage, int to) __attribute__((always_inline)) {
    const int64_t at = stage < stop ? stage : stop - 1;    // read again, not multiplied
    load_pieces<T>(gate_row + first, at, g[to]);
    load_pieces<T>(up_row + first, at, u[to]);
    load_pieces<T>(x_row + first, at, v[to]);
  };
  const auto multiply = [&](int from) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      gated = multiply_pieces<T>(g[from][s], v[from][s], gated);
      raised = multiply_pieces<T>(u[from][s], v[from][s], raised);
    }
  };
  if (begin < stop) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) load(begin + k, k);
    for (int64_t stage = begin; stage < stop; stage += kAhead) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (stage + k < stop) multiply(k);
        if (stage + k + kAhead < stop) load(stage + k + kAhead, k);
      }
    }
  }
  if (wave == kRowWaves - 1 && whole * kValues < columns) {
    const int64_t at = whole * kValues + first;
    load_last<T>(gate_row, at, columns, g[0]);
    load_last<T>(up_row, at, columns, u[0]);
    load_last<T>(x_row, at, columns, v[0]);
    multiply(0);
  }
  sums[0][wave][lane] = gated;
  sums[1][wave][lane] = raised;
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int f = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int from = (f >> 2) * 16 + row;                    // the lane that holds it
  float total[2] = {};
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w)
#pragma unroll
    for (int half = 0; half < 2; ++half)
      total[half] += reinterpret_cast<const float*>(&sums[half][w][from])[f & 3];
  if (row >= rows || f0 + f >= width) return;
  if (pre) {
    pre[row * width + f0 + f] = total[0];
    pre[(rows + row) * width + f0 + f] = total[1];
  }
  y[row * stride + f0 + f] = static_cast<T>(activated(total[0], activation) * total[1]);
}

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

template <class T>
int run_rows(const ns_gated_args* a, hipStream_t stream) {
  const int64_t groups = (a->width + 15) / 16;
  if (groups > INT32_MAX) return fail("the projection is too large for one launch");
  gated_rows<T><<<dim3(static_cast<unsigned>(groups)), dim3(64 * kRowWaves), 0, stream>>>(
      static_cast<const T*>(a->x), a->x_stride, static_cast<const T*>(a->gate), a->gate_stride,
      static_cast<const T*>(a->up), a->up_stride, a->rows, a->columns, a->width, a->activation,
      static_cast<T*>(a->y), a->y_stride, a->pre);
  return launched("gated projection");
}

template <class G>
int tiles_of(const ns_gated_args* a, dim3* grid, uint32_t* tiles_m, uint32_t* tiles_n) {
  const int64_t high = (a->rows + G::rows_m - 1) / G::rows_m;
  const int64_t wide = (a->width + G::rows_n / 2 - 1) / (G::rows_n / 2);
  if (high > INT32_MAX / 4 / wide) return fail("the projection is too large for one launch");
  *grid = dim3(static_cast<unsigned>(high * wide));
  *tiles_m = static_cast<uint32_t>(high);
  *tiles_n = static_cast<uint32_t>(wide);
  return NS_OK;
}

template <class G, class T>
int run_tiles(const ns_gated_args* a, const Rows& x, const Rows& gate, const Rows& up, int64_t pieces,
              hipStream_t stream) {
  dim3 grid;
  uint32_t tiles_m, tiles_n;
  if (int rc = tiles_of<G>(a, &grid, &tiles_m, &tiles_n)) return rc;
  gated_tiles<G, T><<<grid, dim3(G::threads), 0, stream>>>(
      x, gate, up, static_cast<uint32_t>(pieces), a->activation, static_cast<T*>(a->y), a->y_stride, a->pre,
      tiles_m, tiles_n);
  return launched("gated projection");
}

template <class G>
int run_split(const ns_gated_args* a, const Rows& x, const Rows& gate, const Rows& up, int64_t pieces,
              hipStream_t stream) {
  dim3 grid;
  uint32_t tiles_m, tiles_n;
  if (int rc = tiles_of<G>(a, &grid, &tiles_m, &tiles_n)) return rc;
  gated_split<G><<<grid, dim3(G::threads), 0, stream>>>(
      x, gate, up, static_cast<uint32_t>(pieces / (kThirds / 16)), a->activation, static_cast<float*>(a->y),
      a->y_stride, a->pre, tiles_m, tiles_n);
  return launched("gated projection");
}

template <class T>
int run(const ns_gated_args* a, hipStream_t stream) {
  if (few_rows(a)) return run_rows<T>(a, stream);
  const PackedForward w = packed_forward(a);
  auto* space = static_cast<uint8_t*>(a->workspace);
  const int64_t k = a->columns;
  Rows x = plain_rows(a->x, a->x_stride, a->rows, k, a->type);
  Rows gate = plain_rows(a->gate, a->gate_stride, a->width, k, a->type);
  Rows up = plain_rows(a->up, a->up_stride, a->width, k, a->type);
  PackJobs jobs{};
  if (w.pack_x) add_pack(&jobs, &x, a->x, a->x_stride, w.pieces, w.thirds, space + w.x);
  if (w.pack_weights) {
    add_pack(&jobs, &gate, a->gate, a->gate_stride, w.pieces, w.thirds, space + w.gate);
    add_pack(&jobs, &up, a->up, a->up_stride, w.pieces, w.thirds, space + w.up);
  }
  if (int rc = run_packs(jobs, k, w.pieces, a->type, w.thirds, stream)) return rc;
  const GemmSize size = gemm_size(a->rows, 2 * a->width, a->type, w.thirds);
  if constexpr (sizeof(T) == 4) {
    if (w.thirds)
      return size == GemmSize::kMiddle ? run_split<MiddleSplit>(a, x, gate, up, w.pieces, stream)
                                       : run_split<SmallSplit>(a, x, gate, up, w.pieces, stream);
  } else {
    if (size == GemmSize::kLarge) return run_tiles<LargeGemm, T>(a, x, gate, up, w.pieces, stream);
  }
  return size == GemmSize::kMiddle ? run_tiles<MiddleGemm, T>(a, x, gate, up, w.pieces, stream)
                                   : run_tiles<SmallGemm, T>(a, x, gate, up, w.pieces, stream);
}

}  // namespace

bool few_rows(const ns_gated_args* a) { return a->rows <= kFewRows; }

int check_gated(const ns_gated_args* a) {
  if (!a) return fail("projection arguments are required");
  if (a->rows < 0 || a->columns < 0 || a->width < 0) return fail("sizes must not be negative");
  if (a->type != NS_TYPE_F32 && a->type != NS_TYPE_BF16 && a->type != NS_TYPE_F16)
    return fail("unknown element type");
  if (a->activation != NS_GATE_SILU && a->activation != NS_GATE_GELU)
    return fail("unknown activation");
  if (a->columns > NS_GATED_MAX_COLUMNS || a->width > NS_GATED_MAX_COLUMNS ||
      a->rows > INT32_MAX)
    return fail("a gated projection takes at most %d columns each way", NS_GATED_MAX_COLUMNS);
  return NS_OK;
}

}  // namespace ns

extern "C" {

int64_t ns_gated_forward_bytes(const ns_gated_args* a) {
  ns::clear_error();
  if (ns::check_gated(a) || a->rows == 0 || a->width == 0) return 0;
  return ns::few_rows(a) ? 0 : ns::packed_forward(a).bytes;
}

int ns_gated_forward(const ns_gated_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_gated(a)) return rc;
  if (a->rows == 0 || a->width == 0) return NS_OK;
  if (!a->y || (a->columns && (!a->x || !a->gate || !a->up)))
    return ns::fail("x, the weights and the output are required");
  if (int64_t bytes = ns_gated_forward_bytes(a))
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16)
      return ns::fail("the projection needs its workspace of %lld bytes, 16-byte aligned",
                      static_cast<long long>(bytes));
  auto queue = static_cast<hipStream_t>(stream);
  if (a->type == NS_TYPE_F32) return ns::run<float>(a, queue);
  if (a->type == NS_TYPE_BF16) return ns::run<__bf16>(a, queue);
  return ns::run<_Float16>(a, queue);
}

}  // extern "C"
