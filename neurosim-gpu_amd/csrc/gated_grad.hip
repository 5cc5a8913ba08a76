// Backward of the gated projection (gfx950), with g = x gate^T, u = x up^T as the forward kept
// them in float32:
//   dg = dy u f'(g),  du = dy f(g)
//   dx = [dg du] [gate; up],  [dgate; dup] = [dg du]^T x
// The sums of dx run over columns of y, those of the weights over rows of x, and the tile
// kernels read their operands along the sum.  So dg and du, rounded once to the operands' type (the
// matrix cores multiply 16-bit numbers with 16-bit numbers; two parts of each would double the
// products), are written both ways by the pass that computes them, and x and the weights are
// transposed first: passes over memory that cost some tenth of the products: 8192 x 4096 to 8192 in bf16, products
// 755 to 850 us each (1.3 to 1.5 PFLOP/s, the matrix cores 73% busy), dg and du 267, transposes 102.
#include "ns_gated.h"

namespace ns {
namespace {

constexpr int kSide = 64;      // of a transposed tile

// The job that lane `id` of a launch belongs to; `id` becomes its place there.
__device__ __forceinline__ PackJob own_job(const PackJobs& jobs, int64_t& id) {
  PackJob own = jobs.of[0];
  int64_t before = 0;
#pragma unroll
  for (int k = 1; k < 3; ++k)
    if (k < jobs.count && id >= jobs.of[k - 1].end) {
      own = jobs.of[k];
      before = jobs.of[k - 1].end;
    }
  id -= before;
  return own;
}

// Rows as they are, zeros behind them up to whole pieces; a lane per piece.
template <class T>
__global__ __launch_bounds__(kThreads) void pack_kernel(PackJobs jobs, int64_t columns, uint32_t pieces) {
  constexpr int kValues = 16 / sizeof(T);
  int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const PackJob job = own_job(jobs, id);
  if (id >= job.rows * pieces) return;
  const int64_t row = id / pieces, first = (id - row * pieces) * kValues;
  const T* const in = static_cast<const T*>(job.from) + row * job.stride;
  Pack<T, kValues> v;
  if (first + kValues <= columns) {
    v = load_pack<T, kValues>(in + first);
  } else {
#pragma unroll
    for (int k = 0; k < kValues; ++k) v.v[k] = first + k < columns ? in[first + k] : T{};
  }
  store_pack<T, kValues>(reinterpret_cast<T*>(job.to) + id * kValues, v);
}

// float32 rows in thirds; a lane per eight columns.
__global__ __launch_bounds__(kThreads) void thirds_kernel(PackJobs jobs, int64_t columns, uint32_t blocks) {
  int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t lanes = 4 * static_cast<int64_t>(blocks);
  const PackJob job = own_job(jobs, id);
  if (id >= job.rows * lanes) return;
  const int64_t row = id / lanes, first = (id - row * lanes) * 8;
  const float* const in = static_cast<const float*>(job.from) + row * job.stride;
  float v[8];
  if (first + 8 <= columns) {
    const Pack<float, 8> all = load_pack<float, 8>(in + first);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = all.v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = first + j < columns ? in[first + j] : 0.0f;
  }
  store_thirds(job.to + row * blocks * kThirds, first, v);
}

// A square of values on its way from rows to columns: both ways eight values a lane, eight lanes to
// a line.
constexpr int kWide = 8, kSquareLanes = kSide / kWide, kLines = kThreads / kSquareLanes;
template <class T>
struct Square {
  T at[kSide][kSide + 4 / sizeof(T)];
};

// Eight values from column k on (a multiple of 8) of a laid-out row that starts at `row`: in thirds
// for float32.
template <class T>
__device__ __forceinline__ void store_laid(uint8_t* row, int64_t k, const Pack<T, kWide>& v) {
  if constexpr (sizeof(T) == 4)
    store_thirds(row, k, v.v);
  else
    *reinterpret_cast<v4i*>(row + 2 * k) = __builtin_bit_cast(v4i, v);
}

// Stores columns c0 .. of the square, of which `columns` exist, as laid-out rows of `to`, `stride`
// bytes apart, from column r0 on, up to `filled`, whole pieces.
template <class T>
__device__ __forceinline__ void store_turned(const Square<T>& square, uint8_t* to, int64_t stride,
                                             int64_t r0, int64_t filled, int64_t c0, int64_t columns) {
  const int r = threadIdx.x % kSquareLanes * kWide;
#pragma unroll
  for (int k = 0; k < kSide; k += kLines) {
    const int c = k + threadIdx.x / kSquareLanes;
    if (r0 + r >= filled || c0 + c >= columns) continue;
    Pack<T, kWide> v;
#pragma unroll
    for (int j = 0; j < kWide; ++j) v.v[j] = square.at[r + j][c];
    store_laid<T>(to + (c0 + c) * stride, r0 + r, v);
  }
}

// Laid-out rows of what are columns of `from`: value r of row c is from[r][c] for r < rows, zero for
// rows <= r < filled; rows begin at `to`, `stride` bytes apart.
struct Turn {
  const void* from;
  int64_t from_stride, rows, columns, filled;
  uint8_t* to;
  int64_t stride;
  uint32_t tiles_c, end;                   // of its workgroups, in the launch
};
// Up to three matrices in one launch.
struct Turns {
  Turn of[3];
  int count;
};
template <class T>
__global__ __launch_bounds__(kThreads) void transpose_kernel(Turns turns) {
  __shared__ Square<T> square;
  uint32_t id = blockIdx.x;
  Turn t = turns.of[0];
#pragma unroll
  for (int k = 1; k < 3; ++k)
    if (k < turns.count && blockIdx.x >= turns.of[k - 1].end) {
      t = turns.of[k];
      id = blockIdx.x - turns.of[k - 1].end;
    }
  const uint32_t tile_r = uniform(id / t.tiles_c), tile_c = id - tile_r * t.tiles_c;
  const int64_t r0 = static_cast<int64_t>(tile_r) * kSide, c0 = static_cast<int64_t>(tile_c) * kSide;
  const int side = threadIdx.x % kSquareLanes * kWide;
#pragma unroll
  for (int k = 0; k < kSide; k += kLines) {
    const int line = k + threadIdx.x / kSquareLanes;
    const int64_t r = r0 + line, left = t.columns - c0 - side;
    const T* const in = static_cast<const T*>(t.from) + r * t.from_stride + c0 + side;
    Pack<T, kWide> v{};
    if (r < t.rows && left >= kWide) {
      v = load_pack<T, kWide>(in);
    } else if (r < t.rows) {
#pragma unroll
      for (int j = 0; j < kWide; ++j)
        if (j < left) v.v[j] = in[j];
    }
#pragma unroll
    for (int j = 0; j < kWide; ++j) square.at[line][side + j] = v.v[j];
  }
  __syncthreads();
  store_turned<T>(square, t.to, t.stride, r0, t.filled, c0, t.columns);
}

// float16 holds neither a product dy u beyond 65504 nor, to all its bits, one below 2^-14, though the
// gradients that they are summed to may well be in its range.  So its dg and du are rounded as multiples
// of a power of two, one for each row of [dg du] (a row of dx) and one for each of their columns (a row
// of the weights' gradients): that which brings the largest finite one to [2^14, 2^15).  The product's
// sums are multiplied back in float32.  Where a number is still below float16's normal ones, it is off
// by at most 2^-39 of the largest.  Finding them costs a pass over what dg and du come from: a training
// pass of 8192 x 4096 to 8192 2916 -> 3107 us, of 1000 x 500 to 1000 126 -> 135.  bfloat16 has float32's
// range and needs none of this.
template <class T>
constexpr bool kRanged = __is_same(T, _Float16);

// The largest finite sizes, as bits of a float32 (whose order is theirs).
struct Extremes {
  uint32_t* row;               // [M], or NULL
  uint32_t* column;            // [2 F], or NULL
};
__device__ __forceinline__ uint32_t size_bits(float v) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu;
  return bits < 0x7F800000u ? bits : 0;
}
// 2^(14 - e) of a largest size 2^e .. 2^(e+1), at most 2^126, and its inverse.
__device__ __forceinline__ float into_range(uint32_t largest) {
  const uint32_t e = largest >> 23 < 15 ? 15 : largest >> 23;
  return __builtin_bit_cast(float, (268 - e) << 23);
}
__device__ __forceinline__ float out_of_range(uint32_t largest) {
  const uint32_t e = largest >> 23 < 15 ? 15 : largest >> 23;
  return __builtin_bit_cast(float, (e - 14) << 23);
}

// Eight neighbouring values of both products and of dy, zeros where there are none.
template <class T>
struct GateInputs {
  Pack<float, kWide> gate, raised;
  Pack<T, kWide> up;
};
template <class T>
__device__ __forceinline__ GateInputs<T> load_gate_inputs(const float* pre, const T* dy, int64_t dy_stride,
                                                          int64_t m, int64_t f, int64_t rows,
                                                          int64_t width) {
  GateInputs<T> in{};
  const int64_t plane = rows * width, left = width - f;
  if (m < rows && left >= kWide) {
    in.gate = load_pack<float, kWide>(pre + m * width + f);
    in.raised = load_pack<float, kWide>(pre + plane + m * width + f);
    in.up = load_pack<T, kWide>(dy + m * dy_stride + f);
  } else if (m < rows) {
#pragma unroll
    for (int j = 0; j < kWide; ++j) {
      if (j >= left) continue;
      in.gate.v[j] = pre[m * width + f + j];
      in.raised.v[j] = pre[plane + m * width + f + j];
      in.up.v[j] = dy[m * dy_stride + f + j];
    }
  }
  return in;
}

// dg and du of value j.
struct GateGradients {
  float gate, up;
};
template <class T>
__device__ __forceinline__ GateGradients gate_gradients_of(const GateInputs<T>& in, int j, int activation) {
  const Activation a = activated_slope(in.gate.v[j], activation);
  const float own = static_cast<float>(in.up.v[j]);
  return GateGradients{own * in.raised.v[j] * a.slope, own * a.value};
}

__global__ __launch_bounds__(kThreads) void clear_words(uint32_t* words, int64_t count) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id < count) words[id] = 0;
}

// The extremes of dg and du, a workgroup per square.  The largest of some numbers is the same in any
// order, so the atomics change no result.
template <class T>
__global__ __launch_bounds__(kThreads) void gate_extremes(const float* pre, const T* dy, int64_t dy_stride,
                                                          int64_t rows, int64_t width, int activation,
                                                          Extremes to, uint32_t tiles_f) {
  __shared__ uint32_t own[2][kSide];
  const uint32_t tile_m = uniform(blockIdx.x / tiles_f), tile_f = blockIdx.x - tile_m * tiles_f;
  const int64_t m0 = static_cast<int64_t>(tile_m) * kSide, f0 = static_cast<int64_t>(tile_f) * kSide;
  const int side = threadIdx.x % kSquareLanes * kWide;
  if (threadIdx.x < 2 * kSide) own[threadIdx.x / kSide][threadIdx.x % kSide] = 0;
  __syncthreads();
  uint32_t largest[2][kWide] = {};
#pragma unroll
  for (int k = 0; k < kSide; k += kLines) {
    const int64_t m = m0 + k + threadIdx.x / kSquareLanes;
    const GateInputs<T> in = load_gate_inputs<T>(pre, dy, dy_stride, m, f0 + side, rows, width);
    uint32_t of_row = 0;
#pragma unroll
    for (int j = 0; j < kWide; ++j) {
      const GateGradients d = gate_gradients_of<T>(in, j, activation);
      const uint32_t size[2] = {size_bits(d.gate), size_bits(d.up)};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        of_row = of_row > size[half] ? of_row : size[half];
        largest[half][j] = largest[half][j] > size[half] ? largest[half][j] : size[half];
      }
    }
#pragma unroll
    for (int step = 1; step < kSquareLanes; step *= 2) {
      const uint32_t other = __shfl_xor(of_row, step);
      of_row = of_row > other ? of_row : other;
    }
    if (to.row && m < rows && threadIdx.x % kSquareLanes == 0) atomicMax(to.row + m, of_row);
  }
  if (!to.column) return;
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int j = 0; j < kWide; ++j) atomicMax(&own[half][side + j], largest[half][j]);
  __syncthreads();
  const int half = threadIdx.x / kSide;
  const int64_t f = f0 + threadIdx.x % kSide;
  if (half < 2 && f < width) atomicMax(to.column + half * width + f, own[half][threadIdx.x % kSide]);
}

// dg and du: as laid-out rows [M][2 F'], du behind dg, and as columns [2 F][M'], each padded with
// zeros to whole pieces (F', M').
template <class T>
__global__ __launch_bounds__(kThreads) void gate_gradients(const float* pre, const T* dy, int64_t dy_stride,
                                                           int64_t rows, int64_t width, int activation,
                                                           uint8_t* by_row, int64_t row_half,
                                                           int64_t row_stride, uint8_t* by_column,
                                                           int64_t filled, int64_t column_stride,
                                                           Extremes extremes, uint32_t tiles_f) {
  __shared__ Square<T> square[2];
  const uint32_t tile_m = uniform(blockIdx.x / tiles_f), tile_f = blockIdx.x - tile_m * tiles_f;
  const int64_t m0 = static_cast<int64_t>(tile_m) * kSide, f0 = static_cast<int64_t>(tile_f) * kSide;
  const int side = threadIdx.x % kSquareLanes * kWide;
  const int64_t f = f0 + side;
  float of_column[2][kWide];
  if constexpr (kRanged<T>) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int j = 0; j < kWide; ++j)
        of_column[half][j] =
            into_range(by_column && f + j < width ? extremes.column[half * width + f + j] : 0);
  }
#pragma unroll
  for (int k = 0; k < kSide; k += kLines) {
    const int line = k + threadIdx.x / kSquareLanes;
    const int64_t m = m0 + line;
    const GateInputs<T> in = load_gate_inputs<T>(pre, dy, dy_stride, m, f, rows, width);
    float of_row = 1.0f;
    if constexpr (kRanged<T>) of_row = into_range(by_row && m < rows ? extremes.row[m] : 0);
    Pack<T, kWide> g, u;
#pragma unroll
    for (int j = 0; j < kWide; ++j) {
      // Zeros where there is nothing: rows and columns of padding stay zero.
      const GateGradients d = gate_gradients_of<T>(in, j, activation);
      if constexpr (kRanged<T>) {
        g.v[j] = static_cast<T>(d.gate * of_row);
        u.v[j] = static_cast<T>(d.up * of_row);
        square[0].at[line][side + j] = static_cast<T>(d.gate * of_column[0][j]);
        square[1].at[line][side + j] = static_cast<T>(d.up * of_column[1][j]);
      } else {
        g.v[j] = static_cast<T>(d.gate);
        u.v[j] = static_cast<T>(d.up);
        square[0].at[line][side + j] = g.v[j];
        square[1].at[line][side + j] = u.v[j];
      }
    }
    if (by_row && m < rows && f < row_half) {
      store_laid<T>(by_row + m * row_stride, f, g);
      store_laid<T>(by_row + m * row_stride, row_half + f, u);
    }
  }
  if (!by_column) return;
  __syncthreads();
  store_turned<T>(square[0], by_column, column_stride, m0, filled, f0, width);
  store_turned<T>(square[1], by_column + width * column_stride, column_stride, m0, filled, f0, width);
}

// out = a b^T, one workgroup per tile; kRanged types have a's rows' largest sizes and undo their factors.
template <class G, class T>
__global__ __launch_bounds__(G::threads, 512 / G::threads) void gemm_tiles(Rows a, Rows b, uint32_t pieces, T* out,
                                                         int64_t stride, const uint32_t* largest,
                                                         uint32_t tiles_m, uint32_t tiles_n) {
  __shared__ union {
    v4i stages[G::stages * G::rows * 8];
    Strip<G, T> strip[G::WM * G::WN];
  } lds;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const TilePlace tile = tile_place(tiles_m, tiles_n);
  const int64_t m0 = static_cast<int64_t>(tile.m) * G::rows_m;
  const int64_t n0 = static_cast<int64_t>(tile.n) * G::rows_n;
  GemmPlace p;
  p.lane = lane;
  p.wave = wave;
  p.stride_a = static_cast<uint32_t>(a.stride);
  p.stride_b = static_cast<uint32_t>(b.stride);
  p.pieces = pieces;
  p.a = rows_buffer(a, m0, G::rows_m, pieces);
  const Second<false> second{{rows_buffer(b, n0, G::rows_n, pieces)}, {}};
  v4f sum[G::MI][G::NJ] = {};
  gemm_tile<G, T, false>(p, second, lds.stages, sum);
  const int64_t m = m0 + 16 * (wave / G::WN) * G::MI, n = n0 + 16 * (wave % G::WN) * G::NJ;
  if constexpr (kRanged<T>) {
#pragma unroll
    for (int i = 0; i < G::MI; ++i) {
      const int64_t row = m + 16 * i + (lane & 15);
      const float back = out_of_range(row < a.rows ? largest[row] : 0);
#pragma unroll
      for (int j = 0; j < G::NJ; ++j) sum[i][j] *= back;
    }
  }
  store_tiles<G, T, false>(out + m * stride + n, stride, sum, nullptr, a.rows - m, b.rows - n, lane,
                           lds.strip[wave]);
}

// The same for float32 rows in thirds.
template <class G>
__global__ __launch_bounds__(G::threads) void split_tiles(Rows a, Rows b, uint32_t blocks, float* out,
                                                          int64_t stride, uint32_t tiles_m,
                                                          uint32_t tiles_n) {
  __shared__ union {
    uint8_t stages[G::stages * G::stage_bytes];
    Strip<G, float> strip[G::waves];
    v4i aligned;
  } lds;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const TilePlace tile = tile_place(tiles_m, tiles_n);
  const int64_t m0 = static_cast<int64_t>(tile.m) * G::rows_m;
  const int64_t n0 = static_cast<int64_t>(tile.n) * G::rows_n;
  const uint32_t pieces = blocks * (kThirds / 16);
  const v4i second = rows_buffer(b, n0, G::rows_n, pieces);
  const SplitPlace<G> p = split_place<G, false>(lane, wave, blocks, rows_buffer(a, m0, G::rows_m, pieces),
                                                static_cast<uint32_t>(a.stride), second, second,
                                                static_cast<uint32_t>(b.stride));
  v4f sum[G::MI][G::NJ] = {};
  split_tile<G>(p, lds.stages, sum);
  const int64_t m = m0 + 16 * (wave / G::WN) * G::MI, n = n0 + 16 * (wave % G::WN) * G::NJ;
  store_tiles<G, float, false>(out + m * stride + n, stride, sum, nullptr, a.rows - m, b.rows - n, lane,
                               lds.strip[wave]);
}

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

int tile_grid(int64_t tiles_m, int64_t tiles_n, dim3* grid) {
  if (tiles_n < 1 || tiles_m > INT32_MAX / 4 / tiles_n)
    return fail("the projection is too large for one launch");
  *grid = dim3(static_cast<unsigned>(tiles_m * tiles_n));
  return NS_OK;
}

int add_turn(Turns* turns, const void* from, int64_t from_stride, int64_t rows, int64_t columns, int64_t filled,
             uint8_t* to, int64_t stride) {
  const int64_t tiles_r = (filled + kSide - 1) / kSide, tiles_c = (columns + kSide - 1) / kSide;
  const uint32_t before = turns->count ? turns->of[turns->count - 1].end : 0;
  dim3 grid;
  if (int rc = tile_grid(tiles_r, tiles_c, &grid)) return rc;   // a quarter of 2^31 at most, each
  turns->of[turns->count++] = Turn{from, from_stride, rows, columns, filled, to, stride,
                                   static_cast<uint32_t>(tiles_c), before + grid.x};
  return NS_OK;
}

template <class T>
int run_turns(const Turns& turns, hipStream_t stream) {
  transpose_kernel<T><<<dim3(turns.of[turns.count - 1].end), dim3(kThreads), 0, stream>>>(turns);
  return launched("transposition");
}

template <class G, class T>
int product_of(const Rows& a, const Rows& b, int64_t pieces, T* out, int64_t stride, const uint32_t* largest,
               hipStream_t stream) {
  const int64_t tiles_m = (a.rows + G::rows_m - 1) / G::rows_m;
  const int64_t tiles_n = (b.rows + G::rows_n - 1) / G::rows_n;
  const auto count_m = static_cast<uint32_t>(tiles_m), count_n = static_cast<uint32_t>(tiles_n);
  dim3 grid;
  if (int rc = tile_grid(tiles_m, tiles_n, &grid)) return rc;
  if constexpr (sizeof(T) == 4)
    split_tiles<G><<<grid, dim3(G::threads), 0, stream>>>(
        a, b, static_cast<uint32_t>(pieces / (kThirds / 16)), out, stride, count_m, count_n);
  else
    gemm_tiles<G, T><<<grid, dim3(G::threads), 0, stream>>>(a, b, static_cast<uint32_t>(pieces), out, stride,
                                                            largest, count_m, count_n);
  return launched("product");
}

template <class T>
int product(const Rows& a, const Rows& b, int64_t pieces, int32_t type, T* out, int64_t stride,
            const uint32_t* largest, hipStream_t stream) {
  const GemmSize size = gemm_size(a.rows, b.rows, type, sizeof(T) == 4);
  if constexpr (sizeof(T) == 4) {
    return size == GemmSize::kMiddle ? product_of<MiddleSplit, T>(a, b, pieces, out, stride, largest, stream)
                                     : product_of<SmallSplit, T>(a, b, pieces, out, stride, largest, stream);
  } else {
    switch (size) {
      case GemmSize::kLarge: return product_of<LargeGemm, T>(a, b, pieces, out, stride, largest, stream);
      case GemmSize::kMiddle: return product_of<MiddleGemm, T>(a, b, pieces, out, stride, largest, stream);
      default: return product_of<SmallGemm, T>(a, b, pieces, out, stride, largest, stream);
    }
  }
}

// The backward's workspace: dg and du as laid-out rows of 2 F' values and as columns of M', the
// weights transposed (rows of 2 F'), x transposed (rows of M'), and for float16 the largest sizes of
// dg's and du's rows and columns.
struct BackwardSpace {
  int64_t half, filled;                    // F' and M'
  int64_t row_bytes, column_bytes;         // of rows of 2 F', and of M'
  int64_t by_column, weights, x, extremes, bytes;
  int64_t row_extremes, column_extremes;   // how many
};
BackwardSpace backward_space(const ns_gated_args* a) {
  BackwardSpace w{};
  const bool thirds = a->type == NS_TYPE_F32;
  w.half = whole_values(a->width, thirds);
  w.filled = whole_values(a->rows, thirds);
  w.row_bytes = pieces_of(2 * w.half, a->type, thirds) * 16;
  w.column_bytes = pieces_of(w.filled, a->type, thirds) * 16;
  w.by_column = a->dx ? a->rows * w.row_bytes : 0;
  w.weights = w.by_column + (a->dweights ? 2 * a->width * w.column_bytes : 0);
  w.x = w.weights + (a->dx ? a->columns * w.row_bytes : 0);
  w.extremes = w.x + (a->dweights ? a->columns * w.column_bytes : 0);
  const bool ranged = a->type == NS_TYPE_F16;
  w.row_extremes = ranged && a->dx ? a->rows : 0;
  w.column_extremes = ranged && a->dweights ? 2 * a->width : 0;
  w.bytes = w.extremes + 4 * (w.row_extremes + w.column_extremes);
  return w;
}

template <class T>
int run_backward(const ns_gated_args* a, hipStream_t stream) {
  const BackwardSpace w = backward_space(a);
  auto* const space = static_cast<uint8_t*>(a->workspace);
  uint8_t* const by_row = a->dx ? space : nullptr;
  uint8_t* const by_column = a->dweights ? space + w.by_column : nullptr;
  uint8_t* const weights = space + w.weights;
  uint8_t* const x = space + w.x;
  const int64_t tiles_m = (w.filled + kSide - 1) / kSide, tiles_f = (w.half + kSide - 1) / kSide;
  dim3 grid;
  if (int rc = tile_grid(tiles_m, tiles_f, &grid)) return rc;
  Extremes extremes{};
  if constexpr (kRanged<T>) {
    auto* const words = reinterpret_cast<uint32_t*>(space + w.extremes);
    const int64_t count = w.row_extremes + w.column_extremes;      // 2^22 at most
    extremes = Extremes{by_row ? words : nullptr, by_column ? words + w.row_extremes : nullptr};
    clear_words<<<dim3(static_cast<unsigned>((count + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream>>>(
        words, count);
    if (int rc = launched("gate gradients' range")) return rc;
    gate_extremes<T><<<grid, dim3(kThreads), 0, stream>>>(
        a->pre, static_cast<const T*>(a->dy), a->dy_stride, a->rows, a->width, a->activation, extremes,
        static_cast<uint32_t>(tiles_f));
    if (int rc = launched("gate gradients' range")) return rc;
  }
  gate_gradients<T><<<grid, dim3(kThreads), 0, stream>>>(
      a->pre, static_cast<const T*>(a->dy), a->dy_stride, a->rows, a->width, a->activation, by_row, w.half,
      w.row_bytes, by_column, w.filled, w.column_bytes, extremes, static_cast<uint32_t>(tiles_f));
  if (int rc = launched("gate gradients")) return rc;
  // Small calls pay by the launch, so x is turned with the weights; a large one is turned when its
  // product is next, from whose caches it then comes.  Us, all at once / x later: 1000 x 500 to 1000 in
  // float32 117 / 121, 3885 x 1031 to 1500 517 / 515, 8192 x 4096 to 8192 in bf16 2862 / 2820.
  constexpr int64_t kSmall = 8 << 20;
  const bool together = a->rows * a->columns * type_size(a->type) <= kSmall;
  Turns turns{};
  if (a->dx) {
    if (int rc = add_turn(&turns, a->gate, a->gate_stride, a->width, a->columns, w.half, weights, w.row_bytes))
      return rc;
    if (int rc = add_turn(&turns, a->up, a->up_stride, a->width, a->columns, w.half, weights + w.row_bytes / 2,
                          w.row_bytes))
      return rc;
    if (a->dweights && together)
      if (int rc = add_turn(&turns, a->x, a->x_stride, a->rows, a->columns, w.filled, x, w.column_bytes)) return rc;
    if (int rc = run_turns<T>(turns, stream)) return rc;
    const Rows left{by_row, w.row_bytes, a->rows}, right{weights, w.row_bytes, a->columns};
    if (int rc = product<T>(left, right, w.row_bytes / 16, a->type, static_cast<T*>(a->dx), a->columns,
                            extremes.row, stream))
      return rc;
  }
  if (a->dweights) {
    if (!a->dx || !together) {
      turns.count = 0;
      if (int rc = add_turn(&turns, a->x, a->x_stride, a->rows, a->columns, w.filled, x, w.column_bytes)) return rc;
      if (int rc = run_turns<T>(turns, stream)) return rc;
    }
    const Rows left{by_column, w.column_bytes, 2 * a->width}, right{x, w.column_bytes, a->columns};
    return product<T>(left, right, w.column_bytes / 16, a->type, static_cast<T*>(a->dweights), a->columns,
                      extremes.column, stream);
  }
  return NS_OK;
}

}  // namespace

void add_pack(PackJobs* jobs, Rows* rows, const void* data, int64_t stride, int64_t pieces, bool thirds,
              uint8_t* to) {
  const int64_t lanes = thirds ? pieces / (kThirds / 16) * 4 : pieces;     // of a row
  const int64_t before = jobs->count ? jobs->of[jobs->count - 1].end : 0;
  jobs->of[jobs->count++] = PackJob{data, stride, rows->rows, to, before + rows->rows * lanes};
  rows->data = to;
  rows->stride = pieces * 16;
}

int run_packs(const PackJobs& jobs, int64_t columns, int64_t pieces, int32_t type, bool thirds,
              hipStream_t stream) {
  const int64_t lanes = jobs.count ? jobs.of[jobs.count - 1].end : 0, groups = (lanes + kThreads - 1) / kThreads;
  if (groups == 0) return NS_OK;
  if (groups > INT32_MAX) return fail("the projection is too large for one launch");
  const dim3 grid(static_cast<unsigned>(groups)), threads(kThreads);
  if (thirds)
    thirds_kernel<<<grid, threads, 0, stream>>>(jobs, columns, static_cast<uint32_t>(pieces / (kThirds / 16)));
  else if (type == NS_TYPE_F32)
    pack_kernel<float><<<grid, threads, 0, stream>>>(jobs, columns, static_cast<uint32_t>(pieces));
  else
    pack_kernel<_Float16><<<grid, threads, 0, stream>>>(jobs, columns, static_cast<uint32_t>(pieces));
  return launched("rows' layout");
}

// The size whose rounds of tiles over the 256 compute units take the least time.  In units of 0.1
// us for 32 stages (2048 columns of 16 bits): a round of large tiles 45 to 51 us; of middle ones
// 16.2 with two on a compute unit and 24 alone; of small ones 6.2 where there are many, 22 with
// two on a compute unit and 14 alone, where a stage's way from memory to LDS takes longer than its
// products.  float32 in thirds, 32 columns at a time, is bound by its products, and tiles alone
// count: 34 and 12.9 for 32 stages of 32 columns; as it is, at a sixteenth of bfloat16's rate, 60 and
// 15.7.  us, small / middle / large, of M x K to F in bf16: 64 x 4096 to 8192
// 28.8 / 58.8 / 91; 256 x 1024 to 4096 9.9 / 13.2 / 23.5; 512 x 4096 to 4096 50 / 41.8 / 72.6; 2048^3
// 51 / 32.4 / 40.6; 3000 x 700 to 5000 89 / 68 / 61; 4096^3 406 / 259 / 205; in float32 3885 x 1031 to
// 1500 248 / 233.
GemmSize gemm_size(int64_t m, int64_t n, int32_t type, bool thirds) {
  const auto tiles = [=](int64_t side) { return (m + side - 1) / side * ((n + side - 1) / side); };
  const auto rounds = [](int64_t count, int64_t at_once) { return (count + at_once - 1) / at_once; };
  const int64_t few = tiles(64), some = tiles(128);
  if (type == NS_TYPE_F32) {
    const int64_t middle = (thirds ? 340 : 600) * rounds(some, 256);
    return middle <= (thirds ? 129 : 157) * rounds(few, 256) ? GemmSize::kMiddle : GemmSize::kSmall;
  }
  const auto most = [](int64_t a, int64_t b) { return a > b ? a : b; };
  const int64_t small = most(few <= 256 ? 140 : 220, 62 * rounds(few, 256));
  const int64_t middle = most(240 * rounds(some, 512), 162 * rounds(some, 256));
  const int64_t large = 450 * rounds(tiles(256), 256);
  if (large <= middle && large <= small) return GemmSize::kLarge;
  return middle <= small ? GemmSize::kMiddle : GemmSize::kSmall;
}

}  // namespace ns

extern "C" {

int64_t ns_gated_backward_bytes(const ns_gated_args* a) {
  ns::clear_error();
  if (ns::check_gated(a) || a->rows == 0 || a->width == 0 || a->columns == 0) return 0;
  return ns::backward_space(a).bytes;
}

int ns_gated_backward(const ns_gated_args* a, void* stream) {
  ns::clear_error();
  if (int rc = ns::check_gated(a)) return rc;
  if (a->rows > NS_GATED_MAX_ROWS)
    return ns::fail("a backward takes at most %d rows", NS_GATED_MAX_ROWS);
  if (a->rows == 0 || a->width == 0 || a->columns == 0)
    return ns::fail("a backward has at least one row, column and result");
  if (!a->dx && !a->dweights) return NS_OK;
  if (!a->pre || !a->dy || !a->x || !a->gate || !a->up)
    return ns::fail("the forward's sums, dy, x and the weights are required");
  if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16)
    return ns::fail("the backward needs its workspace, 16-byte aligned");
  auto queue = static_cast<hipStream_t>(stream);
  if (a->type == NS_TYPE_F32) return ns::run_backward<float>(a, queue);
  if (a->type == NS_TYPE_BF16) return ns::run_backward<__bf16>(a, queue);
  return ns::run_backward<_Float16>(a, queue);
}

}  // extern "C"
