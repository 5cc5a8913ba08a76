// Backward of the gated projection (gfx950), with g = x gate^T, u = x up^T as the forward kept
// them in float32:
//   dg = dy u f'(g),  du = dy f(g)
//   dx = [dg du] [gate; up],  [dgate; dup] = [dg du]^T x
// The sums of dx run over columns of y, those of the weights over rows of x, and the tile
// kernels read their operands along the sum.  So dg and du, rounded once, are written both
// ways by the pass that computes them, and x and the weights are transposed first: passes
// over memory that cost some tenth of the products.
#include "ns_gated.h"

namespace ns {
namespace {

constexpr int kSide = 64;      // of a transposed tile

// Rows as they are, zeros behind them up to whole pieces; a lane per piece.
template <class T>
__global__ __launch_bounds__(kThreads) void pack_kernel(const T* from, int64_t stride, int64_t rows,
                                                        int64_t columns, uint32_t pieces, T* to) {
  constexpr int kValues = 16 / sizeof(T);
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= rows * pieces) return;
  const int64_t row = id / pieces, first = (id - row * pieces) * kValues;
  const T* const in = from + row * stride;
  Pack<T, kValues> v;
  if (first + kValues <= columns) {
    v = load_pack<T, kValues>(in + first);
  } else {
#pragma unroll
    for (int k = 0; k < kValues; ++k) v.v[k] = first + k < columns ? in[first + k] : T{};
  }
  store_pack<T, kValues>(to + id * kValues, v);
}

// A square of values on its way from rows to columns: both ways in 16-byte pieces, eight (of
// float32 sixteen) lanes to a line.
template <class T>
struct Square {
  static constexpr int V = 16 / sizeof(T), lanes = kSide / V, lines = kThreads / lanes;
  T at[kSide][kSide + 4 / sizeof(T)];
};

// Stores columns c0 .. of the square, of which `columns` exist, as rows of `to` from r0 on, up to
// `filled`, whole pieces.
template <class T>
__device__ __forceinline__ void store_turned(const Square<T>& square, T* to, int64_t stride, int64_t r0,
                                             int64_t filled, int64_t c0, int64_t columns) {
  using S = Square<T>;
  const int r = threadIdx.x % S::lanes * S::V;
#pragma unroll
  for (int k = 0; k < kSide; k += S::lines) {
    const int c = k + threadIdx.x / S::lanes;
    if (r0 + r >= filled || c0 + c >= columns) continue;
    Pack<T, S::V> v;
#pragma unroll
    for (int j = 0; j < S::V; ++j) v.v[j] = square.at[r + j][c];
    store_pack<T, S::V>(to + (c0 + c) * stride + r0 + r, v);
  }
}

// to[c][r] = from[r][c] for r < rows, c < columns, and zeros for rows <= r < filled.
template <class T>
__global__ __launch_bounds__(kThreads) void transpose_kernel(const T* from, int64_t stride, int64_t rows,
                                                             int64_t columns, int64_t filled, T* to,
                                                             int64_t to_stride, uint32_t tiles_c) {
  using S = Square<T>;
  __shared__ S square;
  const uint32_t tile_r = uniform(blockIdx.x / tiles_c), tile_c = blockIdx.x - tile_r * tiles_c;
  const int64_t r0 = static_cast<int64_t>(tile_r) * kSide, c0 = static_cast<int64_t>(tile_c) * kSide;
  const int side = threadIdx.x % S::lanes * S::V;
#pragma unroll
  for (int k = 0; k < kSide; k += S::lines) {
    const int line = k + threadIdx.x / S::lanes;
    const int64_t r = r0 + line, left = columns - c0 - side;
    const T* const in = from + r * stride + c0 + side;
    Pack<T, S::V> v{};
    if (r < rows && left >= S::V) {
      v = load_pack<T, S::V>(in);
    } else if (r < rows) {
#pragma unroll
      for (int j = 0; j < S::V; ++j)
        if (j < left) v.v[j] = in[j];
    }
#pragma unroll
    for (int j = 0; j < S::V; ++j) square.at[line][side + j] = v.v[j];
  }
  __syncthreads();
  store_turned<T>(square, to, to_stride, r0, filled, c0, columns);
}

// dg and du: as rows [M][2 F'], du behind dg, and as columns [2 F][M'], each padded with zeros to
// whole pieces (F', M').
template <class T>
__global__ __launch_bounds__(kThreads) void gate_gradients(const float* pre, const T* dy, int64_t dy_stride,
                                                           int64_t rows, int64_t width, int activation,
                                                           T* by_row, int64_t row_half, T* by_column,
                                                           int64_t filled, uint32_t tiles_f) {
  using S = Square<T>;
  __shared__ S square[2];
  const uint32_t tile_m = uniform(blockIdx.x / tiles_f), tile_f = blockIdx.x - tile_m * tiles_f;
  const int64_t m0 = static_cast<int64_t>(tile_m) * kSide, f0 = static_cast<int64_t>(tile_f) * kSide;
  const int side = threadIdx.x % S::lanes * S::V;
  const int64_t plane = rows * width, f = f0 + side, left = width - f;
#pragma unroll
  for (int k = 0; k < kSide; k += S::lines) {
    const int line = k + threadIdx.x / S::lanes;
    const int64_t m = m0 + line;
    Pack<float, S::V> gate{}, raised{};
    Pack<T, S::V> up{}, g, u;
    if (m < rows && left >= S::V) {
      gate = load_pack<float, S::V>(pre + m * width + f);
      raised = load_pack<float, S::V>(pre + plane + m * width + f);
      up = load_pack<T, S::V>(dy + m * dy_stride + f);
    } else if (m < rows) {
#pragma unroll
      for (int j = 0; j < S::V; ++j) {
        if (j >= left) continue;
        gate.v[j] = pre[m * width + f + j];
        raised.v[j] = pre[plane + m * width + f + j];
        up.v[j] = dy[m * dy_stride + f + j];
      }
    }
#pragma unroll
    for (int j = 0; j < S::V; ++j) {
      // Zeros where there is nothing: rows and columns of padding stay zero.
      const Activation a = activated_slope(gate.v[j], activation);
      const float own = static_cast<float>(up.v[j]);
      g.v[j] = static_cast<T>(own * raised.v[j] * a.slope);
      u.v[j] = static_cast<T>(own * a.value);
      square[0].at[line][side + j] = g.v[j];
      square[1].at[line][side + j] = u.v[j];
    }
    if (by_row && m < rows && f < row_half) {
      store_pack<T, S::V>(by_row + m * 2 * row_half + f, g);
      store_pack<T, S::V>(by_row + m * 2 * row_half + row_half + f, u);
    }
  }
  if (!by_column) return;
  __syncthreads();
  store_turned<T>(square[0], by_column, filled, m0, filled, f0, width);
  store_turned<T>(square[1], by_column + width * filled, filled, m0, filled, f0, width);
}

// out = a b^T, one workgroup per tile.
template <class G, class T>
__global__ __launch_bounds__(G::threads, 512 / G::threads) void gemm_tiles(Rows a, Rows b, uint32_t pieces, T* out,
                                                         int64_t stride, uint32_t tiles_m,
                                                         uint32_t tiles_n) {
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
  store_tiles<G, T, false>(out + m * stride + n, stride, sum, nullptr, a.rows - m, b.rows - n, lane,
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

template <class T>
int transpose(const void* from, int64_t stride, int64_t rows, int64_t columns, int64_t filled, T* to,
              int64_t to_stride, hipStream_t stream) {
  const int64_t tiles_r = (filled + kSide - 1) / kSide, tiles_c = (columns + kSide - 1) / kSide;
  dim3 grid;
  if (int rc = tile_grid(tiles_r, tiles_c, &grid)) return rc;
  transpose_kernel<T><<<grid, dim3(kThreads), 0, stream>>>(static_cast<const T*>(from), stride, rows,
                                                           columns, filled, to, to_stride,
                                                           static_cast<uint32_t>(tiles_c));
  return launched("transposition");
}

template <class G, class T>
int product_of(const Rows& a, const Rows& b, int64_t pieces, T* out, int64_t stride, hipStream_t stream) {
  const int64_t tiles_m = (a.rows + G::rows_m - 1) / G::rows_m;
  const int64_t tiles_n = (b.rows + G::rows_n - 1) / G::rows_n;
  dim3 grid;
  if (int rc = tile_grid(tiles_m, tiles_n, &grid)) return rc;
  gemm_tiles<G, T><<<grid, dim3(G::threads), 0, stream>>>(a, b, static_cast<uint32_t>(pieces), out,
                                                          stride, static_cast<uint32_t>(tiles_m),
                                                          static_cast<uint32_t>(tiles_n));
  return launched("product");
}

template <class T>
int product(const Rows& a, const Rows& b, int64_t pieces, int32_t type, T* out, int64_t stride,
            hipStream_t stream) {
  switch (gemm_size(a.rows, b.rows, type)) {
    case GemmSize::kLarge:
      if constexpr (sizeof(T) == 2) return product_of<LargeGemm, T>(a, b, pieces, out, stride, stream);
      [[fallthrough]];
    case GemmSize::kMiddle: return product_of<MiddleGemm, T>(a, b, pieces, out, stride, stream);
    default: return product_of<SmallGemm, T>(a, b, pieces, out, stride, stream);
  }
}

// The backward's workspace.
struct BackwardSpace {
  int64_t half, filled;                    // F' and M'
  int64_t by_row, by_column, weights, x, bytes;
};
BackwardSpace backward_space(const ns_gated_args* a) {
  BackwardSpace w{};
  const int64_t e = type_size(a->type);
  w.half = whole_values(a->width, a->type);
  w.filled = whole_values(a->rows, a->type);
  w.by_column = a->dx ? a->rows * 2 * w.half * e : 0;
  w.weights = w.by_column + (a->dweights ? 2 * a->width * w.filled * e : 0);
  w.x = w.weights + (a->dx ? a->columns * 2 * w.half * e : 0);
  w.bytes = w.x + (a->dweights ? a->columns * w.filled * e : 0);
  return w;
}

template <class T>
int run_backward(const ns_gated_args* a, hipStream_t stream) {
  const BackwardSpace w = backward_space(a);
  auto* space = static_cast<uint8_t*>(a->workspace);
  T* const by_row = a->dx ? reinterpret_cast<T*>(space + w.by_row) : nullptr;
  T* const by_column = a->dweights ? reinterpret_cast<T*>(space + w.by_column) : nullptr;
  T* const weights = reinterpret_cast<T*>(space + w.weights);
  T* const x = reinterpret_cast<T*>(space + w.x);
  const int64_t e = sizeof(T), tiles_m = (w.filled + kSide - 1) / kSide;
  const int64_t tiles_f = (w.half + kSide - 1) / kSide;
  dim3 grid;
  if (int rc = tile_grid(tiles_m, tiles_f, &grid)) return rc;
  gate_gradients<T><<<grid, dim3(kThreads), 0, stream>>>(
      a->pre, static_cast<const T*>(a->dy), a->dy_stride, a->rows, a->width, a->activation, by_row,
      w.half, by_column, w.filled, static_cast<uint32_t>(tiles_f));
  if (int rc = launched("gate gradients")) return rc;
  if (a->dx) {
    if (int rc = transpose<T>(a->gate, a->gate_stride, a->width, a->columns, w.half, weights, 2 * w.half,
                              stream))
      return rc;
    if (int rc = transpose<T>(a->up, a->up_stride, a->width, a->columns, w.half, weights + w.half,
                              2 * w.half, stream))
      return rc;
    const Rows left{reinterpret_cast<const uint8_t*>(by_row), 2 * w.half * e, a->rows};
    const Rows right{reinterpret_cast<const uint8_t*>(weights), 2 * w.half * e, a->columns};
    if (int rc = product<T>(left, right, 2 * w.half * e / 16, a->type, static_cast<T*>(a->dx), a->columns,
                            stream))
      return rc;
  }
  if (a->dweights) {
    if (int rc = transpose<T>(a->x, a->x_stride, a->rows, a->columns, w.filled, x, w.filled, stream))
      return rc;
    const Rows left{reinterpret_cast<const uint8_t*>(by_column), w.filled * e, 2 * a->width};
    const Rows right{reinterpret_cast<const uint8_t*>(x), w.filled * e, a->columns};
    return product<T>(left, right, w.filled * e / 16, a->type, static_cast<T*>(a->dweights), a->columns,
                      stream);
  }
  return NS_OK;
}

template <class T>
int run_pack(Rows* rows, const void* data, int64_t stride, int64_t columns, int64_t pieces, uint8_t* to,
             hipStream_t stream) {
  const int64_t groups = (rows->rows * pieces + kThreads - 1) / kThreads;
  if (groups > INT32_MAX) return fail("the projection is too large for one launch");
  pack_kernel<T><<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, stream>>>(
      static_cast<const T*>(data), stride, rows->rows, columns, static_cast<uint32_t>(pieces),
      reinterpret_cast<T*>(to));
  rows->data = to;
  rows->stride = pieces * 16;
  return launched("rows' layout");
}

}  // namespace

int pack_rows(Rows* rows, const void* data, int64_t stride, int64_t columns, int32_t type, uint8_t* to,
              hipStream_t stream) {
  const int64_t pieces = pieces_of(columns, type);
  if (pieces == 0) return NS_OK;
  return type == NS_TYPE_F32 ? run_pack<float>(rows, data, stride, columns, pieces, to, stream)
                             : run_pack<_Float16>(rows, data, stride, columns, pieces, to, stream);
}

// The size whose rounds of tiles over the 256 compute units take the least time.  In units of 0.1
// us for 32 stages (2048 columns of 16 bits): a round of large tiles 45 to 51 us; of middle ones
// 16.2 with two on a compute unit and 24 alone; of small ones 6.2 where there are many, 22 with
// two on a compute unit and 14 alone, where a stage's way from memory to LDS takes longer than its
// products.  float32 multiplies at a sixteenth of the rate, so tiles alone count: 60 and 15.7, and
// large ones gain nothing.  us, small / middle / large, of M x K to F in bf16: 64 x 4096 to 8192
// 28.8 / 58.8 / 91; 256 x 1024 to 4096 9.9 / 13.2 / 23.5; 512 x 4096 to 4096 50 / 41.8 / 72.6; 2048^3
// 51 / 32.4 / 40.6; 3000 x 700 to 5000 89 / 68 / 61; 4096^3 406 / 259 / 205; in float32 3885 x 1031 to
// 1500 248 / 233.
GemmSize gemm_size(int64_t m, int64_t n, int32_t type) {
  const auto tiles = [=](int64_t side) { return (m + side - 1) / side * ((n + side - 1) / side); };
  const auto rounds = [](int64_t count, int64_t at_once) { return (count + at_once - 1) / at_once; };
  const int64_t few = tiles(64), some = tiles(128);
  if (type == NS_TYPE_F32)
    return 600 * rounds(some, 256) <= 157 * rounds(few, 256) ? GemmSize::kMiddle : GemmSize::kSmall;
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
