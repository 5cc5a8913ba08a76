// Product of two microscaled 4-bit matrices, y = a b^T + bias (gfx950).
//
// The matrix cores take e2m1 codes and block scales as they are stored: in
// mfma_scale 16x16x128, lane l holds row l%16 of an operand, block l/16 of four (16 bytes
// of codes, one scale byte), so a lane's operand is one 16-byte load; the 16x16 result has
// column l%16 and rows 4*(l/16) .. +3 in lane l's four registers.
#include "ns_signal.h"
#include "neurosim_hip_mx.h"

namespace ns {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));

struct MxView {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t rows, blocks;
};

struct MxOperand {
  v4i codes;
  int scale;
};

// Block `block` of row `row` (past the matrix: zeros, scale 1).
__device__ __forceinline__ MxOperand load_block(const MxView& m, int64_t row, int64_t block,
                                                int64_t stop) {
  MxOperand o{{0, 0, 0, 0}, 127};
  if (row < m.rows && block < stop) {
    o.codes = *reinterpret_cast<const v4i*>(m.codes + (row * m.blocks + block) * 16);
    o.scale = m.scales[row * m.blocks + block];
  }
  return o;
}

__device__ __forceinline__ v4f mx_mfma(const MxOperand& a, const MxOperand& b, v4f c) {
  const v8i wide_a = {a.codes[0], a.codes[1], a.codes[2], a.codes[3], 0, 0, 0, 0};
  const v8i wide_b = {b.codes[0], b.codes[1], b.codes[2], b.codes[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide_a, wide_b, c, 4, 4, 0, a.scale, 0,
                                                          b.scale);
}

// One wavefront per 32x32 tile and part of K.
template <class T>
__global__ __launch_bounds__(kThreads) void product_tiles(MxView a, MxView b, const float* bias,
                                                          T* out, int64_t stride, int64_t tiles_n,
                                                          int64_t tiles, int64_t splits,
                                                          float* partials) {
  const int lane = threadIdx.x & 63;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
  if (id >= tiles * splits) return;
  const int64_t split = id / tiles, tile = id - split * tiles;
  const int64_t m0 = tile / tiles_n * 32, n0 = tile % tiles_n * 32;
  const int64_t steps = (a.blocks + 3) / 4, per = (steps + splits - 1) / splits;
  const int64_t first = split * per * 4;
  int64_t stop = first + per * 4;
  stop = stop < a.blocks ? stop : a.blocks;
  v4f sum[2][2] = {};
  for (int64_t block = first; block < stop; block += 4) {
    MxOperand x[2], y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[i] = load_block(a, m0 + 16 * i + (lane & 15), block + (lane >> 4), stop);
      y[i] = load_block(b, n0 + 16 * i + (lane & 15), block + (lane >> 4), stop);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) sum[i][j] = mx_mfma(x[i], y[j], sum[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t m = m0 + 16 * i + 4 * (lane >> 4) + r, n = n0 + 16 * j + (lane & 15);
        if (m < a.rows && n < b.rows) {
          if (splits > 1)
            partials[(split * a.rows + m) * b.rows + n] = sum[i][j][r];
          else
            out[m * stride + n] = static_cast<T>(sum[i][j][r] + (bias ? bias[n] : 0.0f));
        }
      }
}

// The parts of K added in order.
template <class T>
__global__ __launch_bounds__(kThreads) void add_splits(const float* __restrict__ partials,
                                                       int64_t splits, int64_t rows, int64_t columns,
                                                       const float* bias, T* out, int64_t stride) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= rows * columns) return;
  float sum = 0.0f;
  for (int64_t k = 0; k < splits; ++k) sum += partials[k * rows * columns + id];
  const int64_t m = id / columns, n = id - m * columns;
  out[m * stride + n] = static_cast<T>(sum + (bias ? bias[n] : 0.0f));
}

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

MxView view(const ns_mx_matrix& m) {
  return MxView{m.codes, m.scales, m.rows, (m.columns + NS_MX_BLOCK - 1) / NS_MX_BLOCK};
}

template <class T>
int run(const ns_mx_product_args* p, hipStream_t stream) {
  const MxView a = view(p->a), b = view(p->b);
  const int64_t tiles_n = (b.rows + 31) / 32, tiles = (a.rows + 31) / 32 * tiles_n;
  const int64_t groups = (tiles * p->splits + 3) / 4;
  if (groups > INT32_MAX) return fail("the product is too large for one launch");
  product_tiles<T><<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, stream>>>(
      a, b, p->bias, static_cast<T*>(p->out), p->stride, tiles_n, tiles, p->splits, p->partials);
  if (int rc = launched("product")) return rc;
  if (p->splits == 1) return NS_OK;
  const int64_t adds = (a.rows * b.rows + kThreads - 1) / kThreads;
  if (adds > INT32_MAX) return fail("the product is too large for one launch");
  add_splits<T><<<dim3(static_cast<unsigned>(adds)), dim3(kThreads), 0, stream>>>(
      p->partials, p->splits, a.rows, b.rows, p->bias, static_cast<T*>(p->out), p->stride);
  return launched("product parts");
}

int check_operand(const ns_mx_matrix& m, const char* what) {
  if (m.rows < 0 || m.columns < 0) return fail("%s: rows and columns must not be negative", what);
  if (m.rows && m.columns && (!m.codes || !m.scales))
    return fail("%s: codes and scales are required", what);
  if (reinterpret_cast<uintptr_t>(m.codes) % 16) return fail("%s: codes must be 16-byte aligned", what);
  return NS_OK;
}

}  // namespace
}  // namespace ns

extern "C" {

int32_t ns_mx_product_splits(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0) return 1;
  const int64_t tiles = (m + 31) / 32 * ((n + 31) / 32), steps = (k + 127) / 128;
  int64_t splits = 4096 / tiles;
  if (splits > steps / 4) splits = steps / 4;
  if (splits < 1) splits = 1;
  const int64_t per = (steps + splits - 1) / splits;   // no empty part
  return static_cast<int32_t>((steps + per - 1) / per);
}

int ns_mx_product(const ns_mx_product_args* p, void* stream) {
  ns::clear_error();
  if (!p) return ns::fail("product arguments are required");
  if (int rc = ns::check_operand(p->a, "a")) return rc;
  if (int rc = ns::check_operand(p->b, "b")) return rc;
  if (p->a.columns != p->b.columns) return ns::fail("the operands need the same number of columns");
  if (p->splits < 1) return ns::fail("a product has at least one part");
  if (p->a.rows == 0 || p->b.rows == 0) return NS_OK;
  if (!p->out) return ns::fail("the output is required");
  if (p->splits > 1 && !p->partials) return ns::fail("a split product needs its workspace");
  auto queue = static_cast<hipStream_t>(stream);
  switch (p->type) {
    case NS_TYPE_F32: return ns::run<float>(p, queue);
    case NS_TYPE_BF16: return ns::run<__bf16>(p, queue);
    case NS_TYPE_F16: return ns::run<_Float16>(p, queue);
    default: return ns::fail("unknown element type");
  }
}

}  // extern "C"
