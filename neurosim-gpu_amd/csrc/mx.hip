// Microscaled 4-bit rows (gfx950): quantising float rows, and reading them back.
//
// Both are one pass over memory.  Four neighbouring lanes share a block of 32 values,
// eight values each, so a wavefront's loads and stores are whole runs of a row; the
// block's largest magnitude is joined over its lanes by two DPP steps.  Magnitudes are
// compared as integers: on non-negative floats the order is the same, and infinities and
// NaN come out on top.
#include "ns_signal.h"
#include "neurosim_hip_mx.h"

namespace ns {
namespace {

constexpr int kLaneValues = 8;

template <class T>
struct Eight {
  T v[kLaneValues];
};

// Eight values of a row from k (zeros past K).
template <class T>
__device__ __forceinline__ void load_eight(const T* row, int64_t k, int64_t width, float (&out)[8]) {
  if (k + kLaneValues <= width) {
    const Pack<T, 8> v = load_pack<T, 8>(row + k);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = static_cast<float>(v.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = k + i < width ? static_cast<float>(row[k + i]) : 0.0f;
  }
}

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  uint32_t o = __builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true);
  v = o > v ? o : v;
  o = __builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true);
  return o > v ? o : v;
}

// The scale byte of a block whose largest magnitude has these bits: biased exponent of
// float32 less 2, which is floor(log2) + 127 - 2 for normal values; subnormal ones lie
// below the smallest scale, 2^-127, times 4, as does zero.
__device__ __forceinline__ uint32_t scale_byte(uint32_t peak) {
  if (peak >= 0x7F800000u) return 255u;
  const uint32_t exponent = peak >> 23;
  return exponent > 2u ? exponent - 2u : 0u;
}

// 2^(byte - 127) as float32 (byte 0: the subnormal 2^-127).
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __builtin_bit_cast(float, byte ? byte << 23 : 0x00400000u);
}

template <class T>
__global__ __launch_bounds__(kThreads) void quantize(const T* x, int64_t stride, int64_t rows,
                                                     int64_t width, int64_t blocks, uint8_t* codes,
                                                     uint8_t* scales) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t block = id >> 2;
  const int part = threadIdx.x & 3;
  if (block >= rows * blocks) return;               // whole quads
  const int64_t row = block / blocks, k = (block - row * blocks) * NS_MX_BLOCK + part * kLaneValues;
  float v[8];
  load_eight(x + row * stride, k, width, v);
  uint32_t peak = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t size = __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu;
    peak = size > peak ? size : peak;
  }
  const uint32_t byte = scale_byte(quad_max(peak));
  uint32_t packed = 0;
  if (byte != 255u) {
    // The conversion divides by the scale, rounds to nearest even and saturates.
    const float unit = scale_value(byte);
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v[0], v[1], unit, 0);
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v[2], v[3], unit, 1);
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v[4], v[5], unit, 2);
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v[6], v[7], unit, 3);
  }
  reinterpret_cast<uint32_t*>(codes)[id] = packed;
  if (part == 0) scales[block] = static_cast<uint8_t>(byte);
}

template <class T>
__global__ __launch_bounds__(kThreads) void dequantize(const uint8_t* codes, const uint8_t* scales,
                                                       int64_t rows, int64_t width, int64_t blocks,
                                                       T* out, int64_t stride) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t block = id >> 2;
  if (block >= rows * blocks) return;
  const int64_t row = block / blocks,
                k = (block - row * blocks) * NS_MX_BLOCK + (threadIdx.x & 3) * kLaneValues;
  const uint32_t packed = reinterpret_cast<const uint32_t*>(codes)[id], byte = scales[block];
  const float unit = byte == 255u ? __builtin_nanf("") : scale_value(byte);
  Pack<T, 8> v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // Codes to values with a unit scale, then one multiply: exact in float32.
    const ns_v2f two = e2m1_pair(packed >> (8 * i) & 255u);
    v.v[2 * i] = static_cast<T>(two.x * unit);
    v.v[2 * i + 1] = static_cast<T>(two.y * unit);
  }
  T* to = out + row * stride + k;
  if (k + kLaneValues <= width) {
    store_pack<T, 8>(to, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < width) to[i] = v.v[i];
  }
}

int check_matrix(const ns_mx_matrix* m) {
  if (!m) return fail("a quantised matrix is required");
  if (m->rows < 0 || m->columns < 0) return fail("rows and columns must not be negative");
  if (m->rows && m->columns && (!m->codes || !m->scales))
    return fail("codes and scales are required");
  if (reinterpret_cast<uintptr_t>(m->codes) % 16) return fail("codes must be 16-byte aligned");
  return NS_OK;
}

int rows_grid(const ns_mx_matrix* m, dim3* grid) {
  const int64_t blocks = (m->columns + NS_MX_BLOCK - 1) / NS_MX_BLOCK;
  const int64_t groups = (m->rows * blocks * 4 + kThreads - 1) / kThreads;
  if (groups > INT32_MAX) return fail("the matrix is too large for one launch");
  *grid = dim3(static_cast<unsigned>(groups));
  return NS_OK;
}

template <class T>
int run_rows(const ns_mx_matrix* m, void* x, int64_t stride, bool back, hipStream_t stream) {
  dim3 grid;
  if (int rc = rows_grid(m, &grid)) return rc;
  const int64_t blocks = (m->columns + NS_MX_BLOCK - 1) / NS_MX_BLOCK;
  if (back)
    dequantize<T><<<grid, dim3(kThreads), 0, stream>>>(m->codes, m->scales, m->rows, m->columns,
                                                       blocks, static_cast<T*>(x), stride);
  else
    quantize<T><<<grid, dim3(kThreads), 0, stream>>>(static_cast<const T*>(x), stride, m->rows,
                                                     m->columns, blocks, m->codes, m->scales);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(back ? "dequantise" : "quantise", err);
}

int run_types(const ns_mx_matrix* m, void* x, int64_t stride, int32_t type, bool back, void* stream) {
  clear_error();
  if (int rc = check_matrix(m)) return rc;
  if (m->rows == 0 || m->columns == 0) return NS_OK;
  if (!x) return fail("the float rows are required");
  auto queue = static_cast<hipStream_t>(stream);
  switch (type) {
    case NS_TYPE_F32: return run_rows<float>(m, x, stride, back, queue);
    case NS_TYPE_BF16: return run_rows<__bf16>(m, x, stride, back, queue);
    case NS_TYPE_F16: return run_rows<_Float16>(m, x, stride, back, queue);
    default: return fail("unknown element type");
  }
}

}  // namespace
}  // namespace ns

extern "C" {

int ns_mx_quantize(const ns_mx_matrix* matrix, const void* x, int64_t stride, int32_t type,
                   void* stream) {
  return ns::run_types(matrix, const_cast<void*>(x), stride, type, false, stream);
}

int ns_mx_dequantize(const ns_mx_matrix* matrix, void* out, int64_t stride, int32_t type,
                     void* stream) {
  return ns::run_types(matrix, out, stride, type, true, stream);
}

}  // extern "C"
