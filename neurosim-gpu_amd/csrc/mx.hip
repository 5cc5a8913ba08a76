// Microscaled 4-bit rows (gfx950): quantising float rows, and reading them back.
//
// Both are one pass over memory: 16384 x 8192 in bf16 (340 MB) 57 us to quantise, 48 to read
// back, 6 and 7 TB/s.  Quantising, four neighbouring lanes share a block of 32 values, eight
// values each, so a wavefront's loads and stores are whole runs of a row; the
// block's largest magnitude is joined over its lanes by two DPP steps.  Magnitudes are
// compared as integers: on non-negative floats the order is the same, and infinities and
// NaN come out on top.
#include <type_traits>

#include "ns_signal.h"
#include "neurosim_hip_mx.h"

namespace ns {
namespace {

constexpr int kLaneValues = 8;

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

// Pieces (of a few values of a block) per thread, a workgroup's width apart: several requests on their
// way at a time.  Places are counted in I, 32 bits where the pieces allow: a 64-bit division
// per piece would cost more than the rest of its work.
constexpr int kPieces = 4;

template <class I>
struct Piece {
  I block, row;
  int64_t k;
  bool inside;
};

template <class I, int kValues = kLaneValues>
__device__ __forceinline__ Piece<I> piece_at(I first, int i, I total, I blocks) {
  Piece<I> p;
  const I id = first + i * kThreads + threadIdx.x;
  p.inside = id < total;
  constexpr int kLanes = NS_MX_BLOCK / kValues;            // per block
  p.block = (p.inside ? id : 0) / kLanes;
  p.row = p.block / blocks;
  p.k = static_cast<int64_t>(p.block - p.row * blocks) * NS_MX_BLOCK +
        (threadIdx.x & (kLanes - 1)) * kValues;
  return p;
}

template <class T, class I>
__global__ __launch_bounds__(kThreads) void quantize(const T* x, int64_t stride, I total,
                                                     int64_t width, I blocks, uint8_t* codes,
                                                     uint8_t* scales) {
  const I first = static_cast<I>(blockIdx.x) * (kPieces * kThreads);
  Piece<I> at[kPieces];
  float v[kPieces][8];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    at[i] = piece_at<I>(first, i, total, blocks);
    load_eight(x + at[i].row * stride, at[i].k, width, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    uint32_t peak = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t size = __builtin_bit_cast(uint32_t, v[i][k]) & 0x7FFFFFFFu;
      peak = size > peak ? size : peak;
    }
    const uint32_t byte = scale_byte(quad_max(peak));    // whole quads are inside or not
    // The conversion divides by the scale, rounds to nearest even and saturates.
    const float unit = scale_value(byte);
    uint32_t packed = 0;
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v[i][0], v[i][1], unit, 0);
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v[i][2], v[i][3], unit, 1);
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v[i][4], v[i][5], unit, 2);
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v[i][6], v[i][7], unit, 3);
    if (byte == 255u) packed = 0;
    if (at[i].inside) {
      reinterpret_cast<uint32_t*>(codes)[first + i * kThreads + threadIdx.x] = packed;
      if ((threadIdx.x & 3) == 0) scales[at[i].block] = static_cast<uint8_t>(byte);
    }
  }
}

// A piece is 16 bytes of the values, so that a wavefront's store is one run of a row (eight
// values a piece in float32 too: 226 us instead of 85 for 16384 x 8192).  kStream: past the
// caches, the values being several times their codes.
template <class T, class I, bool kStream>
__global__ __launch_bounds__(kThreads) void dequantize(const uint8_t* codes, const uint8_t* scales,
                                                       I total, int64_t width, I blocks, T* out,
                                                       int64_t stride) {
  constexpr int kValues = 16 / sizeof(T);
  typedef std::conditional_t<kValues == 8, uint32_t, uint16_t> Codes;
  const I first = static_cast<I>(blockIdx.x) * (kPieces * kThreads);
  Piece<I> at[kPieces];
  uint32_t packed[kPieces], byte[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    at[i] = piece_at<I, kValues>(first, i, total, blocks);
    const I id = first + i * kThreads + threadIdx.x;
    packed[i] = reinterpret_cast<const Codes*>(codes)[at[i].inside ? id : 0];
    byte[i] = scales[at[i].block];
  }
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const float unit = byte[i] == 255u ? __builtin_nanf("") : scale_value(byte[i]);
    Pack<T, kValues> v;
#pragma unroll
    for (int k = 0; k < kValues / 2; ++k) {
      // Codes to values with a unit scale, then one multiply: exact in float32.
      const ns_v2f two = e2m1_pair(packed[i] >> (8 * k) & 255u);
      v.v[2 * k] = static_cast<T>(two.x * unit);
      v.v[2 * k + 1] = static_cast<T>(two.y * unit);
    }
    if (!at[i].inside) continue;
    T* to = out + at[i].row * stride + at[i].k;
    if (at[i].k + kValues <= width) {
      stream_pack<T, kValues, kStream>(to, v);
    } else {
#pragma unroll
      for (int k = 0; k < kValues; ++k)
        if (at[i].k + k < width) to[k] = v.v[k];
    }
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

template <class T, class I>
void launch_rows(const ns_mx_matrix* m, void* x, int64_t stride, bool back, int64_t total,
                 int64_t blocks, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((total + kPieces * kThreads - 1) / (kPieces * kThreads)));
  if (back) {
    // us, past the caches and through them: 16384 x 8192 in bf16 49 / 60, float32 85 / 112; where
    // two stores share a piece of 32 bytes, the same (16384 x 8191 65 / 65, float32 127 / 127).
    const bool whole = (reinterpret_cast<uintptr_t>(x) | stride * sizeof(T)) % 32 == 0;
    const auto kernel = whole ? dequantize<T, I, true> : dequantize<T, I, false>;
    kernel<<<grid, dim3(kThreads), 0, stream>>>(m->codes, m->scales, static_cast<I>(total),
                                                m->columns, static_cast<I>(blocks),
                                                static_cast<T*>(x), stride);
  } else {
    quantize<T, I><<<grid, dim3(kThreads), 0, stream>>>(
        static_cast<const T*>(x), stride, static_cast<I>(total), m->columns, static_cast<I>(blocks),
        m->codes, m->scales);
  }
}

template <class T>
int run_rows(const ns_mx_matrix* m, void* x, int64_t stride, bool back, hipStream_t stream) {
  const int64_t blocks = (m->columns + NS_MX_BLOCK - 1) / NS_MX_BLOCK;
  const int64_t lanes = NS_MX_BLOCK / (back ? 16 / static_cast<int>(sizeof(T)) : kLaneValues);
  const int64_t total = m->rows * blocks * lanes;
  if (total / (kPieces * kThreads) >= INT32_MAX) return fail("the matrix is too large for one launch");
  // The last workgroup's pieces too have to be counted within I.
  if (total <= UINT32_MAX - kPieces * kThreads)
    launch_rows<T, uint32_t>(m, x, stride, back, total, blocks, stream);
  else
    launch_rows<T, int64_t>(m, x, stride, back, total, blocks, stream);
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
