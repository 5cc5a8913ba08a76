// 4-bit integer rows with a scale per group (gfx950): quantisation, and reading back.
#include "ns_q4.h"

namespace ns {
namespace {

__device__ __forceinline__ float to_scale_type(float s, int32_t type) {
  if (type == NS_TYPE_F32) return s;
  if (type == NS_TYPE_BF16) return static_cast<float>(static_cast<__bf16>(s));
  return static_cast<float>(static_cast<_Float16>(s));
}

__device__ __forceinline__ void store_scale(void* to, int64_t at, float s, int32_t type) {
  if (type == NS_TYPE_F32) static_cast<float*>(to)[at] = s;
  else if (type == NS_TYPE_BF16) static_cast<__bf16*>(to)[at] = static_cast<__bf16>(s);
  else static_cast<_Float16*>(to)[at] = static_cast<_Float16>(s);
}

// kLanes neighbouring lanes per group, eight values (a 32-bit word of codes) each at a time.
// The values are read twice: for their range, and, from the caches, for the codes.
template <class T, int kLanes>
__global__ __launch_bounds__(kThreads) void q4_quantize(const T* x, int64_t stride, Q4View w,
                                                        uint8_t* codes, void* scales, uint8_t* zeros) {
  constexpr int V = 8;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (kThreads / kLanes) + threadIdx.x / kLanes;
  // Lanes past the last group take it again without storing: all lanes meet below.
  const bool own = id < w.rows * w.groups;
  const int64_t at = own ? id : w.rows * w.groups - 1;
  const int64_t row = at / w.groups, first = (at - row * w.groups) * w.group;
  const int64_t stop = first + w.group < w.columns ? first + w.group : w.columns;
  const T* const from = x + row * stride;
  const int lane = threadIdx.x % kLanes;
  float low = 0.0f, high = 0.0f;
  bool finite = true;
  for (int64_t k = first + lane * V; k < stop; k += kLanes * V) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float v = k + j < stop ? static_cast<float>(from[k + j]) : 0.0f;
      finite = finite && fabsf(v) < __builtin_inff();
      low = fminf(low, v);
      high = fmaxf(high, v);
    }
  }
#pragma unroll
  for (int step = 1; step < kLanes; step *= 2) {
    low = fminf(low, __shfl_xor(low, step));
    high = fmaxf(high, __shfl_xor(high, step));
    finite = __shfl_xor(static_cast<int>(finite), step) && finite;
  }
  float scale = zeros ? high / 15.0f - low / 15.0f : fmaxf(high, -low) / 7.0f;
  scale = to_scale_type(scale, w.scale_type);
  const bool good = finite && scale < __builtin_inff(), some = good && scale > 0.0f;
  float zero = zeros ? 0.0f : 8.0f;
  if (zeros && some) zero = fminf(fmaxf(rintf(-low / scale), 0.0f), 15.0f);
  if (own && lane == 0) {
    store_scale(scales, at, good ? scale : __builtin_nanf(""), w.scale_type);
    if (zeros) zeros[at] = static_cast<uint8_t>(zero);
  }
  if (!own) return;
  // The last group's words go on to the end of the row's last 16 bytes, codes of zero.
  const int64_t filled = stop == w.columns ? w.blocks * 32 : stop;
  for (int64_t k = first + lane * V; k < filled; k += kLanes * V) {
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float code = good ? zero : 0.0f;
      if (k + j < stop && some)
        code = fminf(fmaxf(rintf(static_cast<float>(from[k + j]) / scale) + zero, 0.0f), 15.0f);
      if (k + j < stop) word |= static_cast<uint32_t>(code) << (4 * j);
    }
    *reinterpret_cast<uint32_t*>(codes + row * w.blocks * 16 + k / 2) = word;
  }
}

// A thread takes eight values of a group.
template <class T>
__global__ __launch_bounds__(kThreads) void q4_dequantize(Q4View w, T* out, int64_t stride) {
  constexpr int V = 8;
  const int64_t words = w.blocks * 4, id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= w.rows * words) return;
  const int64_t row = id / words, k = (id - row * words) * V;
  if (k >= w.columns) return;
  const int64_t at = row * w.groups + k / w.group;
  const float scale = q4_scale(w, at), zero = w.zeros ? static_cast<float>(w.zeros[at]) : 8.0f;
  const uint32_t word = *reinterpret_cast<const uint32_t*>(w.codes + row * w.blocks * 16 + k / 2);
  Pack<T, V> v;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float value = (static_cast<float>(word >> (4 * j) & 15u) - zero) * scale;
    // A float32 value in every type: joined with the conversion it would be rounded differently.
    asm volatile("" : "+v"(value));
    v.v[j] = static_cast<T>(value);
  }
  T* const to = out + row * stride + k;
  if (k + V <= w.columns) {
    store_pack<T, V>(to, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (k + j < w.columns) to[j] = v.v[j];
  }
}

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

template <class T, int kLanes>
int run_quantize(const ns_q4_matrix* m, const void* x, int64_t stride, hipStream_t stream) {
  const Q4View w = q4_view(*m);
  const int64_t per = kThreads / kLanes, blocks = (w.rows * w.groups + per - 1) / per;
  if (blocks > INT32_MAX) return fail("the matrix is too large for one launch");
  q4_quantize<T, kLanes><<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream>>>(
      static_cast<const T*>(x), stride, w, m->codes, m->scales, m->zeros);
  return launched("4-bit quantisation");
}

template <class T>
int run_groups(const ns_q4_matrix* m, const void* x, int64_t stride, hipStream_t stream) {
  switch (m->group) {
    case 32: return run_quantize<T, 4>(m, x, stride, stream);
    case 64: return run_quantize<T, 8>(m, x, stride, stream);
    default: return run_quantize<T, 16>(m, x, stride, stream);
  }
}

template <class T>
int run_dequantize(const ns_q4_matrix* m, void* out, int64_t stride, hipStream_t stream) {
  const Q4View w = q4_view(*m);
  const int64_t blocks = (w.rows * w.blocks * 4 + kThreads - 1) / kThreads;
  if (blocks > INT32_MAX) return fail("the matrix is too large for one launch");
  q4_dequantize<T><<<dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream>>>(
      w, static_cast<T*>(out), stride);
  return launched("4-bit values");
}

}  // namespace
}  // namespace ns

extern "C" {

int ns_q4_quantize(const ns_q4_matrix* m, const void* x, int64_t stride, int32_t type, void* stream) {
  ns::clear_error();
  if (!m) return ns::fail("the matrix is required");
  if (int rc = ns::check_q4(*m)) return rc;
  if (m->rows == 0 || m->columns == 0) return NS_OK;
  if (!x) return ns::fail("the values are required");
  auto queue = static_cast<hipStream_t>(stream);
  switch (type) {
    case NS_TYPE_F32: return ns::run_groups<float>(m, x, stride, queue);
    case NS_TYPE_BF16: return ns::run_groups<__bf16>(m, x, stride, queue);
    case NS_TYPE_F16: return ns::run_groups<_Float16>(m, x, stride, queue);
    default: return ns::fail("unknown element type");
  }
}

int ns_q4_dequantize(const ns_q4_matrix* m, void* out, int64_t stride, int32_t type, void* stream) {
  ns::clear_error();
  if (!m) return ns::fail("the matrix is required");
  if (int rc = ns::check_q4(*m)) return rc;
  if (m->rows == 0 || m->columns == 0) return NS_OK;
  if (!out) return ns::fail("the values' place is required");
  auto queue = static_cast<hipStream_t>(stream);
  switch (type) {
    case NS_TYPE_F32: return ns::run_dequantize<float>(m, out, stride, queue);
    case NS_TYPE_BF16: return ns::run_dequantize<__bf16>(m, out, stride, queue);
    case NS_TYPE_F16: return ns::run_dequantize<_Float16>(m, out, stride, queue);
    default: return ns::fail("unknown element type");
  }
}

}  // extern "C"
