// Dropout from a counter-based generator (gfx950): the mask is computed where it is used,
// forwards and backwards, and never stored.
//
// A thread takes eight neighbouring elements, one counter: ten rounds of two 32 x 32 -> 64
// products give eight 16-bit numbers.  (16 bits: one part in 65536 of the drop rate, which
// the scale follows, for half the rounds that 32 bits would cost.)  Bound by memory: 16,384 x 4096
// in bf16 onto a residual 73 us, 5.5 TB/s, back 42, 6.4 TB/s; the vector ALU is half busy.
#include "ns_signal.h"
#include "neurosim_hip_block.h"

namespace ns {
namespace {

// Philox4x32 with 10 rounds (Salmon et al. 2011): c 128 bits, key 64.
__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p0 = static_cast<uint64_t>(c[0]) * 0xD2511F53u;
    const uint64_t p1 = static_cast<uint64_t>(c[2]) * 0xCD9E8D57u;
    const uint32_t next0 = static_cast<uint32_t>(p1 >> 32) ^ c[1] ^ k0;
    const uint32_t next2 = static_cast<uint32_t>(p0 >> 32) ^ c[3] ^ k1;
    c[1] = static_cast<uint32_t>(p1);
    c[3] = static_cast<uint32_t>(p0);
    c[0] = next0;
    c[2] = next2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

template <class T>
__global__ __launch_bounds__(kThreads) void dropout(int64_t count, uint32_t threshold, float scale,
                                                    const T* x, const T* residual, T* out,
                                                    const int64_t* seed_data, int64_t seed,
                                                    int64_t offset) {
  constexpr int V = 8;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t first = at * V;
  if (first >= count) return;
  const uint64_t key = static_cast<uint64_t>(seed_data ? *seed_data : seed);
  uint32_t c[4] = {static_cast<uint32_t>(at), static_cast<uint32_t>(static_cast<uint64_t>(at) >> 32),
                   static_cast<uint32_t>(offset),
                   static_cast<uint32_t>(static_cast<uint64_t>(offset) >> 32)};
  const auto value = [&](T v, T more, int j) __attribute__((always_inline)) {
    const uint32_t number = j & 1 ? c[j / 2] >> 16 : c[j / 2] & 0xFFFFu;
    const float dropped = number >= threshold ? static_cast<float>(v) * scale : 0.0f;
    return static_cast<T>(residual ? static_cast<float>(more) + dropped : dropped);
  };
  if (first + V <= count) {
    const Pack<T, V> in = load_pack<T, V>(x + first);
    Pack<T, V> more{};
    if (residual) more = load_pack<T, V>(residual + first);
    philox(c, static_cast<uint32_t>(key), static_cast<uint32_t>(key >> 32));
    Pack<T, V> y;
#pragma unroll
    for (int j = 0; j < V; ++j) y.v[j] = value(in.v[j], more.v[j], j);
    store_pack<T, V>(out + first, y);
  } else {
    philox(c, static_cast<uint32_t>(key), static_cast<uint32_t>(key >> 32));
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (first + j < count)
        out[first + j] = value(x[first + j], residual ? residual[first + j] : T{}, j);
  }
}

template <class T>
int run(const ns_dropout_args* a, hipStream_t stream) {
  const int64_t per = 8 * kThreads, groups = (a->count + per - 1) / per;
  if (groups > INT32_MAX) return fail("the tensor is too large for one launch");
  const float scale = a->threshold < 65536 ? 65536.0f / (65536 - a->threshold) : 0.0f;
  dropout<T><<<dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, stream>>>(
      a->count, static_cast<uint32_t>(a->threshold), scale, static_cast<const T*>(a->x),
      static_cast<const T*>(a->residual), static_cast<T*>(a->out), a->seed_data, a->seed, a->offset);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch("dropout", err);
}

}  // namespace
}  // namespace ns

extern "C" int ns_dropout(const ns_dropout_args* a, void* stream) {
  ns::clear_error();
  if (!a) return ns::fail("dropout arguments are required");
  if (a->count < 0) return ns::fail("the element count must not be negative");
  if (a->threshold < 0 || a->threshold > 65536) return ns::fail("the threshold is 0 to 65536");
  if (a->type != NS_TYPE_F32 && a->type != NS_TYPE_BF16 && a->type != NS_TYPE_F16)
    return ns::fail("unknown element type");
  if (a->count == 0) return NS_OK;
  if (!a->x || !a->out) return ns::fail("x and the output are required");
  auto queue = static_cast<hipStream_t>(stream);
  if (a->type == NS_TYPE_F32) return ns::run<float>(a, queue);
  if (a->type == NS_TYPE_BF16) return ns::run<__bf16>(a, queue);
  return ns::run<_Float16>(a, queue);
}
