// Products a b^T of float32 rows on the bfloat16 matrix cores, at float32's precision.
//
// A float32 x is three bfloat16 parts x0 + x1 + x2, exactly: each takes, rounded to nearest, the
// eight leading bits of what the ones before it left, at most 2^-8 and 2^-16 of x.  Six of
// the nine products of two numbers' parts are summed; x1 y2, x2 y1 and x2 y2, left out, are together
// at most 2^-23 of x y, as much as two roundings of a float32 product.  The matrix cores multiply
// bfloat16 16 times as fast as float32, so six products take 3/8 of the time of one in float32.
// Parts below bfloat16's least number, 2^-133, are lost: an x below 2^-109 keeps fewer bits.
//
// Rows lie in thirds: for every 32 columns 64 bytes of x0, of x1 and of x2, zeros past the last
// column.  A stage is one such block of every row of both operands; in LDS a part's 64 bytes of a
// row follow the next row's, its 16-byte piece k at place k ^ third_turn(row).
#pragma once

#include "ns_gemm.h"

namespace ns {

constexpr int kThirds = 192;   // bytes of 32 columns of a row

// x's three parts.  What rounds past the largest bfloat16 is cut off instead; infinities and NaN
// are their first part alone.
struct Thirds {
  __bf16 part[3];
};
__device__ __forceinline__ Thirds thirds_of(float x) {
  Thirds t;
  __bf16 first = static_cast<__bf16>(x);
  const bool finite = fabsf(x) < __builtin_inff();
  if (finite && !(fabsf(static_cast<float>(first)) < __builtin_inff()))
    first = __builtin_bit_cast(__bf16, static_cast<uint16_t>(__builtin_bit_cast(uint32_t, x) >> 16));
  const float rest = finite ? x - static_cast<float>(first) : 0.0f;
  t.part[0] = first;
  t.part[1] = static_cast<__bf16>(rest);
  t.part[2] = static_cast<__bf16>(rest - static_cast<float>(t.part[1]));
  return t;
}

// Eight columns, from column k (a multiple of 8) on, of a row that starts at `row`.
__device__ __forceinline__ void store_thirds(uint8_t* row, int64_t k, const float (&v)[8]) {
  Pack<__bf16, 8> out[3];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const Thirds t = thirds_of(v[j]);
#pragma unroll
    for (int p = 0; p < 3; ++p) out[p].v[j] = t.part[p];
  }
  uint8_t* const at = row + k / 32 * kThirds + k % 32 * 2;
#pragma unroll
  for (int p = 0; p < 3; ++p) *reinterpret_cast<v4i*>(at + 64 * p) = __builtin_bit_cast(v4i, out[p]);
}

// Geometry of a tile: WM x WN wavefronts, each MI x NJ results of 16x16; `stages` of them in LDS.
template <int kMI, int kNJ, int kWM, int kWN, int kStages>
struct SplitTile {
  static constexpr int MI = kMI, NJ = kNJ, WM = kWM, WN = kWN, stages = kStages;
  static constexpr int rows_m = 16 * MI * WM, rows_n = 16 * NJ * WN, rows = rows_m + rows_n;
  static constexpr int waves = WM * WN, threads = 64 * waves;
  static constexpr int stage_bytes = rows * kThirds;
  // Strips of 16 rows that a wavefront requests of each operand, three pieces a lane.
  static constexpr int strips_a = MI * WM / waves, strips_b = NJ * WN / waves;
  static constexpr int loads = 3 * (strips_a + strips_b);
  static_assert(strips_a * waves == MI * WM && strips_b * waves == NJ * WN, "whole strips");
};

// 0, 2, 3, 1 for the quarters of 16 rows: so the 16 lanes whose pieces LDS gives at a time, two
// quarters each of two neighbouring pieces, find them in different banks.
__device__ __forceinline__ uint32_t third_turn(uint32_t row) { return 0x78u >> (2 * (row >> 2 & 3)) & 3; }

// What a wavefront asks for: 16 rows of a third a request, a piece a lane.
template <class G>
struct SplitPlace {
  int lane, wave;
  uint32_t blocks;
  v4i a, b[G::strips_b];                         // buffers; the second operand's, by strip
  uint32_t at_a[G::strips_a], at_b[G::strips_b]; // the lane's piece of the first block
};

// `one` and `other` as in ns_gemm.h: kPair, strips of the first half of a wavefront's are the one
// matrix's, the others the other one's.
template <class G, bool kPair>
__device__ __forceinline__ SplitPlace<G> split_place(int lane, int wave, uint32_t blocks, const v4i& a,
                                                     uint32_t stride_a, const v4i& one, const v4i& other,
                                                     uint32_t stride_b) {
  SplitPlace<G> p;
  p.lane = lane;
  p.wave = wave;
  p.blocks = blocks;
  p.a = a;
  const uint32_t row = lane >> 2, piece = (lane & 3) ^ third_turn(row);
#pragma unroll
  for (int s = 0; s < G::strips_a; ++s)
    p.at_a[s] = (16 * (wave + s * G::waves) + row) * stride_a + piece * 16;
#pragma unroll
  for (int s = 0; s < G::strips_b; ++s) {
    const uint32_t strip = wave + s * G::waves;
    const uint32_t local = kPair ? strip / G::NJ * (G::NJ / 2) + strip % (G::NJ / 2) : strip;
    const bool first = !kPair || strip % G::NJ < G::NJ / 2;
    p.at_b[s] = (16 * local + row) * stride_b + piece * 16;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      p.b[s][k] = static_cast<int>(uniform(static_cast<uint32_t>(first ? one[k] : other[k])));
  }
  return p;
}

// Request I of a stage, into the stage's place `to`.
template <class G, int I>
__device__ __forceinline__ void request_third(const SplitPlace<G>& p, uint32_t block, uint32_t to) {
  constexpr int part = I % 3, s = I / 3;
  const bool inside = block < p.blocks;
  const uint32_t within = block * kThirds + 64 * part;
  if constexpr (s < G::strips_a) {
    to_lds_16(p.a, inside ? p.at_a[s] + within : kNone,
              to + part * (G::rows * 64) + (p.wave + s * G::waves) * 1024);
  } else {
    constexpr int t = s - G::strips_a;
    to_lds_16(p.b[t], inside ? p.at_b[t] + within : kNone,
              to + part * (G::rows * 64) + G::rows_m * 64 + (p.wave + t * G::waves) * 1024);
  }
}
template <class G, int I = 0>
__device__ __forceinline__ void request_thirds(const SplitPlace<G>& p, uint32_t block, uint32_t to) {
  request_third<G, I>(p, block, to);
  if constexpr (I + 1 < G::loads) request_thirds<G, I + 1>(p, block, to);
}

template <class G>
struct SplitFragments {
  v4i a[G::MI][3], b[G::NJ][3];
  static constexpr int count = 3 * (G::MI + G::NJ);
};
struct SplitBase {
  uint32_t a, b;                                 // of a wavefront's first strips of the first third
};
template <class G>
__device__ __forceinline__ SplitBase split_base(uint32_t stage, int wm, int wn, int lane) {
  const uint32_t row = lane & 15, place = (lane >> 4) ^ third_turn(row);
  const uint32_t at = stage + row * 64 + place * 16;
  SplitBase base{at + wm * (G::MI * 1024), at + G::rows_m * 64 + wn * (G::NJ * 1024)};
  // One register each, here: left to itself the compiler keeps every strip's.
  asm volatile("" : "+v"(base.a), "+v"(base.b));
  return base;
}
// Fragment I.
template <class G, int I>
__device__ __forceinline__ void read_third(const SplitBase& from, SplitFragments<G>& f) {
  constexpr int part = I % 3, s = I / 3;
  const auto read = [](uint32_t at) {
    return *(const __attribute__((address_space(3))) v4i*)static_cast<uintptr_t>(at);
  };
  if constexpr (s < G::MI) f.a[s][part] = read(from.a + part * (G::rows * 64) + s * 1024);
  else f.b[s - G::MI][part] = read(from.b + part * (G::rows * 64) + (s - G::MI) * 1024);
}
template <class G, int I = 0>
__device__ __forceinline__ void read_thirds(const SplitBase& from, SplitFragments<G>& f) {
  read_third<G, I>(from, f);
  if constexpr (I + 1 < SplitFragments<G>::count) read_thirds<G, I + 1>(from, f);
}

// Column strip C / 6 of a stage, the product C % 6 of parts: MI instructions, beside one read of the
// next stage's fragments and half a request.  (All reads and requests first kept the matrix cores
// waiting: 3885 x 1031 to 1500 and back 581 us.)
template <class G, int C = 0>
__device__ __forceinline__ void split_products(const SplitPlace<G>& p, uint32_t ahead, uint32_t now,
                                               const SplitBase& from, SplitFragments<G>& f,
                                               SplitFragments<G>& next, v4f (&sum)[G::MI][G::NJ]) {
  constexpr int kFirst[6] = {2, 0, 1, 1, 0, 0}, kSecond[6] = {0, 2, 1, 0, 1, 0};   // small ones first
  constexpr int j = C / 6, k = C % 6;
  constexpr int kReads = SplitFragments<G>::count;
  static_assert(kReads <= 12 * G::NJ && G::loads <= 3 * G::NJ, "a product's share");
  if constexpr (C < kReads) read_third<G, C>(from, next);
  if constexpr (C + 6 * G::NJ < kReads) read_third<G, C + 6 * G::NJ>(from, next);
  if constexpr (C % 2 == 0 && C / 2 < G::loads) request_third<G, C / 2>(p, ahead, now);
#pragma unroll
  for (int i = 0; i < G::MI; ++i)
    sum[i][j] = multiply_pieces<__bf16>(f.b[j][kFirst[k]], f.a[i][kSecond[k]], sum[i][j]);
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (C + 1 < 6 * G::NJ) split_products<G, C + 1>(p, ahead, now, from, f, next, sum);
}

// Multiplies a stage's fragments while the next one's are read; `now` is the place of the stage,
// which all have read to its end, and takes the stage after the G::stages - 1 that are on their way.
template <class G>
__device__ __forceinline__ void split_stage(const SplitPlace<G>& p, int wm, int wn, uint32_t ahead,
                                            uint32_t now, uint32_t then, SplitFragments<G>& f,
                                            SplitFragments<G>& next, v4f (&sum)[G::MI][G::NJ]) {
  // The next stage has arrived for all; those behind it may be on their way.
  wait_barrier<wait_loads_and_lds((G::stages - 2) * G::loads)>();
  split_products<G>(p, ahead, now, split_base<G>(then, wm, wn, p.lane), f, next, sum);
}

// The sums of a workgroup's tile; `stages` holds G::stages stages.  One barrier a stage.
template <class G>
__device__ __forceinline__ void split_tile(const SplitPlace<G>& p, const void* stages,
                                           v4f (&sum)[G::MI][G::NJ]) {
  constexpr uint32_t kStage = G::stage_bytes;
  const int wm = p.wave / G::WN, wn = p.wave % G::WN;
  const uint32_t lds = lds_address(stages), end = lds + G::stages * kStage;
  SplitFragments<G> even, odd;
#pragma unroll
  for (int k = 0; k < G::stages; ++k) request_thirds<G>(p, k, lds + k * kStage);
  wait_barrier<wait_loads((G::stages - 1) * G::loads)>();
  read_thirds<G>(split_base<G>(lds, wm, wn, p.lane), even);
  uint32_t now = lds;
  // Blocks past the last read as zeros: an odd number of them is filled up with one.
  for (uint32_t block = 0; block < p.blocks; block += 2) {
    uint32_t then = now + kStage < end ? now + kStage : lds;
    split_stage<G>(p, wm, wn, block + G::stages, now, then, even, odd, sum);
    now = then;
    then = now + kStage < end ? now + kStage : lds;
    split_stage<G>(p, wm, wn, block + 1 + G::stages, now, then, odd, even, sum);
    now = then;
  }
  wait_barrier<0>();                                       // before LDS is used anew
}

}  // namespace ns
