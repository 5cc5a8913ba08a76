// Products a b^T of rows of float32, bfloat16 or float16 on the matrix cores, tile by tile.
//
// All types go the same way through the memories, as 16-byte pieces of rows: a stage is 128
// bytes (eight pieces) of every row of both operands, two of them in LDS, multiplied in two
// steps.  In an instruction (16x16x32 of 16-bit values, four 16x16x4 of float32) lane l holds a
// piece of row l%16, so the four quarters of a wavefront hold four pieces of a row; which ones
// they are does not matter as long as both operands agree.  The 16x16 result has column l%16
// of the first operand's rows and rows 4*(l/16) .. +3 in lane l's four registers.
#pragma once

#include "ns_tiles.h"

namespace ns {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// c + the products of one piece per lane of both operands.
template <class T>
__device__ __forceinline__ v4f multiply_pieces(v4i a, v4i b, v4f c) {
  if constexpr (sizeof(T) == 4) {
    const v4f x = __builtin_bit_cast(v4f, a), y = __builtin_bit_cast(v4f, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[k], y[k], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, __bf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a),
                                                   __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                  __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
}

// Rows of an operand: whole 16-byte pieces at 16-byte aligned addresses.
struct Rows {
  const uint8_t* data;
  int64_t stride;              // bytes from row to row, a multiple of 16, below kMostStride
  int64_t rows;
};
constexpr int64_t kMostStride = 1 << 23;   // 256 rows of a tile are addressed in 31 bits

// Geometry of a tile: WM x WN wavefronts, each MI x NJ results of 16x16; `stages` of them in LDS.
template <int kMI, int kNJ, int kWM, int kWN, int kStages>
struct GemmTile {
  static constexpr int MI = kMI, NJ = kNJ, WM = kWM, WN = kWN, stages = kStages;
  static constexpr int rows_m = 16 * MI * WM, rows_n = 16 * NJ * WN, rows = rows_m + rows_n;
  static constexpr int threads = 64 * WM * WN;
  static constexpr int loads = rows * 8 / threads;          // 16-byte pieces per thread and stage
  static constexpr int loads_a = rows_m * 8 / threads;
  static constexpr int per_round = threads / 8;             // rows per load instruction of all waves
  static_assert(rows_m % per_round == 0 && rows_n % per_round == 0, "a round reads one operand");
  static_assert(MI % NJ == 0 && loads % NJ == 0, "a column's share of reads and requests");
};

// A tile's rows of an operand as a buffer, whose reads past its end give zeros.
__device__ __forceinline__ v4i rows_buffer(const Rows& m, int64_t row, int rows, uint32_t pieces) {
  const int64_t left = m.rows - row;
  const int own = static_cast<int>(left < rows ? left : rows);
  const uint32_t bytes = own > 0 ? (own - 1) * static_cast<uint32_t>(m.stride) + pieces * 16 : 0;
  return describe(m.data + (own > 0 ? row : 0) * m.stride, bytes);
}

// The second operand's rows of a tile: of one matrix, or (kPair) of two, whose rows are dealt to
// the wavefronts so that each has as many strips of the one as of the other, for the same columns
// of the result: strips j < NJ/2 of a wavefront are the first one's, the others the second one's.
template <bool kPair>
struct Second {
  v4i buffer[kPair ? 2 : 1];
  v4i own;                     // kPair, where a wavefront requests of one of them only: that one
};

// Where a round requests as many rows as a wavefront multiplies of one matrix, rounds take the
// two in turn; else a wavefront's requests are all of the same one.
template <class G>
constexpr bool kInTurn = G::per_round == 8 * G::NJ;

template <class G>
__device__ __forceinline__ Second<true> second_pair(const v4i& one, const v4i& other, int wave) {
  static_assert(kInTurn<G> || G::per_round % (16 * G::NJ) == 0, "a request is of one matrix");
  const bool first = (8 * wave >> 4) % G::NJ < G::NJ / 2;
  Second<true> b{{one, other}, {}};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    b.own[k] = static_cast<int>(uniform(static_cast<uint32_t>(first ? one[k] : other[k])));
  return b;
}

struct GemmPlace {
  int lane, wave;
  uint32_t row, piece;         // of the lane in a request
  uint32_t stride_a, stride_b, pieces;
  v4i a;
};

// Requests piece `at` (of the lane) of round I of a stage.
template <class G, bool kPair, int I>
__device__ __forceinline__ void request_round(const GemmPlace& p, const Second<kPair>& b, uint32_t at,
                                              uint32_t to) {
  const bool inside = at < p.pieces;
  const uint32_t place = to + 16 * 64 * p.wave + 16 * (I * G::threads);
  if constexpr (I < G::loads_a) {
    const uint32_t offset = (p.row + G::per_round * I) * p.stride_a + at * 16;
    to_lds_16(p.a, inside ? offset : kNone, place);
  } else {
    constexpr int first = G::per_round * (I - G::loads_a);
    if constexpr (kPair) {
      // Eight rows of one wavefront's request lie in one strip.
      const uint32_t strip = (first + 8 * p.wave) >> 4, j = strip % G::NJ;
      const uint32_t local = (strip / G::NJ * (G::NJ / 2) + j % (G::NJ / 2)) * 16 + (8 * p.wave & 8);
      const uint32_t offset = (local + (p.lane >> 3)) * p.stride_b + at * 16;
      constexpr int in_turn = (I - G::loads_a) & 1;
      to_lds_16(kInTurn<G> ? b.buffer[in_turn] : b.own, inside ? offset : kNone, place);
    } else {
      const uint32_t offset = (p.row + first) * p.stride_b + at * 16;
      to_lds_16(b.buffer[0], inside ? offset : kNone, place);
    }
  }
}

template <class G, bool kPair, int I = 0>
__device__ __forceinline__ void request_stage(const GemmPlace& p, const Second<kPair>& b, uint32_t at,
                                              uint32_t to) {
  request_round<G, kPair, I>(p, b, at, to);
  if constexpr (I + 1 < G::loads) request_stage<G, kPair, I + 1>(p, b, at, to);
}

// A wavefront's operands of one step.
template <class G>
struct GemmFragments {
  v4i a[G::MI], b[G::NJ];
};

// LDS addresses of a wavefront's first strips of a step; the other strips lie at constant
// distances.
struct GemmBase {
  uint32_t a, b;
};
template <class G>
__device__ __forceinline__ GemmBase gemm_base(uint32_t stage, int step, int wm, int wn, int lane) {
  const uint32_t row = lane & 15, place = (2 * (lane >> 4) + step) ^ turn(row);
  const uint32_t at = stage + (row * 8 + place) * 16;
  GemmBase base{at + wm * (G::MI * 16 * 128), at + (G::rows_m + wn * G::NJ * 16) * 128};
  // One register each, here: left to itself the compiler keeps every strip's.
  asm volatile("" : "+v"(base.a), "+v"(base.b));
  return base;
}

// Multiplies column strip J, reading a share of the next step's operands meanwhile and (kAsk)
// requesting a share of a stage to come.
template <class G, class T, bool kPair, bool kAsk, int J = 0>
__device__ __forceinline__ void gemm_columns(GemmFragments<G>& f, const GemmBase& from,
                                             GemmFragments<G>& next, const GemmPlace& p,
                                             const Second<kPair>& b, uint32_t at, uint32_t to,
                                             v4f (&sum)[G::MI][G::NJ]) {
  constexpr int kPer = G::MI / G::NJ, kRounds = G::loads / G::NJ;
  next.b[J] = read_code(from.b, J);
#pragma unroll
  for (int i = kPer * J; i < kPer * (J + 1); ++i) next.a[i] = read_code(from.a, i);
  if constexpr (kAsk) {
    request_round<G, kPair, kRounds * J>(p, b, at, to);
    if constexpr (kRounds > 1) request_round<G, kPair, kRounds * J + 1>(p, b, at, to);
    static_assert(kRounds <= 2, "requests of a column");
  }
  // The empty statements keep the products of a column in its place: the compiler would gather
  // them before the barrier, and wait there for operands that were to arrive meanwhile.
  asm volatile("" : "+v"(f.b[J]));
#pragma unroll
  for (int i = 0; i < G::MI; ++i) sum[i][J] = multiply_pieces<T>(f.b[J], f.a[i], sum[i][J]);
#pragma unroll
  for (int i = 0; i < G::MI; ++i) asm volatile("" : "+v"(sum[i][J]));
  if constexpr (J + 1 < G::NJ)
    gemm_columns<G, T, kPair, kAsk, J + 1>(f, from, next, p, b, at, to, sum);
}

// The sums of a workgroup's tile over pieces [0, pieces) of its rows.  `stages` is the LDS of
// G::stages stages.  While a stage's second step is multiplied, the first of the next one is read,
// and a stage to come is requested into the place that all have read to its end: one barrier a
// stage, after its first step.
template <class G, class T, bool kPair>
__device__ __forceinline__ void gemm_tile(GemmPlace p, const Second<kPair>& b, v4i* stages,
                                          v4f (&sum)[G::MI][G::NJ]) {
  constexpr uint32_t kStage = G::rows * 128;
  const int wm = p.wave / G::WN, wn = p.wave % G::WN;
  const uint32_t lds = lds_address(stages);
  p.row = 8 * p.wave + (p.lane >> 3);
  p.piece = (p.lane & 7) ^ turn(p.row);
  const int count = static_cast<int>(p.pieces + 7) / 8;
  GemmFragments<G> even, odd;
#pragma unroll
  for (int k = 0; k < G::stages; ++k) request_stage<G, kPair>(p, b, p.piece + 8 * k, lds + k * kStage);
  wait_barrier<wait_loads((G::stages - 1) * G::loads)>();
  const GemmBase begin = gemm_base<G>(lds, 0, wm, wn, p.lane);
#pragma unroll
  for (int i = 0; i < G::MI; ++i) even.a[i] = read_code(begin.a, i);
#pragma unroll
  for (int j = 0; j < G::NJ; ++j) even.b[j] = read_code(begin.b, j);
  // Stages past the last read as zeros and are not multiplied.
  uint32_t now = lds;
  for (int stage = 0; stage < count; ++stage) {
    const uint32_t then = now + kStage < lds + G::stages * kStage ? now + kStage : lds;
    gemm_columns<G, T, kPair, false>(even, gemm_base<G>(now, 1, wm, wn, p.lane), odd, p, b, 0, 0, sum);
    // This stage is read by all, and the next one has arrived for all; those behind it may be on
    // their way.
    wait_barrier<wait_loads_and_lds((G::stages - 2) * G::loads)>();
    gemm_columns<G, T, kPair, true>(odd, gemm_base<G>(then, 0, wm, wn, p.lane), even, p, b,
                                    p.piece + 8 * (stage + G::stages), now, sum);
    now = then;
  }
  wait_barrier<0>();                                       // before LDS is used anew
}

// Workgroups are dealt to the XCDs in turn: each XCD gets a run of tiles, in bands of four
// rows, so that those it multiplies at a time share panels in its L2.
struct TilePlace {
  uint32_t m, n;
};
__device__ __forceinline__ TilePlace tile_place(uint32_t tiles_m, uint32_t tiles_n) {
  constexpr uint32_t kBand = 4;
  const uint32_t share = tiles_m * tiles_n / kXcds;
  const uint32_t tile = blockIdx.x < share * kXcds ? blockIdx.x % kXcds * share + blockIdx.x / kXcds
                                                   : blockIdx.x;
  const uint32_t band = uniform(tile / (kBand * tiles_n)), in_band = tile - band * kBand * tiles_n;
  const uint32_t high = tiles_m - kBand * band < kBand ? tiles_m - kBand * band : kBand;
  const uint32_t n = uniform(in_band / high);
  return TilePlace{kBand * band + in_band - n * high, n};
}

}  // namespace ns
