// Product of float rows and a matrix of 4-bit integers with group scales (gfx950):
// y[m][n] = sum over groups g of scale[n][g] * sum over k in g of x[m][k] (code[n][k] - zero[n][g]).
//
// For few rows the codes' bytes are what has to be read, so their way through the registers has to be
// short.  The sum over a group runs on the matrix cores: a code u is put, by a shift and one
// and-or, into the mantissa of 16 as the 16-bit number 16 + u, two at a time, and sum x (16 + u) -
// (16 + zero) sum x is scaled in float32, the sums of x coming from the same instruction with ones
// as weights.  16-bit rows go in as they are.  For float32 rows the 16 + zero that is taken off
// again would cost some bits where x has a mean, so a row goes in as x - c, c its mean over the
// group, rounded to float32 and split into three bfloat16 parts, with a fourth row of ones that
// gives c its share: sum x (u - zero) = sum (x - c)(u - zero) + c (sum (16 + u) - count (16 +
// zero)), whose factor of c is exact.
//
// Operands and their products are exact, the sums are float32's: a group's is off by some 2^-24 of
// (16 + zero) sum |x|, for float32 rows of (16 + zero) sum |x - c| (sums go over 128 columns at most).
// That is some five times what a sum of x (u - zero) would be off by, and counts columns whose
// weight is zero: one value much larger than its group's others costs them bits there too.
//
// What bounds it now: requests.  One of 16 rows, 64 bytes each, takes a compute unit some 50 cycles
// whatever it brings, and the instruction's layout asks for such ones, of the codes (33.5 MB of 16 x
// 8192 to 8192: 17.2 us, 2.0 TB/s; without x, 13.1) and of x; 1 x 1024 to 50,000 10.1 us, of which
// the call's way through the host takes 9.  With more rows, the vector ALU beside the matrix cores:
// 33 x 50,000 to 1000 22.9, some 3 of them to add 49 parts of K; without any loads about 2 less.
//
// In the 16x16x32 instruction the rows of x are the first operand and 16 rows of the weight the
// second, so a lane's four results are four rows of x (for float32: one row's three parts and the
// ones) of its own row of the weight, whose codes it loaded and whose scales it needs.
#include "ns_q4.h"
#include "ns_gemm.h"

namespace ns {
namespace {

constexpr int kQ4Waves = 8, kQ4Threads = 64 * kQ4Waves;
constexpr int kStage = 128;                    // columns a wavefront takes at a time
constexpr int kRing = 1;                       // stages requested ahead

// Rows of x that 16 rows of the instruction hold.
template <class T>
constexpr int kTileRows = sizeof(T) == 4 ? 4 : 16;

// Columns of x in LDS at a time: room for two workgroups on a compute unit, with their factors (20 x
// 1024 to 50,000 in bf16 16.0 us, with 1024 columns 22.9).
constexpr int chunk_columns(int tiles) { return tiles == 1 ? 1024 : 512; }

// What a workgroup does: CT tiles of x's rows, S strips of 16 rows of the weight per wavefront,
// NG groups (or parts of one) per stage.
template <int kCT, int kS, int kNG>
struct Q4Tile {
  static constexpr int CT = kCT, S = kS, NG = kNG;
  static constexpr int chunk = chunk_columns(CT);
  static constexpr int stages = chunk / kStage, sub = kStage / NG;
  // Two tiles and strips leave a compute unit's registers to two workgroups, which hide each other's
  // waits; the others request the next chunk of x while one is multiplied, where registers last.  Us,
  // that way and the other: 20 x 1024 to 50,000 in bf16 16.1 / 22.4, 8 x 1024 to 50,000 in float32 16.7 /
  // 18.4, though 24 x 8192 to 8192 in groups of 32 26.7 / 25.2; 33 x 50,000 to 1000 26.0 / 24.8.
  static constexpr bool kTwo = CT == 2 && S == 2;
  static constexpr bool kNext = !kTwo && (CT * S < 8 || NG == 1);
};

struct Q4Place {
  uint32_t m_tiles, strip_groups, splits, parts;   // parts: wavefronts that share a strip
  uint32_t chunks, per_split;                      // chunks of columns, and of a split
};

// Codes 0 .. 3 and 4 .. 7 of a word as four registers of two 16-bit numbers 16 + u: codes i and
// i + 4 in register i.  The rows of x lie in that order too.
template <bool kHalf>
__device__ __forceinline__ v4i sixteen_plus(uint32_t word) {
  constexpr int at = kHalf ? 6 : 3;            // the place of u in the mantissa
  // The mask in a register: then and and or are one instruction, which takes one constant from
  // elsewhere (33 x 50,000 to 1000 then 24.3 us, else 24.8; 1 x 1024 to 50,000 10.1, else 10.7).
  uint32_t mask = kHalf ? 0x03C003C0u : 0x00780078u;
  constexpr uint32_t sixteen = kHalf ? 0x4C004C00u : 0x41804180u;
  asm("" : "+v"(mask));
  v4i out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t moved = 4 * i > at ? word >> (4 * i > at ? 4 * i - at : 0)
                                      : word << (4 * i > at ? 0 : at - 4 * i);
    out[i] = static_cast<int>((moved & mask) | sixteen);
  }
  return out;
}

template <class T>
__device__ __forceinline__ v4f q4_multiply(v4i x, v4i w, v4f sum) {
  if constexpr (__is_same(T, _Float16)) return multiply_pieces<_Float16>(x, w, sum);
  else return multiply_pieces<__bf16>(x, w, sum);
}

// A lane of quarter q has words 0 .. 3 of block q of its row's four; after this, word q of blocks
// 0 .. 3: a step of the instruction then takes one block, whose group is one.
__device__ __forceinline__ void swap_lanes_32(uint32_t& a, uint32_t& b) {
  const auto both = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = both[0];
  b = both[1];
}
__device__ __forceinline__ void swap_lanes_16(uint32_t& a, uint32_t& b) {
  const auto both = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = both[0];
  b = both[1];
}
__device__ __forceinline__ void deal_blocks(uint32_t (&w)[4]) {
  swap_lanes_32(w[0], w[2]);
  swap_lanes_32(w[1], w[3]);
  swap_lanes_16(w[0], w[1]);
  swap_lanes_16(w[2], w[3]);
}

// The sum over kLanes neighbouring lanes, in every one of them.
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int step = 1; step < kLanes; step *= 2) v += __shfl_xor(v, step);
  return v;
}

// What a group's sums are multiplied with, and what their offset is: -(16 + zero).
struct Q4Factors {
  float scale, offset;
};

template <class G, class T>
struct Q4Centres {};
template <class G>
struct Q4Centres<G, float> {
  float centre[G::chunk / G::sub][4 * G::CT];
};
template <class G, class T>
struct Q4Lds : Q4Centres<G, T> {
  v4i x[G::chunk / 64][16 * G::CT][8];         // pieces of eight columns, at place piece ^ turn(row)
  Q4Factors factors[G::stages * 16 * G::S * kQ4Waves][G::NG];
};

__device__ __forceinline__ int pair_of(float a, float b) {
  typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(int, v2bf{static_cast<__bf16>(a), static_cast<__bf16>(b)});
}

// A thread's pieces of a chunk of x's rows, on their way to LDS.
template <class G, class T>
struct Q4Rows {
  static constexpr int blocks = G::chunk / 8;              // of a row
  static constexpr int count = kTileRows<T> * G::CT * blocks / kQ4Threads;
  static_assert(kTileRows<T> * G::CT * blocks % kQ4Threads == 0, "whole pieces per thread");
  Pack<T, 8> v[count];
};

// Requests them.  Rows that do not exist are not read, nor is the chunk after the last.
template <class G, class T>
__device__ __forceinline__ void ask_rows(const T* x, int64_t stride, int64_t rows, int64_t first,
                                         int64_t columns, Q4Rows<G, T>& to) {
  using R = Q4Rows<G, T>;
#pragma unroll
  for (int u = 0; u < R::count; ++u) {
    const int i = threadIdx.x + u * kQ4Threads, r = i / R::blocks, b = i % R::blocks;
    const int64_t left = columns - first - 8 * b;
    const T* const from = x + r * stride + first + 8 * b;
    to.v[u] = Pack<T, 8>{};
    if (r < rows && left >= 8) {
      to.v[u] = load_pack<T, 8>(from);
    } else if (r < rows && left > 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) to.v[u].v[j] = from[j];
    }
  }
}

// Puts them into LDS.
template <class G, class T>
__device__ __forceinline__ void place_rows(const Q4Rows<G, T>& rows_of_x, int64_t rows, int64_t first,
                                           int64_t columns, Q4Lds<G, T>& lds) {
  using R = Q4Rows<G, T>;
  constexpr int kLanes = G::sub / 8;
#pragma unroll
  for (int u = 0; u < R::count; ++u) {
    const int i = threadIdx.x + u * kQ4Threads, r = i / R::blocks, b = i % R::blocks;
    if (r >= rows) break;
    const Pack<T, 8>& raw = rows_of_x.v[u];
    const int group = b / kLanes, line = b / 8, piece = b % 8;
    if constexpr (sizeof(T) == 2) {
      Pack<T, 8> turned;
#pragma unroll
      for (int j = 0; j < 4; ++j) turned.v[2 * j] = raw.v[j], turned.v[2 * j + 1] = raw.v[j + 4];
      lds.x[line][r][piece ^ turn(r)] = __builtin_bit_cast(v4i, turned);
    } else {
      const int64_t left = columns - first - 8 * b, behind = columns - (first + group * G::sub);
      const float count = behind < G::sub ? (behind > 0 ? static_cast<float>(behind) : 0.0f)
                                          : static_cast<float>(G::sub);
      float sum = 0.0f, rest[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += raw.v[j];
      const float centre = count > 0.0f ? lanes_sum<kLanes>(sum) / count : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) rest[j] = j < left ? raw.v[j] - centre : 0.0f;
      const int slot = 16 * (r >> 2) + 4 * (r & 3);
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        float own[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          own[j] = static_cast<float>(static_cast<__bf16>(rest[j]));
          rest[j] -= own[j];
        }
        lds.x[line][slot + part][piece ^ turn(slot + part)] =
            v4i{pair_of(own[0], own[4]), pair_of(own[1], own[5]), pair_of(own[2], own[6]),
                pair_of(own[3], own[7])};
      }
      float one[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) one[j] = j < left ? 1.0f : 0.0f;
      lds.x[line][slot + 3][piece ^ turn(slot + 3)] =
          v4i{pair_of(one[0], one[4]), pair_of(one[1], one[5]), pair_of(one[2], one[6]),
              pair_of(one[3], one[7])};
      if (b % kLanes == 0) lds.centre[group][r] = centre;
    }
  }
}

// Scales and zeros as they are in memory, so that nothing waits for them before they are used.
template <int NG>
struct Q4Scales {
  uint32_t scale[NG], zeros;                     // of 32 bits each, or of 16 side by side; bytes
};

// Scales and zeros of groups first .. first + NG - 1 of a row that begins at `at`; past its last
// group, where x is zero, that one's.
template <int NG>
__device__ __forceinline__ void load_scales(const Q4View& w, int64_t at, int first, Q4Scales<NG>& to) {
  const int groups = static_cast<int>(w.groups);
  to.zeros = 0x08080808u;
  if (w.scale_type == NS_TYPE_F32 || first + NG > groups) {
#pragma unroll
    for (int g = 0; g < NG; ++g) to.scale[g] = 0;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int64_t own = at + (first + g < groups ? first + g : groups - 1);
      if (w.scale_type == NS_TYPE_F32)
        to.scale[g] = static_cast<const uint32_t*>(w.scales)[own];
      else
        to.scale[g / 2] |= static_cast<uint32_t>(static_cast<const uint16_t*>(w.scales)[own]) << (g % 2 * 16);
    }
    if (w.zeros) {
      to.zeros = 0;
#pragma unroll
      for (int g = 0; g < NG; ++g)
        to.zeros |= static_cast<uint32_t>(w.zeros[at + (first + g < groups ? first + g : groups - 1)]) << (8 * g);
    }
  } else {
    to.scale[0] = 0;
    __builtin_memcpy(to.scale, static_cast<const uint16_t*>(w.scales) + at + first, 2 * NG);
    if (w.zeros) {
      to.zeros = 0;
      __builtin_memcpy(&to.zeros, w.zeros + at + first, NG);
    }
  }
}

template <int NG>
__device__ __forceinline__ uint32_t raw_scale(const Q4Scales<NG>& s, int g, int32_t type) {
  const uint32_t half = g & 1 ? s.scale[g / 2] >> 16 : s.scale[g / 2] & 0xFFFFu;
  return type == NS_TYPE_F32 ? s.scale[g] : half;
}
template <int NG>
__device__ __forceinline__ float zero_offset(const Q4Scales<NG>& s, int g) {
  return -16.0f - static_cast<float>(s.zeros >> (8 * g) & 255u);
}

__device__ __forceinline__ float scale_value(uint32_t raw, int32_t type) {
  if (type == NS_TYPE_F32) return __builtin_bit_cast(float, raw);
  if (type == NS_TYPE_BF16) return __builtin_bit_cast(float, raw << 16);
  return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(raw)));
}

// A workgroup's factors come through LDS, laid there by threads that read a row's neighbouring
// ones: read where they are used, 2 to 8 bytes of 16 rows at a time, they take as long as the codes
// (1 x 8192 to 8192, groups of 128, in bf16 16.7 us, so 12.6).  By stage, then row, rows turned by
// the stage so that neighbouring threads store to different banks; of 2^shift stages from `base` on,
// `rows` rows (a power of two) from `row` on, kEach of them a thread.
struct Q4Table {
  int64_t row;
  int rows, shift, base, last;                   // of the last stage there is
  uint32_t per_group;                            // stages of a group, where it has some
};

template <int NG>
__device__ __forceinline__ int factors_place(const Q4Table& t, int stage, int row) {
  const int turn = 1 << t.shift < 32 / NG ? 32 / NG >> t.shift : 1;
  return (stage << __builtin_ctz(t.rows)) + (row ^ (stage * turn & (t.rows - 1)));
}

template <int NG, int kEach>
__device__ __forceinline__ void ask_factors(const Q4View& w, const Q4Table& t, Q4Scales<NG> (&to)[kEach]) {
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int id = threadIdx.x + u * kQ4Threads, stage = t.base + (id & ((1 << t.shift) - 1));
    const int64_t n = t.row + (id >> t.shift), row = n < w.rows ? n : w.rows - 1;
    const int at = stage < t.last ? stage : t.last;
    if (u * kQ4Threads < t.rows << t.shift)
      load_scales<NG>(w, row * w.groups, NG == 1 ? static_cast<int>(at / t.per_group) : at * NG, to[u]);
  }
}

template <int NG, int kEach>
__device__ __forceinline__ void place_factors(const Q4View& w, const Q4Table& t, const Q4Scales<NG> (&from)[kEach],
                                              Q4Factors (*to)[NG]) {
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int id = threadIdx.x + u * kQ4Threads;
    if (id >= t.rows << t.shift) break;
    Q4Factors* const place = to[factors_place<NG>(t, id & ((1 << t.shift) - 1), id >> t.shift)];
#pragma unroll
    for (int g = 0; g < NG; ++g)
      place[g] = Q4Factors{scale_value(raw_scale(from[u], g, w.scale_type), w.scale_type),
                           zero_offset(from[u], g)};
  }
}

template <class G, class T>
__global__ __launch_bounds__(kQ4Threads, G::kTwo ? 4 : 2) void q4_product(Q4View w, Q4Place p, const T* x,
                                                         int64_t x_stride, int64_t rows,
                                                         const float* bias, T* out, int64_t stride,
                                                         float* partials) {
  __shared__ union {
    Q4Lds<G, T> in;
    v4f sums[kQ4Waves][G::S][G::CT][64];
  } lds;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), q = lane >> 4;
  // Each XCD gets a run of workgroups, the rows' tiles of a strip group side by side, so that its
  // codes are read into one L2.
  const uint32_t share = gridDim.x / kXcds;
  uint32_t id = blockIdx.x < share * kXcds ? blockIdx.x % kXcds * share + blockIdx.x / kXcds : blockIdx.x;
  const uint32_t line = uniform(id / p.m_tiles), m_tile = id - line * p.m_tiles;
  const uint32_t split = uniform(line / p.strip_groups), strip_group = line - split * p.strip_groups;
  const uint32_t part = wave % p.parts;
  const int64_t m0 = static_cast<int64_t>(m_tile) * (kTileRows<T> * G::CT);
  const int64_t n0 =
      (static_cast<int64_t>(strip_group) * (kQ4Waves / p.parts) + wave / p.parts) * (16 * G::S);

  const int stages = static_cast<int>((w.blocks + 3) / 4), blocks = static_cast<int>(w.blocks);
  const int first_chunk = static_cast<int>(split * p.per_split);
  const int last_chunk = first_chunk + static_cast<int>(p.per_split) < static_cast<int>(p.chunks)
                             ? first_chunk + static_cast<int>(p.per_split) : static_cast<int>(p.chunks);
  const int limit = last_chunk * G::stages < stages ? last_chunk * G::stages : stages;
  const uint32_t per_group = G::NG == 1 ? static_cast<uint32_t>(w.group / kStage) : 1;

  // A lane's rows of the weight.
  const uint8_t* codes[G::S];
#pragma unroll
  for (int s = 0; s < G::S; ++s) {
    const int64_t n = n0 + 16 * s + (lane & 15), row = n < w.rows ? n : w.rows - 1;
    codes[s] = w.codes + row * blocks * 16;
  }
  uint32_t ring[kRing][G::S][4];
  const auto load = [&](int stage, uint32_t (&to)[G::S][4]) __attribute__((always_inline)) {
    // Past the last block, x is zero: any codes do.
    const int block = 4 * stage + q < blocks ? 4 * stage + q : blocks - 1;
#pragma unroll
    for (int s = 0; s < G::S; ++s)
      __builtin_memcpy(to[s], codes[s] + static_cast<uint32_t>(block) * 16, 16);
  };
  // The factors of the workgroup's rows.
  const int own_rows = kQ4Waves / static_cast<int>(p.parts) * (16 * G::S);
  const int first_row = static_cast<int>(wave / p.parts) * (16 * G::S);
  Q4Table table{static_cast<int64_t>(strip_group) * own_rows, own_rows, __builtin_ctz(G::stages), 0, limit - 1,
                per_group};

  constexpr int kOnes = __is_same(T, _Float16) ? 0x3C003C00 : 0x3F803F80;
  const v4i ones = {kOnes, kOnes, kOnes, kOnes};
  v4f total[G::S][G::CT] = {};
  const auto compute = [&](int stage, uint32_t (&from)[G::S][4]) __attribute__((always_inline)) {
    const int own = stage % G::stages;                   // in the chunk
    const Q4Factors* by[G::S];
#pragma unroll
    for (int s = 0; s < G::S; ++s)
      by[s] = lds.in.factors[factors_place<G::NG>(table, own, first_row + 16 * s + (lane & 15))];
#pragma unroll
    for (int s = 0; s < G::S; ++s) deal_blocks(from[s]);
#pragma unroll
    for (int g = 0; g < G::NG; ++g) {
      v4f sum[G::S][G::CT] = {}, taken[G::CT] = {};
      constexpr int kSteps = 4 / G::NG;
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        const int e = g * kSteps + step;
        v4i rows_of_x[G::CT];
#pragma unroll
        for (int t = 0; t < G::CT; ++t) {
          rows_of_x[t] = lds.in.x[2 * own + e / 2][16 * t + (lane & 15)][(4 * (e & 1) + q) ^ turn(lane & 15)];
          taken[t] = q4_multiply<T>(rows_of_x[t], ones, taken[t]);
        }
#pragma unroll
        for (int s = 0; s < G::S; ++s) {
          const v4i codes = sixteen_plus<__is_same(T, _Float16)>(from[s][e]);
#pragma unroll
          for (int t = 0; t < G::CT; ++t) sum[s][t] = q4_multiply<T>(rows_of_x[t], codes, sum[s][t]);
        }
      }
      const int group = own * G::NG + g;
#pragma unroll
      for (int s = 0; s < G::S; ++s) {
        const float offset = by[s][g].offset, scale = by[s][g].scale;
#pragma unroll
        for (int t = 0; t < G::CT; ++t) {
          float own_sum[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) own_sum[i] = fmaf(offset, taken[t][i], sum[s][t][i]);
          if constexpr (sizeof(T) == 4) {
            const float parts = (own_sum[2] + own_sum[1]) + own_sum[0];
            const float whole = fmaf(lds.in.centre[group][4 * t + q], own_sum[3], parts);
            total[s][t][0] = fmaf(scale, whole, total[s][t][0]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) total[s][t][i] = fmaf(scale, own_sum[i], total[s][t][i]);
          }
        }
      }
      // Four groups one after the other: side by side they do not fit the registers.
      if constexpr (G::NG == 4) {
#pragma unroll
        for (int s = 0; s < G::S; ++s)
#pragma unroll
          for (int t = 0; t < G::CT; ++t) asm volatile("" : "+v"(total[s][t]) :: "memory");
      }
    }
  };

  // The wavefronts of a strip take its stages in turn; a chunk has a multiple of kRing for each.
  const int step = static_cast<int>(p.parts);
  int stage = first_chunk * G::stages + static_cast<int>(part);
  const T* const own_x = x + m0 * x_stride;
#pragma unroll
  for (int u = 0; u < kRing; ++u)
    if (stage + u * step < limit) load(stage + u * step, ring[u]);
  Q4Rows<G, T> rows_of_x;
  Q4Scales<G::NG> raw[G::stages * 16 * G::S * kQ4Waves / kQ4Threads];
  const auto ask = [&](int chunk) __attribute__((always_inline)) {
    ask_rows<G, T>(own_x, x_stride, rows - m0, static_cast<int64_t>(chunk) * G::chunk, w.columns, rows_of_x);
    table.base = chunk * G::stages;
    ask_factors<G::NG>(w, table, raw);
  };
  if (G::kNext) ask(first_chunk);
  for (int chunk = first_chunk; chunk < last_chunk; ++chunk) {
    const int64_t first = static_cast<int64_t>(chunk) * G::chunk;
    if (!G::kNext) ask(chunk);
    if (chunk > first_chunk) __syncthreads();              // all have read the one before
    place_rows<G, T>(rows_of_x, rows - m0, first, w.columns, lds.in);
    place_factors<G::NG>(w, table, raw, lds.in.factors);
    __syncthreads();
    if (G::kNext && chunk + 1 < last_chunk) ask(chunk + 1);
    for (int end = (chunk + 1) * G::stages; stage < end; stage += kRing * step) {
#pragma unroll
      for (int u = 0; u < kRing; ++u) {
        const int now = stage + u * step;
        if (now < limit) {
          compute(now, ring[u]);
          if (now + kRing * step < limit) load(now + kRing * step, ring[u]);
        }
      }
    }
  }

  if (p.parts > 1) {
    __syncthreads();
#pragma unroll
    for (int s = 0; s < G::S; ++s)
#pragma unroll
      for (int t = 0; t < G::CT; ++t) lds.sums[wave][s][t][lane] = total[s][t];
    __syncthreads();
    if (part) return;
    for (int other = 1; other < step; ++other)
#pragma unroll
      for (int s = 0; s < G::S; ++s)
#pragma unroll
        for (int t = 0; t < G::CT; ++t) total[s][t] += lds.sums[wave + other][s][t][lane];
  }
#pragma unroll
  for (int s = 0; s < G::S; ++s) {
    const int64_t n = n0 + 16 * s + (lane & 15);
    if (n >= w.rows) continue;
    const float more = bias ? bias[n] : 0.0f;
#pragma unroll
    for (int t = 0; t < G::CT; ++t)
#pragma unroll
      for (int i = 0; i < (sizeof(T) == 4 ? 1 : 4); ++i) {
        const int64_t m = m0 + (sizeof(T) == 4 ? 4 * t + q : 16 * t + 4 * q + i);
        if (m >= rows) continue;
        if (p.splits > 1) partials[(split * rows + m) * w.rows + n] = total[s][t][i];
        else out[m * stride + n] = static_cast<T>(total[s][t][i] + more);
      }
  }
}

// Up to 16 rows of 16 bits go from memory to registers: a workgroup's wavefronts share S strips
// and take their stages in turn, so each reads its own part of x, without barriers but for the
// factors and for the sums at the end.
constexpr int kRowRing = 1, kFactorStages = 8 * kQ4Waves;

template <int NG, int S>
struct Q4RowStage {
  v4i x[4];
  uint32_t codes[S][4];
};

template <class T, int NG, int S>
__global__ __launch_bounds__(kQ4Threads) void q4_rows(Q4View w, Q4Place p, const T* x, int64_t x_stride,
                                                      int64_t rows, const float* bias, T* out,
                                                      int64_t stride, float* partials) {
  __shared__ union {
    Q4Factors factors[kFactorStages * 16 * S][NG];
    v4f sums[kQ4Waves][S][64];
  } lds;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), q = lane >> 4;
  const uint32_t split = uniform(blockIdx.x / p.strip_groups), strip_group = blockIdx.x - split * p.strip_groups;
  const int part = static_cast<int>(wave % p.parts), step = static_cast<int>(p.parts);
  const int own_rows = kQ4Waves / step * (16 * S);         // of the workgroup
  const int64_t group_row = static_cast<int64_t>(strip_group) * own_rows;
  const int first_row = wave / step * (16 * S);
  const int blocks = static_cast<int>(w.blocks), stages = (blocks + 3) / 4;
  const int begin = static_cast<int>(split * p.per_split);
  const int limit = begin + static_cast<int>(p.per_split) < stages ? begin + static_cast<int>(p.per_split) : stages;
  const uint32_t per_group = NG == 1 ? static_cast<uint32_t>(w.group / kStage) : 1;
  const int64_t m = (lane & 15) < rows ? lane & 15 : rows - 1;
  const T* const own_x = x + m * x_stride + 8 * q;
  const uint8_t* codes[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int64_t n = group_row + first_row + 16 * s + (lane & 15), row = n < w.rows ? n : w.rows - 1;
    codes[s] = w.codes + row * blocks * 16;
  }
  const int whole = static_cast<int>(w.columns / kStage);  // stages that lie within the columns
  Q4RowStage<NG, S> ring[kRowRing];
  const auto load = [&](int stage, Q4RowStage<NG, S>& to) __attribute__((always_inline)) {
    const int block = 4 * stage + q < blocks ? 4 * stage + q : blocks - 1;
#pragma unroll
    for (int s = 0; s < S; ++s)
      __builtin_memcpy(to.codes[s], codes[s] + static_cast<uint32_t>(block) * 16, 16);
    const T* const from = own_x + static_cast<int64_t>(stage) * kStage;
    if (stage < whole) {
#pragma unroll
      for (int e = 0; e < 4; ++e) __builtin_memcpy(&to.x[e], from + 32 * e, 16);
    } else {
      const int left = static_cast<int>(w.columns - static_cast<int64_t>(stage) * kStage) - 8 * q;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        Pack<T, 8> v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v.v[j] = 32 * e + j < left ? from[32 * e + j] : T{};
        to.x[e] = __builtin_bit_cast(v4i, v);
      }
    }
  };
  // Factors of up to 8 `step` stages at a time; no more than there are stages of (a power of two).
  int shift = __builtin_ctz(kFactorStages / kQ4Waves * p.parts);
  while (shift > 0 && 1 << (shift - 1) >= limit - begin) --shift;
  const int span = 1 << shift;
  Q4Table table{group_row, own_rows, shift, begin, limit - 1, per_group};
  constexpr int kOnes = __is_same(T, _Float16) ? 0x3C003C00 : 0x3F803F80;
  const v4i ones = {kOnes, kOnes, kOnes, kOnes};
  v4f total[S] = {};
  const auto compute = [&](Q4RowStage<NG, S>& from, int place) __attribute__((always_inline)) {
    const Q4Factors* by[S];
#pragma unroll
    for (int s = 0; s < S; ++s)
      by[s] = lds.factors[factors_place<NG>(table, place, first_row + 16 * s + (lane & 15))];
#pragma unroll
    for (int s = 0; s < S; ++s) deal_blocks(from.codes[s]);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      v4f sum[S] = {}, taken = {};
#pragma unroll
      for (int e = g * (4 / NG); e < (g + 1) * (4 / NG); ++e) {
        // Values 0 .. 7 in the order that sixteen_plus leaves the codes in.
        v4i v;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] = static_cast<int>(__builtin_amdgcn_perm(
              static_cast<uint32_t>(from.x[e][2 + i / 2]), static_cast<uint32_t>(from.x[e][i / 2]),
              i & 1 ? 0x07060302u : 0x05040100u));
        taken = q4_multiply<T>(v, ones, taken);
#pragma unroll
        for (int s = 0; s < S; ++s)
          sum[s] = q4_multiply<T>(v, sixteen_plus<__is_same(T, _Float16)>(from.codes[s][e]), sum[s]);
      }
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const Q4Factors own = by[s][g];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          total[s][i] = fmaf(own.scale, fmaf(own.offset, taken[i], sum[s][i]), total[s][i]);
      }
      // One group after the other, in few registers.
#pragma unroll
      for (int s = 0; s < S; ++s) asm volatile("" : "+v"(total[s]) :: "memory");
    }
  };
#pragma unroll
  for (int u = 0; u < kRowRing; ++u)
    if (begin + part + u * step < limit) load(begin + part + u * step, ring[u]);
  for (int base = begin; base < limit; base += span) {
    if (base > begin) __syncthreads();                     // all have read the factors before
    Q4Scales<NG> raw[kFactorStages * 16 * S / kQ4Threads];
    table.base = base;
    ask_factors<NG>(w, table, raw);
    place_factors<NG>(w, table, raw, lds.factors);
    __syncthreads();
    const int end = base + span < limit ? base + span : limit;
    for (int stage = base + part; stage < end; stage += kRowRing * step) {
#pragma unroll
      for (int u = 0; u < kRowRing; ++u) {
        const int now = stage + u * step;
        if (now < end) {
          compute(ring[u], now - base);
          if (now + kRowRing * step < limit) load(now + kRowRing * step, ring[u]);
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < S; ++s) lds.sums[wave][s][lane] = total[s];
  __syncthreads();
  // The workgroup's strips, 256 results each, a column of the weight's rows by its threads.
  for (int id = threadIdx.x; id < own_rows * 16; id += kQ4Threads) {
    const int strip = id >> 8, column = id & 15, row = id >> 4 & 15, first = strip / S * step;
    const int from = (row >> 2) * 16 + column;             // the lane that holds it
    const int64_t n = group_row + 16 * strip + column;
    if (row >= rows || n >= w.rows) continue;
    float value = 0.0f;
    for (int k = 0; k < step; ++k)
      value += reinterpret_cast<const float*>(&lds.sums[first + k][strip % S][from])[row & 3];
    if (p.splits > 1) partials[(split * rows + row) * w.rows + n] = value;
    else out[row * stride + n] = static_cast<T>(value + (bias ? bias[n] : 0.0f));
  }
}

// The parts of K added in order, kAhead requested at a time: 32 of many parts (33 x 50,000 to 1000,
// 49 parts, with 32 / 8 22.9 / 24.3 us), 8 of few (40 x 4096 to 4096, 8 parts, 14.4 / 13.4).
constexpr int kAddThreads = 64;
template <class T, uint32_t kAhead>
__global__ __launch_bounds__(kAddThreads) void add_splits(const float* __restrict__ partials,
                                                       uint32_t splits, int64_t rows, int64_t columns,
                                                       const float* bias, T* out, int64_t stride) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kAddThreads + threadIdx.x;
  if (id >= rows * columns) return;
  float sum = 0.0f;
  for (uint32_t k = 0; k < splits; k += kAhead) {
    float v[kAhead];
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u)
      v[u] = partials[(k + u < splits ? k + u : k) * rows * columns + id];
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) sum += k + u < splits ? v[u] : 0.0f;
  }
  const int64_t m = id / columns, n = id - m * columns;
  out[m * stride + n] = static_cast<T>(sum + (bias ? bias[n] : 0.0f));
}

// y = bias where there is nothing to sum.
template <class T>
__global__ __launch_bounds__(kThreads) void bias_rows(int64_t rows, int64_t columns, const float* bias,
                                                      T* out, int64_t stride) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= rows * columns) return;
  const int64_t m = id / columns, n = id - m * columns;
  out[m * stride + n] = static_cast<T>(bias ? bias[n] : 0.0f);
}

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

// How a product is cut: tiles of x's rows per workgroup (0: q4_rows), strips per wavefront,
// wavefronts that share a strip, and parts of K that workgroups share, so that 2048 wavefronts or
// more stream codes.
struct Q4Plan {
  int tiles, strips;
  Q4Place place;
  int64_t groups;              // workgroups
};

Q4Plan rows_plan(int64_t m, int64_t n, int64_t k) {
  Q4Plan plan{};
  const int64_t stages = (k + kStage - 1) / kStage;
  // More strips a wavefront read x less often, but leave fewer workgroups; with few rows x costs
  // little.  Us with one / two / four: 8 x 4096 to 8192 10.0 / 9.0 / 12.2, 16 x 8192 to 8192 23.3 / 17.2 / 24.9,
  // 16 x 4096 to 12,288 19.1 / 15.4 / 13.9, 16 x 4096 to 16,384 22.8 / 15.2 / 14.0, 4 x 2048 to 32,768 15.8 /
  // 12.2 / 14.1.
  plan.strips = n <= 16 * 256 ? 1 : m <= 8 || n < 64 * 192 ? 2 : 4;
  const int64_t strips = (n + 16 * plan.strips - 1) / (16 * plan.strips);
  int64_t parts = 1;
  // Four stages a wavefront and more: with two 8 x 1024 to 50,000 takes 15.9 us, not 14.3, and 4 x 2048
  // to 32,768 14.1, not 12.2.
  while (parts < kQ4Waves && stages >= 8 * parts) parts *= 2;
  const int64_t strip_groups = (strips * parts + kQ4Waves - 1) / kQ4Waves;
  int64_t splits = 1;
  if (strip_groups < 128) {
    splits = 512 / strip_groups;
    splits = splits < stages / (4 * parts) ? splits : stages / (4 * parts);
    splits = splits > 1 ? splits : 1;
  }
  const int64_t per = (stages + splits - 1) / splits;
  splits = (stages + per - 1) / per;                       // no empty part
  plan.groups = strip_groups * splits;
  plan.place = Q4Place{1, static_cast<uint32_t>(strip_groups), static_cast<uint32_t>(splits),
                       static_cast<uint32_t>(parts), 0, static_cast<uint32_t>(per)};
  return plan;
}

Q4Plan q4_plan(int64_t m, int64_t n, int64_t k, int32_t type) {
  if (type != NS_TYPE_F32 && m <= 16) return rows_plan(m, n, k);
  Q4Plan plan{};
  const int64_t per_tile = type == NS_TYPE_F32 ? 4 : 16, tiles = (m + per_tile - 1) / per_tile;
  plan.tiles = tiles <= 2 ? static_cast<int>(tiles) : tiles == 3 && type != NS_TYPE_F32 ? 3 : 4;
  const int64_t m_tiles = (tiles + plan.tiles - 1) / plan.tiles;
  const int64_t columns = chunk_columns(plan.tiles), chunks = (k + columns - 1) / columns;
  // Two strips a wavefront halve what is read of x from LDS for each, but also the wavefronts.  Us,
  // one / two, bf16: 40 x 4096 to 4096 13.9 / 16.3, 64 x 2048 to 16,384 25.7 / 25.5, 33 x 50,000 to 1000
  // 28.2 / 24.8.
  const bool few = type != NS_TYPE_F32 && m_tiles * ((n + 15) / 16) * chunks <= 2048;
  plan.strips = plan.tiles == 1 || few ? 1 : 2;
  const int64_t strips = (n + 16 * plan.strips - 1) / (16 * plan.strips);
  int64_t parts = 1;
  while (parts * 2 <= 4 / plan.tiles && m_tiles * strips * parts < 2048) parts *= 2;
  const int64_t waves = m_tiles * strips * parts;
  int64_t splits = waves < 2048 ? 2048 / waves : 1;
  splits = splits < chunks ? splits : chunks;
  const int64_t per = splits > 0 ? (chunks + splits - 1) / splits : 1;
  splits = per > 0 ? (chunks + per - 1) / per : 1;         // no empty part
  const int64_t strip_groups = (strips * parts + kQ4Waves - 1) / kQ4Waves;
  plan.groups = m_tiles * strip_groups * splits;
  plan.place = Q4Place{static_cast<uint32_t>(m_tiles), static_cast<uint32_t>(strip_groups),
                       static_cast<uint32_t>(splits), static_cast<uint32_t>(parts),
                       static_cast<uint32_t>(chunks), static_cast<uint32_t>(per)};
  return plan;
}

template <class G, class T>
int run_tile(const ns_q4_product_args* a, const Q4Plan& plan, hipStream_t stream) {
  q4_product<G, T><<<dim3(static_cast<unsigned>(plan.groups)), dim3(kQ4Threads), 0, stream>>>(
      q4_view(a->weight), plan.place, static_cast<const T*>(a->x), a->x_stride, a->rows, a->bias,
      static_cast<T*>(a->out), a->stride, a->workspace);
  return launched("4-bit product");
}

template <class T, int kNG, int kS>
int run_rows(const ns_q4_product_args* a, const Q4Plan& plan, hipStream_t stream) {
  q4_rows<T, kNG, kS><<<dim3(static_cast<unsigned>(plan.groups)), dim3(kQ4Threads), 0, stream>>>(
      q4_view(a->weight), plan.place, static_cast<const T*>(a->x), a->x_stride, a->rows, a->bias,
      static_cast<T*>(a->out), a->stride, a->workspace);
  return launched("4-bit product");
}

template <class T, int kNG>
int run_groups(const ns_q4_product_args* a, const Q4Plan& plan, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (plan.tiles == 0)
      return plan.strips == 1   ? run_rows<T, kNG, 1>(a, plan, stream)
             : plan.strips == 2 ? run_rows<T, kNG, 2>(a, plan, stream)
                                : run_rows<T, kNG, 4>(a, plan, stream);
    if (plan.tiles == 3)
      return plan.strips == 1 ? run_tile<Q4Tile<3, 1, kNG>, T>(a, plan, stream)
                              : run_tile<Q4Tile<3, 2, kNG>, T>(a, plan, stream);
    if (plan.strips == 1)
      return plan.tiles == 2 ? run_tile<Q4Tile<2, 1, kNG>, T>(a, plan, stream)
                             : run_tile<Q4Tile<4, 1, kNG>, T>(a, plan, stream);
  } else {
    if (plan.tiles == 1) return run_tile<Q4Tile<1, 1, kNG>, T>(a, plan, stream);
  }
  if (plan.tiles == 2) return run_tile<Q4Tile<2, 2, kNG>, T>(a, plan, stream);
  return run_tile<Q4Tile<4, 2, kNG>, T>(a, plan, stream);
}

template <class T>
int run(const ns_q4_product_args* a, hipStream_t stream) {
  const int64_t m = a->rows, n = a->weight.rows, results = (m * n + kThreads - 1) / kThreads;
  if (results > INT32_MAX) return fail("the product is too large for one launch");
  if (a->weight.columns == 0) {
    bias_rows<T><<<dim3(static_cast<unsigned>(results)), dim3(kThreads), 0, stream>>>(
        m, n, a->bias, static_cast<T*>(a->out), a->stride);
    return launched("4-bit product");
  }
  const Q4Plan plan = q4_plan(m, n, a->weight.columns, a->type);
  if (plan.groups > INT32_MAX) return fail("the product is too large for one launch");
  if (plan.place.splits > 1 && !a->workspace) return fail("the product needs its workspace");
  int rc;
  switch (a->weight.group) {
    case 32: rc = run_groups<T, 4>(a, plan, stream); break;
    case 64: rc = run_groups<T, 2>(a, plan, stream); break;
    default: rc = run_groups<T, 1>(a, plan, stream); break;
  }
  if (rc || plan.place.splits == 1) return rc;
  const dim3 grid(static_cast<unsigned>((m * n + kAddThreads - 1) / kAddThreads));
  if (plan.place.splits > 24)
    add_splits<T, 32><<<grid, dim3(kAddThreads), 0, stream>>>(
        a->workspace, plan.place.splits, m, n, a->bias, static_cast<T*>(a->out), a->stride);
  else
    add_splits<T, 8><<<grid, dim3(kAddThreads), 0, stream>>>(
        a->workspace, plan.place.splits, m, n, a->bias, static_cast<T*>(a->out), a->stride);
  return launched("4-bit product parts");
}

}  // namespace
}  // namespace ns

extern "C" {

int64_t ns_q4_product_floats(int64_t m, int64_t n, int64_t k, int32_t type) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const ns::Q4Plan plan = ns::q4_plan(m, n, k, type);
  return plan.place.splits > 1 ? plan.place.splits * m * n : 0;
}

int ns_q4_product(const ns_q4_product_args* a, void* stream) {
  ns::clear_error();
  if (!a) return ns::fail("product arguments are required");
  if (int rc = ns::check_q4(a->weight)) return rc;
  if (a->rows < 0) return ns::fail("rows must not be negative");
  if (a->rows == 0 || a->weight.rows == 0) return NS_OK;
  if ((a->weight.columns && !a->x) || !a->out) return ns::fail("x and the output are required");
  auto queue = static_cast<hipStream_t>(stream);
  switch (a->type) {
    case NS_TYPE_F32: return ns::run<float>(a, queue);
    case NS_TYPE_BF16: return ns::run<__bf16>(a, queue);
    case NS_TYPE_F16: return ns::run<_Float16>(a, queue);
    default: return ns::fail("unknown element type");
  }
}

}  // extern "C"
