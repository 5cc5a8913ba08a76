// Product of two microscaled 4-bit matrices, y = a b^T + bias (gfx950).
//
// The matrix cores take e2m1 codes and block scales as they are stored: in
// mfma_scale 16x16x128, lane l holds row l%16 of an operand, block l/16 of four (16 bytes
// of codes, one scale byte), so a lane's operand is one 16-byte load; the 16x16 result has
// column l%16 and rows 4*(l/16) .. +3 in lane l's four registers.
#include <cstddef>

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

// Geometry of a tile kernel: WM x WN wavefronts, each MI x NJ results of 16x16; K goes in
// stages of KS steps of 128 values.
template <int kMI, int kNJ, int kWM, int kWN, int kKS>
struct Tile {
  static constexpr int MI = kMI, NJ = kNJ, WM = kWM, WN = kWN, KS = kKS;
  static constexpr int rows_m = 16 * MI * WM, rows_n = 16 * NJ * WN, rows = rows_m + rows_n;
  static constexpr int threads = 64 * WM * WN;
  static constexpr int loads = rows * KS * 4 / threads;    // 16-byte pieces per thread and stage
  static constexpr int scale_rows = (rows + threads - 1) / threads;
  static_assert(rows * KS * 4 % threads == 0, "whole pieces per thread");
  static_assert(rows_m % (threads / 8) == 0, "a load instruction reads one operand");
  static_assert(KS == 2, "a stage's scales of a row are one 8-byte word");
};

// One stage's operands in LDS.  Codes: rows of 8 blocks, 128 bytes, a whole cache line each,
// with block k of row r at place k ^ (r/2 % 8): a fragment, blocks 4s .. 4s+3 of 16 rows, is then
// read without bank conflicts (so it is with r % 8; blocks 0, 2, 4, 6 would conflict).  Scale
// bytes of (step 0, step 1) as one 16-bit word per (wavefront row, lane, strip), so a lane reads
// all its strips' scales at once and the instruction picks the byte it needs.
template <class G>
struct Stage {
  v4i codes[G::rows * 8];
  uint16_t scales_a[G::WM][64][G::MI];
  uint16_t scales_b[G::WN][64][G::NJ];
};

// The rows a tile reads of one operand, as a buffer whose reads past its end give zeros.
struct MxPanel {
  __amdgpu_buffer_rsrc_t codes;
  const uint8_t* scales;       // of the panel's first row
  int blocks;
  int last;                    // last row
  uint32_t row_bytes;
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return __builtin_amdgcn_readfirstlane(v);
}

__device__ __forceinline__ MxPanel panel(const MxView& m, int64_t row, int rows) {
  const uint32_t own = uniform(static_cast<uint32_t>(m.rows - row < rows ? m.rows - row : rows));
  const uint32_t row_bytes = uniform(static_cast<uint32_t>(m.blocks) * 16);
  const uint64_t base = reinterpret_cast<uint64_t>(m.codes + row * row_bytes);
  const uint64_t low = uniform(static_cast<uint32_t>(base)), high = uniform(base >> 32);
  return MxPanel{__builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(high << 32 | low), 0,
                                                   static_cast<int>(own * row_bytes), 0x00020000),
                 m.scales + row * m.blocks, static_cast<int>(m.blocks), static_cast<int>(own) - 1,
                 row_bytes};
}

// Requests stage `block` .. of both panels' codes straight into LDS, eight rows of 128 bytes
// per instruction: lane l fills place l%8 of row l/8.  Rows that do not exist read as zeros;
// so do, in a row's last, partial stage (kWhole false), blocks from `stop` on.  (With 16 rows
// of 64 bytes per instruction, in the order the fragments are read in, the product of 4096 x
// 4096 by 32768 took 377 us: the L1 fetched every line twice.)
template <bool kWhole>
__device__ __forceinline__ void read_piece(const MxPanel& m, bool inside, uint32_t row,
                                           uint32_t column, v4i* to) {
  const uint32_t offset = kWhole || inside ? row * m.row_bytes + column : 0xFFFFFFF0u;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      m.codes, reinterpret_cast<__attribute__((address_space(3))) void*>(reinterpret_cast<uintptr_t>(to)),
      16, static_cast<int>(offset), 0, 0, 0);
}

template <class G, bool kWhole>
__device__ __forceinline__ void request_codes(const MxPanel& a, const MxPanel& b, int block, int stop,
                                              int wave, int lane, Stage<G>& to) {
  constexpr int kPerRound = G::threads / 8;                // rows per load instruction of all waves
  const uint32_t row = 8 * wave + (lane >> 3);
  const int at = block + static_cast<int>((lane & 7) ^ (row >> 1 & 7));
  const uint32_t column = static_cast<uint32_t>(at) * 16;
  const bool inside = at < stop;
  constexpr int kLoadsA = G::rows_m / kPerRound;           // the first ones are a's
#pragma unroll
  for (int i = 0; i < kLoadsA; ++i)
    read_piece<kWhole>(a, inside, row + kPerRound * i, column, &to.codes[i * G::threads + 64 * wave]);
#pragma unroll
  for (int i = kLoadsA; i < G::loads; ++i)
    read_piece<kWhole>(b, inside, row + kPerRound * (i - kLoadsA), column,
                       &to.codes[i * G::threads + 64 * wave]);
}

// A thread's rows' scale bytes of a stage (past K: scale 1).
template <class G>
struct Scales {
  uint32_t word[G::scale_rows][2];
};

template <class G, bool kWhole>
__device__ __forceinline__ void request_scales(const MxPanel& a, const MxPanel& b, int block,
                                               int stop, Scales<G>& next) {
#pragma unroll
  for (int i = 0; i < G::scale_rows; ++i) {
    const int piece = i * G::threads + static_cast<int>(threadIdx.x);
    if (G::rows % G::threads == 0 || piece < G::rows) {
      const bool of_a = piece < G::rows_m;
      const int own = of_a ? piece : piece - G::rows_m, end = of_a ? a.last : b.last;
      // A row that does not exist reads the last one's: its results are not stored.
      const uint8_t* from = (of_a ? a.scales : b.scales) +
                            static_cast<int64_t>(own < end ? own : end) * a.blocks + block;
      if constexpr (kWhole) {
        __builtin_memcpy(next.word[i], from, 8);
      } else {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          next.word[i][w] = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            next.word[i][w] |= (block + 4 * w + k < stop ? from[4 * w + k] : 127u) << (8 * k);
        }
      }
    }
  }
}

template <class G>
__device__ __forceinline__ void place_scales(const Scales<G>& next, Stage<G>& to) {
#pragma unroll
  for (int i = 0; i < G::scale_rows; ++i) {
    const int row = i * G::threads + static_cast<int>(threadIdx.x);
    if (G::rows % G::threads == 0 || row < G::rows) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint16_t two = static_cast<uint16_t>((next.word[i][0] >> (8 * k) & 255u) |
                                                   (next.word[i][1] >> (8 * k) & 255u) << 8);
        const int strip = row >> 4, lane = 16 * k + (row & 15);
        if (row < G::rows_m)
          to.scales_a[strip / G::MI][lane][strip % G::MI] = two;
        else
          to.scales_b[(strip - G::rows_m / 16) / G::NJ][lane][(strip - G::rows_m / 16) % G::NJ] = two;
      }
    }
  }
}

// y^T strips: with b's rows as the instruction's first operand, a lane's four results are
// four neighbouring columns of one row of y.
template <int kByteA, int kByteB>
__device__ __forceinline__ v4f mx_mfma(v4i a, v4i b, v4f c, int scale_a, int scale_b) {
  const v8i wide_a = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  const v8i wide_b = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide_a, wide_b, c, 4, 4, kByteA, scale_a,
                                                          kByteB, scale_b);
}

template <int kStrips>
__device__ __forceinline__ void load_scales(const uint16_t* from, int (&to)[(kStrips + 1) / 2]) {
  to[(kStrips + 1) / 2 - 1] = 0;
  __builtin_memcpy(to, from, 2 * kStrips);
}

// A wavefront's operands of a stage.
template <class G>
struct Fragments {
  v4i a[G::KS][G::MI], b[G::KS][G::NJ];
  int scale_a[(G::MI + 1) / 2], scale_b[(G::NJ + 1) / 2];
};

template <class G>
__device__ __forceinline__ void read_fragments(const Stage<G>& from, int wm, int wn, int lane,
                                               Fragments<G>& f) {
  load_scales<G::MI>(from.scales_a[wm][lane], f.scale_a);
  load_scales<G::NJ>(from.scales_b[wn][lane], f.scale_b);
#pragma unroll
  for (int s = 0; s < G::KS; ++s) {
    const int place = (4 * s + (lane >> 4)) ^ (lane >> 1 & 7);
#pragma unroll
    for (int i = 0; i < G::MI; ++i)
      f.a[s][i] = from.codes[((wm * G::MI + i) * 16 + (lane & 15)) * 8 + place];
#pragma unroll
    for (int j = 0; j < G::NJ; ++j)
      f.b[s][j] = from.codes[(G::rows_m + (wn * G::NJ + j) * 16 + (lane & 15)) * 8 + place];
  }
}

template <class G, int S = 0, int J = 0, int I = 0>
__device__ __forceinline__ void multiply(const Fragments<G>& f, v4f (&sum)[G::MI][G::NJ]) {
  sum[I][J] = mx_mfma<2 * (J & 1) + S, 2 * (I & 1) + S>(f.b[S][J], f.a[S][I], sum[I][J],
                                                        f.scale_b[J / 2], f.scale_a[I / 2]);
  if constexpr (I + 1 < G::MI)
    multiply<G, S, J, I + 1>(f, sum);
  else if constexpr (J + 1 < G::NJ)
    multiply<G, S, J + 1, 0>(f, sum);
  else if constexpr (S + 1 < G::KS)
    multiply<G, S + 1, 0, 0>(f, sum);
}

// What a wavefront's lanes have written to LDS is read by others of them: no read or write
// moves past this in the program (in LDS they stay in order by themselves).  kPath tells ways
// apart that differ in how they store only: the compiler would join them to one of the two.
template <int kPath>
__device__ __forceinline__ void lanes_meet() { asm volatile("" :: "i"(kPath) : "memory"); }

// A wavefront's results, from row m0, column n0, of which `rows` and `columns` exist.  They
// go strip by strip (16 rows) through LDS, so that each store instruction writes whole lines
// of eight rows or more; rows are padded by 16 bytes, so that the rows of a column do not all
// meet one bank (four cycles of conflicts an access are left).  (Stored from the
// registers, 32 bytes a row, the 8192^3 product spent 75 us of 418 on it.)
template <class G, class T>
struct Strip {
  static constexpr int kWide = 16 / sizeof(T);                        // values per lane and store
  static constexpr int kLanes = 16 * G::NJ / kWide;                   // lanes per row
  static constexpr int kRows = 64 / kLanes < 16 ? 64 / kLanes : 16;   // rows per store
  T values[16][16 * G::NJ + kWide];
};

// kStream: past the caches, for results too large to be read again from there (8192^3 331 ->
// 306 us, 8000 x 50,000 by 1024 497 -> 382), where every lane writes whole halves of 32 bytes
// that no other store shares (5000 rows by 700, us past and through the caches: 31,040 columns
// 128 / 134; 31,016, 16 bytes off a line, 171 / 139; 31,013 194 / 144).
template <class G, class T, bool kStream>
__device__ __forceinline__ void store_tiles(T* to, int64_t stride, const v4f (&sum)[G::MI][G::NJ],
                                            const float* bias, int64_t rows, int64_t columns, int lane,
                                            Strip<G, T>& strip) {
  using S = Strip<G, T>;
  const int row = lane / S::kLanes, column = lane % S::kLanes * S::kWide;
  const bool wide = column + S::kWide <= columns;
#pragma unroll
  for (int i = 0; i < G::MI; ++i) {
#pragma unroll
    for (int j = 0; j < G::NJ; ++j) {
      Pack<T, 4> y;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = 16 * j + 4 * (lane >> 4) + r;
        y.v[r] = static_cast<T>(sum[i][j][r] + (bias && n < columns ? bias[n] : 0.0f));
      }
      __builtin_memcpy(&strip.values[lane & 15][16 * j + 4 * (lane >> 4)], &y, sizeof(y));
    }
    lanes_meet<kStream>();
#pragma unroll
    for (int r = 0; r < 16; r += S::kRows) {
      if (row >= S::kRows || 16 * i + r + row >= rows) continue;
      T* at = to + (16 * i + r + row) * stride + column;
      Pack<T, S::kWide> y;
      __builtin_memcpy(&y, &strip.values[r + row][column], sizeof(y));
      if (wide) {
        stream_pack<T, S::kWide, kStream>(at, y);
      } else {
#pragma unroll
        for (int k = 0; k < S::kWide; ++k)
          if (column + k < columns) at[k] = y.v[k];
      }
    }
    lanes_meet<kStream>();
  }
}

// All this wavefront's loads have arrived, those into LDS too.
__device__ __forceinline__ void wait_all() { __builtin_amdgcn_s_waitcnt(0); }

// Keeps the sums' computation before what follows in the program.
template <class G>
__device__ __forceinline__ void hold(v4f (&sum)[G::MI][G::NJ]) {
#pragma unroll
  for (int i = 0; i < G::MI; ++i)
#pragma unroll
    for (int j = 0; j < G::NJ; ++j) asm volatile("" : "+v"(sum[i][j]));
}

// Tiles of y, one workgroup per tile and part of K.  Two stages of LDS: while one is
// multiplied, the next one is loaded.  33 x 1000 by 50,000 (64 x 64 tiles, 28 parts): 10 us,
// and 4 for the parts' sums.
template <class G, class T>
__global__ __launch_bounds__(G::threads) void product_tiles(MxView a, MxView b, const float* bias,
                                                            T* out, int64_t stride, uint32_t tiles_m,
                                                            uint32_t tiles_n, uint32_t splits,
                                                            float* partials) {
  __shared__ union {
    Stage<G> stages[2];
    Strip<G, T> strip[G::WM * G::WN];
    Strip<G, float> partial[G::WM * G::WN];
  } lds;
  Stage<G>(&stages)[2] = lds.stages;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int wm = wave / G::WN, wn = wave % G::WN;
  // Divisions run on the vector ALU; their results are the same in every lane, and have to
  // be known as such for the panels' buffers.
  const uint32_t split = uniform(blockIdx.x / (tiles_m * tiles_n));
  const uint32_t tile = blockIdx.x - split * (tiles_m * tiles_n);
  const uint32_t tile_m = uniform(tile / tiles_n), tile_n = tile - tile_m * tiles_n;
  const int64_t m0 = static_cast<int64_t>(tile_m) * G::rows_m;
  const int64_t n0 = static_cast<int64_t>(tile_n) * G::rows_n;
  const int blocks = static_cast<int>(a.blocks);           // at most 2^18
  const int all = (blocks + 4 * G::KS - 1) / (4 * G::KS);
  const int per = static_cast<int>(uniform((all + splits - 1u) / splits));
  const int first = static_cast<int>(split) * per * (4 * G::KS);
  const int stop = first + per * (4 * G::KS) < blocks ? first + per * (4 * G::KS) : blocks;
  const MxPanel pa = panel(a, m0, G::rows_m), pb = panel(b, n0, G::rows_n);
  v4f sum[G::MI][G::NJ] = {};
  Scales<G> next;
  Fragments<G> f;
  const int whole_stop = first + (stop - first) / (4 * G::KS) * (4 * G::KS);
  int now = 0;
  if (first < whole_stop) {
    request_codes<G, true>(pa, pb, first, stop, wave, lane, stages[0]);
    request_scales<G, true>(pa, pb, first, stop, next);
    place_scales<G>(next, stages[0]);
  }
  for (int block = first; block < whole_stop; block += 4 * G::KS) {
    // The stage's codes and scales have arrived, and the other stage is read to its end.
    wait_all();
    __syncthreads();
    read_fragments<G>(stages[now], wm, wn, lane, f);
    // The last whole stage requests itself again, which nothing reads.
    const int ahead = block + 4 * G::KS < whole_stop ? block + 4 * G::KS : block;
    now ^= 1;
    request_codes<G, true>(pa, pb, ahead, stop, wave, lane, stages[now]);
    request_scales<G, true>(pa, pb, ahead, stop, next);
    multiply<G>(f, sum);
    hold<G>(sum);
    place_scales<G>(next, stages[now]);
  }
  if (whole_stop < stop) {
    wait_all();
    __syncthreads();
    request_codes<G, false>(pa, pb, whole_stop, stop, wave, lane, stages[now]);
    request_scales<G, false>(pa, pb, whole_stop, stop, next);
    place_scales<G>(next, stages[now]);
    wait_all();
    __syncthreads();
    read_fragments<G>(stages[now], wm, wn, lane, f);
    multiply<G>(f, sum);
  }
  const int64_t m = m0 + 16 * wm * G::MI, n = n0 + 16 * wn * G::NJ;
  // LDS is used anew: the stages are read to their end, and the last requests, which nothing
  // reads, have arrived.
  wait_all();
  __syncthreads();
  if (splits > 1) {
    store_tiles<G, float, false>(partials + (split * a.rows + m) * b.rows + n, b.rows, sum, nullptr,
                          a.rows - m, b.rows - n, lane, lds.partial[wave]);
  } else {
    store_tiles<G, T, false>(out + m * stride + n, stride, sum, bias ? bias + n : nullptr,
                             a.rows - m, b.rows - n, lane, lds.strip[wave]);
  }
}

// Large tiles.  Scales too go straight into LDS, nothing passes through registers on its way
// there; their rows have to be whole 32-bit words, and where they are not (K no multiple of
// 128) pad_scales lays them out so first.  Half a stage (one step
// of 128 values) is multiplied while the fragments of the next half are read and the next
// stages' requests leave one by one between the products, so that neither LDS, nor the
// requests' addresses, nor the barrier keep the matrix cores waiting for long: one barrier a
// stage, after its first half, when all have read the stage to its end and the next one has
// arrived.  On one card 8192^3 in bf16 takes 270 us, 4.07 PFLOP/s, 4096 x 4096 by 32768 264 us,
// 4.16 PFLOP/s: 61% of the rate at which these instructions issue from registers (6.8).  (On
// the way, the first of them on another card: 418 us with both steps' fragments read at once
// and a wait for all requests; 366 with two barriers a stage; 336 like this with all requests
// right behind the barrier; 324 spread; 304 with streamed results and bands of tiles.)  What
// bounds it: of the second's 264 us the products alone, in this frame, take 189, with the
// fragments' reads 219; the requests alone take 124 without those for scales, and slow the
// rest down while they pass through the same LDS.
// The requests are inline assembly because the compiler, which cannot tell the two buffers
// apart, would wait for all of them before it reads either; they write LDS only, no registers,
// and the barriers' waits count them.
struct alignas(16) WordPanel {
  v4i codes, scales;           // buffer descriptors
  uint32_t row_bytes, blocks, scale_bytes;   // a row's codes, blocks, and scales with their padding
};

__device__ __forceinline__ v4i describe(const uint8_t* base, uint32_t bytes) {
  const uint64_t address = reinterpret_cast<uint64_t>(base);
  return v4i{static_cast<int>(uniform(static_cast<uint32_t>(address))),
             static_cast<int>(uniform(static_cast<uint32_t>(address >> 32))),
             static_cast<int>(uniform(bytes)), 0x00020000};
}

__device__ __forceinline__ WordPanel word_panel(const MxView& m, int64_t row, int rows) {
  const uint32_t own = static_cast<uint32_t>(m.rows - row < rows ? m.rows - row : rows);
  const uint32_t blocks = uniform(static_cast<uint32_t>(m.blocks)), scales = (blocks + 3) & ~3u;
  return WordPanel{describe(m.codes + row * m.blocks * 16, own * blocks * 16),
                   describe(m.scales + row * scales, own * scales), blocks * 16, blocks, scales};
}

// 16 bytes per lane from `offset` of a buffer to LDS at `to` + 16 * lane.  The address is in m0,
// which the compiler sets; a request right behind that needs one wait state.
__device__ __forceinline__ void to_lds_16(const v4i& buffer, uint32_t offset, uint32_t to) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "{m0}"(to), "v"(offset), "s"(buffer) : "memory");
}

// Where row r keeps block k of a stage: place k ^ turn(r).  Four neighbouring lanes then ask
// for 64 neighbouring bytes (blocks of one step side by side: requests alone 183 us instead
// of 124, without scales), and the fragment reads, whose quarters hold rows 0-3 and 12-15 of
// one block with rows 4-11 of the next but one, meet no bank twice: bit 2 of the turn tells
// the two sets of rows apart.  (Counted by themselves: these reads no conflict cycle, a 16-bit
// read of scales two, a strip's write or read four; at 8192^3 6.5 and 1.6 million of 41.7 million
// cycles that LDS works.)
__device__ __forceinline__ uint32_t turn(uint32_t row) {
  return (row >> 1 & 7) ^ (row & 4);
}

template <class G>
struct WordStages {
  v4i codes[2][G::rows * 8];
  uint32_t scales[2][G::rows * 4];   // words 4r .. are row r's of two stages
};

// What a wavefront asks for: per stage G::loads pieces of codes, eight rows of 128 bytes each;
// per two stages one piece of scales, 16 bytes of 64 rows (4 bytes of 32 rows a stage: 4096 x
// 4096 by 32768 277 us instead of 264).
struct StageRequests {
  uint32_t row, at, to;        // row and block of the lane's codes; LDS address of the stage
  bool inside;
};
struct ScaleRequests {
  uint32_t block, wave, lane, to;
  bool wanted;
};

template <class G>
__device__ __forceinline__ StageRequests stage_requests(const WordPanel& a, int block, int wave,
                                                        int lane, uint32_t to) {
  StageRequests q;
  q.row = 8 * wave + (lane >> 3);
  q.at = block + ((lane & 7) ^ turn(q.row));
  q.inside = q.at < a.blocks;
  q.to = to + 16 * 64 * wave;
  return q;
}

constexpr uint32_t kNone = 0xFFFFFFF0u;                    // past every buffer: reads as zeros

template <class G, int I>
__device__ __forceinline__ void request_codes(const WordPanel& a, const WordPanel& b,
                                              const StageRequests& q) {
  constexpr int kPerRound = G::threads / 8, kLoadsA = G::rows_m / kPerRound;
  const WordPanel& m = I < kLoadsA ? a : b;
  const uint32_t r = q.row + kPerRound * (I < kLoadsA ? I : I - kLoadsA);
  to_lds_16(m.codes, q.inside ? r * m.row_bytes + q.at * 16 : kNone, q.to + 16 * (I * G::threads));
}

// Scales of two stages.  Past a row's words these are the next row's, and are not used.
template <class G>
__device__ __forceinline__ void request_scales(const WordPanel& a, const WordPanel& b,
                                               const ScaleRequests& q) {
  static_assert(G::rows == G::threads && G::rows_m % 64 == 0, "one row per lane, of one operand");
  const bool of_a = 64 * q.wave < G::rows_m;
  const WordPanel& m = of_a ? a : b;
  const uint32_t r = 64 * q.wave + q.lane - (of_a ? 0 : G::rows_m);
  to_lds_16(m.scales, q.block < a.blocks ? r * a.scale_bytes + q.block : kNone, q.to + 16 * 64 * q.wave);
}

template <class G, int I = 0>
__device__ __forceinline__ void request_all_codes(const WordPanel& a, const WordPanel& b,
                                                  const StageRequests& q) {
  request_codes<G, I>(a, b, q);
  if constexpr (I + 1 < G::loads) request_all_codes<G, I + 1>(a, b, q);
}
// A wavefront's operands: of one step of a stage, and a stage's scales (byte s: step s).
// Lane l's blocks are 2(l/16) and 2(l/16) + 1, so that its two scale bytes are one word.
template <class G>
struct StepFragments {
  v4i a[G::MI], b[G::NJ];
};
template <class G>
struct StageScales {
  int a[G::MI / 2], b[G::NJ];  // a: two strips a register
};

// LDS addresses of a wavefront's first strips of a step, per lane; the other strips lie at
// constant distances.
struct StepBase {
  uint32_t codes_a, codes_b, scales_a, scales_b;
};

template <class G>
__device__ __forceinline__ StepBase step_base(uint32_t stage, uint32_t stage_scales, int step, int wm,
                                              int wn, int lane) {
  constexpr int kScaleBytes = 16;                          // per row
  const uint32_t row = lane & 15, place = (2 * (lane >> 4) + step) ^ turn(row);
  const uint32_t codes = stage + (row * 8 + place) * 16;
  const uint32_t scales = stage_scales + row * kScaleBytes + 2 * (lane >> 4);
  StepBase base{codes + wm * (G::MI * 16 * 128), codes + (G::rows_m + wn * G::NJ * 16) * 128,
                scales + wm * (G::MI * 16 * kScaleBytes),
                scales + (G::rows_m + wn * G::NJ * 16) * kScaleBytes};
  // One register each, here: left to itself the compiler keeps every strip's.
  asm volatile("" : "+v"(base.codes_a), "+v"(base.codes_b), "+v"(base.scales_a), "+v"(base.scales_b));
  return base;
}

__device__ __forceinline__ v4i read_code(uint32_t base, int strip) {
  return *(const __attribute__((address_space(3))) v4i*)static_cast<uintptr_t>(base + strip * (16 * 128));
}
__device__ __forceinline__ int read_scale(uint32_t base, int strip) {
  return *(const __attribute__((address_space(3))) uint16_t*)static_cast<uintptr_t>(base + strip * (16 * 16));
}

// Multiplies column strip J of step S, reading strip J of the next step meanwhile (and, where
// that begins a stage, its scales), and requesting codes of the stage after that (S 1) or the
// scales of stages to come (S 0).
template <class G, int S, int J>
__device__ __forceinline__ void column(StepFragments<G>& f, const StageScales<G>& scales,
                                       const StepBase& from, StepFragments<G>& next,
                                       StageScales<G>& next_scales, const WordPanel& pa,
                                       const WordPanel& pb, const StageRequests& q,
                                       const ScaleRequests& to_come, int keep, v4f (&sum)[G::MI][G::NJ]) {
  constexpr int kPer = G::MI / G::NJ;                      // a's strips per column
  static_assert(kPer == 2, "a column reads two strips of a");
  static_assert(G::loads == 2 * G::NJ, "a column requests two pieces");
  int pair[2];
  next.b[J] = read_code(from.codes_b, J);
#pragma unroll
  for (int i = kPer * J; i < kPer * (J + 1); ++i) next.a[i] = read_code(from.codes_a, i);
  if constexpr (S == 1) {
    next_scales.b[J] = read_scale(from.scales_b, J);
    pair[0] = read_scale(from.scales_a, kPer * J);
    pair[1] = read_scale(from.scales_a, kPer * J + 1);
    request_codes<G, 2 * J>(pa, pb, q);
    request_codes<G, 2 * J + 1>(pa, pb, q);
  } else if constexpr (J == 0) {
    if (to_come.wanted) request_scales<G>(pa, pb, to_come);
  }
  // The empty statements keep the products of a column in its place: the compiler would gather
  // them before the barrier, and wait there for operands that were to arrive meanwhile.
  asm volatile("" : "+v"(f.b[J]));
#pragma unroll
  for (int i = 0; i < G::MI; ++i)
    sum[i][J] = i & 1 ? mx_mfma<S, 2 + S>(f.b[J], f.a[i], sum[i][J], scales.b[J], scales.a[i / 2])
                      : mx_mfma<S, S>(f.b[J], f.a[i], sum[i][J], scales.b[J], scales.a[i / 2]);
#pragma unroll
  for (int i = 0; i < G::MI; ++i) asm volatile("" : "+v"(sum[i][J]));
  if constexpr (S == 1) {
    next_scales.b[J] &= keep;
    next_scales.a[J] = (pair[0] | pair[1] << 16) & keep;
  }
  if constexpr (J + 1 < G::NJ)
    column<G, S, J + 1>(f, scales, from, next, next_scales, pa, pb, q, to_come, keep, sum);
}

// s_waitcnt: vmcnt in bits 0-3 and 14-15, expcnt 4-6, lgkmcnt 8-11.
constexpr int wait_loads(int n) { return (n & 15) | (n >> 4) << 14 | 7 << 4 | 15 << 8; }
template <int kWait>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(kWait);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Both operands' rows of scales, a's then b's, in whole words with zeros behind them; a
// wavefront per row.  8192 x 8192 by 8160: 6 us, and the product with it 344; tiles of the same
// size that took such scales through registers needed 425.
__global__ __launch_bounds__(kThreads) void pad_scales(MxView a, MxView b, uint32_t* out) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
  if (row >= a.rows + b.rows) return;
  const uint8_t* from = row < a.rows ? a.scales + row * a.blocks : b.scales + (row - a.rows) * b.blocks;
  const int64_t words = (a.blocks + 3) / 4;
  for (int64_t w = threadIdx.x & 63; w < words; w += 64) {
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (4 * w + k < a.blocks) word |= static_cast<uint32_t>(from[4 * w + k]) << (8 * k);
    out[row * words + w] = word;
  }
}

__device__ __forceinline__ uint32_t lds_address(const void* at) {
  return uniform(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) const void*)at)));
}

template <class G, class T>
__global__ __launch_bounds__(G::threads) void product_word_tiles(MxView a, MxView b,
                                                                 const float* bias, T* out,
                                                                 int64_t stride, uint32_t tiles_m,
                                                                 uint32_t tiles_n) {
  __shared__ union {
    WordStages<G> stages;
    Strip<G, T> strip[G::WM * G::WN];
  } lds;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int wm = wave / G::WN, wn = wave % G::WN;
  // Workgroups are dealt to the XCDs in turn: each XCD gets a run of tiles, in bands of four
  // rows, so that the 32 it multiplies at a time share four panels of a and eight of b in its
  // L2 (4096 x 4096 by 32768 251 -> 238 us, 3000 x 50,000 by 4096 399 -> 359, against rows of
  // tiles dealt one by one).
  constexpr uint32_t kBand = 4;
  const uint32_t share = tiles_m * tiles_n / kXcds;
  const uint32_t tile = blockIdx.x < share * kXcds ? blockIdx.x % kXcds * share + blockIdx.x / kXcds
                                                   : blockIdx.x;
  const uint32_t band = uniform(tile / (kBand * tiles_n)), in_band = tile - band * kBand * tiles_n;
  const uint32_t high = tiles_m - kBand * band < kBand ? tiles_m - kBand * band : kBand;
  const uint32_t tile_n = uniform(in_band / high), tile_m = kBand * band + in_band - tile_n * high;
  const int64_t m0 = static_cast<int64_t>(tile_m) * G::rows_m;
  const int64_t n0 = static_cast<int64_t>(tile_n) * G::rows_n;
  const WordPanel pa = word_panel(a, m0, G::rows_m), pb = word_panel(b, n0, G::rows_n);
  const int stages = (static_cast<int>(pa.blocks) + 7) / 8;
  const uint32_t codes = lds_address(&lds.stages.codes), scales_at = lds_address(&lds.stages.scales);
  constexpr uint32_t kCodes = sizeof(lds.stages.codes[0]), kScales = sizeof(lds.stages.scales[0]);

  v4f sum[G::MI][G::NJ] = {};
  StepFragments<G> even, odd;  // operands of a stage's first and second step
  StageScales<G> scales, next_scales;
  request_all_codes<G>(pa, pb, stage_requests<G>(pa, 0, wave, lane, codes));
  request_scales<G>(pa, pb, ScaleRequests{0, static_cast<uint32_t>(wave),
                                                     static_cast<uint32_t>(lane), scales_at, true});
  request_all_codes<G>(pa, pb, stage_requests<G>(pa, 8, wave, lane, codes + kCodes));
  wait_barrier<wait_loads(G::loads)>();
  const StepBase begin = step_base<G>(codes, scales_at, 0, wm, wn, lane);
  const int keep = 2 * (lane >> 4) < static_cast<int>(pa.blocks) ? -1 : 0;
#pragma unroll
  for (int i = 0; i < G::MI; ++i) {
    even.a[i] = read_code(begin.codes_a, i);
    if (i & 1)
      scales.a[i / 2] =
          (read_scale(begin.scales_a, i - 1) | read_scale(begin.scales_a, i) << 16) & keep;
  }
#pragma unroll
  for (int j = 0; j < G::NJ; ++j) {
    even.b[j] = read_code(begin.codes_b, j);
    scales.b[j] = read_scale(begin.scales_b, j) & keep;
  }
  // Stages past the last read as zeros and are not multiplied.
  for (int stage = 0; stage < stages; ++stage) {
    const uint32_t now = codes + (stage & 1 ? kCodes : 0), then = codes + (stage & 1 ? 0 : kCodes);
    const int after = stage + 1;
    // The other half of the scales is read to its end: the last barrier saw to it.
    const ScaleRequests to_come{8u * (stage + 2), static_cast<uint32_t>(wave),
                                static_cast<uint32_t>(lane),
                                scales_at + ((stage & 2) ? 0 : kScales), !(stage & 1)};
    column<G, 0, 0>(even, scales, step_base<G>(now, scales_at, 1, wm, wn, lane), odd, next_scales, pa,
                    pb, StageRequests{}, to_come, 0, sum);
    // This stage is read by all, and the next one has arrived for all.
    wait_barrier<0>();
    // Blocks past K have codes of zero, but their scales, another row's, may be NaN.
    const int keep = 8 * after + 2 * (lane >> 4) < static_cast<int>(pa.blocks) ? -1 : 0;
    column<G, 1, 0>(odd, scales,
                    step_base<G>(then, scales_at + (after & 2 ? kScales : 0) + 8 * (after & 1), 0, wm,
                                 wn, lane),
                    even, next_scales, pa, pb, stage_requests<G>(pa, 8 * (stage + 2), wave, lane, now),
                    to_come, keep, sum);
    scales = next_scales;
  }
  wait_barrier<0>();                                       // before LDS is used anew
  const int64_t m = m0 + 16 * wm * G::MI, n = n0 + 16 * wn * G::NJ;
  T* const to = out + m * stride + n;
  const float* const more = bias ? bias + n : nullptr;
  if ((reinterpret_cast<uintptr_t>(out) | stride * sizeof(T)) % 32 == 0)
    store_tiles<G, T, true>(to, stride, sum, more, a.rows - m, b.rows - n, lane, lds.strip[wave]);
  else
    store_tiles<G, T, false>(to, stride, sum, more, a.rows - m, b.rows - n, lane, lds.strip[wave]);
}

// Few rows of a (up to 16) and few columns: bound by b's bytes, each read once, and by the way
// from a request to its use.  A workgroup takes 16 columns of y (rows of b) straight from
// memory to registers, four stages of K requested ahead; its four wavefronts take a quarter of
// K each and meet in LDS.
// A sum over K may take its blocks in any order, as long as both operands do: lane l takes
// blocks 2(l/16) and 2(l/16) + 1 of a stage for its two steps, so that four lanes read a whole
// line of a row and a row's two scale bytes are one 16-bit word.  16 x 4096 by 4096 takes 6 us with its call.
struct RowPanel {
  __amdgpu_buffer_rsrc_t codes;
  const uint8_t* scales;       // of the lane's row
  uint32_t row_offset;
  int blocks;
};

// Rows row .. row + 15 of an operand (past its last row: none).
__device__ __forceinline__ RowPanel row_panel(const MxView& m, int64_t row, int lane) {
  const MxPanel p = panel(m, row < m.rows ? row : m.rows - 1, row < m.rows ? 16 : 0);
  const int own = (lane & 15) < p.last ? (lane & 15) : p.last > 0 ? p.last : 0;
  return RowPanel{p.codes, p.scales + static_cast<int64_t>(own) * p.blocks,
                  static_cast<uint32_t>(lane & 15) * p.row_bytes, p.blocks};
}

struct RowStage {
  v4i codes[2];
  int scales;                  // byte 0: first step, byte 1: second
};

// Blocks and rows that do not exist read as zeros with scale 1.
__device__ __forceinline__ void load_row_stage(const RowPanel& p, int block, RowStage& to) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint32_t offset = block + s < p.blocks ? p.row_offset + (block + s) * 16u : 0xFFFFFFF0u;
    to.codes[s] = __builtin_bit_cast(
        v4i, __builtin_amdgcn_raw_buffer_load_b128(p.codes, static_cast<int>(offset), 0, 0));
  }
  if (p.blocks >= 2) {
    // The row's last word holds the last block's byte second.
    const int at = block < p.blocks - 2 ? block : p.blocks - 2;
    uint16_t two;
    __builtin_memcpy(&two, p.scales + at, 2);
    to.scales = block <= p.blocks - 2 ? two : block == p.blocks - 1 ? two >> 8 | 127 << 8 : 0x7F7F;
  } else {
    to.scales = block == 0 ? p.scales[0] | 127 << 8 : 0x7F7F;
  }
}

constexpr int kRowsAhead = 4;   // stages
constexpr int kWaves = kThreads / 64;

// A workgroup's wavefronts share a strip of 16 columns, a part of K each.
template <class T>
__global__ __launch_bounds__(kThreads) void product_rows(MxView a, MxView b, const float* bias,
                                                         T* out, int64_t stride) {
  __shared__ v4f sums[kWaves][64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const RowPanel pa = row_panel(a, 0, lane), pb = row_panel(b, n0, lane);
  const int blocks = static_cast<int>(a.blocks), stages = (blocks + 7) / 8;
  const int per = (stages + kWaves - 1) / kWaves, first = wave * per;
  const int stop = first + per < stages ? first + per : stages;

  v4f sum = {};
  RowStage x[kRowsAhead], y[kRowsAhead];
  const int mine = 2 * (lane >> 4);
  // A stage past the end reads as zeros.
  const auto load = [&](int stage, int to) __attribute__((always_inline)) {
    const int block = 8 * (stage < stop ? stage : stages) + mine;
    load_row_stage(pb, block, y[to]);
    load_row_stage(pa, block, x[to]);
  };
  if (first < stop) {
#pragma unroll
    for (int u = 0; u < kRowsAhead; ++u) load(first + u, u);
  }
  for (int stage = first; stage < stop; stage += kRowsAhead) {
#pragma unroll
    for (int u = 0; u < kRowsAhead; ++u) {
      sum = mx_mfma<0, 0>(y[u].codes[0], x[u].codes[0], sum, y[u].scales, x[u].scales);
      sum = mx_mfma<1, 1>(y[u].codes[1], x[u].codes[1], sum, y[u].scales, x[u].scales);
      if (stage + kRowsAhead < stop) load(stage + kRowsAhead + u, u);
    }
  }
  sums[wave][lane] = sum;
  __syncthreads();
  const int column = threadIdx.x & 15, m = threadIdx.x >> 4;
  const int from = (column >> 2) * 16 + m;                 // the lane that holds it
  const int64_t n = n0 + column;
  float total = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    total += reinterpret_cast<const float*>(&sums[w][from])[column & 3];
  if (m < a.rows && n < b.rows)
    out[m * stride + n] = static_cast<T>(total + (bias ? bias[n] : 0.0f));
}

// The parts of K added in order, eight requested at a time.
template <class T>
__global__ __launch_bounds__(kThreads) void add_splits(const float* __restrict__ partials,
                                                       uint32_t splits, int64_t rows,
                                                       int64_t columns, const float* bias, T* out,
                                                       int64_t stride) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= rows * columns) return;
  float sum = 0.0f;
  constexpr uint32_t kAhead = 8;
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

int launched(const char* what) {
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? NS_OK : fail_launch(what, err);
}

MxView view(const ns_mx_matrix& m) {
  return MxView{m.codes, m.scales, m.rows, (m.columns + NS_MX_BLOCK - 1) / NS_MX_BLOCK};
}

using Large = Tile<8, 4, 2, 4, 2>;   // 256 x 256
using Small = Tile<2, 2, 2, 2, 2>;   // 64 x 64

constexpr int64_t kFewRows = 16;     // product_rows

// Which kernel multiplies M x N by K.  us, 64 x 64 tiles against 256 x 256: 4096^3 86 / 51;
// 2048 x 4096 by 1024 (128 large tiles, half the compute units) 16.7 / 17.7; 2048^3 (64) 13.8 /
// 21.  One small tile high or wide, the large ones are mostly empty: 33 x 50,000 by 1024 8.0 /
// 13.2, by 4096 23 / 29, 64 x 50,000 by 4096 29 / 30, 50,000 x 64 by 1024 8.2 / 17.7; two high,
// 128 x 50,000 by 1024 15.6 / 16.3, by 4096 47 / 32.  product_rows saves small tiles the cut of
// K and its launch where both have few columns and not too many of K: product_rows / tiles, 16 x
// 4096 by 4096 6.0 / 9.5, 1 x 12,000 by 6000 8.6 / 13; but 1 x 50,000 by 1024 8.5 / 6.8, 16 x
// 50,000 by 1024 13.2 / 7.1, 16 x 8192 by 16,384 26 / 17, 1 x 1000 by 50,000 11.3 / 10.1.
enum class Kernel { kRows, kSmall, kLarge };
Kernel kernel_of(int64_t m, int64_t n, int64_t k) {
  if (m <= kFewRows && n < 16 * 1024 && k <= 8 * 1024) return Kernel::kRows;
  if (m <= Small::rows_m || n <= Small::rows_n) return Kernel::kSmall;
  return (m + 255) / 256 * ((n + 255) / 256) >= 192 ? Kernel::kLarge : Kernel::kSmall;
}

// Parts that the small tiles cut K into where they are few.  A part's sums are written, read
// again and cost a launch (4 us), so parts are long: seven stages or more, sixteen where the
// tiles alone give every compute unit one.  (product_rows, whose wavefronts share K, gains
// nothing: 8 x 2000 by 8192 whole 7.5, in two parts 11.6; 16 x 8000 by 8192 12.8 / 16.3.)  us,
// whole / cut: 256 x 4096 by 4096 11.4 / 16.2 (2 parts of 8 stages), 1024 x 1024 by 8192 24.3 /
// 21.7 (2 of 16), 64 x 8192 by 8192 18.1 (2 of 16) / 15.4 (4 of 8), 33 x 1000 by 50,000 15.5 (16
// of 13) / 14 (28 of 7).  Seven stages at least against eight: 33 x 1000 by 60,000 13.8 / 14.2,
// by 50,000 13.0 / 13.3, by 30,000 11.8 / 11.8; 33 x 2000 by 30,000 12.7 / 13.3, by 60,000 18.1 /
// 18.1; 33 x 500 by 16,384 to 60,000, 64 x 8192 by 8192 and 100 x 2000 by 16,384 the same.
int64_t parts_of_k(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0) return 1;
  if (kernel_of(m, n, k) != Kernel::kSmall) return 1;
  const int64_t stages = (k + 255) / 256, tiles = (m + 63) / 64 * ((n + 63) / 64);
  const int64_t most = stages / (tiles >= 256 ? 16 : 7);
  const int64_t parts = 512 / tiles < most ? 512 / tiles : most;
  if (parts <= 1) return 1;
  const int64_t per = (stages + parts - 1) / parts;   // no empty part
  return (stages + per - 1) / per;
}

// The workspace: a's codes and scales (float rows), then the parts' sums, or both operands'
// scales in whole words.
struct Workspace {
  int64_t scales, rest, bytes;
};

int64_t word_bytes(int64_t blocks) { return (blocks + 3) / 4 * 4; }

Workspace workspace_of(int64_t m, int64_t n, int64_t k, bool float_rows) {
  const int64_t blocks = (k + NS_MX_BLOCK - 1) / NS_MX_BLOCK, parts = parts_of_k(m, n, k);
  Workspace w{};
  w.scales = float_rows ? m * blocks * 16 : 0;
  w.rest = float_rows ? (m * blocks * 17 + 15) / 16 * 16 : 0;
  w.bytes = w.rest + (parts > 1 ? parts * m * n * 4 : 0);
  if (kernel_of(m, n, k) == Kernel::kLarge) w.bytes += (m + n) * word_bytes(blocks);
  return w;
}

template <class G, class T>
int run_tiles(const ns_mx_product_args* p, int64_t parts, float* partials, hipStream_t stream) {
  const MxView a = view(p->a), b = view(p->b);
  const int64_t tiles_m = (a.rows + G::rows_m - 1) / G::rows_m;
  const int64_t tiles_n = (b.rows + G::rows_n - 1) / G::rows_n;
  const int64_t groups = tiles_m * tiles_n * parts;
  if (groups > INT32_MAX) return fail("the product is too large for one launch");
  product_tiles<G, T><<<dim3(static_cast<unsigned>(groups)), dim3(G::threads), 0, stream>>>(
      a, b, p->bias, static_cast<T*>(p->out), p->stride, static_cast<uint32_t>(tiles_m),
      static_cast<uint32_t>(tiles_n), static_cast<uint32_t>(parts), partials);
  return launched("product");
}

template <class T>
int run_large(const ns_mx_product_args* p, void* words, hipStream_t stream) {
  using G = Large;
  MxView a = view(p->a), b = view(p->b);
  const int64_t tiles_m = (a.rows + G::rows_m - 1) / G::rows_m;
  const int64_t tiles_n = (b.rows + G::rows_n - 1) / G::rows_n;
  const int64_t copies = (a.rows + b.rows + kThreads / 64 - 1) / (kThreads / 64);
  if (tiles_m * tiles_n > INT32_MAX || copies > INT32_MAX)
    return fail("the product is too large for one launch");
  if (a.blocks % 4 || reinterpret_cast<uintptr_t>(a.scales) % 4 ||
      reinterpret_cast<uintptr_t>(b.scales) % 4) {
    auto* to = static_cast<uint8_t*>(words);
    pad_scales<<<dim3(static_cast<unsigned>(copies)), dim3(kThreads), 0, stream>>>(
        a, b, static_cast<uint32_t*>(words));
    if (int rc = launched("product scales")) return rc;
    a.scales = to;
    b.scales = to + a.rows * word_bytes(a.blocks);
  }
  product_word_tiles<G, T><<<dim3(static_cast<unsigned>(tiles_m * tiles_n)), dim3(G::threads), 0,
                             stream>>>(a, b, p->bias, static_cast<T*>(p->out), p->stride,
                                       static_cast<uint32_t>(tiles_m),
                                       static_cast<uint32_t>(tiles_n));
  return launched("product");
}

template <class T>
int run_rows(const ns_mx_product_args* p, hipStream_t stream) {
  const int64_t strips = (p->b.rows + 15) / 16;            // fewer than 1024 (kernel_of)
  product_rows<T><<<dim3(static_cast<unsigned>(strips)), dim3(kThreads), 0, stream>>>(
      view(p->a), view(p->b), p->bias, static_cast<T*>(p->out), p->stride);
  return launched("product");
}

template <class T>
int run_kernel(const ns_mx_product_args* p, int64_t parts, float* partials, hipStream_t stream) {
  const Kernel kernel = kernel_of(p->a.rows, p->b.rows, p->a.columns);
  switch (p->a.columns || kernel == Kernel::kRows ? kernel : Kernel::kSmall) {
    case Kernel::kLarge: return run_large<T>(p, partials, stream);
    case Kernel::kSmall: return run_tiles<Small, T>(p, parts, partials, stream);
    default: return run_rows<T>(p, stream);
  }
}

template <class T>
int run(const ns_mx_product_args* p, float* partials, hipStream_t stream) {
  const int64_t rows = p->a.rows, columns = p->b.rows;
  const int64_t parts = parts_of_k(rows, columns, p->a.columns);
  if (int rc = run_kernel<T>(p, parts, partials, stream)) return rc;
  if (parts == 1) return NS_OK;
  const int64_t adds = (rows * columns + kThreads - 1) / kThreads;
  if (adds > INT32_MAX) return fail("the product is too large for one launch");
  add_splits<T><<<dim3(static_cast<unsigned>(adds)), dim3(kThreads), 0, stream>>>(
      partials, static_cast<uint32_t>(parts), rows, columns, p->bias, static_cast<T*>(p->out),
      p->stride);
  return launched("product parts");
}

int check_operand(const ns_mx_matrix& m, const char* what) {
  if (m.columns && (!m.codes || !m.scales))
    return fail("%s: codes and scales are required", what);
  if (reinterpret_cast<uintptr_t>(m.codes) % 16) return fail("%s: codes must be 16-byte aligned", what);
  return NS_OK;
}

}  // namespace
}  // namespace ns

extern "C" {

int64_t ns_mx_product_bytes(int64_t m, int64_t n, int64_t k, int32_t float_rows) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  return ns::workspace_of(m, n, k, float_rows != 0).bytes;
}

int ns_mx_product(const ns_mx_product_args* args, void* stream) {
  ns::clear_error();
  if (!args) return ns::fail("product arguments are required");
  ns_mx_product_args p = *args;
  const int64_t m = p.a.rows, n = p.b.rows, k = p.a.columns;
  if (p.a.columns != p.b.columns) return ns::fail("the operands need the same number of columns");
  // A tile's rows of codes are addressed in 31 bits.
  if (k > NS_MX_MAX_COLUMNS) return ns::fail("a product takes at most %d columns", NS_MX_MAX_COLUMNS);
  if (m < 0 || n < 0 || k < 0) return ns::fail("rows and columns must not be negative");
  if (m == 0 || n == 0) return NS_OK;
  if (k > 0) {
    const ns::Workspace w = ns::workspace_of(m, n, k, p.x != nullptr);
    auto* space = static_cast<uint8_t*>(p.workspace);
    if (w.bytes && (!space || reinterpret_cast<uintptr_t>(space) % 16))
      return ns::fail("the product needs its workspace, 16-byte aligned");
    if (p.x) {
      p.a.codes = space;
      p.a.scales = space + w.scales;
      if (int rc = ns_mx_quantize(&p.a, p.x, p.x_stride, p.x_type, stream)) return rc;
    }
    p.workspace = space + w.rest;
  }
  if (int rc = ns::check_operand(p.a, "a")) return rc;
  if (int rc = ns::check_operand(p.b, "b")) return rc;
  if (!p.out) return ns::fail("the output is required");
  auto queue = static_cast<hipStream_t>(stream);
  auto* partials = static_cast<float*>(p.workspace);
  switch (p.type) {
    case NS_TYPE_F32: return ns::run<float>(&p, partials, queue);
    case NS_TYPE_BF16: return ns::run<__bf16>(&p, partials, queue);
    case NS_TYPE_F16: return ns::run<_Float16>(&p, partials, queue);
    default: return ns::fail("unknown element type");
  }
}

}  // extern "C"
