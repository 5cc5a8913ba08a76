// What the kernels share that multiply tiles of matrices on the matrix cores: operands
// straight into LDS, waits, and results out of the registers in whole lines.
#pragma once

#include "ns_signal.h"

namespace ns {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return __builtin_amdgcn_readfirstlane(v);
}

__device__ __forceinline__ v4i describe(const uint8_t* base, uint32_t bytes) {
  const uint64_t address = reinterpret_cast<uint64_t>(base);
  return v4i{static_cast<int>(uniform(static_cast<uint32_t>(address))),
             static_cast<int>(uniform(static_cast<uint32_t>(address >> 32))),
             static_cast<int>(uniform(bytes)), 0x00020000};
}


constexpr uint32_t kNone = 0xFFFFFFF0u;                    // past every buffer: reads as zeros

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

__device__ __forceinline__ v4i read_code(uint32_t base, int strip) {
  return *(const __attribute__((address_space(3))) v4i*)static_cast<uintptr_t>(base + strip * (16 * 128));
}
__device__ __forceinline__ uint32_t lds_address(const void* at) {
  return uniform(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) const void*)at)));
}


// All this wavefront's loads have arrived, those into LDS too.
__device__ __forceinline__ void wait_all() { __builtin_amdgcn_s_waitcnt(0); }

// s_waitcnt: vmcnt in bits 0-3 and 14-15, expcnt 4-6, lgkmcnt 8-11.
constexpr int wait_loads(int n) { return (n & 15) | (n >> 4) << 14 | 7 << 4 | 15 << 8; }
// The same, and all of LDS's answers.
constexpr int wait_loads_and_lds(int n) { return (n & 15) | (n >> 4) << 14 | 7 << 4; }
template <int kWait>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(kWait);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
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

}  // namespace ns
