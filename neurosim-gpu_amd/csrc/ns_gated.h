// What the forward and the backward of the gated projection share: activations, sizes of
// tiles, and operands laid out as the tile kernels read them.
#pragma once

#include "ns_split.h"
#include "neurosim_hip_block.h"

namespace ns {

// Small tiles run where few fit the card, each waiting for its stages: four of them in LDS (64 x
// 4096 to 8192 in bf16 28.8 us, with three 31.2, with two 48.4).
using LargeGemm = GemmTile<8, 4, 2, 4, 2>;    // 256 x 256
using MiddleGemm = GemmTile<4, 4, 2, 2, 2>;   // 128 x 128
using SmallGemm = GemmTile<2, 2, 2, 2, 4>;    // 64 x 64
using MiddleSplit = SplitTile<4, 4, 2, 2, 3>; // 128 x 128
using SmallSplit = SplitTile<2, 2, 2, 2, 2>;  // 64 x 64

// x times the normal distribution's mass below x; erfc keeps the relative accuracy of small ones.
__device__ __forceinline__ float mass_below(float x) { return 0.5f * erfcf(-0.70710678118654752f * x); }

__device__ __forceinline__ float activated(float x, int activation) {
  return x * (activation == NS_GATE_SILU ? sigmoid(x) : mass_below(x));
}

struct Activation {
  float value, slope;
};
__device__ __forceinline__ Activation activated_slope(float x, int activation) {
  if (activation == NS_GATE_SILU) {
    const float s = sigmoid(x);
    return Activation{x * s, s * fmaf(x, 1.0f - s, 1.0f)};
  }
  const float below = mass_below(x);
  const float density = 0.39894228040143268f * __builtin_amdgcn_exp2f(-0.5f * kLog2e * x * x);
  return Activation{x * below, fmaf(x, density, below)};
}

inline int64_t type_size(int32_t type) { return type == NS_TYPE_F32 ? 4 : 2; }
// n up to whole pieces, and the 16-byte pieces of a laid-out row of n values, as they are or in thirds.
inline int64_t whole_values(int64_t n, bool thirds) { return thirds ? (n + 31) / 32 * 32 : (n + 7) / 8 * 8; }
inline int64_t pieces_of(int64_t n, int32_t type, bool thirds) {
  return thirds ? (n + 31) / 32 * (kThirds / 16) : (n * type_size(type) + 15) / 16;
}

enum class GemmSize { kSmall, kMiddle, kLarge };
GemmSize gemm_size(int64_t m, int64_t n, int32_t type, bool thirds);

// Whether the tile kernels read these rows where they lie.
inline bool plain(const void* data, int64_t stride, int64_t rows, int64_t columns, int32_t type) {
  const int64_t e = type_size(type);
  return reinterpret_cast<uintptr_t>(data) % 16 == 0 && columns * e % 16 == 0 &&
         (rows <= 1 || (stride * e % 16 == 0 && stride >= columns && stride * e <= kMostStride));
}
inline Rows plain_rows(const void* data, int64_t stride, int64_t rows, int64_t columns, int32_t type) {
  return Rows{static_cast<const uint8_t*>(data),
              rows <= 1 ? pieces_of(columns, type, false) * 16 : stride * type_size(type), rows};
}

// Whether a forward lays float32 rows out in thirds, a pass over the operands that few rows or small
// products do not repay.  Us, as they are / in thirds, M x K to F: 64 x 4096 to 4096 72 / 163, 256 x
// 2048 to 2048 37.6 / 56.3, 512 x 2048 to 2048 68.0 / 67.3, 1000 x 500 to 1000 20.6 / 24.7, 700 x 3000 to 900
// 98 / 85, 1024 x 1024 to 2048 67 / 49, 2048^3 243 / 164.
inline bool in_thirds(const ns_gated_args* a) {
  constexpr int64_t kRepays = 200, kProducts = 1500000000;
  const int64_t results = a->rows * a->width;
  return a->type == NS_TYPE_F32 && results >= kRepays * (a->rows + 2 * a->width) &&
         results >= kProducts / (a->columns > 0 ? a->columns : kProducts);
}

// What has to be laid out anew for the forward, and where in the workspace.
struct PackedForward {
  bool thirds, pack_x, pack_weights;
  int64_t pieces;                          // of a row
  int64_t x, gate, up, bytes;
};
inline PackedForward packed_forward(const ns_gated_args* a) {
  PackedForward w{};
  w.thirds = in_thirds(a);
  w.pieces = pieces_of(a->columns, a->type, w.thirds);
  const int64_t row = w.pieces * 16;
  w.pack_x = w.thirds || !plain(a->x, a->x_stride, a->rows, a->columns, a->type);
  w.pack_weights = w.thirds || !plain(a->gate, a->gate_stride, a->width, a->columns, a->type) ||
                   !plain(a->up, a->up_stride, a->width, a->columns, a->type) ||
                   (a->width > 1 && a->gate_stride != a->up_stride);
  w.gate = w.pack_x ? a->rows * row : 0;
  w.up = w.gate + (w.pack_weights ? a->width * row : 0);
  w.bytes = w.up + (w.pack_weights ? a->width * row : 0);
  return w;
}

// Rows to copy, dense and filled up with zeros, as they are or in thirds: up to three matrices of as
// many columns in one launch, since small calls pay by the launch.
struct PackJob {
  const void* from;
  int64_t stride, rows;
  uint8_t* to;
  int64_t end;                             // of its lanes, in the launch
};
struct PackJobs {
  PackJob of[3];
  int count;
};
void add_pack(PackJobs* jobs, Rows* rows, const void* data, int64_t stride, int64_t pieces, bool thirds,
              uint8_t* to);
int run_packs(const PackJobs& jobs, int64_t columns, int64_t pieces, int32_t type, bool thirds,
              hipStream_t stream);

int check_gated(const ns_gated_args* a);
bool few_rows(const ns_gated_args* a);

}  // namespace ns
