// What the kernels of 4-bit integer weights share: the matrix, its scales and checks.
#pragma once

#include "ns_signal.h"
#include "neurosim_hip_q4.h"

namespace ns {

struct Q4View {
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;
  int64_t rows, columns, group;
  int64_t blocks, groups;      // of a row: 32 columns, and scales
  int32_t scale_type;
};

__device__ __forceinline__ float q4_scale(const Q4View& w, int64_t at) {
  if (w.scale_type == NS_TYPE_F32) return static_cast<const float*>(w.scales)[at];
  if (w.scale_type == NS_TYPE_BF16) return static_cast<float>(static_cast<const __bf16*>(w.scales)[at]);
  return static_cast<float>(static_cast<const _Float16*>(w.scales)[at]);
}

inline Q4View q4_view(const ns_q4_matrix& m) {
  Q4View w{m.codes, m.scales, m.zeros, m.rows, m.columns, m.group, (m.columns + 31) / 32, 0,
           m.scale_type};
  w.groups = (m.columns + m.group - 1) / m.group;
  return w;
}

inline int check_q4(const ns_q4_matrix& m) {
  if (m.rows < 0 || m.columns < 0) return fail("rows and columns must not be negative");
  if (m.columns > NS_Q4_MAX_COLUMNS) return fail("a 4-bit row has at most %d columns", NS_Q4_MAX_COLUMNS);
  if (m.group != 32 && m.group != 64 && (m.group <= 0 || m.group % 128 || m.group > NS_Q4_MAX_COLUMNS))
    return fail("a group has 32, 64 or a multiple of 128 columns, up to %d", NS_Q4_MAX_COLUMNS);
  if (m.scale_type != NS_TYPE_F32 && m.scale_type != NS_TYPE_BF16 && m.scale_type != NS_TYPE_F16)
    return fail("unknown element type of the scales");
  if (m.rows && m.columns && (!m.codes || !m.scales)) return fail("codes and scales are required");
  if (reinterpret_cast<uintptr_t>(m.codes) % 16) return fail("codes must be 16-byte aligned");
  return NS_OK;
}

}  // namespace ns
