// Rotary positions on several axes (time, height, width of a token): pair i of a head turns by the position of the axis
// whose section holds i, sections one after the other.
#pragma once
#include "common.h"

namespace kgc {

constexpr int ROPE_MAX_AXES = 4;
struct RopeAxes {
  int n;                       // 0: one position per token
  int end[ROPE_MAX_AXES];      // axis a: pairs [end[a - 1], end[a])
  int64_t stride;              // positions of axis a: + a * stride
  int rows;                    // of the cos / sin table
};

// cos and sin of pairs i .. i + 7 of token t (positions outside the table: its nearest row)
__device__ __forceinline__ void axes_cos_sin(const RopeAxes& ax, const int64_t* __restrict__ positions, int t,
                                             const float* __restrict__ cos_sin, int d, int i, float (&cc)[8],
                                             float (&sn)[8]) {
  auto axis_of = [&](int p) {
    int a = 0;
#pragma unroll
    for (int k = 0; k < ROPE_MAX_AXES - 1; ++k) a += k < ax.n - 1 && p >= ax.end[k] ? 1 : 0;
    return a;
  };
  auto row_of = [&](int a) {
    const int64_t p = positions[a * ax.stride + t];
    return cos_sin + (p < 0 ? 0 : p >= ax.rows ? ax.rows - 1 : p) * d;
  };
  const int first = axis_of(i), last = axis_of(i + 7);
  if (first == last) {
    const float* cs = row_of(first) + i;
    const float4 c0 = *reinterpret_cast<const float4*>(cs), c1 = *reinterpret_cast<const float4*>(cs + 4);
    const float4 s0 = *reinterpret_cast<const float4*>(cs + d / 2), s1 = *reinterpret_cast<const float4*>(cs + d / 2 + 4);
    cc[0] = c0.x; cc[1] = c0.y; cc[2] = c0.z; cc[3] = c0.w;
    cc[4] = c1.x; cc[5] = c1.y; cc[6] = c1.z; cc[7] = c1.w;
    sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w;
    sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float* cs = row_of(axis_of(i + j)) + i + j;
    cc[j] = cs[0];
    sn[j] = cs[d / 2];
  }
}

}  // namespace kgc
