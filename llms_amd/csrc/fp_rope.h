// fp_rope.h — QK-norm and rotate-half RoPE of one head row, shared by the kernels
// that put q, k and v where attention reads them (fp_attn.hip, fp_kv8.hip).
#pragma once

#include "fp_norm.h"

namespace fp {

// Sum over the LPH (8 or 16) consecutive lanes of a head.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
  v += dpp_f32<0xb1>(v);                            // quad_perm [1,0,3,2]
  v += dpp_f32<0x4e>(v);                            // quad_perm [2,3,0,1]
  v += dpp_f32<0x141>(v);                           // row_half_mirror: sums of 8
  if constexpr (LPH == 16) v += dpp_f32<0x140>(v);  // row_mirror: sums of 16
  return v;
}

// One head row per LPH = D / 8 lanes: lane j holds elements 4j .. 4j+3 of the
// first half (lo) and of the second (hi), so a rotate-half pair sits in one lane.
// g NULL: no norm (the caller has normalised the row). cr, sr: the row's cos and sin.
// Rounded where torch's bf16 ops round: the norm, its weight, each product and the sum.
template <int D>
__device__ __forceinline__ void norm_rope_row(u32x2& lo, u32x2& hi, const uint16_t* g, float eps,
                                              const uint16_t* cr, const uint16_t* sr, int j) {
  constexpr int LPH = D / 8;
  uint32_t x[8] = {lo.x & 0xffffu, lo.x >> 16, lo.y & 0xffffu, lo.y >> 16,
                   hi.x & 0xffffu, hi.x >> 16, hi.y & 0xffffu, hi.y >> 16};
  if (g) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = bf16_bits_to_f32(x[e]);
      s += __fmul_rn(f, f);
    }
    const float r = rms_scale(head_sum<LPH>(s), D, eps);
    const u32x2 gl = *reinterpret_cast<const u32x2*>(g + 4 * j);
    const u32x2 gh = *reinterpret_cast<const u32x2*>(g + D / 2 + 4 * j);
    const uint32_t gb[8] = {gl.x & 0xffffu, gl.x >> 16, gl.y & 0xffffu, gl.y >> 16,
                            gh.x & 0xffffu, gh.x >> 16, gh.y & 0xffffu, gh.y >> 16};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = norm_bf16(x[e], gb[e], r);
  }
  uint32_t y[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x1 = bf16_bits_to_f32(x[e]), x2 = bf16_bits_to_f32(x[4 + e]);
    const int d = 4 * j + e;
    const float c1 = bf16_bits_to_f32(cr[d]), c2 = bf16_bits_to_f32(cr[D / 2 + d]);
    const float s1 = bf16_bits_to_f32(sr[d]), s2 = bf16_bits_to_f32(sr[D / 2 + d]);
    y[e] = f32_to_bf16_bits(round_bf16(__fmul_rn(x1, c1)) + round_bf16(__fmul_rn(-x2, s1)));
    y[4 + e] = f32_to_bf16_bits(round_bf16(__fmul_rn(x2, c2)) + round_bf16(__fmul_rn(x1, s2)));
  }
  lo = u32x2{y[0] | (y[1] << 16), y[2] | (y[3] << 16)};
  hi = u32x2{y[4] | (y[5] << 16), y[6] | (y[7] << 16)};
}

}  // namespace fp
