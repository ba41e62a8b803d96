// kt_wave.h -- device helpers shared by the decoder's kernels (kt_decoder.hip, kt_kv8.hip):
// reductions over a wave, and the rotary positions as the reference rounds them.
#pragma once

#include "kt_common.h"

namespace kt {

// Sum and maximum over a wave without LDS round trips: inside each row of 16 lanes by DPP
// exchanges (quad xor 1, quad xor 2, half-row mirror, row mirror: every lane of a row ends
// with the same row total, the two operands of each add being the same pair), then the
// four row totals read into scalars and combined in one fixed order, so every lane holds
// the same bits. Needs every lane of the wave active.
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float lane_value(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ float wave_sum_dpp(float v) {
    v += dpp_move<0xB1>(v);   // quad_perm [1,0,3,2]
    v += dpp_move<0x4E>(v);   // quad_perm [2,3,0,1]
    v += dpp_move<0x141>(v);  // row_half_mirror
    v += dpp_move<0x140>(v);  // row_mirror
    return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}
__device__ __forceinline__ float wave_max_dpp(float v) {
    v = fmaxf(v, dpp_move<0xB1>(v));
    v = fmaxf(v, dpp_move<0x4E>(v));
    v = fmaxf(v, dpp_move<0x141>(v));
    v = fmaxf(v, dpp_move<0x140>(v));
    return fmaxf(fmaxf(lane_value(v, 0), lane_value(v, 16)), fmaxf(lane_value(v, 32), lane_value(v, 48)));
}

// RoPE.applyInPlace's rotation of pair (x1, x2) = (row[i], row[i + half]) at pos (K/RoPE.kt:
// 117-137): theta = pos * invFreq[i] in fp32, cos and sin in double rounded to float, no
// contraction.
__device__ __forceinline__ float rope_cos(int32_t pos, float inv_freq_i) {
    return static_cast<float>(cos(static_cast<double>(static_cast<float>(pos) * inv_freq_i)));
}
__device__ __forceinline__ float rope_sin(int32_t pos, float inv_freq_i) {
    return static_cast<float>(sin(static_cast<double>(static_cast<float>(pos) * inv_freq_i)));
}
__device__ __forceinline__ void rope_cos_sin(int32_t pos, float inv_freq_i, float& c, float& s) {
    c = rope_cos(pos, inv_freq_i);
    s = rope_sin(pos, inv_freq_i);
}
// The same by one argument reduction for both.
__device__ __forceinline__ void rope_sin_cos(int32_t pos, float inv_freq_i, float& c, float& s) {
    double cd, sd;
    sincos(static_cast<double>(static_cast<float>(pos) * inv_freq_i), &sd, &cd);
    c = static_cast<float>(cd);
    s = static_cast<float>(sd);
}
__device__ __forceinline__ void rope_apply(float x1, float x2, float c, float s, float& y1, float& y2) {
#pragma clang fp contract(off)
    y1 = x1 * c - x2 * s;
    y2 = x1 * s + x2 * c;
}

}  // namespace kt
