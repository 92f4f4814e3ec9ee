/*
 * wave.h - Sums and maxima over a wave's 64 lanes by VALU moves.
 */
#ifndef W4A16_WAVE_H
#define W4A16_WAVE_H

#include <hip/hip_runtime.h>

namespace w4a16 {

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_zero(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false); }

/* The sum of v over the lanes up to and with this one: row shifts within 16 lanes, then the rows'
 * last lanes carried to the rows behind (six VALU moves; shuffles are six round trips through LDS). */
__device__ __forceinline__ int wave_upto(int v) {
    v += dpp_or_zero<0x111, 0xF>(v);
    v += dpp_or_zero<0x112, 0xF>(v);
    v += dpp_or_zero<0x114, 0xF>(v);
    v += dpp_or_zero<0x118, 0xF>(v);
    v += dpp_or_zero<0x142, 0xA>(v); /* row_bcast:15 into rows 1 and 3 */
    v += dpp_or_zero<0x143, 0xC>(v); /* row_bcast:31 into rows 2 and 3 */
    return v;
}

/* The largest of v >= 0 over the lanes. */
__device__ __forceinline__ int wave_most(int v) {
    auto with = [&](int o) { v = o > v ? o : v; };
    with(dpp_or_zero<0x111, 0xF>(v));
    with(dpp_or_zero<0x112, 0xF>(v));
    with(dpp_or_zero<0x114, 0xF>(v));
    with(dpp_or_zero<0x118, 0xF>(v));
    with(dpp_or_zero<0x142, 0xA>(v));
    with(dpp_or_zero<0x143, 0xC>(v));
    return __builtin_amdgcn_readlane(v, 63);
}

template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_or_least(float v) {
    constexpr int kLeast = (int)0xFF800000u; /* -infinity */
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(kLeast, __builtin_bit_cast(int, v), CTRL, ROWS, 0xF, false));
}

/* The largest of v over the lanes; NaN are none. */
__device__ __forceinline__ float wave_most(float v) {
    v = fmaxf(v, dpp_or_least<0x111, 0xF>(v));
    v = fmaxf(v, dpp_or_least<0x112, 0xF>(v));
    v = fmaxf(v, dpp_or_least<0x114, 0xF>(v));
    v = fmaxf(v, dpp_or_least<0x118, 0xF>(v));
    v = fmaxf(v, dpp_or_least<0x142, 0xA>(v));
    v = fmaxf(v, dpp_or_least<0x143, 0xC>(v));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double v) {
    const uint2 b = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, make_uint2((uint32_t)__builtin_amdgcn_update_dpp(0, (int)b.x, CTRL, ROWS, 0xF, false),
                                                 (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b.y, CTRL, ROWS, 0xF, false)));
}

/* As wave_upto, in FP64. */
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp_or_zero<0x111, 0xF>(v);
    v += dpp_or_zero<0x112, 0xF>(v);
    v += dpp_or_zero<0x114, 0xF>(v);
    v += dpp_or_zero<0x118, 0xF>(v);
    v += dpp_or_zero<0x142, 0xA>(v); /* row_bcast:15 into rows 1 and 3 */
    v += dpp_or_zero<0x143, 0xC>(v); /* row_bcast:31 into rows 2 and 3 */
    return v;
}

__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint2 b = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, make_uint2((uint32_t)__builtin_amdgcn_readlane((int)b.x, lane),
                                                 (uint32_t)__builtin_amdgcn_readlane((int)b.y, lane)));
}

__device__ __forceinline__ double wave_sum(double v) { return lane_f64(wave_scan(v), 63); }

} // namespace w4a16

#endif /* W4A16_WAVE_H */
