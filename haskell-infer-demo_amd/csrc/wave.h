/*
 * wave.h - Sums and maxima of integers over a wave's 64 lanes by VALU moves.
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

} // namespace w4a16

#endif /* W4A16_WAVE_H */
