// q4k_scan.h -- 64-bit sums over the lanes of a wave, in the registers' own moves between lanes.
#pragma once

#include <hip/hip_runtime.h>

namespace q4k {

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp64(double x) {  // 0 where no lane is
    const unsigned long long b = __double_as_longlong(x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
    return __longlong_as_double(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double wave_scan(double x) {  // inclusive
    x += dpp64<0x111, 0xf>(x);  // row_shr:1, 2, 4, 8 within 16 lanes
    x += dpp64<0x112, 0xf>(x);
    x += dpp64<0x114, 0xf>(x);
    x += dpp64<0x118, 0xf>(x);
    x += dpp64<0x142, 0xa>(x);  // the last lane of rows 0 and 2 to the next row
    x += dpp64<0x143, 0xc>(x);  // of row 1 to rows 2 and 3
    return x;
}
// What lies before each lane, from an inclusive scan: the lane before's, 0 in the first.  (Less the
// lane's own it would lose what is 2^-53 of that.)
__device__ __forceinline__ double wave_before(double inclusive) { return dpp64<0x138, 0xf>(inclusive); }  // wave_shr:1
__device__ __forceinline__ double lane_of(double x, int lane) {
    const unsigned long long b = __double_as_longlong(x);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __longlong_as_double(((unsigned long long)hi << 32) | lo);
}

}  // namespace q4k
