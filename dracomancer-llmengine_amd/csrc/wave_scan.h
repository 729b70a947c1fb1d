// wave_scan.h -- prefix sums over a wave's lanes and values held in scalar
// registers (gfx950, DPP row moves and row broadcasts: no LDS).
#pragma once
#include <hip/hip_runtime.h>

namespace draco {

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long uni(long v) {
    return (long)((unsigned long)(unsigned)uni((int)v) | (unsigned long)(unsigned)uni((int)(v >> 32)) << 32);
}

// Inclusive sums over the lanes, and lane l's value.
template <int CTRL, int ROWS>
__device__ __forceinline__ long dpp_up(long v) {  // 0 where no lane lies that far back
    const int lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xF, false);
    return (long)((unsigned long)(unsigned)lo | (unsigned long)(unsigned)hi << 32);
}
__device__ __forceinline__ long wave_scan(long v) {
    v += dpp_up<0x111, 0xF>(v);  // within rows of 16: 1, 2, 4 and 8 lanes back
    v += dpp_up<0x112, 0xF>(v);
    v += dpp_up<0x114, 0xF>(v);
    v += dpp_up<0x118, 0xF>(v);
    v += dpp_up<0x142, 0xA>(v);  // a row's last lane to the next row, then lane 31 to the upper half
    v += dpp_up<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ long lane_of(long v, int l) {
    return (long)((unsigned long)(unsigned)__builtin_amdgcn_readlane((int)v, l) |
                  (unsigned long)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32);
}
}  // namespace draco
