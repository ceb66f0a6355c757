// Running sums, sums and the largest value of a wave's 64 lanes for the operators on the caller's device buffers.
#pragma once
#include "hipdec_common.h"

// Double precision over the 64 lanes of a wave by data-parallel moves (an LDS round trip per step is 0.1 us, six of them
// in a row for every sum).  Inclusive running sum; the total is lane 63's.
template <int CTRL, int ROW_MASK> __device__ __forceinline__ double dpp_get64(double v) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROW_MASK, 0xf, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROW_MASK, 0xf, false));
}
__device__ __forceinline__ double wave_scan_f64(double v) {
    v += dpp_get64<0x111, 0xf>(v);   // row_shr:1
    v += dpp_get64<0x112, 0xf>(v);   // row_shr:2
    v += dpp_get64<0x114, 0xf>(v);   // row_shr:4
    v += dpp_get64<0x118, 0xf>(v);   // row_shr:8
    v += dpp_get64<0x142, 0xa>(v);   // row_bcast:15 into rows 1 and 3
    v += dpp_get64<0x143, 0xc>(v);   // row_bcast:31 into rows 2 and 3
    return v;
}
// a lane's value in every lane (the lane the same for the whole wave)
__device__ __forceinline__ double wave_read_f64(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
// the lane before's value, 0 in lane 0
__device__ __forceinline__ double wave_before_f64(double v) { return dpp_get64<0x138, 0xf>(v); }   // wave_shr:1
template <int CTRL, int ROW_MASK> __device__ __forceinline__ float dpp_max(float v) {
    const int i = __float_as_int(v);
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, ROW_MASK, 0xf, false)));
}
// the largest of the 64 lanes, in every lane
__device__ __forceinline__ float wave_max_dpp(float v) {
    v = dpp_max<0x111, 0xf>(v);
    v = dpp_max<0x112, 0xf>(v);
    v = dpp_max<0x114, 0xf>(v);
    v = dpp_max<0x118, 0xf>(v);
    v = dpp_max<0x142, 0xa>(v);
    v = dpp_max<0x143, 0xc>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
