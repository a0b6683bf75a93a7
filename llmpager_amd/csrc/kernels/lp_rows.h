// What the kernels over rows of logits (lp_logits.hip, lp_verify.hip) share.
#pragma once
#include "lp_device.h"

using namespace lp;
using namespace lpk;

namespace {

// Over the wave by row shares of 16 lanes (neighbours, pairs, the halves of eight,
// the halves), then the four rows' from scalar registers: no LDS round trips.
template <int CTRL>
__device__ __forceinline__ double add_dpp(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, false);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    v = add_dpp<0x140>(add_dpp<0x141>(add_dpp<0x4e>(add_dpp<0xb1>(v))));
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    double t = 0.0;
#pragma unroll
    for (int l = 0; l < 64; l += 16)
        t += __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), l) << 32 |
                                            (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, l));
    return t;
}
// (NaN counts as nothing)
__device__ __forceinline__ float wave_top(float v) {
    return __uint_as_float(wave_reduce_u32(__float_as_uint(v), 0xff800000u, [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}

}  // namespace
