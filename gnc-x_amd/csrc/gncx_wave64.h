// gncx_wave64.h -- sums of 64-bit values over the lanes of a wave.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace gncx::dev {

// v and another lane's, through DPP (no LDS round trip, unlike a shuffle)
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ double dpp_add_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROW_MASK, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROW_MASK, 0xf, false);
    return v + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Sum over the wave, returned in every lane: wave_sum's steps.
__device__ __forceinline__ double wave_sum_f64(double v) {
    v = dpp_add_f64<0xb1>(v);
    v = dpp_add_f64<0x4e>(v);
    v = dpp_add_f64<0x141>(v);
    v = dpp_add_f64<0x140>(v);
    v = dpp_add_f64<0x142, 0xa>(v);
    v = dpp_add_f64<0x143, 0xc>(v);
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), 63);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), 63);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

}  // namespace gncx::dev
