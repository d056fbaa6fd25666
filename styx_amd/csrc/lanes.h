// lanes.h -- sums, maxima and running sums over a wave by lane permutes (the
// VALU's, no LDS round trip), for values of 32 and 64 bits.
#pragma once

#include "common.h"

namespace styx {

template <int CTRL, int ROWS = 0xF, bool ZERO = true> __device__ __forceinline__ uint32_t dpp_u(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, ZERO);
}
// step applied to the words of a value of 4 or 8 bytes
template <typename T, typename Step> __device__ __forceinline__ T by_words(T v, Step step)
{
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, step(__builtin_bit_cast(uint32_t, v)));
    } else {
        static_assert(sizeof(T) == 8, "4 or 8 bytes");
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(T, (uint64_t)step((uint32_t)(u >> 32)) << 32 | step((uint32_t)u));
    }
}
// op over the wave, every lane getting the result: each step pairs a lane
// with one of the other half of its block (bfly's steps, qdot.h)
template <typename T, typename Op> __device__ __forceinline__ T wave_all(T v, Op op)
{
    v = op(v, by_words(v, [](uint32_t x) { return dpp_u<0xB1>(x); }));
    v = op(v, by_words(v, [](uint32_t x) { return dpp_u<0x4E>(x); }));
    v = op(v, by_words(v, [](uint32_t x) { return dpp_u<0x141>(x); }));
    v = op(v, by_words(v, [](uint32_t x) { return dpp_u<0x140>(x); }));
    // of the two words that a swap returns one is the lane's own, the other
    // its partner's
    v = op(v, by_words(v, [](uint32_t x) {
               const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
               return (threadIdx.x & 16) ? r[0] : r[1];
           }));
    v = op(v, by_words(v, [](uint32_t x) {
               const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
               return (threadIdx.x & 32) ? r[0] : r[1];
           }));
    return v;
}
template <typename T> __device__ __forceinline__ T wave_total(T v)
{
    return wave_all(v, [](T a, T b) { return a + b; });
}
template <typename T> __device__ __forceinline__ T wave_most(T v)
{
    return wave_all(v, [](T a, T b) { return a > b ? a : b; });
}
// Inclusive sums of whole numbers in the order of the lanes: within rows of
// 16, then the rows' last lanes passed on (row_bcast:15 to rows 1 and 3, :31
// to the upper half).
template <typename T> __device__ __forceinline__ T wave_upto(T v)
{
    v += by_words(v, [](uint32_t x) { return dpp_u<0x111>(x); });
    v += by_words(v, [](uint32_t x) { return dpp_u<0x112>(x); });
    v += by_words(v, [](uint32_t x) { return dpp_u<0x114>(x); });
    v += by_words(v, [](uint32_t x) { return dpp_u<0x118>(x); });
    v += by_words(v, [](uint32_t x) { return dpp_u<0x142, 0xA, false>(x); });
    v += by_words(v, [](uint32_t x) { return dpp_u<0x143, 0xC, false>(x); });
    return v;
}
// The value of one lane (uniform).
template <typename T> __device__ __forceinline__ T of_lane(T v, int lane)
{
    return by_words(v, [lane](uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, lane); });
}

}  // namespace styx
