// What the two passes of the root-mean-square norm share: how lanes hold a row, sums over them.
#pragma once

#include <type_traits>

#include "rows8.hpp"

namespace kge {

// A value as another lane of a group of 2 * WIDTH has it, the sum so far being the same in WIDTH lanes (or as it is in them: the swaps give both halves).
__device__ __forceinline__ float other_half(float v, int width)
{
    const int b = __float_as_int(v);
    if (width == 1) return __int_as_float(dpp<0xB1>(b));    // quad_perm 1 0 3 2
    if (width == 2) return __int_as_float(dpp<0x4E>(b));    // quad_perm 2 3 0 1
    if (width == 4) return __int_as_float(dpp<0x141>(b));   // row_half_mirror
    return __int_as_float(dpp<0x140>(b));                   // row_mirror
}
__device__ __forceinline__ double other_half(double v, int width)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const float lo = other_half(__int_as_float((int)b), width), hi = other_half(__int_as_float((int)(b >> 32)), width);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__float_as_int(hi) << 32 | (uint32_t)__float_as_int(lo));
}
__device__ __forceinline__ float both_halves(float v, bool wide)  // the sum over two rows of sixteen lanes, or (wide) over two halves of the wave
{
    const uint32_t b = __float_as_uint(v);
    const auto r = wide ? __builtin_amdgcn_permlane32_swap(b, b, false, false) : __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ double both_halves(double v, bool wide)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t x = (uint32_t)b, y = (uint32_t)(b >> 32);
    const auto lo = wide ? __builtin_amdgcn_permlane32_swap(x, x, false, false) : __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const auto hi = wide ? __builtin_amdgcn_permlane32_swap(y, y, false, false) : __builtin_amdgcn_permlane16_swap(y, y, false, false);
    return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) + __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
}
// sum over `lanes` neighbouring lanes (a power of two from 4 to 64), the same in each of them.  No step goes through LDS.
template <class V>
__device__ __forceinline__ V lanes_sum(V v, int lanes)
{
    v += other_half(v, 1);
    v += other_half(v, 2);
    if (lanes > 4) v += other_half(v, 4);
    if (lanes > 8) v += other_half(v, 8);
    if (lanes > 16) v = both_halves(v, false);
    if (lanes > 32) v = both_halves(v, true);
    return v;
}
// sum over 128 or 256 neighbouring threads of a workgroup of 256, the same in each of them; `turn` changes from one call to the next, so that one barrier a call
// is enough
template <class V>
__device__ __forceinline__ V waves_sum(V v, int lanes, V (&part)[2][4], int turn)
{
    v = lanes_sum(v, 64);
    if ((threadIdx.x & 63) == 0) part[turn & 1][threadIdx.x >> 6] = v;
    __syncthreads();
    const V *p = part[turn & 1];
    const int pair = threadIdx.x >> 7 << 1;
    return lanes == 128 ? p[pair] + p[pair + 1] : (p[0] + p[1]) + (p[2] + p[3]);
}

// How a row is held in registers: `pieces` of eight columns a lane (1, 2 or 4; 0: it is too long for that), by `lanes` lanes: a power of two from 4 to 64, or
// 128 or 256, which are several waves.  Two pieces where that still makes `enough` waves, so that they share what a row costs besides; one where it does not; four
// only where rows are too long for fewer.  Forward passes with one, two and four pieces (us): 65536 x 2048 bf16 188, 186, 204, to 8 bits 184, 192, 253;
// 30000 x 300 to 8 bits 32, 25, 25; 65536 x 128 13.0, 11.4, 11.7; 4096 x 1024 to 8 bits 10.0, 11, 14.1.
struct Hold {
    int pieces, lanes;
};
inline Hold hold_of(int64_t rows, int64_t cols, int64_t enough)
{
    const int64_t need = ceil_div(cols, 8);
    if (need > 256 * 4) return Hold{0, 256};
    int pieces = need > 4 && rows * need / 128 >= enough ? 2 : 1, lanes = 4;
    while ((int64_t)lanes * pieces < need && lanes < 256) lanes *= 2;
    while ((int64_t)lanes * pieces < need) pieces *= 2;
    return Hold{pieces, lanes};
}

// A thread's place among the 256 of a workgroup, `lanes` of which hold a row (WAVES: whole waves, all of whose lanes then know that they work on the same one).
template <bool WAVES>
__device__ __forceinline__ void place_in_rows(int lanes, int *lane, uint32_t *group)
{
    *lane = threadIdx.x & (lanes - 1);
    *group = threadIdx.x >> (31 - __builtin_clz(lanes));
    if (WAVES) *group = (uint32_t)__builtin_amdgcn_readfirstlane((int)*group);
}

// How r is kept in 32 bits: as it is, or where it does not fit (2^128 and more: rows whose root mean square is below 2^-128, which only an eps below 2^-256 leaves so) as
// -r 2^-64.  The row's numbers are then taken times 2^64, which rounds none of them, and so is what is multiplied by r again.
__device__ __forceinline__ void to_reach(float kept, float (&v)[8])
{
    if (kept < 0.0f)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= 0x1p64f;
}

// What a sum loses when it is rounded to 16 bits, in sixteenths of a step, -8 .. 7: four bits an element, eight of a row in a word.  bf16: the difference of the two numbers'
// bits, in units of 2^12 (a step at the sum: below a power of two that it was rounded up to, half of the step there); fp16, whose small numbers are evenly spaced: in sixteenths
// of the step at the result.  With it the gradients are those of the sum itself, to 2^-13: from the rounded one alone dweight would be off by 1.4 times its own rounding, and dx of short
// rows, where g - n mean(g n) cancels, by several times.
__device__ __forceinline__ int step_exponent(float h)  // of 1/16 of a step of fp16 at h
{
    const int e = (int)(__float_as_uint(h) >> 23 & 0xFF);
    return (e > 113 ? e : 113) - 127 - 14;
}
template <class T>
__device__ __forceinline__ uint32_t rest_of(const float (&sum)[8])
{
    uint32_t word = 0;
    if constexpr (std::is_same<T, bf16_t>::value) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t lost = __float_as_uint(sum[e]) - __float_as_uint((float)(T)sum[e]), q = (lost + 0x8800u) >> 12;  // (rounded, and 8 more; of a tie downwards 16)
            word |= (q < 15u ? q : 15u) << (4 * e);
        }
        return word ^ 0x88888888u;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float h = (float)(T)sum[e];
        const float q = rintf(__builtin_amdgcn_ldexpf(sum[e] - h, -step_exponent(h)));  // (of what is not finite NaN, and -8 below, which changes neither)
        word |= ((uint32_t)(int)fminf(fmaxf(q, -8.0f), 7.0f) & 15u) << (4 * e);
    }
    return word;
}
template <class T>
__device__ __forceinline__ void add_rest(float (&h)[8], uint32_t word)
{
    if constexpr (std::is_same<T, bf16_t>::value) {
        word ^= 0x88888888u;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = __uint_as_float(__float_as_uint(h[e]) - 0x8000u + ((word >> (4 * e) & 15u) << 12));  // (NaN stays NaN)
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int q = (int)(word << (28 - 4 * e)) >> 28;
        h[e] += __builtin_amdgcn_ldexpf((float)q, step_exponent(h[e]));
    }
}

// calls f with (pieces, whether several waves hold a row) as compile-time values; not for pieces == 0
template <class F>
inline void with_hold(const Hold &h, F &&f)
{
    using std::integral_constant;
    auto waves = [&](auto pieces) {
        if (h.lanes > 64) f(pieces, std::true_type{});
        else f(pieces, std::false_type{});
    };
    if (h.pieces == 1) waves(integral_constant<int, 1>{});
    else if (h.pieces == 2) waves(integral_constant<int, 2>{});
    else waves(integral_constant<int, 4>{});
}

inline int check_norm(const kge_rms_norm *n)
{
    if (!n) return KGE_EINVAL;
    if (!known_type(n->type) || !(known_type(n->out_type) || n->out_type == KGE_E4M3) || !(n->eps >= 0.0) || n->eps > 1.7976931348623157e308) return KGE_EINVAL;
    const int64_t most = (int64_t)1 << 31;
    if (n->rows < 0 || n->cols < 0 || n->rows >= most || n->cols >= most) return KGE_ESHAPE;
    return KGE_OK;
}

}  // namespace kge
