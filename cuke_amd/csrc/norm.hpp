// What the two passes of the root-mean-square norm share: how lanes hold a row, sums over them.
#pragma once

#include <type_traits>

#include "rows8.hpp"

namespace kge {

// sum over `lanes` neighbouring lanes (a power of two, 64 at most), the same in each of them
template <class V>
__device__ __forceinline__ V lanes_sum(V v, int lanes)
{
    for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor(v, o, kWave);
    return v;
}
// sum over 128 or 256 neighbouring threads of a workgroup of 256, the same in each of them; `part` may be written again behind the next barrier
template <class V>
__device__ __forceinline__ V waves_sum(V v, int lanes, V *part)
{
    v = lanes_sum(v, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    const int pair = threadIdx.x >> 7 << 1;
    return lanes == 128 ? part[pair] + part[pair + 1] : (part[0] + part[1]) + (part[2] + part[3]);
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

// What a sum loses when it is rounded to 16 bits, in sixteenths of a step of the result there, -8 .. 7: four bits an element, eight of a row in a word.  With it the
// gradients are those of the sum itself, to 2^-13: from the rounded one alone dweight would be off by 1.4 times its own rounding, and dx of short rows,
// where g - n mean(g n) cancels, by several times.
template <class T>
__device__ __forceinline__ int step_exponent(float h)  // of 1/16 of a step of T at h
{
    const int e = (int)(__float_as_uint(h) >> 23 & 0xFF), least = std::is_same<T, bf16_t>::value ? 1 : 113;
    return (e > least ? e : least) - 127 - (std::is_same<T, bf16_t>::value ? 11 : 14);
}
template <class T>
__device__ __forceinline__ uint32_t rest_of(const float (&sum)[8])
{
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float h = (float)(T)sum[e];
        const float q = rintf(__builtin_amdgcn_ldexpf(sum[e] - h, -step_exponent<T>(h)));  // (NaN of what is not finite: 0 below)
        word |= ((uint32_t)(int)fminf(fmaxf(q, -8.0f), 7.0f) & 15u) << (4 * e);
    }
    return word;
}
template <class T>
__device__ __forceinline__ void add_rest(float (&h)[8], uint32_t word)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int q = (int)(word << (28 - 4 * e)) >> 28;
        h[e] += __builtin_amdgcn_ldexpf((float)q, step_exponent<T>(h[e]));
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
