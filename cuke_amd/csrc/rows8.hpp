// Rows in 8 bits (kge_rows8): e4m3 numbers with a power of two for each block of 32 columns.  Four lanes with eight consecutive columns each hold a block.
#pragma once

#include "features.hpp"

namespace kge {

struct e4m3_t {};  // the type of an output in 8 bits

struct Rows8 {
    uint8_t *q;
    int64_t q_stride;
    uint8_t *scale;
    int64_t scale_stride;
};

inline int64_t q_width(int64_t cols) { return 32 * ceil_div(cols, 32); }
inline int64_t scale_width(int64_t cols) { return 4 * ceil_div(cols, 128); }
inline Rows8 rows8_of(const kge_rows8 *r)
{
    return r ? Rows8{static_cast<uint8_t *>(r->q), r->q_stride, static_cast<uint8_t *>(r->scale), r->scale_stride} : Rows8{};
}
// whether the arrays are there and lie as the header says
inline int check_rows8(const kge_rows8 *r, int64_t rows, int64_t cols)
{
    if (!r) return KGE_EINVAL;
    if (r->q_stride % 16 != 0 || r->scale_stride % 4 != 0 || r->q_stride < q_width(cols) || r->scale_stride < scale_width(cols)) return KGE_ESHAPE;
    if (rows > 0 && cols > 0 && (!r->q || !r->scale || !aligned16(r->q) || reinterpret_cast<uintptr_t>(r->scale) % 4 != 0)) return KGE_EINVAL;
    return KGE_OK;
}

// kge_unpack8 of rows that have been checked; y [rows, cols] with any cols up to q_width() (what lies behind a row's end is zero)
void launch_unpack8(int type, const Rows8 &in, int64_t rows, int64_t cols, void *y, int64_t y_stride, hipStream_t st);

template <int CTRL>
__device__ __forceinline__ int dpp(int v)
{
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ float quad_max(float v)  // over four neighbouring lanes, none below 0
{
    v = fmaxf(v, __int_as_float(dpp<0xB1>(__float_as_int(v))));
    return fmaxf(v, __int_as_float(dpp<0x4E>(__float_as_int(v))));
}

// The byte of the least power of two that brings `top` (finite, not negative) to 448 = 1.75 2^8 at most: a mantissa above 1.75 carries into the exponent.
__device__ __forceinline__ int scale_byte(float top)
{
    const int e = (int)((__float_as_uint(top) + 0x1FFFFFu) >> 23) - 8;
    return e > 0 ? e : 0;
}
__device__ __forceinline__ float scale_inverse(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }  // (of the bytes above: 0 .. 247)
__device__ __forceinline__ float scale_value(int byte)
{
    return byte == 0 ? 0x1p-127f : (byte == 255 ? __builtin_nanf("") : __uint_as_float((uint32_t)byte << 23));
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

// eight values, each 448 at most or not finite (NaN then, by the instruction too), to e4m3
__device__ __forceinline__ uint2 to_e4m3(const float (&v)[8])
{
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}
__device__ __forceinline__ void from_e4m3(uint2 q, float scale, float (&v)[8])
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, true);
    const f2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, true);
    v[0] = a[0] * scale, v[1] = a[1] * scale, v[2] = b[0] * scale, v[3] = b[1] * scale;
    v[4] = c[0] * scale, v[5] = c[1] * scale, v[6] = d[0] * scale, v[7] = d[1] * scale;
}

// the largest of eight values that is finite (a maximum passes NaN over; infinities are rare enough to be looked for afterwards)
__device__ __forceinline__ float top_of(const float (&v)[8])
{
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
    if (!finite(top)) {
        top = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, finite(v[e]) ? fabsf(v[e]) : 0.0f);
    }
    return top;
}

}  // namespace kge
