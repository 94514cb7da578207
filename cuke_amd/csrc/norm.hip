// Root-mean-square norm of rows with a residual's addition in front of it, to rows of a type or of 8 bits (kge_rms_norm_fwd).
//
//   h = x + residual,  r = (mean h^2 + eps)^-1/2,  y = h r weight
//
// One pass: a row waits in registers while its squares are summed.  The sum is one of 64-bit products (the matrix and vector units form them at the pace of 32-bit
// ones, and memory is slower than either): no value of a type overflows in it, and with it any element can be formed again in 64 bits.
#include <type_traits>

#include "norm.hpp"

namespace kge {

struct NormArgs {
    const void *x, *residual, *weight;
    int64_t x_stride, residual_stride;
    int64_t rows, cols;
    double eps, share;  // share: 1 / cols
    void *y;
    int64_t y_stride;
    Rows8 y8;
    void *h;
    int64_t h_stride;
    float *rstd;
    uint32_t *rest;  // [rows][ceil(cols / 8)], or NULL
    int lanes;       // of a row
};

template <class T>
__device__ __forceinline__ double sum_at(const NormArgs &a, int64_t row, int64_t col)
{
    double h = (double)(float)static_cast<const T *>(a.x)[row * a.x_stride + col];
    if (a.residual) h += (double)(float)static_cast<const T *>(a.residual)[row * a.residual_stride + col];
    return h;
}
// r of a row as it is kept (to_reach()), to half a unit of its last place and 2^-40: the instruction's 2^-23 and a step of Newton's method
__device__ __forceinline__ float root(const NormArgs &a, double sum)
{
    const double m = fma(sum, a.share, a.eps), r = __builtin_amdgcn_rsq(m);
    const double better = r * fma(-0.5 * m * r, r, 1.5), v = r > 0.0 && r < 1e300 ? better : r;  // (of 0 and infinity the step would make NaN)
    const float f = (float)v;
    return finite(f) || !(v < 1e300) ? f : -(float)fmin(v * 0x1p-64, 0x1.fffffep127);  // (beyond that rows are zeros)
}
// r in 64 bits, and an element of the result, from memory
__device__ __forceinline__ double root64(const NormArgs &a, double sum) { return 1.0 / sqrt(sum / (double)a.cols + a.eps); }
template <class T>
__device__ __forceinline__ double result_at(const NormArgs &a, int64_t row, int64_t col, double r)
{
    const double y = sum_at<T>(a, row, col) * r;
    return a.weight ? y * (double)(float)static_cast<const T *>(a.weight)[col] : y;
}
// to 32 bits towards zero, the last bit set where that was not exact: what is rounded further from there lands where the 64-bit value does
__device__ __forceinline__ float to_odd(double d)
{
    float f = (float)d;
    if (!finite(f) || (double)f == d) return f;
    uint32_t b = __float_as_uint(f);
    if (fabs((double)f) > fabs(d)) --b;
    return __uint_as_float(b | 1u);
}
template <class T>
__device__ __forceinline__ float top_in_64(const NormArgs &a, int64_t row, int64_t col, double sum)
{
    const double r = root64(a, sum);
    float top = 0.0f;
#pragma unroll 1
    for (int e = 0; e < 8 && col + e < a.cols; ++e) {
        const float v = fabsf(to_odd(result_at<T>(a, row, col + e, r)));
        top = fmaxf(top, finite(v) ? v : 0.0f);
    }
    return top;
}
// the bytes of q that differ from `other` formed again (one, as a rule)
template <class T>
__device__ __forceinline__ uint2 settle(const NormArgs &a, int64_t row, int64_t col, double sum, float inverse, uint2 q, uint2 other)
{
    uint64_t all = (uint64_t)q.y << 32 | q.x, differ = all ^ ((uint64_t)other.y << 32 | other.x);
    const double r = root64(a, sum);
#pragma unroll 1
    while (differ) {
        const int shift = __builtin_ctzll(differ) & ~7;
        const uint64_t mask = 0xFFull << shift;
        differ &= ~mask;
        if (col + shift / 8 >= a.cols) continue;
        const float v = to_odd(result_at<T>(a, row, col + shift / 8, r) * (double)inverse);
        all = (all & ~mask) | (uint64_t)((uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xFFu) << shift;
    }
    return make_uint2((uint32_t)all, (uint32_t)(all >> 32));
}

// Eight consecutive results (fp32, each within 6 units of its last place; zero behind the row's end) to 8 bits; the lanes of a block come together.  A value that another
// rounding of fp32 would put on the other side of a border of e4m3, one in 100000, is formed again in 64 bits, and so is a block's largest value at the border
// of two powers: to see that, every value is rounded twice, 16 units apart.
constexpr float kUp = 1.0f + 0x1p-21f, kDown = 1.0f - 0x1p-21f;
template <class T>
__device__ __forceinline__ void store_e4m3(const NormArgs &a, int64_t row, int64_t col, double sum, const float (&y)[8], bool there)
{
    const int64_t width = (a.cols + 31) / 32 * 32;
    const float top = quad_max(top_of(y));
    int byte = scale_byte(top * kDown);
    if (byte != scale_byte(top * kUp)) byte = scale_byte(quad_max(top_in_64<T>(a, row, col, sum)));
    const float inverse = scale_inverse(byte), down = inverse * kDown, up = inverse * kUp;
    float low[8], high[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) low[e] = y[e] * down, high[e] = y[e] * up;
    uint2 q = to_e4m3(low);
    const uint2 other = to_e4m3(high);
    if (q.x != other.x || q.y != other.y) q = settle<T>(a, row, col, sum, inverse, q, other);
    if (there && col < width) {
        *reinterpret_cast<uint2 *>(a.y8.q + row * a.y8.q_stride + col) = q;
        if ((col & 31) == 0) a.y8.scale[row * a.y8.scale_stride + col / 32] = (uint8_t)byte;
    }
}
// zeros behind a row's last scale
__device__ __forceinline__ void finish_scales(const NormArgs &a, int64_t row, int lane)
{
    const int64_t blocks = (a.cols + 31) / 32, at = blocks + lane;
    if (lane < 3 && at < (blocks + 3) / 4 * 4) a.y8.scale[row * a.y8.scale_stride + at] = 0;
}

// A row is held in registers, C pieces of eight columns a lane, by `lanes` lanes (WAVES: by two or four waves).  FULL: rows are whole pieces.
// Bound by memory where rows are many: 65536 x 2048 bf16 with a residual and rest (1.14 GB) 185 us, 6.2 TB/s; a copy of 2 GB reaches 5.0.  Of few rows by what a wave
// has to do for its share of one: 4096 x 1024 to 8 bits (29 MB) 9.4 us, to bf16 7.7, of which a launch, a row's read and, requested behind its sum, the
// weight's are 4.
template <class T, class O, int C, bool WAVES, bool FULL>
__global__ __launch_bounds__(256) void rms_norm_kernel(NormArgs a)
{
    __shared__ double part[2][4];
    int turn = 0;
    int lane;
    uint32_t group;
    place_in_rows<WAVES>(a.lanes, &lane, &group);
    const int lanes = a.lanes, groups = 256 >> (31 - __builtin_clz(lanes));
    auto column = [&](int c) { return 8 * (c * lanes + lane); };
    auto valid = [&](int c) { return (int)a.cols - column(c); };
    auto load = [&](const void *from, int64_t at, int c, float(&v)[8]) {
        const T *p = static_cast<const T *>(from) + at + column(c);
        if (FULL ? valid(c) > 0 : valid(c) >= 8) {
            const auto q = Pack<T, 8>::load(p).v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)q[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
            if (FULL || valid(c) <= 0) return;
            // (a row's end in three loads at most)
            const int four = valid(c) & 4, two = valid(c) & 2;
            if (four) {
                const auto q = Pack<T, 4>::load(p).v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (float)q[e];
            }
            if (two) {
                const auto q = Pack<T, 2>::load(p + four).v;
                if (four) v[4] = (float)q[0], v[5] = (float)q[1];
                else v[0] = (float)q[0], v[1] = (float)q[1];
            }
            if (valid(c) & 1) {
                const float q = (float)p[four + two];
#pragma unroll
                for (int e = 0; e < 7; e += 2)
                    if (e == four + two) v[e] = q;
            }
        }
    };
    for (int64_t row0 = (int64_t)blockIdx.x * groups; row0 < a.rows; row0 += (int64_t)gridDim.x * groups) {
        const bool there = row0 + group < a.rows;
        const int64_t row = (uint32_t)row0 + (there ? group : 0u);  // (lanes without a row of their own go along)
        float h[C][8];
        double sum = 0.0;
#pragma unroll
        for (int c = 0; c < C; ++c) load(a.x, row * a.x_stride, c, h[c]);
        if (a.residual) {
            float more[C][8];
#pragma unroll
            for (int c = 0; c < C; ++c) load(a.residual, row * a.residual_stride, c, more[c]);
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) h[c][e] += more[c][e];
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (a.h && there) store8(static_cast<T *>(a.h) + row * a.h_stride + column(c), h[c], FULL && valid(c) > 0 ? 8 : valid(c));
            if constexpr (sizeof(T) == 2)
                if (a.rest && there && valid(c) > 0) a.rest[row * ((a.cols + 7) / 8) + column(c) / 8] = rest_of<T>(h[c]);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fma((double)h[c][e], (double)h[c][e], sum);
        }
        sum = WAVES ? waves_sum(sum, lanes, part, turn++) : lanes_sum(sum, lanes);
        const float kept = root(a, sum), r = fabsf(kept);
        if (a.rstd && there && lane == 0) a.rstd[row] = kept;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            to_reach(kept, h[c]);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[c][e] *= r;
            if (a.weight) {
                float w[8];
                load(a.weight, 0, c, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[c][e] *= w[e];
            }
            if constexpr (std::is_same<O, e4m3_t>::value) store_e4m3<T>(a, row, column(c), sum, h[c], there);
            else if (there) store8(static_cast<O *>(a.y) + row * a.y_stride + column(c), h[c], FULL && valid(c) > 0 ? 8 : valid(c));
        }
        if constexpr (std::is_same<O, e4m3_t>::value)
            if (there) finish_scales(a, row, lane);
    }
}

// The same of rows that registers do not hold: a workgroup goes over a row twice.
template <class T, class O>
__global__ __launch_bounds__(256) void rms_norm_long_kernel(NormArgs a)
{
    __shared__ double part[2][4];
    int turn = 0;
    auto load = [&](int64_t row, int64_t col, float(&h)[8]) {
        const int64_t left = a.cols - col;
        const int valid = (int)(left < 8 ? left : 8);
        load8(static_cast<const T *>(a.x) + row * a.x_stride + col, valid, h);
        if (!a.residual) return valid;
        float more[8];
        load8(static_cast<const T *>(a.residual) + row * a.residual_stride + col, valid, more);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] += more[e];
        return valid;
    };
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        double sum = 0.0;
        for (int64_t col = 8 * threadIdx.x; col < a.cols; col += 8 * 256) {
            float h[8];
            load(row, col, h);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fma((double)h[e], (double)h[e], sum);
        }
        sum = waves_sum(sum, 256, part, turn++);
        const float kept = root(a, sum), r = fabsf(kept);
        if (a.rstd && threadIdx.x == 0) a.rstd[row] = kept;
        for (int64_t col0 = 0; col0 < a.cols; col0 += 8 * 256) {  // (all lanes come along)
            const int64_t col = col0 + 8 * threadIdx.x;
            float h[8];
            const int valid = load(row, col, h);
            if (a.h) store8(static_cast<T *>(a.h) + row * a.h_stride + col, h, valid);
            if constexpr (sizeof(T) == 2)
                if (a.rest && valid > 0) a.rest[row * ((a.cols + 7) / 8) + col / 8] = rest_of<T>(h);
            to_reach(kept, h);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] *= r;
            if (a.weight) {
                float w[8];
                load8(static_cast<const T *>(a.weight) + col, valid, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] *= w[e];
            }
            if constexpr (std::is_same<O, e4m3_t>::value) store_e4m3<T>(a, row, col, sum, h, true);
            else store8(static_cast<O *>(a.y) + row * a.y_stride + col, h, valid);
        }
        if constexpr (std::is_same<O, e4m3_t>::value) finish_scales(a, row, threadIdx.x);
    }
}

template <class T, class O>
static void launch_norm(const NormArgs &args, hipStream_t st)
{
    NormArgs a = args;
    const Hold hold = hold_of(a.rows, a.cols, 8192);
    a.lanes = hold.lanes;
    const int64_t blocks = ceil_div(a.rows, 256 / hold.lanes);
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20))), block(256);
    if (hold.pieces == 0) {
        hipLaunchKernelGGL((rms_norm_long_kernel<T, O>), grid, block, 0, st, a);
        return;
    }
    with_hold(hold, [&](auto pieces, auto waves) {
        if (a.cols % 8 == 0) hipLaunchKernelGGL((rms_norm_kernel<T, O, decltype(pieces)::value, decltype(waves)::value, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((rms_norm_kernel<T, O, decltype(pieces)::value, decltype(waves)::value, false>), grid, block, 0, st, a);
    });
}
template <class T>
static void launch_norm(const NormArgs &a, int out_type, hipStream_t st)
{
    if (out_type == KGE_E4M3) launch_norm<T, e4m3_t>(a, st);
    else if (out_type == KGE_F32) launch_norm<T, float>(a, st);
    else if (out_type == KGE_BF16) launch_norm<T, bf16_t>(a, st);
    else launch_norm<T, half_t>(a, st);
}

}  // namespace kge

using namespace kge;

extern "C" {

int kge_rms_norm_fwd(const kge_rms_norm *norm, void *y, int64_t y_stride, const kge_rows8 *y8, void *h, int64_t h_stride, float *rstd,
                     void *rest, void *stream)
{
    if (const int rc = check_norm(norm)) return rc;
    if (norm->x_stride < norm->cols || (norm->residual && norm->residual_stride < norm->cols) || (h && h_stride < norm->cols)) return KGE_ESHAPE;
    const bool eight = norm->out_type == KGE_E4M3;
    if (eight) {
        if (const int rc = check_rows8(y8, norm->rows, norm->cols)) return rc;
    } else if (y_stride < norm->cols) {
        return KGE_ESHAPE;
    }
    if (norm->rows == 0 || norm->cols == 0) return KGE_OK;
    if (!norm->x || (!eight && !y) || reinterpret_cast<uintptr_t>(rest) % 4 != 0) return KGE_EINVAL;
    const NormArgs a{norm->x, norm->residual, norm->weight, norm->x_stride, norm->residual_stride, norm->rows, norm->cols, norm->eps, 1.0 / (double)norm->cols,
                     y, y_stride, rows8_of(eight ? y8 : nullptr), h, h_stride, rstd, static_cast<uint32_t *>(rest), 0};
    hipStream_t st = as_stream(stream);
    KGE_CLEAR_LAUNCH_ERRORS();
    if (norm->type == KGE_F32) launch_norm<float>(a, norm->out_type, st);
    else if (norm->type == KGE_BF16) launch_norm<bf16_t>(a, norm->out_type, st);
    else launch_norm<half_t>(a, norm->out_type, st);
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

}  // extern "C"
