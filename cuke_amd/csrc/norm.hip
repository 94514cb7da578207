// Root-mean-square norm of rows with a residual's addition in front of it, to rows of a type or of 8 bits, and its gradients (kge_rms_norm_fwd,
// kge_rms_norm_bwd).
#include "linear_tile.hpp"
#include "rows8.hpp"

namespace kge {

struct NormArgs {
    const void *x, *residual, *weight;
    int64_t x_stride, residual_stride;
    int64_t rows, cols;
    double eps;
    void *y;
    int64_t y_stride;
    Rows8 y8;
    void *h;
    int64_t h_stride;
    float *rstd;
    int lanes;  // of a row: a power of two from 4 to 64
};

// sum over `lanes` neighbouring lanes (a power of two), the same in each of them
template <class V>
__device__ __forceinline__ V lanes_sum(V v, int lanes)
{
    for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor(v, o, kWave);
    return v;
}
// sum over a workgroup of 256, the same in each thread; `part` is free to be written again after the next barrier
template <class V>
__device__ __forceinline__ V block_sum(V v, V *part)
{
    v = lanes_sum(v, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

template <class T>
__device__ __forceinline__ double sum_at(const NormArgs &a, int64_t row, int64_t col)
{
    double h = (double)(float)static_cast<const T *>(a.x)[row * a.x_stride + col];
    if (a.residual) h += (double)(float)static_cast<const T *>(a.residual)[row * a.residual_stride + col];
    return h;
}
// an element of the result in 64 bits, from memory
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

// Eight consecutive results (fp32, each within 4 units of its last place; zero behind the row's end) to 8 bits; the lanes of a block come together.  A value that another rounding of fp32
// would put on the other side of a border of e4m3, one in 40000, is formed again in 64 bits, and so is a block's largest value at the border of two powers.
constexpr float kUp = 1.0f + 0x1p-20f, kDown = 1.0f - 0x1p-20f;
template <class T>
__device__ __forceinline__ void store_e4m3(const NormArgs &a, int64_t row, int64_t col, double r, const float (&y)[8], bool there)
{
    const int64_t width = (a.cols + 31) / 32 * 32;
    float top = quad_max(top_of(y));
    int byte = scale_byte(top * kDown);
    if (byte != scale_byte(top * kUp)) {
        top = 0.0f;
        for (int e = 0; e < 8; ++e) {
            const float v = col + e < a.cols ? fabsf(to_odd(result_at<T>(a, row, col + e, r))) : 0.0f;
            top = fmaxf(top, finite(v) ? v : 0.0f);
        }
        top = quad_max(top);
        byte = scale_byte(top);
    }
    const float inverse = scale_inverse(byte);
    float low[8], high[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) low[e] = y[e] * inverse * kDown, high[e] = y[e] * inverse * kUp;
    uint2 q = to_e4m3(low);
    const uint2 other = to_e4m3(high);
    if (q.x != other.x || q.y != other.y) {
#pragma unroll
        for (int e = 0; e < 8; ++e) low[e] = y[e] * inverse;
        for (int e = 0; e < 8; ++e) {
            if (((e < 4 ? q.x ^ other.x : q.y ^ other.y) >> (8 * (e & 3)) & 0xFF) == 0) continue;
            const float v = col + e < a.cols ? to_odd(result_at<T>(a, row, col + e, r) * (double)inverse) : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (u == e) low[u] = v;
        }
        q = to_e4m3(low);
    }
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

// A row is held in registers, C pieces of eight columns a lane: by `lanes` lanes of a wave (BLOCK: by the workgroup).
template <class T, class O, int C, bool BLOCK>
__global__ __launch_bounds__(256) void rms_norm_kernel(NormArgs a)
{
    __shared__ double part[4];
    const int lanes = BLOCK ? 256 : a.lanes, lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = 256 / lanes;
    for (int64_t row0 = (int64_t)blockIdx.x * groups; row0 < a.rows; row0 += (int64_t)gridDim.x * groups) {
        const bool there = row0 + group < a.rows;
        const int64_t row = there ? row0 + group : a.rows - 1;  // (lanes without a row of their own go along)
        float h[C][8];
        double sum = 0.0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t col = 8 * ((int64_t)c * lanes + lane), left = a.cols - col;
            load8(static_cast<const T *>(a.x) + row * a.x_stride + col, (int)(left < 8 ? left : 8), h[c]);
        }
        if (a.residual) {
            float more[C][8];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int64_t col = 8 * ((int64_t)c * lanes + lane), left = a.cols - col;
                load8(static_cast<const T *>(a.residual) + row * a.residual_stride + col, (int)(left < 8 ? left : 8), more[c]);
            }
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) h[c][e] += more[c][e];
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t col = 8 * ((int64_t)c * lanes + lane), left = a.cols - col;
            if (a.h && there) store8(static_cast<T *>(a.h) + row * a.h_stride + col, h[c], (int)(left < 8 ? left : 8));
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fma((double)h[c][e], (double)h[c][e], sum);
        }
        sum = BLOCK ? block_sum(sum, part) : lanes_sum(sum, lanes);
        const double r64 = 1.0 / sqrt(sum / (double)a.cols + a.eps);
        const float r = (float)r64;
        if (a.rstd && there && lane == 0) a.rstd[row] = r;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t col = 8 * ((int64_t)c * lanes + lane), left = a.cols - col;
            const int valid = (int)(left < 8 ? left : 8);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[c][e] *= r;
            if (a.weight) {
                float w[8];
                load8(static_cast<const T *>(a.weight) + col, valid, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[c][e] *= w[e];
            }
            if constexpr (std::is_same<O, e4m3_t>::value) store_e4m3<T>(a, row, col, r64, h[c], there);
            else if (there) store8(static_cast<O *>(a.y) + row * a.y_stride + col, h[c], valid);
        }
        if constexpr (std::is_same<O, e4m3_t>::value)
            if (there) finish_scales(a, row, lane);
    }
}

// The same of rows that registers do not hold: a workgroup goes over a row twice.
template <class T, class O>
__global__ __launch_bounds__(256) void rms_norm_long_kernel(NormArgs a)
{
    __shared__ double part[4];
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
        sum = block_sum(sum, part);
        const double r64 = 1.0 / sqrt(sum / (double)a.cols + a.eps);
        const float r = (float)r64;
        if (a.rstd && threadIdx.x == 0) a.rstd[row] = r;
        for (int64_t col0 = 0; col0 < a.cols; col0 += 8 * 256) {  // (all lanes come along)
            const int64_t col = col0 + 8 * threadIdx.x;
            float h[8];
            const int valid = load(row, col, h);
            if (a.h) store8(static_cast<T *>(a.h) + row * a.h_stride + col, h, valid);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] *= r;
            if (a.weight) {
                float w[8];
                load8(static_cast<const T *>(a.weight) + col, valid, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] *= w[e];
            }
            if constexpr (std::is_same<O, e4m3_t>::value) store_e4m3<T>(a, row, col, r64, h, true);
            else store8(static_cast<O *>(a.y) + row * a.y_stride + col, h, valid);
        }
        if constexpr (std::is_same<O, e4m3_t>::value) finish_scales(a, row, threadIdx.x);
    }
}

// ---- gradients -------------------------------------------------------------------------------------
struct NormGradArgs {
    const void *h, *dy, *dh, *weight;
    int64_t h_stride, dy_stride, dh_stride;
    const float *rstd;
    int64_t rows, cols, quads, rows_each;
    void *dx;     // or NULL
    int64_t dx_stride;
    float *sums;  // [ranges][4 quads]: dweight's over a range of rows, or NULL
    int lanes;
};

// With n = h r: dx = r (g - n mean(g n)) + dh, dweight = sum dy n.  A workgroup takes a range of rows; a lane's columns are the same in all of them,
// so dweight's sums wait in registers until its end.
template <class T, class D, int C, bool BLOCK>
__global__ __launch_bounds__(256) void rms_norm_grad_kernel(NormGradArgs a)
{
    __shared__ float part[4];
    __shared__ float s_sum[BLOCK ? 1 : 256][8];
    const int lanes = BLOCK ? 256 : a.lanes, lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = 256 / lanes;
    const int64_t first = (int64_t)blockIdx.x * a.rows_each, last = first + a.rows_each < a.rows ? first + a.rows_each : a.rows;
    const float share = 1.0f / (float)a.cols;
    float sum[C][8] = {};
    for (int64_t row0 = first; row0 < last; row0 += groups) {
        const bool there = row0 + group < last;
        const int64_t row = there ? row0 + group : last - 1;
        float n[C][8], g[C][8], dot = 0.0f;
        const float r = a.rstd[row];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t col = 8 * ((int64_t)c * lanes + lane), left = a.cols - col;
            const int valid = (int)(left < 8 ? left : 8);
            load8(static_cast<const T *>(a.h) + row * a.h_stride + col, valid, n[c]);
            load8(static_cast<const D *>(a.dy) + row * a.dy_stride + col, valid, g[c]);
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t col = 8 * ((int64_t)c * lanes + lane), left = a.cols - col;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                n[c][e] *= r;
                if (there) sum[c][e] = fmaf(g[c][e], n[c][e], sum[c][e]);
            }
            if (a.weight) {
                float w[8];
                load8(static_cast<const T *>(a.weight) + col, (int)(left < 8 ? left : 8), w);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[c][e] *= w[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) dot = fmaf(g[c][e], n[c][e], dot);
        }
        if (!a.dx) continue;
        const float mean = (BLOCK ? block_sum(dot, part) : lanes_sum(dot, lanes)) * share;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t col = 8 * ((int64_t)c * lanes + lane), left = a.cols - col;
            const int valid = (int)(left < 8 ? left : 8);
            float d[8] = {};
            if (a.dh) load8(static_cast<const T *>(a.dh) + row * a.dh_stride + col, valid, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = fmaf(r, g[c][e] - n[c][e] * mean, d[e]);
            if (there) store8(static_cast<T *>(a.dx) + row * a.dx_stride + col, d, valid);
        }
    }
    if (!a.sums) return;
    float *to = a.sums + (int64_t)blockIdx.x * a.quads * 4;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int64_t col = 8 * ((int64_t)c * lanes + lane);
        if constexpr (!BLOCK) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) s_sum[threadIdx.x][e] = sum[c][e];
            __syncthreads();
            if (group) continue;
            for (int k = 1; k < groups; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[c][e] += s_sum[k * lanes + lane][e];
        }
        if (col < a.cols) *reinterpret_cast<float4 *>(to + col) = make_float4(sum[c][0], sum[c][1], sum[c][2], sum[c][3]);
        if (col + 4 < a.cols) *reinterpret_cast<float4 *>(to + col + 4) = make_float4(sum[c][4], sum[c][5], sum[c][6], sum[c][7]);
    }
}

// dx of rows that registers do not hold
template <class T, class D>
__global__ __launch_bounds__(256) void rms_norm_grad_long_kernel(NormGradArgs a)
{
    __shared__ float part[4];
    auto load = [&](int64_t row, int64_t col, float r, float(&n)[8], float(&g)[8]) {
        const int64_t left = a.cols - col;
        const int valid = (int)(left < 8 ? left : 8);
        load8(static_cast<const T *>(a.h) + row * a.h_stride + col, valid, n);
        load8(static_cast<const D *>(a.dy) + row * a.dy_stride + col, valid, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) n[e] *= r;
        if (!a.weight) return valid;
        float w[8];
        load8(static_cast<const T *>(a.weight) + col, valid, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] *= w[e];
        return valid;
    };
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float r = a.rstd[row];
        float dot = 0.0f;
        for (int64_t col = 8 * threadIdx.x; col < a.cols; col += 8 * 256) {
            float n[8], g[8];
            load(row, col, r, n, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) dot = fmaf(g[e], n[e], dot);
        }
        const float mean = block_sum(dot, part) * (1.0f / (float)a.cols);
        for (int64_t col = 8 * threadIdx.x; col < a.cols; col += 8 * 256) {
            float n[8], g[8], d[8] = {};
            const int valid = load(row, col, r, n, g);
            if (a.dh) load8(static_cast<const T *>(a.dh) + row * a.dh_stride + col, valid, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = fmaf(r, g[e] - n[e] * mean, d[e]);
            store8(static_cast<T *>(a.dx) + row * a.dx_stride + col, d, valid);
        }
    }
}
// dweight's sums over ranges of rows, of such rows: eight columns a thread
template <class T, class D>
__global__ __launch_bounds__(256) void rms_norm_long_sums_kernel(NormGradArgs a)
{
    const int64_t first = (int64_t)blockIdx.y * a.rows_each, last = first + a.rows_each < a.rows ? first + a.rows_each : a.rows;
    const int64_t col = 8 * ((int64_t)blockIdx.x * 256 + threadIdx.x), left = a.cols - col;
    if (left <= 0) return;
    const int valid = (int)(left < 8 ? left : 8);
    float sum[8] = {};
    for (int64_t row = first; row < last; ++row) {
        const float r = a.rstd[row];
        float n[8], g[8];
        load8(static_cast<const T *>(a.h) + row * a.h_stride + col, valid, n);
        load8(static_cast<const D *>(a.dy) + row * a.dy_stride + col, valid, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = fmaf(g[e], n[e] * r, sum[e]);
    }
    float *to = a.sums + (int64_t)blockIdx.y * a.quads * 4 + col;
    *reinterpret_cast<float4 *>(to) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    if (valid > 4) *reinterpret_cast<float4 *>(to + 4) = make_float4(sum[4], sum[5], sum[6], sum[7]);
}

template <class T>
__global__ __launch_bounds__(256) void norm_join_kernel(SumArgs j)
{
    __shared__ float4 lds[256];
    join_sums<T, 256>(j, blockIdx.x, lds);
}

// ---- launches --------------------------------------------------------------------------------------
// How a row is held: pieces a lane and lanes, or a workgroup.  As few lanes as hold it in four pieces each leave the others to other rows; what
// is wasted behind a row's end counts first.
struct Hold {
    int pieces, lanes;  // pieces 0: not in registers
};
static Hold hold_of(int64_t cols)
{
    const int64_t need = ceil_div(cols, 8);
    if (need > 256 * 4) return Hold{0, 256};
    if (need > 64 * 4) return Hold{need > 256 * 2 ? 4 : 2, 256};
    Hold best{4, 64};
    for (int lanes = 4; lanes <= 64; lanes *= 2)
        for (int pieces = 1; pieces <= 4; ++pieces)
            if ((int64_t)lanes * pieces >= need && lanes * pieces < best.lanes * best.pieces) best = Hold{pieces, lanes};
    return best;
}

template <class T, class O>
static void launch_norm(const NormArgs &args, hipStream_t st)
{
    NormArgs a = args;
    const Hold hold = hold_of(a.cols);
    a.lanes = hold.lanes;
    const int64_t blocks = ceil_div(a.rows, 256 / hold.lanes);
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20))), block(256);
    if (hold.pieces == 0) hipLaunchKernelGGL((rms_norm_long_kernel<T, O>), grid, block, 0, st, a);
    else if (hold.lanes == 256) {
        if (hold.pieces == 4) hipLaunchKernelGGL((rms_norm_kernel<T, O, 4, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((rms_norm_kernel<T, O, 2, true>), grid, block, 0, st, a);
    } else if (hold.pieces == 4) hipLaunchKernelGGL((rms_norm_kernel<T, O, 4, false>), grid, block, 0, st, a);
    else if (hold.pieces == 3) hipLaunchKernelGGL((rms_norm_kernel<T, O, 3, false>), grid, block, 0, st, a);
    else if (hold.pieces == 2) hipLaunchKernelGGL((rms_norm_kernel<T, O, 2, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((rms_norm_kernel<T, O, 1, false>), grid, block, 0, st, a);
}
template <class T>
static void launch_norm(const NormArgs &a, int out_type, hipStream_t st)
{
    if (out_type == KGE_E4M3) launch_norm<T, e4m3_t>(a, st);
    else if (out_type == KGE_F32) launch_norm<T, float>(a, st);
    else if (out_type == KGE_BF16) launch_norm<T, bf16_t>(a, st);
    else launch_norm<T, half_t>(a, st);
}

// Ranges of rows that dweight is summed over.
struct Ranges {
    int64_t rows_each;
    int count;
};
static Ranges ranges_of(int64_t rows, int64_t cols)
{
    const Hold hold = hold_of(cols);
    const int64_t turn = hold.pieces ? 256 / hold.lanes : 8, turns = ceil_div(rows, turn);
    const int64_t across = hold.pieces ? 1 : ceil_div(cols, 2048), want = across < 1024 ? 1024 / across : 1;
    const int64_t each = turn * ceil_div(turns, want);
    return Ranges{each > 0 ? each : 1, (int)ceil_div(rows, each > 0 ? each : 1)};
}

template <class T, class D>
static void launch_grads(const NormGradArgs &args, const Ranges &ranges, void *dweight, hipStream_t st)
{
    NormGradArgs a = args;
    const Hold hold = hold_of(a.cols);
    a.lanes = hold.lanes;
    const dim3 grid((unsigned)ranges.count), block(256);
    if (hold.pieces == 0) {
        // (the sums first: dx may take the place of dy)
        if (a.sums) hipLaunchKernelGGL((rms_norm_long_sums_kernel<T, D>), dim3((unsigned)ceil_div(a.cols, 2048), (unsigned)ranges.count), block, 0, st, a);
        if (a.dx) hipLaunchKernelGGL((rms_norm_grad_long_kernel<T, D>), dim3((unsigned)(a.rows < (1 << 20) ? a.rows : (1 << 20))), block, 0, st, a);
    } else if (hold.lanes == 256) {
        if (hold.pieces == 4) hipLaunchKernelGGL((rms_norm_grad_kernel<T, D, 4, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((rms_norm_grad_kernel<T, D, 2, true>), grid, block, 0, st, a);
    } else if (hold.pieces == 4) hipLaunchKernelGGL((rms_norm_grad_kernel<T, D, 4, false>), grid, block, 0, st, a);
    else if (hold.pieces == 3) hipLaunchKernelGGL((rms_norm_grad_kernel<T, D, 3, false>), grid, block, 0, st, a);
    else if (hold.pieces == 2) hipLaunchKernelGGL((rms_norm_grad_kernel<T, D, 2, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((rms_norm_grad_kernel<T, D, 1, false>), grid, block, 0, st, a);
    if (a.sums) hipLaunchKernelGGL(norm_join_kernel<T>, dim3((unsigned)ceil_div(a.quads, 4)), block, 0, st, SumArgs{a.sums, ranges.count, a.cols, a.quads, dweight});
}
template <class T>
static void launch_grads(const NormGradArgs &a, const Ranges &ranges, int dy_type, void *dweight, hipStream_t st)
{
    if (dy_type == KGE_F32) launch_grads<T, float>(a, ranges, dweight, st);
    else if (dy_type == KGE_BF16) launch_grads<T, bf16_t>(a, ranges, dweight, st);
    else launch_grads<T, half_t>(a, ranges, dweight, st);
}

static int check(const kge_rms_norm *n)
{
    if (!n) return KGE_EINVAL;
    if (!known_type(n->type) || !(known_type(n->out_type) || n->out_type == KGE_E4M3) || !(n->eps >= 0.0) || n->eps > 1.7976931348623157e308) return KGE_EINVAL;
    const int64_t most = (int64_t)1 << 31;
    if (n->rows < 0 || n->cols < 0 || n->rows >= most || n->cols >= most) return KGE_ESHAPE;
    return KGE_OK;
}

}  // namespace kge

using namespace kge;

extern "C" {

int kge_rms_norm_fwd(const kge_rms_norm *norm, void *y, int64_t y_stride, const kge_rows8 *y8, void *h, int64_t h_stride, float *rstd,
                     void *stream)
{
    if (const int rc = check(norm)) return rc;
    if (norm->x_stride < norm->cols || (norm->residual && norm->residual_stride < norm->cols) || (h && h_stride < norm->cols)) return KGE_ESHAPE;
    const bool eight = norm->out_type == KGE_E4M3;
    if (eight) {
        if (const int rc = check_rows8(y8, norm->rows, norm->cols)) return rc;
    } else if (y_stride < norm->cols) {
        return KGE_ESHAPE;
    }
    if (norm->rows == 0 || norm->cols == 0) return KGE_OK;
    if (!norm->x || (!eight && !y)) return KGE_EINVAL;
    const NormArgs a{norm->x, norm->residual, norm->weight, norm->x_stride, norm->residual_stride, norm->rows, norm->cols, norm->eps,
                     y, y_stride, rows8_of(eight ? y8 : nullptr), h, h_stride, rstd, 0};
    hipStream_t st = as_stream(stream);
    KGE_CLEAR_LAUNCH_ERRORS();
    if (norm->type == KGE_F32) launch_norm<float>(a, norm->out_type, st);
    else if (norm->type == KGE_BF16) launch_norm<bf16_t>(a, norm->out_type, st);
    else launch_norm<half_t>(a, norm->out_type, st);
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

size_t kge_rms_norm_bwd_workspace(const kge_rms_norm *norm)
{
    if (check(norm) || norm->rows == 0 || norm->cols == 0) return 0;
    return (size_t)ranges_of(norm->rows, norm->cols).count * ceil_div(norm->cols, 4) * 16;
}

int kge_rms_norm_bwd(const kge_rms_norm *norm, const void *h, int64_t h_stride, const float *rstd, int32_t dy_type, const void *dy,
                     int64_t dy_stride, const void *dh, int64_t dh_stride, void *dx, int64_t dx_stride, void *dweight, void *workspace,
                     size_t workspace_bytes, void *stream)
{
    if (const int rc = check(norm)) return rc;
    if (!known_type(dy_type)) return KGE_EINVAL;
    if (h_stride < norm->cols || dy_stride < norm->cols || (dh && dh_stride < norm->cols) || (dx && dx_stride < norm->cols)) return KGE_ESHAPE;
    if (norm->cols == 0 || (!dx && !dweight)) return KGE_OK;
    if (norm->rows > 0 && (!h || !rstd || !dy)) return KGE_EINVAL;
    const size_t need = dweight ? kge_rms_norm_bwd_workspace(norm) : 0;
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KGE_EWORKSPACE;
    const Ranges ranges = norm->rows ? ranges_of(norm->rows, norm->cols) : Ranges{1, 0};
    const NormGradArgs a{h, dy, dh, norm->weight, h_stride, dy_stride, dh_stride, rstd, norm->rows, norm->cols, ceil_div(norm->cols, 4), ranges.rows_each,
                         dx, dx_stride, dweight ? static_cast<float *>(workspace) : nullptr, 0};
    hipStream_t st = as_stream(stream);
    KGE_CLEAR_LAUNCH_ERRORS();
    if (norm->rows == 0) {  // (dweight is an empty sum)
        if (dweight) {
            const SumArgs none{nullptr, 0, norm->cols, a.quads, dweight};
            const dim3 grid((unsigned)ceil_div(a.quads, 4)), block(256);
            if (norm->type == KGE_F32) hipLaunchKernelGGL(norm_join_kernel<float>, grid, block, 0, st, none);
            else if (norm->type == KGE_BF16) hipLaunchKernelGGL(norm_join_kernel<bf16_t>, grid, block, 0, st, none);
            else hipLaunchKernelGGL(norm_join_kernel<half_t>, grid, block, 0, st, none);
        }
    } else if (norm->type == KGE_F32) launch_grads<float>(a, ranges, dy_type, dweight, st);
    else if (norm->type == KGE_BF16) launch_grads<bf16_t>(a, ranges, dy_type, dweight, st);
    else launch_grads<half_t>(a, ranges, dy_type, dweight, st);
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

}  // extern "C"
