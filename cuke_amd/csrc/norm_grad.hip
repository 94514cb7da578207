// Gradients of the root-mean-square norm (kge_rms_norm_bwd).  With n = h r and g = dy weight:
//   dx = r (g - n mean(g n)) + dh,   dweight = sum over rows of dy n
#include <type_traits>

#include "linear_tile.hpp"
#include "norm.hpp"

namespace kge {

struct NormGradArgs {
    const void *h, *dy, *dh, *weight;
    int64_t h_stride, dy_stride, dh_stride;
    const float *rstd;
    const uint32_t *rest;  // or NULL
    int64_t rows, cols, quads, rows_each;
    void *dx;     // or NULL
    int64_t dx_stride;
    float *sums;  // [ranges][4 quads]: dweight's over a range of rows, or NULL
    int lanes;
    double eps;
};

// Eight elements as they lie in memory, requested ahead of their use.  A row's last piece is moved back to end with the row (rows of at least eight columns), so that
// no load needs a branch; the first `skip` elements belong to the piece before it too.
template <class E>
struct Held {
    typename Pack<E, 8>::type v;
    __device__ __forceinline__ void fetch(const void *row, int at) { v = Pack<E, 8>::load(static_cast<const E *>(row) + at).v; }
    __device__ __forceinline__ void values(float (&f)[8]) const
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
    }
};

// A workgroup takes a range of rows, each held by `lanes` lanes (WAVES: by two or four waves); what the next row needs is requested while the present one is worked on.  A lane's
// columns are the same in all rows, so dweight's sums wait in registers until the range's end.
// 65536 x 2048 bf16 with dh and rest (1.14 GB) 226 us, without 161 (0.81 GB): 5.0 TB/s, what a large copy reaches, but not the forward pass's 6.2; more or fewer ranges, two rows
// requested ahead and dx alone (220) change little.  4096 x 1024 (36 MB, in the caches) 8, and 2.4 for the joining of dweight's sums.
template <class T, class D, int C, bool WAVES, bool DH, bool REST>
__global__ __launch_bounds__(256) void rms_norm_grad_kernel(NormGradArgs a)
{
    __shared__ float part[2][4];
    int turn = 0;
    __shared__ float s_sum[256][8];
    int lane;
    uint32_t group;
    place_in_rows<WAVES>(a.lanes, &lane, &group);
    const int lanes = a.lanes, groups = 256 >> (31 - __builtin_clz(lanes));
    const int64_t first = (int64_t)blockIdx.x * a.rows_each, last = first + a.rows_each < a.rows ? first + a.rows_each : a.rows;
    const float share = 1.0f / (float)a.cols;
    const int cols = (int)a.cols;
    int at[C], skip[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int col = 8 * (c * lanes + lane);
        at[c] = col < cols - 8 ? col : cols - 8, skip[c] = col - at[c];
    }
    float sum[C][8] = {};
    Held<T> h[C], dh[DH ? C : 1], w[C];
    Held<D> dy[C];
    uint32_t rest[REST ? C : 1], rest_end[REST ? C : 1];
    float r;
    const int words = (cols + 7) / 8;
    if (a.weight) {
#pragma unroll
        for (int c = 0; c < C; ++c) w[c].fetch(a.weight, at[c]);
    }
    // the lane's present row, and the one requested ahead (behind the range's end: a row that is there)
    const int64_t mine = first + (first + group < last ? group : 0u);
    const T *row_h = static_cast<const T *>(a.h) + mine * a.h_stride, *row_dh = static_cast<const T *>(a.dh) + (DH ? mine * a.dh_stride : 0);
    const D *row_dy = static_cast<const D *>(a.dy) + mine * a.dy_stride;
    const uint32_t *row_rest = a.rest + (REST ? mine * words : 0);
    const float *row_r = a.rstd + mine;
    T *row_dx = static_cast<T *>(a.dx) + mine * a.dx_stride;
    const int64_t step_h = groups * a.h_stride, step_dy = groups * a.dy_stride, step_dh = groups * a.dh_stride, step_dx = groups * a.dx_stride;
    auto fetch = [&] {
        r = *row_r;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            h[c].fetch(row_h, at[c]);
            dy[c].fetch(row_dy, at[c]);
            if constexpr (DH) dh[c].fetch(row_dh, at[c]);
            if constexpr (REST)  // (a piece that was moved back begins inside a word)
                rest[c] = row_rest[at[c] >> 3], rest_end[c] = row_rest[(at[c] + 7) >> 3];
        }
    };
    fetch();
    for (int64_t row0 = first; row0 < last; row0 += groups) {
        const int64_t row = row0 + group;
        const bool there = row < last;
        float n[C][8], g[C][8], dot = 0.0f;
        const float kept = r, rr = fabsf(kept);
        Held<T> more[DH ? C : 1];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            h[c].values(n[c]), dy[c].values(g[c]);
            if constexpr (REST) add_rest<T>(n[c], __builtin_amdgcn_alignbit(rest_end[c], rest[c], 4 * (at[c] & 7)));
            to_reach(kept, n[c]);
            if constexpr (DH) more[c] = dh[c];
            if (skip[c] > 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < skip[c]) g[c][e] = 0.0f;  // (counted by the piece before)
            }
        }
        if (row + groups < last) {
            row_r += groups, row_h += step_h, row_dy += step_dy;
            if constexpr (DH) row_dh += step_dh;
            if constexpr (REST) row_rest += groups * words;
        }
        fetch();
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                n[c][e] *= rr;
                if (there) sum[c][e] = fmaf(g[c][e], n[c][e], sum[c][e]);
            }
            if (a.weight) {
                float v[8];
                w[c].values(v);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[c][e] *= v[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) dot = fmaf(g[c][e], n[c][e], dot);
        }
        if (!a.dx) continue;
        const float mean = (WAVES ? waves_sum(dot, lanes, part, turn++) : lanes_sum(dot, lanes)) * share;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float d[8] = {};
            if constexpr (DH) more[c].values(d);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[c][e] -= n[c][e] * mean;
            to_reach(kept, g[c]);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = fmaf(rr, g[c][e], d[e]);
            if (!there || skip[c] >= 8) continue;
            T *to = row_dx + at[c];
            if (skip[c] == 0) {
                store8(to, d, 8);
            } else {
#pragma unroll
                for (int e = 1; e < 8; ++e)
                    if (e >= skip[c]) to[e] = (T)d[e];
            }
        }
        row_dx += step_dx;
    }
    if (!a.sums) return;
    float *to = a.sums + (int64_t)blockIdx.x * a.quads * 4;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (groups > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) s_sum[threadIdx.x][e] = sum[c][e];
            __syncthreads();
            if (group) continue;
            for (int k = 1; k < groups; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[c][e] += s_sum[k * lanes + lane][e];
        }
        if (skip[c] == 0) {
            Pack<float, 4> lo, hi;
            lo.v[0] = sum[c][0], lo.v[1] = sum[c][1], lo.v[2] = sum[c][2], lo.v[3] = sum[c][3];
            hi.v[0] = sum[c][4], hi.v[1] = sum[c][5], hi.v[2] = sum[c][6], hi.v[3] = sum[c][7];
            lo.store(to + at[c]), hi.store(to + at[c] + 4);
        } else {
#pragma unroll
            for (int e = 1; e < 8; ++e)
                if (e >= skip[c]) to[at[c] + e] = sum[c][e];
        }
    }
}

// Rows of one to seven columns: a thread a row, dweight's sums in registers until the range's end.  Of one column g - n mean(g n) = g (1 - n^2) = g eps r^2: the difference of two
// nearly equal numbers (eps 1e-6: one or two of fp32's digits are left), the product of what is known.  Bound by launches: 65536 bf16 rows of 1, 4
// and 7 columns 8.3, 8.4 and 8.5 us with the joining of the sums (61, 202 and 294 with a workgroup a row, as the longest rows have).
template <class T, class D>
__global__ __launch_bounds__(256) void rms_norm_grad_few_kernel(NormGradArgs a)
{
    __shared__ float part[4][8];
    const int64_t first = (int64_t)blockIdx.x * a.rows_each, last = first + a.rows_each < a.rows ? first + a.rows_each : a.rows;
    const int cols = (int)a.cols;
    const float share = 1.0f / (float)cols;
    float w[8], sum[8] = {};
    if (a.weight) load8(static_cast<const T *>(a.weight), cols, w);
    for (int64_t row = first + threadIdx.x; row < last; row += 256) {
        const float kept = a.rstd[row], r = fabsf(kept);
        float n[8], g[8], d[8] = {};
        load8(static_cast<const T *>(a.h) + row * a.h_stride, cols, n);
        load8(static_cast<const D *>(a.dy) + row * a.dy_stride, cols, g);
        if (a.dh) load8(static_cast<const T *>(a.dh) + row * a.dh_stride, cols, d);
        if constexpr (sizeof(T) == 2)
            if (a.rest) add_rest<T>(n, a.rest[row]);
        to_reach(kept, n);
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            n[e] *= r;
            sum[e] = fmaf(g[e], n[e], sum[e]);
            if (a.weight) g[e] *= w[e];
            dot = fmaf(g[e], n[e], dot);
        }
        if (!a.dx) continue;
        if (cols == 1) {
            const double whole = kept < 0.0f ? r * 0x1p64 : r;
            d[0] = (float)(a.eps * whole * whole * whole * g[0] + 0.0 * n[0] + d[0]);  // (of what is not finite NaN, as the difference would be)
        } else {
            const float mean = dot * share;
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] -= n[e] * mean;
            to_reach(kept, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = fmaf(r, g[e], d[e]);
        }
        store8(static_cast<T *>(a.dx) + row * a.dx_stride, d, cols);
    }
    if (!a.sums) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float all = lanes_sum(sum[e], 64);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6][e] = all;
    }
    __syncthreads();
    const int e = threadIdx.x;
    if (e < 4 * (int)a.quads) a.sums[(int64_t)blockIdx.x * a.quads * 4 + e] = (part[0][e] + part[1][e]) + (part[2][e] + part[3][e]);
}

// Rows that registers do not hold: dx by a workgroup that goes over a row twice.
template <class T, class D>
__global__ __launch_bounds__(256) void rms_norm_grad_long_kernel(NormGradArgs a)
{
    __shared__ float part[2][4];
    int turn = 0;
    auto load = [&](int64_t row, int64_t col, float kept, float(&n)[8], float(&g)[8]) {
        const int64_t left = a.cols - col;
        const int valid = (int)(left < 8 ? left : 8);
        load8(static_cast<const T *>(a.h) + row * a.h_stride + col, valid, n);
        load8(static_cast<const D *>(a.dy) + row * a.dy_stride + col, valid, g);
        if constexpr (sizeof(T) == 2)
            if (a.rest) add_rest<T>(n, a.rest[row * ((a.cols + 7) / 8) + col / 8]);
        to_reach(kept, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) n[e] *= fabsf(kept);
        if (!a.weight) return valid;
        float w[8];
        load8(static_cast<const T *>(a.weight) + col, valid, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] *= w[e];
        return valid;
    };
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float kept = a.rstd[row];
        float dot = 0.0f;
        for (int64_t col = 8 * threadIdx.x; col < a.cols; col += 8 * 256) {
            float n[8], g[8];
            load(row, col, kept, n, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) dot = fmaf(g[e], n[e], dot);
        }
        const float mean = waves_sum(dot, 256, part, turn++) * (1.0f / (float)a.cols);
        for (int64_t col = 8 * threadIdx.x; col < a.cols; col += 8 * 256) {
            float n[8], g[8], d[8] = {};
            const int valid = load(row, col, kept, n, g);
            if (a.dh) load8(static_cast<const T *>(a.dh) + row * a.dh_stride + col, valid, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] -= n[e] * mean;
            to_reach(kept, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = fmaf(fabsf(kept), g[e], d[e]);
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
        const float kept = a.rstd[row];
        float n[8], g[8];
        load8(static_cast<const T *>(a.h) + row * a.h_stride + col, valid, n);
        load8(static_cast<const D *>(a.dy) + row * a.dy_stride + col, valid, g);
        if constexpr (sizeof(T) == 2)
            if (a.rest) add_rest<T>(n, a.rest[row * ((a.cols + 7) / 8) + col / 8]);
        to_reach(kept, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = fmaf(g[e], n[e] * fabsf(kept), sum[e]);
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
static Hold grad_hold(int64_t rows, int64_t cols)
{
    return cols < 8 ? Hold{0, 1} : hold_of(rows, cols, 4096);  // (rms_norm_grad_few_kernel)
}

// Ranges of rows, one a workgroup, that dweight is summed over: 512 of them (us with 256, 512, 1024 and 2048: 65536 x 2048 bf16 with dh and rest 220, 226, 228, 235, without
// 158, 161, 172, 171; 4096 x 1024 11.8, 12.1, 15.0, 15.0; 30000 x 300 22.3, 20.9, 23.4, 27.9).
struct Ranges {
    int64_t rows_each;
    int count;
};
static Ranges ranges_of(int64_t rows, int64_t cols)
{
    const Hold hold = grad_hold(rows, cols);
    const int64_t turn = hold.pieces || hold.lanes == 1 ? 256 / hold.lanes : 8, turns = ceil_div(rows, turn);
    const int64_t across = hold.pieces || hold.lanes == 1 ? 1 : ceil_div(cols, 2048), most = 512, want = across < most ? most / across : 1;
    const int64_t each = turn * ceil_div(turns, want);
    return Ranges{each > 0 ? each : 1, (int)ceil_div(rows, each > 0 ? each : 1)};
}

template <class T, class D>
static void launch_grads(const NormGradArgs &args, const Ranges &ranges, void *dweight, hipStream_t st)
{
    NormGradArgs a = args;
    const Hold hold = grad_hold(a.rows, a.cols);
    a.lanes = hold.lanes;
    const dim3 grid((unsigned)ranges.count), block(256);
    if (hold.lanes == 1) {
        hipLaunchKernelGGL((rms_norm_grad_few_kernel<T, D>), grid, block, 0, st, a);
    } else if (hold.pieces == 0) {
        // (the sums first: dx may take the place of dy)
        if (a.sums) hipLaunchKernelGGL((rms_norm_long_sums_kernel<T, D>), dim3((unsigned)ceil_div(a.cols, 2048), (unsigned)ranges.count), block, 0, st, a);
        if (a.dx) hipLaunchKernelGGL((rms_norm_grad_long_kernel<T, D>), dim3((unsigned)(a.rows < (1 << 20) ? a.rows : (1 << 20))), block, 0, st, a);
    } else {
        with_hold(hold, [&](auto pieces, auto waves) {
            constexpr int kPieces = decltype(pieces)::value;
            constexpr bool kWaves = decltype(waves)::value;
            if constexpr (sizeof(T) == 2) {
                if (a.rest && a.dh) hipLaunchKernelGGL((rms_norm_grad_kernel<T, D, kPieces, kWaves, true, true>), grid, block, 0, st, a);
                else if (a.rest) hipLaunchKernelGGL((rms_norm_grad_kernel<T, D, kPieces, kWaves, false, true>), grid, block, 0, st, a);
                if (a.rest) return;
            }
            if (a.dh) hipLaunchKernelGGL((rms_norm_grad_kernel<T, D, kPieces, kWaves, true, false>), grid, block, 0, st, a);
            else hipLaunchKernelGGL((rms_norm_grad_kernel<T, D, kPieces, kWaves, false, false>), grid, block, 0, st, a);
        });
    }
    if (a.sums) hipLaunchKernelGGL(norm_join_kernel<T>, dim3((unsigned)ceil_div(a.quads, 4)), block, 0, st, SumArgs{a.sums, ranges.count, a.cols, a.quads, dweight});
}
template <class T>
static void launch_grads(const NormGradArgs &a, const Ranges &ranges, int dy_type, void *dweight, hipStream_t st)
{
    if (dy_type == KGE_F32) launch_grads<T, float>(a, ranges, dweight, st);
    else if (dy_type == KGE_BF16) launch_grads<T, bf16_t>(a, ranges, dweight, st);
    else launch_grads<T, half_t>(a, ranges, dweight, st);
}

}  // namespace kge

using namespace kge;

extern "C" {

size_t kge_rms_norm_bwd_workspace(const kge_rms_norm *norm)
{
    if (check_norm(norm) || norm->rows == 0 || norm->cols == 0) return 0;
    return (size_t)ranges_of(norm->rows, norm->cols).count * ceil_div(norm->cols, 4) * 16;
}

int kge_rms_norm_bwd(const kge_rms_norm *norm, const void *h, int64_t h_stride, const float *rstd, const void *rest, int32_t dy_type, const void *dy,
                     int64_t dy_stride, const void *dh, int64_t dh_stride, void *dx, int64_t dx_stride, void *dweight, void *workspace,
                     size_t workspace_bytes, void *stream)
{
    if (const int rc = check_norm(norm)) return rc;
    if (!known_type(dy_type)) return KGE_EINVAL;
    if (h_stride < norm->cols || dy_stride < norm->cols || (dh && dh_stride < norm->cols) || (dx && dx_stride < norm->cols)) return KGE_ESHAPE;
    if (norm->cols == 0 || (!dx && !dweight)) return KGE_OK;
    if (norm->rows > 0 && (!h || !rstd || !dy || reinterpret_cast<uintptr_t>(rest) % 4 != 0)) return KGE_EINVAL;
    const size_t need = dweight ? kge_rms_norm_bwd_workspace(norm) : 0;
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KGE_EWORKSPACE;
    const Ranges ranges = norm->rows ? ranges_of(norm->rows, norm->cols) : Ranges{1, 0};
    const NormGradArgs a{h, dy, dh, norm->weight, h_stride, dy_stride, dh_stride, rstd, static_cast<const uint32_t *>(rest), norm->rows, norm->cols, ceil_div(norm->cols, 4), ranges.rows_each,
                         dx, dx_stride, dweight ? static_cast<float *>(workspace) : nullptr, 0, norm->eps};
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
