// Rows packed to 8 bits and back (kge_pack8, kge_unpack8).
#include "rows8.hpp"

namespace kge {

struct Places {
    int64_t rows, cols;
    uint32_t each;    // pieces of a row
    int64_t total;
};
__device__ __forceinline__ void place_of(const Places &p, int64_t i, int64_t *row, int64_t *piece)
{
    if (p.total <= 0xFFFFFFFFll) {
        const uint32_t r = (uint32_t)i / p.each;
        *row = r, *piece = (uint32_t)i - r * p.each;
    } else {
        *row = i / p.each, *piece = i - *row * p.each;
    }
}

// Sixteen lanes take 128 columns of a row, eight each: four blocks, whose scales are stored as one word.  One pass, a block's largest value by two exchanges within a quad.
// Bound by memory: 65536 x 1000 bf16 (200 MB) 34 us where the caches have it, 46 where they do not.
template <class T>
__global__ __launch_bounds__(256) void pack8_kernel(const T *x, int64_t x_stride, Rows8 out, Places p)
{
    const int64_t width = (p.cols + 31) / 32 * 32;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.total; i += (int64_t)gridDim.x * 256) {  // (sixteen lanes stay together)
        int64_t row, piece;
        place_of(p, i, &row, &piece);
        const int64_t col = 8 * piece, left = p.cols - col;
        float v[8];
        load8(x + row * x_stride + col, (int)(left < 8 ? left : 8), v);
        const int byte = scale_byte(quad_max(top_of(v)));
        const float inverse = scale_inverse(byte);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= inverse;
        const int lane = threadIdx.x & 15;
        int word = (col & ~31) < p.cols ? byte << (8 * (lane >> 2)) : 0;
        word |= dpp<0x124>(word);  // (rotated by 4, and by 8)
        word |= dpp<0x128>(word);
        if (col < width) *reinterpret_cast<uint2 *>(out.q + row * out.q_stride + col) = to_e4m3(v);
        if (lane == 0) *reinterpret_cast<int *>(out.scale + row * out.scale_stride + col / 32) = word;
    }
}

// Eight columns a thread.  65536 x 1000 to bf16 (200 MB): 30 us.
template <class T>
__global__ __launch_bounds__(256) void unpack8_kernel(Rows8 in, T *y, int64_t y_stride, Places p)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.total; i += (int64_t)gridDim.x * 256) {
        int64_t row, piece;
        place_of(p, i, &row, &piece);
        const int64_t col = 8 * piece, left = p.cols - col;
        float v[8];
        from_e4m3(*reinterpret_cast<const uint2 *>(in.q + row * in.q_stride + col), scale_value(in.scale[row * in.scale_stride + col / 32]), v);
        store8(y + row * y_stride + col, v, (int)(left < 8 ? left : 8));
    }
}

static unsigned grid_for(int64_t items)
{
    const int64_t b = ceil_div(items, 256);
    return (unsigned)(b < 16384 ? b : 16384);
}

template <class T>
static int pack(const void *x, int64_t x_stride, int64_t rows, int64_t cols, const kge_rows8 *out, hipStream_t st)
{
    const int64_t each = 16 * ceil_div(cols, 128);
    const Places p{rows, cols, (uint32_t)each, rows * each};
    KGE_CLEAR_LAUNCH_ERRORS();
    hipLaunchKernelGGL(pack8_kernel<T>, dim3(grid_for(p.total)), dim3(256), 0, st, static_cast<const T *>(x), x_stride, rows8_of(out), p);
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}
void launch_unpack8(int type, const Rows8 &in, int64_t rows, int64_t cols, void *y, int64_t y_stride, hipStream_t st)
{
    const int64_t each = ceil_div(cols, 8);
    const Places p{rows, cols, (uint32_t)each, rows * each};
    const dim3 grid(grid_for(p.total)), block(256);
    if (type == KGE_F32) hipLaunchKernelGGL(unpack8_kernel<float>, grid, block, 0, st, in, static_cast<float *>(y), y_stride, p);
    else if (type == KGE_BF16) hipLaunchKernelGGL(unpack8_kernel<bf16_t>, grid, block, 0, st, in, static_cast<bf16_t *>(y), y_stride, p);
    else hipLaunchKernelGGL(unpack8_kernel<half_t>, grid, block, 0, st, in, static_cast<half_t *>(y), y_stride, p);
}

static bool too_large(int64_t rows, int64_t cols) { return rows < 0 || cols < 0 || rows >= (int64_t)1 << 31 || cols >= (int64_t)1 << 31; }

}  // namespace kge

using namespace kge;

extern "C" {

int kge_pack8(int32_t type, const void *x, int64_t x_stride, int64_t rows, int64_t cols, const kge_rows8 *out, void *stream)
{
    if (!known_type(type)) return KGE_EINVAL;
    if (too_large(rows, cols) || x_stride < cols) return KGE_ESHAPE;
    if (const int rc = check_rows8(out, rows, cols)) return rc;
    if (rows == 0 || cols == 0) return KGE_OK;
    if (!x) return KGE_EINVAL;
    hipStream_t st = as_stream(stream);
    if (type == KGE_F32) return pack<float>(x, x_stride, rows, cols, out, st);
    if (type == KGE_BF16) return pack<bf16_t>(x, x_stride, rows, cols, out, st);
    return pack<half_t>(x, x_stride, rows, cols, out, st);
}

int kge_unpack8(const kge_rows8 *rows8, int64_t rows, int64_t cols, int32_t type, void *y, int64_t y_stride, void *stream)
{
    if (!known_type(type)) return KGE_EINVAL;
    if (too_large(rows, cols) || y_stride < cols) return KGE_ESHAPE;
    if (const int rc = check_rows8(rows8, rows, cols)) return rc;
    if (rows == 0 || cols == 0) return KGE_OK;
    if (!y) return KGE_EINVAL;
    KGE_CLEAR_LAUNCH_ERRORS();
    launch_unpack8(type, rows8_of(rows8), rows, cols, y, y_stride, as_stream(stream));
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

}  // extern "C"
