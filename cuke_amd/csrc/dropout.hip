// Dropout with a mask that is never stored: forward and gradient are the same pass (kge_dropout).
#include "features.hpp"

namespace kge {

// Four elements a thread, one word of the sequence for them.  Bound by memory, x read and y written once; the word's two 64-bit products hide
// behind that: 65536 x 1000 bf16 (262 MB) 53 us, 4.9 TB/s.
template <class T>
__global__ __launch_bounds__(256) void dropout_kernel(const T *x, int64_t x_stride, T *y, int64_t y_stride, int64_t rows, int64_t cols, Drop drop)
{
    const uint64_t base = drop.base();
    const int64_t total = rows * drop.quads;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / drop.quads, quad = i % drop.quads, col = 4 * quad, left = cols - col;
        const int valid = (int)(left < 4 ? left : 4);
        const float4 q = load4(x + row * x_stride + col, valid);
        float v[4] = {q.x, q.y, q.z, q.w};
        if (drop.cut) drop.apply(v, drop.word(base, drop.place(row, quad)));
        store4(y + row * y_stride + col, make_float4(v[0], v[1], v[2], v[3]), valid);
    }
}

template <class T>
static int launch(const void *x, int64_t x_stride, void *y, int64_t y_stride, int64_t rows, int64_t cols, const Drop &d, hipStream_t st)
{
    const int64_t blocks = ceil_div(rows * d.quads, 256);
    KGE_CLEAR_LAUNCH_ERRORS();
    hipLaunchKernelGGL(dropout_kernel<T>, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, static_cast<const T *>(x), x_stride,
                       static_cast<T *>(y), y_stride, rows, cols, d);
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

}  // namespace kge

using namespace kge;

extern "C" int kge_dropout(int32_t type, const void *x, int64_t x_stride, void *y, int64_t y_stride, int64_t rows, int64_t cols, double p,
                           uint64_t seed, uint64_t step, const uint64_t *step_dev, void *stream)
{
    if (!known_type(type) || !drop_ok(p)) return KGE_EINVAL;
    if (rows < 0 || cols < 0 || x_stride < cols || y_stride < cols) return KGE_ESHAPE;
    if (rows == 0 || cols == 0) return KGE_OK;
    if (!x || !y) return KGE_EINVAL;
    const Drop d = make_drop(p, seed, step, step_dev, cols);
    hipStream_t st = as_stream(stream);
    if (type == KGE_F32) return launch<float>(x, x_stride, y, y_stride, rows, cols, d, st);
    if (type == KGE_BF16) return launch<bf16_t>(x, x_stride, y, y_stride, rows, cols, d, st);
    return launch<half_t>(x, x_stride, y, y_stride, rows, cols, d, st);
}
