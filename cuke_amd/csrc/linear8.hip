// Linear layers on rows in 8 bits: y = drop(act(x8 W^T + b)) + residual with a 16-bit weight or one in 8 bits too, and the gradients (kge_linear8_fwd,
// kge_linear8_bwd).
#include "linear_plan.hpp"

namespace kge {

// ---- few rows --------------------------------------------------------------------------------------
// As linear_few_kernel, with rows in 8 bits (and the weight too: W8) widened on their way to the matrix cores.  A wave takes every eighth group of four blocks, a quarter of
// its lanes a block each: 32 numbers in two loads and one scale.  (A step multiplies eight terms of each of the four: which terms meet in it does not matter.)  Bound by a launch and two dependent
// loads: 1 x 1024 -> 512 with both sides in 8 bits 3.3 us, 1 x 4096 -> 2048 6.0.
template <class T>
struct Line8 {
    const uint8_t *q, *scale;  // of the lane's block in the first group
    struct Group {
        uint4 lo, hi;
        int byte;
        __device__ __forceinline__ typename Few<T>::piece widened(int step) const
        {
            const uint4 v = step < 2 ? lo : hi;
            return widen(step & 1 ? make_uint2(v.z, v.w) : make_uint2(v.x, v.y), __int_as_float(byte << 23), T{});
        }
    };
    __device__ __forceinline__ Line8(const Rows8 &s, int64_t row, int quarter) : q(s.q + row * s.q_stride + 32 * quarter), scale(s.scale + row * s.scale_stride + quarter) {}
    __device__ __forceinline__ Group load(int64_t group) const
    {
        const uint4 *p = reinterpret_cast<const uint4 *>(q + 128 * group);
        return Group{p[0], p[1], scale[4 * group]};
    }
};
// 32 terms of a 16-bit weight's row
template <class T>
struct Line16 {
    typedef typename Few<T>::piece piece;
    const T *p;
    struct Group {
        piece v[4];
        __device__ __forceinline__ piece widened(int step) const { return v[step]; }
    };
    __device__ __forceinline__ Line16(const Side &s, int64_t row, int quarter) : p(static_cast<const T *>(s.p) + row * s.stride + 32 * quarter) {}
    __device__ __forceinline__ Group load(int64_t group) const
    {
        Group g;
#pragma unroll
        for (int u = 0; u < 4; ++u) g.v[u] = Few<T>::load(p + 128 * group + 8 * u);
        return g;
    }
    __device__ __forceinline__ Group load(int64_t group, int64_t left) const  // `left` terms of the 32 exist
    {
        Group g;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t rest = left - 8 * u;
            g.v[u] = Few<T>::load(p + 128 * group + 8 * u, rest < 0 ? 0 : (int)(rest < 8 ? rest : 8));
        }
        return g;
    }
};

template <class T, int MF, bool W8>
__global__ __launch_bounds__(kFewWaves *kWave) void linear8_few_kernel(TileArgs t)
{
    using F = Few<T>;
    using Rows = Line8<T>;
    using Weight = typename std::conditional<W8, Line8<T>, Line16<T>>::type;
    static_assert(F::kTerms == 32 && F::kEach == 8, "a step");
    constexpr int kAhead = 2;  // groups whose loads are in flight together
    __shared__ f4 sums[kFewWaves][MF][kWave];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), r = lane & 15, quarter = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16 * MF;
    const int64_t n = n0 + r < t.a.extent ? n0 + r : t.a.extent - 1;  // (rows that do not exist: others, whose sums nobody asks for)
    auto weight = [&] {
        if constexpr (W8) return Weight(t.a8, n, quarter);
        else return Weight(t.a, n, quarter);
    };
    const Weight a = weight();
    auto row = [&](int j) { return m0 + 16 * j + r < t.b.extent ? m0 + 16 * j + r : t.b.extent - 1; };
    const Rows first(t.b8, row(0), quarter), second(t.b8, row(MF - 1), quarter);
    f4 acc[MF] = {};
    const int64_t blocks = (t.k + 31) / 32, full = t.k / 128;  // full: groups all of whose terms exist
    auto multiply = [&](const typename Weight::Group &x, const typename Rows::Group (&y)[MF]) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const typename F::piece p = x.widened(u);
#pragma unroll
            for (int j = 0; j < MF; ++j) acc[j] = F::multiply(p, y[j].widened(u), acc[j]);
        }
    };
    int64_t g = wave;
    for (; g + (kAhead - 1) * kFewWaves < full; g += kAhead * kFewWaves) {
        typename Weight::Group x[kAhead];
        typename Rows::Group y[kAhead][MF];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            x[k] = a.load(g + k * kFewWaves);
#pragma unroll
            for (int j = 0; j < MF; ++j) y[k][j] = (j ? second : first).load(g + k * kFewWaves);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) multiply(x[k], y[k]);
    }
    for (; 4 * g < blocks; g += kFewWaves) {  // (numbers behind a row's end are zero, to the end of its last block; a 16-bit weight's row ends where it ends)
        typename Weight::Group x{};
        typename Rows::Group y[MF]{};
        if (4 * g + quarter < blocks) {
            if constexpr (W8) x = a.load(g);
            else if (g < full) x = a.load(g);
            else x = a.load(g, t.k - 128 * g - 32 * quarter);
#pragma unroll
            for (int j = 0; j < MF; ++j) y[j] = (j ? second : first).load(g);
        }
        multiply(x, y);
    }
#pragma unroll
    for (int j = 0; j < MF; ++j) sums[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave >= MF) return;
    // wave j finishes rows 16 j ..: lane l holds columns 4 (l / 16) .. + 3 of row l % 16
    f4 z = sums[0][wave][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) z += sums[w][wave][lane];
    const int64_t m = m0 + 16 * wave + r, col = n0 + 4 * (lane >> 4), left = t.e.cols - col;
    if (m >= t.e.rows || left <= 0) return;
    const int valid = (int)(left < 4 ? left : 4);
    float4 bias = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (t.e.bias) bias = load4(static_cast<const T *>(t.e.bias) + col, valid);
    float out[1][4] = {{z[0], z[1], z[2], z[3]}};
    finish_quads<T, 1, W8 ? 0 : 8>(t.e, t.e.drop.base(), m, 1, col, valid, out, bias, nullptr);
}

template <class T>
static void launch_few8(int few, bool w8, const TileArgs &t, hipStream_t st)
{
    const dim3 grid((unsigned)ceil_div(t.a.extent, 16), (unsigned)ceil_div(t.b.extent, 16 * few)), block(kFewWaves * kWave);
    if (few == 1 && w8) hipLaunchKernelGGL((linear8_few_kernel<T, 1, true>), grid, block, 0, st, t);
    else if (few == 1) hipLaunchKernelGGL((linear8_few_kernel<T, 1, false>), grid, block, 0, st, t);
    else if (w8) hipLaunchKernelGGL((linear8_few_kernel<T, 2, true>), grid, block, 0, st, t);
    else hipLaunchKernelGGL((linear8_few_kernel<T, 2, false>), grid, block, 0, st, t);
}

// ---- forward pass ----------------------------------------------------------------------------------
// The shapes of linear_plan.hpp with the stages that rows in 8 bits leave room for; those that are other ones where both sides are in 8 bits (a stage's terms are
// then twice as many, and its rows of 128 bytes are whole lines: with 64 terms and four stages, half lines, the largest shape took 349 us for 16384 x 4096 -> 4096 in place of 272).
using LargeB = Shape<256, 256, 64, 2, 4, 3>;
using MiddleB = Shape<128, 128, 64, 2, 4, 3>;
using TallB = Shape<64, 128, 64, 2, 2, 3>;
using LoneB = Shape<64, 128, 64, 2, 4, 4>;
using SmallB = Shape<64, 64, 64, 2, 2, 3>;
using Large8 = Shape<256, 256, 64, 2, 4, 2>;
using Middle8 = Shape<128, 128, 64, 2, 4, 2>;
using Tall8 = Shape<64, 128, 64, 2, 2, 2>;

// Waves a SIMD that the registers have to leave room for: a workgroup of eight whose LDS lets two of them share a CU holds itself to 128 registers (65536 x 512 -> 400:
// 78 us with 136).
template <class S, Eight E>
constexpr int waves_for() { return S::kThreads == 512 && 2 * (S::STAGES * stage_bytes8<S, E>() + (E == kBothSides && grouped_scales<S>() ? 32 * (S::XA + S::XB) : 0)) <= 160 << 10 ? 4 : 1; }

// The weight in 16 bits, rows widened as they leave LDS.  32768 x 2048 -> 2048 bf16: plain 262 us (1.05 PFLOP/s; rows of 16 bits 277), with gelu, drop and act' kept 320 (336).
template <class T, class S>
__global__ __launch_bounds__(S::kThreads, (waves_for<S, kSideB>())) void linear8_forward_kernel(TileArgs t)
{
    constexpr int kStage = stage_bytes8<S, kSideB>();
    __shared__ __align__(16) char stage0[kStage], stage1[kStage], stage2[S::STAGES > 2 ? kStage : 16], stage3[S::STAGES > 3 ? kStage : 16];
    compute_tile<T, false, false, S, true, true, kSideB>(t, blockIdx.x, gridDim.x, stage0, stage1, stage2, stage3);
}
// The matrix cores' own product of 8-bit sides, at twice the pace of the 16-bit one.  It sums eight neighbouring terms at a time and drops of each what lies
// below 2^-13 of the largest one's power (and adds such sums in fp32): of a result some 2^-13, next to nothing beside its rounding to bf16 (2^-9), and of one
// that is small because its terms cancel 2^-13 of the largest of them, which is more of it; too much for fp16 and fp32, which are made of widened numbers.
// 8192 x 8192 x 8192 490 us (2.24 PFLOP/s; 32768 x 2048 -> 2048 160), the matrix cores busy for 59 % of it at the 1.8 GHz that the card's power leaves them;
// 512 us in four waves of 128 x 128 that read LDS a step ahead of the products.
template <class T, class S>
__global__ __launch_bounds__(S::kThreads, (waves_for<S, kBothSides>())) void linear8_answer_kernel(TileArgs t)
{
    constexpr int kStage = stage_bytes8<S, kBothSides>();
    __shared__ __align__(16) char stage0[kStage], stage1[kStage], stage2[S::STAGES > 2 ? kStage : 16], stage3[S::STAGES > 3 ? kStage : 16];
    __shared__ __align__(16) char scales[grouped_scales<S>() ? 32 * (S::XA + S::XB) : 16];
    compute_tile<T, false, false, S, true, true, kBothSides>(t, blockIdx.x, gridDim.x, stage0, stage1, stage2, stage3, scales);
}

template <class T, class S, bool BOTH>
static void launch_tiles(TileArgs &t, hipStream_t st)
{
    t.tiles_a = (int)ceil_div(t.a.extent, S::XA), t.tiles_b = (int)ceil_div(t.b.extent, S::XB);
    const int64_t blocks = (int64_t)t.tiles_a * t.tiles_b;
    if (!blocks) return;
    if constexpr (BOTH && std::is_same<T, bf16_t>::value) hipLaunchKernelGGL((linear8_answer_kernel<T, S>), dim3((unsigned)blocks), dim3(S::kThreads), 0, st, t);
    else if constexpr (!BOTH) hipLaunchKernelGGL((linear8_forward_kernel<T, S>), dim3((unsigned)blocks), dim3(S::kThreads), 0, st, t);
}

// Whether both sides' rows are near enough for the shapes with grouped_scales(), and whether a launch of another shape takes so many tiles.
static bool near_rows(const Rows8 &a, const Rows8 &b) { return a.q_stride < (int64_t)1 << 24 && b.q_stride < (int64_t)1 << 24; }
static bool far_launchable(int64_t a, int64_t b) { return tiles_launchable<TallB>(a, b) || tiles_launchable<LoneB>(a, b) || tiles_launchable<SmallB>(a, b); }

// By forward_cost(); terms of both sides in 8 bits count in pairs.  The shape chosen takes 1.1 % longer than the best one on average over seventeen sizes with a 16-bit weight,
// 1.4 % over as many with one in 8 bits.  Some of them (us; Large, Middle, Tall, Lone, Small; what is chosen in brackets), with a 16-bit weight:
//   32768 x 2048 -> 2048, gelu, drop, act' kept  [329] 370 405 435 474       65536 x 512 -> 400, fp32 residual  79 [76] 76  82 88
//    4096 x 1024 -> 512, gelu, drop, act' kept    47   18  15 [13] 14         2500 x 520 -> 264, gelu           38  21  12  10 [8]
// and with one in 8 bits:
//   32768 x 2048 -> 2048, gelu                   [193] 222 239 343 281       30198 x 488 -> 1392, plain         57 [48] 54  98 68
//    1000 x 2048 -> 2048, gelu                    43   17  16 [12] 13         4096 x 4096 -> 1024, gelu         65 [29; 33 in two stages] 37 40 39
//   16384 x 4096 -> 4096, plain                  [269] 341 465 665 580       65536 x 512 -> 2048, gelu and residual  387 [297] 321 530 329
template <class T>
static void launch_forward8(TileArgs &t, bool both, hipStream_t st)
{
    const int64_t moved = (t.e.out_f32 ? 4 : 2) * (t.e.residual ? 2 : 1) + (t.e.slope ? 1 : 0);
    int64_t epilogue = 64 * moved + (t.e.act > KGE_ACT_RELU ? 192 : 0) + (t.e.drop.cut ? 192 : 0);
    if (both) epilogue = epilogue * 13 / 10;
    const bool near = !both || near_rows(t.a8, t.b8);
    const double large = near ? forward_cost<LargeB>(t, epilogue + (t.e.residual ? 256 : 0), 1, 1.0, 1.0) : INFINITY;
    const double middle = near ? forward_cost<MiddleB>(t, epilogue, 2, both ? 0.7 : 0.73, both ? 3.5 : 2.5) : INFINITY, tall = forward_cost<TallB>(t, epilogue, 3, both ? 0.45 : 0.5, 2.3);
    const double small = forward_cost<SmallB>(t, epilogue, 3, both ? 0.4 : 0.45, 0.9), lone = forward_cost<LoneB>(t, epilogue, 1, both ? 0.35 : 0.4, 0.9);
    if (lone < large && lone < middle && lone < tall && lone < small) both ? launch_tiles<T, LoneB, true>(t, st) : launch_tiles<T, LoneB, false>(t, st);
    else if (large <= middle && large <= tall && large <= small) both ? launch_tiles<T, Large8, true>(t, st) : launch_tiles<T, LargeB, false>(t, st);
    else if (middle <= tall && middle <= small) {
        // (a tile a CU at most: nothing but its own stages hides its waits)
        if (both) tiles_of(t.a.extent, t.b.extent, 128) <= 256 ? launch_tiles<T, MiddleB, true>(t, st) : launch_tiles<T, Middle8, true>(t, st);
        else launch_tiles<T, MiddleB, false>(t, st);
    } else if (tall <= small) both ? launch_tiles<T, Tall8, true>(t, st) : launch_tiles<T, TallB, false>(t, st);
    else both ? launch_tiles<T, SmallB, true>(t, st) : launch_tiles<T, SmallB, false>(t, st);
}

// ---- gradients -------------------------------------------------------------------------------------
// dW = dz^T x8, dx = dz W and the bias's gradient in one launch, as linear_grads_kernel; W and X: the shapes of the two products.  32768 x 2048 x 2048 bf16 475 us (rows
// of 16 bits 465): dW alone 245 in place of 234, for the numbers that are widened between its products.
using MiddleA = Shape<128, 128, 32, 4, 2, 4>;
using SmallA = Shape<64, 64, 32, 2, 2, 4>;
template <class T, class W, class X>
__global__ __launch_bounds__(W::kThreads, W::kThreads == 512 && W::XA * W::XB <= 128 * 128 ? 4 : 1) void linear8_grads_kernel(TileArgs dw, TileArgs dx, SumArgs db, int64_t dw_blocks, int64_t dx_blocks)
{
    static_assert(W::kThreads == X::kThreads && W::XA == X::XA && W::XB == X::XB && W::STAGES >= X::STAGES, "one grid, and arrays of the larger one");
    static_assert(W::K == 32, "kFarthest");
    constexpr int kA = side_bytes<W, true>() > side_bytes<X, true>() ? side_bytes<W, true>() : side_bytes<X, true>();
    constexpr int kB = side_bytes<W, false>() > side_bytes<X, false>() ? side_bytes<W, false>() : side_bytes<X, false>();
    __shared__ __align__(16) char stage0[kB], stage1[kB], stage2[W::STAGES > 2 ? kB : 16], stage3[W::STAGES > 3 ? kB : 16];
    __shared__ __align__(16) char wide0[kA], wide1[kA], wide2[X::STAGES > 2 ? kA : 16], wide3[X::STAGES > 3 ? kA : 16];
    const int64_t block = blockIdx.x, products = dw_blocks + dx_blocks, before = dx.k > dw.k_each ? dx_blocks : 0;
    if (block >= products) join_sums<T, W::kThreads>(db, block - products, reinterpret_cast<float4 *>(stage0));
    else if (block >= before && block < before + dw_blocks)
        compute_tile<T, true, true, W, false, true, kSideA>(dw, block - before, dw_blocks, stage0, stage1, stage2, stage3, wide0, wide1);
    else
        compute_tile<T, true, false, X, false, true, kNoSideApart>(dx, before ? block : block - dw_blocks, dx_blocks, stage0, stage1, stage2, stage3, wide0, wide1, wide2,
                                                                   wide3);
}

template <class T, class W, class X>
static void launch_grads8(TileArgs &dw, TileArgs &dx, const SumArgs &db, bool want_dw, bool want_dx, hipStream_t st)
{
    for (TileArgs *t : {&dw, &dx}) t->tiles_a = (int)ceil_div(t->a.extent, W::XA), t->tiles_b = (int)ceil_div(t->b.extent, W::XB);
    const int64_t nw = want_dw ? (int64_t)dw.tiles_a * dw.tiles_b * dw.splits : 0, nx = want_dx ? (int64_t)dx.tiles_a * dx.tiles_b : 0;
    const int64_t nb = db.out ? ceil_div(db.quads, 4) : 0;
    if (nw + nx + nb) hipLaunchKernelGGL((linear8_grads_kernel<T, W, X>), dim3((unsigned)(nw + nx + nb)), dim3(W::kThreads), 0, st, dw, dx, db, nw, nx);
}

// ---- a layer's plan --------------------------------------------------------------------------------
struct Plan8 {
    bool pack_w;         // the weight is copied (one in 8 bits: widened) for the tiles
    int few;             // few_rows() of the forward pass
    size_t slope, w;     // bytes of each in a saved block, in this order
    int64_t quads;
    int sum_blocks;
    int64_t sum_rows;
};

static Plan8 plan8_of(const kge_linear *l, bool w8 = false)
{
    Plan8 p;
    p.quads = ceil_div(l->out, 4);
    p.pack_w = w8 ? !(l->type == KGE_BF16 && l->out_type == KGE_BF16) : !lies_ready(l->type, l->weight, l->weight_stride, l->in);
    // (a weight whose rows share a channel is worth copying where many rows are multiplied by it)
    if (!w8 && l->weight_stride % 2048 == 0 && l->in >= 1024 && l->out >= 1024 && l->rows >= 8192) p.pack_w = true;
    p.few = few_rows(l->type, l->rows, l->in, l->out, p.pack_w);
    p.slope = l->act == KGE_ACT_NONE ? 0 : up256((size_t)l->rows * p.quads * 4);
    p.w = p.pack_w ? packed_bytes(l->type, l->out, l->in) : 0;
    sum_ranges(l->rows, l->out, &p.sum_blocks, &p.sum_rows);
    return p;
}

// what kge_linear_fwd asks of a layer, with a weight that is read where `weight8` lies
static int check8(const kge_linear *l, bool weight8)
{
    if (!l || l->type == KGE_F32) return KGE_EINVAL;
    kge_linear as = *l;
    as.x = &as, as.x_stride = as.in;
    if (weight8) as.weight = &as, as.weight_stride = as.in;
    return check(&as);
}

template <class T>
static int forward8(const kge_linear *l, const kge_rows8 *x8, const kge_rows8 *w8, bool keep, void *y, int64_t y_stride, char *slope, char *pw, hipStream_t st)
{
    const Plan8 p = plan8_of(l, w8 != nullptr);
    TileArgs t{};
    t.splits = 1;
    t.e = Ends{y, y_stride, l->bias, l->residual, l->residual_stride, slope, l->rows, l->out, p.quads,
               make_drop(l->p, l->seed, l->step, l->step_dev, l->out), l->act, l->out_type == KGE_F32, passing(l, y, y_stride)};
    t.b8 = rows8_of(x8), t.a8 = rows8_of(w8);
    t.b = Side{x8->q, x8->q_stride / 2, l->rows};
    t.k = l->in, t.k8 = q_width(l->in) / 2;
    const bool both = w8 && !p.pack_w && !p.few;
    if (both) {  // (elements of both sides: pairs of terms)
        t.a = Side{w8->q, w8->q_stride / 2, l->out};
        t.k = t.k8;
    } else if (w8) {
        if (!p.few && l->in > 0) launch_unpack8(l->type, t.a8, l->out, up8(l->in), pw, pitch_of(l->type, l->in), st);
        t.a = Side{pw, pitch_of(l->type, l->in), l->out};
    } else {
        if (p.pack_w && (keep || !p.few)) launch_pack(l, false, true, nullptr, pw, st);
        t.a = side_of(l->weight, l->weight_stride, p.pack_w && !p.few, pw, l->type, l->in, l->out);
    }
    if (p.few) {
        launch_few8<T>(p.few, w8 != nullptr, t, st);
        KGE_CHECK_LAUNCH();
        return KGE_OK;
    }
    t.k_each = split_length(t.k, 1);
    launch_forward8<T>(t, both, st);
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

template <class T>
static int backward8(const kge_linear *l, const kge_rows8 *x8, const Plan8 &p, const GradPlan &g, const void *dy, int64_t dy_stride, const char *saved, void *dx,
                     void *dw, void *db, char *ws, hipStream_t st)
{
    const int64_t width8 = up8(l->out);
    const bool ready = l->act == KGE_ACT_NONE && nearbyint(l->p * 65536.0) == 0.0 && l->out_type == l->type && lies_ready(l->type, dy, dy_stride, l->out);
    char *dz = ws;
    float *sums = reinterpret_cast<float *>(ws + packed_bytes(l->type, l->rows, l->out));
    float *part = reinterpret_cast<float *>(reinterpret_cast<char *>(sums) + up256((size_t)p.sum_blocks * p.quads * 16));
    const bool want_dz = !ready && (dx || dw);
    if ((want_dz || db) && l->rows > 0 && l->out > 0) {
        GradArgs a{dy, dy_stride, p.slope ? saved : nullptr, l->rows, l->out, p.quads, p.sum_rows,
                   make_drop(l->p, l->seed, l->step, l->step_dev, l->out), want_dz ? dz : nullptr, width8, pitch_of(l->type, l->out), db ? sums : nullptr, 4};
        while (a.lanes < 64 && 8 * a.lanes < width8) a.lanes *= 2;
        const dim3 grid((unsigned)ceil_div(width8, 8 * a.lanes), (unsigned)p.sum_blocks);
        if (l->out_type == KGE_F32) hipLaunchKernelGGL((linear_dz_kernel<T, float, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((linear_dz_kernel<T, T, true>), grid, dim3(256), 0, st, a);
    }
    const int64_t in_quads = ceil_div(l->in, 4);
    TileArgs tx{}, tw{};
    tx.a = side_of(l->weight, l->weight_stride, p.pack_w, saved + p.slope, l->type, l->in, l->in);
    tx.b = side_of(dy, dy_stride, !ready, dz, l->type, l->out, l->rows);
    tx.k = l->out, tx.splits = 1, tx.k_each = split_length(l->out, 1);
    tx.e.y = dx, tx.e.y_stride = l->in, tx.e.rows = l->rows, tx.e.cols = l->in, tx.e.quads = in_quads;
    tw.a.extent = l->in, tw.a8 = rows8_of(x8);
    tw.b = tx.b, tw.b.extent = l->out;
    tw.k = l->rows, tw.splits = g.dw_splits, tw.k_each = split_length(l->rows, tw.splits);
    tw.partial = tw.splits > 1 ? part : nullptr;
    tw.e.y = dw, tw.e.y_stride = l->in, tw.e.rows = l->out, tw.e.cols = l->in, tw.e.quads = in_quads;
    const SumArgs sum{sums, p.sum_blocks, l->out, p.quads, db};
    if (g.tile == 256) launch_grads8<T, Large, Large>(tw, tx, sum, dw != nullptr, dx != nullptr, st);
    else if (g.tile == 128) launch_grads8<T, MiddleA, MiddleA>(tw, tx, sum, dw != nullptr, dx != nullptr, st);
    else launch_grads8<T, SmallA, SmallA>(tw, tx, sum, dw != nullptr, dx != nullptr, st);
    if (dw && tw.partial) launch_join<T>(JoinArgs{part, l->out, l->in, in_quads, tw.splits, dw}, st);
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

}  // namespace kge

using namespace kge;

// Bytes between rows of x8 that the backward pass takes: a stage's 32 rows are addressed with 32 bits.
constexpr int64_t kFarthest = (int64_t)1 << 26;

static size_t backward8_bytes(const kge_linear *l, const Plan8 &p, const GradPlan &g)
{
    return packed_bytes(l->type, l->rows, l->out) + up256((size_t)p.sum_blocks * p.quads * 16) +
           (g.dw_splits > 1 ? (size_t)g.dw_splits * l->out * ceil_div(l->in, 4) * 16 : 0);
}

extern "C" {

size_t kge_linear8_saved_bytes(const kge_linear *lin)
{
    if (check8(lin, false)) return 0;
    const Plan8 p = plan8_of(lin);
    return p.slope + p.w;
}

size_t kge_linear8_fwd_workspace(const kge_linear *lin, const kge_rows8 *weight8, int for_backward)
{
    if (check8(lin, weight8 != nullptr)) return 0;
    const Plan8 p = plan8_of(lin, weight8 != nullptr);
    return for_backward || p.few ? 0 : p.w;
}

int kge_linear8_fwd(const kge_linear *lin, const kge_rows8 *x8, const kge_rows8 *weight8, void *y, int64_t y_stride, int for_backward, void *saved,
                    size_t saved_bytes, void *workspace, size_t workspace_bytes, void *stream)
{
    if (const int rc = check8(lin, weight8 != nullptr)) return rc;
    if (const int rc = check_rows8(x8, lin->rows, lin->in)) return rc;
    if (weight8) {
        if (for_backward) return KGE_EINVAL;
        if (const int rc = check_rows8(weight8, lin->out, lin->in)) return rc;
    }
    if (lin->rows == 0 || lin->out == 0) return KGE_OK;
    if (!y) return KGE_EINVAL;
    if (y_stride < lin->out) return KGE_ESHAPE;
    const Plan8 p = plan8_of(lin, weight8 != nullptr);
    if (weight8 && !p.pack_w && !p.few && !near_rows(rows8_of(x8), rows8_of(weight8)) && !far_launchable(lin->out, lin->rows)) return KGE_ESHAPE;
    const size_t need_saved = for_backward ? p.slope + p.w : 0, need = for_backward || p.few ? 0 : p.w;
    if (need_saved && (!saved || saved_bytes < need_saved || !aligned16(saved))) return KGE_EWORKSPACE;
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KGE_EWORKSPACE;
    char *slope = for_backward && p.slope ? static_cast<char *>(saved) : nullptr;
    char *pw = for_backward ? static_cast<char *>(saved) + p.slope : static_cast<char *>(workspace);
    hipStream_t st = as_stream(stream);
    KGE_CLEAR_LAUNCH_ERRORS();
    if (lin->type == KGE_BF16) return forward8<bf16_t>(lin, x8, weight8, for_backward != 0, y, y_stride, slope, pw, st);
    return forward8<half_t>(lin, x8, weight8, for_backward != 0, y, y_stride, slope, pw, st);
}

size_t kge_linear8_bwd_workspace(const kge_linear *lin)
{
    if (check8(lin, false)) return 0;
    const GradPlan g = grad_plan(lin);
    return g.tile ? backward8_bytes(lin, plan8_of(lin), g) : 0;
}

int kge_linear8_bwd(const kge_linear *lin, const kge_rows8 *x8, const void *dy, int64_t dy_stride, const void *saved, size_t saved_bytes, void *dx,
                    void *dweight, void *dbias, void *workspace, size_t workspace_bytes, void *stream)
{
    if (const int rc = check8(lin, false)) return rc;
    if (const int rc = check_rows8(x8, lin->rows, lin->in)) return rc;
    if (dy_stride < lin->out || x8->q_stride >= kFarthest || x8->scale_stride >= kFarthest) return KGE_ESHAPE;
    if (lin->rows > 0 && lin->out > 0 && !dy) return KGE_EINVAL;
    const Plan8 p = plan8_of(lin);
    const GradPlan g = grad_plan(lin);
    if (!g.tile || (dx && !g.dx)) return KGE_ESHAPE;
    const size_t need_saved = p.slope + p.w, need = backward8_bytes(lin, p, g);
    if (need_saved && (!saved || saved_bytes < need_saved || !aligned16(saved))) return KGE_EWORKSPACE;
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KGE_EWORKSPACE;
    hipStream_t st = as_stream(stream);
    KGE_CLEAR_LAUNCH_ERRORS();
    const char *s = static_cast<const char *>(saved);
    char *ws = static_cast<char *>(workspace);
    if (lin->type == KGE_BF16) return backward8<bf16_t>(lin, x8, p, g, dy, dy_stride, s, dx, dweight, dbias, ws, st);
    return backward8<half_t>(lin, x8, p, g, dy, dy_stride, s, dx, dweight, dbias, ws, st);
}

}  // extern "C"
