// Linear layers with a fused epilogue, y = drop(act(x W^T + b)) + residual, and their gradients (kge_linear_fwd, kge_linear_bwd).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "linear_tile.hpp"

namespace kge {

// ---- operands as the matrix cores take them --------------------------------------------------------
static int64_t up8(int64_t n) { return (n + 7) & ~int64_t(7); }
static size_t up256(size_t n) { return (n + 255) & ~size_t(255); }
// Elements between the rows of an array that is laid out here: whole chunks, and not a multiple of 4096 bytes, at which all rows of a tile fall on
// one channel of the L2 (32768 x 2048 x 2048 bf16: forward 303 us with the weight so, 277 with 128 bytes more a row; dx 300 and 254).
static int64_t pitch_of(int type, int64_t width)
{
    const int64_t w = up8(width);
    return w > 0 && w * type_bytes(type) % 4096 == 0 ? w + 64 : w;
}
static size_t packed_bytes(int type, int64_t rows, int64_t width) { return up256((size_t)rows * pitch_of(type, width) * type_bytes(type)); }

// Whether an array can be read as it lies: fp32 always, 16 bits where rows start on 16 bytes and are whole chunks of 8 elements.
static bool lies_ready(int type, const void *p, int64_t stride, int64_t width) { return type == KGE_F32 || (aligned16(p) && stride % 8 == 0 && width % 8 == 0); }

// Rows of 16-bit elements of up to two arrays of one width (a layer's x and weight) copied to whole chunks, zeros behind their end, in one launch:
// two cost 2 us more.  Bound by memory: 2048 x 2048 in 5.5 us, most of it the launch.
struct PackArgs {
    const uint16_t *src[2];
    int64_t stride[2], rows[2];
    uint16_t *dst[2];
    int64_t width, pitch;
};
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a)
{
    typedef uint16_t chunk __attribute__((ext_vector_type(8)));
    const int64_t chunks = (a.width + 7) / 8, total = (a.rows[0] + a.rows[1]) * chunks;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        int64_t row = i / chunks;
        const int64_t col = 8 * (i - row * chunks), left = a.width - col;
        const bool second = row >= a.rows[0];
        if (second) row -= a.rows[0];
        const uint16_t *src = (second ? a.src[1] : a.src[0]) + row * (second ? a.stride[1] : a.stride[0]) + col;
        chunk v;
        if (left >= 8) {
            v = Pack<uint16_t, 8>::load(src).v;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < left ? src[e] : (uint16_t)0;
        }
        *reinterpret_cast<chunk *>((second ? a.dst[1] : a.dst[0]) + row * a.pitch + col) = v;
    }
}

// ---- gradient at the products ----------------------------------------------------------------------
// dz = drop(dy) act'(z) in the layer's type, and its column sums over a range of rows.  Bound by memory (dy and act' read, dz written).  Eight
// elements a lane, kGradRows rows at a time per group of lanes, so that enough loads are in flight; `lanes` of a wave (a power of two) take a
// row, or 512 columns of it, and the sums stay in registers from row to row.  32768 x 2048 bf16 (403 MB) 82 us, 4.9 TB/s.
struct GradArgs {
    const void *dy;
    int64_t dy_stride;
    const void *slope;  // [rows][4 quads] or NULL
    int64_t rows, cols, quads, rows_each;
    Drop drop;
    void *dz;  // [rows][pitch], whole chunks of it written; or NULL
    int64_t width8, pitch;
    float *sums;  // [gridDim.y][4 quads] or NULL
    int lanes;
};
constexpr int kGradRows = 2;

template <class T, class O>
__global__ __launch_bounds__(256) void linear_dz_kernel(GradArgs g)
{
    __shared__ float s_sum[256][8];
    const int lane = threadIdx.x % g.lanes, group = threadIdx.x / g.lanes, groups = 256 / g.lanes;
    const int64_t col = ((int64_t)blockIdx.x * g.lanes + lane) * 8;
    const int64_t first = (int64_t)blockIdx.y * g.rows_each, last = first + g.rows_each < g.rows ? first + g.rows_each : g.rows;
    const int64_t left = g.cols - col;
    const int valid = (int)(left < 8 ? left : 8);
    const uint64_t base = g.drop.base(), step = g.drop.place(groups, 0);
    float sum[8] = {};
    if (col < g.width8) {
        uint64_t place = g.drop.place(first + group, col >> 2);
        for (int64_t row0 = first + group; row0 < last; row0 += kGradRows * groups) {
            float v[kGradRows][8], s[kGradRows][8];
#pragma unroll
            for (int r = 0; r < kGradRows; ++r) {
                const int64_t row = row0 + r * groups < last ? row0 + r * groups : row0;
                load8(static_cast<const O *>(g.dy) + row * g.dy_stride + col, valid, v[r]);
                if (g.slope) {
                    const int64_t at = row * 4 * g.quads + col;
                    const int kept = (int)(4 * g.quads - col < 8 ? 4 * g.quads - col : 8);
                    if (sizeof(T) == 4) load8(static_cast<const float *>(g.slope) + at, kept, s[r]);
                    else load8(static_cast<const uint16_t *>(g.slope) + at, kept, s[r]);
                }
            }
#pragma unroll
            for (int r = 0; r < kGradRows; ++r, place += step) {
                const int64_t row = row0 + r * groups;
                if (row >= last) break;
                if (g.slope) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < valid) v[r][e] *= sizeof(T) == 4 ? s[r][e] : slope_from_fixed(s[r][e]);
                }
                if (g.drop.cut) {  // (last: a dropped element's gradient is zero)
                    g.drop.apply(v[r], Drop::word(base, place));
                    g.drop.apply(v[r] + 4, Drop::word(base, place + 0x9E3779B97F4A7C15ull));
                }
                if (g.dz) store8(static_cast<T *>(g.dz) + row * g.pitch + col, v[r], 8);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += v[r][e];
            }
        }
    }
    if (!g.sums) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) s_sum[threadIdx.x][e] = sum[e];
    __syncthreads();
    if (group || valid <= 0) return;
    for (int k = 1; k < groups; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += s_sum[k * g.lanes + lane][e];
    float *to = g.sums + (int64_t)blockIdx.y * g.quads * 4 + col;
    *reinterpret_cast<float4 *>(to) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    if (valid > 4) *reinterpret_cast<float4 *>(to + 4) = make_float4(sum[4], sum[5], sum[6], sum[7]);
}

// ---- partial sums joined ---------------------------------------------------------------------------
// A weight's gradient: out[row][col] = sum over n parts of part[.][row][col].  SHARE threads take a quad, each every SHARE-th part: many parts of a
// small gradient are many loads one after another otherwise (63 parts of 34 x 102: 7.2 us with one, 4.0 with eight).  Bound by memory where the
// gradient is large: 4 parts of 2048 x 2048 (75 MB) 18 us.
struct JoinArgs {
    const float *part;
    int64_t rows, cols, quads;
    int n;
    void *out;
};

template <class T, int SHARE>
__global__ __launch_bounds__(256) void linear_join_kernel(JoinArgs j)
{
    __shared__ float4 sums[SHARE > 1 ? 256 : 1];
    constexpr int kQuads = 256 / SHARE;
    const int64_t i = (int64_t)blockIdx.x * kQuads + threadIdx.x % kQuads, each = j.rows * j.quads;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (i < each) {
        const float4 *p = reinterpret_cast<const float4 *>(j.part) + i;
#pragma unroll 4
        for (int k = threadIdx.x / kQuads; k < j.n; k += SHARE) {
            const float4 v = p[k * each];
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
    }
    if constexpr (SHARE > 1) {
        sums[threadIdx.x] = s;
        __syncthreads();
        if (threadIdx.x >= kQuads) return;
#pragma unroll
        for (int k = 1; k < SHARE; ++k) {
            const float4 v = sums[threadIdx.x + k * kQuads];
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
    }
    if (i >= each) return;
    const int64_t row = i / j.quads, col = 4 * (i % j.quads), left = j.cols - col;
    store4(static_cast<T *>(j.out) + row * j.cols + col, s, (int)(left < 4 ? left : 4));
}

// ---- products --------------------------------------------------------------------------------------
// Larger tiles read less and multiply faster, smaller ones waste less at the edges and in the last round over the card, and where several share a
// CU each hides the other's epilogue.  Forward passes by tile (us; Large, Middle, Tall, Lone, Small; what is chosen in brackets):
//   32768 x 2048 -> 2048 bf16, gelu and drop   [336] 382  424  521  485       65536 x 512 -> 400, plain         [50] 50  56  75  62
//   65536 x 512 -> 400, fp32 residual            88 [75]  80  102   84        20000 x 304 -> 800, plain          36 [26] 29  37  30
//   16384 x 768 -> 512, plain                    29 [20]  27   27   25         8192 x 768 -> 512, fp32 residual  37  19 [17] 20  20
//    4096 x 1024 -> 512, gelu and drop           45  18   15  [12]  13         2500 x 520 -> 264, gelu and drop  36  19  12   9  [8]
// Lone's four stages keep a CU busy that has one tile.  Middle has eight waves (four: 27.6 us where it takes 25.6, 16384 x 768 -> 512) and shorter
// stages in the gradients, whose epilogue is short (8192 x 768 -> 512 38.7 and 36.1 us); Tall is slower with eight (20000 x 304 -> 800 40 and 44).
// fp32 (MiddleF, SmallF, DeepF): 4033 x 1200 -> 1352 [117] 131; 8192 x 1024 -> 1024 [110] 140; 8192 x 768 -> 512 [45] 45 62; 2048 x 1024 -> 1024 47
// [40]; 851 x 1968 -> 1016 48 [34]; 2500 x 520 -> 264 17 [13]; 27717 x 102 -> 34 [12] 15.  DeepF's eight waves share a tile's terms in halves, so
// that a CU with one tile has two waves a SIMD to hide splitting and waits; the same in 16 bits loses to Small (2500 x 520 -> 264 7.0 and 7.3).
using Large = Shape<256, 256, 32, 2, 4, 4>;
using Middle = Shape<128, 128, 64, 2, 4, 2>;
using MiddleG = Shape<128, 128, 32, 2, 4, 4>;
using Tall = Shape<64, 128, 64, 2, 2, 2>;
using Lone = Shape<64, 128, 64, 2, 4, 4>;
using Small = Shape<64, 64, 64, 2, 2, 3>;
using MiddleF = Shape<128, 128, 32, 2, 4, 2>;
using SmallF = Shape<64, 64, 32, 2, 2, 2>;
using DeepF = Shape<64, 64, 64, 2, 2, 2, 2>;

static int64_t tiles_of(int64_t a, int64_t b, int x) { return ceil_div(a, x) * ceil_div(b, x); }
constexpr int64_t kMostThreads = (int64_t(1) << 32) - 1;  // of a launch
template <class S>
static bool launchable(int64_t blocks) { return blocks <= kMostThreads / S::kThreads; }
template <class S>
static bool tiles_launchable(int64_t a, int64_t b) { return launchable<S>(ceil_div(a, S::XA) * ceil_div(b, S::XB)); }

template <class T, class S, bool WHOLE = true>
static void launch_forward(TileArgs &t, hipStream_t st)
{
    t.tiles_a = (int)ceil_div(t.a.extent, S::XA), t.tiles_b = (int)ceil_div(t.b.extent, S::XB);
    const int64_t blocks = (int64_t)t.tiles_a * t.tiles_b;
    if (blocks) hipLaunchKernelGGL((linear_forward_kernel<T, S, WHOLE>), dim3((unsigned)blocks), dim3(S::kThreads), 0, st, t);
}

// What a forward pass costs in tiles of a shape: rounds over the card, times the tiles a round holds on a CU (`share` at most), times a tile's area,
// times its terms and its epilogue's worth of terms (64 for a byte moved an element, 192 for gelu or silu and 192 for dropping), each at the shape's
// pace beside the largest tiles'; a CU that holds fewer tiles than it could waits more.  Over 24 sizes, each with six epilogues, the shape chosen
// takes 1 % longer than the best one on average, and 28 % at most.
template <class S>
static double forward_cost(const TileArgs &t, int64_t epilogue, int share, double pace, double epilogue_pace)
{
    const int64_t tiles = ceil_div(t.a.extent, S::XA) * ceil_div(t.b.extent, S::XB), a_cu = ceil_div(tiles, 256);
    if (!launchable<S>(tiles)) return INFINITY;
    const int64_t at_once = a_cu < share ? a_cu : share, rounds = ceil_div(tiles, 256 * (at_once > 0 ? at_once : 1));
    return (double)rounds * at_once * S::XA * S::XB * ((double)t.k / pace + epilogue / epilogue_pace) / (0.4 + 0.6 * at_once / share);
}

template <class T>
static void launch_forward(TileArgs &t, hipStream_t st)
{
    const int64_t out = sizeof(T) == 4 || t.e.out_f32 ? 4 : 2, moved = out * (t.e.residual ? 2 : 1) + (t.e.slope ? (int64_t)sizeof(T) : 0);
    const int64_t epilogue = 64 * moved + (t.e.act > KGE_ACT_RELU ? 192 : 0) + (t.e.drop.cut ? 192 : 0);
    if constexpr (sizeof(T) == 4) {
        const bool whole = t.k % 4 == 0;
        const double middle = forward_cost<MiddleF>(t, epilogue, 1, 1.0, 1.0), small = forward_cost<SmallF>(t, epilogue, 3, 0.7, 0.7);
        const double deep = forward_cost<DeepF>(t, epilogue, 1, 0.55, 0.55);
        if (deep < middle && deep < small) whole ? launch_forward<T, DeepF, true>(t, st) : launch_forward<T, DeepF, false>(t, st);
        else if (middle <= small) whole ? launch_forward<T, MiddleF, true>(t, st) : launch_forward<T, MiddleF, false>(t, st);
        else whole ? launch_forward<T, SmallF, true>(t, st) : launch_forward<T, SmallF, false>(t, st);
    } else {
        // (a residual hides behind nothing in the largest tiles: 30198 x 488 -> 1392, plain and with one, 90 and 124 us; Middle 91 and 95)
        const double large = forward_cost<Large>(t, epilogue + (t.e.residual ? 256 : 0), 1, 1.0, 1.0), middle = forward_cost<Middle>(t, epilogue, 2, 0.73, 2.5);
        const double tall = forward_cost<Tall>(t, epilogue, 3, 0.53, 2.3), small = forward_cost<Small>(t, epilogue, 3, 0.47, 0.9);
        const double lone = forward_cost<Lone>(t, epilogue, 1, 0.41, 0.9);
        if (lone < large && lone < middle && lone < tall && lone < small) launch_forward<T, Lone>(t, st);
        else if (large <= middle && large <= tall && large <= small) launch_forward<T, Large>(t, st);
        else if (middle <= tall && middle <= small) launch_forward<T, Middle>(t, st);
        else if (tall <= small) launch_forward<T, Tall>(t, st);
        else launch_forward<T, Small>(t, st);
    }
}

// Few output elements: how many times 16 rows a workgroup of linear_few_kernel takes, or 0 where tiles are faster.  copies: whether tiles would need
// an operand copied first.  Measured with gelu and drop (us; tiles, 16 rows, 32 rows): 1 x 768 -> 512 bf16 6.4, 3.5, 3.7; 256 x 4096 -> 512 17.1,
// 16.8, 13.3; 512 x 768 -> 400 6.9, 8.0, 6.9; 512 x 2048 -> 512 11.0, 16.9, 13.5; 2000 x 200 -> 100 5.4, 4.0, 4.1; 1000 x 300 -> 200, with copies, 11.8, 9.5, 9.4; fp32, whose tiles
// wait for one another longer: 37 x 300 -> 200 12.3, 3.4, 3.9; 256 x 768 -> 2048 22.2, 24.1, 19.3; 512 x 2048 -> 1024 48.8, 58.4, 44.9, and
// 512 x 2048 -> 2048 49.7, 113, 87.
static int few_rows(int type, int64_t rows, int64_t in, int64_t out, bool copies)
{
    const int64_t blocks = tiles_of(rows, out, 16);
    if (blocks <= 400) return 1;
    return blocks <= (type == KGE_F32 ? 2048 : (copies || in <= 512 ? 1024 : 768)) ? 2 : 0;
}

template <class T>
static void launch_few(int few, const TileArgs &t, hipStream_t st)
{
    const dim3 grid((unsigned)ceil_div(t.a.extent, 16), (unsigned)ceil_div(t.b.extent, 16 * few)), block(kFewWaves * kWave);
    if (few == 1) hipLaunchKernelGGL((linear_few_kernel<T, 1>), grid, block, 0, st, t);
    else hipLaunchKernelGGL((linear_few_kernel<T, 2>), grid, block, 0, st, t);
}

static int64_t split_length(int64_t k, int splits) { return ceil_div(ceil_div(k, splits), 64) * 64; }

// The tiles of a backward pass and the parts that dW's sums over rows are split into: what is expected to end first.  Workgroups for the longer
// sums start first, `slots` at a time, the others fill what they leave; a tile takes so many us a term and some besides, and parts cost a launch, and
// bytes written and read.  The paces are those that fit some six plans of each of 17 sizes, within 8 % on average.  Some of what they decide (us):
// 65536 x 256 -> 128 bf16 in 33 parts 41, in 128 49; 16384 x 768 -> 512 in tiles of 128 54, of 256 64; 32768 x 2048 -> 2048 745 and 632; 1500 x 4000
// -> 120 in one part of tiles of 64 17, in 6 of 128 22; fp32 9000 x 100 -> 1500 with dx's longer sums first 95, with dW's 105; 512 x 768 -> 400 in DeepF's
// tiles 16, in SmallF's 20.
struct GradPlan {
    int tile, dw_splits;  // tile: 256, 128 or 64; 0: no launch takes this many
    bool deep;            // DeepF
    bool dx;              // whether the launch takes dx beside dW
};
// When n jobs of length a each, then m of length b, are done by `slots` workers.
static double jobs_end(int64_t n, double a, int64_t m, double b, int64_t slots)
{
    const int64_t late = n % slots;
    const double first = (double)(n / slots) * a, second = late ? first + a : first;  // when the workers without and with a last job of the first kind are free
    if (m == 0) return second;
    auto whole = [&](double from, double t) { return from + std::ceil((t - from) / b - 1e-6) * b; };
    double t = first + (double)m * b / (double)(slots - late);
    if (t <= second || !late) return std::max(second, whole(first, t));
    t = ((double)m * b + (double)(slots - late) * first + (double)late * second) / (double)slots;
    return std::max(second, std::min(whole(first, t), whole(second, t)));
}
static GradPlan grad_plan(int type, int64_t rows, int64_t in, int64_t out, bool with_dx = true)
{
    struct Pace {
        int tile, threads, slots;
        double a_term, besides;  // us
        double alone;            // how much longer a long sum takes where nothing else hides its waits
        bool deep;
    };
    static const Pace kHalf[] = {{64, Small::kThreads, 256, 0.0026, 1.0, 2.3, false}, {128, MiddleG::kThreads, 256, 0.0066, 3.0, 1.4, false},
                                 {256, Large::kThreads, 256, 0.0260, 8.1, 1.0, false}};
    static const Pace kFloat[] = {{64, SmallF::kThreads, 512, 0.0268, 3.5, 1.0, false}, {128, MiddleF::kThreads, 256, 0.0393, 6.7, 1.0, false},
                                  {64, DeepF::kThreads, 256, 0.0165, 5.0, 1.0, true}};
    const bool f32 = type == KGE_F32;
    const Pace *paces = f32 ? kFloat : kHalf;
    const double parts_launch = f32 ? 7.0 : 5.0, part = (double)out * (double)in * 8.0 / (f32 ? 16e6 : 40e6);  // us
    GradPlan best{0, 1, false, with_dx};
    double best_end = INFINITY;
    for (int i = 0; i < 3; ++i) {
        const Pace &p = paces[i];
        const int64_t dw = tiles_of(out, in, p.tile), dx = with_dx ? tiles_of(rows, in, p.tile) : 0;
        const double b = (double)out * p.a_term + p.besides;
        for (int parts = 1; parts <= 64; parts += parts < 8 ? 1 : parts / 4) {
            const int64_t each = split_length(rows, parts), n = dw * ceil_div(rows, each > 0 ? each : 1);
            if (parts > 1 && (each < 128 || out * ceil_div(in, 4) > kMostThreads - 256)) break;  // (joining takes a thread a quad)
            if (n + dx + ceil_div(out, 16) > kMostThreads / p.threads) continue;
            const double a = (double)each * p.a_term + p.besides;
            double end = out > each ? jobs_end(dx, b, n, a, p.slots) : jobs_end(n, a, dx, b, p.slots);
            end = std::max(end, p.alone * (double)std::max(each, out) * p.a_term);
            if (parts > 1) end += parts_launch + parts * part;
            if (end < best_end) best_end = end, best = GradPlan{p.tile, parts, p.deep, with_dx};
        }
    }
    return best;
}
static GradPlan grad_plan(const kge_linear *l)
{
    const GradPlan g = grad_plan(l->type, l->rows, l->in, l->out);
    return g.tile ? g : grad_plan(l->type, l->rows, l->in, l->out, false);
}

template <class T, class S, bool WHOLE = true>
static void launch_grads(TileArgs &dw, TileArgs &dx, const SumArgs &db, bool want_dw, bool want_dx, hipStream_t st)
{
    for (TileArgs *t : {&dw, &dx}) t->tiles_a = (int)ceil_div(t->a.extent, S::XA), t->tiles_b = (int)ceil_div(t->b.extent, S::XB);
    const int64_t nw = want_dw ? (int64_t)dw.tiles_a * dw.tiles_b * dw.splits : 0, nx = want_dx ? (int64_t)dx.tiles_a * dx.tiles_b : 0;
    const int64_t nb = db.out ? ceil_div(db.quads, 4) : 0;
    if (nw + nx + nb) hipLaunchKernelGGL((linear_grads_kernel<T, S, WHOLE>), dim3((unsigned)(nw + nx + nb)), dim3(S::kThreads), 0, st, dw, dx, db, nw, nx);
}

template <class T>
static void launch_grads(const GradPlan &g, TileArgs &dw, TileArgs &dx, const SumArgs &db, bool want_dw, bool want_dx, hipStream_t st)
{
    if constexpr (sizeof(T) == 4) {
        const bool whole = dw.a.extent % 4 == 0 && dw.b.extent % 4 == 0;  // in and out
        if (g.deep) whole ? launch_grads<T, DeepF, true>(dw, dx, db, want_dw, want_dx, st) : launch_grads<T, DeepF, false>(dw, dx, db, want_dw, want_dx, st);
        else if (g.tile == 128) whole ? launch_grads<T, MiddleF, true>(dw, dx, db, want_dw, want_dx, st) : launch_grads<T, MiddleF, false>(dw, dx, db, want_dw, want_dx, st);
        else whole ? launch_grads<T, SmallF, true>(dw, dx, db, want_dw, want_dx, st) : launch_grads<T, SmallF, false>(dw, dx, db, want_dw, want_dx, st);
    } else {
        if (g.tile == 256) launch_grads<T, Large>(dw, dx, db, want_dw, want_dx, st);
        else if (g.tile == 128) launch_grads<T, MiddleG>(dw, dx, db, want_dw, want_dx, st);
        else launch_grads<T, Small>(dw, dx, db, want_dw, want_dx, st);
    }
}

// ---- a layer's plan --------------------------------------------------------------------------------
struct Plan {
    bool pack_x, pack_w;
    int few;             // few_rows() of the forward pass
    bool pack_few;       // whether its operands are copied for it where they have to be for tiles
    size_t slope, x, w;  // bytes of each in a saved block, in this order
    int64_t quads;
    int sum_blocks;      // ranges of rows the bias's gradient is summed over
    int64_t sum_rows;
};

static Plan plan_of(const kge_linear *l)
{
    Plan p;
    p.quads = ceil_div(l->out, 4);
    p.pack_x = !lies_ready(l->type, l->x, l->x_stride, l->in);
    p.pack_w = !lies_ready(l->type, l->weight, l->weight_stride, l->in);
    p.few = few_rows(l->type, l->rows, l->in, l->out, p.pack_x || p.pack_w);
    // (a weight whose rows share a channel is worth copying where many rows are multiplied by it)
    if (l->type != KGE_F32 && l->weight_stride % 2048 == 0 && l->in >= 1024 && l->out >= 1024 && l->rows >= 8192) p.pack_w = true;
    // (rows that start anywhere are read as they lie, at a third of the pace: 2110 x 1283 -> 56 21 us; that is less than the copies' launches up to
    // some 8 MB)
    p.pack_few = p.few && (ceil_div(l->rows, 16 * p.few) * ceil_div(l->out, 16) * (16 + 16 * p.few)) * l->in * 2 > 8 << 20;
    p.slope = l->act == KGE_ACT_NONE ? 0 : up256((size_t)l->rows * p.quads * 4 * type_bytes(l->type));
    p.x = p.pack_x ? packed_bytes(l->type, l->rows, l->in) : 0;
    p.w = p.pack_w ? packed_bytes(l->type, l->out, l->in) : 0;
    // ranges of at least 8 rows, about 2048 workgroups in all: few turns each, so that a range is not one wait after another
    const int64_t across = ceil_div(up8(l->out), 512), want = across > 0 && across < 2048 ? 2048 / across : 1;
    p.sum_rows = ceil_div(l->rows, want);
    if (p.sum_rows < 8) p.sum_rows = 8;
    p.sum_blocks = (int)ceil_div(l->rows, p.sum_rows);
    return p;
}

static int check(const kge_linear *l)
{
    if (!l) return KGE_EINVAL;
    if (!known_type(l->type) || (l->out_type != l->type && l->out_type != KGE_F32)) return KGE_EINVAL;
    if (l->act < KGE_ACT_NONE || l->act > KGE_ACT_SILU || !drop_ok(l->p)) return KGE_EINVAL;
    const int64_t most = (int64_t)1 << 31;
    if (l->rows < 0 || l->in < 0 || l->out < 0 || l->rows >= most || l->in >= most || l->out >= most) return KGE_ESHAPE;
    if (l->x_stride < l->in || l->weight_stride < l->in || (l->residual && l->residual_stride < l->out)) return KGE_ESHAPE;
    if (ceil_div(l->rows, 32) * ceil_div(l->out, 32) >= most || ceil_div(l->rows, 32) * ceil_div(l->in, 32) >= most ||
        ceil_div(l->in, 32) * ceil_div(l->out, 32) >= most)
        return KGE_ESHAPE;
    const int64_t a = l->out, b = l->rows;  // (some shape's tiles have to fit a launch; the choices leave out those that do not)
    if (l->type == KGE_F32 ? !tiles_launchable<MiddleF>(a, b) && !tiles_launchable<SmallF>(a, b) && !tiles_launchable<DeepF>(a, b)
                           : !tiles_launchable<Large>(a, b) && !tiles_launchable<Middle>(a, b) && !tiles_launchable<Tall>(a, b) && !tiles_launchable<Lone>(a, b) &&
                                 !tiles_launchable<Small>(a, b))
        return KGE_ESHAPE;
    if ((l->rows > 0 && l->in > 0 && !l->x) || (l->in > 0 && l->out > 0 && !l->weight)) return KGE_EINVAL;
    return KGE_OK;
}

static int grid_for(int64_t items)
{
    const int64_t b = ceil_div(items, 256);
    return (int)(b < 8192 ? b : 8192);
}

static void launch_pack(const kge_linear *l, bool x, bool weight, void *px, void *pw, hipStream_t st)
{
    const PackArgs a{{static_cast<const uint16_t *>(l->x), static_cast<const uint16_t *>(l->weight)}, {l->x_stride, l->weight_stride},
                     {x ? l->rows : 0, weight ? l->out : 0}, {static_cast<uint16_t *>(px), static_cast<uint16_t *>(pw)}, l->in, pitch_of(KGE_BF16, l->in)};
    const int64_t total = (a.rows[0] + a.rows[1]) * (up8(l->in) / 8);
    if (total) hipLaunchKernelGGL(pack_kernel, dim3(grid_for(total)), dim3(256), 0, st, a);
}

// an operand where it lies, or its packed copy
static Side side_of(const void *p, int64_t stride, bool packed, const void *copy, int type, int64_t width, int64_t extent)
{
    if (packed) return Side{copy, pitch_of(type, width), extent};
    return Side{p, stride, extent};
}

// Whether y is written past the caches: large (64 MB), in fp32, rows of whole 64-byte pieces.  65536 x 512 -> 400 with an fp32 residual 72 to 62 us,
// and 83 to 80 where its inputs come from memory; 100000 x 256 -> 256 46 to 42; rows of 4000 bytes lose (102 to 114).
static int passing(const kge_linear *l, const void *y, int64_t y_stride)
{
    return l->out_type == KGE_F32 && l->rows * y_stride >= (int64_t)16 << 20 && y_stride % 16 == 0 && reinterpret_cast<uintptr_t>(y) % 64 == 0;
}

template <class T>
static int forward(const kge_linear *l, const Plan &p, bool pack, void *y, int64_t y_stride, char *slope, char *px, char *pw, hipStream_t st)
{
    if (pack && (p.pack_x || p.pack_w)) launch_pack(l, p.pack_x, p.pack_w, px, pw, st);
    TileArgs t{};
    t.a = side_of(l->weight, l->weight_stride, p.pack_w && pack, pw, l->type, l->in, l->out);
    t.b = side_of(l->x, l->x_stride, p.pack_x && pack, px, l->type, l->in, l->rows);
    t.k = l->in, t.splits = 1, t.k_each = split_length(l->in, 1);
    t.e = Ends{y, y_stride, l->bias, l->residual, l->residual_stride, slope, l->rows, l->out, p.quads,
               make_drop(l->p, l->seed, l->step, l->step_dev, l->out), l->act, l->out_type == KGE_F32, passing(l, y, y_stride)};
    if (p.few) launch_few<T>(p.few, t, st);
    else launch_forward<T>(t, st);
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

template <class T>
static int backward(const kge_linear *l, const Plan &p, const GradPlan &g, const void *dy, int64_t dy_stride, const char *saved, void *dx, void *dw, void *db,
                    char *ws, hipStream_t st)
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
        if (l->out_type == KGE_F32) hipLaunchKernelGGL((linear_dz_kernel<T, float>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((linear_dz_kernel<T, T>), grid, dim3(256), 0, st, a);
    }
    const int64_t in_quads = ceil_div(l->in, 4);
    TileArgs tx{}, tw{};
    tx.a = side_of(l->weight, l->weight_stride, p.pack_w, saved + p.slope + p.x, l->type, l->in, l->in);
    tx.b = side_of(dy, dy_stride, !ready, dz, l->type, l->out, l->rows);
    tx.k = l->out, tx.splits = 1, tx.k_each = split_length(l->out, 1);
    tx.e.y = dx, tx.e.y_stride = l->in, tx.e.rows = l->rows, tx.e.cols = l->in, tx.e.quads = in_quads;
    tw.a = side_of(l->x, l->x_stride, p.pack_x, saved + p.slope, l->type, l->in, l->in);
    tw.b = tx.b, tw.b.extent = l->out;
    tw.k = l->rows, tw.splits = g.dw_splits, tw.k_each = split_length(l->rows, tw.splits);
    tw.partial = tw.splits > 1 ? part : nullptr;
    tw.e.y = dw, tw.e.y_stride = l->in, tw.e.rows = l->out, tw.e.cols = l->in, tw.e.quads = in_quads;
    launch_grads<T>(g, tw, tx, SumArgs{sums, p.sum_blocks, l->out, p.quads, db}, dw != nullptr, dx != nullptr, st);
    if (dw && tw.partial) {
        const JoinArgs j{part, l->out, l->in, in_quads, tw.splits, dw};
        const int64_t quads = j.rows * j.quads;
        if (quads && quads <= 65536 && j.n >= 8) hipLaunchKernelGGL((linear_join_kernel<T, 8>), dim3((unsigned)ceil_div(quads, 32)), dim3(256), 0, st, j);
        else if (quads) hipLaunchKernelGGL((linear_join_kernel<T, 1>), dim3((unsigned)ceil_div(quads, 256)), dim3(256), 0, st, j);
    }
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

}  // namespace kge

using namespace kge;

static size_t backward_bytes(const kge_linear *l, const Plan &p, const GradPlan &g)
{
    return packed_bytes(l->type, l->rows, l->out) + up256((size_t)p.sum_blocks * p.quads * 16) +
           (g.dw_splits > 1 ? (size_t)g.dw_splits * l->out * ceil_div(l->in, 4) * 16 : 0);
}

extern "C" {

size_t kge_linear_saved_bytes(const kge_linear *lin)
{
    if (check(lin)) return 0;
    const Plan p = plan_of(lin);
    return p.slope + p.x + p.w;
}

size_t kge_linear_fwd_workspace(const kge_linear *lin, int for_backward)
{
    if (check(lin)) return 0;
    const Plan p = plan_of(lin);
    return for_backward || (p.few && !p.pack_few) ? 0 : p.x + p.w;
}

int kge_linear_fwd(const kge_linear *lin, void *y, int64_t y_stride, int for_backward, void *saved, size_t saved_bytes, void *workspace,
                   size_t workspace_bytes, void *stream)
{
    if (const int rc = check(lin)) return rc;
    if (lin->rows == 0 || lin->out == 0) return KGE_OK;
    if (!y) return KGE_EINVAL;
    if (y_stride < lin->out) return KGE_ESHAPE;
    const Plan p = plan_of(lin);
    const size_t need_saved = for_backward ? p.slope + p.x + p.w : 0, need = for_backward || (p.few && !p.pack_few) ? 0 : p.x + p.w;
    const bool pack = for_backward || !p.few || p.pack_few;
    if (need_saved && (!saved || saved_bytes < need_saved || !aligned16(saved))) return KGE_EWORKSPACE;
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KGE_EWORKSPACE;
    char *slope = for_backward && p.slope ? static_cast<char *>(saved) : nullptr;
    char *px = for_backward ? static_cast<char *>(saved) + p.slope : static_cast<char *>(workspace);
    hipStream_t st = as_stream(stream);
    KGE_CLEAR_LAUNCH_ERRORS();
    if (lin->type == KGE_F32) return forward<float>(lin, p, pack, y, y_stride, slope, px, px + p.x, st);
    if (lin->type == KGE_BF16) return forward<bf16_t>(lin, p, pack, y, y_stride, slope, px, px + p.x, st);
    return forward<half_t>(lin, p, pack, y, y_stride, slope, px, px + p.x, st);
}

size_t kge_linear_bwd_workspace(const kge_linear *lin)
{
    if (check(lin)) return 0;
    const GradPlan g = grad_plan(lin);
    return g.tile ? backward_bytes(lin, plan_of(lin), g) : 0;
}

int kge_linear_bwd(const kge_linear *lin, const void *dy, int64_t dy_stride, const void *saved, size_t saved_bytes, void *dx, void *dweight,
                   void *dbias, void *workspace, size_t workspace_bytes, void *stream)
{
    if (const int rc = check(lin)) return rc;
    if (dy_stride < lin->out) return KGE_ESHAPE;
    if (lin->rows > 0 && lin->out > 0 && !dy) return KGE_EINVAL;
    const Plan p = plan_of(lin);
    const GradPlan g = grad_plan(lin);
    if (!g.tile || (dx && !g.dx)) return KGE_ESHAPE;
    const size_t need_saved = p.slope + p.x + p.w, need = backward_bytes(lin, p, g);
    if (need_saved && (!saved || saved_bytes < need_saved || !aligned16(saved))) return KGE_EWORKSPACE;
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return KGE_EWORKSPACE;
    hipStream_t st = as_stream(stream);
    KGE_CLEAR_LAUNCH_ERRORS();
    const char *s = static_cast<const char *>(saved);
    char *ws = static_cast<char *>(workspace);
    if (lin->type == KGE_F32) return backward<float>(lin, p, g, dy, dy_stride, s, dx, dweight, dbias, ws, st);
    if (lin->type == KGE_BF16) return backward<bf16_t>(lin, p, g, dy, dy_stride, s, dx, dweight, dbias, ws, st);
    return backward<half_t>(lin, p, g, dy, dy_stride, s, dx, dweight, dbias, ws, st);
}

}  // extern "C"
