// Linear layers with a fused epilogue, y = drop(act(x W^T + b)) + residual, and their gradients (kge_linear_fwd, kge_linear_bwd).
#include "linear_plan.hpp"

namespace kge {

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
    sum_ranges(l->rows, l->out, &p.sum_blocks, &p.sum_rows);
    return p;
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
    if (dw && tw.partial) launch_join<T>(JoinArgs{part, l->out, l->in, in_quads, tw.splits, dw}, st);
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
