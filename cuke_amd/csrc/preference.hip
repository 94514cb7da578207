// Preference loss of positive and negative scores against a frozen reference's, with its gradients (kge_preference_loss).
#include <float.h>

#include "features.hpp"

namespace kge {

struct PreferArgs {
    const void *pos, *neg, *ref_pos, *ref_neg;
    const uint8_t *mask;
    int64_t B, N, neg_stride, ref_stride, mask_stride;
    float beta, sign, smoothing, heat, target, inv_batch;  // heat: temperature * log2(e); target: 1 / (2 beta)
    int kind;
    float *dpos, *dneg, *loss;
    double *part_loss;  // one per workgroup of rows, or per segment
    float2 *stats;      // [B][segments]: largest score, sum of weights relative to it
    float *part_back;   // [B][segments]
    int64_t segments;
    double scale;
    int lanes;          // of a wave that share a row
};

// f(d) and f'(d).  The product beta d is rounded by itself (no fused multiply-add), so that the hinge's corner is where the rounded
// product says.
__device__ __forceinline__ float prefer(const PreferArgs &a, float d, float *slope)
{
    if (a.kind == KGE_PREFER_SQUARE) {
        const float g = d - a.target;
        *slope = 2.0f * g;
        return g * g;
    }
    const float z = __fmul_rn(a.beta, d);
    if (a.kind == KGE_PREFER_HINGE) {
        *slope = z < 1.0f ? -a.beta : (z >= 1.0f ? 0.0f : z);  // (a NaN stays one)
        return z >= 1.0f ? 0.0f : 1.0f - z;
    }
    // log(1 + exp(-z)) = max(-z, 0) + log(1 + e), e = exp(-|z|); what 1 + e rounds away is put back to first order, so that pairs far apart keep
    // their small loss; sigma(-z) without cancellation.  Of the two terms in |z| one is zero; a term whose factor is zero is not there, however
    // large z is
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(z)), u = 1.0f + e, inv = __builtin_amdgcn_rcpf(u);
    const float soft = fmaf(e - (u - 1.0f), inv, 0.69314718f * __builtin_amdgcn_logf(u));
    *slope = a.beta * (a.smoothing - (z > 0.0f ? e : 1.0f) * inv);
    const float share = z > 0.0f ? a.smoothing : 1.0f - a.smoothing;
    return share != 0.0f ? fmaf(share, fabsf(z), soft) : soft;
}

// Sums and maxima over the lanes that share a row: `lanes` of a wave, or a whole workgroup of four waves.
struct Group {
    int lanes;
    __device__ __forceinline__ float max(float v) const
    {
        for (int o = lanes >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
        return v;
    }
    __device__ __forceinline__ float sum(float v) const
    {
        for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
        return v;
    }
};
struct Workgroup {
    float *s;  // [4]
    __device__ __forceinline__ float max(float v) const
    {
        v = Group{kWave}.max(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    }
    __device__ __forceinline__ float sum(float v) const
    {
        v = Group{kWave}.sum(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        return (s[0] + s[1]) + (s[2] + s[3]);
    }
};

// The weight of a score so far above (below) the one that has weight 1.
__device__ __forceinline__ float weight_of(const PreferArgs &a, float above) { return __builtin_amdgcn_exp2f(a.heat * above); }
// What scores are measured against where the largest is `top`.  Where there is none, or all are infinitely low, none of them has a weight.
__device__ __forceinline__ float base_of(float top) { return top == -INFINITY ? 0.0f : top; }

// The part of a row a lane holds in registers: C quads, `apart` elements from one to the next.
template <class T, int C>
struct Held {
    float v[C][4], ref[C][4], w[C][4];
    uint32_t on;  // one bit an element

    __device__ __forceinline__ void load(const PreferArgs &a, int64_t b, int64_t n0, int64_t apart, int64_t end, bool with_ref)
    {
        const T *neg = static_cast<const T *>(a.neg) + b * a.neg_stride, *from = static_cast<const T *>(a.ref_neg) + b * a.ref_stride;
        const uint8_t *mask = a.mask + b * a.mask_stride;
        on = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t n = n0 + c * apart, left = end - n;
            const int valid = left < 4 ? (left > 0 ? (int)left : 0) : 4;
            const float4 q = load4(neg + n, valid);
            v[c][0] = q.x, v[c][1] = q.y, v[c][2] = q.z, v[c][3] = q.w;
            float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (with_ref && a.ref_neg) r = load4(from + n, valid);
            ref[c][0] = r.x, ref[c][1] = r.y, ref[c][2] = r.z, ref[c][3] = r.w;
            uint32_t bits = (1u << valid) - 1u;
            if (a.mask) {
                uint32_t there = 0;
                if (valid == 4) {
                    const auto m = Pack<uint8_t, 4>::load(mask + n).v;
                    there = (m[0] ? 1u : 0u) | (m[1] ? 2u : 0u) | (m[2] ? 4u : 0u) | (m[3] ? 8u : 0u);
                } else {
                    for (int e = 0; e < valid; ++e) there |= mask[n + e] ? 1u << e : 0u;
                }
                bits &= there;
            }
            on |= bits << (4 * c);
        }
    }
    // The largest score (of distances: the smallest, negated), then the weights relative to `top` and their sum.  The maximum is a score, not an
    // exponent: exponents of scores near the end of the range would be infinite, and those of scores far from zero lose their differences' bits.
    __device__ __forceinline__ float top(const PreferArgs &a) const
    {
        float t = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4 * C; ++i)
            if (on >> i & 1u) t = fmaxf(t, a.sign * v[i / 4][i % 4]);
        return t;
    }
    __device__ __forceinline__ float weigh(const PreferArgs &a, float top)
    {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * C; ++i) {
            float &x = w[i / 4][i % 4];
            x = on >> i & 1u ? (a.heat != 0.0f ? weight_of(a, fmaf(a.sign, v[i / 4][i % 4], -top)) : 1.0f) : 0.0f;
            sum += x;
        }
        return sum;
    }
    // losses and gradients; inv: one over the row's sum of weights
    __device__ __forceinline__ void finish(const PreferArgs &a, int64_t b, int64_t n0, int64_t apart, int64_t end, float p, float inv, float *loss, float *back) const
    {
        float l = 0.0f, k = 0.0f;
        const float up = a.sign * a.inv_batch;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float g[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float slope;
                const float f = prefer(a, a.sign * (p - (v[c][e] - ref[c][e])), &slope), x = w[c][e] * inv;
                // (A pair without a weight adds nothing, also where its loss, and then perhaps its slope, is infinite; a NaN stays one.  16384 x 1024
                // takes 1.3 us for asking; a second pass over lanes that hold such a pair spills registers, and takes more.)
                const bool there = (on >> (4 * c + e) & 1u) && !(x == 0.0f && f == INFINITY);
                l += there ? x * f : 0.0f;
                g[e] = there ? x * slope * up : 0.0f;
                k += g[e];
            }
            const int64_t n = n0 + c * apart, left = end - n;
            if (a.dneg && left > 0) store4(a.dneg + b * a.N + n, make_float4(-g[0], -g[1], -g[2], -g[3]), (int)(left < 4 ? left : 4));
        }
        *loss = l, *back = k;
    }
};

template <class T>
__device__ __forceinline__ float positive(const PreferArgs &a, int64_t b)
{
    return (float)static_cast<const T *>(a.pos)[b] - (a.ref_pos ? (float)static_cast<const T *>(a.ref_pos)[b] : 0.0f);
}

__device__ __forceinline__ double block_total(double v)
{
    __shared__ double s[16];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < (int)blockDim.x >> 6; ++w) t += s[w];
    return t;
}

// Rows of at most 1024 pairs, each read once and held in the registers of `lanes` lanes of a wave: bound by memory (16384 x 1024 fp32 with
// reference, mask and weights: 218 MB in 50 us, 4.4 TB/s), of 16-bit scores by vector instructions (the same in bf16, 151 MB: 51 us; with even weights and no
// mask 44).  A workgroup leaves one partial loss; a single one writes the loss itself.
template <class T, int C>
__global__ __launch_bounds__(1024) void preference_rows_kernel(PreferArgs a)
{
    const int lane = threadIdx.x % a.lanes, groups = blockDim.x / a.lanes;
    const Group g{a.lanes};
    double total = 0.0;
    // (every lane of a wave takes every turn: the sums are of whole waves)
    for (int64_t first = (int64_t)blockIdx.x * groups; first < a.B; first += (int64_t)gridDim.x * groups) {
        const int64_t b = first + threadIdx.x / a.lanes, n0 = 4 * lane, apart = 4 * a.lanes;
        const bool row = b < a.B;
        Held<T, C> h;
        float p = 0.0f, loss = 0.0f, back = 0.0f;
        h.load(a, row ? b : 0, n0, apart, row ? a.N : 0, true);
        if (row && a.N > 0) p = positive<T>(a, b);  // (rows of no pairs: the arrays may be NULL)
        const float top = a.heat != 0.0f ? base_of(g.max(h.top(a))) : 0.0f;
        const float sum = g.sum(h.weigh(a, top));
        h.finish(a, row ? b : 0, n0, apart, row ? a.N : 0, p, sum != 0.0f ? 1.0f / sum : 0.0f, &loss, &back);
        loss = g.sum(loss), back = g.sum(back);
        if (row && lane == 0) {
            total += (double)loss;
            if (a.dpos) a.dpos[b] = back;
        }
    }
    total = block_total(total);
    if (threadIdx.x) return;
    if (gridDim.x == 1) *a.loss = (float)(total * a.scale);
    else a.part_loss[blockIdx.x] = total;
}

// Longer rows, in segments of kSegment pairs that a workgroup holds in its registers.  Their weights' sum is not known before all have been read:
// one pass leaves every segment's largest score and its sum (there is none where weights are even and no pair is masked), a second
// joins them and reads the scores again, mostly from the caches (64 x 40943 bf16 with reference and mask, 24 MB: 4.4 and 9.8 us; with weights 5.3 and
// 10.2).  Bound by the
// latency of each pass, a row's sums end before its gradients begin; of large batches by vector instructions and memory alike (2048 x 40943 so, 755 MB:
// 330 us, with weights 343; with neither, in one pass, 178).  Segments of 1024 pairs take 5 to 45 % longer there, of 4096 up to 35 % where rows are few.
constexpr int kSegmentQuads = 2, kSegment = 256 * 4 * kSegmentQuads;
constexpr int64_t kMostSegments = ((int64_t(1) << 32) - 1) / 256;  // a launch has fewer than 2^32 threads

template <class T>
__global__ __launch_bounds__(256) void preference_stats_kernel(PreferArgs a)
{
    __shared__ float s[4];
    const Workgroup g{s};
    const int64_t b = blockIdx.x / a.segments, seg = blockIdx.x % a.segments, n0 = seg * kSegment + 4 * threadIdx.x;
    Held<T, kSegmentQuads> h;
    h.load(a, b, n0, 1024, a.N, false);
    const float top = a.heat != 0.0f ? base_of(g.max(h.top(a))) : 0.0f;
    const float sum = g.sum(h.weigh(a, top));
    if (threadIdx.x == 0) a.stats[b * a.segments + seg] = make_float2(top, sum);
}

template <class T>
__global__ __launch_bounds__(256) void preference_segment_kernel(PreferArgs a)
{
    __shared__ float s[4];
    const Workgroup g{s};
    const int64_t b = blockIdx.x / a.segments, seg = blockIdx.x % a.segments, n0 = seg * kSegment + 4 * threadIdx.x;
    Held<T, kSegmentQuads> h;
    h.load(a, b, n0, 1024, a.N, true);
    float top = 0.0f, sum = (float)a.N;
    if (a.stats) {
        const float2 *st = a.stats + b * a.segments;
        // (a segment none of whose pairs has a weight is left out)
        float t = -INFINITY, u = 0.0f;
        for (int64_t i = threadIdx.x; i < a.segments; i += 256)
            if (st[i].y != 0.0f) t = fmaxf(t, st[i].x);
        top = base_of(g.max(t));
        for (int64_t i = threadIdx.x; i < a.segments; i += 256) {
            const float2 v = st[i];
            if (v.y != 0.0f) u += v.y * weight_of(a, v.x - top);
        }
        sum = g.sum(u);
    }
    h.weigh(a, top);
    float loss, back;
    h.finish(a, b, n0, 1024, a.N, positive<T>(a, b), sum != 0.0f ? 1.0f / sum : 0.0f, &loss, &back);
    loss = g.sum(loss), back = g.sum(back);
    if (threadIdx.x) return;
    a.part_loss[b * a.segments + seg] = (double)loss;
    a.part_back[b * a.segments + seg] = back;
}

// The first workgroup adds the n partial losses up, the others (there are some behind segments only) a row's gradient a wave.
constexpr int kTotalThreads = 1024;
__global__ __launch_bounds__(kTotalThreads) void preference_total_kernel(PreferArgs a, int64_t n)
{
    if (blockIdx.x == 0) {
        double t = 0.0;
        for (int64_t i = threadIdx.x; i < n; i += kTotalThreads) t += a.part_loss[i];
        t = block_total(t);
        if (threadIdx.x == 0) *a.loss = (float)(t * a.scale);
        return;
    }
    const int64_t b = (int64_t)(blockIdx.x - 1) * (kTotalThreads / kWave) + (threadIdx.x >> 6);
    if (b >= a.B) return;
    float t = 0.0f;
    for (int64_t i = threadIdx.x & 63; i < a.segments; i += 64) t += a.part_back[b * a.segments + i];
    t = Group{kWave}.sum(t);
    if ((threadIdx.x & 63) == 0) a.dpos[b] = t;
}

constexpr int64_t kRowBlocks = 2048;  // workgroups of rows, and so partial losses, at most

static bool in_segments(const kge_preference *p) { return p->n_neg > 1024; }
static int64_t segments_of(const kge_preference *p) { return ceil_div(p->n_neg, kSegment); }

// Lanes to a row: enough that each holds a quad (of the longest rows four), a power of two.
static int lanes_of(int64_t n)
{
    int lanes = 1;
    while (lanes < 64 && 4 * lanes < n) lanes *= 2;
    return lanes;
}

template <class T>
static void launch_rows(PreferArgs &a, hipStream_t st)
{
    a.lanes = lanes_of(a.N);
    // A batch this small takes one workgroup of at most two turns, which needs no second launch to add partial losses up (8192 x 1 pairs in
    // eight turns: 15.8 us)
    const bool one = a.B * a.lanes <= 2048;
    const int threads = one ? 1024 : 256;
    const int64_t want = ceil_div(a.B, threads / a.lanes);
    const dim3 grid((unsigned)(one ? 1 : (want < kRowBlocks ? want : kRowBlocks))), block(threads);
    if (a.N <= 256) hipLaunchKernelGGL((preference_rows_kernel<T, 1>), grid, block, 0, st, a);
    else if (a.N <= 512) hipLaunchKernelGGL((preference_rows_kernel<T, 2>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((preference_rows_kernel<T, 4>), grid, block, 0, st, a);
    if (grid.x > 1) hipLaunchKernelGGL(preference_total_kernel, dim3(1), dim3(kTotalThreads), 0, st, a, (int64_t)grid.x);
}

template <class T>
static void launch_segments(PreferArgs &a, hipStream_t st)
{
    const dim3 grid((unsigned)(a.B * a.segments));
    if (a.stats) hipLaunchKernelGGL(preference_stats_kernel<T>, grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL(preference_segment_kernel<T>, grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL(preference_total_kernel, dim3((unsigned)(1 + (a.dpos ? ceil_div(a.B, kTotalThreads / kWave) : 0))), dim3(kTotalThreads), 0, st, a, a.B * a.segments);
}

static int check(const kge_preference *p)
{
    if (!p) return KGE_EINVAL;
    if (!known_type(p->type) || p->kind < KGE_PREFER_SIGMOID || p->kind > KGE_PREFER_SQUARE) return KGE_EINVAL;
    if (!(p->beta > 0.0f && p->beta <= FLT_MAX) || (p->sign != 1.0f && p->sign != -1.0f) || !(p->temperature >= 0.0f && p->temperature <= FLT_MAX)) return KGE_EINVAL;
    if (!(p->smoothing >= 0.0f && p->smoothing <= 1.0f) || (p->smoothing != 0.0f && p->kind != KGE_PREFER_SIGMOID)) return KGE_EINVAL;
    if (p->batch < 0 || p->n_neg < 0) return KGE_ESHAPE;
    if (p->batch >= (int64_t)1 << 40 || p->n_neg >= (int64_t)1 << 40) return KGE_ESHAPE;
    if (in_segments(p) && p->batch > kMostSegments / segments_of(p)) return KGE_ESHAPE;
    if (p->neg_stride < p->n_neg || (p->ref_neg && p->ref_neg_stride < p->n_neg) || (p->mask && p->mask_stride < p->n_neg)) return KGE_ESHAPE;
    if ((p->ref_pos == nullptr) != (p->ref_neg == nullptr) && p->batch > 0 && p->n_neg > 0) return KGE_EINVAL;
    if (p->batch > 0 && p->n_neg > 0 && (!p->pos || !p->neg)) return KGE_EINVAL;
    return KGE_OK;
}

}  // namespace kge

using namespace kge;

extern "C" {

size_t kge_preference_workspace(const kge_preference *pref)
{
    if (check(pref)) return 0;
    if (!in_segments(pref)) return sizeof(double) * (size_t)(pref->batch < kRowBlocks ? pref->batch : kRowBlocks);
    return (size_t)pref->batch * segments_of(pref) * (sizeof(double) + sizeof(float2) + sizeof(float));
}

int kge_preference_loss(const kge_preference *pref, float *loss, float *dpos, float *dneg, void *workspace, size_t workspace_bytes, void *stream)
{
    if (const int rc = check(pref)) return rc;
    if (!loss) return KGE_EINVAL;
    const size_t need = kge_preference_workspace(pref);
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7u))) return KGE_EWORKSPACE;
    hipStream_t st = as_stream(stream);
    PreferArgs a{};
    a.pos = pref->pos, a.neg = pref->neg, a.ref_pos = pref->ref_pos, a.ref_neg = pref->ref_neg, a.mask = pref->mask;
    a.B = pref->batch, a.N = pref->n_neg, a.neg_stride = pref->neg_stride, a.ref_stride = pref->ref_neg_stride, a.mask_stride = pref->mask_stride;
    a.beta = pref->beta, a.sign = pref->sign, a.smoothing = pref->smoothing, a.heat = fminf(pref->temperature * 1.44269504f, FLT_MAX);
    a.target = 0.5f / pref->beta, a.inv_batch = a.B > 0 ? 1.0f / (float)a.B : 0.0f, a.scale = a.B > 0 ? 1.0 / (double)a.B : 0.0;
    a.kind = pref->kind, a.dpos = dpos, a.dneg = dneg, a.loss = loss, a.part_loss = static_cast<double *>(workspace);
    KGE_CLEAR_LAUNCH_ERRORS();
    if (!in_segments(pref)) {
        if (pref->type == KGE_F32) launch_rows<float>(a, st);
        else if (pref->type == KGE_BF16) launch_rows<bf16_t>(a, st);
        else launch_rows<half_t>(a, st);
    } else if (a.B > 0) {
        a.segments = segments_of(pref);
        float2 *stats = reinterpret_cast<float2 *>(a.part_loss + a.B * a.segments);
        a.part_back = reinterpret_cast<float *>(stats + a.B * a.segments);
        a.stats = a.mask || a.heat != 0.0f ? stats : nullptr;
        if (pref->type == KGE_F32) launch_segments<float>(a, st);
        else if (pref->type == KGE_BF16) launch_segments<bf16_t>(a, st);
        else launch_segments<half_t>(a, st);
    } else {
        hipLaunchKernelGGL(preference_total_kernel, dim3(1), dim3(kTotalThreads), 0, st, a, (int64_t)0);
    }
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

}  // extern "C"
