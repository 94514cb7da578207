// Preference loss of positive and negative scores against a frozen reference's, with its gradients (kge_preference_loss).
#include <float.h>

#include "features.hpp"

namespace kge {

struct PreferArgs {
    const void *pos, *neg, *ref_pos, *ref_neg;
    const uint8_t *mask;
    int64_t B, N, neg_stride, ref_stride, mask_stride;
    float beta, sign, smoothing, temperature, target, inv_batch;  // target: 1 / (2 beta)
    int kind;
    float *dpos, *dneg;
    double *row_loss;
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
        *slope = z < 1.0f ? -a.beta : 0.0f;
        return z < 1.0f ? 1.0f - z : 0.0f;
    }
    // log(1 + exp(-z)) = max(-z, 0) + log(1 + exp(-|z|)); sigma(-z) without cancellation
    const float e = __expf(-fabsf(z)), soft = log1pf(e), s = (z > 0.0f ? e : 1.0f) / (1.0f + e);
    *slope = a.beta * (a.smoothing - s);
    return soft + (1.0f - a.smoothing) * fmaxf(-z, 0.0f) + a.smoothing * fmaxf(z, 0.0f);
}

__device__ __forceinline__ float block_sum(float v, float *s)
{
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return s[0] + s[1] + s[2] + s[3];
}
__device__ __forceinline__ float block_max(float v, float *s)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

// One workgroup a row: the largest weight's exponent, the sum of weights, then loss and gradients.
template <class T>
__global__ __launch_bounds__(256) void preference_row_kernel(PreferArgs a)
{
    __shared__ float s[4];
    for (int64_t b = blockIdx.x; b < a.B; b += gridDim.x) {
        const T *neg = static_cast<const T *>(a.neg) + b * a.neg_stride;
        const T *ref = a.ref_neg ? static_cast<const T *>(a.ref_neg) + b * a.ref_stride : nullptr;
        const uint8_t *mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
        const float heat = a.temperature * a.sign;
        float top = -INFINITY;
        if (heat != 0.0f)
            for (int64_t n = threadIdx.x; n < a.N; n += 256)
                if (!mask || mask[n]) top = fmaxf(top, heat * (float)neg[n]);
        top = heat != 0.0f ? block_max(top, s) : 0.0f;
        float sum = 0.0f;
        for (int64_t n = threadIdx.x; n < a.N; n += 256)
            if (!mask || mask[n]) sum += heat != 0.0f ? __expf(heat * (float)neg[n] - top) : 1.0f;
        sum = block_sum(sum, s);
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        const float p = (float)static_cast<const T *>(a.pos)[b] - (a.ref_pos ? (float)static_cast<const T *>(a.ref_pos)[b] : 0.0f);
        float loss = 0.0f, back = 0.0f;
        for (int64_t n = threadIdx.x; n < a.N; n += 256) {
            float g = 0.0f;
            if (!mask || mask[n]) {
                const float v = (float)neg[n];
                const float w = (heat != 0.0f ? __expf(heat * v - top) : 1.0f) * inv;
                float slope;
                const float f = prefer(a, a.sign * (p - (v - (ref ? (float)ref[n] : 0.0f))), &slope);
                loss += w * f;
                g = w * slope * a.sign * a.inv_batch;
                back += g;
            }
            if (a.dneg) a.dneg[b * a.N + n] = -g;
        }
        loss = block_sum(loss, s);
        back = block_sum(back, s);
        if (threadIdx.x == 0) {
            a.row_loss[b] = (double)loss;
            if (a.dpos) a.dpos[b] = back;
        }
    }
}

__global__ __launch_bounds__(256) void preference_total_kernel(const double *rows, int64_t n, double scale, float *loss)
{
    __shared__ double s[256];
    double t = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 256) t += rows[i];
    s[threadIdx.x] = t;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = (float)(s[0] * scale);
}

static int check(const kge_preference *p)
{
    if (!p) return KGE_EINVAL;
    if (!known_type(p->type) || p->kind < KGE_PREFER_SIGMOID || p->kind > KGE_PREFER_SQUARE) return KGE_EINVAL;
    if (!(p->beta > 0.0f && p->beta <= FLT_MAX) || (p->sign != 1.0f && p->sign != -1.0f) || !(p->temperature >= 0.0f && p->temperature <= FLT_MAX)) return KGE_EINVAL;
    if (!(p->smoothing >= 0.0f && p->smoothing <= 1.0f) || (p->smoothing != 0.0f && p->kind != KGE_PREFER_SIGMOID)) return KGE_EINVAL;
    if (p->batch < 0 || p->n_neg < 0) return KGE_ESHAPE;
    if (p->neg_stride < p->n_neg || (p->ref_neg && p->ref_neg_stride < p->n_neg) || (p->mask && p->mask_stride < p->n_neg)) return KGE_ESHAPE;
    if ((p->ref_pos == nullptr) != (p->ref_neg == nullptr) && p->batch > 0 && p->n_neg > 0) return KGE_EINVAL;
    if (p->batch > 0 && p->n_neg > 0 && (!p->pos || !p->neg)) return KGE_EINVAL;
    return KGE_OK;
}

}  // namespace kge

using namespace kge;

extern "C" {

size_t kge_preference_workspace(const kge_preference *pref) { return check(pref) ? 0 : sizeof(double) * (size_t)pref->batch; }

int kge_preference_loss(const kge_preference *pref, float *loss, float *dpos, float *dneg, void *workspace, size_t workspace_bytes, void *stream)
{
    if (const int rc = check(pref)) return rc;
    if (!loss) return KGE_EINVAL;
    const size_t need = kge_preference_workspace(pref);
    if (need && (!workspace || workspace_bytes < need)) return KGE_EWORKSPACE;
    hipStream_t st = as_stream(stream);
    double *rows = static_cast<double *>(workspace);
    PreferArgs a{pref->pos, pref->neg, pref->ref_pos, pref->ref_neg, pref->mask, pref->batch, pref->n_neg, pref->neg_stride,
                 pref->ref_neg_stride, pref->mask_stride, pref->beta, pref->sign, pref->smoothing, pref->temperature, 0.5f / pref->beta,
                 pref->batch > 0 ? 1.0f / (float)pref->batch : 0.0f, pref->kind, dpos, dneg, rows};
    KGE_CLEAR_LAUNCH_ERRORS();
    if (pref->batch > 0) {
        const dim3 grid((unsigned)(pref->batch < 65536 ? pref->batch : 65536));
        if (pref->type == KGE_F32) hipLaunchKernelGGL(preference_row_kernel<float>, grid, dim3(256), 0, st, a);
        else if (pref->type == KGE_BF16) hipLaunchKernelGGL(preference_row_kernel<bf16_t>, grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(preference_row_kernel<half_t>, grid, dim3(256), 0, st, a);
    }
    hipLaunchKernelGGL(preference_total_kernel, dim3(1), dim3(256), 0, st, rows, pref->batch, pref->batch > 0 ? 1.0 / (double)pref->batch : 0.0, loss);
    KGE_CHECK_LAUNCH();
    return KGE_OK;
}

}  // extern "C"
