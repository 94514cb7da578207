// What the feature operators (linear layers, dropout, the preference loss) share: element types, activations, the random bits of a
// dropped element.
#pragma once

#include <math.h>

#include "common.hpp"

namespace kge {

typedef _Float16 half_t;
typedef __bf16 bf16_t;

inline int64_t type_bytes(int type) { return type == KGE_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == KGE_F32 || type == KGE_BF16 || type == KGE_F16; }

// V consecutive elements of a row, at whatever address the row's stride leaves them (dword loads take any dword, the 16-bit forms any
// pair of bytes: gfx950 runs with unaligned access on).
template <class E, int V>
struct Pack {
    typedef E type __attribute__((ext_vector_type(V), aligned(sizeof(E))));
    type v;
    __device__ __forceinline__ static Pack load(const E *p) { return Pack{*reinterpret_cast<const type *>(p)}; }
    __device__ __forceinline__ void store(E *p) const { *reinterpret_cast<type *>(p) = v; }
};

// eight elements of which `valid` exist (any number: none below 1, all above 7), as floats; the rest are zero
template <class E>
__device__ __forceinline__ void load8(const E *p, int valid, float (&v)[8])
{
    if (valid >= 8) {
        const auto q = Pack<E, 8>::load(p).v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)q[e];
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < valid ? (float)p[e] : 0.0f;
}
template <class E>
__device__ __forceinline__ void store8(E *p, const float (&v)[8], int valid)
{
    if (valid >= 8) {
        Pack<E, 8> q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q.v[e] = (E)v[e];
        q.store(p);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < valid) p[e] = (E)v[e];
}

// four elements of which `valid` (0 .. 4) exist, as floats; the rest are zero
template <class E>
__device__ __forceinline__ float4 load4(const E *p, int valid)
{
    if (valid >= 4) {
        const auto q = Pack<E, 4>::load(p).v;
        return make_float4((float)q[0], (float)q[1], (float)q[2], (float)q[3]);
    }
    return make_float4(valid > 0 ? (float)p[0] : 0.0f, valid > 1 ? (float)p[1] : 0.0f, valid > 2 ? (float)p[2] : 0.0f, 0.0f);
}
template <class E>
__device__ __forceinline__ void store4(E *p, float4 v, int valid)
{
    if (valid >= 4) {
        Pack<E, 4> q;
        q.v[0] = (E)v.x, q.v[1] = (E)v.y, q.v[2] = (E)v.z, q.v[3] = (E)v.w;
        q.store(p);
        return;
    }
    if (valid > 0) p[0] = (E)v.x;
    if (valid > 1) p[1] = (E)v.y;
    if (valid > 2) p[2] = (E)v.z;
}

// ---- activations -----------------------------------------------------------------------------------
// Phi(z), the normal distribution, and exp(-z^2 / 2): erfc(x) = exp(-x^2) t P(t), t = 1 / (1 + 0.4 x), x = |z| / sqrt 2, with P of
// degree 8 fitted in 64 bits to a relative error of 1.3e-7 over 0 <= x <= 200.  One exponential and one reciprocal serve the
// activation and its derivative; the lower tail keeps its relative accuracy (1 - erf would not).
__device__ __forceinline__ void normal_cdf(float z, float *cdf, float *bell)
{
    const float x = fabsf(z) * 0.70710678f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.4f, x, 1.0f));
    float p = 0.05027035f;
    p = fmaf(p, t, -0.18293487f);
    p = fmaf(p, t, 0.16914065f);
    p = fmaf(p, t, -0.00565531f);
    p = fmaf(p, t, 0.14145454f);
    p = fmaf(p, t, 0.16853582f);
    p = fmaf(p, t, 0.20784353f);
    p = fmaf(p, t, 0.22566955f);
    p = fmaf(p, t, 0.22567586f);
    const float e = __builtin_amdgcn_exp2f(-0.72134752f * z * z);
    const float tail = 0.5f * e * t * p;
    *cdf = z < 0.0f ? tail : 1.0f - tail;
    *bell = e;
}

// act(z) in place, and act'(z), of V values (the branch is the launch's, not the value's)
template <int V>
__device__ __forceinline__ void activate(float (&z)[V], int act, float (&slope)[V])
{
    if (act == KGE_ACT_GELU) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float cdf, bell;
            normal_cdf(z[v], &cdf, &bell);
            slope[v] = fmaf(z[v] * 0.39894228f, bell, cdf);
            z[v] *= cdf;
        }
    } else if (act == KGE_ACT_SILU) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z[v]));
            slope[v] = s * fmaf(z[v], 1.0f - s, 1.0f);
            z[v] *= s;
        }
    } else if (act == KGE_ACT_RELU) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            slope[v] = z[v] > 0.0f ? 1.0f : (z[v] <= 0.0f ? 0.0f : z[v]);  // (a NaN stays one)
            z[v] = z[v] < 0.0f ? 0.0f : z[v];
        }
    }
}

// The derivative as it is kept for the backward pass of 16-bit layers: every one of them lies in [-0.13, 1.13], so 16 bits of fixed
// point hold it to 1.02e-5 (0 and 1 exactly; a nearly dead unit's below 1e-5, of gelu from about z = -5 down, becomes 0), where bf16 would add an error as large as that of the gradient's own rounding; 0, which no derivative
// comes near, is NaN.  Layers in fp32 keep it in fp32.
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ us2 slopes_to_fixed(float a, float b)  // (one conversion to two unsigned normalised numbers; it makes 0 of NaN)
{
    constexpr float k1 = 49152.0f / 65535.0f, k0 = 8192.0f / 65535.0f;
    return __builtin_bit_cast(us2, __builtin_amdgcn_cvt_pknorm_u16(fmaf(a, k1, k0), fmaf(b, k1, k0)));
}
__device__ __forceinline__ float slope_from_fixed(float q) { return q == 0.0f ? __builtin_nanf("") : (q - 8192.0f) * (1.0f / 49152.0f); }

// The derivative as layers on rows in 8 bits keep it: unsigned fixed point in steps of 1 / 200 from -0.135 (0 and 1 exactly), so off by 0.0025 at most and by
// 0.0014 in the mean square: of z of N(0, 1) that is 0.0022 (gelu) or 0.0023 (silu) of act', somewhat more than rounding it to bf16 would cost (0.0019, 0.0017) and ten times what
// rounding it to fp16 would (0.0002).  It is taken for the byte an element that it saves, kept and moved twice; 16-bit rows keep act' to 1e-5.  0, which no derivative comes
// near, is NaN.
__device__ __forceinline__ uint32_t slopes_to_bytes(float a, float b, float c, float d)
{
    auto place = [](float v) { return v == v ? fmaf(v, 200.0f, 27.0f) : 0.0f; };
    uint32_t w = __builtin_amdgcn_cvt_pk_u8_f32(place(a), 0, 0);
    w = __builtin_amdgcn_cvt_pk_u8_f32(place(b), 1, w);
    w = __builtin_amdgcn_cvt_pk_u8_f32(place(c), 2, w);
    return __builtin_amdgcn_cvt_pk_u8_f32(place(d), 3, w);
}
__device__ __forceinline__ float slope_from_byte(float q) { return q == 0.0f ? __builtin_nanf("") : (q - 27.0f) * 0.005f; }

// ---- random bits -----------------------------------------------------------------------------------
__host__ __device__ __forceinline__ uint64_t mix64(uint64_t z)  // splitmix64
{
    z += 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

// Which elements of a [rows, cols] block are dropped (kge_dropout's comment in the header defines it): four elements of a row share one
// 64-bit word, 16 bits each, so a mask costs two 64-bit products per four elements and is made again wherever it is needed.
struct Drop {
    uint64_t mixed_seed;       // mix64(seed ^ constant)
    uint64_t step;
    const uint64_t *step_dev;  // added to step, or NULL
    uint32_t cut;              // dropped where the 16 bits are below it; 0: nothing is dropped
    float scale;
    int64_t quads;             // words per row
    __device__ __forceinline__ uint64_t base() const { return cut ? mix64(mixed_seed ^ (step + (step_dev ? *step_dev : 0))) : 0; }
    // a quad's place in the sequence: places of rows a fixed distance apart differ by a constant (no product per quad)
    __device__ __forceinline__ uint64_t place(int64_t row, int64_t quad) const { return (uint64_t)(row * quads + quad) * 0x9E3779B97F4A7C15ull; }
    __device__ __forceinline__ static uint64_t word(uint64_t base, uint64_t place) { return mix64(base ^ place); }
    __device__ __forceinline__ void apply(float *v, uint64_t w) const
    {
        // (four elements; a dropped one is zero whatever it was)
        const uint32_t lo = (uint32_t)w, hi = (uint32_t)(w >> 32);
        v[0] = (lo & 0xFFFFu) >= cut ? v[0] * scale : 0.0f, v[1] = (lo >> 16) >= cut ? v[1] * scale : 0.0f;
        v[2] = (hi & 0xFFFFu) >= cut ? v[2] * scale : 0.0f, v[3] = (hi >> 16) >= cut ? v[3] * scale : 0.0f;
    }
};

inline bool drop_ok(double p) { return p >= 0.0 && p <= 1.0; }
inline Drop make_drop(double p, uint64_t seed, uint64_t step, const uint64_t *step_dev, int64_t cols)
{
    Drop d;
    d.mixed_seed = mix64(seed ^ 0xD1B54A32D192ED03ull);
    d.step = step, d.step_dev = step_dev;
    d.cut = (uint32_t)nearbyint(p * 65536.0);
    d.scale = d.cut < 65536u ? (float)(65536.0 / (65536.0 - d.cut)) : 0.0f;
    d.quads = ceil_div(cols, 4);
    return d;
}

}  // namespace kge
