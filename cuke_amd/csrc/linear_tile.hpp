// Matrix products of the linear layers on the matrix cores: out[m][n] = sum over k of side a (n, k) and side b (m, k).
//
// Each side lies in memory in one of two ways: ALONG rows (row = its index, the sum runs inside the row) or ACROSS them (the sum runs
// over rows, the index inside).  y = x W^T has both sides along, dx = dz W one across, dW = dz^T x both: no operand is ever transposed in
// memory.  A tile that lies across is turned by the transposing LDS reads on its way to the matrix cores.  16-bit tiles go to LDS 16 bytes a lane
// without passing through registers; fp32 ones are taken through registers, where every value becomes three bf16 parts (mfma_split.hpp), of
// whose nine products six are formed.
#pragma once

#include "features.hpp"
#include "mfma_split.hpp"

namespace kge {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

template <class E>
struct Mfma;
template <>
struct Mfma<bf16_t> {
    __device__ __forceinline__ static floatx16 go(s16x8 a, s16x8 b, floatx16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mfma<half_t> {
    __device__ __forceinline__ static floatx16 go(s16x8 a, s16x8 b, floatx16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// One side of a product.  16 bits: rows start 16-byte aligned and a multiple of 8 elements apart; elements between the last one and the next
// multiple of 8 belong to the row and, where the sum runs inside it, are zero.  fp32: rows as they lie.
struct Side {
    const void *p;
    int64_t stride;  // elements between rows
    int64_t extent;  // indices
};

struct Ends {
    void *y;
    int64_t y_stride;
    const void *bias;
    const void *residual;
    int64_t residual_stride;
    void *slope;  // [rows][quads * 4], or NULL
    int64_t rows, cols, quads;
    Drop drop;
    int act;
    int out_f32;  // y and residual in fp32
    int passing;  // y, in fp32 and its quads on 16 bytes, is written past the caches
};

struct TileArgs {
    Side a, b;      // a: the columns of the output, b: its rows
    int64_t k;      // terms of every sum
    int64_t k_each; // per split, a multiple of 64
    int tiles_a, tiles_b, splits;
    float *partial; // where a sum is split: [splits][rows][quads * 4] in fp32, to be joined; else NULL
    Ends e;
};

static __device__ __align__(16) const uint32_t zero_chunk[4] = {0, 0, 0, 0};  // what chunks outside a side read

__device__ __forceinline__ void chunk_to_lds(const void *src, void *lds)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src, (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

// A tile of X indices by K (32 or 64) terms in LDS, as 16-byte chunks.  Along: K / 8 chunks a row, chunk j in slot j ^ (row / 2 % 8) (K = 32: j ^
// (row / 4 % 4)), so that the 128-bit reads of sixteen consecutive rows fall on distinct banks of the 64.  Across: X / 8 chunks a row of terms, pairs of chunks permuted by the row so
// that the transposing reads of four rows (and of both halves of a wave, where the row is long enough) do.
template <int X, int K, bool ACROSS, int THREADS>
struct Tile {
    static constexpr int kChunks = X * K / 8;
    static constexpr int kRounds = kChunks / THREADS;
    static constexpr int kRow = ACROSS ? X / 8 : K / 8;  // chunks a row
    static_assert(kChunks % THREADS == 0, "whole rounds");
    static_assert(K == 32 || K == 64, "turn() knows these rows");

    __device__ __forceinline__ static int turn(int row)
    {
        if (!ACROSS) return K == 64 ? (row >> 1) & 7 : (row >> 2) & 3;
        return X >= 256 ? 2 * (2 * (row & 3) + 8 * ((row >> 3) & 1)) : (X >= 128 ? 4 * (row & 3) : 2 * (row & 3));
    }

    // The chunks a thread brings in: where the next ones come from, and how far they are from the ones behind them.
    template <class E>
    struct Feed {
        const char *from[kRounds];
        int64_t step[kRounds];
        int term[kRounds];  // of the chunk, within the tile

        __device__ __forceinline__ void start(const Side &s, int64_t first, int64_t k)
        {
            const E *p = static_cast<const E *>(s.p);
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int c = r * THREADS + (int)threadIdx.x, row = c / kRow, j = (c % kRow) ^ turn(row);
                const int64_t index = first + (ACROSS ? 8 * j : row);
                term[r] = ACROSS ? row : 8 * j;
                const bool there = index < s.extent;
                from[r] = there ? reinterpret_cast<const char *>(p + (ACROSS ? (k + row) * s.stride + index : index * s.stride + k + 8 * j))
                                : reinterpret_cast<const char *>(zero_chunk);
                step[r] = there ? (ACROSS ? K * s.stride : K) * (int64_t)sizeof(E) : 0;
            }
        }
        // the next tile, of which `left` terms exist (none, behind the end)
        __device__ __forceinline__ void load(int64_t left, char *lds)
        {
            const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                chunk_to_lds(term[r] < left ? from[r] : reinterpret_cast<const char *>(zero_chunk), lds + 16 * (r * THREADS + wave * 64));
                from[r] += step[r];
            }
        }
    };

    // The same of an fp32 side: a chunk's eight values wait in registers (two tiles' at a time) until they go to LDS as parts.  A quad that
    // exists as a whole or not at all needs no branch, behind which its load would be waited for; only where rows are no whole quads (not WHOLE) and
    // a tile holds their end are values taken one at a time.
    template <bool WHOLE>
    struct FloatFeed {
        const float *from[kRounds];
        int64_t step;
        int term[kRounds], there[kRounds];  // there: how many of a chunk's indices exist (across; along: of its row, all or none)
        bool ends;                          // across: the tile holds the end of its rows, inside a quad
        float held[2][kRounds][8];

        __device__ __forceinline__ void start(const Side &s, int64_t first, int64_t k)
        {
            const float *p = static_cast<const float *>(s.p);
            step = ACROSS ? K * s.stride : K;
            ends = ACROSS && first + X > s.extent && s.extent % 4 != 0;
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int c = r * THREADS + (int)threadIdx.x, row = c / kRow, j = (c % kRow) ^ turn(row);
                const int64_t index = first + (ACROSS ? 8 * j : row), rest = s.extent - index;
                term[r] = ACROSS ? row : 8 * j;
                there[r] = rest <= 0 ? 0 : (ACROSS && rest < 8 ? (int)rest : 8);
                from[r] = p + (ACROSS ? (k + row) * s.stride + index : index * s.stride + k + 8 * j);
            }
        }
        __device__ __forceinline__ void fetch(int set, int64_t left)
        {
            const int most = (int)(left < K ? left : K);
            const bool single = !WHOLE && (ACROSS ? ends : most > 0 && most % 4 != 0);
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int rest = most - term[r], valid = ACROSS ? (rest > 0 ? there[r] : 0) : (rest < there[r] ? rest : there[r]);
                if (single) {
                    load8(from[r], valid, held[set][r]);
                } else {
                    const float *zero = reinterpret_cast<const float *>(zero_chunk);
                    // (said to be global memory: the choice between two objects would make flat loads of these, which count with the LDS's)
                    typedef const __attribute__((address_space(1))) f4u *quad;
                    const f4u a = *(quad)(valid > 0 ? from[r] : zero), b = *(quad)(valid > 4 ? from[r] + 4 : zero);
#pragma unroll
                    for (int e = 0; e < 4; ++e) held[set][r][e] = a[e], held[set][r][4 + e] = b[e];
                }
                from[r] += step;
            }
        }
        __device__ __forceinline__ void put(int set, char *lds, int plane_bytes)
        {
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                // (an infinite value, or one that rounds to infinity, and NaN make NaN of the second part and so of every sum they enter, which is
                // then formed again)
                bf16x4 lo[kSplitParts], hi[kSplitParts];
                bf16x8 part[kSplitParts];
                // (The compiler has been seen to let the parts overwrite the values they are still to be taken from, where both are tuples of
                // registers: each value passes through a register of its own.)
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = held[set][r][e];
                    asm("" : "+v"(v[e]));
                }
                split_quad(make_float4(v[0], v[1], v[2], v[3]), lo);
                split_quad(make_float4(v[4], v[5], v[6], v[7]), hi);
#pragma unroll
                for (int k = 0; k < kSplitParts; ++k) part[k] = __builtin_shufflevector(lo[k], hi[k], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int k = 0; k < kSplitParts; ++k) *reinterpret_cast<bf16x8 *>(lds + k * plane_bytes + 16 * (r * THREADS + (int)threadIdx.x)) = part[k];
            }
        }
    };

    // eight terms of an index for each lane: index at + lane % 32, terms 16 step + 8 (lane / 32) .. + 7
    __device__ __forceinline__ static s16x8 read(const char *lds, int at, int step, int lane)
    {
        if (!ACROSS) {
            const int row = at + (lane & 31), j = 2 * step + (lane >> 5);
            return *reinterpret_cast<const s16x8 *>(lds + 16 * (row * kRow + (j ^ turn(row))));
        }
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const int row = 16 * step + 8 * (lane >> 5) + ((lane & 15) >> 2), index = at + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        const char *p = lds + 16 * (row * kRow + ((index >> 3) ^ turn(row))) + 2 * (index & 7);
        const char *q = lds + 16 * ((row + 4) * kRow + ((index >> 3) ^ turn(row + 4))) + 2 * (index & 7);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)q);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// The sums of four (`valid`) output elements of a row by fp32 instructions, for fp32 sides.  Not for speed: it runs where a sum is not finite.
template <bool A_ACROSS, bool B_ACROSS>
__device__ __noinline__ float4 plain_sums(Side a, Side b, int64_t n, int valid, int64_t m, int64_t k0, int64_t k1)
{
    const float *pa = static_cast<const float *>(a.p), *pb = static_cast<const float *>(b.p);
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int v = 0; v < valid; ++v)
        for (int64_t k = k0; k < k1; ++k)
            s[v] = fmaf(pa[A_ACROSS ? k * a.stride + n + v : (n + v) * a.stride + k], pb[B_ACROSS ? k * b.stride + m : m * b.stride + k], s[v]);
    return make_float4(s[0], s[1], s[2], s[3]);
}

// Four elements of a residual's row as they lie in memory, requested ahead of their use (a 16-bit row's fill half of it).
struct Raw4 {
    f4 v;
    template <class T>
    __device__ __forceinline__ void fetch(const Ends &e, int64_t row, int64_t col)
    {
        const int64_t at = (row < e.rows ? row : e.rows - 1) * e.residual_stride + (col < e.cols ? col : e.cols - 4);
        typedef float pair __attribute__((ext_vector_type(2), aligned(2)));
        if (sizeof(T) == 4 || e.out_f32) {
            v = Pack<float, 4>::load(static_cast<const float *>(e.residual) + at).v;
        } else {
            const pair q = *reinterpret_cast<const pair *>(static_cast<const T *>(e.residual) + at);
            v[0] = q[0], v[1] = q[1];
        }
    }
    template <class T>
    __device__ __forceinline__ f4 value(const Ends &e) const
    {
        if constexpr (sizeof(T) == 2) {
            typedef T quad __attribute__((ext_vector_type(4)));
            typedef float pair __attribute__((ext_vector_type(2)));
            const quad q = __builtin_bit_cast(quad, pair{v[0], v[1]});
            if (!e.out_f32) return f4{(float)q[0], (float)q[1], (float)q[2], (float)q[3]};
        }
        return v;
    }
};

// Four consecutive columns (`valid` of them exist) of R rows, `apart` rows from one to the next, through the layer's epilogue.  T: the layer's
// type.  R rows at a time, so that one's arithmetic hides another's latencies where few waves run.  ahead: the rows' residuals, or NULL.
template <class T, int R>
__device__ __forceinline__ void finish_quads(const Ends &e, uint64_t base, int64_t first, int apart, int64_t col, int valid, float (&z)[R][4], float4 bias,
                                             const Raw4 *ahead)
{
    float res[R][4];
    if (ahead) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const f4 v = ahead[r].value<T>(e);
            res[r][0] = v[0], res[r][1] = v[1], res[r][2] = v[2], res[r][3] = v[3];
        }
    } else if (e.residual) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = first + r * apart, at = (row < e.rows ? row : e.rows - 1) * e.residual_stride + col;
            const float4 v = sizeof(T) == 4 || e.out_f32 ? load4(static_cast<const float *>(e.residual) + at, valid)
                                                         : load4(static_cast<const T *>(e.residual) + at, valid);
            res[r][0] = v.x, res[r][1] = v.y, res[r][2] = v.z, res[r][3] = v.w;
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) z[r][0] += bias.x, z[r][1] += bias.y, z[r][2] += bias.z, z[r][3] += bias.w;
    if (e.act != KGE_ACT_NONE) {
        float flat[4 * R], slope[4 * R];
#pragma unroll
        for (int i = 0; i < 4 * R; ++i) flat[i] = z[i / 4][i % 4];
        activate(flat, e.act, slope);
#pragma unroll
        for (int i = 0; i < 4 * R; ++i) z[i / 4][i % 4] = flat[i];
        if (e.slope) {  // (rows of whole quads)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t row = first + r * apart, at = row * 4 * e.quads + col;
                if (row >= e.rows) continue;
                if (sizeof(T) == 4) {
                    *reinterpret_cast<float4 *>(static_cast<float *>(e.slope) + at) = make_float4(slope[4 * r], slope[4 * r + 1], slope[4 * r + 2], slope[4 * r + 3]);
                } else {
                    const us2 lo = slopes_to_fixed(slope[4 * r], slope[4 * r + 1]), hi = slopes_to_fixed(slope[4 * r + 2], slope[4 * r + 3]);
                    const ushort4 q = {lo[0], lo[1], hi[0], hi[1]};
                    *reinterpret_cast<ushort4 *>(static_cast<uint16_t *>(e.slope) + at) = q;
                }
            }
        }
    }
    if (e.drop.cut) {
        const uint64_t place = e.drop.place(first, col >> 2), step = e.drop.place(apart, 0);
#pragma unroll
        for (int r = 0; r < R; ++r) e.drop.apply(z[r], Drop::word(base, place + r * step));
    }
    if (e.residual) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int v = 0; v < 4; ++v) z[r][v] += res[r][v];
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t row = first + r * apart, at = row * e.y_stride + col;
        if (row >= e.rows) continue;
        const float4 v = make_float4(z[r][0], z[r][1], z[r][2], z[r][3]);
        if (e.passing && valid >= 4) {
            __builtin_nontemporal_store(f4{v.x, v.y, v.z, v.w}, reinterpret_cast<f4 *>(static_cast<float *>(e.y) + at));
            continue;
        }
        if (sizeof(T) == 4 || e.out_f32) store4(static_cast<float *>(e.y) + at, v, valid);
        else store4(static_cast<T *>(e.y) + at, v, valid);
    }
}

// Workgroups are dealt to the eight XCDs in turn (wherever the count starts); consecutive tiles go to one XCD, whose L2 then holds the rows and columns they share:
// eight rows of tiles at a time, walked column by column.
__device__ __forceinline__ void tile_of(int64_t block, int64_t blocks, const TileArgs &t, int *ta, int *tb, int *split)
{
    const int64_t xcd = block & 7, each = blocks >> 3, more = blocks & 7;
    const int64_t id = xcd * each + (xcd < more ? xcd : more) + (block >> 3);
    const int64_t tiles = (int64_t)t.tiles_a * t.tiles_b;
    *split = (int)(id / tiles);
    const int64_t q = id % tiles, band = (int64_t)8 * t.tiles_a;
    const int64_t first = q / band * 8, wide = t.tiles_b - first < 8 ? t.tiles_b - first : 8;
    *tb = (int)(first + q % band % wide), *ta = (int)(q % band / wide);
}

// A wave's own loads have landed but for the last `out` (LDS reads and writes all have), and every wave's have: what the stage in turn holds
// may be read, and the stage read last may be written.
template <int OUT>
__device__ __forceinline__ void stage_ready()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((OUT & 15) | (OUT >> 4) << 14 | 7 << 4);  // vmcnt(OUT) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void lds_ready()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);  // lgkmcnt(0): loads to registers stay in flight
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A workgroup of WA x WB waves computes XA columns by XB rows, K terms at a time.  16 bits: STAGES tiles are in LDS, in arrays of their own (so
// that the compiler sees that the one being read is none of those being written); STAGES - 1 are requested ahead, and one barrier a tile both
// publishes the next and frees the last.  fp32: two stages, two more tiles in registers.  SHARE > 1: as many groups of WA x WB waves each multiply
// their share of every tile's terms, and join their sums in LDS before the epilogue.
// Bound by the matrix cores where sums are long: 32768 x 2048 -> 2048 bf16 plain 277 us (992 TFLOP/s; a large library product of this card 1383, both
// held by its power), its gradients 470 (1170); fp32 8192 x 1024 -> 1024 103 us (1.0 PFLOP/s of bf16 products).  Where they are short, by waits: a
// CU's first tiles and its epilogues, which more workgroups a CU hide.
template <int XA_, int XB_, int K_, int WA_, int WB_, int STAGES_, int SHARE_ = 1>
struct Shape {
    static constexpr int XA = XA_, XB = XB_, K = K_, WA = WA_, WB = WB_, STAGES = STAGES_, SHARE = SHARE_, kThreads = WA * WB * SHARE * kWave;
};
template <class T, class S>
constexpr int stage_bytes() { return (S::XA + S::XB) * S::K * 2 * (sizeof(T) == 4 ? kSplitParts : 1); }

// T: the layer's type.  LAYER: sums go through the layer's epilogue; else they are stored in its type, or as parts of split sums.  WHOLE: an fp32
// side's rows are whole quads.
template <class T, bool A_ACROSS, bool B_ACROSS, class S, bool LAYER, bool WHOLE>
__device__ __forceinline__ void compute_tile(const TileArgs &t, int64_t block, int64_t blocks, char *stage0, char *stage1, char *stage2, char *stage3)
{
    constexpr bool kFloat = sizeof(T) == 4;
    using E = typename std::conditional<kFloat, bf16_t, T>::type;
    constexpr int PLANES = kFloat ? kSplitParts : 1, K = S::K, STAGES = S::STAGES, WA = S::WA, WB = S::WB, SHARE = S::SHARE;
    using A = Tile<S::XA, K, A_ACROSS, S::kThreads>;
    using B = Tile<S::XB, K, B_ACROSS, S::kThreads>;
    constexpr int kBytesA = S::XA * K * 2, kBytesB = S::XB * K * 2, kStage = stage_bytes<T, S>();
    constexpr int FA = S::XA / WA / 32, FB = S::XB / WB / 32;
    static_assert(STAGES >= 2 && STAGES <= 4 && (!kFloat || STAGES == 2), "stages");

    int ta, tb, split;
    tile_of(block, blocks, t, &ta, &tb, &split);
    const int64_t n0 = (int64_t)ta * S::XA, m0 = (int64_t)tb * S::XB;
    const int64_t k0 = split * t.k_each, k1 = k0 + t.k_each < t.k ? k0 + t.k_each : t.k;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wa = (wave % WA) * (S::XA / WA), wb = (SHARE > 1 ? wave / WA % WB : wave / WA) * (S::XB / WB), part = SHARE > 1 ? wave / (WA * WB) : 0;  // of every tile's terms

    floatx16 acc[FA][FB] = {}, low[kFloat ? FA : 1][kFloat ? FB : 1] = {};
    int64_t left = k1 - k0;  // terms not requested yet
    const int tiles = left > 0 ? (int)((left + K - 1) / K) : 0;
    auto stage = [&](int u) -> char * { return u == 0 ? stage0 : (u == 1 ? stage1 : (u == 2 ? stage2 : stage3)); };
    auto multiply = [&](const char *lds) {
#pragma unroll
        for (int u = 0; u < K / 16 / SHARE; ++u) {
            const int step = part * (K / 16 / SHARE) + u;
            s16x8 a[FA][PLANES], b[FB][PLANES];
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
#pragma unroll
                for (int j = 0; j < FB; ++j) b[j][p] = B::read(lds + PLANES * kBytesA + p * kBytesB, wb + 32 * j, step, lane);
#pragma unroll
                for (int i = 0; i < FA; ++i) a[i][p] = A::read(lds + p * kBytesA, wa + 32 * i, step, lane);
            }
#pragma unroll
            for (int i = 0; i < FA; ++i)
#pragma unroll
                for (int j = 0; j < FB; ++j) {
                    if constexpr (!kFloat) {
                        acc[i][j] = Mfma<E>::go(a[i][0], b[j][0], acc[i][j]);
                    } else {
#pragma unroll
                        for (int u = 0; u < kSplitTerms - 1; ++u) low[i][j] = Mfma<E>::go(a[i][kTermA[u]], b[j][kTermB[u]], low[i][j]);
                        acc[i][j] = Mfma<E>::go(a[i][0], b[j][0], acc[i][j]);
                    }
                }
        }
    };
    if constexpr (kFloat) {
        typename A::template FloatFeed<WHOLE> feed_a;
        typename B::template FloatFeed<WHOLE> feed_b;
        feed_a.start(t.a, n0, k0), feed_b.start(t.b, m0, k0);
        auto fetch = [&](int set) { feed_a.fetch(set, left), feed_b.fetch(set, left), left -= K; };
        auto put = [&](int set, char *lds) { feed_a.put(set, lds, kBytesA), feed_b.put(set, lds + PLANES * kBytesA, kBytesB); };
        // (in this order: the loop waits for the older of two tiles' loads only where the entry leaves them in the loop's own order)
        fetch(0);
        __builtin_amdgcn_sched_barrier(0);
        fetch(1);
        __builtin_amdgcn_sched_barrier(0);
        put(0, stage0);
        __builtin_amdgcn_sched_barrier(0);
        fetch(0);
        __builtin_amdgcn_sched_barrier(0);
        auto turn = [&](int u) {
            lds_ready();
            put(1 - u, stage(1 - u));
            fetch(1 - u);
            multiply(stage(u));
        };
        int at = 0;
        for (; at + 2 <= tiles; at += 2) turn(0), turn(1);
        if (at < tiles) turn(0);
    } else {
        typename A::template Feed<E> feed_a;
        typename B::template Feed<E> feed_b;
        constexpr int kLoads = A::kRounds + B::kRounds;  // per thread and tile
        feed_a.start(t.a, n0, k0), feed_b.start(t.b, m0, k0);
        auto load = [&](char *lds) { feed_a.load(left, lds), feed_b.load(left, lds + kBytesA), left -= K; };
        // (tiles behind the end are requested too, as zeros: the number of loads in flight is then always the same)
#pragma unroll
        for (int u = 0; u < STAGES - 1; ++u) load(stage(u));
        int at = 0;
        for (; at + STAGES <= tiles; at += STAGES)
#pragma unroll
            for (int u = 0; u < STAGES; ++u) {
                stage_ready<kLoads * (STAGES - 2)>();
                load(stage((u + STAGES - 1) % STAGES));
                multiply(stage(u));
            }
#pragma unroll
        for (int u = 0; u < STAGES - 1; ++u) {
            if (at + u >= tiles) break;
            stage_ready<kLoads * (STAGES - 2)>();
            load(stage((u + STAGES - 1) % STAGES));
            multiply(stage(u));
        }
    }

    // No load may still be on its way to LDS: the sums go there next, a strip of 32 rows by 64 (or 32) of the wave's columns at a time, so that they
    // come back row by row and memory is written (and a residual read) in whole lines.  Quads are permuted within a row as chunks are above.  A
    // strip's residuals are requested all at once and ahead of everything else that is done with it.
    constexpr int kGroup = FA < 2 ? 1 : 2, kQuads = 8 * kGroup, kStrip = 32 * kQuads * 16, kPerStage = kStage / kStrip;
    constexpr int kApart = 64 / kQuads, kRows = 4 / SHARE, kTurns = 32 / (kApart * kRows * SHARE);  // rows a read covers, reads a turn, turns of a wave in a strip
    constexpr int kStrips = FA / kGroup * FB;
    static_assert(FA % kGroup == 0 && kPerStage >= 1 && (WA * WB + kPerStage - 1) / kPerStage <= STAGES, "a strip for every wave");
    static_assert(SHARE == 1 || (kStrips == 1 && kPerStage >= SHARE * WA * WB), "waves that share a strip");
    const int quad = lane % kQuads, row0 = lane / kQuads + part * kTurns * kApart * kRows;
    const bool ahead = LAYER && t.e.residual && t.e.cols % 4 == 0;
    Raw4 held[kTurns][kRows];
    auto column = [&](int strip) { return n0 + wa + strip / FB * 32 * kGroup + 4 * quad; };
    auto line = [&](int strip, int turn) { return m0 + wb + strip % FB * 32 + row0 + turn * kApart * kRows; };
    auto fetch_strip = [&](int strip) {
#pragma unroll
        for (int u = 0; u < kTurns; ++u)
#pragma unroll
            for (int k = 0; k < kRows; ++k) held[u][k].template fetch<T>(t.e, line(strip, u) + k * kApart, column(strip));
    };
    if constexpr (LAYER)
        if (ahead) fetch_strip(0);
    stage_ready<0>();
    auto skew = [](int row) { return kQuads == 16 ? row & 15 : (row >> 1) & 7; };
    char *lds = stage(wave / kPerStage) + wave % kPerStage * kStrip;
    uint64_t base = 0;
    if constexpr (LAYER) base = t.e.drop.base();
    // (one copy of what is done with a strip: unrolled, the epilogue alone would fill the instruction cache)
#pragma unroll 1
    for (int strip = 0; strip < kStrips; ++strip) {
        const int64_t col = column(strip);
        const int valid = (int)(t.e.cols - col < 4 ? t.e.cols - col : 4);
        float4 bias = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if constexpr (LAYER) {
            if (t.e.bias) bias = load4(static_cast<const T *>(t.e.bias) + (valid > 0 ? col : 0), valid);
            if (ahead && strip > 0) fetch_strip(strip);
        }
        // lane l holds columns 8 (v / 4) + 4 (l / 32) + v % 4 of row l % 32
#pragma unroll
        for (int f = 0; f < kStrips; ++f) {
            if (f != strip) continue;
#pragma unroll
            for (int i = 0; i < kGroup; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float z[4];
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        z[v] = acc[f / FB * kGroup + i][f % FB][4 * q + v];
                        if constexpr (kFloat) z[v] += low[f / FB * kGroup + i][f % FB][4 * q + v];
                    }
                    const int row = lane & 31, at = 8 * i + 2 * q + (lane >> 5);
                    *reinterpret_cast<float4 *>(lds + 16 * (row * kQuads + (at ^ skew(row)))) = make_float4(z[0], z[1], z[2], z[3]);
                }
        }
        if constexpr (SHARE > 1) lds_ready();  // (one strip: nothing is written to again)
        if (valid <= 0) continue;
#pragma unroll
        for (int u = 0; u < kTurns; ++u) {
            const int64_t first = line(strip, u);
            float z[kRows][4];
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                const int r = row0 + (u * kRows + k) * kApart;
                const char *from = (SHARE > 1 ? stage0 + wave % (WA * WB) * kStrip : lds) + 16 * (r * kQuads + (quad ^ skew(r)));
                float4 v = *reinterpret_cast<const float4 *>(from);
#pragma unroll
                for (int p = 1; p < SHARE; ++p) {
                    const float4 more = *reinterpret_cast<const float4 *>(from + p * WA * WB * kStrip);
                    v.x += more.x, v.y += more.y, v.z += more.z, v.w += more.w;
                }
                if constexpr (kFloat) {
                    // (an infinite operand's parts, or leading parts that were rounded up, may have made this of a finite sum)
                    const int64_t row = first + k * kApart;
                    if ((not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w)) && row < t.e.rows)
                        v = plain_sums<A_ACROSS, B_ACROSS>(t.a, t.b, col, valid, row, k0, k1);
                }
                z[k][0] = v.x, z[k][1] = v.y, z[k][2] = v.z, z[k][3] = v.w;
            }
            if constexpr (LAYER) {
                finish_quads<T, kRows>(t.e, base, first, kApart, col, valid, z, bias, ahead ? held[u] : nullptr);
            } else {
#pragma unroll
                for (int k = 0; k < kRows; ++k) {
                    const int64_t row = first + k * kApart;
                    const float4 v = make_float4(z[k][0], z[k][1], z[k][2], z[k][3]);
                    if (row >= t.e.rows) continue;
                    if (t.partial) *reinterpret_cast<float4 *>(t.partial + ((int64_t)split * t.e.rows + row) * 4 * t.e.quads + col) = v;
                    else store4(static_cast<T *>(t.e.y) + row * t.e.y_stride + col, v, valid);
                }
            }
        }
    }
}

// y = drop(act(x W^T + b)) + residual.  The epilogue is fused: with gelu, drop and act' kept 32768 x 2048 -> 2048 bf16 takes 336 us, 59 more than the
// plain product, where a pass over memory of its own would take 100 or more.
template <class T, class S, bool WHOLE>
__global__ __launch_bounds__(S::kThreads) void linear_forward_kernel(TileArgs t)
{
    constexpr int kStage = stage_bytes<T, S>();
    __shared__ __align__(16) char stage0[kStage], stage1[kStage], stage2[S::STAGES > 2 ? kStage : 16], stage3[S::STAGES > 3 ? kStage : 16];
    compute_tile<T, false, false, S, true, WHOLE>(t, blockIdx.x, gridDim.x, stage0, stage1, stage2, stage3);
}

// out[col] = sum over n parts of part[.][col]: few columns, many parts, so a quad is shared by a quarter of the workgroup.
struct SumArgs {
    const float *part;  // [n][4 quads]
    int n;
    int64_t cols, quads;
    void *out;
};
template <class T, int THREADS>
__device__ __forceinline__ void join_sums(const SumArgs &j, int64_t block, float4 *lds)
{
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int64_t quad = block * 4 + threadIdx.x % 4;
    if (quad < j.quads) {
        const float4 *p = reinterpret_cast<const float4 *>(j.part) + quad;
#pragma unroll 4
        for (int k = threadIdx.x / 4; k < j.n; k += THREADS / 4) {
            const float4 v = p[k * j.quads];
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
    }
    // (a tree: the order of the sums is the same in every call)
    for (int o = THREADS / 2; o >= 4; o >>= 1) {
        lds[threadIdx.x] = s;
        __syncthreads();
        if ((int)threadIdx.x < o) {
            const float4 v = lds[threadIdx.x + o];
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        __syncthreads();
    }
    if (threadIdx.x >= 4 || quad >= j.quads) return;
    const int64_t left = j.cols - 4 * quad;
    store4(static_cast<T *>(j.out) + 4 * quad, s, (int)(left < 4 ? left : 4));
}

// dW = dz^T x, dx = dz W and the bias's gradient in one launch: workgroups for the longer sums start first, the last ones join the column sums that
// the kernel before this one has left.
template <class T, class S, bool WHOLE>
__global__ __launch_bounds__(S::kThreads) void linear_grads_kernel(TileArgs dw, TileArgs dx, SumArgs db, int64_t dw_blocks, int64_t dx_blocks)
{
    constexpr int kStage = stage_bytes<T, S>();
    __shared__ __align__(16) char stage0[kStage], stage1[kStage], stage2[S::STAGES > 2 ? kStage : 16], stage3[S::STAGES > 3 ? kStage : 16];
    const int64_t block = blockIdx.x, products = dw_blocks + dx_blocks, before = dx.k > dw.k_each ? dx_blocks : 0;  // dx's in front of dW's
    if (block >= products) join_sums<T, S::kThreads>(db, block - products, reinterpret_cast<float4 *>(stage0));
    else if (block >= before && block < before + dw_blocks) compute_tile<T, true, true, S, false, WHOLE>(dw, block - before, dw_blocks, stage0, stage1, stage2, stage3);
    else compute_tile<T, true, false, S, false, WHOLE>(dx, before ? block : block - dw_blocks, dx_blocks, stage0, stage1, stage2, stage3);
}

// ---- few rows --------------------------------------------------------------------------------------
// The forward pass of a few rows reads the weight once and does next to nothing with it, so what counts is how soon all of it is on its way: a
// workgroup takes 16 columns and 16 or 32 rows, its eight waves take every eighth stretch of the sum, straight from memory into the matrix
// cores' registers (fp32: by fp32 instructions), and join their sums in LDS.  Rows may lie anywhere.  Bound by the latency of a launch and of two
// loads: 1 x 1024 -> 512 bf16 3.5 us, 37 x 300 -> 200 fp32 3.4 (an empty launch takes 2).
constexpr int kFewWaves = 8;

template <class T>
struct Few;  // what a lane holds of a row for one step of kTerms terms: those from 8 (or 4) * (lane / 16) on
template <class T>
struct FewHalf {
    static constexpr int kTerms = 32, kEach = 8;
    typedef short piece __attribute__((ext_vector_type(8)));
    __device__ __forceinline__ static piece load(const T *p) { return Pack<short, 8>::load(reinterpret_cast<const short *>(p)).v; }
    __device__ __forceinline__ static piece load(const T *p, int valid)
    {
        piece v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < valid ? reinterpret_cast<const short *>(p)[e] : (short)0;
        return v;
    }
};
template <>
struct Few<bf16_t> : FewHalf<bf16_t> {
    __device__ __forceinline__ static f4 multiply(piece a, piece b, f4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Few<half_t> : FewHalf<half_t> {
    __device__ __forceinline__ static f4 multiply(piece a, piece b, f4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Few<float> {
    static constexpr int kTerms = 16, kEach = 4;
    typedef f4 piece;
    __device__ __forceinline__ static piece load(const float *p) { return Pack<float, 4>::load(p).v; }
    __device__ __forceinline__ static piece load(const float *p, int valid)
    {
        const float4 v = load4(p, valid);
        return f4{v.x, v.y, v.z, v.w};
    }
    __device__ __forceinline__ static f4 multiply(piece a, piece b, f4 c)
    {
        // (an instruction takes one term of each lane; which four terms meet in it does not matter)
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

template <class T, int MF>
__global__ __launch_bounds__(kFewWaves *kWave) void linear_few_kernel(TileArgs t)
{
    using F = Few<T>;
    constexpr int kAhead = 4;  // steps whose loads are in flight together
    __shared__ f4 sums[kFewWaves][MF][kWave];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), r = lane & 15, k0 = F::kEach * (lane >> 4);
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16 * MF;
    const int64_t n = n0 + r < t.a.extent ? n0 + r : t.a.extent - 1;  // (rows that do not exist: others, whose sums nobody asks for)
    const T *a = static_cast<const T *>(t.a.p) + n * t.a.stride + k0, *b[MF];
#pragma unroll
    for (int j = 0; j < MF; ++j) {
        const int64_t m = m0 + 16 * j + r;
        b[j] = static_cast<const T *>(t.b.p) + (m < t.b.extent ? m : t.b.extent - 1) * t.b.stride + k0;
    }
    f4 acc[MF] = {};
    const int64_t full = t.k / F::kTerms;
    int64_t s = wave;
    for (; s + (kAhead - 1) * kFewWaves < full; s += kAhead * kFewWaves) {
        typename F::piece x[kAhead], y[kAhead][MF];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t at = (s + u * kFewWaves) * F::kTerms;
            x[u] = F::load(a + at);
#pragma unroll
            for (int j = 0; j < MF; ++j) y[u][j] = F::load(b[j] + at);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int j = 0; j < MF; ++j) acc[j] = F::multiply(x[u], y[u][j], acc[j]);
    }
    for (; s < full; s += kFewWaves) {
        const typename F::piece x = F::load(a + s * F::kTerms);
#pragma unroll
        for (int j = 0; j < MF; ++j) acc[j] = F::multiply(x, F::load(b[j] + s * F::kTerms), acc[j]);
    }
    if (s == full && full * F::kTerms < t.k) {  // the wave whose turn it is takes what is left
        const int64_t at = full * F::kTerms, left = t.k - at - k0;
        const int valid = left < 0 ? 0 : (int)(left < F::kEach ? left : F::kEach);
        const typename F::piece x = F::load(a + at, valid);
#pragma unroll
        for (int j = 0; j < MF; ++j) acc[j] = F::multiply(x, F::load(b[j] + at, valid), acc[j]);
    }
#pragma unroll
    for (int j = 0; j < MF; ++j) sums[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave >= MF) return;
    // wave j finishes rows 16 j ..: lane l holds columns 4 (l / 16) .. + 3 of row l % 16
    f4 z = sums[0][wave][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) z += sums[w][wave][lane];
    const int64_t row = m0 + 16 * wave + r, col = n0 + 4 * (lane >> 4), left = t.e.cols - col;
    if (row >= t.e.rows || left <= 0) return;
    const int valid = (int)(left < 4 ? left : 4);
    float4 bias = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (t.e.bias) bias = load4(static_cast<const T *>(t.e.bias) + col, valid);
    float out[1][4] = {{z[0], z[1], z[2], z[3]}};
    finish_quads<T, 1>(t.e, t.e.drop.base(), row, 1, col, valid, out, bias, nullptr);
}

}  // namespace kge
