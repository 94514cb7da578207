// Matrix products of the linear layers on the matrix cores: out[m][n] = sum over k of side a (n, k) and side b (m, k).
//
// Each side lies in memory in one of two ways: ALONG rows (row = its index, the sum runs inside the row) or ACROSS them (the sum runs
// over rows, the index inside).  y = x W^T has both sides along, dx = dz W one across, dW = dz^T x both: no operand is ever transposed in
// memory.  A tile that lies across is turned by the transposing LDS reads on its way to the matrix cores.  16-bit tiles go to LDS 16 bytes a lane
// without passing through registers; fp32 ones are taken through registers, where every value becomes three bf16 parts (mfma_split.hpp), of
// whose nine products six are formed.  Rows in 8 bits go through registers too, where they become 16-bit ones (every e4m3 number times a power of two is
// one: of bf16 from 2^-130 up, of fp16 from 2^-21 to 65520; smaller ones are rounded), or, where both sides are in 8 bits, to LDS as they lie: the matrix cores take them with
// their powers.
#pragma once

#include <type_traits>

#include "features.hpp"
#include "mfma_split.hpp"
#include "rows8.hpp"

namespace kge {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef int i8v __attribute__((ext_vector_type(8)));

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

// Which sides of a product are rows in 8 bits.  kNoSideApart: neither, but side a in the arrays that another product of the launch needs for such a side.
enum Eight { kNoSide = 0, kSideA = 1, kSideB = 2, kBothSides = 3, kNoSideApart = 4 };

struct TileArgs {
    Side a, b;      // a: the columns of the output, b: its rows (one in 8 bits: its extent, and what lies in memory is in a8 or b8)
    int64_t k;      // terms of every sum
    int64_t k8;     // side b in 8 bits: pairs of terms that its rows hold, zeros behind their end among them
    int64_t k_each; // per split, a multiple of 64
    int tiles_a, tiles_b, splits;
    float *partial; // where a sum is split: [splits][rows][quads * 4] in fp32, to be joined; else NULL
    Ends e;
    Rows8 a8, b8;
};

static __device__ __align__(16) const uint32_t zero_chunk[4] = {0, 0, 0, 0};  // what chunks outside a side read

__device__ __forceinline__ void chunk_to_lds(const void *src, void *lds)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src, (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}
__device__ __forceinline__ void word_to_lds(const void *src, void *lds)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src, (__attribute__((address_space(3))) void *)lds, 4, 0, 0);
}

// eight e4m3 numbers times the power of two whose exponent byte is in bits 23 .. 30 of `power`, as 16-bit numbers
__device__ __forceinline__ s16x8 widen(uint2 q, float power, bf16_t)
{
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    const pair a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.x, power, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.x, power, true);
    const pair c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.y, power, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q.y, power, true);
    return __builtin_bit_cast(s16x8, __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ s16x8 widen(uint2 q, float power, half_t)
{
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    const pair a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q.x, power, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q.x, power, true);
    const pair c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q.y, power, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q.y, power, true);
    return __builtin_bit_cast(s16x8, __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7));
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
        typename std::conditional<ACROSS, int64_t, int>::type step[kRounds];
        int term;  // of the first chunk, within the tile (along rows of all of them: rounds are whole turns of turn())
        static_assert(ACROSS || THREADS / kRow % 16 == 0, "one term for all rounds");
        __device__ __forceinline__ int term_of(int r) const { return ACROSS ? term + r * (THREADS / kRow) : term; }

        __device__ __forceinline__ void start(const Side &s, int64_t first, int64_t k)
        {
            const E *p = static_cast<const E *>(s.p);
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int c = r * THREADS + (int)threadIdx.x, row = c / kRow, j = (c % kRow) ^ turn(row);
                const int64_t index = first + (ACROSS ? 8 * j : row);
                if (r == 0) term = ACROSS ? row : 8 * j;
                const bool there = index < s.extent;
                from[r] = there ? reinterpret_cast<const char *>(p + (ACROSS ? (k + row) * s.stride + index : index * s.stride + k + 8 * j))
                                : reinterpret_cast<const char *>(zero_chunk);
                if constexpr (ACROSS) step[r] = there ? K * s.stride * (int64_t)sizeof(E) : 0;
                else step[r] = there ? K * (int)sizeof(E) : 0;
            }
        }
        // the next tile, all of whose terms exist
        __device__ __forceinline__ void load_whole(char *lds)
        {
            const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                chunk_to_lds(from[r], lds + 16 * (r * THREADS + wave * 64));
                from[r] += step[r];
            }
        }
        // the next tile, of which `left` terms exist (none, behind the end)
        __device__ __forceinline__ void load(int64_t left, char *lds)
        {
            const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                chunk_to_lds(term_of(r) < left ? from[r] : reinterpret_cast<const char *>(zero_chunk), lds + 16 * (r * THREADS + wave * 64));
                from[r] += step[r];
            }
        }
    };

    // The same along rows, addressed with 32 bits from where the tile begins (its rows less than 2^32 bytes): an index that does not exist is another one, whose sums go
    // nowhere.
    struct NearFeed {
        const char *from;
        uint32_t at[kRounds];
        int term;
        __device__ __forceinline__ void start(const Side &s, int64_t first, int64_t k)  // (elements of 16 bits)
        {
            from = static_cast<const char *>(s.p) + 2 * (first * s.stride + k);
            const int last = (int)(s.extent - first < X ? s.extent - first : X) - 1;
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int c = r * THREADS + (int)threadIdx.x, row = c / kRow, j = (c % kRow) ^ turn(row);
                if (r == 0) term = 8 * j;
                at[r] = (uint32_t)(row < last ? row : last) * (2 * (uint32_t)s.stride) + 16 * j;
            }
        }
        __device__ __forceinline__ uint32_t offset(int r) const
        {
            uint32_t v = at[r];
            asm volatile("" : "+v"(v));  // (the compiler would hold an address of 64 bits for each)
            return v;
        }
        __device__ __forceinline__ void load_whole(char *lds)
        {
            const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
            for (int r = 0; r < kRounds; ++r) chunk_to_lds(from + offset(r), lds + 16 * (r * THREADS + wave * 64));
            from += 2 * K;
        }
        __device__ __forceinline__ void load(int64_t left, char *lds)
        {
            const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
            for (int r = 0; r < kRounds; ++r) chunk_to_lds(term < left ? from + at[r] : reinterpret_cast<const char *>(zero_chunk), lds + 16 * (r * THREADS + wave * 64));
            from += 2 * K;
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

    // The same of a side in 8 bits across rows: a chunk's eight numbers and its block's scale wait in registers, two tiles' at a time, and go to LDS as 16-bit ones.
    // Read through buffers that end with the tile's rows: what lies behind comes back as zeros, so that every load is made and none needs an address of its own.
    // (An index that does not exist may be another row's: its sums go nowhere.)
    template <class E>
    struct ByteFeed {
        static constexpr int kTurnRows = THREADS / kRow;  // rows a round covers: turn() is the same in all of them
        static_assert(ACROSS && kTurnRows % 16 == 0, "chunk j of a row is the same in every round");
        const uint8_t *q, *scale;       // of the next tile's first row
        int64_t q_step, scale_step;     // bytes of a tile's rows
        int q_whole, q_last, scale_whole, scale_last;  // bytes from there to the end of a tile's rows: of whole tiles, and of the last one
        int left;                       // tiles not requested yet
        uint32_t q_at, scale_at, q_round, scale_round;  // the lane's chunk, and how far those of its rounds are apart
        uint2 held[2][kRounds];
        int byte[2][kRounds];

        // terms: rows from k on, more than none
        __device__ __forceinline__ void start(const Rows8 &s, int64_t extent, int64_t first, int64_t k, int64_t terms, int tiles)
        {
            const int row = threadIdx.x / kRow, j = (threadIdx.x % kRow) ^ turn(row);
            q = s.q + k * s.q_stride + first, scale = s.scale + k * s.scale_stride + (first >> 5);
            q_step = K * s.q_stride, scale_step = K * s.scale_stride, left = tiles;
            const int width = (int)((extent + 31) / 32 * 32 - first), q_row = (int)s.q_stride, scale_row = (int)s.scale_stride;  // (K rows are less than 2^31)
            const int last = (int)((terms - 1) % K);
            q_whole = (K - 1) * q_row + width, q_last = last * q_row + width;
            scale_whole = (K - 1) * scale_row + width / 32, scale_last = last * scale_row + width / 32;
            q_at = row * q_row + 8 * j, scale_at = row * scale_row + (j >> 2);
            q_round = kTurnRows * q_row, scale_round = kTurnRows * scale_row;
        }
        __device__ __forceinline__ void fetch(int set)  // the next tile; behind the last one zeros
        {
            constexpr int kFormat = 0x00020000;  // raw, 32 bits an element
            const auto from = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(q), 0, left > 1 ? q_whole : (left == 1 ? q_last : 0), kFormat);
            const auto of = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(scale), 0, left > 1 ? scale_whole : (left == 1 ? scale_last : 0), kFormat);
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const u2 v = __builtin_bit_cast(u2, __builtin_amdgcn_raw_buffer_load_b64(from, q_at + r * q_round, 0, 0));
                held[set][r] = make_uint2(v[0], v[1]);
                byte[set][r] = __builtin_amdgcn_raw_buffer_load_b8(of, scale_at + r * scale_round, 0, 0);
            }
            q += q_step, scale += scale_step, --left;
        }
        __device__ __forceinline__ void put(int set, char *lds)
        {
#pragma unroll
            for (int r = 0; r < kRounds; ++r)
                *reinterpret_cast<s16x8 *>(lds + 16 * (r * THREADS + (int)threadIdx.x)) = widen(held[set][r], __int_as_float(byte[set][r] << 23), E{});
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

// 32 terms of 8 bits of an index for each lane (of a tile along rows whose elements are pairs of terms): index at + lane % 32, terms 64 step + 16 (lane / 32) .. + 15
// and 32 on from there.  The instruction's first block of 32 terms is the first half of what all lanes hold; its scale is that of lane % 32, the second's that of
// lane % 32 + 32.
template <class TILE>
__device__ __forceinline__ i8v read_eight(const char *lds, int at, int step, int lane)
{
    const int row = at + (lane & 31), j = 4 * step + (lane >> 5), turn = TILE::turn(lane & 31);
    const s16x8 lo = *reinterpret_cast<const s16x8 *>(lds + 16 * (row * TILE::kRow + (j ^ turn)));
    const s16x8 hi = *reinterpret_cast<const s16x8 *>(lds + 16 * (row * TILE::kRow + ((j + 2) ^ turn)));
    return __builtin_bit_cast(i8v, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15));
}

// 16 terms of 8 bits of an index for each lane (of such a tile): index at + lane % 32, terms 32 block + 16 (lane / 32) .. + 15; and eight of 16 bits of a tile whose
// elements are terms: chunk `chunk`.
template <class TILE>
__device__ __forceinline__ uint4 read_sixteen(const char *lds, int at, int block, int lane)
{
    const int row = at + (lane & 31), j = 2 * block + (lane >> 5);
    return *reinterpret_cast<const uint4 *>(lds + 16 * (row * TILE::kRow + (j ^ TILE::turn(lane & 31))));
}
template <class TILE>
__device__ __forceinline__ s16x8 read_chunk(const char *lds, int at, int chunk, int lane)
{
    const int row = at + (lane & 31);
    return *reinterpret_cast<const s16x8 *>(lds + 16 * (row * TILE::kRow + (chunk ^ TILE::turn(lane & 31))));
}

// The scales of a tile, a word (four blocks: 128 terms, of which a tile has all or half) an index: XA of side a, then XB of side b, then what no index asks for.
// Every thread brings in one, so that all waves have as many loads on their way.
template <int XA, int XB, int THREADS, int BLOCKS>
struct ScaleFeed {
    static_assert(XA + XB <= THREADS && (BLOCKS == 2 || BLOCKS == 4), "a word a thread");
    const uint8_t *from;
    int there;  // all ones, or 0
    __device__ __forceinline__ void start(const Rows8 &a, int64_t extent_a, int64_t n0, const Rows8 &b, int64_t extent_b, int64_t m0)
    {
        const int i = threadIdx.x;
        const bool second = i >= XA;
        const int64_t index = second ? m0 + i - XA : n0 + i;
        const bool yes = second ? i < XA + XB && index < extent_b : index < extent_a;
        from = yes ? (second ? b.scale + index * b.scale_stride : a.scale + index * a.scale_stride) : reinterpret_cast<const uint8_t *>(zero_chunk);
        there = yes ? -1 : 0;
    }
    __device__ __forceinline__ void load(int tile, bool more, char *lds)  // (behind the end: zeros)
    {
        const uint8_t *p = more ? from + (tile * BLOCKS & ~3 & there) : reinterpret_cast<const uint8_t *>(zero_chunk);
        word_to_lds(p, lds + 4 * 64 * __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6));
    }
    // where a tile's first block is in a word
    __device__ __forceinline__ static int shift(int tile) { return BLOCKS == 4 ? 0 : 16 * (tile & 1); }
};

// The scales of both sides for tiles of 128 terms in two stages: 16 bytes (512 terms, four tiles') an index at a time, a quarter of the indices with each of the four tiles before,
// so that four lanes read one line.
template <int XA, int XB, int THREADS>
struct ScaleGroups {
    static constexpr int kIndices = XA + XB, kBytes = 16 * kIndices, kOnce = kIndices < THREADS ? kIndices : THREADS;  // kOnce: words that a load brings in
    static_assert(kIndices % kOnce == 0 && XA % (kOnce / 4) == 0 && (kIndices / 4) % (kOnce / 4) == 0, "the indices of a load are all of one side");
    const uint8_t *a, *b;
    int64_t a_stride, b_stride;
    int a_last, b_last, last;  // indices and words there are, less one: what does not exist is another one, whose sums nobody asks for or whose numbers are zero
    __device__ __forceinline__ ScaleGroups(const TileArgs &t, int64_t n0, int64_t m0)
        : a(t.a8.scale + n0 * t.a8.scale_stride), b(t.b8.scale + m0 * t.b8.scale_stride), a_stride(t.a8.scale_stride), b_stride(t.b8.scale_stride),
          a_last((int)(t.a.extent - n0 < XA ? t.a.extent - n0 : XA) - 1), b_last((int)(t.b.extent - m0 < XB ? t.b.extent - m0 : XB) - 1), last((int)((t.k + 63) / 64) - 1)
    {
    }
    // part `quarter` % 4 of group `quarter` / 4, to the one of two buffers that belongs to it
    __device__ __forceinline__ void load(int quarter, char *buffers) const
    {
        const int group = quarter >> 2, part = quarter & 3, i = (int)threadIdx.x % kOnce, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) % (kOnce / 64);
        const int word = 4 * group + (i & 3);
#pragma unroll
        for (int first = 0; first < kIndices; first += kOnce) {
            const int index0 = part * (kIndices / 4) + first / 4;
            const bool second = index0 >= XA;
            const uint8_t *from = second ? b : a;
            const int64_t stride = second ? b_stride : a_stride;
            const int most = second ? b_last : a_last, index = index0 - (second ? XA : 0) + (i >> 2);
            word_to_lds(from + (uint32_t)(index < most ? index : most) * stride + 4 * (word < last ? word : last),
                        buffers + (group & 1) * kBytes + 4 * (part * kIndices + first + 64 * wave));
        }
    }
    __device__ __forceinline__ static int word(const char *buffers, int index, int tile)
    {
        return *reinterpret_cast<const int *>(buffers + (tile >> 2 & 1) * kBytes + 16 * index + 4 * (tile & 3));
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
// type.  R rows at a time, so that one's arithmetic hides another's latencies where few waves run.  ahead: the rows' residuals, or NULL.  KEEP: the bits that act' is
// kept in (16: those of the type; 0: it is not kept).
template <class T, int R, int KEEP = 16>
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
        if (KEEP > 0 && e.slope) {  // (rows of whole quads)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t row = first + r * apart, at = row * 4 * e.quads + col;
                if (row >= e.rows) continue;
                if (KEEP == 8) {
                    *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(e.slope) + at) = slopes_to_bytes(slope[4 * r], slope[4 * r + 1], slope[4 * r + 2], slope[4 * r + 3]);
                } else if (sizeof(T) == 4) {
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
template <class S, bool A>
constexpr int side_bytes() { return (A ? S::XA : S::XB) * S::K * 2; }
// Side b in 8 bits, or both (whose tiles have twice as many terms as S::K says); the scales lie behind them.
// Whether both sides' scales come in by groups (ScaleGroups): where tiles are large enough for a word an index and tile to be as many lines as the numbers are (32768 x 2048 -> 2048
// 186 us with words, 160 with groups; 65536 x 512 -> 2048 with gelu, of 128 x 128 tiles, 213 and 200).  The rows of a tile's side have to be less than 2^32 bytes, which is for the launch to see.
template <class S>
constexpr bool grouped_scales() { return S::K == 64 && S::STAGES == 2 && S::XA * S::XB >= 128 * 128; }
template <class S, Eight E>
constexpr int stage_bytes8() { return S::XA * S::K * 2 + S::XB * S::K * (E == kSideB ? 1 : 2) + (E == kBothSides && grouped_scales<S>() ? 0 : 4 * S::kThreads); }

// T: the layer's type.  LAYER: sums go through the layer's epilogue; else they are stored in its type, or as parts of split sums.  WHOLE: an fp32
// side's rows are whole quads.  EIGHT: the sides that are rows in 8 bits.  Side a goes through registers to two arrays of its own (wide0, wide1), so that its writes do
// not wait for the other's loads; side b goes to LDS as it lies, in elements that are pairs of terms (the stride of Side in pairs), and so do both (TileArgs::k in
// pairs too).
template <class T, bool A_ACROSS, bool B_ACROSS, class S, bool LAYER, bool WHOLE, Eight EIGHT = kNoSide>
__device__ __forceinline__ void compute_tile(const TileArgs &t, int64_t block, int64_t blocks, char *stage0, char *stage1, char *stage2, char *stage3,
                                             char *wide0 = nullptr, char *wide1 = nullptr, char *wide2 = nullptr, char *wide3 = nullptr)
{
    constexpr bool kFloat = sizeof(T) == 4;
    using E = typename std::conditional<kFloat, bf16_t, T>::type;
    constexpr int PLANES = kFloat ? kSplitParts : 1, K = S::K, STAGES = S::STAGES, WA = S::WA, WB = S::WB, SHARE = S::SHARE;
    using A = Tile<S::XA, K, A_ACROSS, S::kThreads>;
    using B = Tile<S::XB, EIGHT == kSideB ? K / 2 : K, B_ACROSS, S::kThreads>;  // (of a side in 8 bits that goes to LDS as it lies: elements are pairs of terms)
    constexpr int kBytesA = S::XA * K * 2, kBytesB = S::XB * K * (EIGHT == kSideB ? 1 : 2), kStage = EIGHT == kSideB ? kBytesA + kBytesB : stage_bytes<T, S>();
    constexpr bool kScales = EIGHT == kSideB || EIGHT == kBothSides;
    static_assert(EIGHT == kNoSide || (!kFloat && SHARE == 1 && (!kScales || (!A_ACROSS && !B_ACROSS)) && (!kScales || K == 64)), "sides in 8 bits");
    constexpr int FA = S::XA / WA / 32, FB = S::XB / WB / 32;
    static_assert(STAGES >= 2 && STAGES <= 4 && (!kFloat || STAGES == 2), "stages");

    constexpr bool kGrouped = EIGHT == kBothSides && grouped_scales<S>();
    constexpr bool kWideA = EIGHT == kSideA || EIGHT == kNoSideApart;
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
    auto wide = [&](int u) -> char * { return u == 0 ? wide0 : (u == 1 ? wide1 : (u == 2 ? wide2 : wide3)); };
    using Scales = ScaleFeed<EIGHT == kBothSides && !kGrouped ? S::XA : 0, S::XB, kScales ? S::kThreads : S::XA + S::XB, EIGHT == kBothSides ? 4 : 2>;
    auto multiply_steps = [&](int u, int tile, int first, int last) {
        const char *la = EIGHT == kSideA ? wide(tile & 1) : (kWideA ? wide(u) : stage(u)), *lb = kWideA ? stage(u) : la + PLANES * kBytesA;
        if constexpr (EIGHT == kSideB) {
            // (32 terms at a time: a lane's sixteen of side b are half a block, which one scale widens; side a's are read to match)
            int sb[FB];
#pragma unroll
            for (int j = 0; j < FB; ++j) sb[j] = *reinterpret_cast<const int *>(lb + kBytesB + 4 * (wb + 32 * j + (lane & 31))) >> Scales::shift(tile);
            // (where a wave has one product or two, all of a tile is read before the first of it is widened: little else hides the reads' latency)
            constexpr int kAhead = FA * FB <= 2 ? K / 32 : 1;
            static_assert(K / 32 % kAhead == 0, "whole turns");
#pragma unroll
            for (int u = 0; u < K / 32; u += kAhead) {
                s16x8 a[kAhead][FA][2];
                uint4 q[kAhead][FB];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
#pragma unroll
                    for (int j = 0; j < FB; ++j) q[k][j] = read_sixteen<B>(lb, wb + 32 * j, u + k, lane);
#pragma unroll
                    for (int i = 0; i < FA; ++i)
#pragma unroll
                        for (int v = 0; v < 2; ++v) a[k][i][v] = read_chunk<A>(la, wa + 32 * i, 4 * (u + k) + 2 * (lane >> 5) + v, lane);
                }
                if (kAhead > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    s16x8 b[FB][2];
#pragma unroll
                    for (int j = 0; j < FB; ++j) {
                        const float power = __int_as_float((sb[j] >> 8 * (u + k) & 0xFF) << 23);
                        b[j][0] = widen(make_uint2(q[k][j].x, q[k][j].y), power, E{}), b[j][1] = widen(make_uint2(q[k][j].z, q[k][j].w), power, E{});
                    }
#pragma unroll
                    for (int v = 0; v < 2; ++v)
#pragma unroll
                        for (int i = 0; i < FA; ++i)
#pragma unroll
                            for (int j = 0; j < FB; ++j) acc[i][j] = Mfma<E>::go(a[k][i][v], b[j][v], acc[i][j]);
                }
            }
            return;
        }
        if constexpr (EIGHT == kBothSides) {
            // (half a wave gives the first block's scales, the other the second's: its byte of a word is moved to where the instruction looks)
            int sa[FA], sb[FB];
            const char *scales = lb + kBytesB;
            const int shift = Scales::shift(tile) + 8 * (lane >> 5);
#pragma unroll
            for (int j = 0; j < FB; ++j) sb[j] = *reinterpret_cast<const int *>(scales + 4 * (S::XA + wb + 32 * j + (lane & 31))) >> shift;
#pragma unroll
            for (int i = 0; i < FA; ++i) sa[i] = *reinterpret_cast<const int *>(scales + 4 * (wa + 32 * i + (lane & 31))) >> shift;
#pragma unroll
            for (int u = 0; u < K / 32; ++u) {
                i8v a[FA], b[FB];
#pragma unroll
                for (int j = 0; j < FB; ++j) b[j] = read_eight<B>(lb, wb + 32 * j, u, lane);
#pragma unroll
                for (int i = 0; i < FA; ++i) a[i] = read_eight<A>(la, wa + 32 * i, u, lane);
#pragma unroll
                for (int i = 0; i < FA; ++i)
#pragma unroll
                    for (int j = 0; j < FB; ++j)
                        acc[i][j] = u == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[i], b[j], acc[i][j], 0, 0, 0, sa[i], 0, sb[j])
                                           : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[i], b[j], acc[i][j], 0, 0, 2, sa[i], 2, sb[j]);
            }
            return;
        }
#pragma unroll
        for (int u = first; u < last; ++u) {
            const int step = part * (K / 16 / SHARE) + u;
            s16x8 a[FA][PLANES], b[FB][PLANES];
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
#pragma unroll
                for (int j = 0; j < FB; ++j) b[j][p] = B::read(lb + p * kBytesB, wb + 32 * j, step, lane);
#pragma unroll
                for (int i = 0; i < FA; ++i) a[i][p] = A::read(la + p * kBytesA, wa + 32 * i, step, lane);
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
    auto multiply = [&](int u, int tile) { multiply_steps(u, tile, 0, K / 16 / SHARE); };
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
            multiply(u, 0);
        };
        int at = 0;
        for (; at + 2 <= tiles; at += 2) turn(0), turn(1);
        if (at < tiles) turn(0);
    } else if constexpr (EIGHT == kSideA) {
        // The 16-bit side is requested STAGES - 1 tiles ahead; the other one's numbers come to registers three tiles ahead and to LDS one tile ahead.  Only what the
        // turn before this one has requested may still be on its way at the barrier: the compiler, which cannot count loads to registers among those to LDS,
        // would otherwise wait for all of them before it uses a register.
        constexpr int kOut = (STAGES > 2 ? B::kRounds : 0) + 2 * A::kRounds;
        typename A::template ByteFeed<E> bytes;
        typename B::template Feed<E> feed;
        bytes.start(t.a8, t.a.extent, n0, k0, k1 - k0, tiles), feed.start(t.b, m0, k0);
        auto fetch = [&](int set) { bytes.fetch(set); };
        auto load = [&](char *lds, auto whole) {
            if constexpr (decltype(whole)::value) feed.load_whole(lds);
            else feed.load(left, lds);
            left -= K;
        };
        fetch(0);
        __builtin_amdgcn_sched_barrier(0);
        fetch(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < STAGES - 1; ++u) load(stage(u), std::false_type{});
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        bytes.put(0, wide0);
        __builtin_amdgcn_sched_barrier(0);
        fetch(0);
        __builtin_amdgcn_sched_barrier(0);
        auto in_order = [] {  // (what is still in flight is counted: no load moves in front of one that is written before it; all else may)
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0x38F);
        };
        // (the next tile is widened between the products, which it hides behind: in front of them it would keep the matrix cores waiting)
        auto turn = [&](int u, int set, auto whole) {
            __builtin_amdgcn_sched_barrier(0);
            stage_ready<kOut>();
            __builtin_amdgcn_sched_barrier(0);
            load(stage((u + STAGES - 1) % STAGES), whole);
            in_order();
            multiply_steps(u, set, 0, K / 32);
            bytes.put(1 - set, wide(1 - set));
            in_order();
            fetch(1 - set);
            in_order();
            multiply_steps(u, set, K / 32, K / 16);
        };
        constexpr int kTurns = STAGES % 2 ? 2 * STAGES : STAGES;
        int at = 0;
        for (const int whole = (int)((k1 - k0) / K); at + kTurns + STAGES - 1 <= whole; at += kTurns)  // (what is requested here are whole tiles)
#pragma unroll
            for (int u = 0; u < kTurns; ++u) turn(u % STAGES, u & 1, std::true_type{});
        for (; at + kTurns <= tiles; at += kTurns)
#pragma unroll
            for (int u = 0; u < kTurns; ++u) turn(u % STAGES, u & 1, std::false_type{});
#pragma unroll
        for (int u = 0; u < kTurns - 1; ++u) {
            if (at + u >= tiles) break;
            turn(u % STAGES, u & 1, std::false_type{});
        }
    } else if constexpr (kGrouped) {
        typename A::NearFeed feed_a;
        typename B::NearFeed feed_b;
        ScaleGroups<S::XA, S::XB, S::kThreads> scales(t, n0, m0);
        feed_a.start(t.a, n0, k0), feed_b.start(t.b, m0, k0);
        auto load = [&](int u, auto whole) {
            if constexpr (decltype(whole)::value) feed_a.load_whole(stage(u)), feed_b.load_whole(stage(u) + kBytesA);
            else feed_a.load(left, stage(u)), feed_b.load(left, stage(u) + kBytesA);
            left -= K;
        };
        int sa[FA], sb[FB];
        // (half a wave gives the first block's scales, the other the second's: its byte of a word is moved to where the instruction looks)
        auto multiply_eight = [&](int u, auto step) {
            constexpr int kStep = decltype(step)::value, kByte = 2 * kStep;
            i8v a[FA], b[FB];
#pragma unroll
            for (int j = 0; j < FB; ++j) b[j] = read_eight<B>(stage(u) + kBytesA, wb + 32 * j, kStep, lane);
#pragma unroll
            for (int i = 0; i < FA; ++i) a[i] = read_eight<A>(stage(u), wa + 32 * i, kStep, lane);
            if constexpr (kStep == 0) {
#pragma unroll
                for (int j = 0; j < FB; ++j) sb[j] >>= 8 * (lane >> 5);
#pragma unroll
                for (int i = 0; i < FA; ++i) sa[i] >>= 8 * (lane >> 5);
            }
#pragma unroll
            for (int i = 0; i < FA; ++i)
#pragma unroll
                for (int j = 0; j < FB; ++j) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[i], b[j], acc[i][j], 0, 0, kByte, sa[i], kByte, sb[j]);
        };
        if (tiles > 0)  // (a side of no terms has no scales)
            for (int q = 0; q < 4; ++q) scales.load(q, wide0);
        load(0, std::false_type{});
        // (a tile's scales are read in front of what is requested: behind it, the compiler would wait for that)
        auto turn = [&](int u, int tile, auto whole) {
            stage_ready<0>();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < FB; ++j) sb[j] = scales.word(wide0, S::XA + wb + 32 * j + (lane & 31), tile);
#pragma unroll
            for (int i = 0; i < FA; ++i) sa[i] = scales.word(wide0, wa + 32 * i + (lane & 31), tile);
            __builtin_amdgcn_sched_barrier(0);
            load(1 - u, whole);
            scales.load(tile + 4, wide0);
            multiply_eight(u, std::integral_constant<int, 0>{});
            multiply_eight(u, std::integral_constant<int, 1>{});
        };
        int at = 0;
        for (const int whole = (int)((k1 - k0) / K); at + 3 <= whole; at += 2) turn(0, at, std::true_type{}), turn(1, at + 1, std::true_type{});
        for (; at + 2 <= tiles; at += 2) turn(0, at, std::false_type{}), turn(1, at + 1, std::false_type{});
        if (at < tiles) turn(0, at, std::false_type{});
    } else {
        typename A::template Feed<E> feed_a;
        typename B::template Feed<E> feed_b;
        Scales scales;
        constexpr int kLoads = A::kRounds + B::kRounds + kScales;  // per thread and tile
        feed_a.start(t.a, n0, k0), feed_b.start(t.b, m0, k0);
        if constexpr (kScales) scales.start(t.a8, t.a.extent, n0, t.b8, t.b.extent, m0);
        int64_t left8 = t.k8;  // (side b in 8 bits: pairs of terms, of which zeros behind the row's end are some)
        int loaded = 0;
        auto load = [&](int u, auto whole) {
            char *to_a = EIGHT == kNoSideApart ? wide(u) : stage(u), *to_b = EIGHT == kNoSideApart ? stage(u) : stage(u) + kBytesA;
            if constexpr (decltype(whole)::value) feed_a.load_whole(to_a), feed_b.load_whole(to_b);
            else feed_a.load(left, to_a), feed_b.load(EIGHT == kSideB ? left8 : left, to_b);
            if constexpr (kScales) scales.load(loaded, decltype(whole)::value || loaded < tiles, stage(u) + kBytesA + kBytesB);
            if constexpr (EIGHT != kNoSide) ++loaded, left8 -= K / 2;
            left -= K;
        };
        // (tiles behind the end are requested too, as zeros: the number of loads in flight is then always the same)
#pragma unroll
        for (int u = 0; u < STAGES - 1; ++u) load(u, std::false_type{});
        int at = 0;
        if constexpr (EIGHT != kNoSide)
            for (const int whole = (int)((k1 - k0) / K); at + 2 * STAGES - 1 <= whole; at += STAGES)  // (what is requested here are whole tiles)
#pragma unroll
                for (int u = 0; u < STAGES; ++u) {
                    stage_ready<kLoads * (STAGES - 2)>();
                    load((u + STAGES - 1) % STAGES, std::true_type{});
                    multiply(u, at + u);
                }
        for (; at + STAGES <= tiles; at += STAGES)
#pragma unroll
            for (int u = 0; u < STAGES; ++u) {
                stage_ready<kLoads * (STAGES - 2)>();
                load((u + STAGES - 1) % STAGES, std::false_type{});
                multiply(u, at + u);
            }
#pragma unroll
        for (int u = 0; u < STAGES - 1; ++u) {
            if (at + u >= tiles) break;
            stage_ready<kLoads * (STAGES - 2)>();
            load((u + STAGES - 1) % STAGES, std::false_type{});
            multiply(u, at + u);
        }
    }

    // No load may still be on its way to LDS: the sums go there next, a strip of 32 rows by 64 (or 32) of the wave's columns at a time, so that they
    // come back row by row and memory is written (and a residual read) in whole lines.  Quads are permuted within a row as chunks are above.  A
    // strip's residuals are requested all at once and ahead of everything else that is done with it.
    constexpr bool kRoom = EIGHT != kSideA || WA * WB <= STAGES * (kBytesB / 8192) + 2 * (kBytesA / 8192);  // for strips of 64 columns
    constexpr int kGroup = FA < 2 || !kRoom ? 1 : 2, kQuads = 8 * kGroup, kStrip = 32 * kQuads * 16;
    constexpr int kPerStage = (kWideA ? kBytesB : kStage) / kStrip, kPerWide = kBytesA / kStrip;
    constexpr int kApart = 64 / kQuads, kRows = EIGHT == kSideB && FA * FB == 8 ? 2 : 4 / SHARE, kTurns = 32 / (kApart * kRows * SHARE);  // rows a read covers, reads a turn, turns of a wave in a strip
    constexpr int kStrips = FA / kGroup * FB;
    static_assert(FA % kGroup == 0 && kPerStage >= 1 && WA * WB <= STAGES * kPerStage + (EIGHT == kSideA ? 2 : (kWideA ? STAGES : 0)) * kPerWide, "a strip for every wave");
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
    if constexpr (kWideA)
        if (wave >= STAGES * kPerStage) lds = wide((wave - STAGES * kPerStage) / kPerWide) + (wave - STAGES * kPerStage) % kPerWide * kStrip;
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
                finish_quads<T, kRows, EIGHT == kNoSide ? 16 : (EIGHT == kBothSides ? 0 : 8)>(t.e, base, first, kApart, col, valid, z, bias, ahead ? held[u] : nullptr);
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
