// mx4_rows.hpp -- products of rows of an MXFP4 matrix with a few tokens whose values keep their
// type or are MXFP8, a group of 256 terms at a time, by single waves.
//
// Both operands go to the bf16 matrix cores.  An MXFP4 value is a bf16 one, its block's code included
// (elements have 2 bits, and bf16 fp32's exponents), and so is an MXFP8 one (4 bits); dense
// values are exact sums of bf16 pieces: bf16 as they are, fp16 as 2 (8 and 3 bits), fp32 as 3 (8
// each).  So products are exact, and sums are held in fp32.  Two ends are bf16's: what of an MXFP8 value or a
// piece lies below 2^-133 is rounded to it (codes 0 to 2, whose least bits are 2^-136), and a value of 2^128
// or more, MXFP4's under codes 253 and 254 and MXFP8's from 247 on, is an infinity, behind the last term
// too, where X's zeros make it NaN; neither quantiser writes one.  (To clear such elements there took 2-3 % of
// the small calls: moe 1 x 2048 x 1024, 8 of 64, 16.4 -> 16.9 us in a graph, though no group of it is ragged.)
//   The scaled 4- and 8-bit instruction would take an eighth of the time, but it aligns the 128 terms of
// a product to their largest, and drops what lies some 2^-14 below: blocks with small scales beside
// one with a large one (1000 terms with codes 2^50 apart: off by 5e-5 of the result).
//
// v_mfma_f32_16x16x32_bf16: lane l holds terms 8 (l / 16) .. + 7 of row l % 16 of each operand; its
// result has row 4 * (l / 16) + e of the first operand and row l % 16 of the second at register e.
//
// Neighbouring lanes of a fragment are different rows, and a CU's load unit takes a cycle for each
// line that a quad of lanes meets: read straight from memory, fragments bound all of it (16 tokens x
// 8192 x 8192: 17.4 us, of which the tokens' 7.4).  So a wave loads whole runs of rows, and turns
// them round in LDS of its own; nothing there is shared, and no wave waits for another.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "layer.hpp"
#include "mx4_strip.hpp"
#include "pieces.hpp"

namespace sbx {

typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ inline __amdgpu_buffer_rsrc_t buffer_of(const uint8_t* base, int bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), (short)0, bytes, kRsrcWord3);
}

// The scale that a conversion takes for a code: its exponent field is what counts (0: 2^-127, 255: NaN).
__device__ inline float scale_of_code(uint32_t code) { return __builtin_bit_cast(float, code << 23); }

// ---- rows of MXFP4 ----

// 256 terms of 16 N rows.  In registers as loaded: 16 bytes (chunk lane % 8 of a row's 128) of rows
// 8 i + lane / 8, and the 8 codes of rows 16 i + lane % 16.
template <int N>
struct Rows4 {
    u32x4 v[2 * N];
    u32x2 code[N];
};

template <int N>
struct Source4 {
    const uint8_t *rows, *codes;
    int64_t lds;
    int bytes, count, ld, at[2 * N], lane;

    // `count_` rows of nb blocks (or 16 N of more), the first of them in `rows` and `codes`.
    __device__ inline void init(int64_t ld_, int64_t lds_, int count_, int nb, int lane_)
    {
        count = min(count_, 16 * N);
        ld = (int)ld_;
        lds = lds_;
        lane = lane_;
        bytes = strip_bytes(count, ld, nb);
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) {
            const int row = 8 * i + lane / 8;
            at[i] = row < count ? row * ld + lane % 8 * 16 : kOutside;
        }
    }

    __device__ inline void move(const uint8_t* P, const uint8_t* S, int64_t first)
    {
        rows = P + first * ld;
        codes = S + 8 * first;
    }

    // Group g, `left` blocks up to the last: zeros, not from memory, past it and past the last row
    // (a range check is certain to test the vector offset: mx4_strip.hpp).
    __device__ inline void load(Rows4<N>& d, int g, int left) const
    {
        const __amdgpu_buffer_rsrc_t v = buffer_of(rows, bytes);
        const __amdgpu_buffer_rsrc_t c = buffer_of(codes + g * lds, left > 0 ? 8 * count : 0);
        const int from = left > 0 ? 128 * g : 0;
#pragma unroll
        for (int i = 0; i < 2 * N; ++i)
            d.v[i] = __builtin_bit_cast(
                u32x4, __builtin_amdgcn_raw_buffer_load_b128(v, lane % 8 < left ? at[i] : kOutside, from, 0));
#pragma unroll
        for (int i = 0; i < N; ++i)
            d.code[i] = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_raw_buffer_load_b64(c, lane % 16 * 8 + 128 * i, 0, 0));
    }
};

// The first `left` of eight bytes, zeros for the others: codes of blocks past the last one (whose
// elements are zeros, and whose codes may be NaN's), 8-bit elements past the last term.
__device__ inline u32x2 first_bytes(u32x2 x, int left)
{
    const uint32_t lo = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << 8 * left) - 1;
    const uint32_t hi = left >= 8 ? ~0u : left <= 4 ? 0u : (1u << 8 * (left - 4)) - 1;
    return u32x2{x[0] & lo, x[1] & hi};
}

// Four lanes' blocks for the matrix cores: word b of lane group q becomes word q of block b.
__device__ inline u32x4 by_blocks(u32x4 v)
{
    auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
    auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4{c[0], c[1], d[0], d[1]};
}

__device__ inline bf16x8 values4(uint32_t word, float scale)
{
    const bf16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0),
                 v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1),
                 v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2),
                 v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3);
    return bf16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}

// Between a wave's writes to its LDS and the reads of other lanes' (and those and the next writes):
// LDS serves a wave in order, so only the compiler has to keep it.
__device__ inline void in_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// A wave's LDS for rows: 2 KiB for each 16.  Chunk c of row x lies at place c ^ (x / 2 % 8) of its
// 128 bytes: LDS serves 16 bytes a lane to lanes 0-3, 12-15 and 20-27, then to the others of 0-31,
// then to 32-63 likewise, and no two of such 16 meet in a bank.
constexpr int rows4_bytes(int n) { return 2048 * n; }

// The rows' values as fragments, a block of 32 terms each, through the wave's LDS.
template <int N>
__device__ inline void fragments(const Rows4<N>& d, char* lds, int lane, bf16x8 (&to)[N][8])
{
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
        const int row = 8 * i + lane / 8;
        *(u32x4*)(lds + row * 128 + (lane % 8 ^ row / 2 % 8) * 16) = d.v[i];
    }
    in_order();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int row = 16 * i + lane % 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u32x4 w = by_blocks(*(const u32x4*)(lds + row * 128 + (4 * h + lane / 16 ^ row / 2 % 8) * 16));
#pragma unroll
            for (int b = 0; b < 4; ++b) to[i][4 * h + b] = values4(w[b], scale_of_code(d.code[i][h] >> 8 * b & 255));
        }
    }
    in_order();
}

// ---- tokens ----

template <typename T>
constexpr int kBf16Pieces = sizeof(T) == 4 ? 3 : std::is_same<T, f16_t>::value ? 2 : 1;

// Eight values as bf16 pieces, the largest first; what is left for the last one is rounded to it (of
// 2 pieces for fp16 and 3 for fp32 nothing is lost).  An infinity's lower pieces are zeros.
template <int N>
__device__ inline void split(const float (&x)[8], bf16x8 (&to)[N])
{
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
    for (int n = 0; n + 1 < N; ++n) {
        u32x4 w;  // the upper halves of two words
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, rest[2 * i + 1]),
                                         __builtin_bit_cast(uint32_t, rest[2 * i]), 0x07060302);
        to[n] = __builtin_bit_cast(bf16x8, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float top = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, rest[i]) & 0xffff0000);
            const float left = rest[i] - top;
            rest[i] = n == 0 && __builtin_isinf(x[i]) ? 0.0f : left;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) to[N - 1][i] = (bf16_t)rest[i];
}

// 256 terms of a tile of TOKENS (2, 8 or 16) tokens: a lane loads 8 terms, 8 (lane % 32) .., of tokens
// 2 i + lane / 32, makes their pieces, and writes them to LDS.  Piece n of token t is row x = n TOKENS + t
// there, of 512 bytes, its chunk c (8 terms) at place c ^ (x % 16), for the same reason as above.
//   A fragment's 16 rows are 16 of these, pieces of a token among them: so that fp16's two of 8 tokens take
// one instruction a block, as bf16's 16 tokens do, and three of two tokens one.  Each piece has sums of its
// own, added at the end, the largest piece's first.
constexpr int tokens_bytes(int pieces, int tokens) { return 512 * pieces * tokens; }
constexpr int fragments_of(int pieces, int tokens) { return (pieces * tokens + 15) / 16; }

template <int PIECES, int TOKENS>
__device__ inline void put_tokens(char* lds, int i, int lane, const bf16x8 (&x)[PIECES], int first = 0)
{
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
        const int row = n * TOKENS + first + 2 * i + lane / 32;
        *(bf16x8*)(lds + row * 512 + (lane % 32 ^ row % 16) * 16) = x[n];
    }
}

// A block's fragment f: rows 16 f + lane % 16 (past the last: again the first ones, whose sums nobody takes).
template <int PIECES, int TOKENS>
__device__ inline bf16x8 get_tokens(const char* lds, int b, int f, int lane)
{
    constexpr int ROWS = PIECES * TOKENS;
    const int row = ROWS >= 16 * f + 16 ? 16 * f + lane % 16 : 16 * f + lane % 16 % (ROWS - 16 * f);
    return *(const bf16x8*)(lds + row * 512 + (4 * b + lane / 16 ^ row % 16) * 16);
}

// Tokens of type T: rows anywhere within 2 GiB.
template <typename T, int TOKENS>
struct DenseTokens {
    static constexpr int PIECES = kBf16Pieces<T>, PER = 8 * sizeof(T) / 16, LOADS = TOKENS / 2;
    struct Values {
        Piece<T> v[LOADS][PER];
    };
    const T* base;
    int bytes, k, at[LOADS];

    // Token t of the tile lies offset_of(t) bytes from base, or is not there (kOutside); `bytes` to the
    // last one's end.  k >= 8 terms.
    template <typename F>
    __device__ inline void init(const T* base_, int bytes_, int k_, F&& offset_of, int lane)
    {
        base = base_;
        bytes = bytes_;
        k = k_;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) at[i] = offset_of(2 * i + lane / 32);
    }
    // Group g.  A piece that reaches past the rows' end is read that much earlier (put moves it).
    __device__ inline void load(Values& d, int g, int lane) const
    {
        const __amdgpu_buffer_rsrc_t v = buffer_of((const uint8_t*)base, bytes);
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int c = min(256 * g + lane % 32 * 8 + Piece<T>::N * p, k - Piece<T>::N) * (int)sizeof(T);
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                d.v[i][p] = __builtin_bit_cast(
                    Piece<T>, __builtin_amdgcn_raw_buffer_load_b128(v, at[i] == kOutside ? kOutside : at[i] + c, 0, 0));
        }
    }
    // To LDS, as tokens first .. of a tile of TILE.
    template <int TILE = TOKENS>
    __device__ inline void put(Values& d, char* lds, int g, int lane, int first = 0) const
    {
        if (256 * g + 256 > k)
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
#pragma unroll
                for (int p = 0; p < PER; ++p)
                    trim_piece<Cut::Ragged>(d.v[i][p], 256 * g + lane % 32 * 8 + Piece<T>::N * p, k);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            bf16x8 x[PIECES];
            if constexpr (PIECES == 1)
                x[0] = __builtin_bit_cast(bf16x8, d.v[i][0]);
            else {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = (float)d.v[i][e / Piece<T>::N].v[e % Piece<T>::N];
                split(f, x);
            }
            put_tokens<PIECES, TILE>(lds, i, lane, x, first);
        }
    }
};

// Tokens that are rows of an MXFP8 matrix.
template <int TOKENS>
struct Mx8Tokens {
    static constexpr int PIECES = 1, LOADS = TOKENS / 2;
    struct Values {
        u32x2 v[LOADS];
        uint32_t code[LOADS];
    };
    const uint8_t *rows, *codes;
    int64_t lds;
    int bytes, count, ld, nb, k;

    // Rows first .. (n in all) of k terms.
    __device__ inline void init(const uint8_t* P, int64_t ld_, const uint8_t* S, int64_t lds_, int first, int n, int k_)
    {
        k = k_;
        nb = (k + 31) / 32;
        count = min(n - first, TOKENS);
        ld = (int)ld_;
        lds = lds_;
        rows = P + first * ld_;
        bytes = (count - 1) * ld + 32 * nb;
        codes = S + 8 * (int64_t)first;
    }
    // Group g: zeros past the last block and the last row.
    __device__ inline void load(Values& d, int g, int lane) const
    {
        const int left = nb - 8 * g;
        const __amdgpu_buffer_rsrc_t v = buffer_of(rows, bytes);
        const __amdgpu_buffer_rsrc_t c = buffer_of(codes + g * lds, left > 0 ? 8 * count : 0);
        const int from = left > 0 ? 256 * g : 0, block = lane % 32 / 4;  // (counts inside alone: mx4_strip.hpp)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int t = 2 * i + lane / 32;
            const bool inside = t < count && block < left;
            d.v[i] = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_raw_buffer_load_b64(v, inside ? t * ld + lane % 32 * 8 : kOutside, from, 0));
            d.code[i] = __builtin_amdgcn_raw_buffer_load_b8(c, inside ? 8 * t + block : kOutside, 0, 0);
        }
    }
    __device__ inline void put(Values& d, char* lds_, int g, int lane) const
    {
        if (256 * g + 256 > k)
#pragma unroll
            for (int i = 0; i < LOADS; ++i) d.v[i] = first_bytes(d.v[i], k - 256 * g - lane % 32 * 8);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const float scale = scale_of_code(d.code[i] & 255);
            const bf16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d.v[i][0], scale, false),
                         v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d.v[i][0], scale, true),
                         v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d.v[i][1], scale, false),
                         v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d.v[i][1], scale, true);
            const bf16x8 x[1] = {bf16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]}};
            put_tokens<1, TOKENS>(lds_, i, lane, x);
        }
    }
};

// Tokens that lie as bf16 pieces already: a piece of token t offset_of(t) bytes from its base, zeros to
// a whole group; the pieces' bases are `stride` apart.
template <int PIECES_, int TOKENS>
struct PieceTokens {
    static constexpr int PIECES = PIECES_, LOADS = TOKENS / 2;
    struct Values {
        u32x4 v[LOADS][PIECES];
    };
    const uint8_t* base;
    int64_t stride;
    int at[LOADS];

    // A token that is not there (kOutside) is not read.
    template <typename F>
    __device__ inline void move(F&& offset_of, int lane)
    {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int from = offset_of(2 * i + lane / 32);
            at[i] = from == kOutside ? kOutside : from + lane % 32 * 16;
        }
    }
    __device__ inline void load(Values& d, int g) const
    {
#pragma unroll
        for (int n = 0; n < PIECES; ++n) {
            const __amdgpu_buffer_rsrc_t v = buffer_of(base + n * stride, 0x7fffffff);
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                d.v[i][n] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(v, at[i], g * 512, 0));
        }
    }
    __device__ inline void put(const Values& d, char* lds, int lane) const
    {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            bf16x8 x[PIECES];
#pragma unroll
            for (int n = 0; n < PIECES; ++n) x[n] = __builtin_bit_cast(bf16x8, d.v[i][n]);
            put_tokens<PIECES, TOKENS>(lds, i, lane, x);
        }
    }
};

// A workgroup's barrier for what lies in LDS; loads from memory go on.
__device__ inline void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// acc[f][i]: rows 4 (lane / 16) + e of block i of w, row 16 f + lane % 16 of the tile in LDS.
template <int PIECES, int TOKENS, int N>
__device__ inline void multiply(f32x4 (&acc)[fragments_of(PIECES, TOKENS)][N], const bf16x8 (&w)[N][8], const char* lds,
                                int lane)
{
    in_order();
#pragma unroll
    for (int b = 0; b < 8; ++b)
#pragma unroll
        for (int f = 0; f < fragments_of(PIECES, TOKENS); ++f) {
            const bf16x8 x = get_tokens<PIECES, TOKENS>(lds, b, f, lane);
#pragma unroll
            for (int i = 0; i < N; ++i)
                acc[f][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i][b], x, acc[f][i], 0, 0, 0);
        }
    in_order();
}

}  // namespace sbx
