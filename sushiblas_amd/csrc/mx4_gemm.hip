// mx4_gemm.hip -- C = alpha * A * B^T + beta * C of two MXFP4 matrices (mx4.hpp).
//
// v_mfma_scale_f32_16x16x128: lane l holds row l % 16 of its operand and the
// 32 elements of block l / 16 of four, with the block's code in a byte of
// another register; products are exact and sums are held in fp32.  Its result
// has row 4 * (l / 16) + e of the first operand and row l % 16 of the second
// at register e.  B is given first, so a lane holds neighbouring columns of C.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mx4.hpp"
#include "mx4_plan.hpp"
#include "mx4_strip.hpp"

namespace sbx {
namespace {

// c += b * a^T, with byte H of the codes.  As assembly, so that the sums stay
// where they are: given the builtin, the compiler moves the 256 sums of a 128 x 128
// wave between registers (400 moves per 128 products).  It knows nothing of the
// unit's latency then: the caller keeps two instructions between a VALU write of an
// operand and its use here, and waits (settle) before it reads sums.
template <int H>
__device__ inline void mma(f32x4& c, i32x4 b, int code_b, i32x4 a, int code_a)
{
    if constexpr (H == 0)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+a"(c)
                     : "v"(b), "v"(a), "v"(code_b), "v"(code_a));
    else
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] "
                     "cbsz:4 blgp:4"
                     : "+a"(c)
                     : "v"(b), "v"(a), "v"(code_b), "v"(code_a));
}

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ inline i32x8 widen(i32x4 v)
{
    return i32x8{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
}

template <int MB, int NB>
__device__ inline void settle(f32x4 (&acc)[MB][NB])
{
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) asm volatile("" : "+a"(acc[i][j]));
}

// A buffer descriptor in scalar registers.
__device__ inline i32x4 descriptor(const uint8_t* base, int64_t bytes)
{
    const uint64_t at = (uint64_t)base;
    i32x4 d;
    d[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)at);
    d[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32) & 0xffff);
    d[2] = __builtin_amdgcn_readfirstlane((int)(bytes < 0 ? 0 : bytes));
    d[3] = kRsrcWord3;
    return d;
}

// Loads 16 bytes per lane straight to LDS, to `lds` + 16 * lane.  As assembly, because
// the compiler makes every LDS read after the builtin wait for all such loads; the caller
// waits.  It writes no register.
__device__ inline void load_lds(uint32_t lds, int voff, i32x4 rsrc, int soff)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds),
                 "v"(voff), "s"(rsrc), "s"(soff)
                 : "memory", "m0");
}
template <int N>
__device__ inline void wait_loads_and_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// 16 bytes of results, from or to memory that is aligned to the element only.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[16 / sizeof(T)];
};

template <typename T>
__device__ inline T result(float acc, float c, const Mx4GemmArgs& p)
{
    const float v = p.beta != 0.0f ? p.alpha * acc + p.beta * c : p.alpha * acc;
    return (T)(p.relu ? (v > 0.0f ? v : 0.0f) : v);
}

// A piece of neighbouring results of a row, `left` (or none) of them inside C, which is at c.
template <typename T>
__device__ inline Vec<T> finish(const float (&acc)[16 / sizeof(T)], const T* c, int left, const Mx4GemmArgs& p)
{
    constexpr int V = 16 / sizeof(T);
    Vec<T> o, in = {};
    if (p.beta != 0.0f) {
        if (left >= V)
            in = *(const Vec<T>*)c;
        else
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e < left) in.v[e] = c[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) o.v[e] = result<T>(acc[e], (float)in.v[e], p);
    return o;
}

template <typename T>
__device__ inline void store(T* c, const Vec<T>& o, int left, const Mx4GemmArgs& p)
{
    constexpr int V = 16 / sizeof(T);
    if (left >= V) {
        // Rows of whole 64 bytes go past the L2s, that keep the operands then (8192^2 x 512 to bf16
        // 60.5 -> 55.1 us, 4096^2 x 1024 23.4 -> 16.7 us); of others an L2 has to put the pieces
        // together (4095 x 3001 x 2047 to fp32 27.7 us, past them 38.4).
        typedef u32x4 __attribute__((aligned(2))) loose_t;
        if (p.past)
            __builtin_nontemporal_store(__builtin_bit_cast(u32x4, o), (loose_t*)c);
        else
            *(Vec<T>*)c = o;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < left) c[e] = o.v[e];
    }
}

// Tile of BM x BN = (16 MB WM) x (16 NB WN) of C by WM x WN waves of 16 MB x 16 NB,
// 256 terms at a time through NS LDS stages; KG groups of such waves share the terms.
//
// A stage holds the tile's rows of 128 bytes (8 blocks, a cache line) and their 8 codes.
// It is filled by loads that go straight to LDS, which place lanes' 16 bytes one after
// another: a wave's instruction fills 8 rows, and the order in which a row's blocks lie
// is permuted by the address each lane reads instead: block b of row x at place
// b ^ swizzle(x).  LDS has 64 banks, and serves 16 bytes a lane to lanes 0-3, 12-15,
// 20-27, then to the others of 0-31, then 32-63 likewise; with the swizzles below no
// two of such 16 lanes of a fragment read meet (SQ_LDS_BANK_CONFLICT: 8 % of the LDS
// cycles, one for each read of codes, which are 2 bytes a lane).
//   A stage is multiplied in two halves; lane group q takes block 2q + h of a row in
// half h, so its codes for both are one 16-bit read.
//   While a half is multiplied, the next is read from LDS: A's block i into its own
// place once the pass over it is done, B's blocks into a second set.  Between the
// halves of stage t every wave has read all of it: a barrier there frees its place for
// t + 2, and sees t + 1 arrived, asked for a whole stage's time before.
//   B's block j holds the tile's rows 16 G (j / G) + 4 (j % G) + 4 G (i / 4) + i % 4 at
// its index i (G: 2, or all 3 blocks), so that a lane's results of G blocks are 4 G
// neighbouring columns.
//   What bounds it.  8192^3 to bf16, 237-257 us (4.3-4.6 PFLOP/s; these products
// straight from registers 8.66, which is 2.07 GHz): without loads and LDS reads 166 us, at 2.08 GHz
// with the matrix units 76 % busy -- each round's first stage and C's way out are not hidden; with
// them power holds 1.82-1.9 GHz and the units are 57 % busy, beside the operands' way from the L2s
// (2.6 GB, 10 TB/s).  A
// stage's loads asked for at once 290 us against 284 spread, results straight from the registers
// 284 against 261, reads of a pass in a row 261 against 256; four waves of 128 x 128 527 against
// 503 us at 16384 terms.
// 4096 x 1024 x 4096 on 128^2 tiles 15.2-16.9 us: a stage 0.57 us, its products alone 0.25, its
// LDS reads 0.29, both without the loads 0.48-0.51: LDS and the matrix units, which overlap in part.
// 4095 x 3001 x 2047 to fp32 22.9-25.0 us: C, 49 MB in rows that no line begins with (of 3004
// columns 22.5).  512^3 to fp32 4.6: launch, the first stage's way, C's.
template <typename T, int WM, int WN, int KG, int MB, int NB, int NS>
__global__ void __launch_bounds__(64 * WM * WN * KG, 2) mx4_gemm_kernel(Mx4GemmArgs p, int tiles_m, int tiles_n)
{
    constexpr int WAVES = WM * WN, BM = 16 * MB * WM, BN = 16 * NB * WN;
    constexpr int CA = (BM + 127) / 128 * 1024, CB = (BN + 127) / 128 * 1024;  // codes
    constexpr int OFF_B = BM * 128, OFF_SA = OFF_B + BN * 128, OFF_SB = OFF_SA + CA;
    constexpr int STAGE = OFF_SB + CB;
    constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;  // loads per wave and stage
    constexpr int NCA = CA / 1024, NC = NCA + CB / 1024;     // of codes, one by each of the first waves
    constexpr int PER_PASS = (LA + LB + MB - 1) / MB;
    static_assert(LA * 8 * WAVES == BM && LB * 8 * WAVES == BN && NC <= WAVES, "whole wave-wide loads");
    static_assert(MB >= NB && (NB % 2 == 0 || NB == 3), "");
    constexpr int GB = NB % 2 ? NB : 2;  // blocks of B that interleave
    __shared__ __align__(16) char lds_all[KG * NS * STAGE];
    const int lane = threadIdx.x % 64, wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int kg = wave_all / WAVES, wave = wave_all % WAVES;  // group, and wave of the group
    const int r = lane % 16, q = lane / 16;
    char* lds = lds_all + kg * NS * STAGE;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds_all + kg * NS * STAGE;
    // Neighbouring tiles to one XCD (workgroups are dealt to the 8 in turn), in columns of 8
    // tiles of rows: the XCD's tiles of one time share both operands in its L2.
    int id = blockIdx.x;
    const int total = tiles_m * tiles_n, per_xcd = total / 8;
    if (id < per_xcd * 8) id = id % 8 * per_xcd + id / 8;
    const int group = 8 * tiles_n, g0 = id / group * 8;
    const int gh = tiles_m - g0 < 8 ? tiles_m - g0 : 8;
    const int m0 = (g0 + id % group % gh) * BM, n0 = id % group / gh * BN;
    const int nb = (p.k + 31) / 32, nk = (nb + 8 * KG - 1) / (8 * KG);  // stages of a group

    const int rows_a = p.m - m0 < BM ? p.m - m0 : BM, rows_b = p.n - n0 < BN ? p.n - n0 : BN;
    i32x4 da = descriptor(p.A + (int64_t)m0 * p.lda, (int64_t)(rows_a - 1) * p.lda + 16 * nb);
    i32x4 db = descriptor(p.B + (int64_t)n0 * p.ldb, (int64_t)(rows_b - 1) * p.ldb + 16 * nb);

    // what this lane loads: 16 bytes of a row (rows past the operand's end lie past the
    // descriptor's); the swizzles of rows 8 apart are alike or two
    auto swz_a = [](int x) { return (x >> 1 & 1) ^ (x & 8 ? 6 : 0); };
    auto swz_b = [](int x) { return (x >> 1 & 1) ^ (x % (16 * GB) >= 8 * GB ? 6 : 0); };
    int va[LA], vb[LB], ca[LA], cb[LB];
#pragma unroll
    for (int j = 0; j < LA; ++j) {
        const int x = (wave * LA + j) * 8 + lane / 8;
        ca[j] = lane % 8 ^ swz_a(x);
        va[j] = (int)(x * p.lda) + ca[j] * 16;
    }
#pragma unroll
    for (int j = 0; j < LB; ++j) {
        const int x = (wave * LB + j) * 8 + lane / 8;
        cb[j] = lane % 8 ^ swz_b(x);
        vb[j] = (int)(x * p.ldb) + cb[j] * 16;
    }
    // and codes: the first NC waves, 128 rows of A or of B each
    const bool code_b = wave >= NCA;
    const int code_row = (code_b ? wave - NCA : wave) * 128;
    const int code_left = (code_b ? rows_b : rows_a) - code_row;
    const uint8_t* code_at = code_b ? p.SB + 8 * (int64_t)(n0 + code_row) : p.SA + 8 * (int64_t)(m0 + code_row);
    const int64_t code_step = code_b ? p.ldsb : p.ldsa;
    code_at += kg * code_step;

    // Load x < LA + LB of stage t; the codes go with the last.  Blocks past the last one,
    // and all of a stage past the last, are zeros, whatever lies there.
    auto load_part = [&](int t, int x) {
        const uint32_t at = lds0 + t % NS * STAGE;
        const int tk = t * KG + kg, left = nb - 8 * tk;
        const int from = min(tk, (nb - 1) / 8) * 128;  // (counts inside alone: mx4_strip.hpp)
        if (x < LA)
            load_lds(at + (wave * LA + x) * 1024, ca[x % LA] < left ? va[x % LA] : kOutside, da, from);
        else
            load_lds(at + OFF_B + (wave * LB + x - LA) * 1024, cb[(x - LA) % LB] < left ? vb[(x - LA) % LB] : kOutside,
                     db, from);
        if (x == LA + LB - 1 && wave < NC) {
            const uint64_t s = (uint64_t)code_at;
            const int n = left <= 0 || code_left <= 0 ? 0 : code_left > 128 ? 1024 : 8 * code_left;
            load_lds(at + OFF_SA + wave * 1024, lane * 16,
                     i32x4{(int)(uint32_t)s, (int)(uint32_t)(s >> 32) & 0xffff, n, kRsrcWord3}, 0);
            code_at += KG * code_step;
        }
    };
    // Codes past the last block may be NaN's: the last stage's are cleared.
    auto clear_codes = [&](int t) {
        if (t == nk - 1 && nb % 8) {
            const uint64_t mask = (1ull << nb % 8 * 8) - 1;
            if (nb / 8 == t * KG + kg)
                for (int i = threadIdx.x % (64 * WAVES); i < (CA + CB) / 8; i += 64 * WAVES)
                    ((uint64_t*)(lds + t % NS * STAGE + OFF_SA))[i] &= mask;
            __syncthreads();
        }
    };

    i32x4 fa[MB], fb[2][NB];
    int sa[MB], sb[NB], sb_next[NB];
    const int wm = wave % WM * (16 * MB), wn = wave / WM * (16 * NB);
    const int rb = r / 4 * (4 * GB) + r % 4;
    int at_a[2], at_b[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        at_a[h] = (wm + r) * 128 + (2 * q + h ^ swz_a(r)) * 16;
        at_b[h] = OFF_B + (wn + rb) * 128 + (2 * q + h ^ swz_b(rb)) * 16;
    }
    const int at_sa = OFF_SA + (wm + r) * 8 + 2 * q, at_sb = OFF_SB + (wn + rb) * 8 + 2 * q;
    auto read_a = [&](auto half, int i, const char* at) {
        fa[i] = *(const i32x4*)(at + at_a[decltype(half)::value] + i * 2048);
    };
    auto read_b = [&](auto half, int j, const char* at) {
        constexpr int H = decltype(half)::value;
        fb[H][j] = *(const i32x4*)(at + at_b[H] + j / GB * (GB * 2048) + j % GB * 512);
    };
    auto read_sa = [&](int i, const char* at) { sa[i] = *(const uint16_t*)(at + at_sa + i * 128); };
    auto read_sb = [&](int j, const char* at) {
        sb_next[j] = *(const uint16_t*)(at + at_sb + j / GB * (GB * 128) + j % GB * 32);
    };
    // Codes as whole registers: without this the compiler widens them at their use, too
    // near before it (see mma).
    auto whole = [](int& code) { asm volatile("" : "+v"(code)); };
    constexpr std::integral_constant<int, 0> first{};
    constexpr std::integral_constant<int, 1> second{};

    f32x4 acc[MB][NB] = {};
    // Multiplies half H of a stage and reads the next half, from the stage at `at`.
    // beside(i): what else goes with pass i.  Reads begin after the first pass (so A's block
    // i is read a pass later than its place is free).
    auto multiply = [&](auto half, const char* at, auto&& beside) {
        constexpr int H = decltype(half)::value;
        constexpr std::integral_constant<int, 1 - H> next{};
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            if (i > 2 && H == 1) {  // codes read two passes before
                whole(sa[i - 3]);
                if (i - 3 < NB) whole(sb_next[i - 3]);
            }
            // one instruction of the reads after each product: a wave issues in order, and what
            // comes in a row keeps the matrix unit waiting
            const int x0 = i - 1, x1 = i == MB - 1 ? i : i - 1;  // A's blocks read in this pass
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                mma<H>(acc[i][j], fb[H][j], sb[j], fa[i], sa[i]);
                if (i == 0) {
                    if (j == 0) beside(i);
                } else {
                    if (j == 0) read_a(next, x0, at);
                    if (j == (NB > 2 ? 1 : 0) && H == 1) read_sa(x0, at);
                    if (j == NB / 2 && x0 < NB) read_b(next, x0, at);
                    if (j == NB - 1 && x0 < NB && H == 1) read_sb(x0, at);
                    if (j == NB - 1 && x1 > x0) {
                        read_a(next, x1, at);
                        if (H == 1) read_sa(x1, at);
                        if (x1 < NB) {
                            read_b(next, x1, at);
                            if (H == 1) read_sb(x1, at);
                        }
                    }
                    if (j == NB - 1) beside(i);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (H == 1) {
#pragma unroll
            for (int i = MB - 3 > 0 ? MB - 3 : 0; i < MB; ++i) whole(sa[i]);
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                whole(sb_next[j]);
                sb[j] = sb_next[j];
                whole(sb[j]);
            }
            asm volatile("s_nop 1");
        }
    };

    if (nk > 0) {
        // (a descriptor that vector instructions wrote may be read 5 instructions later)
        asm volatile("s_nop 4" : "+s"(da), "+s"(db));
#pragma unroll
        for (int x = 0; x < NS * (LA + LB); ++x) load_part(x / (LA + LB), x % (LA + LB));
        wait_loads_and_barrier<(NS - 1) * (LA + LB)>();  // (the waves that load codes wait for more)
        clear_codes(0);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            read_a(first, i, lds);
            read_sa(i, lds);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            read_b(first, j, lds);
            read_sb(j, lds);
        }
#pragma unroll
        for (int i = 0; i < MB; ++i) whole(sa[i]);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            sb[j] = sb_next[j];
            whole(sb[j]);
        }
        asm volatile("s_nop 1");
        for (int t = 0; t < nk; ++t) {
            multiply(first, lds + t % NS * STAGE, [](int) {});
            // (after the last stage: what lies there)
            multiply(second, lds + (t + 1) % NS * STAGE, [&](int i) {
                if (i == 0) {
                    wait_loads_and_barrier<(NS - 2) * (LA + LB)>();
                    clear_codes(t + 1);
                }
                // spread over the passes: a wave that asks for all of them at once waits its
                // turn at the CU's one load unit instead of multiplying
#pragma unroll
                for (int x = i * PER_PASS; x < (i + 1) * PER_PASS && x < LA + LB; ++x) load_part(t + NS, x);
            });
        }
        wait_loads_and_barrier<0>();  // nothing more is written to LDS
    }
    settle(acc);

    // The groups' sums: each takes over half of the rows, and gives the others'.
    constexpr int MINE = MB / KG;
    if constexpr (KG == 2) {
        f32x4* trade = (f32x4*)lds_all;
        static_assert(WAVES * MB * NB * 64 * 16 <= KG * NS * STAGE, "");
#pragma unroll
        for (int i = 0; i < MINE; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j)
                trade[((kg * WAVES + wave) * MINE + i) * NB * 64 + j * 64 + lane] = kg ? acc[i][j] : acc[MINE + i][j];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MINE; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j)
                acc[i][j] = (kg ? acc[MINE + i][j] : acc[i][j]) +
                            trade[(((1 - kg) * WAVES + wave) * MINE + i) * NB * 64 + j * 64 + lane];
        __syncthreads();
    }
    constexpr int V = 16 / sizeof(T), COLS = 16 * NB, PITCH = COLS + 4;
    constexpr int PER_ROW = COLS / V, PIECES = 16 * PER_ROW;
    // Out through LDS, 16 rows of the wave's at a time, so that an instruction stores whole
    // rows of them (from the registers it would store 32 columns of 16 rows).  Neighbouring lanes
    // store neighbouring pieces of a row; where those of fp32 are not aligned, the same piece of
    // neighbouring rows instead: 3001 x 4095 x 2047 24.5 us in place of 32.0, 4095^2 x 1000 23.7
    // in place of 34.1, 2047 x 2049 x 512 11.6 and 10.8.  Not for 16 bits (4095^2 x 1000 28.7
    // against 23.3), nor for C's that the MALL does not hold (8191^2 x 500 128 against 105).
    static_assert(2 * 16 * PITCH * 4 * WAVES <= NS * STAGE, "");
    float* out = (float*)lds_all + wave_all * 2 * 16 * PITCH;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        float* half = out + i % 2 * 16 * PITCH;
#pragma unroll
        for (int j = 0; j < NB; ++j)
            *(f32x4*)(half + r * PITCH + j / GB * (16 * GB) + 4 * GB * q + j % GB * 4) = acc[i][j];
#pragma unroll
        for (int x = 0; x < PIECES; x += 64) {
            const int piece = PIECES % 64 && x + lane >= PIECES ? PIECES - 1 : x + lane;
            int row = piece / PER_ROW, col = piece % PER_ROW * V;
            if (V == 4 && p.down) {
                constexpr int ROWS = PER_ROW % 8 ? 16 : 8;  // by 64 / ROWS pieces an instruction
                row = x / 64 * ROWS % 16 + lane % ROWS;
                col = (x / 64 * ROWS / 16 * (64 / ROWS) + lane / ROWS) * V;
            }
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = half[row * PITCH + col + e];
            const int m = m0 + wm + 16 * (kg * MINE + i) + row, n = n0 + wn + col;
            if (x + lane < PIECES && m < p.m) {
                T* c = (T*)p.C + (int64_t)m * p.ldc + n;
                store(c, finish<T>(v, c, p.n - n, p), p.n - n, p);
            }
        }
    }
}

// Products with a narrow operand Y (a few tokens, or the columns of a narrow C) and any number of
// rows of the wide one X (XA: A, else B), or with a small C over many terms (mx4_plan.hpp): a
// workgroup takes 16 XB rows of X and all of Y, its eight waves each an eighth of the terms, in
// groups of 256 by turns, straight from memory to registers (a lane's 32 neighbouring bytes of a
// row; the group after is under way meanwhile).  The waves' sums are added up in LDS, in order.
//   Bound by memory: 1 x 8192 x 8192 (36 MB) 8.4 us, 9.8 a call with the launch between, 1 x 28672
// x 8192 27 us (4.6 TB/s; a copy reaches 5.2).  Blocks of 64 neighbouring bytes an instruction, in
// place of 32 a lane, took as long.
constexpr int kSkinnyWaves = 8;

template <int N>
struct Group {
    i32x4 v[N][2];
    int code[N];  // two codes in its low bytes
};

// The rows of an operand that a workgroup takes, and the lane's place in them (mx4_strip.hpp).
template <int N>
struct Strip {
    const uint8_t *rows, *codes;
    int64_t lds;
    int bytes, count, ld, lane, at[N], code_at;

    __device__ inline void init(const uint8_t* P, int64_t ld_, const uint8_t* S, int64_t lds_, int first, int n,
                                int nb, int lane_)
    {
        count = min(n - first, 16 * N);
        ld = (int)ld_;
        lds = lds_;
        lane = lane_;
        rows = P + first * ld_;
        bytes = strip_bytes(count, ld, nb);
        codes = S + 8 * (int64_t)first;
#pragma unroll
        for (int i = 0; i < N; ++i) at[i] = strip_lane(lane, i, count, ld);
        code_at = lane % 16 * 8 + lane / 16 * 2;
    }

    // Group g (256 terms), with `left` blocks up to the last: zeros, not from memory, past it
    // and past the last row.  The codes of a group's 8 blocks are all there.
    __device__ inline void load(Group<N>& d, int g, int left) const
    {
        const __amdgpu_buffer_rsrc_t v =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(rows), (short)0, bytes, kRsrcWord3);
        const __amdgpu_buffer_rsrc_t c = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(codes) + g * lds, (short)0, left > 0 ? 8 * count : 0, kRsrcWord3);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int from = strip_scalar(i, g, count, ld, left);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                d.v[i][h] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                          v, strip_vector(at[i], lane, h, left), from, 0));
            d.code[i] = __builtin_amdgcn_raw_buffer_load_b16(c, code_at + 128 * i, 0, 0);
        }
    }
};

// Codes past the last block may be NaN's and are cleared (the elements there are zeros):
// `mine` of the lane's two blocks are inside.
template <int N>
__device__ inline void clip(Group<N>& d, int mine)
{
#pragma unroll
    for (int i = 0; i < N; ++i) d.code[i] = mine >= 2 ? d.code[i] : mine == 1 ? d.code[i] & 0xff : 0;
}

template <typename T, int YB, int XB, bool XA>
__global__ void __launch_bounds__(64 * kSkinnyWaves, YB * XB >= 4 ? 2 : 4) mx4_skinny_kernel(Mx4GemmArgs p)
{
    const int nx = XA ? p.m : p.n, ny = XA ? p.n : p.m;
    constexpr int PITCH = 16 * YB + 4;
    __shared__ float part[kSkinnyWaves][16 * PITCH];

    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int r = lane % 16, q = lane / 16;
    const int x0 = block_x() * (16 * XB), y0 = blockIdx.y * (16 * YB);
    if (x0 >= nx) return;
    const int nb = (p.k + 31) / 32, groups = (nb + 7) / 8;
    Strip<XB> sx;
    Strip<YB> sy;
    sx.init(XA ? p.A : p.B, XA ? p.lda : p.ldb, XA ? p.SA : p.SB, XA ? p.ldsa : p.ldsb, x0, nx, nb, lane);
    sy.init(XA ? p.B : p.A, XA ? p.ldb : p.lda, XA ? p.SB : p.SA, XA ? p.ldsb : p.ldsa, y0, ny, nb, lane);

    f32x4 acc[XB][YB] = {};
    auto load = [&](Group<XB>& x, Group<YB>& y, int g) {
        sx.load(x, g, nb - 8 * g);
        sy.load(y, g, nb - 8 * g);
    };
    auto multiply = [&](Group<XB>& x, Group<YB>& y, int g) {
        const int left = nb - 8 * g;
        if (left < 8) {
            clip(x, left - 2 * q);
            clip(y, left - 2 * q);
        }
#pragma unroll
        for (int i = 0; i < XB; ++i)
#pragma unroll
            for (int j = 0; j < YB; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    widen(x.v[i][0]), widen(y.v[j][0]), acc[i][j], 4, 4, 0, x.code[i], 0, y.code[j]);
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    widen(x.v[i][1]), widen(y.v[j][1]), acc[i][j], 4, 4, 1, x.code[i], 1, y.code[j]);
            }
    };
    // (no branch around loads, also past the last group: the compiler would wait for all of them)
    constexpr int W = kSkinnyWaves;
    Group<XB> x0g, x1g;
    Group<YB> y0g, y1g;
    load(x0g, y0g, wave);
    for (int g = wave; g < groups; g += 2 * W) {
        load(x1g, y1g, g + W);
        multiply(x0g, y0g, g);
        load(x0g, y0g, g + 2 * W);
        multiply(x1g, y1g, g + W);
    }
    T* C = (T*)p.C;
#pragma unroll
    for (int i = 0; i < XB; ++i) {
        if (i > 0) __syncthreads();
#pragma unroll
        for (int j = 0; j < YB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[wave][(4 * q + e) * PITCH + 16 * j + r] = acc[i][j][e];
        __syncthreads();
        for (int t = threadIdx.x; t < 16 * 16 * YB; t += 64 * kSkinnyWaves) {
            const int dx = XA ? t / (16 * YB) : t % 16, dy = XA ? t % (16 * YB) : t / 16;  // C's rows run along n
            const int xr = x0 + 16 * i + dx;
            if (xr >= nx || y0 + dy >= ny) continue;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kSkinnyWaves; ++w) v += part[w][dx * PITCH + dy];
            T* c = C + (XA ? (int64_t)xr * p.ldc + y0 + dy : (int64_t)(y0 + dy) * p.ldc + xr);
            *c = result<T>(v, p.beta != 0.0f ? (float)*c : 0.0f, p);
        }
    }
}

template <typename T, int YB, int XB>
hipError_t launch_skinny(const Mx4GemmArgs& a, hipStream_t s)
{
    auto grid = [](int x, int y) {
        return grid_of((x + 16 * XB - 1) / (16 * XB), (unsigned)((y + 16 * YB - 1) / (16 * YB)));
    };
    if (a.m <= a.n)
        mx4_skinny_kernel<T, YB, XB, false><<<grid(a.n, a.m), 64 * kSkinnyWaves, 0, s>>>(a);
    else
        mx4_skinny_kernel<T, YB, XB, true><<<grid(a.m, a.n), 64 * kSkinnyWaves, 0, s>>>(a);
    return hipGetLastError();
}

template <typename T, int WM, int WN, int KG, int MB, int NB, int NS>
hipError_t launch_tile(const Mx4GemmArgs& a, hipStream_t s)
{
    constexpr int BM = 16 * MB * WM, BN = 16 * NB * WN;
    const int tm = (a.m + BM - 1) / BM, tn = (a.n + BN - 1) / BN;
    if ((int64_t)tm * tn * (64 * WM * WN * KG) > kMaxThreads) return hipErrorNotSupported;
    mx4_gemm_kernel<T, WM, WN, KG, MB, NB, NS><<<(unsigned)(tm * tn), 64 * WM * WN * KG, 0, s>>>(a, tm, tn);
    return hipGetLastError();
}

template <typename T>
hipError_t launch(const Mx4GemmArgs& a, hipStream_t s)
{
    switch (mx4_kernel(a.m, a.n, a.k)) {
    case Mx4Kernel::Narrow2: return launch_skinny<T, 1, 2>(a, s);
    case Mx4Kernel::Narrow: return launch_skinny<T, 1, 1>(a, s);
    case Mx4Kernel::Tile64: return launch_tile<T, 2, 2, 1, 2, 2, 2>(a, s);
    case Mx4Kernel::Tile64Groups: return launch_tile<T, 2, 2, 2, 2, 2, 4>(a, s);
    case Mx4Kernel::Tile128Stages: return launch_tile<T, 2, 4, 1, 4, 2, 4>(a, s);
    case Mx4Kernel::Tile128: return launch_tile<T, 2, 2, 1, 4, 4, 2>(a, s);
    case Mx4Kernel::Tile256x192: return launch_tile<T, 2, 4, 1, 8, 3, 2>(a, s);
    case Mx4Kernel::Tile192x256: return launch_tile<T, 2, 4, 1, 6, 4, 2>(a, s);
    case Mx4Kernel::Tile256: return launch_tile<T, 2, 4, 1, 8, 4, 2>(a, s);
    default: return hipErrorNotSupported;
    }
}

}  // namespace

hipError_t launch_mx4_gemm(int dtype, const Mx4GemmArgs& a, hipStream_t s)
{
    switch (dtype) {
    case 0: return launch<float>(a, s);
    case 2: return launch<bf16_t>(a, s);
    default: return launch<f16_t>(a, s);
    }
}

}  // namespace sbx
