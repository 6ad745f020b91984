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

namespace sbx {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kRsrcWord3 = 0x00020000;
constexpr int kOutside = (int)0x80000000u;  // an offset past every descriptor's end: reads zeros

// c += b * a^T.  As assembly, so that the sums stay where they are: given the
// builtin, the compiler moves the 256 sums of a 128 x 128 wave between registers
// (400 moves per 128 products).  It knows nothing of the unit's latency then: the
// caller keeps two instructions between a VALU write of an operand and its use here
// (there are none in the loop), and waits (settle) before it reads sums.
__device__ inline void mma(f32x4& c, i32x4 b, int code_b, i32x4 a, int code_a)
{
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                 : "+a"(c)
                 : "v"(b), "v"(a), "v"(code_b), "v"(code_a));
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

// 16 (or 4) bytes per lane from memory to LDS at `lds` + 16 (4) * lane.  As
// assembly, because the compiler makes every LDS read after the builtin wait
// for all of them; load_stage's caller waits.  They write no register.
__device__ inline void load16_lds(uint32_t lds, int voff, i32x4 rsrc, int soff)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds),
                 "v"(voff), "s"(rsrc), "s"(soff)
                 : "memory");
}
__device__ inline void load4_lds(uint32_t lds, int voff, i32x4 rsrc)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds),
                 "v"(voff), "s"(rsrc)
                 : "memory");
}
template <int N>
__device__ inline void wait_loads_and_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
    T v[8];
};

// Eight neighbouring results of a row, `left` of them inside C.
template <typename T>
__device__ inline void store8(T* c, const float (&acc)[8], int left, const Mx4GemmArgs& p)
{
    if (left >= 8) {
        Eight<T> o, in;
        if (p.beta != 0.0f) in = *(const Eight<T>*)c;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = p.alpha * acc[e];
            if (p.beta != 0.0f) v += p.beta * (float)in.v[e];
            o.v[e] = (T)(p.relu ? (v > 0.0f ? v : 0.0f) : v);
        }
        *(Eight<T>*)c = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e < left) {
                float v = p.alpha * acc[e];
                if (p.beta != 0.0f) v += p.beta * (float)c[e];
                c[e] = (T)(p.relu ? (v > 0.0f ? v : 0.0f) : v);
            }
        }
    }
}

// Tile of (32 MB) x (32 NB) of C by 2 x 2 waves of 16 MB x 16 NB, 128 terms at a
// time through a ring of four LDS stages.
//
// A stage holds the tile's rows of 64 bytes (4 blocks) and their 4 codes.  It is
// filled by loads that go straight to LDS, which place lanes' 16 bytes one after
// another: a wave's instruction fills 16 rows, and the order in which a row's four
// blocks lie is permuted by the address each lane reads instead, so that the 16
// lanes of a fragment read meet no bank twice (block b of row x at place
// b ^ swizzle(x)).
//   Stage t + 3 is asked for while t is multiplied and t + 1 is read from LDS
// into the other set of registers, so a load has two stages' time to arrive and
// neither LDS latency nor memory's is waited for.  One barrier per stage: after it,
// t + 1 is there for all waves, and all have read t, the last reader of t - 1's
// place being past its reads since before the last barrier.
//   B's block j holds the tile's rows 32 (j / 2) + 4 (j % 2) + 8 (i / 4) + i % 4 at
// its index i, so that a lane's results of blocks j, j + 1 are 8 neighbouring columns.
template <typename T, int MB, int NB>
__global__ void __launch_bounds__(256, MB * NB >= 64 ? 1 : 2) mx4_gemm_kernel(Mx4GemmArgs p, int tiles_m, int tiles_n)
{
    constexpr int BM = 32 * MB, BN = 32 * NB;
    constexpr int OFF_B = BM * 64, OFF_SA = OFF_B + BN * 64, OFF_SB = OFF_SA + BM * 4;
    constexpr int STAGE = OFF_SB + BN * 4;
    constexpr int LA = BM / 64, LB = BN / 64;            // 16-byte loads per wave and stage
    constexpr int SI = (BM + BN) / 64;                   // wave-wide loads of codes per stage
    constexpr int LS = SI >= 4 ? SI / 4 : 1;             // of them per wave (waves over SI repeat one)
    constexpr int LOADS = LA + LB + LS;
    static_assert(BM % 64 == 0 && BN % 64 == 0, "whole wave-wide loads");
    __shared__ __align__(16) char lds[4 * STAGE];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int r = lane % 16, q = lane / 16;
    // Neighbouring tiles to one XCD (workgroups are dealt to the 8 in turn), in columns of 8
    // tiles of rows: the XCD's tiles of one time share both operands in its L2.
    int id = blockIdx.x;
    const int total = tiles_m * tiles_n, per_xcd = total / 8;
    if (id < per_xcd * 8) id = id % 8 * per_xcd + id / 8;
    const int group = 8 * tiles_n, g0 = id / group * 8;
    const int gh = tiles_m - g0 < 8 ? tiles_m - g0 : 8;
    const int m0 = (g0 + id % group % gh) * BM, n0 = id % group / gh * BN;
    const int nb = (p.k + 31) / 32, nk = (nb + 3) / 4;

    const int rows_a = p.m - m0 < BM ? p.m - m0 : BM, rows_b = p.n - n0 < BN ? p.n - n0 : BN;
    i32x4 da = descriptor(p.A + (int64_t)m0 * p.lda, (int64_t)(rows_a - 1) * p.lda + 16 * nb);
    i32x4 db = descriptor(p.B + (int64_t)n0 * p.ldb, (int64_t)(rows_b - 1) * p.ldb + 16 * nb);

    // what this lane loads: a row's 16 bytes
    auto swz_a = [](int x) { return ((x >> 1 ^ x >> 3) & 1) | (x >> 1 & 2); };
    auto swz_b = [](int x) { return ((x >> 1 ^ x >> 4) & 1) | (x >> 2 & 2); };
    // (A's rows of a wave's loads are 16 apart and permuted alike, B's in two ways)
    int va[LA], vb[LB];
    const int ca = lane % 4 ^ swz_a(lane / 4);
    const int cb[2] = {lane % 4 ^ swz_b(wave * LB * 16 + lane / 4), lane % 4 ^ swz_b((wave * LB + 1) * 16 + lane / 4)};
#pragma unroll
    for (int j = 0; j < LA; ++j) va[j] = (int)(((wave * LA + j) * 16 + lane / 4) * p.lda) + ca * 16;
#pragma unroll
    for (int j = 0; j < LB; ++j) vb[j] = (int)(((wave * LB + j) * 16 + lane / 4) * p.ldb) + cb[j % 2] * 16;

    // codes: 64 rows of A or of B, their groups' addresses in turn
    uint64_t sp[LS];
    int64_t ss[LS];
    int sn[LS];
#pragma unroll
    for (int j = 0; j < LS; ++j) {
        const int i = (wave * LS + j) % SI;
        const bool b = i >= BM / 64;
        const int x = (b ? i - BM / 64 : i) * 64;
        const int left = (b ? rows_b : rows_a) - x;
        sp[j] = b ? (uint64_t)(p.SB + 8 * (int64_t)(n0 + x)) : (uint64_t)(p.SA + 8 * (int64_t)(m0 + x));
        ss[j] = b ? p.ldsb : p.ldsa;
        sn[j] = left > 0 ? 8 * left : 0;
    }

    auto load_stage = [&](int t) {  // for t = 0, 1, 2 ..
        const uint32_t at = lds0 + (t & 3) * STAGE;
        // blocks past the last one are zeros, whatever lies there
        const bool out_a = 4 * t + ca >= nb, out_b[2] = {4 * t + cb[0] >= nb, 4 * t + cb[1] >= nb};
#pragma unroll
        for (int j = 0; j < LA; ++j)
            load16_lds(at + (wave * LA + j) * 1024, out_a ? kOutside : va[j], da, t * 64);
#pragma unroll
        for (int j = 0; j < LB; ++j)
            load16_lds(at + OFF_B + (wave * LB + j) * 1024, out_b[j % 2] ? kOutside : vb[j], db, t * 64);
#pragma unroll
        for (int j = 0; j < LS; ++j) {
            const i32x4 d = {(int)(uint32_t)sp[j], (int)(uint32_t)(sp[j] >> 32) & 0xffff, t < nk ? sn[j] : 0, kRsrcWord3};
            load4_lds(at + OFF_SA + (wave * LS + j) % SI * 256, lane * 8 + t % 2 * 4, d);
            sp[j] += t & 1 ? ss[j] : 0;
        }
    };

    i32x4 fa[2][MB], fb[NB];
    int sa[2][MB], sb[NB];
    const int wm = wave % 2 * (16 * MB), wn = wave / 2 * (16 * NB);
    const int rb = r / 4 * 8 + r % 4;
    const int at_a = (wm + r) * 64 + (q ^ swz_a(r)) * 16, at_b = OFF_B + (wn + rb) * 64 + (q ^ swz_b(rb)) * 16;
    const int at_sa = OFF_SA + (wm + r) * 4 + q, at_sb = OFF_SB + (wn + rb) * 4 + q;
    auto read_a = [&](auto set, int i, const char* at) {
        constexpr int S = decltype(set)::value;
        fa[S][i] = *(const i32x4*)(at + at_a + i * 1024);
        sa[S][i] = *(const uint8_t*)(at + at_sa + i * 64);
    };
    auto read_b = [&](int j, const char* at) {
        fb[j] = *(const i32x4*)(at + at_b + j / 2 * 2048 + j % 2 * 256);
        sb[j] = *(const uint8_t*)(at + at_sb + j / 2 * 128 + j % 2 * 16);
    };
    // Codes as whole registers: without this the compiler widens them from bytes
    // at their use, too near before it (see mma).
    auto whole = [](int& code) { asm volatile("" : "+v"(code)); };
    // Codes past the last block may be NaN's: the last stage's are cleared.
    auto clear_codes = [&](int t) {
        if (t == nk - 1 && nb % 4) {
            for (int i = threadIdx.x; i < BM + BN; i += 256)
                ((uint32_t*)(lds + (t & 3) * STAGE + OFF_SA))[i] &= (1u << nb % 4 * 8) - 1;
            __syncthreads();
        }
    };

    f32x4 acc[MB][NB] = {};
    // Multiplies stage t, and reads t + 1: its A blocks into the other registers in the
    // first half of the passes, its B block j into the place of pass j's.
    auto step = [&](auto set, int t) {
        constexpr int S = decltype(set)::value;
        constexpr int PER = 2 * MB / NB;  // A blocks read in a pass
        static_assert(PER * NB == 2 * MB && NB % 2 == 0, "");
        wait_loads_and_barrier<LOADS>();
        clear_codes(t + 1);
        load_stage(t + 3);
        const char* at = lds + ((t + 1) & 3) * STAGE;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            whole(sb[j == 0 ? NB - 1 : j - 1]);  // what the pass before read
            if (j > 0 && j <= NB / 2)
#pragma unroll
                for (int i = 0; i < PER; ++i) whole(sa[1 - S][(j - 1) * PER + i]);
#pragma unroll
            for (int i = 0; i < MB; ++i) mma(acc[i][j], fb[j], sb[j], fa[S][i], sa[S][i]);
            read_b(j, at);
            if (j < NB / 2)
#pragma unroll
                for (int i = 0; i < PER; ++i) read_a(std::integral_constant<int, 1 - S>{}, j * PER + i, at);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if (nk > 0) {
        // (a descriptor that vector instructions wrote may be read 5 instructions later)
        asm volatile("s_nop 4" : "+s"(da), "+s"(db));
        load_stage(0);
        load_stage(1);
        load_stage(2);
        wait_loads_and_barrier<2 * LOADS>();
        clear_codes(0);
#pragma unroll
        for (int i = 0; i < MB; ++i) read_a(std::integral_constant<int, 0>{}, i, lds);
#pragma unroll
        for (int j = 0; j < NB; ++j) read_b(j, lds);
#pragma unroll
        for (int i = 0; i < MB; ++i) whole(sa[0][i]);
#pragma unroll
        for (int j = 0; j < NB; ++j) whole(sb[j]);
        for (int t = 0; t < nk; t += 2) {  // (of an odd number, a stage of zeros is the last)
            step(std::integral_constant<int, 0>{}, t);
            step(std::integral_constant<int, 1>{}, t + 1);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is written to LDS past the end
    }
    settle(acc);

    T* C = (T*)p.C;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int m = m0 + wm + 16 * i + r;
        if (m >= p.m) continue;
#pragma unroll
        for (int j = 0; j < NB; j += 2) {
            const int n = n0 + wn + 16 * j + 8 * q;
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = acc[i][j][e];
                v[4 + e] = acc[i][j + 1][e];
            }
            if (n < p.n) store8(C + (int64_t)m * p.ldc + n, v, p.n - n, p);
        }
    }
}

template <typename T, int MB, int NB>
hipError_t launch_tile(const Mx4GemmArgs& a, hipStream_t s)
{
    constexpr int BM = 32 * MB, BN = 32 * NB;
    const int tm = (a.m + BM - 1) / BM, tn = (a.n + BN - 1) / BN;
    if ((int64_t)tm * tn > 0x7fffffff) return hipErrorInvalidValue;
    mx4_gemm_kernel<T, MB, NB><<<(unsigned)(tm * tn), 256, 0, s>>>(a, tm, tn);
    return hipGetLastError();
}

template <typename T>
hipError_t launch(const Mx4GemmArgs& a, hipStream_t s)
{
    auto tiles = [&](int64_t b) { return (a.m + b - 1) / b * ((a.n + b - 1) / b); };
    if (tiles(256) >= 128) return launch_tile<T, 8, 8>(a, s);
    if (tiles(128) >= 128) return launch_tile<T, 4, 4>(a, s);
    return launch_tile<T, 2, 2>(a, s);
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
