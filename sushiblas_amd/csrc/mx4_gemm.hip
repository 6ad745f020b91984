// mx4_gemm.hip -- C = alpha * A * B^T + beta * C of two MXFP4 matrices (mx4.hpp).
//
// v_mfma_scale_f32_16x16x128: lane l holds row l % 16 of its operand and the
// 32 elements of block l / 16 of four, with the block's code in a byte of
// another register; products are exact and sums are held in fp32.  Its result
// has row 4 * (l / 16) + i of A and row l % 16 of B at register i.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx4.hpp"

namespace sbx {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Registers of one 16-row operand block for 128 elements: its row's 32 of them
// and their code, zeros outside the matrix.
struct Frag {
    i32x4 v;
    int code;
};

__device__ inline Frag load_frag(const uint8_t* P, int64_t ldp, const uint8_t* S, int64_t lds,
                                 int row, int rows, int b, int nb)
{
    Frag f{{0, 0, 0, 0}, 0};
    if (row < rows && b < nb) {
        f.v = *(const i32x4*)(P + row * ldp + (int64_t)b * 16);
        f.code = S[b / 8 * lds + (int64_t)row * 8 + b % 8];
    }
    return f;
}

__device__ inline i32x8 widen(i32x4 v)
{
    return i32x8{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
}

// 64 x 64 of C per workgroup, 32 x 32 per wave, operands straight from memory.
template <typename T>
__global__ void __launch_bounds__(256) mx4_gemm_kernel(Mx4GemmArgs p)
{
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int r = lane % 16, q = lane / 16;
    const int tiles_m = (p.m + 63) / 64;
    const int m0 = (int)(blockIdx.x % tiles_m) * 64 + wave % 2 * 32;
    const int n0 = (int)(blockIdx.x / tiles_m) * 64 + wave / 2 * 32;
    const int nb = (p.k + 31) / 32;
    f32x4 acc[2][2] = {};
    for (int b = 0; b < nb; b += 4) {
        Frag fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fa[i] = load_frag(p.A, p.lda, p.SA, p.ldsa, m0 + 16 * i + r, p.m, b + q, nb);
            fb[i] = load_frag(p.B, p.ldb, p.SB, p.ldsb, n0 + 16 * i + r, p.n, b + q, nb);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    widen(fa[i].v), widen(fb[j].v), acc[i][j], 4, 4, 0, fa[i].code, 0, fb[j].code);
    }
    T* C = (T*)p.C;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int m = m0 + 16 * i + 4 * q + e, n = n0 + 16 * j + r;
                if (m >= p.m || n >= p.n) continue;
                T* c = C + (int64_t)m * p.ldc + n;
                float v = p.alpha * acc[i][j][e];
                if (p.beta != 0.0f) v += p.beta * (float)*c;
                *c = (T)(p.relu ? (v > 0.0f ? v : 0.0f) : v);
            }
}

template <typename T>
hipError_t launch(const Mx4GemmArgs& a, hipStream_t s)
{
    const int64_t tiles = ((int64_t)a.m + 63) / 64 * (((int64_t)a.n + 63) / 64);
    mx4_gemm_kernel<T><<<(unsigned)tiles, 256, 0, s>>>(a);
    return hipGetLastError();
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
