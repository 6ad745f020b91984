// mx4_quantize.hip -- to MXFP4 (mx4.hpp) and back.
//
// A block's scale is 2^E, E = floor(log2 max|v|) - 2 (2: the exponent of e2m1's
// largest value) and not below -127; elements are v / 2^E rounded to nearest
// even and saturated at 6.  A block with an infinity or a NaN becomes NaN.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx4.hpp"

namespace sbx {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The code of a block whose largest magnitude has these bits (an integer
// comparison orders magnitudes, NaN last).
__device__ inline uint32_t block_code(uint32_t top)
{
    const uint32_t e = top >> 23;
    return e >= 255 ? 255u : e > 2 ? e - 2 : 0u;
}

__device__ inline u32x4 pack_block(const float (&v)[32], uint32_t code)
{
    u32x4 out = {0, 0, 0, 0};
    if (code == 255) return out;
    const float scale = __builtin_bit_cast(float, code << 23);  // its exponent field is what counts
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * i], v[8 * i + 1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * i + 2], v[8 * i + 3], scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * i + 4], v[8 * i + 5], scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * i + 6], v[8 * i + 7], scale, 3);
        out[i] = w;
    }
    return out;
}

// The value at (row, col) that is quantised, 0 outside the matrix.
template <typename T>
__device__ inline float value(const DropoutArgs& a, int64_t row, int64_t col)
{
    if (row >= a.rows || col >= a.cols) return 0.0f;
    float x = (float)((const T*)a.X)[row * a.ldx + col];
    if (a.threshold) {
        const uint32_t keep = keep_bits(a, (uint32_t)row, (uint32_t)(col / 8));
        x = keep >> (col % 8) & 1 ? x * (float)a.scale : 0.0f;
    }
    if (a.gate && !((float)((const T*)a.gate)[row * a.ldg + col] > 0.0f)) x = 0.0f;
    return x;
}

// One thread per block: TURN, of the transpose.
template <typename T, bool TURN>
__global__ void __launch_bounds__(256) quantize_kernel(DropoutArgs a, Mx4Out o)
{
    const int64_t nr = TURN ? a.cols : a.rows, nk = TURN ? a.rows : a.cols;
    const int64_t nb = (nk + 31) / 32, groups = (nb + 7) / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nr * groups * 8;
         i += (int64_t)gridDim.x * 256) {
        const int64_t r = i % nr, b = i / nr;
        float v[32];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            v[j] = TURN ? value<T>(a, b * 32 + j, r) : value<T>(a, r, b * 32 + j);
            const uint32_t m = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;
            top = top > m ? top : m;
        }
        const uint32_t code = block_code(top);
        if (b < nb) *(u32x4*)(o.P + r * o.ldp + b * 16) = pack_block(v, code);
        o.S[b / 8 * o.lds + r * 8 + b % 8] = (uint8_t)code;  // past the last block: 0
    }
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(int64_t rows, int64_t cols, const uint8_t* P,
                                                         int64_t ldp, const uint8_t* S, int64_t lds,
                                                         T* Y, int64_t ldy)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols;
         i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / cols, c = i % cols, b = c / 32;
        const uint32_t n = P[r * ldp + c / 2] >> (c % 2 * 4) & 15;
        const uint32_t code = S[b / 8 * lds + r * 8 + b % 8];
        const uint32_t e = n >> 1 & 3, f = n & 1;
        // (2 + f) 2^(e - 2), or f 2^-1 without the implicit bit
        float v = e ? (float)(2 + f) * (float)(1 << (e - 1)) * 0.5f : (float)f * 0.5f;
        v = n & 8 ? -v : v;
        Y[r * ldy + c] = (T)(code == 255 ? __builtin_nanf("") : ldexpf(v, (int)code - 127));
    }
}

unsigned blocks_of(int64_t items)
{
    const int64_t b = (items + 255) / 256;
    return (unsigned)(b > 16384 ? 16384 : b < 1 ? 1 : b);
}

template <typename T>
hipError_t quantize(const DropoutArgs& a, const Mx4Out& rows, const Mx4Out& cols, hipStream_t s)
{
    auto items = [](int64_t nr, int64_t nk) { return nr * ((nk + 255) / 256) * 8; };
    if (rows.P) quantize_kernel<T, false><<<blocks_of(items(a.rows, a.cols)), 256, 0, s>>>(a, rows);
    if (cols.P) quantize_kernel<T, true><<<blocks_of(items(a.cols, a.rows)), 256, 0, s>>>(a, cols);
    return hipGetLastError();
}

template <typename T>
hipError_t dequantize(int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp, const uint8_t* S,
                      int64_t lds, void* Y, int64_t ldy, hipStream_t s)
{
    dequantize_kernel<T><<<blocks_of(rows * cols), 256, 0, s>>>(rows, cols, P, ldp, S, lds, (T*)Y, ldy);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mx4_quantize(int dtype, const DropoutArgs& a, const Mx4Out& rows,
                               const Mx4Out& cols, hipStream_t s)
{
    switch (dtype) {
    case 0: return quantize<float>(a, rows, cols, s);
    case 2: return quantize<bf16_t>(a, rows, cols, s);
    default: return quantize<f16_t>(a, rows, cols, s);
    }
}

hipError_t launch_mx4_dequantize(int dtype, int64_t rows, int64_t cols, const uint8_t* P,
                                 int64_t ldp, const uint8_t* S, int64_t lds, void* Y, int64_t ldy,
                                 hipStream_t s)
{
    switch (dtype) {
    case 0: return dequantize<float>(rows, cols, P, ldp, S, lds, Y, ldy, s);
    case 2: return dequantize<bf16_t>(rows, cols, P, ldp, S, lds, Y, ldy, s);
    default: return dequantize<f16_t>(rows, cols, P, ldp, S, lds, Y, ldy, s);
    }
}

}  // namespace sbx
