// mx4_quantize.hip -- to MXFP4 (mx4.hpp) and back.
//
// A block's scale is 2^E, E = floor(log2 max|v|) - 2 (2: the exponent of e2m1's
// largest value) and not below -127; elements are v / 2^E rounded to nearest
// even and saturated at 6.  A block with an infinity or a NaN becomes NaN.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mx4.hpp"

namespace sbx {
namespace {

// The code of a block whose largest magnitude has these bits (an integer
// comparison orders magnitudes, NaN last).
__device__ inline uint32_t block_code(uint32_t top)
{
    const uint32_t e = top >> 23;
    return e >= 255 ? 255u : e > 2 ? e - 2 : 0u;
}

// The same from bits that other lanes hold too (DPP: lane ^ 1 and ^ 2; lane ^ 8 of 16).
template <int CTRL>
__device__ inline uint32_t max_dpp(uint32_t x)
{
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
    return x > y ? x : y;
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kXor8 = 0x128;

__device__ inline uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// Eight elements of a block with this code.
__device__ inline uint32_t pack8(float a, float b, float c, float d, float e, float f, float g, float h,
                                 uint32_t code)
{
    const float scale = __builtin_bit_cast(float, code << 23);  // its exponent field is what counts
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a, b, scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, c, d, scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, e, f, scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, g, h, scale, 3);
    return code == 255 ? 0 : w;
}

// Eight values of a row, from memory that is aligned to the element only.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
    T v[8];
};

// A workgroup takes 8 RPT rows by 256 columns, a lane RPT rows by 8 columns: its loads are
// 16 bytes of 16-bit values, its 8 columns of a row one call of the generator, and its column
// of 16 rows half a block.  A row's block lies in 4 neighbouring lanes, a column's in
// 32 / RPT lanes 8 apart.  One pass makes both forms; their packed elements go out as whole
// lines that the L2 gathers from the four waves (P) or that one instruction writes (PT).
// MASKED: with dropout or a gate.
template <typename T, int RPT, bool MASKED>
__global__ void __launch_bounds__(256) quantize_kernel(DropoutArgs a, Mx4Out ro, Mx4Out co, int col_tiles)
{
    constexpr int ROWS = 8 * RPT, SPAN = 32 / RPT;
    __shared__ __align__(8) uint8_t row_codes[ROWS][8];
    __shared__ __align__(4) uint8_t col_codes[256][ROWS / 32];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t tile_r = (int64_t)(blockIdx.x / col_tiles) * ROWS, tile_c = (int64_t)(blockIdx.x % col_tiles) * 256;
    const int64_t r0 = tile_r + lane / 8 * RPT, c0 = tile_c + wave * 64 + lane % 8 * 8;
    const int64_t nb_r = (a.cols + 31) / 32, nb_c = (a.rows + 31) / 32;  // blocks of a row, of a column

    float v[RPT][8];
    if (tile_r + ROWS <= a.rows && tile_c + wave * 64 + 64 <= a.cols) {
        Eight<T> x[RPT];
#pragma unroll
        for (int i = 0; i < RPT; ++i) x[i] = *(const Eight<T>*)((const T*)a.X + (r0 + i) * a.ldx + c0);
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = (float)x[i].v[e];
        if (MASKED && a.gate) {
            Eight<T> g[RPT];
#pragma unroll
            for (int i = 0; i < RPT; ++i) g[i] = *(const Eight<T>*)((const T*)a.gate + (r0 + i) * a.ldg + c0);
#pragma unroll
            for (int i = 0; i < RPT; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = (float)g[i].v[e] > 0.0f ? v[i][e] : 0.0f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[i][e] = 0.0f;
                if (r0 + i < a.rows && c0 + e < a.cols) {
                    v[i][e] = (float)((const T*)a.X)[(r0 + i) * a.ldx + c0 + e];
                    if (MASKED && a.gate && !((float)((const T*)a.gate)[(r0 + i) * a.ldg + c0 + e] > 0.0f))
                        v[i][e] = 0.0f;
                }
            }
    }
    if (MASKED && a.threshold) {
        const float scale = (float)a.scale;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const uint32_t keep = keep_bits(a, (uint32_t)(r0 + i), (uint32_t)(c0 / 8));
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = keep >> e & 1 ? v[i][e] * scale : 0.0f;
        }
    }

    if (ro.P) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[i][e]));
            const uint32_t code = block_code(max_dpp<kXor2>(max_dpp<kXor1>(top)));
            const uint32_t w = pack8(v[i][0], v[i][1], v[i][2], v[i][3], v[i][4], v[i][5], v[i][6], v[i][7], code);
            if (r0 + i < a.rows && c0 < 32 * nb_r) *(uint32_t*)(ro.P + (r0 + i) * ro.ldp + c0 / 2) = w;
            if (lane % 4 == 0) row_codes[lane / 8 * RPT + i][wave * 2 + lane % 8 / 4] = (uint8_t)code;
        }
    }
    if (co.P) {
        typedef typename std::conditional<RPT == 16, uint2, uint16_t>::type part_t;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < RPT; ++i) top = max(top, magnitude(v[i][e]));
            top = max_dpp<kXor8>(top);
            if (SPAN == 8) {
                top = max(top, (uint32_t)__shfl_xor((int)top, 16));
                top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            }
            const uint32_t code = block_code(top);
            part_t w;
            if constexpr (RPT == 16) {
                w.x = pack8(v[0][e], v[1][e], v[2][e], v[3][e], v[4][e], v[5][e], v[6][e], v[7][e], code);
                w.y = pack8(v[8][e], v[9][e], v[10][e], v[11][e], v[12][e], v[13][e], v[14][e], v[15][e], code);
            } else {
                w = (part_t)pack8(v[0][e], v[1][e], v[2][e], v[3][e], 0, 0, 0, 0, code);
            }
            if (c0 + e < a.cols && r0 < 32 * nb_c) *(part_t*)(co.P + (c0 + e) * co.ldp + r0 / 2) = w;
            if (lane / 8 % SPAN == 0) col_codes[wave * 64 + lane % 8 * 8 + e][lane / 8 / SPAN] = (uint8_t)code;
        }
    }
    __syncthreads();
    // 8 codes of a row, ROWS / 32 of a column; those past the last block are 0, and so are all of a
    // tile past the last row, there to complete a column's group
    if (ro.P && threadIdx.x < ROWS && tile_r + threadIdx.x < a.rows)
        *(uint2*)(ro.S + tile_c / 256 * ro.lds + (tile_r + threadIdx.x) * 8) = *(const uint2*)row_codes[threadIdx.x];
    if (co.P && tile_c + threadIdx.x < a.cols) {
        uint8_t* s = co.S + tile_r / 256 * co.lds + (tile_c + threadIdx.x) * 8 + tile_r / 32 % 8;
        if constexpr (ROWS == 128) *(uint32_t*)s = *(const uint32_t*)col_codes[threadIdx.x];
        else *s = col_codes[threadIdx.x][0];
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

template <typename T, int RPT>
hipError_t quantize_by(const DropoutArgs& a, const Mx4Out& rows, const Mx4Out& cols, hipStream_t s)
{
    // whole groups of 256 rows where the columns' codes are wanted: each is written to its end
    const int64_t r = cols.P ? (a.rows + 255) / 256 * 256 : a.rows;
    const int64_t rt = (r + 8 * RPT - 1) / (8 * RPT), ct = (a.cols + 255) / 256;
    if (rt * ct > 0x7fffffff) return hipErrorInvalidValue;
    if (a.threshold || a.gate)
        quantize_kernel<T, RPT, true><<<(unsigned)(rt * ct), 256, 0, s>>>(a, rows, cols, (int)ct);
    else
        quantize_kernel<T, RPT, false><<<(unsigned)(rt * ct), 256, 0, s>>>(a, rows, cols, (int)ct);
    return hipGetLastError();
}

template <typename T>
hipError_t quantize(const DropoutArgs& a, const Mx4Out& rows, const Mx4Out& cols, hipStream_t s)
{
    return a.rows * a.cols >= (int64_t)4 << 20 ? quantize_by<T, 16>(a, rows, cols, s)
                                               : quantize_by<T, 4>(a, rows, cols, s);
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
