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

typedef float f32x2 __attribute__((ext_vector_type(2)));

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

// The scale a conversion takes: its exponent field is what counts (0: 2^-127).
__device__ inline float scale_of(uint32_t code) { return __builtin_bit_cast(float, code << 23); }

constexpr int RPT = 4, ROWS = 8 * RPT;  // rows of a lane, of a workgroup

// Eight values of a row, from memory that is aligned to the element only.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
    T v[8];
};

// The lane's rows of 8 values; past an edge, values from the nearest place inside.
template <typename T>
__device__ inline void load_rows(Eight<T> (&x)[RPT], const void* X, int64_t ld, int64_t r0, int64_t c0,
                                 bool whole, const DropoutArgs& a)
{
    if (whole) {  // (the wave's 64 columns are inside)
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int64_t r = r0 + i < a.rows ? r0 + i : a.rows - 1;
            x[i] = *(const Eight<T>*)((const T*)X + r * ld + c0);
        }
    } else {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int64_t r = r0 + i < a.rows ? r0 + i : a.rows - 1;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[i].v[e] = ((const T*)X)[r * ld + (c0 + e < a.cols ? c0 + e : a.cols - 1)];
            __builtin_amdgcn_sched_barrier(0);  // (a row at a time: addresses take registers)
        }
    }
}

// A workgroup takes 32 rows by 256 columns, a lane 4 rows (RPT) by 8 columns: its loads are
// 16 bytes of 16-bit values, and its 8 columns of a row one call of the generator.  A row's
// block lies in 4 neighbouring lanes, a column's in 8 lanes 8 apart, so one pass over X makes
// both forms in registers.  What leaves in small pieces (4 bytes of P, 2 of PT a lane) the L2
// gathers into lines.  MASKED: with dropout or a gate.
//   Bound by HBM where X is large: 8192^2 bf16, both forms, 35.5 us for 205 MB (5.8 TB/s);
// 8 or 16 rows a lane store larger pieces but leave fewer waves (34.9 and 37.0 us; with
// dropout and gate 73.0, 73.2 and 112 us).
template <typename T, bool MASKED>
__global__ void __launch_bounds__(256) quantize_kernel(DropoutArgs a, Mx4Out ro, Mx4Out co, int col_tiles)
{
    __shared__ __align__(8) uint8_t row_codes[ROWS][8];
    __shared__ uint8_t col_codes[256];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t tile_r = (int64_t)(blockIdx.x / col_tiles) * ROWS, tile_c = (int64_t)(blockIdx.x % col_tiles) * 256;
    const int64_t r0 = tile_r + lane / 8 * RPT, c0 = tile_c + wave * 64 + lane % 8 * 8;
    const int64_t nb_r = (a.cols + 31) / 32, nb_c = (a.rows + 31) / 32;  // blocks of a row, of a column

    Eight<T> x[RPT], g[RPT];
    const bool whole = tile_c + wave * 64 + 64 <= a.cols;
    load_rows<T>(x, a.X, a.ldx, r0, c0, whole, a);
    if (MASKED && a.gate) load_rows<T>(g, a.gate, a.ldg, r0, c0, whole, a);
    uint32_t keep[RPT][4];  // (made while the loads are on their way)
    if (MASKED && a.threshold) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) keep_words(a, (uint32_t)(r0 + i), (uint32_t)(c0 / 8), keep[i]);
    }
    float v[RPT][8];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = (float)x[i].v[e];
    if (MASKED && a.threshold) {
        const float scale = (float)a.scale;
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = kept(a, keep[i], e) ? v[i][e] * scale : 0.0f;
    }
    if (MASKED && a.gate) {
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = (float)g[i].v[e] > 0.0f ? v[i][e] : 0.0f;
    }
    if (tile_r + ROWS > a.rows || tile_c + 256 > a.cols) {  // zeros outside
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = r0 + i < a.rows && c0 + e < a.cols ? v[i][e] : 0.0f;
    }

    if (ro.P) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[i][e]));
            const uint32_t code = block_code(max_dpp<kXor2>(max_dpp<kXor1>(top)));
            const float scale = scale_of(code);
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][0], v[i][1], scale, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][2], v[i][3], scale, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][4], v[i][5], scale, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][6], v[i][7], scale, 3);
            if (code == 255) w = 0;
            if (r0 + i < a.rows && c0 < 32 * nb_r) *(uint32_t*)(ro.P + (r0 + i) * ro.ldp + c0 / 2) = w;
            if (lane % 4 == 0) row_codes[lane / 8 * RPT + i][wave * 2 + lane % 8 / 4] = (uint8_t)code;
        }
    }
    if (co.P) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < RPT; ++i) top = max(top, magnitude(v[i][e]));
            top = max_dpp<kXor8>(top);
            top = max(top, (uint32_t)__shfl_xor((int)top, 16));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            const uint32_t code = block_code(top);
            const float scale = scale_of(code);
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0][e], v[1][e], scale, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2][e], v[3][e], scale, 1);
            if (c0 + e < a.cols && r0 < 32 * nb_c)
                *(uint16_t*)(co.P + (c0 + e) * co.ldp + r0 / 2) = (uint16_t)(code == 255 ? 0 : w);
            if (lane < 8) col_codes[wave * 64 + lane * 8 + e] = (uint8_t)code;
        }
    }
    __syncthreads();
    // 8 codes of a row, one of a column; those past the last block are 0, and so are all of a
    // tile past the last row, there to complete a column's group
    if (ro.P && threadIdx.x < ROWS && tile_r + threadIdx.x < a.rows)
        *(uint2*)(ro.S + tile_c / 256 * ro.lds + (tile_r + threadIdx.x) * 8) = *(const uint2*)row_codes[threadIdx.x];
    if (co.P && tile_c + threadIdx.x < a.cols)
        co.S[tile_r / 256 * co.lds + (tile_c + threadIdx.x) * 8 + tile_r / 32 % 8] = col_codes[threadIdx.x];
}

// Threads form TX chunks of 8 columns by 256 / TX rows, kRows times.
constexpr int kRows = 4;

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp,
                                                         const uint8_t* S, int64_t lds, T* Y, int64_t ldy, int tx,
                                                         int col_tiles)
{
    const int64_t c0 = ((int64_t)(blockIdx.x % col_tiles) * tx + threadIdx.x % tx) * 8;
    const int per = 256 / tx;
    const int64_t r0 = (int64_t)(blockIdx.x / col_tiles) * (per * kRows) + threadIdx.x / tx;
    if (c0 >= cols) return;
    uint32_t w[kRows], code[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int64_t r = r0 + i * per < rows ? r0 + i * per : rows - 1;  // (a row past the last is not stored)
        w[i] = *(const uint32_t*)(P + r * ldp + c0 / 2);
        code[i] = S[c0 / 256 * lds + r * 8 + c0 / 32 % 8];
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int64_t r = r0 + i * per;
        if (r >= rows) break;
        const float scale = scale_of(code[i]);
        f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 0),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 1),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 2),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 3)};
        Eight<T> y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y.v[e] = (T)(code[i] == 255 ? __builtin_nanf("") : v[e / 2][e % 2]);
        T* to = Y + r * ldy + c0;
        if (c0 + 8 <= cols)
            *(Eight<T>*)to = y;
        else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c0 + e < cols) to[e] = y.v[e];
    }
}

template <typename T>
hipError_t quantize(const DropoutArgs& a, const Mx4Out& rows, const Mx4Out& cols, hipStream_t s)
{
    // whole groups of 256 rows where the columns' codes are wanted: each is written to its end
    const int64_t r = cols.P ? (a.rows + 255) / 256 * 256 : a.rows;
    const int64_t rt = (r + ROWS - 1) / ROWS, ct = (a.cols + 255) / 256;
    if (rt * ct > 0x7fffffff) return hipErrorInvalidValue;
    if (a.threshold || a.gate)
        quantize_kernel<T, true><<<(unsigned)(rt * ct), 256, 0, s>>>(a, rows, cols, (int)ct);
    else
        quantize_kernel<T, false><<<(unsigned)(rt * ct), 256, 0, s>>>(a, rows, cols, (int)ct);
    return hipGetLastError();
}

template <typename T>
hipError_t dequantize(int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp, const uint8_t* S,
                      int64_t lds, void* Y, int64_t ldy, hipStream_t s)
{
    const int64_t chunks = (cols + 7) / 8;
    int tx = 1;
    while (tx < 256 && tx < chunks) tx *= 2;
    const int64_t ct = (chunks + tx - 1) / tx, rt = (rows + 256 / tx * kRows - 1) / (256 / tx * kRows);
    if (rt * ct > 0x7fffffff) return hipErrorInvalidValue;
    dequantize_kernel<T><<<(unsigned)(rt * ct), 256, 0, s>>>(rows, cols, P, ldp, S, lds, (T*)Y, ldy, tx, (int)ct);
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
