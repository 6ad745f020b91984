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

typedef float f32x2 __attribute__((ext_vector_type(2)));

// The code of a block whose largest magnitude has these bits.
__device__ inline uint32_t block_code(uint32_t top)
{
    const uint32_t e = top >> 23;
    return e == 255 ? 255u : __builtin_elementwise_sub_sat(e, 2u);
}

// The larger magnitude, NaN if there is one.
__device__ inline float larger(float a, float b) { return __builtin_elementwise_maximum(fabsf(a), fabsf(b)); }

// The larger bits (magnitudes are in integer order, NaN last) of two lanes.
template <int CTRL>
__device__ inline uint32_t max_dpp(uint32_t x, uint32_t other)
{
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)other, CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kXor8 = 0x128;  // DPP: lane ^ 1, ^ 2, ^ 8 of 16

// The scale a conversion takes: its exponent field is what counts (0: 2^-127).
__device__ inline float scale_of(uint32_t code) { return __builtin_bit_cast(float, code << 23); }

constexpr int RPT = 4;     // rows of a lane
constexpr int TILE = 128;  // rows and columns of a workgroup

// The lane's rows of 8 values; past an edge, values from the nearest place inside.
template <typename T>
__device__ inline void load_rows(Eight<T> (&x)[RPT], const void* X, int64_t ld, int64_t r0, int64_t c0,
                                 bool inside, bool whole, const DropoutArgs& a)
{
    if (inside) {
        const T* from = (const T*)X + r0 * ld + c0;
#pragma unroll
        for (int i = 0; i < RPT; ++i) x[i] = *(const Eight<T>*)(from + i * ld);
    } else if (whole) {  // (the wave's 64 columns are inside)
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

// A workgroup takes 128 by 128 values, a wave 32 rows by 64 columns, a lane 4 rows (RPT) by 8
// columns: its loads are 16 bytes of 16-bit values, and its 8 columns of a row one call of the
// generator.  A row's block lies in 4 neighbouring lanes, a column's in 8 lanes 8 apart, so one
// pass over X makes both forms in registers.  They are gathered in LDS and leave 64 bytes of a
// row at a time, past the L2s.
//   Bound by HBM: 8192^2 bf16 33-37 us to both forms (205 MB, 5.5-6.2 TB/s), 25.5-27.1 to the rows'
// alone (170 MB, 6.3-6.7 TB/s), 25.7-26.1 to the columns', fp32 53, 44 and 45; stored through the L2s 45.9 and 33.7 us, straight from the lanes (4 bytes of
// P, 2 of PT each: the L2s take as long for a request of 16 bytes as for one of 64) 53.2 and 34.8.
// With dropout and gate 57.3 us, the generator's and the selects' VALU work beside.
template <typename T, bool DROP, bool GATE>
__global__ void __launch_bounds__(512, 4) quantize_kernel(DropoutArgs a, Mx4Out ro, Mx4Out co, int col_tiles)
{
    const uint32_t tile = block_x();  // (those past the last row's store nothing)
    constexpr int PITCH_P = 72, PITCH_PT = 68;  // (no bank is met twice by a wave's writes)
    __shared__ uint32_t row_codes[TILE], col_codes[TILE];
    __shared__ __align__(8) uint8_t row_elems[TILE * PITCH_P];
    __shared__ __align__(4) uint8_t col_elems[TILE * PITCH_PT];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t tile_r = (int64_t)(tile / col_tiles) * TILE, tile_c = (int64_t)(tile % col_tiles) * TILE;
    const int rl = wave / 2 * 32 + lane / 8 * RPT, cl = wave % 2 * 64 + lane % 8 * 8;  // in the tile
    const int64_t r0 = tile_r + rl, c0 = tile_c + cl;

    Eight<T> x[RPT], g[RPT];
    const bool inside = tile_r + TILE <= a.rows && tile_c + TILE <= a.cols;
    const bool whole = tile_c + wave % 2 * 64 + 64 <= a.cols;
    load_rows<T>(x, a.X, a.ldx, r0, c0, inside, whole, a);
    if (GATE) load_rows<T>(g, a.gate, a.ldg, r0, c0, inside, whole, a);
    float v[RPT][8];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        uint32_t keep[4];
        if (DROP) keep_words(a, (uint32_t)(r0 + i), (uint32_t)(c0 / 8), keep);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[i][e] = (float)x[i].v[e];
            if (DROP) v[i][e] *= (float)a.scale;
            if (DROP || GATE)
                v[i][e] = (!DROP || kept(a, keep, e)) && (!GATE || (float)g[i].v[e] > 0.0f) ? v[i][e] : 0.0f;
        }
    }
    if (!inside) {  // zeros outside
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = r0 + i < a.rows && c0 + e < a.cols ? v[i][e] : 0.0f;
    }

    if (ro.P) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const float top = larger(larger(larger(v[i][0], v[i][1]), larger(v[i][2], v[i][3])),
                                     larger(larger(v[i][4], v[i][5]), larger(v[i][6], v[i][7])));
            uint32_t bits = __builtin_bit_cast(uint32_t, top);
            bits = max_dpp<kXor1>(bits, bits);
            bits = max_dpp<kXor2>(bits, bits);
            const uint32_t code = block_code(bits);
            const float scale = scale_of(code);
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][0], v[i][1], scale, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][2], v[i][3], scale, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][4], v[i][5], scale, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[i][6], v[i][7], scale, 3);
            w = code == 255 ? 0 : w;
            *(uint32_t*)(row_elems + (rl + i) * PITCH_P + cl / 2) = w;
            ((uint8_t*)(row_codes + rl + i))[cl / 32] = (uint8_t)code;  // (by four lanes)
        }
    }
    if (co.P) {
        // The columns' largest: 8 of 4 rows in each lane; lanes 32, 16 and 8 apart trade halves
        // of theirs until each has one column's of all 32 rows.
        uint32_t t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            t[e] = __builtin_bit_cast(uint32_t, larger(larger(v[0][e], v[1][e]), larger(v[2][e], v[3][e])));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const auto x = __builtin_amdgcn_permlane32_swap(t[e], t[e + 4], false, false);
            t[e] = max(x[0], x[1]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const auto x = __builtin_amdgcn_permlane16_swap(t[e], t[e + 2], false, false);
            t[e] = max(x[0], x[1]);
        }
        const bool odd = lane & 8;
        // byte wave / 2 of a column's word, 8 columns of this lane
        uint32_t* codes = col_codes + cl;
        ((uint8_t*)(codes + lane / 8))[wave / 2] =
            (uint8_t)block_code(max_dpp<kXor8>(odd ? t[1] : t[0], odd ? t[0] : t[1]));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t c = ((const uint8_t*)(codes + e))[wave / 2];
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0][e], v[1][e], scale_of(c), 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2][e], v[3][e], scale_of(c), 1);
            *(uint16_t*)(col_elems + (cl + e) * PITCH_PT + rl / 2) = (uint16_t)(c == 255 ? 0 : w);
        }
    }
    __syncthreads();
    // Codes past the last block are 0, and so are all of a tile past the last row or column, there
    // to complete a group of 8.
    const int t = threadIdx.x;
    if (ro.P) {
        const int64_t row = tile_r + t / 4, c = tile_c + t % 4 * 32;
        if (row < a.rows && c < a.cols) {
            const uint2* w = (const uint2*)(row_elems + t / 4 * PITCH_P + t % 4 * 16);
            __builtin_nontemporal_store(u32x4{w[0].x, w[0].y, w[1].x, w[1].y}, (u32x4*)(ro.P + row * ro.ldp + c / 2));
        }
        if (t < TILE && tile_r + t < a.rows)
            *(uint32_t*)(ro.S + tile_c / 256 * ro.lds + (tile_r + t) * 8 + tile_c / 32 % 8) = row_codes[t];
    }
    if (co.P) {
        const int64_t col = tile_c + t / 4, r = tile_r + t % 4 * 32;
        if (col < a.cols && r < a.rows) {
            const uint32_t* w = (const uint32_t*)(col_elems + t / 4 * PITCH_PT + t % 4 * 16);
            __builtin_nontemporal_store(u32x4{w[0], w[1], w[2], w[3]}, (u32x4*)(co.P + col * co.ldp + r / 2));
        }
        if (t < TILE && tile_c + t < a.cols && tile_r / 256 * 256 < a.rows)
            *(uint32_t*)(co.S + tile_r / 256 * co.lds + (tile_c + t) * 8 + tile_r / 32 % 8) = col_codes[t];
    }
}

// Threads form TX pieces of 16 bytes of a row's values by 256 / TX rows, as many times as give a
// thread 32 values.
//   Bound by HBM: 8192^2 to bf16 25.4 us (170 MB, 6.7 TB/s), to fp32 45.6 (304 MB, 6.7 TB/s); rows
// that begin inside a line cost more: 8191 x 8190 33.4 and 67.0.
template <typename T>
constexpr int kRows = 32 / Piece<T>::N;

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp,
                                                         const uint8_t* S, int64_t lds, T* Y, int64_t ldy, int tx,
                                                         int col_tiles)
{
    constexpr int N = Piece<T>::N, R = kRows<T>;
    typedef typename std::conditional<N == 8, uint32_t, uint16_t>::type elems_t;
    const int64_t c0 = ((int64_t)(blockIdx.x % col_tiles) * tx + threadIdx.x % tx) * N;
    const int per = 256 / tx;
    const int64_t r0 = (int64_t)(blockIdx.x / col_tiles) * (per * R) + threadIdx.x / tx;
    if (c0 >= cols) return;
    uint32_t w[R], code[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t r = r0 + i * per < rows ? r0 + i * per : rows - 1;  // (a row past the last is not stored)
        w[i] = *(const elems_t*)(P + r * ldp + c0 / 2);
        code[i] = S[c0 / 256 * lds + r * 8 + c0 / 32 % 8];
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t r = r0 + i * per;
        if (r >= rows) break;
        const float scale = scale_of(code[i]);
        f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 0),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 1)};
        if constexpr (N == 8) {
            v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 2);
            v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 3);
        }
        Piece<T> y;
#pragma unroll
        for (int e = 0; e < N; ++e) y.v[e] = (T)(code[i] == 255 ? __builtin_nanf("") : v[e / 2][e % 2]);
        T* to = Y + r * ldy + c0;
        if (c0 + N <= cols)
            store_past(to, y);
        else
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (c0 + e < cols) to[e] = y.v[e];
    }
}

template <typename T>
hipError_t quantize(const DropoutArgs& a, const Mx4Out& rows, const Mx4Out& cols, hipStream_t s)
{
    // whole groups of 8 blocks along a form's axis: their codes are written to the end
    const int64_t rt = cols.P ? (a.rows + 255) / 256 * 2 : (a.rows + TILE - 1) / TILE;
    const int64_t ct = rows.P ? (a.cols + 255) / 256 * 2 : (a.cols + TILE - 1) / TILE;
    if (rt * ct > 0x7fffffff) return hipErrorNotSupported;
    const dim3 grid = grid_of(rt * ct);
    if (a.threshold && a.gate) quantize_kernel<T, true, true><<<grid, 512, 0, s>>>(a, rows, cols, (int)ct);
    else if (a.threshold) quantize_kernel<T, true, false><<<grid, 512, 0, s>>>(a, rows, cols, (int)ct);
    else if (a.gate) quantize_kernel<T, false, true><<<grid, 512, 0, s>>>(a, rows, cols, (int)ct);
    else quantize_kernel<T, false, false><<<grid, 512, 0, s>>>(a, rows, cols, (int)ct);
    return hipGetLastError();
}

template <typename T>
hipError_t dequantize(int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp, const uint8_t* S,
                      int64_t lds, void* Y, int64_t ldy, hipStream_t s)
{
    const int64_t pieces = (cols + Piece<T>::N - 1) / Piece<T>::N;
    int tx = 1;
    while (tx < 256 && tx < pieces) tx *= 2;
    const int64_t per = 256 / tx * kRows<T>;
    const int64_t ct = (pieces + tx - 1) / tx, rt = (rows + per - 1) / per;
    if (rt * ct * 256 > kMaxThreads) return hipErrorNotSupported;
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
