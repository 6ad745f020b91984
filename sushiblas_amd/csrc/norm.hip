// norm.hip -- the root-mean-square norm of rows, with the addition of a residual before it,
// results in the input's type or MXFP8, and its gradient (layer.hpp).
//
// Sums of squares and the factor 1 / sqrt(mean + eps) are held in 64 bits, and the norm is their
// product with the values in 64, rounded to 32 once: so that the 8-bit form, whose steps are
// 2^-3 of a value, does not depend on the order of a sum.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "layer.hpp"
#include "pieces.hpp"

namespace sbx {
namespace {

// COUNT sums over the THREADS lanes of a row, from 16 (four rows to a wave) to a workgroup's 1024.
// Between waves through LDS: `slot` alternates, so that one barrier is enough.
template <int THREADS, int COUNT>
__device__ inline void row_sums(double (&x)[COUNT], double (&part)[2][16][COUNT], int slot)
{
#pragma unroll
    for (int i = 0; i < COUNT; ++i) x[i] = THREADS == 16 ? sum16(x[i]) : sum64(x[i]);
    if constexpr (THREADS > 64) {
        const int wave = threadIdx.x / 64, first = wave / (THREADS / 64) * (THREADS / 64);
        if (threadIdx.x % 64 == 0)
#pragma unroll
            for (int i = 0; i < COUNT; ++i) part[slot][wave][i] = x[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            x[i] = part[slot][first][i];
#pragma unroll
            for (int w = 1; w < THREADS / 64; ++w) x[i] += part[slot][first + w][i];
        }
    }
}

template <int CTRL>
__device__ inline uint32_t max_lane(uint32_t x)
{
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true));
}

// Piece `c` .. of the norm to MXFP8; the lanes of a block of 32 are neighbours.
template <typename T>
__device__ inline void store_mx8(const Mx4Out& q, int64_t row, int c, int cols, const float (&v)[Piece<T>::N])
{
    constexpr int N = Piece<T>::N;
    uint32_t top = 0;  // magnitudes are in the order of their bits, NaN last
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffff);
    top = max_lane<kDppXor1>(top);
    top = max_lane<kDppXor2>(top);
    if constexpr (N == 4) top = max_lane<kDppHalfMirror>(top);
    const uint32_t e = top >> 23;
    const uint32_t code = e == 255 ? 255u : __builtin_elementwise_sub_sat(e, 8u);
    const float scale = __builtin_bit_cast(float, (254 - code) << 23);  // 2^(127 - code)
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        float s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = __builtin_amdgcn_fmed3f(v[4 * i + j] * scale, -448.0f, 448.0f);
        w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
        w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], (int)w[i], true);
        if (code == 255) w[i] = 0;
    }
    const int nb = (cols + 31) / 32, b = c / 32;
    if (b >= nb) return;
    uint8_t* p = q.P + row * q.ldp + c;
    if constexpr (N == 8)
        *(uint64_t*)p = (uint64_t)w[1] << 32 | w[0];
    else
        *(uint32_t*)p = w[0];
    if (c % 32 == 0) {
        uint8_t* s = q.S + b / 8 * q.lds + 8 * row;
        s[b % 8] = (uint8_t)code;
        if (b == nb - 1)
            for (int i = nb % 8; i % 8; ++i) s[i] = 0;  // past the row's last block
    }
}

// H and the norm's results for a piece.
template <Cut CUT, typename T>
__device__ inline void emit(const NormArgs& a, int64_t row, int c, const Piece<T>& h, const Piece<T>& w, double rs)
{
    constexpr int N = Piece<T>::N;
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)((double)(float)h.v[i] * rs * (double)(float)w.v[i]);
    if (a.H) store_piece<CUT>((T*)a.H + row * a.ldh, c, (int)a.cols, h);
    if (a.Y) {
        Piece<T> y;
#pragma unroll
        for (int i = 0; i < N; ++i) y.v[i] = (T)v[i];
        store_piece<CUT>((T*)a.Y + row * a.ldy, c, (int)a.cols, y);
    }
    if (a.q.P) store_mx8<T>(a.q, row, c, (int)a.cols, v);
}

template <typename T>
__device__ inline void add(Piece<T>& x, const Piece<T>& r)
{
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) x.v[i] = (T)((float)x.v[i] + (float)r.v[i]);
}

template <typename T>
__device__ inline double square(const Piece<T>& h)
{
    double sq = 0.0;
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) sq += (double)(float)h.v[i] * (double)(float)h.v[i];
    return sq;
}

// Rows that THREADS lanes hold in PIECES pieces each, so that X and R are read once.
//   Bound by HBM: 8192^2 bf16 with the residual 102 us (537 MB, 5.3 TB/s; a copy reaches 5.1), fp32 199,
// to MXFP8 93; 16384 x 512 bf16 13.7.  Rows that begin inside lines: 2047 x 4095 fp16 14.7 us
// (67 MB, 4.6 TB/s).  One row is a launch: 2.3 us for 4096 (5.5-6.5 a call), by as many lanes as it has pieces.
template <typename T, Cut CUT, int THREADS, int PIECES>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) norm_kernel(NormArgs a)
{
    constexpr int N = Piece<T>::N, ROWS = THREADS < 256 ? 256 / THREADS : 1;
    __shared__ double part[2][16][1];
    const int c0 = threadIdx.x % THREADS * N, cols = (int)a.cols;
    Piece<T> w[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) w[p] = whole_piece<CUT>((const T*)a.W, c0 + p * THREADS * N, cols);
    int slot = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS; row < a.rows;
         row += (int64_t)gridDim.x * ROWS, slot ^= 1) {
        Piece<T> h[PIECES], r[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
            h[p] = load_piece<CUT>((const T*)a.X + row * a.ldx, c0 + p * THREADS * N, cols);
        if (a.R) {
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
                r[p] = load_piece<CUT>((const T*)a.R + row * a.ldr, c0 + p * THREADS * N, cols);
#pragma unroll
            for (int p = 0; p < PIECES; ++p) add(h[p], r[p]);
        }
#pragma unroll
        for (int p = 0; p < PIECES; ++p) trim_piece<CUT>(h[p], c0 + p * THREADS * N, cols);
        double sq[1] = {};
#pragma unroll
        for (int p = 0; p < PIECES; ++p) sq[0] += square(h[p]);
        row_sums<THREADS>(sq, part, slot);
        const double rs = rsqrt(sq[0] / (double)a.cols + a.eps);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            keep_packed(h[p]);
            keep_packed(w[p]);
        }
#pragma unroll
        for (int p = 0; p < PIECES; ++p) emit<CUT>(a, row, c0 + p * THREADS * N, h[p], w[p], rs);
    }
}

// Longer rows, read twice: 2047 x 33000 bf16 with the residual 146 us for 540 MB, 4096 x 16392 fp32 253 for 1074
// (3.7 and 4.2 TB/s of what has to move).
template <typename T, Cut CUT>
__global__ void __launch_bounds__(1024) norm_long_kernel(NormArgs a)
{
    constexpr int N = Piece<T>::N, STEP = 1024 * N;
    __shared__ double part[2][16][1];
    const int cols = (int)a.cols, end = (cols + STEP - 1) / STEP * STEP;
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, slot ^= 1) {
        const T *x = (const T*)a.X + row * a.ldx, *r = (const T*)a.R + row * a.ldr;
        auto load = [&](int c) {
            Piece<T> h = load_piece<CUT>(x, c, cols);
            if (a.R) add(h, load_piece<CUT>(r, c, cols));
            trim_piece<CUT>(h, c, cols);
            return h;
        };
        double sq[1] = {};
        for (int c = threadIdx.x * N; c < end; c += STEP) sq[0] += square(load(c));
        row_sums<1024>(sq, part, slot);
        const double rs = rsqrt(sq[0] / (double)a.cols + a.eps);
        // (results may lie where X or R is read: a thread writes what it alone reads, but for the
        // piece across the row's end, which is read with values before it, and drops those)
        for (int c = threadIdx.x * N; c < end; c += STEP)
            emit<CUT>(a, row, c, load(c), whole_piece<CUT>((const T*)a.W, c, cols), rs);
    }
}

// What a row's gradient takes from its sums of squares and of dy w h: s = 1 / sqrt(mean + eps) as s g w, g
// and w powers of two that halve its exponent, and m = s^2 mean(dy w h).  Since eps may be 0, s may pass what 32
// bits hold, and dy w lie past them where dy w s does not.
struct RowGrad {
    float g, w, s, m;
    __device__ inline RowGrad(const double (&sum)[2], double per_col, double eps)
    {
        const double rs = rsqrt(sum[0] * per_col + eps);
        const int e = max(min(__builtin_amdgcn_frexp_exp(rs), 252), -252), half = e / 2;  // (0 of an infinity and NaN)
        g = __builtin_bit_cast(float, (uint32_t)(127 + half) << 23);
        w = __builtin_bit_cast(float, (uint32_t)(127 + e - half) << 23);
        s = (float)__builtin_ldexp(rs, -e);
        m = (float)(sum[1] * per_col * rs * rs);
    }
    // Of a wave's only row, in scalar registers.
    __device__ inline void keep_once()
    {
        auto once = [](float& x) {
            x = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
        };
        once(g);
        once(w);
        once(s);
        once(m);
    }
};

// The gradient of a piece of a row, its input's gradient stored and its share of W's added to dw: with
// n = h s, dx = s dy w - n m + dr.  (dy g and w's w stay within 32 bits where dy w s does, unless it is
// w below 2^-50 or above 2^63 that brings it back: 64 bits throughout take 1-3 % more, and 39.8 us for
// 4095 x 3001 bf16, whose registers they pass.)
template <Cut CUT, typename T>
__device__ inline void grad_piece(const NormGradArgs& a, int64_t row, int c, const Piece<T>& h, const Piece<T>& dy,
                                  const Piece<T>& dr, const Piece<T>& w, const RowGrad& by, float (&dw)[Piece<T>::N])
{
    Piece<T> dx;
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) {
        const float g = (float)dy.v[i], n = (float)h.v[i] * by.g * (by.w * by.s);
        const float v = g * by.g * ((float)w.v[i] * by.w) * by.s - n * by.m;
        dx.v[i] = (T)(a.DR ? v + (float)dr.v[i] : v);
        dw[i] += g * n;
    }
    store_piece<CUT>((T*)a.DX + row * a.lddx, c, (int)a.cols, dx);
}

template <typename T>
__device__ inline void grad_sums(const Piece<T>& h, const Piece<T>& dy, const Piece<T>& w, double (&sum)[2])
{
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) {
        const double x = (double)(float)h.v[i];
        sum[0] += x * x;
        sum[1] += x * ((double)(float)dy.v[i] * (double)(float)w.v[i]);
    }
}

// THREADS lanes to a row, PIECES pieces of it in each; the workgroup's rows' share of W's gradient
// stays in registers over its rows, and is added up in LDS at the end, in order.
//   Bound by HBM where each workgroup has many rows: 8192 x 4096 bf16 51.5-53 us (268 MB, 5.1 TB/s), and
// 1.5-4 for the parts.  With few (4095 x 3001 bf16: 4 each, 24 us and 4.6 for the parts, for 98 MB) by the way from a row's
// loads over its sums to its stores, which nothing overlaps but the other waves' own.  More parts,
// for two workgroups a CU, would cost their way through memory.
template <typename T, Cut CUT, int THREADS, int PIECES>
__global__ void __launch_bounds__(1024) grad_kernel(NormGradArgs a)
{
    constexpr int N = Piece<T>::N, ROWS = 1024 / THREADS;
    __shared__ double part[2][16][2];
    const int c0 = threadIdx.x % THREADS * N, cols = (int)a.cols;
    const double per_col = 1.0 / (double)a.cols;
    Piece<T> w[PIECES];
    float dw[PIECES][N] = {};
#pragma unroll
    for (int p = 0; p < PIECES; ++p) w[p] = whole_piece<CUT>((const T*)a.W, c0 + p * THREADS * N, cols);
    int slot = 0;
    for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.rows; base += (int64_t)gridDim.x * ROWS, slot ^= 1) {
        // (a row past the last: the last one again, and nothing of it kept)
        const int64_t mine = base + threadIdx.x / THREADS;
        const bool inside = mine < a.rows;
        const int64_t row = inside ? mine : a.rows - 1;
        Piece<T> h[PIECES], dy[PIECES], dr[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            h[p] = load_piece<CUT>((const T*)a.H + row * a.ldh, c0 + p * THREADS * N, cols);
            dy[p] = load_piece<CUT>((const T*)a.DY + row * a.lddy, c0 + p * THREADS * N, cols);
        }
        if (a.DR)
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
                dr[p] = load_piece<CUT>((const T*)a.DR + row * a.lddr, c0 + p * THREADS * N, cols);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            trim_piece<CUT>(h[p], c0 + p * THREADS * N, cols);
            trim_piece<CUT>(dy[p], c0 + p * THREADS * N, cols);
        }
        double sum[2] = {};
#pragma unroll
        for (int p = 0; p < PIECES; ++p) grad_sums(h[p], dy[p], w[p], sum);
        row_sums<THREADS>(sum, part, slot);
        RowGrad by(sum, per_col, a.eps);
        if constexpr (THREADS >= 64) by.keep_once();
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            keep_packed(h[p]);
            keep_packed(dy[p]);
            keep_packed(w[p]);
        }
        if (a.DR)
#pragma unroll
            for (int p = 0; p < PIECES; ++p) trim_piece<CUT>(dr[p], c0 + p * THREADS * N, cols);
        if (inside)
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
                grad_piece<CUT>(a, row, c0 + p * THREADS * N, h[p], dy[p], dr[p], w[p], by, dw[p]);
    }
    if (!a.DW) return;
    float* to = a.part + blockIdx.x * a.cols;
    __shared__ float sums[ROWS > 1 ? 1024 * N : 1];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        if constexpr (ROWS > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) sums[threadIdx.x * N + i] = dw[p][i];
            __syncthreads();
            for (int c = threadIdx.x; c < THREADS * N; c += 1024) {
                float v = sums[c];
                for (int g = 1; g < ROWS; ++g) v += sums[g * THREADS * N + c];
                if (p * THREADS * N + c < cols) to[p * THREADS * N + c] = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (c0 + p * THREADS * N + i < cols) to[c0 + p * THREADS * N + i] = dw[p][i];
        }
    }
}

// Longer rows, read twice; a workgroup's share of W's gradient lies in memory: 4096 x 16384 fp32 301 us for 1074 MB,
// 4096 x 16385 bf16 286 for 537.
template <typename T, Cut CUT>
__global__ void __launch_bounds__(1024) grad_long_kernel(NormGradArgs a)
{
    constexpr int N = Piece<T>::N, STEP = 1024 * N;
    __shared__ double part[2][16][2];
    const int cols = (int)a.cols, end = (cols + STEP - 1) / STEP * STEP;
    const double per_col = 1.0 / (double)a.cols;
    const T* W = (const T*)a.W;
    float* to = a.part + blockIdx.x * a.cols;
    bool first = true;
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, first = false, slot ^= 1) {
        const T *H = (const T*)a.H + row * a.ldh, *DY = (const T*)a.DY + row * a.lddy;
        double sum[2] = {};
        for (int c = threadIdx.x * N; c < end; c += STEP)
            grad_sums(whole_piece<CUT>(H, c, cols), whole_piece<CUT>(DY, c, cols),
                      whole_piece<CUT>(W, c, cols), sum);
        row_sums<1024>(sum, part, slot);
        const RowGrad by(sum, per_col, a.eps);
        for (int c = threadIdx.x * N; c < end; c += STEP) {
            typedef Piece<float> four_t;
            float dw[N] = {};
            const bool inside = c + N <= cols;
            if (a.DW && !first) {
                if (inside)
#pragma unroll
                    for (int i = 0; i < N; i += 4) *(four_t*)(dw + i) = *(const four_t*)(to + c + i);
                else
#pragma unroll
                    for (int i = 0; i < N; ++i) dw[i] = c + i < cols ? to[c + i] : 0.0f;
            }
            Piece<T> dr = {};
            if (a.DR) dr = whole_piece<CUT>((const T*)a.DR + row * a.lddr, c, cols);
            grad_piece<CUT>(a, row, c, whole_piece<CUT>(H, c, cols), whole_piece<CUT>(DY, c, cols), dr,
                       whole_piece<CUT>(W, c, cols), by, dw);
            if (a.DW) {
                if (inside)
#pragma unroll
                    for (int i = 0; i < N; i += 4) *(four_t*)(to + c + i) = *(const four_t*)(dw + i);
                else
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (c + i < cols) to[c + i] = dw[i];
            }
        }
    }
}

// W's gradient from its parts (none: zeros): 64 columns a workgroup at a time, its 16 waves every 16th part each.
__global__ void __launch_bounds__(1024) parts_kernel(const float* part, int parts, int64_t cols, float* DW)
{
    __shared__ float sums[16][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    for (int64_t c0 = (int64_t)blockIdx.x * 64; c0 < cols; c0 += (int64_t)gridDim.x * 64) {
        const int64_t c = c0 + lane;
        float v = 0.0f;
        if (c < cols)
#pragma unroll 4
            for (int i = wave; i < parts; i += 16) v += part[i * cols + c];
        __syncthreads();
        sums[wave][lane] = v;
        __syncthreads();
        if (wave > 0 || c >= cols) continue;
#pragma unroll
        for (int i = 1; i < 16; ++i) v += sums[i][lane];
        DW[c] = v;
    }
}

// Threads form TX pieces of 16 bytes of a row's values by 256 / TX rows.
template <typename T>
__global__ void __launch_bounds__(256) dequantize8_kernel(int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp,
                                                          const uint8_t* S, int64_t lds, T* Y, int64_t ldy, int tx,
                                                          int col_tiles)
{
    constexpr int N = Piece<T>::N, R = 4;
    typedef typename std::conditional<N == 8, uint64_t, uint32_t>::type elems_t;
    const int64_t c = ((int64_t)(blockIdx.x % col_tiles) * tx + threadIdx.x % tx) * N;
    const int per = 256 / tx;
    const int64_t r0 = (int64_t)(blockIdx.x / col_tiles) * (per * R) + threadIdx.x / tx;
    if (c >= cols) return;
    elems_t w[R];
    uint32_t code[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t r = r0 + i * per < rows ? r0 + i * per : rows - 1;  // (a row past the last is not stored)
        w[i] = *(const elems_t*)(P + r * ldp + c);
        code[i] = S[c / 256 * lds + r * 8 + c / 32 % 8];
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t r = r0 + i * per;
        if (r >= rows) break;
        // 2^(code - 127), by halves: 2^-127 is not normal, and its product with an element exact
        const float half = __builtin_bit_cast(float, (code[i] / 2 + 64) << 23),
                    rest = __builtin_bit_cast(float, (code[i] - code[i] / 2 + 63) << 23);
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        float v[N];
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            const int word = (int)(uint32_t)(w[i] >> (e == 4 ? 32 : 0));
            const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
            v[e] = lo[0]; v[e + 1] = lo[1]; v[e + 2] = hi[0]; v[e + 3] = hi[1];
        }
        Piece<T> y;
#pragma unroll
        for (int e = 0; e < N; ++e) y.v[e] = (T)(code[i] == 255 ? __builtin_nanf("") : v[e] * half * rest);
        store_piece<Cut::Ragged>(Y + r * ldy, (int)c, (int)cols, y);
    }
}

template <typename T, Cut CUT, int THREADS, int PIECES>
hipError_t launch_norm(const NormArgs& a, hipStream_t s)
{
    constexpr int ROWS = THREADS < 256 ? 256 / THREADS : 1, MOST = 256 * 2048 / (THREADS < 256 ? 256 : THREADS);
    const int64_t groups = (a.rows + ROWS - 1) / ROWS;
    norm_kernel<T, CUT, THREADS, PIECES>
        <<<(unsigned)(groups < MOST ? groups : MOST), THREADS < 256 ? 256 : THREADS, 0, s>>>(a);
    return hipGetLastError();
}

template <typename T, Cut CUT>
hipError_t norm(const NormArgs& a, int64_t pieces, hipStream_t s)
{
    if (pieces <= 16) return launch_norm<T, CUT, 16, 1>(a, s);
    if constexpr (CUT != Cut::Short) {
        if (pieces <= 64) return launch_norm<T, CUT, 64, 1>(a, s);
        // few rows: as many lanes as there are pieces, for latency
        const bool few = a.rows < 512;
        if (pieces <= 256) {
            if (few) return launch_norm<T, CUT, 256, 1>(a, s);
            return pieces <= 128 ? launch_norm<T, CUT, 64, 2>(a, s) : launch_norm<T, CUT, 64, 4>(a, s);
        }
        if (pieces <= 512) return few ? launch_norm<T, CUT, 512, 1>(a, s) : launch_norm<T, CUT, 256, 2>(a, s);
        if (pieces <= 1024) return few ? launch_norm<T, CUT, 1024, 1>(a, s) : launch_norm<T, CUT, 256, 4>(a, s);
        if (pieces <= 2048) return launch_norm<T, CUT, 512, 4>(a, s);
        if constexpr (sizeof(T) == 4)  // (of 16 bits they would not fit the registers)
            if (pieces <= 4096) return launch_norm<T, CUT, 1024, 4>(a, s);
        norm_long_kernel<T, CUT><<<(unsigned)(a.rows < 512 ? a.rows : 512), 1024, 0, s>>>(a);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t norm(const NormArgs& a, hipStream_t s)
{
    const int64_t pieces = (a.cols + Piece<T>::N - 1) / Piece<T>::N;
    switch (cut_of<T>(a.cols)) {
    case Cut::Whole: return norm<T, Cut::Whole>(a, pieces, s);
    case Cut::Ragged: return norm<T, Cut::Ragged>(a, pieces, s);
    default: return norm<T, Cut::Short>(a, pieces, s);
    }
}

// The only part is W's gradient.
NormGradArgs whole(NormGradArgs a, int parts)
{
    if (parts == 1) a.part = a.DW;
    return a;
}

template <typename T, Cut CUT, int THREADS, int PIECES>
int launch_grad(const NormGradArgs& a, hipStream_t s)
{
    constexpr int ROWS = 1024 / THREADS;
    // Up to two turns go to one workgroup, which writes W's gradient itself: a second launch costs as much or more
    // (4 x 4096 bf16, one turn, 6.8 us against 10.1; 128 x 128, two, 6.6 against 9.7; 8 x 4096, two, 10.0 either way).
    const int64_t groups = (a.rows + ROWS - 1) / ROWS;
    const int parts = groups <= 2 ? 1 : groups < kNormGradParts ? (int)groups : kNormGradParts;
    grad_kernel<T, CUT, THREADS, PIECES><<<parts, 1024, 0, s>>>(whole(a, parts));
    return parts;
}

// Returns how many parts W's gradient has.
template <typename T, Cut CUT>
int norm_grad(const NormGradArgs& a, int64_t pieces, hipStream_t s)
{
    if (pieces <= 16) return launch_grad<T, CUT, 16, 1>(a, s);
    if constexpr (CUT != Cut::Short) {
        if (pieces <= 64) return launch_grad<T, CUT, 64, 1>(a, s);
        if (pieces <= 128) return launch_grad<T, CUT, 64, 2>(a, s);
        if (pieces <= 256) return launch_grad<T, CUT, 128, 2>(a, s);
        if (pieces <= 512) return launch_grad<T, CUT, 256, 2>(a, s);
        if (pieces <= 1024) return launch_grad<T, CUT, 512, 2>(a, s);
        if (pieces <= 2048) return launch_grad<T, CUT, 1024, 2>(a, s);
        const int parts = a.rows < kNormGradParts ? (int)a.rows : kNormGradParts;
        grad_long_kernel<T, CUT><<<parts, 1024, 0, s>>>(whole(a, parts));
        return parts;
    }
    return 0;
}

template <typename T>
int norm_grad(const NormGradArgs& a, hipStream_t s)
{
    const int64_t pieces = (a.cols + Piece<T>::N - 1) / Piece<T>::N;
    switch (cut_of<T>(a.cols)) {
    case Cut::Whole: return norm_grad<T, Cut::Whole>(a, pieces, s);
    case Cut::Ragged: return norm_grad<T, Cut::Ragged>(a, pieces, s);
    default: return norm_grad<T, Cut::Short>(a, pieces, s);
    }
}

template <typename T>
hipError_t dequantize8(int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp, const uint8_t* S, int64_t lds,
                       void* Y, int64_t ldy, hipStream_t s)
{
    const int64_t pieces = (cols + Piece<T>::N - 1) / Piece<T>::N;
    int tx = 1;
    while (tx < 256 && tx < pieces) tx *= 2;
    const int64_t per = 256 / tx * 4, ct = (pieces + tx - 1) / tx, rt = (rows + per - 1) / per;
    if (rt * ct * 256 > kMaxThreads) return hipErrorNotSupported;
    dequantize8_kernel<T><<<(unsigned)(rt * ct), 256, 0, s>>>(rows, cols, P, ldp, S, lds, (T*)Y, ldy, tx, (int)ct);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rms_norm(int dtype, const NormArgs& a, hipStream_t s)
{
    switch (dtype) {
    case 0: return norm<float>(a, s);
    case 2: return norm<bf16_t>(a, s);
    default: return norm<f16_t>(a, s);
    }
}

hipError_t launch_rms_norm_grad(int dtype, const NormGradArgs& a, hipStream_t s)
{
    int parts = 0;
    if (a.rows > 0) {
        switch (dtype) {
        case 0: parts = norm_grad<float>(a, s); break;
        case 2: parts = norm_grad<bf16_t>(a, s); break;
        default: parts = norm_grad<f16_t>(a, s);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (!a.DW || parts == 1) return hipSuccess;
    const int64_t tiles = (a.cols + 63) / 64;
    parts_kernel<<<(unsigned)(tiles < 65536 ? tiles : 65536), 1024, 0, s>>>(a.part, parts, a.cols, a.DW);
    return hipGetLastError();
}

hipError_t launch_mx8_dequantize(int dtype, int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp,
                                 const uint8_t* S, int64_t lds, void* Y, int64_t ldy, hipStream_t s)
{
    switch (dtype) {
    case 0: return dequantize8<float>(rows, cols, P, ldp, S, lds, Y, ldy, s);
    case 2: return dequantize8<bf16_t>(rows, cols, P, ldp, S, lds, Y, ldy, s);
    default: return dequantize8<f16_t>(rows, cols, P, ldp, S, lds, Y, ldy, s);
    }
}

}  // namespace sbx
