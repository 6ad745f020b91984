// dropout.hip -- dropout whose mask is a function of the element's place, so
// that none is stored (see DropoutArgs): Y = keep ? X * scale : 0, and with a
// gate only where gate > 0.  Forward and backward pass are the same kernel.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx4.hpp"

namespace sbx {
namespace {

template <typename T>
struct Arith {
    typedef float type;
};
template <>
struct Arith<double> {
    typedef double type;
};

// Threads form TX pieces of 16 bytes of a row (8 columns share a call of the generator: threads
// of fp32 make it twice, of fp64 four times) by 256 / TX rows.
//   Bound by HBM: 8192^2 bf16 43.7 us (268 MB, 6.1 TB/s), with a gate 65.3; fp32 91.5 (537 MB, 5.9
// TB/s; a call of the generator for 8 values, which leaves a lane 32 bytes apart from the next,
// 102), with a gate 132.6; fp64 175-217 (1.07 GB, 4.9-6.1 TB/s), with a gate 254.  The generator makes 792 G calls/s: 8192^2 in 11 us, under the loads.
// Small ones are a launch: fp32 512 x 1024 3.3 us, 5.5 a call.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs a, T* Y, int64_t ldy, int tx)
{
    typedef typename Arith<T>::type R;
    constexpr int N = Piece<T>::N;
    const int64_t c0 = ((int64_t)blockIdx.x * tx + threadIdx.x % tx) * N;
    if (c0 >= a.cols) return;
    const R scale = (R)a.scale;
    const int rows_per = 256 / tx;
    for (int64_t row = (int64_t)blockIdx.y * rows_per + threadIdx.x / tx; row < a.rows;
         row += (int64_t)gridDim.y * rows_per) {
        const T* x = (const T*)a.X + row * a.ldx + c0;
        const T* g = a.gate ? (const T*)a.gate + row * a.ldg + c0 : nullptr;
        T* y = Y + row * ldy + c0;
        uint32_t keep[4];
        if (a.threshold) {
            keep_words(a, (uint32_t)row, (uint32_t)(c0 / 8), keep);
#pragma unroll
            for (int from = N; from < 8; from += N)  // the piece's words first
                if (c0 % 8 == from)
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) keep[i] = keep[from / 2 + i];
        }
        if (c0 + N <= a.cols) {
            const Piece<T> xv = *(const Piece<T>*)x;
            Piece<T> yv;
#pragma unroll
            for (int i = 0; i < N; ++i)
                yv.v[i] = !a.threshold || kept(a, keep, i) ? (T)((R)xv.v[i] * scale) : (T)0;
            if (g) {
                const Piece<T> gv = *(const Piece<T>*)g;
#pragma unroll
                for (int i = 0; i < N; ++i) yv.v[i] = gv.v[i] > (T)0 ? yv.v[i] : (T)0;
            }
            store_past(y, yv);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (c0 + i >= a.cols) continue;
                const bool on = (!a.threshold || kept(a, keep, i)) && (!g || g[i] > (T)0);
                y[i] = on ? (T)((R)x[i] * scale) : (T)0;
            }
        }
    }
}

template <typename T>
hipError_t launch(const DropoutArgs& a, void* Y, int64_t ldy, hipStream_t s)
{
    const int64_t pieces = (a.cols + Piece<T>::N - 1) / Piece<T>::N;
    int tx = 1;
    while (tx < 256 && tx < pieces) tx *= 2;
    const int64_t gx = (pieces + tx - 1) / tx, rows_per = 256 / tx;
    int64_t gy = (a.rows + rows_per - 1) / rows_per;
    if (gy > 65535) gy = 65535;
    dropout_kernel<T><<<dim3((unsigned)gx, (unsigned)gy), 256, 0, s>>>(a, (T*)Y, ldy, tx);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_dropout(int dtype, const DropoutArgs& a, void* Y, int64_t ldy, hipStream_t s)
{
    switch (dtype) {
    case 0: return launch<float>(a, Y, ldy, s);
    case 1: return launch<double>(a, Y, ldy, s);
    case 2: return launch<bf16_t>(a, Y, ldy, s);
    default: return launch<f16_t>(a, Y, ldy, s);
    }
}

}  // namespace sbx
