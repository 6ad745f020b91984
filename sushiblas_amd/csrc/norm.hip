// norm.hip -- the root-mean-square norm of rows, with the addition of a residual before it,
// results in the input's type or MXFP8, and its gradient (layer.hpp).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "layer.hpp"

namespace sbx {
namespace {

// The sum over a workgroup of 256, in every thread.
__device__ inline double total(double v)
{
    __shared__ double part[4];
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    __syncthreads();
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    return part[0] + part[1] + part[2] + part[3];
}

template <typename T>
__device__ inline T sum_at(const NormArgs& a, int64_t row, int64_t c)
{
    const T x = ((const T*)a.X)[row * a.ldx + c];
    return a.R ? (T)((float)x + (float)((const T*)a.R)[row * a.ldr + c]) : x;
}

template <typename T>
__global__ void __launch_bounds__(256) norm_kernel(NormArgs a)
{
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        double sq = 0.0;
        for (int64_t c = threadIdx.x; c < a.cols; c += 256) {
            const double h = (double)(float)sum_at<T>(a, row, c);
            sq += h * h;
        }
        const double rs = 1.0 / sqrt(total(sq) / (double)a.cols + a.eps);
        // a thread to a block of 32
        const int64_t nb = (a.cols + 31) / 32;
        for (int64_t b = threadIdx.x; b < (nb + 7) / 8 * 8; b += 256) {
            float v[32], top = 0.0f;
            bool fine = true;
            for (int i = 0; i < 32; ++i) {
                const int64_t c = b * 32 + i;
                v[i] = 0.0f;
                if (c >= a.cols) continue;
                const T h = sum_at<T>(a, row, c);
                v[i] = (float)((double)(float)h * rs * (double)(float)((const T*)a.W)[c]);
                if (a.H) ((T*)a.H)[row * a.ldh + c] = h;
                if (a.Y) ((T*)a.Y)[row * a.ldy + c] = (T)v[i];
                fine = fine && __builtin_isfinite(v[i]);
                top = fmaxf(top, fabsf(v[i]));
            }
            if (!a.q.P) continue;
            int code = fine ? (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 8 : 255;
            if (code < 0) code = 0;
            a.q.S[b / 8 * a.q.lds + 8 * row + b % 8] = b < nb ? code : 0;
            if (b >= nb) continue;
            const double up = code == 255 ? 0.0 : ldexp(1.0, 127 - code);
            for (int i = 0; i < 32; i += 2) {
                const float x = code == 255 ? 0.0f : fminf(fmaxf((float)(v[i] * up), -448.0f), 448.0f);
                const float y = code == 255 ? 0.0f : fminf(fmaxf((float)(v[i + 1] * up), -448.0f), 448.0f);
                *(uint16_t*)(a.q.P + row * a.q.ldp + b * 32 + i) =
                    (uint16_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false);
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) grad_kernel(NormGradArgs a)
{
    for (int64_t c = threadIdx.x; a.DW && c < a.cols; c += 256) a.part[blockIdx.x * a.cols + c] = 0.0f;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *h = (const T*)a.H + row * a.ldh, *dy = (const T*)a.DY + row * a.lddy, *w = (const T*)a.W;
        double sq = 0.0, along = 0.0;
        for (int64_t c = threadIdx.x; c < a.cols; c += 256) {
            const double x = (double)(float)h[c];
            sq += x * x;
            along += x * (double)(float)w[c] * (double)(float)dy[c];
        }
        const double rs = 1.0 / sqrt(total(sq) / (double)a.cols + a.eps);
        along = total(along) / (double)a.cols * rs * rs;
        for (int64_t c = threadIdx.x; c < a.cols; c += 256) {
            const double x = (double)(float)h[c], g = (double)(float)dy[c];
            double dx = rs * (g * (double)(float)w[c] - x * along);
            if (a.DR) dx += (double)(float)((const T*)a.DR)[row * a.lddr + c];
            if (a.DW) a.part[blockIdx.x * a.cols + c] += (float)(g * x * rs);
            ((T*)a.DX)[row * a.lddx + c] = (T)(float)dx;
        }
    }
}

__global__ void __launch_bounds__(256) parts_kernel(const float* part, int parts, int64_t cols, float* DW)
{
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float v = 0.0f;
    for (int i = 0; i < parts; ++i) v += part[i * cols + c];
    DW[c] = v;
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize8_kernel(int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp,
                                                          const uint8_t* S, int64_t lds, T* Y, int64_t ldy)
{
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
        if (c >= cols) return;
        const uint32_t code = S[c / 256 * lds + row * 8 + c / 32 % 8];
        const float v = __builtin_amdgcn_cvt_f32_fp8(P[row * ldp + c], 0);
        Y[row * ldy + c] = (T)(code == 255 ? __builtin_nanf("") : (float)ldexp((double)v, (int)code - 127));
    }
}

}  // namespace

hipError_t launch_rms_norm(int dtype, const NormArgs& a, hipStream_t s)
{
    const unsigned grid = (unsigned)(a.rows < 65536 ? a.rows : 65536);
    switch (dtype) {
    case 0: norm_kernel<float><<<grid, 256, 0, s>>>(a); break;
    case 2: norm_kernel<bf16_t><<<grid, 256, 0, s>>>(a); break;
    default: norm_kernel<f16_t><<<grid, 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

hipError_t launch_rms_norm_grad(int dtype, const NormGradArgs& a, hipStream_t s)
{
    const int parts = norm_grad_parts(a.rows);
    if (parts) {
        switch (dtype) {
        case 0: grad_kernel<float><<<parts, 256, 0, s>>>(a); break;
        case 2: grad_kernel<bf16_t><<<parts, 256, 0, s>>>(a); break;
        default: grad_kernel<f16_t><<<parts, 256, 0, s>>>(a);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || !a.DW) return e;
    }
    parts_kernel<<<(unsigned)((a.cols + 255) / 256), 256, 0, s>>>(a.part, parts, a.cols, a.DW);
    return hipGetLastError();
}

hipError_t launch_mx8_dequantize(int dtype, int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp,
                                 const uint8_t* S, int64_t lds, void* Y, int64_t ldy, hipStream_t s)
{
    const dim3 grid((unsigned)((cols + 255) / 256), (unsigned)(rows < 65535 ? rows : 65535));
    switch (dtype) {
    case 0: dequantize8_kernel<float><<<grid, 256, 0, s>>>(rows, cols, P, ldp, S, lds, (float*)Y, ldy); break;
    case 2: dequantize8_kernel<bf16_t><<<grid, 256, 0, s>>>(rows, cols, P, ldp, S, lds, (bf16_t*)Y, ldy); break;
    default: dequantize8_kernel<f16_t><<<grid, 256, 0, s>>>(rows, cols, P, ldp, S, lds, (f16_t*)Y, ldy);
    }
    return hipGetLastError();
}

}  // namespace sbx
