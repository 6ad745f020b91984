// mx4_linear.hip -- Y = alpha * X * B^T + beta * Y for a few rows of X, dense or MXFP8, and an
// MXFP4 matrix B (layer.hpp).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "layer.hpp"

namespace sbx {
namespace {

// One wave to a result.
template <typename T>
__global__ void __launch_bounds__(256) linear_kernel(Mx4LinearArgs a)
{
    const int lane = threadIdx.x % 64;
    const int64_t n = (int64_t)block_x() * 4 + threadIdx.x / 64;
    if (n >= a.n) return;
    const int nb = (a.k + 31) / 32;
    for (int64_t m = blockIdx.y; m < a.m; m += gridDim.y) {
        float sum = 0.0f;
        for (int b = lane; b < nb; b += 64) {
            const float s = __builtin_bit_cast(float, (uint32_t)a.SB[b / 8 * a.ldsb + 8 * n + b % 8] << 23);
            const uint8_t* w = a.B + n * a.ldb + 16 * b;
            float s8 = 1.0f;
            if (a.SX) {
                const uint32_t code = a.SX[b / 8 * a.ldsx + 8 * m + b % 8];
                s8 = code == 255 ? __builtin_nanf("") : code ? __builtin_bit_cast(float, code << 23) : 0x1p-127f;
            }
            float dot = 0.0f;
            for (int i = 0; i < 32; ++i) {
                const int64_t c = 32 * b + i;
                if (c >= a.k) break;
                const float x = a.SX ? __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)a.X)[m * a.ldx + c], 0) * s8
                                     : (float)((const T*)a.X)[m * a.ldx + c];
                dot += x * __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i / 2] >> i % 2 * 4, s, 0)[0];
            }
            sum += dot;
        }
        for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
        if (lane == 0) {
            T* y = (T*)a.Y + m * a.ldy + n;
            float v = a.alpha * sum;
            if (a.beta != 0.0f) v += a.beta * (float)*y;
            *y = (T)(a.relu ? (v > 0.0f ? v : 0.0f) : v);
        }
    }
}

template <typename T>
hipError_t launch(const Mx4LinearArgs& a, hipStream_t s)
{
    linear_kernel<T><<<grid_of((a.n + 3) / 4, (unsigned)(a.m < 65535 ? a.m : 65535)), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mx4_linear(int dtype, const Mx4LinearArgs& a, hipStream_t s)
{
    switch (dtype) {
    case 0: return launch<float>(a, s);
    case 2: return launch<bf16_t>(a, s);
    default: return launch<f16_t>(a, s);
    }
}

}  // namespace sbx
