// mx4_moe.hip -- a mixture-of-experts layer for a few tokens, its experts' weights MXFP4
// (layer.hpp).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "layer.hpp"

namespace sbx {
namespace {

__device__ inline double* logits_of(const Mx4MoeArgs& a, const Mx4MoeWork& w) { return (double*)(a.work + w.logits); }
__device__ inline int* chosen_of(const Mx4MoeArgs& a, const Mx4MoeWork& w) { return (int*)(a.work + w.chosen); }
__device__ inline float* weights_of(const Mx4MoeArgs& a, const Mx4MoeWork& w) { return (float*)(a.work + w.weights); }
__device__ inline float* act_of(const Mx4MoeArgs& a, const Mx4MoeWork& w) { return (float*)(a.work + w.act); }

// Logits in 64 bits, so that which experts are chosen does not depend on the order of the sums.
template <typename T>
__global__ void __launch_bounds__(64) logits_kernel(Mx4MoeArgs a, Mx4MoeWork w)
{
    const int e = blockIdx.x, t = blockIdx.y;
    double sum = 0.0;
    for (int c = threadIdx.x; c < a.width; c += 64)
        sum += (double)(float)((const T*)a.X)[t * a.ldx + c] * (double)(float)((const T*)a.WR)[e * a.ldwr + c];
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if (threadIdx.x == 0) logits_of(a, w)[(int64_t)t * a.experts + e] = sum;
}

// Whether logit x of expert i comes before y of j: the higher one, NaN highest, ties by index.
__device__ inline bool before(double x, int i, double y, int j)
{
    const bool nx = x != x, ny = y != y;
    if (nx != ny) return nx;
    return !nx && x != y ? x > y : i < j;
}

__global__ void __launch_bounds__(64) choose_kernel(Mx4MoeArgs a, Mx4MoeWork w)
{
    const int t = blockIdx.x * 64 + threadIdx.x;
    if (t >= a.tokens) return;
    const double* l = logits_of(a, w) + (int64_t)t * a.experts;
    int* chosen = chosen_of(a, w) + t * a.topk;
    double top = 0.0, last = 0.0, sum = 0.0;
    int last_e = -1;
    for (int j = 0; j < a.topk; ++j) {
        int best = -1;
        for (int e = 0; e < a.experts; ++e)
            if ((last_e < 0 || before(last, last_e, l[e], e)) && (best < 0 || before(l[e], e, l[best], best))) best = e;
        chosen[j] = last_e = best;
        last = l[best];
        if (j == 0) top = last;
        if (a.normalize) sum += exp(last - top);
    }
    if (!a.normalize)
        for (int e = 0; e < a.experts; ++e) sum += exp(l[e] - top);
    for (int j = 0; j < a.topk; ++j) {
        const float p = (float)(exp(l[chosen[j]] - top) / sum);
        weights_of(a, w)[t * a.topk + j] = p;
        if (a.weights) a.weights[t * a.topk + j] = p;
        if (a.chosen) a.chosen[t * a.topk + j] = chosen[j];
    }
}

// A wave's product of a row of an MXFP4 matrix.
template <typename T>
__device__ inline float dot(const T* x, const uint8_t* P, const uint8_t* S, int64_t lds, int k)
{
    float sum = 0.0f;
    for (int b = threadIdx.x % 64; b < (k + 31) / 32; b += 64) {
        const float s = __builtin_bit_cast(float, (uint32_t)S[b / 8 * lds + b % 8] << 23);
        for (int i = 0; i < 32 && 32 * b + i < k; ++i)
            sum += (float)x[32 * b + i] *
                   __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(P[16 * b + i / 2] >> i % 2 * 4, s, 0)[0];
    }
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    return sum;
}

template <typename T>
__global__ void __launch_bounds__(64) up_kernel(Mx4MoeArgs a, Mx4MoeWork w)
{
    const int64_t j = blockIdx.x, c = blockIdx.y;  // unit of the hidden layer, choice
    const int64_t g = (int64_t)chosen_of(a, w)[c] * 2 * a.hidden + j, u = g + a.hidden;
    const T* x = (const T*)a.X + c / a.topk * a.ldx;
    const float gate = dot(x, a.W1 + g * a.ld1, a.S1 + 8 * g, a.lds1, a.width);
    const float up = dot(x, a.W1 + u * a.ld1, a.S1 + 8 * u, a.lds1, a.width);
    if (threadIdx.x == 0) act_of(a, w)[c * a.hidden + j] = gate / (1.0f + expf(-gate)) * up;
}

template <typename T>
__global__ void __launch_bounds__(64) down_kernel(Mx4MoeArgs a, Mx4MoeWork w)
{
    const int64_t n = blockIdx.x, t = blockIdx.y;
    float y = 0.0f;
    for (int j = 0; j < a.topk; ++j) {
        const int64_t c = t * a.topk + j, r = (int64_t)chosen_of(a, w)[c] * a.width + n;
        y += weights_of(a, w)[c] * dot(act_of(a, w) + c * a.hidden, a.W2 + r * a.ld2, a.S2 + 8 * r, a.lds2, a.hidden);
    }
    if (threadIdx.x == 0) ((T*)a.Y)[t * a.ldy + n] = (T)y;
}

template <typename T>
hipError_t launch(const Mx4MoeArgs& a, hipStream_t s)
{
    const Mx4MoeWork w = mx4_moe_work(a.tokens, a.hidden, a.experts, a.topk);
    const unsigned choices = (unsigned)(a.tokens * a.topk);
    logits_kernel<T><<<dim3((unsigned)a.experts, (unsigned)a.tokens), 64, 0, s>>>(a, w);
    choose_kernel<<<(unsigned)(a.tokens + 63) / 64, 64, 0, s>>>(a, w);
    up_kernel<T><<<dim3((unsigned)a.hidden, choices), 64, 0, s>>>(a, w);
    down_kernel<T><<<dim3((unsigned)a.width, (unsigned)a.tokens), 64, 0, s>>>(a, w);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mx4_moe(int dtype, const Mx4MoeArgs& a, hipStream_t s)
{
    switch (dtype) {
    case 0: return launch<float>(a, s);
    case 2: return launch<bf16_t>(a, s);
    default: return launch<f16_t>(a, s);
    }
}

}  // namespace sbx
