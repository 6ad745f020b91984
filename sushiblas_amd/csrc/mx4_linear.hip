// mx4_linear.hip -- Y = alpha * X * B^T + beta * Y for a few rows of X, dense or MXFP8, and an
// MXFP4 matrix B (layer.hpp).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "layer.hpp"
#include "mx4_rows.hpp"

namespace sbx {
namespace {

constexpr int kWaves = 8;

template <typename T>
__device__ inline T result(float acc, float y, const Mx4LinearArgs& p)
{
    const float v = p.beta != 0.0f ? p.alpha * acc + p.beta * y : p.alpha * acc;
    return (T)(p.relu ? (v > 0.0f ? v : 0.0f) : v);
}

// A workgroup takes 16 XB rows of B and YB tiles of TOKENS rows of X, its eight waves each an eighth
// of the terms, in groups of 256 by turns: two groups of B are under way beside the one at work, and
// a tile of X.  The waves' sums are added up in LDS, in order.  Which wave has a term does not
// depend on m, so a row's bits do not either.
template <typename T, bool MX8, int TOKENS, int YB, int XB>
__global__ void __launch_bounds__(64 * kWaves, 2) linear_kernel(Mx4LinearArgs p)
{
    typedef typename std::conditional<MX8, Mx8Tokens<TOKENS>, DenseTokens<T, TOKENS>>::type tokens_t;
    constexpr int PIECES = tokens_t::PIECES, PITCH = 16 * YB + 4;
    constexpr int OWN = rows4_bytes(XB) + tokens_bytes(PIECES, TOKENS), PART = 16 * PITCH * 4;
    __shared__ __align__(16) char lds[kWaves * (OWN > PART ? OWN : PART)];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int x0 = block_x() * (16 * XB), y0 = blockIdx.y * (TOKENS * YB);
    if (x0 >= p.n) return;
    char *own = lds + wave * OWN, *tokens_at = own + rows4_bytes(XB);
    const int nb = (p.k + 31) / 32, groups = (nb + 7) / 8, whole = MX8 ? groups : p.k / 256;
    Source4<XB> sw;
    sw.init(p.B, p.ldb, p.SB, p.ldsb, x0, p.n, nb, lane);
    tokens_t sa[YB];
#pragma unroll
    for (int j = 0; j < YB; ++j) {
        const int first = min(y0 + j * TOKENS, p.m - 1);
        if constexpr (MX8)
            sa[j].init((const uint8_t*)p.X, p.ldx, p.SX, p.ldsx, first, p.m, nb);
        else {
            const int ld = (int)(p.ldx * sizeof(T)), count = min(p.m - first, TOKENS);
            sa[j].init((const T*)p.X + first * p.ldx, (count - 1) * ld + p.k * (int)sizeof(T),
                       [&](int t) { return t < count ? t * ld : kOutside; }, lane);
        }
    }

    f32x4 acc[YB][XB] = {};
    Rows4<XB> w0, w1;
    typename tokens_t::Values a;
    auto load_tokens = [&](int j, int g) {  // (a group past the last: the last whole one, not used)
        if constexpr (MX8)
            sa[j].load(a, g, nb - 8 * g, lane);
        else
            sa[j].load(a, min(g, whole - 1));
    };
    auto use = [&](Rows4<XB>& w, int g, bool end) {
        if (nb - 8 * g < 8)
#pragma unroll
            for (int i = 0; i < XB; ++i) w.code[i] = first_codes(w.code[i], nb - 8 * g);
        bf16x8 v[XB][8];
        fragments(w, own, lane, v);
        sw.load(w, g + 2 * kWaves, nb - 8 * (g + 2 * kWaves));
#pragma unroll
        for (int j = 0; j < YB; ++j) {
            if (end)
                if constexpr (!MX8) {
                    if (p.k >= Piece<T>::N)
                        sa[j].template load_end<Cut::Ragged>(a, g, p.k, lane);
                    else
                        sa[j].template load_end<Cut::Short>(a, g, p.k, lane);
                }
            sa[j].put(a, tokens_at, lane);
            if (!end) load_tokens(j + 1 < YB ? j + 1 : 0, j + 1 < YB ? g : g + kWaves);
            multiply<PIECES, TOKENS>(acc[j], v, tokens_at, lane);
        }
    };
    sw.load(w0, wave, nb - 8 * wave);
    sw.load(w1, wave + kWaves, nb - 8 * (wave + kWaves));
    int g = wave;
    if (g < whole) {
        load_tokens(0, g);
        for (; g < whole; g += 2 * kWaves) {
            use(w0, g, false);
            if (g + kWaves < whole) use(w1, g + kWaves, false);
        }
    }
    if (!MX8 && p.k % 256 && whole % kWaves == wave) {
        Rows4<XB> w = whole / kWaves % 2 ? w1 : w0;
        use(w, whole, true);
    }

    __syncthreads();
    float* part = (float*)lds;
    T* Y = (T*)p.Y;
    const int r = lane % 16, q = lane / 16;
#pragma unroll
    for (int i = 0; i < XB; ++i) {
        if (i > 0) __syncthreads();
#pragma unroll
        for (int j = 0; j < YB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[(wave * 16 + 4 * q + e) * PITCH + 16 * j + r] = acc[j][i][e];
        __syncthreads();
        for (int t = threadIdx.x; t < 16 * TOKENS * YB; t += 64 * kWaves) {
            const int dm = t / 16, n = x0 + 16 * i + t % 16, m = y0 + dm;
            if (n >= p.n || m >= p.m) continue;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
                v += part[(w * 16 + t % 16) * PITCH + dm / TOKENS * 16 + dm % TOKENS];
            T* y = Y + (int64_t)m * p.ldy + n;
            *y = result<T>(v, p.beta != 0.0f ? (float)*y : 0.0f, p);
        }
    }
}

template <typename T, bool MX8, int TOKENS, int YB>
hipError_t launch_form(const Mx4LinearArgs& a, hipStream_t s)
{
    const unsigned gy = (unsigned)((a.m + TOKENS * YB - 1) / (TOKENS * YB));
    // two blocks of B's rows a workgroup, where that leaves one for each CU
    if (a.n > 16 * 256)
        linear_kernel<T, MX8, TOKENS, YB, 2><<<grid_of((a.n + 31) / 32, gy), 64 * kWaves, 0, s>>>(a);
    else
        linear_kernel<T, MX8, TOKENS, YB, 1><<<grid_of((a.n + 15) / 16, gy), 64 * kWaves, 0, s>>>(a);
    return hipGetLastError();
}

template <typename T, bool MX8>
hipError_t launch(const Mx4LinearArgs& a, hipStream_t s)
{
    constexpr int TOKENS = MX8 || kBf16Pieces<T> == 1 ? 16 : 8;  // (pieces of 16 would not fit the LDS)
    if (a.m <= 2) return launch_form<T, MX8, 2, 1>(a, s);
    if (a.m <= TOKENS) return launch_form<T, MX8, TOKENS, 1>(a, s);
    if (a.m <= 2 * TOKENS) return launch_form<T, MX8, TOKENS, 2>(a, s);
    return launch_form<T, MX8, TOKENS, 4>(a, s);
}

}  // namespace

hipError_t launch_mx4_linear(int dtype, const Mx4LinearArgs& a, hipStream_t s)
{
    switch (dtype) {
    case 0: return a.SX ? launch<float, true>(a, s) : launch<float, false>(a, s);
    case 2: return a.SX ? launch<bf16_t, true>(a, s) : launch<bf16_t, false>(a, s);
    default: return a.SX ? launch<f16_t, true>(a, s) : launch<f16_t, false>(a, s);
    }
}

}  // namespace sbx
