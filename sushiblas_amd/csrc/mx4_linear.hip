// mx4_linear.hip -- Y = alpha * X * B^T + beta * Y for a few rows of X, dense or MXFP8, and an
// MXFP4 matrix B (layer.hpp).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "layer.hpp"
#include "layer_plan.hpp"
#include "mx4_rows.hpp"

namespace sbx {
namespace {

template <typename T>
__device__ inline T result(float acc, float y, const Mx4LinearArgs& p)
{
    const float v = p.beta != 0.0f ? p.alpha * acc + p.beta * y : p.alpha * acc;
    return (T)(p.relu ? (v > 0.0f ? v : 0.0f) : v);
}

// The groups of terms of one of WAVES waves (or of as many sums), one after another: first, first + WAVES, ..;
// from one of them that differs from block to block of B's rows, and round, where rows lie 4096 bytes apart
// or a multiple: workgroups that are at the same terms of all rows would meet in the same memory channels
// (1 x 8192 x 8192 bf16 12.0 us, so 9.3; 1 x 28672 x 8192 28.4, so 24.0.  1 x 8192 x 12288, rows 6144 apart,
// 12.6, so 12.9).
template <int WAVES>
struct Turns {
    int first, count, start;
    __device__ inline Turns(const Mx4LinearArgs& p, int first_, int groups, int block)
    {
        first = first_;
        count = (groups - first + WAVES - 1) / WAVES;
        start = p.ldb % 4096 == 0 && count > 1 ? (int)((uint32_t)block * 2654435761u >> 16) % count : 0;
    }
    // The i-th; of i >= count one past the last group (zeros where it is loaded).
    __device__ inline int group(int i) const
    {
        return first + WAVES * (i >= count ? i : i + start < count ? i + start : i + start - count);
    }
};

constexpr int kTallRows = 128, kTallTokens = 16;

// A workgroup takes 16 XB rows of B and YB tiles of TOKENS rows of X, its waves a share each of the
// terms, in groups of 256 by turns; AHEAD groups are under way (2 with one tile of X alone).  The waves' sums
// are added up in LDS, in order.
// Which wave has a term does not depend on m, so a row's bits do not either.
//   One token is bound by memory: bf16 1 x 28672 x 8192 23.9 us (125 MB, 5.2 TB/s; the product of
// MXFP4 operands, mx4_gemm.hip, 29.0), 1 x 8192 x 8192 8.2-9.8 (36 MB: 2.3 of it are any kernel's, and there is one
// round).  More tokens are bound by the operands' way through LDS to the matrix cores, which their loads do
// not quite hide behind: without any load bf16 16 x 28672 x 8192 takes 21.5 of its 35 us (with X's alone,
// which each workgroup reads all of, 23.6, with B's 28.5) and 64 x 8192 x 8192 19.1 of 22.1; conversions
// take one (64 rows of B a workgroup take too many registers: 79).
template <typename T, bool MX8, int TOKENS, int YB, int XB, int WAVES, int AHEAD>
__global__ void __launch_bounds__(64 * WAVES, 2) linear_kernel(Mx4LinearArgs p)
{
    typedef typename std::conditional<MX8, Mx8Tokens<TOKENS>, DenseTokens<T, TOKENS>>::type tokens_t;
    constexpr int PIECES = tokens_t::PIECES, FRAGMENTS = fragments_of(PIECES, TOKENS), PITCH = 16 * FRAGMENTS * YB + 4;
    constexpr int OWN = rows4_bytes(XB) + tokens_bytes(PIECES, TOKENS), PART = 16 * PITCH * 4;
    __shared__ __align__(16) char lds[WAVES * (OWN > PART ? OWN : PART)];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int x0 = block_x() * (16 * XB), y0 = blockIdx.y * (TOKENS * YB);
    if (x0 >= p.n) return;
    char *own = lds + wave * OWN, *tokens_at = own + rows4_bytes(XB);
    const int nb = (p.k + 31) / 32, groups = (nb + 7) / 8;
    Source4<XB> sw;
    sw.init(p.ldb, p.ldsb, p.n - x0, nb, lane);
    sw.move(p.B, p.SB, x0);
    tokens_t sa[YB];
#pragma unroll
    for (int j = 0; j < YB; ++j) {
        const int first = min(y0 + j * TOKENS, p.m - 1);
        if constexpr (MX8)
            sa[j].init((const uint8_t*)p.X, p.ldx, p.SX, p.ldsx, first, p.m, p.k);
        else {
            const int ld = (int)(p.ldx * sizeof(T)), count = min(p.m - first, TOKENS);
            sa[j].init((const T*)p.X + first * p.ldx, (count - 1) * ld + p.k * (int)sizeof(T), p.k,
                       [&](int t) { return t < count ? t * ld : kOutside; }, lane);
        }
    }

    f32x4 acc[YB][FRAGMENTS][XB] = {};
    Rows4<XB> w[AHEAD];
    typename tokens_t::Values a[AHEAD];
    // (no branch around a load, and one past the last group reads zeros or the last group again: the
    // compiler would wait for all of them where paths meet)
    const Turns<WAVES> own_turns(p, wave, groups, x0 / (PIECES == 1 ? 32 : kTallRows));
    const int turns = own_turns.count;
    auto group = [&](int i) { return own_turns.group(i); };
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
        const int g = group(d);
        sw.load(w[d], g, nb - 8 * g);
        sa[0].load(a[d], g, lane);
    }
    for (int turn = 0; turn < turns;) {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
            const int g = group(turn), next = group(turn + AHEAD);
            bf16x8 v[XB][8];
            if (nb - 8 * g < 8)
#pragma unroll
                for (int i = 0; i < XB; ++i) w[d].code[i] = first_bytes(w[d].code[i], nb - 8 * g);
            fragments(w[d], own, lane, v);
            sw.load(w[d], next, nb - 8 * next);
#pragma unroll
            for (int j = 0; j < YB; ++j) {
                sa[j].put(a[d], tokens_at, g, lane);
                sa[j + 1 < YB ? j + 1 : 0].load(a[d], j + 1 < YB ? g : next, lane);
                multiply<PIECES, TOKENS>(acc[j], v, tokens_at, lane);
            }
            if (++turn == turns) break;
        }
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
            for (int f = 0; f < FRAGMENTS; ++f)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    part[(wave * 16 + 4 * q + e) * PITCH + 16 * (FRAGMENTS * j + f) + r] = acc[j][f][i][e];
        __syncthreads();
        for (int t = threadIdx.x; t < 16 * TOKENS * YB; t += 64 * WAVES) {
            const int dm = t / 16, n = x0 + 16 * i + t % 16, m = y0 + dm;
            if (n >= p.n || m >= p.m) continue;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
#pragma unroll
                for (int x = 0; x < PIECES; ++x)
                    v += part[(w * 16 + t % 16) * PITCH + 16 * FRAGMENTS * (dm / TOKENS) + x * TOKENS + dm % TOKENS];
            T* y = Y + (int64_t)m * p.ldy + n;
            *y = result<T>(v, p.beta != 0.0f ? (float)*y : 0.0f, p);
        }
    }
}

// Many rows of X in pieces: four waves take 32 rows of B each, and tiles of 16 rows of X lie in LDS for all of
// them, a group after another, the next one on its way; so X is read, and its pieces are made, once for 128
// rows of B.  Four more waves have the same rows and every other group, so that one's products go on while another
// waits for LDS (64 x 8192 x 8192 fp16 33.6 us, by four waves alone 41.4, by linear_kernel 44.5; fp32 40.9, 56.3, 66.6).
//   A row's bits are linear_kernel's: sums of every fourth group stay apart, as its four waves' are.
//   Bound by a wave's own way through LDS and conversions, which two waves to a SIMD do not hide: bf16,
// with nothing to split, gains nothing (24.5 against 25.6; 256 x 8192 x 4096 50.2 against 46.0).
template <typename T>
__global__ void __launch_bounds__(512, 2) linear_tall_kernel(Mx4LinearArgs p)
{
    constexpr int WAVES = 4, SETS = 2, TOKENS = kTallTokens, PER = TOKENS / WAVES;
    typedef DenseTokens<T, PER> tokens_t;
    constexpr int PIECES = tokens_t::PIECES, FRAGMENTS = fragments_of(PIECES, TOKENS), STAGE = tokens_bytes(PIECES, TOKENS);
    __shared__ __align__(16) char lds[SETS * (2 * STAGE + WAVES * rows4_bytes(2))];
    const int lane = threadIdx.x % 64, id = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wave = id % WAVES, set = id / WAVES;
    const int x0 = block_x() * kTallRows, y0 = blockIdx.y * TOKENS;
    if (x0 >= p.n) return;
    const int nb = (p.k + 31) / 32, groups = (nb + 7) / 8, n0 = x0 + 32 * wave;
    char *stage = lds + set * 2 * STAGE, *own = lds + SETS * 2 * STAGE + id * rows4_bytes(2);
    // (past the last row of B or X: that one, not stored)
    const int row = min(n0, p.n - 1), first = min(y0 + PER * wave, p.m - 1);
    Source4<2> sw;
    sw.init(p.ldb, p.ldsb, p.n - row, nb, lane);
    sw.move(p.B, p.SB, row);
    tokens_t sa;
    const int ld = (int)(p.ldx * sizeof(T)), count = min(p.m - first, PER);
    sa.init((const T*)p.X + first * p.ldx, (count - 1) * ld + p.k * (int)sizeof(T), p.k,
            [&](int t) { return t < count ? t * ld : kOutside; }, lane);
    constexpr int SUMS = 4 / SETS;  // of groups 4 i + SETS u + set
    const Turns<4> mine[SUMS] = {{p, set, groups, x0 / kTallRows}, {p, set + SETS, groups, x0 / kTallRows}};
    f32x4 acc[SUMS][FRAGMENTS][2] = {};
    Rows4<2> w;
    typename tokens_t::Values a;
    sa.load(a, mine[0].group(0), lane);
    sw.load(w, mine[0].group(0), nb - 8 * mine[0].group(0));
    sa.template put<TOKENS>(a, stage, mine[0].group(0), lane, PER * wave);
    sa.load(a, mine[1].group(0), lane);
    lds_barrier();
    const int turns = (groups + 3) / 4;  // of all: the last one without a group, perhaps
    for (int turn = 0; turn < turns; ++turn) {
#pragma unroll
        for (int u = 0; u < SUMS; ++u) {
            const int g = mine[u].group(turn), then = mine[1 - u].group(turn + u);
            bf16x8 v[2][8];
            if (nb - 8 * g < 8)
#pragma unroll
                for (int i = 0; i < 2; ++i) w.code[i] = first_bytes(w.code[i], nb - 8 * g);
            fragments(w, own, lane, v);
            sw.load(w, then, nb - 8 * then);
            sa.template put<TOKENS>(a, stage + (1 - u) * STAGE, then, lane, PER * wave);  // its last readers passed the barrier before
            sa.load(a, mine[u].group(turn + 1), lane);
            multiply<PIECES, TOKENS>(acc[u], v, stage + u * STAGE, lane);
            lds_barrier();
        }
    }
    static_assert(WAVES * SUMS * FRAGMENTS * 2 * 64 * 16 <= sizeof(lds), "");
    f32x4* part = (f32x4*)lds + wave * (SUMS * FRAGMENTS * 2 * 64) + lane;
    if (set == 1)
#pragma unroll
        for (int u = 0; u < SUMS; ++u)
#pragma unroll
            for (int x = 0; x < FRAGMENTS; ++x)
#pragma unroll
                for (int i = 0; i < 2; ++i) part[((u * FRAGMENTS + x) * 2 + i) * 64] = acc[u][x][i];
    __syncthreads();
    const int m = y0 + lane % 16;
    if (set == 1 || m >= p.m) return;
    T* Y = (T*)p.Y + m * p.ldy;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f32x4 v = {};
#pragma unroll
        for (int u = 0; u < SUMS; ++u) {
#pragma unroll
            for (int x = 0; x < FRAGMENTS; ++x) v += acc[u][x][i];
#pragma unroll
            for (int x = 0; x < FRAGMENTS; ++x) v += part[((u * FRAGMENTS + x) * 2 + i) * 64];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = n0 + 16 * i + 4 * (lane / 16) + e;
            if (n < p.n) Y[n] = result<T>(v[e], p.beta != 0.0f ? (float)Y[n] : 0.0f, p);
        }
    }
}

// Fewer terms than a piece has, or none.  A thread to a result.
template <typename T>
__global__ void __launch_bounds__(256) few_terms_kernel(Mx4LinearArgs p)
{
    const int64_t n = (int64_t)block_x() * 256 + threadIdx.x;
    if (n >= p.n) return;
    const int m = blockIdx.y;
    float sum = 0.0f;
    if (p.k > 0) {
        const float scale = scale_of_code(p.SB[8 * n]);
        for (int c = 0; c < p.k; ++c)
            sum += (float)((const T*)p.X)[m * p.ldx + c] *
                   __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(p.B[n * p.ldb + c / 2] >> c % 2 * 4, scale, 0)[0];
    }
    T* y = (T*)p.Y + (int64_t)m * p.ldy + n;
    *y = result<T>(sum, p.beta != 0.0f ? (float)*y : 0.0f, p);
}

template <typename T, bool MX8, int TOKENS, int YB, int XB, int WAVES, int AHEAD>
void start(const Mx4LinearArgs& a, hipStream_t s)
{
    const unsigned gy = (unsigned)((a.m + TOKENS * YB - 1) / (TOKENS * YB));
    linear_kernel<T, MX8, TOKENS, YB, XB, WAVES, AHEAD>
        <<<grid_of((a.n + 16 * XB - 1) / (16 * XB), gy), 64 * WAVES, 0, s>>>(a);
}

template <typename T, bool MX8, int TOKENS, int YB>
void launch_rows(const Mx4LinearPlan& p, const Mx4LinearArgs& a, hipStream_t s)
{
    if constexpr (TOKENS == 2 && (MX8 || kBf16Pieces<T> == 1)) {
        if (p.ahead == 2)
            p.waves == 8 ? start<T, MX8, 2, YB, 1, 8, 2>(a, s) : start<T, MX8, 2, YB, 1, 4, 2>(a, s);
        else
            p.waves == 8 ? start<T, MX8, 2, YB, 1, 8, 1>(a, s) : start<T, MX8, 2, YB, 1, 4, 1>(a, s);
    } else {
        p.waves == 8 ? start<T, MX8, TOKENS, YB, 1, 8, 1>(a, s) : start<T, MX8, TOKENS, YB, 2, 4, 1>(a, s);
    }
}

template <typename T, bool MX8>
hipError_t launch(const Mx4LinearArgs& a, hipStream_t s)
{
    constexpr int PIECES = MX8 ? 1 : kBf16Pieces<T>;
    const Mx4LinearPlan p = mx4_linear_plan(PIECES, MX8, a.m, a.n, a.k);
    if (p.form == Mx4LinearPlan::FewTerms) {
        few_terms_kernel<T><<<grid_of((a.n + 255) / 256, (unsigned)a.m), 256, 0, s>>>(a);
    } else if (p.form == Mx4LinearPlan::Tall) {
        if constexpr (PIECES > 1)
            linear_tall_kernel<T><<<grid_of((a.n + kTallRows - 1) / kTallRows,
                                            (unsigned)((a.m + kTallTokens - 1) / kTallTokens)), 512, 0, s>>>(a);
    } else if (p.tokens == 2) {
        launch_rows<T, MX8, 2, 1>(p, a, s);
    } else if (p.tokens == 8) {
        if constexpr (PIECES > 1) {
            if (p.tiles == 1) {
                launch_rows<T, MX8, 8, 1>(p, a, s);
            } else if constexpr (PIECES == 3) {
                launch_rows<T, MX8, 8, 2>(p, a, s);
            }
        }
    } else if constexpr (PIECES < 3) {
        p.tiles == 1 ? launch_rows<T, MX8, 16, 1>(p, a, s) : launch_rows<T, MX8, 16, 2>(p, a, s);
    }
    return hipGetLastError();
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
