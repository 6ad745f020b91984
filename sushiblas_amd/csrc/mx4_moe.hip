// mx4_moe.hip -- a mixture-of-experts layer for a few tokens, its experts' weights MXFP4
// (layer.hpp).
//
// Kernels, each on what the one before wrote to the workspace:
//   prepare  the router's logits, and the tokens as bf16 pieces
//   choose   (more than 8 tokens or 64 experts, and two tokens) each token's experts and shares
//   up       a tile, a few tokens of one expert, by 16 units of the hidden layer a wave: share *
//            silu(G x) * (U x), as bf16 pieces; of fewer tokens and experts it chooses itself, which
//            costs less than a launch
//   down     a tile by 32 results; of one token, 16 results over all of its choices, which the waves share
//   combine  (more than one token) the sum over a token's choices
// Products and pieces: mx4_rows.hpp.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "layer.hpp"
#include "layer_plan.hpp"
#include "mx4_rows.hpp"

namespace sbx {
namespace {

// ---- the router ----

// Pieces that an activation is held in before the second product: the 24 bits of 32, of every type.  Two
// (16 bits) take less of the second product (64 x 4096 x 2048, 4 of 32, bf16 105 us against 112, 8 tokens 70.6
// and 73.0, one token 15.2 and 15.5), but where an expert's terms cancel what is left has none of a result's own bits.
constexpr int kActPieces = 3;

// x in the wave's lower half and y in its upper one, each added to its own other half.
__device__ inline double halves(double x, double y)
{
    const uint64_t a = __builtin_bit_cast(uint64_t, x), b = __builtin_bit_cast(uint64_t, y);
    auto lo = __builtin_amdgcn_permlane32_swap((uint32_t)a, (uint32_t)b, false, false);
    auto hi = __builtin_amdgcn_permlane32_swap((uint32_t)(a >> 32), (uint32_t)(b >> 32), false, false);
    return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) + __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
}
// The same by rows of 16 lanes: x in the even ones, y in the odd ones.
__device__ inline double quarters(double x, double y)
{
    const uint64_t a = __builtin_bit_cast(uint64_t, x), b = __builtin_bit_cast(uint64_t, y);
    auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)a, (uint32_t)b, false, false);
    auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(a >> 32), (uint32_t)(b >> 32), false, false);
    return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) + __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
}

// Four experts and TOKENS (1 or 4) tokens a workgroup, whose four waves take a quarter of the terms each.
// Logits in 64 bits, so that which experts are chosen does not depend on the order of the sums.
// Workgroups past the experts' make pieces.
template <typename T, int TOKENS>
__global__ void __launch_bounds__(256) prepare_kernel(Mx4MoeArgs a, Mx4MoeWork w, int expert_groups)
{
    constexpr int N = Piece<T>::N, PIECES = kBf16Pieces<T>;
    if ((int)blockIdx.x >= expert_groups) {  // 8 terms a thread
        const int per_row = w.x_ld / 16, i = (blockIdx.x - expert_groups) * 256 + threadIdx.x;
        if (blockIdx.y > 0 || i >= per_row * a.tokens) return;
        const int t = i / per_row, c = i % per_row * 8;
        const T* row = (const T*)a.X + t * a.ldx;
        float x[8];
#pragma unroll
        for (int p = 0; p < 8 / N; ++p) {
            const Piece<T> v = a.width > N ? whole_piece<Cut::Ragged>(row, c + N * p, a.width)
                                           : whole_piece<Cut::Short>(row, c + N * p, a.width);
#pragma unroll
            for (int e = 0; e < N; ++e) x[N * p + e] = (float)v.v[e];
        }
        bf16x8 to[PIECES];
        split(x, to);
#pragma unroll
        for (int n = 0; n < PIECES; ++n) *(bf16x8*)(a.work + w.x + n * w.x_stride + (size_t)i * 16) = to[n];
        return;
    }
    __shared__ double part[4][4 * TOKENS];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, e0 = blockIdx.x * 4, t0 = blockIdx.y * TOKENS;
    const T *wr[4], *x[TOKENS];  // (past the last expert or token: the last one again)
#pragma unroll
    for (int i = 0; i < 4; ++i) wr[i] = (const T*)a.WR + min(e0 + i, a.experts - 1) * a.ldwr;
#pragma unroll
    for (int j = 0; j < TOKENS; ++j) x[j] = (const T*)a.X + min(t0 + j, a.tokens - 1) * a.ldx;
    double sum[4][TOKENS] = {};
    auto add = [&](const T(&wv)[4], const T(&xv)[TOKENS]) {
        double wd[4], xd[TOKENS];
#pragma unroll
        for (int i = 0; i < 4; ++i) wd[i] = (double)(float)wv[i];
#pragma unroll
        for (int j = 0; j < TOKENS; ++j) xd[j] = (double)(float)xv[j];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < TOKENS; ++j) sum[i][j] += wd[i] * xd[j];
    };
    const int whole = a.width / N * N;
#pragma unroll 2
    for (int c = threadIdx.x * N; c < whole; c += 256 * N) {
        Piece<T> wv[4], xv[TOKENS];
#pragma unroll
        for (int i = 0; i < 4; ++i) wv[i] = *(const Piece<T>*)(wr[i] + c);
#pragma unroll
        for (int j = 0; j < TOKENS; ++j) xv[j] = *(const Piece<T>*)(x[j] + c);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            T we[4], xe[TOKENS];
#pragma unroll
            for (int i = 0; i < 4; ++i) we[i] = wv[i].v[n];
#pragma unroll
            for (int j = 0; j < TOKENS; ++j) xe[j] = xv[j].v[n];
            add(we, xe);
        }
    }
    if (whole + (int)threadIdx.x < a.width) {
        T we[4], xe[TOKENS];
#pragma unroll
        for (int i = 0; i < 4; ++i) we[i] = wr[i][whole + threadIdx.x];
#pragma unroll
        for (int j = 0; j < TOKENS; ++j) xe[j] = x[j][whole + threadIdx.x];
        add(we, xe);
    }
    // Sums over the wave: of four numbers at a time, so that each row of lanes is left with one of them.
    double* all = &sum[0][0];
#pragma unroll
    for (int i = 0; i < 4 * TOKENS; i += 4) {
        const double two[2] = {halves(all[i], all[i + 1]), halves(all[i + 2], all[i + 3])};
        const double s = sum16(quarters(two[0], two[1]));
        if (lane % 16 == 0) part[wave][i + (lane / 16 % 2 * 2 + lane / 32)] = s;
    }
    __syncthreads();
    const int i = threadIdx.x / TOKENS, j = threadIdx.x % TOKENS;
    if (i < 4 && e0 + i < a.experts && t0 + j < a.tokens)
        ((double*)(a.work + w.logits))[(int64_t)(t0 + j) * a.experts + e0 + i] =
            part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x];
}

// The highest of a wave's words.
__device__ inline uint32_t highest(uint32_t x)
{
    auto dpp = [&](auto ctrl) {
        x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true));
    };
    dpp(std::integral_constant<int, kDppXor1>{});
    dpp(std::integral_constant<int, kDppXor2>{});
    dpp(std::integral_constant<int, kDppHalfMirror>{});
    dpp(std::integral_constant<int, kDppMirror>{});
    const uint32_t a = __builtin_amdgcn_readlane((int)x, 0), b = __builtin_amdgcn_readlane((int)x, 16),
                   c = __builtin_amdgcn_readlane((int)x, 32), d = __builtin_amdgcn_readlane((int)x, 48);
    return max(max(a, b), max(c, d));
}

// A wave's choices for one token, one after another.  EACH: logits a lane has, 64 * EACH >= experts.
constexpr int kMaxExperts = 512;
template <int EACH>
struct Chooser {
    uint64_t key[EACH];  // the logits, by their order; 0: none, or taken already
    double mine, top;

    __device__ __forceinline__ void init(const double* logits, int experts, int lane)
    {
        mine = top = 0.0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            key[i] = 0;
            if (i * 64 + lane < experts) {
                const double l = logits[i * 64 + lane] + 0.0;  // (no negative zero)
                const uint64_t b = __builtin_bit_cast(uint64_t, l);
                key[i] = l != l ? ~0ull : b >> 63 ? ~b : b | 1ull << 63;
            }
        }
    }
    // The j-th expert, the same in all lanes.
    __device__ __forceinline__ int next(int j, int lane)
    {
        uint64_t best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < EACH; ++i)
            if (key[i] > best) {
                best = key[i];
                at = i;
            }
        const uint32_t hi = highest((uint32_t)(best >> 32));
        uint64_t with = __builtin_amdgcn_ballot_w64((uint32_t)(best >> 32) == hi);
        if (with & (with - 1)) {  // several: by the lower words, then the lowest index
            const bool in = with >> lane & 1;
            const uint32_t lo = highest(in ? (uint32_t)best : 0u);
            const bool equal = in && (uint32_t)best == lo;
            const uint32_t first = ~highest(equal ? ~(uint32_t)(at * 64 + lane) : 0u);
            with = __builtin_amdgcn_ballot_w64(equal && (uint32_t)(at * 64 + lane) == first);
        }
        const int winner = __builtin_ctzll(with);
        const int e = __builtin_amdgcn_readlane(at, winner) * 64 + winner;
        const double x = lane_value(__builtin_bit_cast(double, best >> 63 ? best & ~(1ull << 63) : ~best), winner);
        if (j == 0) top = x;
        if (lane == j) mine = x;
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (lane == winner && i == at) key[i] = 0;
        return e;
    }
    // After all: the share of a lane's choice, in lanes below topk.
    __device__ __forceinline__ float share(const double* logits, int experts, int topk, int normalize, int lane) const
    {
        const double own = exp(mine - top);
        double all = 0.0;
        if (normalize) {
            all = lane < topk ? own : 0.0;
        } else {
            for (int e = lane; e < experts; e += 64) all += exp(logits[e] - top);
        }
        return (float)(own / sum64(all));
    }
};

// A wave to a token.
template <int EACH>
__global__ void __launch_bounds__(256) choose_kernel(Mx4MoeArgs a, Mx4MoeWork w)
{
    const int lane = threadIdx.x % 64, t = blockIdx.x * 4 + threadIdx.x / 64;
    if (t >= a.tokens) return;
    const double* logits = (const double*)(a.work + w.logits) + (int64_t)t * a.experts;
    Chooser<EACH> from;
    from.init(logits, a.experts, lane);
    int mine = 0;
    for (int k = 0; k < a.topk; ++k) {
        const int e = from.next(k, lane);
        if (lane == k) mine = e;
    }
    const float p = from.share(logits, a.experts, a.topk, a.normalize, lane);
    if (lane >= a.topk) return;
    const int c = t * a.topk + lane;
    ((int*)(a.work + w.chosen))[c] = mine;
    ((float*)(a.work + w.weights))[c] = p;
    if (a.chosen) a.chosen[c] = mine;
    if (a.weights) a.weights[c] = p;
}

// ---- the experts ----

// The hidden layer's values, times their shares, as pieces.
template <int N>
__device__ inline void store_act(const Mx4MoeArgs& a, const Mx4MoeWork& w, int choice, int unit, const float (&h)[8])
{
    bf16x8 to[kActPieces];
    split(h, to);
#pragma unroll
    for (int n = 0; n < kActPieces; ++n) {
        uint8_t* at = a.work + w.act + n * w.act_stride + (size_t)choice * w.act_ld + 2 * unit;
        const u32x4 v = __builtin_bit_cast(u32x4, to[n]);
        if constexpr (N == 8)
            *(u32x4*)at = v;
        else
            *(u32x2*)at = u32x2{v[0], v[1]};
    }
}
// share * silu(gate) * up.  exp(-gate) passes 32 bits from -88.7 on, where silu times a large up is still an
// ordinary number: so by e = exp(-|gate| / 2), of which negative gates take 1 / (1 + 1 / e^2) = e e / (1 + e^2),
// one e before up and one after.
__device__ inline float act_of(float gate, float up, float share)
{
    const float e = expf(-0.5f * fabsf(gate)), by = gate < 0.0f ? e : 1.0f;
    return share * (gate * by / (1.0f + e * e) * up * by);
}

// The only token's: 16 units of the expert that is its choice blockIdx.y, by eight waves that share the terms.
//   Two workgroups to a CU, for which the registers of a second group of terms ahead are too many: 2048
// terms, 8 x 1024 units 18 MB, with prepare 13.1 us against 15.0.
template <typename T, int EACH>
__global__ void __launch_bounds__(512, 4) up_one_kernel(Mx4MoeArgs a, Mx4MoeWork w)
{
    constexpr int WAVES = 8, TOKENS = 2, PIECES = kBf16Pieces<T>, PITCH = 20;
    constexpr int OWN = rows4_bytes(2) + tokens_bytes(PIECES, TOKENS), PART = 2 * 16 * PITCH * 4;
    __shared__ __align__(16) char lds[WAVES * (OWN > PART ? OWN : PART)];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int j0 = blockIdx.x * 16, choice = blockIdx.y;
    const int nb = (a.width + 31) / 32, groups = (nb + 7) / 8, rows = min(a.hidden - j0, 16);
    PieceTokens<PIECES, TOKENS> sa;
    sa.base = a.work + w.x;
    sa.stride = w.x_stride;
    sa.move([&](int t) { return t > 0 ? kOutside : 0; }, lane);
    typename PieceTokens<PIECES, TOKENS>::Values x;
    sa.load(x, min(wave, groups - 1));
    Chooser<EACH> from;
    from.init((const double*)(a.work + w.logits), a.experts, lane);
    int expert = 0, mine = 0;
    for (int k = 0; k <= choice; ++k) {
        expert = from.next(k, lane);
        if (lane == k) mine = expert;
    }
    char *own = lds + wave * OWN, *tokens_at = own + rows4_bytes(2);
    f32x4 acc[1][2] = {};
    Source4<1> sg, su;
    sg.init(a.ld1, a.lds1, rows > 0 ? rows : 1, nb, lane);
    su = sg;
    // (past the last unit: the last one's rows, not used)
    sg.move(a.W1, a.S1, (int64_t)expert * 2 * a.hidden + min(j0, a.hidden - 1));
    su.move(a.W1, a.S1, (int64_t)expert * 2 * a.hidden + a.hidden + min(j0, a.hidden - 1));
    Rows4<1> wg, wu;
    sg.load(wg, wave, nb - 8 * wave);
    su.load(wu, wave, nb - 8 * wave);
    // the other choices, and the shares, while the weights are under way
    for (int k = choice + 1; k < a.topk; ++k) {
        const int e = from.next(k, lane);
        if (lane == k) mine = e;
    }
    const float shares = from.share((const double*)(a.work + w.logits), a.experts, a.topk, a.normalize, lane);
    const float share = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, shares), choice));
    if (blockIdx.x == 0 && choice == 0 && wave == 0 && lane < a.topk) {
        ((int*)(a.work + w.chosen))[lane] = mine;
        if (a.weights) a.weights[lane] = shares;
        if (a.chosen) a.chosen[lane] = mine;
    }
    for (int g = wave; g < groups; g += WAVES) {
        bf16x8 v[2][8];
        if (nb - 8 * g < 8) {
            wg.code[0] = first_bytes(wg.code[0], nb - 8 * g);
            wu.code[0] = first_bytes(wu.code[0], nb - 8 * g);
        }
        const Rows4<2> both = {{wg.v[0], wg.v[1], wu.v[0], wu.v[1]}, {wg.code[0], wu.code[0]}};
        fragments(both, own, lane, v);
        sg.load(wg, g + WAVES, nb - 8 * (g + WAVES));
        su.load(wu, g + WAVES, nb - 8 * (g + WAVES));
        sa.put(x, tokens_at, lane);
        sa.load(x, min(g + WAVES, groups - 1));
        multiply<PIECES, TOKENS>(acc, v, tokens_at, lane);
    }
    __syncthreads();
    float* part = (float*)lds;
    const int r = lane % 16, q = lane / 16;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[((wave * 2 + i) * 16 + 4 * q + e) * PITCH + r] = acc[0][i][e];
    __syncthreads();
    if (threadIdx.x >= 16) return;
    // a unit a thread, and zeros past the last one, to the row's end
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v)
#pragma unroll
        for (int n = 0; n < PIECES; ++n) {
            g += part[((v * 2) * 16 + threadIdx.x) * PITCH + n * TOKENS];
            u += part[((v * 2 + 1) * 16 + threadIdx.x) * PITCH + n * TOKENS];
        }
    const float h = (int)threadIdx.x < rows ? act_of(g, u, share) : 0.0f;
    float all[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) all[i] = __shfl(h, (int)(threadIdx.x * 8 + i) % 16);
    if (threadIdx.x < 2) store_act<8>(a, w, choice, j0 + 8 * threadIdx.x, all);
}

// A wave's sums of a tile (PIECES of a token in as many columns), of tokens lane % TOKENS.
template <int PIECES, int TOKENS, int N>
__device__ inline f32x4 token_sums(const f32x4 (&acc)[fragments_of(PIECES, TOKENS)][N], int i)
{
    f32x4 v = acc[0][i];
    if constexpr (TOKENS == 16) {
#pragma unroll
        for (int n = 1; n < PIECES; ++n) v += acc[n][i];
    } else if constexpr (TOKENS == 8 && PIECES > 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], 8);  // (the same in either order)
        if constexpr (PIECES == 3) v += acc[1][i];
    }
    return v;
}

// A tile's tokens times two blocks of 16 rows, by a workgroup of four waves (rows stay within a wave:
// mx4_rows.hpp).
//   SPLIT false: the rows are each wave's own, and the tokens' terms are in LDS for all of them, a group
// after another, the next one on its way.  Tokens are read and laid out once for 128 rows.
//   SPLIT true: the waves share the terms of the same rows, a group each by turns, and add up at the end.
// Four times the workgroups, where the others would leave CUs idle.
//   AHEAD: groups of rows under way.  One is enough where a CU has several workgroups (8 x 4096 x 2048, 4 of 32:
// fp32 74 us, with two 85, fp16 70 and 72), but for the first product of tokens of one piece (16 x 2048 x 1024,
// 8 of 64, bf16: 59.3, with two 57.6).
template <int PIECES, int TOKENS, bool SPLIT, int AHEAD>
struct TileProduct {
    static constexpr int STAGE = tokens_bytes(PIECES, TOKENS), STAGES = SPLIT ? kTileWaves : 2;
    static constexpr int BYTES = STAGES * STAGE + kTileWaves * rows4_bytes(2);
    static constexpr int FRAGMENTS = fragments_of(PIECES, TOKENS);
    // a thread's chunks of a piece: of the tokens (its number + THREADS i) / 32
    static constexpr int THREADS = SPLIT ? 64 : 64 * kTileWaves, LOADS = TOKENS * 32 / THREADS;
    f32x4 acc[FRAGMENTS][2];  // SPLIT: the first wave's

    // s0, s1: the rows, at least one of each; x: the tokens' pieces, `stride` apart, token t's offset_of(t)
    // bytes from there or not there (kOutside).
    template <typename F>
    __device__ inline void run(const Source4<1>& s0, const Source4<1>& s1, int nb, const uint8_t* tokens, int64_t stride,
                               F&& offset_of, char* lds, int lane, int wave)
    {
        constexpr int STEP = SPLIT ? kTileWaves : 1;
        const int groups = (nb + 7) / 8, me = SPLIT ? lane : threadIdx.x, first = SPLIT ? wave : 0;
        char *own = lds + STAGES * STAGE + wave * rows4_bytes(2), *stage = lds + (SPLIT ? wave * STAGE : 0);
        int at[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int from = offset_of((me + THREADS * i) / 32);
            at[i] = from == kOutside ? kOutside : from + lane % 32 * 16;
        }
        u32x4 x[LOADS][PIECES];
        auto load_tokens = [&](int g) {
#pragma unroll
            for (int n = 0; n < PIECES; ++n) {
                const __amdgpu_buffer_rsrc_t v = buffer_of(tokens + n * stride, 0x7fffffff);
#pragma unroll
                for (int i = 0; i < LOADS; ++i)
                    x[i][n] = __builtin_bit_cast(
                        u32x4, __builtin_amdgcn_raw_buffer_load_b128(v, at[i], min(g, groups - 1) * 512, 0));
            }
        };
        auto put_tokens = [&](char* to) {
#pragma unroll
            for (int n = 0; n < PIECES; ++n)
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int row = n * TOKENS + (me + THREADS * i) / 32;
                    *(u32x4*)(to + row * 512 + (lane % 32 ^ row % 16) * 16) = x[i][n];
                }
        };
        Rows4<1> w0[AHEAD], w1[AHEAD];
        load_tokens(first);
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
            const int g = first + d * STEP;
            s0.load(w0[d], g, nb - 8 * g);
            s1.load(w1[d], g, nb - 8 * g);
        }
        if constexpr (!SPLIT) {
            put_tokens(stage);
            load_tokens(1);
            lds_barrier();
        }
#pragma unroll
        for (int f = 0; f < FRAGMENTS; ++f) acc[f][0] = acc[f][1] = f32x4{};
        for (int g = first; g < groups;) {
#pragma unroll
            for (int d = 0; d < 2; ++d) {  // (not SPLIT: stage g % 2)
                bf16x8 v[2][8];
                if (nb - 8 * g < 8) {
                    w0[d % AHEAD].code[0] = first_bytes(w0[d % AHEAD].code[0], nb - 8 * g);
                    w1[d % AHEAD].code[0] = first_bytes(w1[d % AHEAD].code[0], nb - 8 * g);
                }
                const Rows4<2> both = {{w0[d % AHEAD].v[0], w0[d % AHEAD].v[1], w1[d % AHEAD].v[0], w1[d % AHEAD].v[1]}, {w0[d % AHEAD].code[0], w1[d % AHEAD].code[0]}};
                fragments(both, own, lane, v);
                const int next = g + AHEAD * STEP;
                s0.load(w0[d % AHEAD], next, nb - 8 * next);
                s1.load(w1[d % AHEAD], next, nb - 8 * next);
                if constexpr (SPLIT) {
                    put_tokens(stage);
                    load_tokens(g + STEP);
                    multiply<PIECES, TOKENS>(acc, v, stage, lane);
                } else {
                    put_tokens(stage + (1 - d) * STAGE);  // its last readers passed the barrier before
                    load_tokens(g + 2);
                    multiply<PIECES, TOKENS>(acc, v, stage + d * STAGE, lane);
                    lds_barrier();
                }
                g += STEP;
                if (g >= groups) break;
            }
        }
        if constexpr (SPLIT) {
            static_assert(kTileWaves * FRAGMENTS * 2 * 64 * 16 <= BYTES, "");
            f32x4* part = (f32x4*)lds;
            __syncthreads();
            if (wave > 0)
#pragma unroll
                for (int f = 0; f < FRAGMENTS; ++f)
#pragma unroll
                    for (int i = 0; i < 2; ++i) part[((wave * FRAGMENTS + f) * 2 + i) * 64 + lane] = acc[f][i];
            __syncthreads();
            if (wave == 0)
#pragma unroll
                for (int f = 0; f < FRAGMENTS; ++f)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int o = 1; o < kTileWaves; ++o) acc[f][i] += part[((o * FRAGMENTS + f) * 2 + i) * 64 + lane];
        }
    }
};

// A workgroup's tile: the blockIdx.y-th when the chunk's choices are sorted by expert and each expert's
// tokens, in order, cut into tiles of TOKENS.  Every workgroup sorts them itself, from the experts chosen:
// as bits, a token chooses an expert once.  (One workgroup that wrote a list for all took 11 us of its
// one CU for 64 tokens and 32 experts, and the list's way through memory.)
constexpr int kMoeChoices = kMoeChunk * 16;
struct Choices {  // in the LDS of the product that comes after
    uint64_t tokens_of[kMaxExperts];  // as bits
    int expert_of[kMoeChoices];
};
template <int TOKENS>
struct Tile {
    int choice_of[TOKENS], expert, skip, total, sums[kTileWaves];

    // Before: nothing in tokens_of.
    static __device__ inline void clear(Choices& x)
    {
        for (int e = threadIdx.x; e < kMaxExperts; e += 64 * kTileWaves) x.tokens_of[e] = 0;
        __syncthreads();
    }
    // A choice of the chunk, by any thread.
    static __device__ inline void put(Choices& x, const Mx4MoeArgs& a, int c, int e)
    {
        x.expert_of[c] = e;
        atomicOr((unsigned long long*)&x.tokens_of[e], 1ull << c / a.topk);
    }
    static __device__ inline void put_all(Choices& x, const Mx4MoeArgs& a, const Mx4MoeWork& w, int first, int count)
    {
        for (int c = threadIdx.x; c < count; c += 64 * kTileWaves)
            put(x, a, c, ((const int*)(a.work + w.chosen))[first + c]);
    }
    // After: whether there is the tile; its tokens' number, its expert and choices (of the chunk).
    __device__ inline int find(const Choices& x, const Mx4MoeArgs& a, int lane, int wave)
    {
        __syncthreads();
        // two experts a thread, of as many waves as that takes: tiles of the experts before
        constexpr int PER = kMaxExperts / (64 * kTileWaves);
        static_assert(PER == 2, "");
        const int used = (a.experts + 2 * 64 - 1) / (2 * 64), e = 2 * threadIdx.x;
        int n0 = 0, n1 = 0, sum = 0;
        if (wave < used) {
            n0 = (__popcll(x.tokens_of[e]) + TOKENS - 1) / TOKENS;
            n1 = (__popcll(x.tokens_of[e + 1]) + TOKENS - 1) / TOKENS;
            sum = n0 + n1;
            for (int d = 1; d < 64; d *= 2) {
                const int v = __shfl_up(sum, d);
                if (lane >= d) sum += v;
            }
            if (lane == 63) sums[wave] = sum;
        }
        if (used > 1) __syncthreads();
        if (wave < used) {
            for (int v = 0; v < wave; ++v) sum += sums[v];
            const int at = blockIdx.y - (sum - n0 - n1);
            if (at >= 0 && at < n0 + n1) {
                expert = at < n0 ? e : e + 1;
                skip = (at < n0 ? at : at - n0) * TOKENS;
            }
            if (wave == used - 1 && lane == 63) total = sum;
        }
        __syncthreads();
        if ((int)blockIdx.y >= total) return 0;
        const uint64_t mask = x.tokens_of[expert];
        if (threadIdx.x < kMoeChunk && (mask >> threadIdx.x & 1)) {
            const int place = __popcll(mask & ((1ull << threadIdx.x) - 1)) - skip;
            if (place >= 0 && place < TOKENS) {
                int c = threadIdx.x * a.topk;
                while (x.expert_of[c] != expert) ++c;  // (it is there)
                choice_of[place] = c;
            }
        }
        __syncthreads();
        return min(__popcll(mask) - skip, TOKENS);
    }
};

struct Shares {
    float of[kFewTokens * 16];
};
template <int TOKENS>
__device__ inline void choose_few(const Mx4MoeArgs& a, const Mx4MoeWork& w, Choices& choices, Shares& shares, int lane,
                                  int wave)
{
    for (int t = wave; t < a.tokens; t += kTileWaves) {
        const double* logits = (const double*)(a.work + w.logits) + t * a.experts;
        Chooser<1> from;
        from.init(logits, a.experts, lane);
        int mine = 0;
        for (int k = 0; k < a.topk; ++k) {
            const int e = from.next(k, lane);
            if (lane == k) mine = e;
        }
        const float p = from.share(logits, a.experts, a.topk, a.normalize, lane);
        if (lane >= a.topk) continue;
        const int c = t * a.topk + lane;
        Tile<TOKENS>::put(choices, a, c, mine);
        shares.of[c] = p;
        if (blockIdx.x > 0 || blockIdx.y > 0) continue;
        ((int*)(a.work + w.chosen))[c] = mine;  // for the second product
        if (a.chosen) a.chosen[c] = mine;
        if (a.weights) a.weights[c] = p;
    }
}

// 16 units a wave (SPLIT: a workgroup): its rows of G and of U.
template <typename T, int TOKENS, bool SPLIT, bool FEW>
__global__ void __launch_bounds__(64 * kTileWaves) up_kernel(Mx4MoeArgs a, Mx4MoeWork w)
{
    constexpr int PIECES = kBf16Pieces<T>;
    typedef TileProduct<PIECES, TOKENS, SPLIT, PIECES == 1 ? 2 : 1> product_t;
    __shared__ __align__(16) char lds[product_t::BYTES];
    __shared__ Tile<TOKENS> tile;
    __shared__ typename std::conditional<FEW, Shares, int>::type shares;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int first = blockIdx.z * kMoeChunk * a.topk;  // the chunk's first choice
    Choices& choices = *(Choices*)lds;
    static_assert(sizeof(Choices) <= product_t::BYTES, "");
    tile.clear(choices);
    if constexpr (FEW)
        choose_few<TOKENS>(a, w, choices, shares, lane, wave);
    else
        tile.put_all(choices, a, w, first, min(a.tokens * a.topk - first, kMoeChunk * a.topk));
    const int count = tile.find(choices, a, lane, wave);
    if (count == 0) return;
    const int expert = __builtin_amdgcn_readfirstlane(tile.expert);
    const int j0 = (SPLIT ? blockIdx.x : blockIdx.x * kTileWaves + wave) * 16, nb = (a.width + 31) / 32, rows = min(a.hidden - j0, 16);
    Source4<1> sg, su;
    sg.init(a.ld1, a.lds1, rows > 0 ? rows : 1, nb, lane);
    su = sg;
    // (past the last unit: the last one's rows, not used)
    sg.move(a.W1, a.S1, (int64_t)expert * 2 * a.hidden + min(j0, a.hidden - 1));
    su.move(a.W1, a.S1, (int64_t)expert * 2 * a.hidden + a.hidden + min(j0, a.hidden - 1));
    product_t product;
    product.run(sg, su, nb, a.work + w.x, w.x_stride,
                [&](int t) { return t < count ? (first + tile.choice_of[t]) / a.topk * w.x_ld : kOutside; }, lds, lane, wave);
    if (SPLIT && wave > 0) return;
    const int t = lane % 16, q = lane / 16;
    const f32x4 gate = token_sums<PIECES, TOKENS>(product.acc, 0), up = token_sums<PIECES, TOKENS>(product.acc, 1);
    if (t >= count) return;
    const int choice = first + tile.choice_of[t];
    float share;
    if constexpr (FEW)
        share = shares.of[choice];
    else
        share = ((const float*)(a.work + w.weights))[choice];
    float h[8] = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = 4 * q + e < rows ? act_of(gate[e], up[e], share) : 0.0f;
    store_act<4>(a, w, choice, j0 + 4 * q, h);
}

// 32 results a wave (SPLIT: a workgroup), of each choice apart.
template <typename T, int TOKENS, bool SPLIT>
__global__ void __launch_bounds__(64 * kTileWaves) down_kernel(Mx4MoeArgs a, Mx4MoeWork w)
{
    constexpr int PIECES = kActPieces;
    typedef TileProduct<PIECES, TOKENS, SPLIT, 1> product_t;
    __shared__ __align__(16) char lds[product_t::BYTES];
    __shared__ Tile<TOKENS> tile;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int first = blockIdx.z * kMoeChunk * a.topk;  // the chunk's first choice
    Choices& choices = *(Choices*)lds;
    static_assert(sizeof(Choices) <= product_t::BYTES, "");
    tile.clear(choices);
    tile.put_all(choices, a, w, first, min(a.tokens * a.topk - first, kMoeChunk * a.topk));
    const int count = tile.find(choices, a, lane, wave);
    if (count == 0) return;
    const int expert = __builtin_amdgcn_readfirstlane(tile.expert);
    const int n0 = (SPLIT ? blockIdx.x : blockIdx.x * kTileWaves + wave) * 32, nb = (a.hidden + 31) / 32;
    Source4<1> s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // (past the last row: that one, not used)
        const int at = min(n0 + 16 * i, a.width - 1);
        s[i].init(a.ld2, a.lds2, a.width - at, nb, lane);
        s[i].move(a.W2, a.S2, (int64_t)expert * a.width + at);
    }
    product_t product;
    product.run(s[0], s[1], nb, a.work + w.act + (size_t)first * w.act_ld, w.act_stride,
                [&](int t) { return t < count ? tile.choice_of[t] * w.act_ld : kOutside; }, lds, lane, wave);
    if (SPLIT && wave > 0) return;
    const int t = lane % 16, q = lane / 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x4 v = token_sums<PIECES, TOKENS>(product.acc, i);
        const int n = n0 + 16 * i + 4 * q;
        // (rows of `out` are whole 16 bytes)
        if (t < count && n < a.width)
            *(f32x4*)(a.work + w.out + ((size_t)(first + tile.choice_of[t]) * w.out_ld + n) * 4) = v;
    }
}

// A token's sum over its choices, in their order.
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(Mx4MoeArgs a, Mx4MoeWork w)
{
    const int n = (blockIdx.x * 256 + threadIdx.x) * 4, t = blockIdx.y;
    if (n >= a.width) return;
    const float* from = (const float*)(a.work + w.out) + (size_t)t * a.topk * w.out_ld + n;
    f32x4 v = {};
    for (int j = 0; j < a.topk; j += 4) {  // four loads under way
        f32x4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *(const f32x4*)(from + (size_t)min(j + i, a.topk - 1) * w.out_ld);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (j + i < a.topk) v += x[i];
    }
    T* y = (T*)a.Y + t * a.ldy + n;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < a.width) y[e] = (T)v[e];
}

// The only token's: 16 results a workgroup.  Its choices times their groups of terms are cut into one run
// for each of 16 waves, whose sums are added up in LDS, in order.
template <typename T>
__global__ void __launch_bounds__(1024) down_one_kernel(Mx4MoeArgs a, Mx4MoeWork w)
{
    constexpr int WAVES = 16, TOKENS = 2, PIECES = kActPieces, OWN = rows4_bytes(1) + tokens_bytes(PIECES, TOKENS);
    __shared__ __align__(16) char lds[WAVES * OWN];
    __shared__ float part[WAVES][16];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int n0 = blockIdx.x * 16, *experts = (const int*)(a.work + w.chosen);
    char *own = lds + wave * OWN, *tokens_at = own + rows4_bytes(1);
    const int nb = (a.hidden + 31) / 32, groups = (nb + 7) / 8;
    const int units = a.topk * groups, from = units * wave / WAVES, to = units * (wave + 1) / WAVES;
    f32x4 acc[1][1] = {};
    if (from < to) {
        struct Place {  // a choice and a group of its terms
            int choice, g;
        };
        auto after = [&](Place p) { return p.g + 1 < groups ? Place{p.choice, p.g + 1} : Place{p.choice + 1, 0}; };
        Source4<1> sw;
        sw.init(a.ld2, a.lds2, a.width - n0, nb, lane);
        PieceTokens<PIECES, TOKENS> sa;
        sa.base = a.work + w.act;
        sa.stride = w.act_stride;
        auto load_rows = [&](Rows4<1>& d, Place p) {  // (past the last choice: the last one again)
            const int e = __builtin_amdgcn_readfirstlane(experts[min(p.choice, a.topk - 1)]);
            sw.move(a.W2, a.S2, (int64_t)e * a.width + n0);
            sw.load(d, p.g, nb - 8 * p.g);
        };
        typename PieceTokens<PIECES, TOKENS>::Values x;
        auto load_tokens = [&](Place p) {
            const int row = min(p.choice, a.topk - 1) * w.act_ld;
            sa.move([&](int t) { return t > 0 ? kOutside : row; }, lane);
            sa.load(x, p.g);
        };
        Rows4<1> rows;
        Place now{from / groups, from % groups}, next = after(now);
        load_rows(rows, now);
        load_tokens(now);
        for (int u = from; u < to; ++u) {
            bf16x8 v[1][8];
            if (nb - 8 * now.g < 8) rows.code[0] = first_bytes(rows.code[0], nb - 8 * now.g);
            fragments(rows, own, lane, v);
            load_rows(rows, next);
            sa.put(x, tokens_at, lane);
            load_tokens(next);
            multiply<PIECES, TOKENS>(acc, v, tokens_at, lane);
            now = next;
            next = after(next);
        }
    }
    // pieces are in columns 0, 2 and 4
    f32x4 sum = acc[0][0];
#pragma unroll
    for (int n = 1; n < PIECES; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += __shfl_down(acc[0][0][e], 2 * n);
    if (lane % 16 == 0)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[wave][lane / 4 + e] = sum[e];
    __syncthreads();
    const int n = n0 + (int)threadIdx.x;
    if (threadIdx.x >= 16 || n >= a.width) return;
    float y = 0.0f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) y += part[v][threadIdx.x];
    ((T*)a.Y)[n] = (T)y;
}

// The products of more than one token, in tiles of UP and DOWN; FEW: that choose in the first one.
template <typename T, int UP, int DOWN, bool FEW>
void launch_tiles(const Mx4MoePlan& p, const Mx4MoeArgs& a, const Mx4MoeWork& w, hipStream_t s)
{
    if constexpr (!FEW) {
        const unsigned waves = (unsigned)((a.tokens + 3) / 4);
        if (p.each == 1)
            choose_kernel<1><<<waves, 256, 0, s>>>(a, w);
        else if (p.each == 2)
            choose_kernel<2><<<waves, 256, 0, s>>>(a, w);
        else
            choose_kernel<8><<<waves, 256, 0, s>>>(a, w);
    }
    const unsigned up_x = (unsigned)(w.act_ld / 32);  // 16 units each, to the end of a row of the workspace
    const unsigned down_x = (unsigned)((a.width + 31) / 32), down_w = (down_x + kTileWaves - 1) / kTileWaves;
    if (p.up_rows)
        up_kernel<T, UP, false, FEW><<<dim3(up_x / kTileWaves, p.up_tiles, p.chunks), 64 * kTileWaves, 0, s>>>(a, w);
    else
        up_kernel<T, UP, true, FEW><<<dim3(up_x, p.up_tiles, p.chunks), 64 * kTileWaves, 0, s>>>(a, w);
    if (p.down_rows)
        down_kernel<T, DOWN, false><<<dim3(down_w, p.down_tiles, p.chunks), 64 * kTileWaves, 0, s>>>(a, w);
    else
        down_kernel<T, DOWN, true><<<dim3(down_x, p.down_tiles, p.chunks), 64 * kTileWaves, 0, s>>>(a, w);
    combine_kernel<T><<<dim3((unsigned)((a.width + 1023) / 1024), (unsigned)a.tokens), 256, 0, s>>>(a, w);
}

template <typename T>
hipError_t launch(const Mx4MoeArgs& a, hipStream_t s)
{
    const Mx4MoeWork w = mx4_moe_work(a.tokens, a.width, a.hidden, a.experts, a.topk);
    const Mx4MoePlan p = mx4_moe_plan(kBf16Pieces<T>, a.tokens, a.width, a.hidden, a.experts, a.topk);
    const int expert_groups = (a.experts + 3) / 4, pieces = (w.x_ld / 16 * a.tokens + 255) / 256;
    const unsigned prepare_x = (unsigned)(expert_groups + pieces);
    if (p.one) {
        prepare_kernel<T, 1><<<prepare_x, 256, 0, s>>>(a, w, expert_groups);
        const dim3 up((unsigned)(w.act_ld / 32), (unsigned)a.topk);
        if (p.each == 1)
            up_one_kernel<T, 1><<<up, 512, 0, s>>>(a, w);
        else if (p.each == 2)
            up_one_kernel<T, 2><<<up, 512, 0, s>>>(a, w);
        else
            up_one_kernel<T, 8><<<up, 512, 0, s>>>(a, w);
        down_one_kernel<T><<<(unsigned)((a.width + 15) / 16), 1024, 0, s>>>(a, w);
    } else {
        prepare_kernel<T, 4><<<dim3(prepare_x, (unsigned)((a.tokens + 3) / 4)), 256, 0, s>>>(a, w, expert_groups);
        constexpr int UP = kBf16Pieces<T> == 1 ? 16 : 8;
        if (p.few)
            launch_tiles<T, UP, 8, true>(p, a, w, s);
        else if (p.down == 16)
            launch_tiles<T, 16, 16, false>(p, a, w, s);
        else
            launch_tiles<T, UP, 8, false>(p, a, w, s);
    }
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
