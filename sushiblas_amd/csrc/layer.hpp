// layer.hpp -- what surrounds a layer with MXFP4 weights: the root-mean-square norm
// and its gradient, the product for a few tokens, the mixture-of-experts layer.
// Their arguments and launchers.
//
// An MXFP8 matrix is an MXFP4 one (mx4.hpp) with e4m3 elements, one a byte: 32 bytes
// a block, codes in the same places, the largest element 448 = 1.75 * 2^8.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx4.hpp"

namespace sbx {

struct NormArgs {
    int64_t rows, cols;
    const void *X, *R, *W;  // R: null, or what is added to X
    int64_t ldx, ldr;
    double eps;
    void *H, *Y;  // the sum, its norm; null: not wanted
    int64_t ldh, ldy;
    Mx4Out q;  // the norm as MXFP8 (P null: not wanted)
};

struct NormGradArgs {
    int64_t rows, cols;
    const void *H, *W, *DY, *DR;  // DR: null, or a gradient that arrives at H beside the norm's
    int64_t ldh, lddy, lddr;
    double eps;
    void* DX;
    int64_t lddx;
    float* DW;    // null: not wanted
    float* part;  // with DW: up to norm_grad_parts(rows) x cols
};

// Groups of rows whose share of DW is summed apart: at most.
constexpr int kNormGradParts = 256;
inline int norm_grad_parts(int64_t rows) { return rows < kNormGradParts ? (int)rows : kNormGradParts; }

struct Mx4LinearArgs {
    int m, n, k;
    const void* X;  // dense of the result's type; with SX e4m3 elements
    int64_t ldx;
    const uint8_t* SX;
    int64_t ldsx;
    const uint8_t *B, *SB;
    int64_t ldb, ldsb;
    void* Y;
    int64_t ldy;
    float alpha, beta;
    int relu;
};

struct Mx4MoeArgs {
    int tokens, width, hidden, experts, topk;
    const void *X, *WR;
    int64_t ldx, ldwr;
    const uint8_t *W1, *S1, *W2, *S2;
    int64_t ld1, lds1, ld2, lds2;
    void* Y;
    int64_t ldy;
    int normalize;
    int* chosen;     // null: not wanted
    float* weights;  // the same
    uint8_t* work;
};

// A mixture's workspace: offsets of its parts, each 256-byte aligned.
struct Mx4MoeWork {
    size_t logits;           // tokens x experts, 64 bits
    size_t chosen, weights;  // tokens x topk
    size_t x, x_stride;      // tokens as bf16 pieces (up to 3, x_stride bytes apart), zeros to x_ld bytes
    size_t act, act_stride;  // the hidden layer times its share, one row a choice, likewise
    size_t out;              // (more than one token) each choice's results, rows of out_ld floats
    size_t bytes;
    int x_ld, act_ld, out_ld;
};
inline Mx4MoeWork mx4_moe_work(int64_t tokens, int64_t width, int64_t hidden, int64_t experts, int64_t topk)
{
    Mx4MoeWork w;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t from = at;
        at += (bytes + 255) / 256 * 256;
        return from;
    };
    w.x_ld = (int)((width + 255) / 256 * 512);
    w.act_ld = (int)((hidden + 255) / 256 * 512);
    w.logits = take(8 * tokens * experts);
    w.chosen = take(4 * tokens * topk);
    w.weights = take(4 * tokens * topk);
    w.x_stride = (size_t)w.x_ld * tokens;
    w.x = take(3 * w.x_stride);
    w.act_stride = (size_t)w.act_ld * tokens * topk;
    w.act = take(3 * w.act_stride);
    w.out_ld = (int)((width + 3) / 4 * 4);
    w.out = take(tokens > 1 ? 4 * (size_t)w.out_ld * tokens * topk : 0);
    w.bytes = at;
    return w;
}

// dtype: an sbx_dtype that the caller has checked.  hipErrorNotSupported: a grid of more than a
// launch takes.
hipError_t launch_rms_norm(int dtype, const NormArgs& a, hipStream_t s);
hipError_t launch_rms_norm_grad(int dtype, const NormGradArgs& a, hipStream_t s);
hipError_t launch_mx8_dequantize(int dtype, int64_t rows, int64_t cols, const uint8_t* P, int64_t ldp,
                                 const uint8_t* S, int64_t lds, void* Y, int64_t ldy, hipStream_t s);
hipError_t launch_mx4_linear(int dtype, const Mx4LinearArgs& a, hipStream_t s);
hipError_t launch_mx4_moe(int dtype, const Mx4MoeArgs& a, hipStream_t s);

}  // namespace sbx
