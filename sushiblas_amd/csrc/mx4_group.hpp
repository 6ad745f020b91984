// mx4_group.hpp -- how the kernels for a narrow operand read an MXFP4 matrix: straight from
// memory to a wave's registers, 256 elements (8 blocks, a group of codes) of 16 rows at a time,
// 32 neighbouring bytes of a row to a lane.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx4_strip.hpp"

namespace sbx {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int kRsrcWord3 = 0x00020000;

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ inline i32x8 widen(i32x4 v)
{
    return i32x8{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
}

template <int N>
struct Group {
    i32x4 v[N][2];
    int code[N];  // two codes in its low bytes
};

// The rows of an operand that a workgroup takes, and the lane's place in them (mx4_strip.hpp).
template <int N>
struct Strip {
    const uint8_t *rows, *codes;
    int64_t lds;
    int bytes, count, ld, lane, at[N], code_at;

    __device__ inline void init(const uint8_t* P, int64_t ld_, const uint8_t* S, int64_t lds_, int first, int n,
                                int nb, int lane_)
    {
        count = min(n - first, 16 * N);
        ld = (int)ld_;
        lds = lds_;
        lane = lane_;
        rows = P + first * ld_;
        bytes = strip_bytes(count, ld, nb);
        codes = S + 8 * (int64_t)first;
#pragma unroll
        for (int i = 0; i < N; ++i) at[i] = strip_lane(lane, i, count, ld);
        code_at = lane % 16 * 8 + lane / 16 * 2;
    }

    // Group g (256 terms), with `left` blocks up to the last: zeros, not from memory, past it
    // and past the last row.  The codes of a group's 8 blocks are all there.
    __device__ inline void load(Group<N>& d, int g, int left) const
    {
        const __amdgpu_buffer_rsrc_t v =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(rows), (short)0, bytes, kRsrcWord3);
        const __amdgpu_buffer_rsrc_t c = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(codes) + g * lds, (short)0, left > 0 ? 8 * count : 0, kRsrcWord3);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int from = strip_scalar(i, g, count, ld, left);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                d.v[i][h] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                          v, strip_vector(at[i], lane, h, left), from, 0));
            d.code[i] = __builtin_amdgcn_raw_buffer_load_b16(c, code_at + 128 * i, 0, 0);
        }
    }
};

// Codes past the last block may be NaN's and are cleared (the elements there are zeros):
// `mine` of the lane's two blocks are inside.
template <int N>
__device__ inline void clip(Group<N>& d, int mine)
{
#pragma unroll
    for (int i = 0; i < N; ++i) d.code[i] = mine >= 2 ? d.code[i] : mine == 1 ? d.code[i] & 0xff : 0;
}

}  // namespace sbx
