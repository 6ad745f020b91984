// pieces.hpp -- 16-byte pieces of a row at any alignment and place, and sums over lanes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx4.hpp"

namespace sbx {

// How a row of `cols` values is cut into pieces of N: whole ones only, with one that straddles its
// end, or shorter than a piece.
enum class Cut { Whole, Ragged, Short };
template <typename T>
inline Cut cut_of(int64_t cols)
{
    constexpr int N = Piece<T>::N;
    return cols % N == 0 ? Cut::Whole : cols > N ? Cut::Ragged : Cut::Short;
}

// Values c .. of a row for trim_piece, without a branch around the load: a piece that reaches past
// the end is read that much earlier.
template <Cut CUT, typename T>
__device__ inline Piece<T> load_piece(const T* row, int c, int cols)
{
    constexpr int N = Piece<T>::N;
    if constexpr (CUT == Cut::Short) {
        u32x4 y = {};
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < cols) {
                if constexpr (sizeof(T) == 2)
                    y[i / 2] |= (uint32_t)((const uint16_t*)row)[c + i] << i % 2 * 16;
                else
                    y[i] = ((const uint32_t*)row)[c + i];
            }
        return __builtin_bit_cast(Piece<T>, y);
    }
    return *(const Piece<T>*)(row + (c + N <= cols ? c : cols - N));
}

// The piece that load_piece read, moved to its place, zeros from the row's end on.  Apart from the
// load, so that all of a lane's loads are under way before the first is waited for; only the waves
// that hold a row's end do more than test for it (the norm of 8192 x 8191 bf16, with the residual,
// 103 us against 159 with the shift at each load).
template <Cut CUT, typename T>
__device__ inline void trim_piece(Piece<T>& x, int c, int cols)
{
    constexpr int N = Piece<T>::N;
    if constexpr (CUT == Cut::Short) return;
    if constexpr (CUT == Cut::Whole) {
        const u32x4 v = __builtin_bit_cast(u32x4, x);
        x = __builtin_bit_cast(Piece<T>, c < cols ? v : u32x4{});
        return;
    }
    if (__builtin_amdgcn_ballot_w64(c + N > cols) == 0) return;
    struct Words {
        uint64_t lo, hi;
    };
    Words v = __builtin_bit_cast(Words, x);
    const int past = c + N - cols, by = past <= 0 ? 0 : past < N ? past * (int)(8 * sizeof(T)) : 128;
    const uint64_t hi = by < 128 ? v.hi : 0;
    v.lo = by < 64 ? v.lo >> by | (hi << 1) << (63 - by) : hi >> (by & 63);
    v.hi = by < 64 ? hi >> by : 0;
    x = __builtin_bit_cast(Piece<T>, v);
}

template <Cut CUT, typename T>
__device__ inline Piece<T> whole_piece(const T* row, int c, int cols)
{
    Piece<T> x = load_piece<CUT>(row, c, cols);
    trim_piece<CUT>(x, c, cols);
    return x;
}

// Stores what of a piece lies inside the row; where rows begin inside lines, past the L2s (the norm
// of 2047 x 4095 fp16, with the residual, 14.7 us against 19.0; aligned ones take as long either way).
template <Cut CUT, typename T>
__device__ inline void store_piece(T* row, int c, int cols, const Piece<T>& y)
{
    constexpr int N = Piece<T>::N;
    if (CUT == Cut::Whole) {
        if (c < cols) *(Piece<T>*)(row + c) = y;
    } else if (c + N <= cols)
        store_past(row + c, y);
    else if (CUT != Cut::Whole)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < cols) row[c + i] = y.v[i];
}

// What follows takes this piece from its registers again: the compiler would keep its values
// converted, in twice as many or four times.
template <typename T>
__device__ inline void keep_packed(Piece<T>& x)
{
    u32x4 v = __builtin_bit_cast(u32x4, x);
    asm("" : "+v"(v));
    x = __builtin_bit_cast(Piece<T>, v);
}

// x of the lane that a DPP control names.
template <int CTRL>
__device__ inline double other_lane(double x)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140;

// The sum over the 16 lanes of a row of the wave, in each.
__device__ inline double sum16(double x)
{
    x += other_lane<kDppXor1>(x);
    x += other_lane<kDppXor2>(x);
    x += other_lane<kDppHalfMirror>(x);
    return x + other_lane<kDppMirror>(x);
}

__device__ inline double lane_value(double x, int lane)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The sum over a wave.
__device__ inline double sum64(double x)
{
    x = sum16(x);
    return lane_value(x, 0) + lane_value(x, 16) + (lane_value(x, 32) + lane_value(x, 48));
}

}  // namespace sbx
