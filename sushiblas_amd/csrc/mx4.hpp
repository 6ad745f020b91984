// mx4.hpp -- the dropout and the microscaled 4-bit (MXFP4) operators: their
// arguments, launchers and shared device code.
//
// An MXFP4 matrix is the OCP microscaling format with e2m1 elements: blocks of
// 32 along a row, v = element * 2^(code - 127), one e8m0 code per block (255:
// the block is NaN).  Elements are packed two a byte, the even one in the low
// half; a row's last block is filled with zeros, so a row takes 16 bytes per
// block.  Codes lie in groups of 8 blocks (256 elements): block b of row r has
// its code at S[(b / 8) * lds + 8 * r + b % 8].  So the codes that a tile of
// rows needs for 256 elements are one run of memory, and a lane of a matrix
// instruction has the codes of its row in one 8-byte load.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "philox.hpp"

namespace sbx {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// Matrices the elementwise operators read, with their dropout.
//   keep(r, c): 16 bits of Philox (key = seed, counter = (c / 8, r, stream_id,
//   kDropoutTag); word c % 8 / 2, its half c % 2) against `threshold`.  The
//   counter comes from the place in the matrix alone, so a backward pass, or
//   another kernel, makes the same mask again and none is stored.  The last
//   counter word keeps it apart from the fills (0 there).
struct DropoutArgs {
    const void* X;
    int64_t ldx;
    const void* gate;  // null, or values that pass where they are > 0
    int64_t ldg;
    int64_t rows, cols;
    uint64_t seed;
    uint32_t stream_id;
    uint32_t threshold;  // 65536 * p, rounded; 0: no dropout
    double scale;        // 65536 / (65536 - threshold): the mean stays, whatever p rounds to
};

constexpr uint32_t kDropoutTag = 0x44524F50;

struct Mx4Out {
    uint8_t* P;  // null: not wanted
    int64_t ldp;
    uint8_t* S;
    int64_t lds;
};

struct Mx4GemmArgs {
    const uint8_t *A, *SA, *B, *SB;
    int64_t lda, ldsa, ldb, ldsb;
    void* C;
    int64_t ldc;
    int m, n, k;
    float alpha, beta;
    int relu;
    int past;  // C's rows are whole 64-byte lines
    int down;  // fp32 pieces of 16 bytes are not aligned, and C is no more than the MALL's half
};

// A launch takes less than 2^32 threads along x: workgroups (of up to 512) past the kGridX-th go
// on along z.  Some at the end have no tile then.
constexpr int64_t kMaxThreads = 0xffffffff;
constexpr int kGridX = 1 << 22;
inline dim3 grid_of(int64_t blocks, unsigned y = 1)
{
    return dim3((unsigned)(blocks < kGridX ? blocks : kGridX), y, (unsigned)((blocks + kGridX - 1) / kGridX));
}
__device__ inline uint32_t block_x() { return blockIdx.z * kGridX + blockIdx.x; }

// dtype: an sbx_dtype that the caller has checked.  hipErrorNotSupported: a grid of more than a
// launch takes.
hipError_t launch_dropout(int dtype, const DropoutArgs& a, void* Y, int64_t ldy, hipStream_t s);
hipError_t launch_mx4_quantize(int dtype, const DropoutArgs& a, const Mx4Out& rows,
                               const Mx4Out& cols, hipStream_t s);
hipError_t launch_mx4_dequantize(int dtype, int64_t rows, int64_t cols, const uint8_t* P,
                                 int64_t ldp, const uint8_t* S, int64_t lds, void* Y, int64_t ldy,
                                 hipStream_t s);
hipError_t launch_mx4_gemm(int dtype, const Mx4GemmArgs& a, hipStream_t s);

// The random numbers of columns 8 * chunk .. + 7 of a row, and whether number e stays.
__device__ inline void keep_words(const DropoutArgs& a, uint32_t row, uint32_t chunk, uint32_t (&w)[4])
{
    philox4x32(a.seed, chunk, row, a.stream_id, kDropoutTag, w);
}
__device__ inline bool kept(const DropoutArgs& a, const uint32_t (&w)[4], int e)
{
    return (e % 2 ? w[e / 2] >> 16 : w[e / 2] & 0xffff) >= a.threshold;
}

// Eight neighbouring values, in memory that is aligned to the element only (the device
// serves such 16-byte accesses).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
    T v[8];
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Sixteen bytes of neighbouring values: what a lane stores at once, so that a wave's instruction
// writes whole lines (fp32 in two such pieces a lane, 32 bytes apart between lanes: 8192^2
// dequantised 114 us, in one 46).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Piece {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};

// Stores it past the L2s.
template <typename T>
__device__ inline void store_past(T* to, const Piece<T>& y)
{
    typedef u32x4 __attribute__((aligned(2))) loose_t;  // (16-byte accesses need no alignment)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, y), (loose_t*)to);
}

}  // namespace sbx
