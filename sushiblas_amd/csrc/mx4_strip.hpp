// mx4_strip.hpp -- where the MXFP4 product's narrow kernel (mx4_gemm.hip) reads an
// operand: a strip of up to 16 N rows, 8 blocks of 32 elements (128 bytes) of each at
// a time.  Plain arithmetic, so that a host program can check it against a matrix's end.
//
// A buffer load's range check is certain to test the vector offset only, not the scalar
// offset that is added to it.  So what lies outside the operand gets a vector offset past
// every descriptor's end (and then reads zeros), and the scalar offset, which moves an
// inner place by rows and groups, counts inside alone.
#pragma once

namespace sbx {

constexpr int kOutside = (int)0x80000000u;  // as an offset, past every descriptor's end

// Bytes from the strip's first row to the end of its last one: `count` rows, ld bytes
// apart, of `blocks` blocks.
constexpr int strip_bytes(int count, int ld, int blocks) { return (count - 1) * ld + 16 * blocks; }

// A lane's place in rows 16 i .. + 15: row lane % 16 of them, blocks 2 (lane / 16) and the
// next of a group; outside past the strip's last row.
constexpr int strip_lane(int lane, int i, int count, int ld)
{
    return 16 * i + lane % 16 < count ? lane % 16 * ld + lane / 16 * 32 : kOutside;
}

// The vector offset of its block `half` (0, 1) of a group with `left` blocks up to the last.
constexpr int strip_vector(int lane_at, int lane, int half, int left)
{
    return lane / 16 * 2 + half < left ? lane_at + 16 * half : kOutside;
}

// The scalar offset of rows 16 i and group g.
constexpr int strip_scalar(int i, int g, int count, int ld, int left)
{
    return left > 0 && 16 * i < count ? 16 * i * ld + 128 * g : 0;
}

}  // namespace sbx
