// MXFP4 matrices: blocks of 32 values along a row, each block 16 bytes of e2m1
// codes (value 2i in the low half of byte i) and one scale byte b for 2^(b - 127)
// (255: the block is NaN). A ragged last block is filled up with zero codes, so a
// row holds ceil(cols / 32) whole blocks and every row of codes is 16-byte sized.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace swb {

constexpr int kMxBlock = 32;       // values per scale
constexpr int kMxBlockBytes = 16;  // bytes of codes per block

__host__ __device__ inline int64_t mx_blocks(int64_t cols) { return (cols + kMxBlock - 1) / kMxBlock; }

// 2^(b - 127) for one scale byte: the byte is the exponent field, except that 0
// is the subnormal 2^-127 and 255 is NaN.
__device__ __forceinline__ float mx_scale(uint32_t b) {
    uint32_t bits = b << 23;
    if (b == 0u) bits = 0x00400000u;
    if (b == 255u) bits = 0x7FC00000u;
    return __uint_as_float(bits);
}

// The four bytes of `w` as pairs of e2m1 codes -> four fp16 pairs (exact), in order.
__device__ __forceinline__ void mx_decode_f16(uint32_t w, uint32_t (&p)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3])
        : "r"(w));
}

// Eight codes -> four bf16 pairs (exact), pair i = (code i, code i + 4). The three
// magnitude bits of a code, moved to the lowest exponent bits and the highest
// mantissa bit, read as bf16, are the value times 2^-126 (subnormals included), so
// one exact multiplication by 2^126 finishes it.
__device__ __forceinline__ void mx_decode_bf16(uint32_t w, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t t = w << (12 - 4 * i);  // code i at bits 12..15, code i + 4 at bits 28..31
        const uint32_t v = (t & 0x80008000u) | ((t >> 6) & 0x01C001C0u);
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(v), "r"(0x7E807E80u));
    }
}

// Two fp32 values (already divided by the block's scale) -> one byte of codes, `lo`
// in the low half: nearest, ties to the even code, beyond 6 to 6.
__device__ __forceinline__ uint32_t mx_encode(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 b;\n\t.reg .b16 h;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n\t"
        "mov.b16 h, {b, 0};\n\t"
        "cvt.u32.u16 %0, h;\n\t}"
        : "=r"(r)
        : "f"(lo), "f"(hi));
    return r;
}

}  // namespace swb
