// Microscaled 4-bit floating point (OCP MX): elements of 4 bits (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives),
// one power of two (E8M0: byte b stands for 2^(b - 127), 255 for not a number) for every 32 elements along a row.
//
//   codes   uint8 [..., R, Kp / 2]: Kp is K rounded up to 128; element 2i in the low half of byte i; zero beyond K
//   scales  uint8 [..., ceil(R / 128), Kp / 128, 512]: a tile of 128 rows by four blocks, the layout in which the tensor
//           cores' scale factors are copied to tensor memory: the byte of row r, block b at
//           (r % 32) * 16 + r % 128 / 32 * 4 + b % 4; zero for blocks beyond K, anything for rows beyond R
//
// A block's exponent is that of its largest magnitude less two (6 = 1.5 * 2^2 is the largest element), at least -127;
// elements round to nearest, ties to the even code, and saturate at 6.  Values are exact in bfloat16.  A block that
// holds an infinity or NaN gets byte 255 and codes 0: all of its values are NaN.
#pragma once

#include "common.cuh"

namespace prism {
namespace mx {

constexpr int BLOCK = 32, GROUP = 128, TILE_ROWS = 128, TILE_BYTES = 512;
constexpr int WORKSPACE_TOO_SMALL = -1;        // an entry's answer before it launches anything

__host__ __device__ __forceinline__ int groups_of(int K) { return (K + GROUP - 1) / GROUP; }

// the scale byte of a block from the bits of its largest magnitude (an integer maximum: NaN and infinity win)
__device__ __forceinline__ int scale_byte(uint32_t most) {
    return most >= 0x7f800000u ? 255 : max((int)(most >> 23) - 2, 0);
}
// 2^(127 - byte), the factor that brings a block's values into the elements' range
__device__ __forceinline__ float scale_inverse(int byte) { return __uint_as_float((uint32_t)(254 - min(byte, 253)) << 23); }
// 2^(byte - 127), NaN for 255
__device__ __forceinline__ float scale_value(int byte) {
    return byte == 255 ? __uint_as_float(0x7fffffffu) : byte ? __uint_as_float((uint32_t)byte << 23) : __uint_as_float(0x00400000u);
}
// the values of a byte's two codes (the low half first), exact in half precision
__device__ __forceinline__ float2 elements2(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(byte));
    float2 v;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(v.x), "=f"(v.y) : "r"(h));
    return v;
}
// two values to 4 bits each, `lo` in the low half of the byte
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}

}  // namespace mx
}  // namespace prism
