// The microscaled 4-bit format (MXFP4) shared by its producers and the product.
//
// A block is 32 consecutive columns of a row.  Its scale is a power of two held as the byte
// e + 127 (E8M0), e = floor(log2(max|x|)) - 2: the largest element lands in [4, 8) and the
// element format E2M1, +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, ends at 6 (values above saturate).  A block
// with a NaN or an infinity gets the NaN byte 255 and zero elements: everything computed from it
// is NaN.  Elements are packed two per byte, the even column in the low half.
//
// Scale bytes lie in tiles of 128 rows x 4 blocks (512 bytes), byte (r % 32) * 16 + (r / 32) * 4 + b
// of a tile for row r and block b: four rows 32 apart make one 16-byte line, which is how tensor
// memory wants them (32 lanes x 4 words), so a tile goes from shared memory into tensor memory in
// one copy.  Tiles follow one another along a row tile's columns: [row tile][column tile][512].
// Bytes of rows and blocks outside the matrix are written as 0 (the scale 2^-127): they meet zero
// elements, and a NaN byte there would turn those into NaN.
#pragma once

#include "b2_common.cuh"

namespace b2 {

constexpr int kMxBlock = 32;          // columns per scale
constexpr int kMxTileRows = 128;      // rows per scale tile
constexpr int kMxTileCols = 128;      // columns per scale tile (4 blocks)
constexpr int kMxTileBytes = 512;

__host__ __device__ __forceinline__ int mx_scale_offset(int row_in_tile, int block) {
  return (row_in_tile & 31) * 16 + (row_in_tile >> 5) * 4 + block;
}

// Scale byte from the exponent field of the block's largest magnitude.  bf16 and fp32 share the
// 8-bit exponent field E: floor(log2) = E - 127, so the byte is E - 2.  E below 2 (and the
// subnormals, E = 0) meets the format's smallest scale, byte 0; E = 255 is an infinity or a NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t exponent_field) {
  return exponent_field == 255u ? 255u : (exponent_field < 2u ? 0u : exponent_field - 2u);
}
// 2^-e, exact for every byte 0..252; 0 for the NaN byte (the block's elements become zeros).
__device__ __forceinline__ float mx_inverse_scale(uint32_t byte) {
  return byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23);
}
// 2^e (the NaN byte gives NaN); byte 0 is 2^-127, a subnormal.
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fc00000u) : (byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23));
}

// Eight fp32 -> eight 4-bit elements in one word, element i in bits 4i..4i+3 (nearest, ties to the
// even code, saturating at 6).
__device__ __forceinline__ uint32_t mx_pack8(const float (&f)[8]) {
  uint32_t d;
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t"
      "}"
      : "=r"(d)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return d;
}

// Eight 4-bit elements of one word -> four packed f16 pairs (exact).
__device__ __forceinline__ void mx_unpack8(uint32_t q, uint32_t (&h)[4]) {
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t"
      "}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(q));
}

// Largest magnitude of packed bf16 pairs as integers: the order of the 15 magnitude bits is the
// order of the values, and a NaN's exponent field stays on top.
__device__ __forceinline__ uint32_t mx_absmax_bits(uint32_t acc, uint32_t w) {
  return __vmaxu2(acc, w & 0x7fff7fffu);
}

// The larger exponent field of eight fp32 values, as packed halves: the upper halves hold it, and
// the order of those (sign dropped) is the order of the values.
__device__ __forceinline__ uint32_t mx_absmax_halves(const float (&f)[8]) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __byte_perm(__float_as_uint(f[2 * i]), __float_as_uint(f[2 * i + 1]), 0x7632) & 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(h[0], h[1]), __vmaxu2(h[2], h[3]));
}
// Scale byte of a block from the packed halves of its four lanes (neighbours).
__device__ __forceinline__ uint32_t mx_block_byte(uint32_t halves) {
  halves = __vmaxu2(halves, __shfl_xor_sync(0xffffffffu, halves, 1));
  halves = __vmaxu2(halves, __shfl_xor_sync(0xffffffffu, halves, 2));
  return mx_scale_byte(max(halves & 0xffffu, halves >> 16) >> 7);
}
// The four blocks' bytes of one row's column tile, from the 16 consecutive lanes that hold its 128
// columns (four lanes per block, all with their block's byte): the word in every lane.
__device__ __forceinline__ uint32_t mx_gather_word(uint32_t byte) {
  uint32_t w = byte << ((threadIdx.x & 12) * 2);
  w |= __shfl_xor_sync(0xffffffffu, w, 4);
  w |= __shfl_xor_sync(0xffffffffu, w, 8);
  return w;
}
// The packed elements of a lane's eight columns under their block's byte.
__device__ __forceinline__ uint32_t mx_quantize8(const float (&f)[8], uint32_t byte) {
  const float inv = mx_inverse_scale(byte);
  const uint64_t inv2 = pack2(inv, inv);
  float s[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(mul2(pack2(f[2 * i], f[2 * i + 1]), inv2), s[2 * i], s[2 * i + 1]);
  return byte == 255u ? 0u : mx_pack8(s);
}

}  // namespace b2
