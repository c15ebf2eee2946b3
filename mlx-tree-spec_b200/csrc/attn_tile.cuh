// Building blocks of the tcgen05 attention kernels: exp2, the shared-memory
// descriptor of an MN-major operand, and the conversion of 8-bit cache codes.
#pragma once

#include "sm100.cuh"

namespace tsb {

TSB_HD float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// MN-major operand, 128-byte swizzle: 64-element rows of 128 B along MN, 8-row
// K groups 1024 B apart (SBO), 64-element MN blocks `lbo` bytes apart (LBO).
TSB_HD uint64_t desc_mnmajor_sw128(uint32_t smem_byte_addr, uint32_t lbo) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_byte_addr >> 4) & 0x3FFF);
  d |= (uint64_t)((lbo >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Byte k of w as the bits of float 2^23 + byte (exact): the byte becomes the
// low mantissa byte of 0x4B000000.
TSB_HD uint32_t byte_2p23(uint32_t w, uint32_t k) { return prmt(w, 0x4B000000u, 0x7540u | k); }

// 8 MLX codes (u8, low byte first) -> 8 bf16 of s*q + b: q exact in float,
// one float fma, round to nearest even (the dequantization of mlx
// dequantize and of the 8-bit staging in attn.cu).
TSB_HD uint4 dequant8_mlx(uint2 w, float s, float b) {
  uint32_t o[4];
  const uint32_t ws[2] = {w.x, w.y};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float q0 = __uint_as_float(byte_2p23(ws[h], 2 * e)) - 8388608.f;
      const float q1 = __uint_as_float(byte_2p23(ws[h], 2 * e + 1)) - 8388608.f;
      o[2 * h + e] = pack_bf16x2(__fmaf_rn(q0, s, b), __fmaf_rn(q1, s, b));
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// 8 int8 codes -> 8 bf16 holding the same integers (exact): flipping the sign
// bit gives q + 128 as an unsigned byte.
TSB_HD uint4 convert8_s8(uint2 w) {
  uint32_t o[4];
  const uint32_t ws[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float q0 = __uint_as_float(byte_2p23(ws[h], 2 * e)) - 8388736.f;  // 2^23 + 128
      const float q1 = __uint_as_float(byte_2p23(ws[h], 2 * e + 1)) - 8388736.f;
      o[2 * h + e] = pack_bf16x2(q0, q1);
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace tsb
