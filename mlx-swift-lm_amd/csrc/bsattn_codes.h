// bsattn_codes.h -- affine codes as fp16 MFMA operands, shared by the
// attention kernels over quantized caches.
#pragma once

#include "bsattn_device.h"

namespace bsattn {

// Codes as the decode kernel's MFMA operands: int8 code c is the fp16
// 1024 + c (byte_to_f16); an int4 word (element e in nibble q_nib(e)) gives
// pairs 0 and 2 (elements 0, 1, 4, 5) as 1024 + c and pairs 1 and 3
// (elements 2, 3, 6, 7) as 1024 + 16 c: pair k's nibbles k and k + 4 sit at
// bits 4 (k & 1) and 16 + 4 (k & 1) once the word is shifted by 8 (k >> 1),
// inside the fp16 mantissa under the exponent of 1024, so a word costs one
// shift and four v_and_or_b32 (base: 0x64006400 in a VGPR).  The other
// operand of each unit-16 element is scaled by 1/16 (kUnit16), so every
// product is q c (or p c) plus 1024 times the other operand, and
// sum (1024 + u c) x = sum x c u + 1024 sum x removes the offset with the sum
// of the same scaled operand.
__device__ __forceinline__ u32x4 nib_to_f16_dec(uint32_t w, uint32_t base) {
  const uint32_t w8 = w >> 8;
  return u32x4{(w & 0x000F000Fu) | base, (w & 0x00F000F0u) | base, (w8 & 0x000F000Fu) | base,
               (w8 & 0x00F000F0u) | base};
}
constexpr float kDecOff = 1024.0f;  // value of code 0 in the decode operands
constexpr float kUnit16 = 0.0625f;  // scale of the other operand at unit-16 int4 elements

// 0x64006400 (two fp16 1024.0) in a VGPR the compiler cannot fold into the
// v_and_or_b32 (a DPP identity move: unlike an inline-asm move, the
// compiler sees its register write, so the MFMA hazard wait states around
// it are inserted)
__device__ __forceinline__ uint32_t f16_pair_1024() {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)0x64006400, 0xE4, 0xF, 0xF, false);
}

// A operand of QK token tile t, k-step s, from the tile's K fragments
template <int KB>
__device__ __forceinline__ u32x4 k_operand(const u32x4* kf, int s, uint32_t base) {
  if constexpr (KB == 4) return nib_to_f16_dec(kf[0][s], base);
  else return byte_to_f16(kf[s >> 1][2 * (s & 1)], kf[s >> 1][2 * (s & 1) + 1]);
}

// B operand of PV dim tile dt, k-step s2, from the V fragments
template <int KB, int KS2>
__device__ __forceinline__ u32x4 v_operand(const u32x4* vf, int dt, int s2, uint32_t base) {
  constexpr int DPF = QCode<KB>::DPF;
  const u32x4& f = vf[(dt / DPF) * KS2 + s2];
  if constexpr (KB == 4) return nib_to_f16_dec(f[dt & 3], base);
  else return byte_to_f16(f[2 * (dt & 1)], f[2 * (dt & 1) + 1]);
}

// products of the fp16 halves
__device__ __forceinline__ uint32_t f16x2_mul(uint32_t x, uint32_t y) {
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) * __builtin_bit_cast(f16x2, y));
}
// x * 1/16 on both fp16 halves (exact unless the result is below fp16's
// normal range)
__device__ __forceinline__ uint32_t f16x2_unit16(uint32_t x) {
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) * f16x2{(_Float16)kUnit16, (_Float16)kUnit16});
}

__device__ __forceinline__ f32x4 mfma_f16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

}  // namespace bsattn
