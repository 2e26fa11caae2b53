// The 8-bit key / value cache shared by kv8.hip (writes, reads back) and attention_kv8.hip (attends).
//
// S sequences x H key heads x cap positions (a multiple of 64).  Per (sequence, head):
//   K  [cap][hd]            one byte a value, rows as they come
//   V  [cap / 16][hd][16]   tiles of 16 positions, TRANSPOSED inside: 16 consecutive bytes are 16 positions of one channel, which is what
//                           the P V product contracts over -- a lane's 16-byte load is an operand of two matrix instructions
//   scales fp32 [cap / block], powers of two, one per `block` (16 / 32 / 64) positions.  value = code * scale, exactly representable in bf16.
// Codes: DT 0 = e4m3 (OCP, largest 448), DT 1 = int8 (largest 127; -128 is never written).
#pragma once
#include "neko_kernels.h"

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;

// two 8-bit codes (bytes 0/1 or, HI, 2/3 of w) -> two bf16 = code * scale.  One instruction for e4m3; int8 goes through fp32.
template <int DT, bool HI>
__device__ __forceinline__ uint32_t kv8_unpack2(uint32_t w, float scale) {
  if constexpr (DT == 0) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
  } else {
    const float a = (float)(signed char)(w >> (HI ? 16 : 0)), b = (float)(signed char)(w >> (HI ? 24 : 8));
    return pack_bf16x2(a * scale, b * scale);
  }
}
// ... and unscaled (the callers that fold the scale into something smaller)
template <int DT, bool HI>
__device__ __forceinline__ uint32_t kv8_unpack2(uint32_t w) {
  if constexpr (DT == 0) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  } else {
    return pack_bf16x2((float)(signed char)(w >> (HI ? 16 : 0)), (float)(signed char)(w >> (HI ? 24 : 8)));
  }
}
// 8 codes -> one matrix operand (element j = code j)
template <int DT>
__device__ __forceinline__ bf16x8_v kv8_frag(uint32_t w0, uint32_t w1) {
  typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_v;
  const u32x4_v u = {kv8_unpack2<DT, false>(w0), kv8_unpack2<DT, true>(w0), kv8_unpack2<DT, false>(w1), kv8_unpack2<DT, true>(w1)};
  return __builtin_bit_cast(bf16x8_v, u);
}
// four values (already divided by the scale, |x| <= qmax) -> four codes, round to nearest even
template <int DT>
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d) {
  if constexpr (DT == 0) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    // x + 1.5 * 2^23: the addition rounds to an integer (nearest even), which is then the low byte of the sum's bit pattern
    constexpr float MAGIC = 12582912.0f;
    const uint32_t u0 = __float_as_uint(a + MAGIC), u1 = __float_as_uint(b + MAGIC), u2 = __float_as_uint(c + MAGIC), u3 = __float_as_uint(d + MAGIC);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u3, u2, 0x0c0c0400u), __builtin_amdgcn_perm(u1, u0, 0x0c0c0400u), 0x05040100u);
  }
}
// one code as fp32
template <int DT>
__device__ __forceinline__ float kv8_code(uint32_t byte) {
  if constexpr (DT == 0) return __uint_as_float(kv8_unpack2<0, false>(byte) << 16);
  else return (float)(signed char)byte;
}
