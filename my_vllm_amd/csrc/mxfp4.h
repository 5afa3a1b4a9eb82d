// The 4-bit KV cache format (MXFP4) shared by the kernels that write and read it.
//
// OCP microscaling FP4: an element is e2m1 (codes 0..7 stand for 0, 0.5, 1,
// 1.5, 2, 3, 4, 6; bit 3 is the sign), and 32 elements share one E8M0 scale, a
// byte b that stands for 2^(b - 127) (255: NaN).  A head's row of 128 elements
// is 64 bytes of elements (element 2i in the low four bits of byte i) and four
// scale bytes.  A page of one KV head is one block of 1088 contiguous bytes:
// its 16 tokens' elements, then their scales, so that a page is read with one
// 16-byte access a lane and one line of scales.
//
// gfx950 converts this format in one instruction a pair
// (v_cvt_scalef32_pk_{bf16,f16}_fp4 and back), scale included; the scale
// operand is an fp32 of which the exponent bits count, so a scale byte shifted
// to bit 23 is the operand (0 counts as 2^-127, 255 gives NaN).
#pragma once

#include "mva_common.h"

namespace mva {

constexpr int kFp4Group = 32;      // elements a scale
constexpr int kFp4RowBytes = 64;   // element bytes of a head's row
constexpr int kFp4RowScales = 4;   // scale bytes of a head's row
constexpr int kFp4PageTokens = 16;
constexpr int kFp4ScaleOffset = kFp4PageTokens * kFp4RowBytes;                           // 1024
constexpr int kFp4BlockBytes = kFp4ScaleOffset + kFp4PageTokens * kFp4RowScales;         // 1088

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

// Scale operand of a scale byte.
__device__ inline float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

template <typename T>
struct Fp4;

template <>
struct Fp4<__bf16> {
  typedef bf16x2 v2;
  // Largest scale byte written: 6 * 2^125 is the largest value read back.
  static constexpr int kMaxScale = 252;
  static constexpr uint32_t kInfBits = 0x7f80;
  // fp32 bits of the magnitude `m` (the low 15 bits of an element).
  __device__ static inline uint32_t f32_bits(uint32_t m) { return m << 16; }
  // Elements 2 kByte and 2 kByte + 1 of eight packed in `w`, times `scale`.
  template <int kByte>
  __device__ static inline v2 unpack(uint32_t w, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, kByte);
  }
  // `w` with byte kByte replaced by the codes of the two elements in x, over
  // `scale` (nearest, ties to even, saturating).
  template <int kByte>
  __device__ static inline uint32_t pack(uint32_t w, uint32_t x, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2, x), scale, kByte);
  }
};

template <>
struct Fp4<_Float16> {
  typedef f16x2 v2;
  static constexpr int kMaxScale = 140;  // 6 * 2^13
  static constexpr uint32_t kInfBits = 0x7c00;
  __device__ static inline uint32_t f32_bits(uint32_t m) {
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m));
  }
  template <int kByte>
  __device__ static inline v2 unpack(uint32_t w, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, kByte);
  }
  template <int kByte>
  __device__ static inline uint32_t pack(uint32_t w, uint32_t x, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2, x), scale, kByte);
  }
};

// Eight elements packed in `w`, times `scale`.
template <typename T>
__device__ inline typename Elem<T>::v8 fp4_unpack8(uint32_t w, float scale) {
  typedef Fp4<T> F;
  const typename F::v2 a = F::template unpack<0>(w, scale), b = F::template unpack<1>(w, scale);
  const typename F::v2 c = F::template unpack<2>(w, scale), d = F::template unpack<3>(w, scale);
  return typename Elem<T>::v8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace mva
