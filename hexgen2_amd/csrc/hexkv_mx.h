// The 4-bit block format: 32 consecutive elements share a power of two, held
// as its biased exponent (byte b: 2^(b - 127), 255: the block is NaN), and
// an element is a sign, two exponent bits and one fraction bit: 0, 0.5, 1, 1.5,
// 2, 3, 4 or 6 times that power, the earlier element in a byte's lower half.
//
// A block's power is the smallest that leaves no element above 6 (a smaller
// one would clip the largest elements, by up to a quarter), and within
// [-125, 126], so that every non-zero value is a normal bf16 number (or, from
// 3.5 times 2^126 up, rounded to 2^128, past bf16's and fp32's range: an infinity to
// every reader): over normally distributed data the error is 0.116 of their deviation.  Since the
// power is exact, x / power is, and the only rounding is the element's own
// (nearest, halfway to the even code).
//
// gfx950 converts both ways (v_cvt_scalef32_pk_*): pinned on the GPU over every
// byte and element, byte 0 (2^-127) and 255 (NaN) among them, and against
// round-half-even over [-6, 6] at several powers.
#pragma once

#include "hexkv_common.h"

namespace hexkv {

constexpr int kMxBlock = 32;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Bytes of one position's row in a 4-bit cache: [2][heads][D / 2] elements,
// [2][heads][D / 32] powers, padded to a multiple of 16 so that every row's
// vectors are aligned.
__host__ __device__ constexpr int64_t mx_row_bytes(int64_t heads, int64_t head_dim) {
  return (2 * heads * (head_dim / 2 + head_dim / kMxBlock) + 15) / 16 * 16;
}

// Whether one of 8 elements reads as an infinity or a NaN: byte 255, 4 and 6
// times 2^126 (kMxLastPower), 2, 3, 4 and 6 times 2^127.
constexpr unsigned int kMxLastPower = 253;
__device__ __forceinline__ bool mx_past(unsigned int w, unsigned int byte) {
  return byte == 255 || (byte == 254 && (w & 0x44444444u)) || (byte == 253 && (w & w << 1 & 0x44444444u));
}

// The float whose exponent field a conversion takes the power from.
__device__ __forceinline__ float mx_scale(unsigned int byte) { return __uint_as_float(byte << 23); }

// The 8 elements of `w` times their power, as bf16 (exact).
__device__ __forceinline__ u32x4 mx_bf16(unsigned int w, float scale) {
  u32x4 r;
  r[0] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
  r[1] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
  r[2] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
  r[3] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  return r;
}

// The same as fp16: exact for powers from 2^-23 to 2^13 (bytes 104 to 140).
__device__ __forceinline__ u32x4 mx_f16(unsigned int w, float scale) {
  u32x4 r;
  r[0] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0));
  r[1] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1));
  r[2] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2));
  r[3] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
  return r;
}
constexpr unsigned int kMxF16Low = 104, kMxF16High = 140;

// The same as fp32.
__device__ __forceinline__ void mx_f32(unsigned int w, float scale, float *f) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
  f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1], f[4] = c[0], f[5] = c[1], f[6] = d[0], f[7] = d[1];
}

// The power's byte for a block whose largest magnitude has the bits `u` (an
// infinity's and a NaN's bits exceed every finite value's): the smallest e
// with 1.f * 2^k <= 1.5 * 2^(e + 2).  A block of zeros takes 2^0, which
// fp16 products read without their detour.
__device__ __forceinline__ unsigned int mx_power(unsigned int u) {
  if (u == 0) return 127;
  if (u >= 0x7f800000u) return 255;
  const int b = static_cast<int>(u >> 23) - 2 + ((u & 0x7fffffu) > 0x400000u ? 1 : 0);
  return static_cast<unsigned int>(min(max(b, 2), 253));
}

// 8 elements of a block with power byte `byte`, as 4 bits each.
__device__ __forceinline__ unsigned int mx_encode(const float *f, unsigned int byte) {
  if (byte == 255) return 0;
  const float scale = mx_scale(byte);
  unsigned int w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0], f[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2], f[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4], f[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6], f[7], scale, 3);
  return w;
}

// The largest magnitude's bits over 8 elements, and over the aligned groups of
// four lanes that hold a block's 32.
__device__ __forceinline__ unsigned int mx_bits(const float *f) {
  unsigned int u = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) u = max(u, __float_as_uint(f[i]) & 0x7fffffffu);
  return u;
}
__device__ __forceinline__ unsigned int mx_block_bits(unsigned int u) {
  u = max(u, static_cast<unsigned int>(
                 __builtin_amdgcn_update_dpp(0, static_cast<int>(u), 0xB1, 0xF, 0xF, true)));  // lane ^ 1
  return max(u, static_cast<unsigned int>(
                    __builtin_amdgcn_update_dpp(0, static_cast<int>(u), 0x4E, 0xF, 0xF, true)));  // lane ^ 2
}

// 8 consecutive elements as fp32; `vec`: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void mx_read8(const T *p, bool vec, float *f) {
  if (vec) {
    if constexpr (sizeof(T) == 2) {
      Elem<T>::to_float(*reinterpret_cast<const u32x4 *>(p), f);
    } else {
      Elem<T>::to_float(*reinterpret_cast<const u32x4 *>(p), f);
      Elem<T>::to_float(*reinterpret_cast<const u32x4 *>(p + 4), f + 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(p[i]);
  }
}

// 8 consecutive elements rounded to T; `vec`: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void mx_write8(T *p, bool vec, const float *f) {
  if (vec) {
    typedef T t __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
    for (int c = 0; c < 8; c += 16 / sizeof(T)) {
      t v;
#pragma unroll
      for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) v[i] = Elem<T>::from_float(f[c + i]);
      *reinterpret_cast<t *>(p + c) = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = Elem<T>::from_float(f[i]);
  }
}

}  // namespace hexkv
