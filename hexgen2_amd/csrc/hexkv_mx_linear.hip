// Products with 4-bit matrices: hexkv_mx_linear.
//
// A wave takes 16 rows of the matrix and up to 64 tokens, 128 of the inner
// dimension at a time: lane (c, g) holds one block (16 bytes, 32 elements) of
// row c, and the tokens' operand the same 32 elements of each token in the
// same order, so the converted block feeds four matrix instructions as it stands.
// The four waves of a workgroup share the inner dimension and join through
// LDS.
//
// bf16 activations meet the matrix as bf16, exact for every power.  fp16 ones
// meet it as fp16, exact for powers from 2^-23 to 2^13; a wave that meets
// another power takes that step in bf16, with each activation as two terms.
// fp32 activations are three bf16 terms.  All sums are fp32.
#include "hexkv_mx.h"

#include <algorithm>

namespace hexkv {

constexpr int kMxlThreads = 256;
constexpr int kMxlWaves = kMxlThreads / 64;

struct MxLinearArgs {
  const void *x;
  int64_t x_stride;  // elements
  const unsigned char *codes, *powers;
  void *out;
  int32_t rows, n, k;
  bool vec;  // x's rows are 16-byte aligned
};

// 8 activations as operand terms: the data type's own bits, or bf16 terms.
template <typename T>
__device__ __forceinline__ u32x4 raw8(const T *p, bool vec) {
  static_assert(sizeof(T) == 2, "16-bit data");
  if (vec) return *reinterpret_cast<const u32x4 *>(p);
  const unsigned short *s = reinterpret_cast<const unsigned short *>(p);
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = s[2 * i] | static_cast<unsigned int>(s[2 * i + 1]) << 16;
  return r;
}

// The first N bf16 terms of 8 floats (each the truncated rest of those before).
template <int N>
__device__ __forceinline__ void terms8(const float *f, u32x4 *t) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x0 = f[2 * i], x1 = f[2 * i + 1];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const unsigned int u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
      t[n][i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
      const float r0 = x0 - __uint_as_float(u0 & 0xffff0000u), r1 = x1 - __uint_as_float(u1 & 0xffff0000u);
      x0 = r0 == r0 ? r0 : 0.f;  // an infinity is its first term alone
      x1 = r1 == r1 ? r1 : 0.f;
    }
  }
}

__device__ __forceinline__ f32x4 mma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma_f16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// acc += 8 elements of the matrix (word w, times scale) times 8 activations.
template <typename T>
__device__ __forceinline__ f32x4 mx_product(unsigned int w, float scale, bool narrow, const T *x, bool live, bool vec,
                                            f32x4 acc) {
  if constexpr (sizeof(T) == 4) {
    float f[8] = {};
    if (live) mx_read8(x, vec, f);
    u32x4 t[3];
    terms8<3>(f, t);
    const u32x4 m = mx_bf16(w, scale);
    acc = mma_bf16(m, t[0], acc);
    acc = mma_bf16(m, t[1], acc);
    return mma_bf16(m, t[2], acc);
  } else {
    u32x4 r = {};
    if (live) r = raw8(x, vec);
    if constexpr (Elem<T>::kDtype == HEXKV_BF16) {
      return mma_bf16(mx_bf16(w, scale), r, acc);
    } else {
      if (narrow) return mma_f16(mx_f16(w, scale), r, acc);
      float f[8];
      Elem<T>::to_float(r, f);
      u32x4 t[2];
      terms8<2>(f, t);
      const u32x4 m = mx_bf16(w, scale);
      return mma_bf16(m, t[1], mma_bf16(m, t[0], acc));
    }
  }
}

// MT: tiles of 16 tokens.
template <typename T, int MT>
__global__ __launch_bounds__(kMxlThreads) void mx_linear_kernel(const MxLinearArgs a) {
  __shared__ f32x4 s_part[kMxlWaves][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int n0 = static_cast<int>(blockIdx.x) * 16, m0 = static_cast<int>(blockIdx.y) * (16 * MT);
  const int64_t row = min(n0 + c, a.n - 1);
  const unsigned char *codes = a.codes + row * (a.k / 2), *powers = a.powers + row * (a.k / kMxBlock);
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{};
  for (int k0 = wave * 128; k0 < a.k; k0 += kMxlWaves * 128) {
    const int k = k0 + g * kMxBlock;  // this lane's block
    u32x4 w = {};
    unsigned int byte = 127;
    if (k < a.k) {
      w = *reinterpret_cast<const u32x4 *>(codes + k / 2);
      byte = powers[k / kMxBlock];
    }
    const bool narrow = !__ballot(byte - kMxF16Low > kMxF16High - kMxF16Low);
    const float scale = mx_scale(byte);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int token = m0 + t * 16 + c;
      const bool live = token < a.rows && k < a.k;
      const T *x = static_cast<const T *>(a.x) + static_cast<int64_t>(live ? token : 0) * a.x_stride + (live ? k : 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[t] = mx_product<T>(w[j], scale, narrow, x + 8 * j, live, a.vec, acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) s_part[wave][t][lane] = acc[t];
  __syncthreads();
  // acc: column c is the token, rows 4 g + i are the matrix's
  if (wave < MT) {
    f32x4 sum = s_part[0][wave][lane];
#pragma unroll
    for (int w = 1; w < kMxlWaves; ++w) sum += s_part[w][wave][lane];
    const int token = m0 + wave * 16 + c, n = n0 + 4 * g;
    if (token < a.rows && n < a.n) {
      T *out = static_cast<T *>(a.out) + static_cast<int64_t>(token) * a.n + n;
      if (n + 4 <= a.n) {
        store4(out, sum);
      } else {
        for (int i = 0; i < a.n - n; ++i) out[i] = Elem<T>::from_float(sum[i]);
      }
    }
  }
}

template <typename T>
static void mx_linear_launch(const MxLinearArgs &a, hipStream_t s) {
  const unsigned gx = static_cast<unsigned>((a.n + 15) / 16);
  if (a.rows <= 16) mx_linear_kernel<T, 1><<<dim3(gx, 1), kMxlThreads, 0, s>>>(a);
  else if (a.rows <= 32) mx_linear_kernel<T, 2><<<dim3(gx, 1), kMxlThreads, 0, s>>>(a);
  else mx_linear_kernel<T, 4><<<dim3(gx, static_cast<unsigned>((a.rows + 63) / 64)), kMxlThreads, 0, s>>>(a);
}

}  // namespace hexkv

extern "C" int hexkv_mx_linear(const void *x, int64_t x_stride, const void *codes, const void *powers, void *out,
                               int rows, int n, int k, int dtype, hexkv_stream_t stream) {
  using namespace hexkv;
  const char *what = "hexkv_mx_linear";
  clear_error();
  if (dtype != HEXKV_F16 && dtype != HEXKV_BF16 && dtype != HEXKV_F32)
    return fail(HEXKV_EINVAL, "%s: unknown dtype %d", what, dtype);
  if (rows < 0 || n < 0 || k < 0) return fail(HEXKV_EINVAL, "%s: negative size", what);
  if (k == 0 || k % kMxBlock) return fail(HEXKV_EINVAL, "%s: k %d is not a positive multiple of %d", what, k, kMxBlock);
  if (rows == 0 || n == 0) return HEXKV_OK;
  if (!x || !codes || !powers || !out) return fail(HEXKV_EINVAL, "%s: null argument", what);
  const int elem = dtype == HEXKV_F32 ? 4 : 2;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & (elem - 1)) || !aligned16(codes))
    return fail(HEXKV_EINVAL, "%s: x/out misaligned, or codes not 16-byte aligned", what);
  if (rows > (1 << 20) || (static_cast<int64_t>(rows) + 63) / 64 * ((n + 15) / 16) >= INT64_C(1) << 24)
    return fail(HEXKV_ERANGE, "%s: over 2^20 tokens, or 2^24 workgroups or more; split the call", what);
  MxLinearArgs a = {};
  a.x = x;
  a.x_stride = x_stride;
  a.codes = static_cast<const unsigned char *>(codes);
  a.powers = static_cast<const unsigned char *>(powers);
  a.out = out;
  a.rows = rows;
  a.n = n;
  a.k = k;
  a.vec = aligned16(x) && x_stride * elem % 16 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == HEXKV_BF16) mx_linear_launch<__bf16>(a, s);
  else if (dtype == HEXKV_F16) mx_linear_launch<_Float16>(a, s);
  else mx_linear_launch<float>(a, s);
  return check_launch(what);
}
