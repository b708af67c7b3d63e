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
  int32_t m_tiles, n_tiles, splits, split_k;
  float *partial;  // [splits][rows][n]
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

// Few tokens (up to 16): a wave takes 16 rows of the matrix, 128 of the inner
// dimension at a time, the workgroup's waves in turn; kAhead of a wave's steps
// are loaded before the first is used.  The activations come straight from the
// caches.
constexpr int kAhead = 4;

template <typename T>
__global__ __launch_bounds__(kMxlThreads) void mx_few_kernel(const MxLinearArgs a) {
  __shared__ f32x4 s_part[kMxlWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int n0 = static_cast<int>(blockIdx.x) * 16;
  const int64_t row = min(n0 + c, a.n - 1);
  const unsigned char *codes = a.codes + row * (a.k / 2), *powers = a.powers + row * (a.k / kMxBlock);
  const T *x = static_cast<const T *>(a.x) + static_cast<int64_t>(c < a.rows ? c : 0) * a.x_stride;
  f32x4 acc = {};
  for (int base = wave * 128; base < a.k; base += kAhead * kMxlWaves * 128) {
    u32x4 w[kAhead];
    unsigned int byte[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const int k = base + s * kMxlWaves * 128 + g * kMxBlock;  // this lane's block
      w[s] = u32x4{};
      byte[s] = 127;
      if (k < a.k) {
        w[s] = *reinterpret_cast<const u32x4 *>(codes + k / 2);
        byte[s] = powers[k / kMxBlock];
      }
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const int k = base + s * kMxlWaves * 128 + g * kMxBlock;
      const bool live = c < a.rows && k < a.k;
      const bool narrow = !__ballot(byte[s] - kMxF16Low > kMxF16High - kMxF16Low);
      const float scale = mx_scale(byte[s]);
      const T *at = x + (live ? k : 0);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float f[8] = {};
          if (live) mx_read8(at + 8 * j, a.vec, f);
          u32x4 t[3];
          terms8<3>(f, t);
          const u32x4 m = mx_bf16(w[s][j], scale);
#pragma unroll
          for (int n = 0; n < 3; ++n) acc = mma_bf16(m, t[n], acc);
        }
      } else {
        u32x4 r[4] = {};
        if (live) {
#pragma unroll
          for (int j = 0; j < 4; ++j) r[j] = raw8(at + 8 * j, a.vec);
        }
        if constexpr (Elem<T>::kDtype == HEXKV_BF16) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc = mma_bf16(mx_bf16(w[s][j], scale), r[j], acc);
        } else if (narrow) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc = mma_f16(mx_f16(w[s][j], scale), r[j], acc);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float f[8];
            Elem<T>::to_float(r[j], f);
            u32x4 t[2];
            terms8<2>(f, t);
            const u32x4 m = mx_bf16(w[s][j], scale);
            acc = mma_bf16(m, t[1], mma_bf16(m, t[0], acc));
          }
        }
      }
    }
  }
  s_part[wave][lane] = acc;
  __syncthreads();
  // acc: column c is the token, rows 4 g + i are the matrix's
  if (wave == 0) {
    f32x4 sum = s_part[0][lane];
#pragma unroll
    for (int w = 1; w < kMxlWaves; ++w) sum += s_part[w][lane];
    const int n = n0 + 4 * g;
    if (c < a.rows && n < a.n) {
      T *out = static_cast<T *>(a.out) + static_cast<int64_t>(c) * a.n + n;
      if (n + 4 <= a.n) {
        store4(out, sum);
      } else {
        for (int i = 0; i < a.n - n; ++i) out[i] = Elem<T>::from_float(sum[i]);
      }
    }
  }
}

// More tokens: a workgroup takes 32 MT WM tokens by 32 NT WN rows of the matrix;
// its waves are WM x WN pieces of that, times WK that share the inner
// dimension.  A step is STEPS times 64 of the inner dimension for each of the
// WK: the tokens' piece of it lies in LDS (two of them, loaded through
// registers while the other is used), in 16-byte chunks permuted within a row so that
// a wave's reads of one chunk of 32 rows meet every bank equally; the matrix
// goes straight to the registers of the waves that convert it, one step
// ahead.  v_mfma_f32_32x32x16: lane (c, h) holds one block of row c, half h of 64,
// and the tokens' operand the same elements.
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T, int MT_, int NT_, int WM_, int WN_, int WK_, int STEPS_>
struct MxTileShape {
  static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, WK = WK_, STEPS = STEPS_;
  static constexpr int kWaves = WM * WN * WK, kThreads = 64 * kWaves;
  static constexpr int kTokens = 32 * MT * WM, kRows = 32 * NT * WN;
  static constexpr int kStep = 64 * WK * STEPS;            // inner dimension of one step
  static constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;   // 16-bit terms of an activation in LDS
  static constexpr int kChunks = kStep / 8;                // 16-byte chunks of a token's row in LDS
  static constexpr int kPlane = kTokens * kChunks;         // chunks of a plane
  static constexpr int kLoads = kPlane / kThreads;         // chunks a thread stages
  static constexpr size_t kLds = size_t{16} * 2 * kPlanes * kPlane;
  static_assert(kPlane % kThreads == 0, "every thread stages as much");
  static_assert(static_cast<size_t>(WK - 1) * WM * WN * MT * NT * 16 * 64 * 4 <= kLds, "the join fits the stage");
};

__device__ __forceinline__ f32x16 mma32_bf16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32_f16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads) void mx_tile_kernel(const MxLinearArgs a) {
  constexpr int MT = S::MT, NT = S::NT, CH = S::kChunks, PL = S::kPlanes;
  constexpr int kSpread = CH >= 16 ? 1 : 16 / CH;  // rows whose chunks fill the banks once
  constexpr int kMask = CH >= 16 ? 15 : CH - 1;
  __shared__ __attribute__((aligned(16))) char s_mem[S::kLds];
  u32x4 *s_x = reinterpret_cast<u32x4 *>(s_mem);  // [2][planes][tokens][chunks]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int wn = wave % S::WN, wm = wave / S::WN % S::WM, wk = wave / (S::WN * S::WM);

  // Consecutive workgroups go to the XCDs in turn: those of one XCD take one
  // piece of the matrix through all its tokens before the next.
  const int local = static_cast<int>(blockIdx.x >> 3);
  const int group = local / a.m_tiles * 8 + static_cast<int>(blockIdx.x & 7);
  const int m0 = (local % a.m_tiles) * S::kTokens;
  if (group >= a.n_tiles * a.splits) return;
  const int n0 = group / a.splits * S::kRows, split = group % a.splits;
  const int k_first = split * a.split_k, k_last = min(a.k, k_first + a.split_k);

  const unsigned char *codes[NT], *powers[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t row = min(n0 + (wn * NT + t) * 32 + c, a.n - 1);
    codes[t] = a.codes + row * (a.k / 2);
    powers[t] = a.powers + row * (a.k / kMxBlock);
  }

  u32x4 stage[PL][S::kLoads];
  const auto fetch_x = [&](int k0) {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int at = i * S::kThreads + tid, token = m0 + at / CH, k = k0 + at % CH * 8;
      const bool live = token < a.rows && k < k_last;
      const T *p = static_cast<const T *>(a.x) + static_cast<int64_t>(live ? token : 0) * a.x_stride + (live ? k : 0);
      if constexpr (PL == 1) {
        stage[0][i] = u32x4{};
        if (live) stage[0][i] = raw8(p, a.vec);
      } else {
        float f[8] = {};
        if (live) mx_read8(p, a.vec, f);
        u32x4 t[3];
        terms8<3>(f, t);
#pragma unroll
        for (int n = 0; n < 3; ++n) stage[n][i] = t[n];
      }
    }
  };
  const auto store_x = [&](int buf) {
#pragma unroll
    for (int n = 0; n < PL; ++n)
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int at = i * S::kThreads + tid, token = at / CH, chunk = at % CH;
        s_x[(buf * PL + n) * S::kPlane + token * CH + (chunk ^ (token / kSpread & kMask))] = stage[n][i];
      }
  };
  struct Weights {
    u32x4 w[S::STEPS][NT];
    unsigned int byte[S::STEPS][NT];
  };
  const auto fetch_w = [&](int k0, Weights &x) {
#pragma unroll
    for (int s = 0; s < S::STEPS; ++s)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int k = k0 + (wk * S::STEPS + s) * 64 + h * kMxBlock;
        x.w[s][t] = u32x4{};
        x.byte[s][t] = 127;
        if (k < k_last) {
          x.w[s][t] = *reinterpret_cast<const u32x4 *>(codes[t] + k / 2);
          x.byte[s][t] = powers[t][k / kMxBlock];
        }
      }
  };

  f32x16 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x16{};

  const auto compute = [&](int buf, const Weights &x) {
#pragma unroll
    for (int s = 0; s < S::STEPS; ++s) {
      bool far = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) far |= x.byte[s][t] - kMxF16Low > kMxF16High - kMxF16Low;
      const auto tokens = [&](int n, int m, int j) {
        const int token = (wm * MT + m) * 32 + c, chunk = (wk * S::STEPS + s) * 8 + h * 4 + j;
        return s_x[(buf * PL + n) * S::kPlane + token * CH + (chunk ^ (token / kSpread & kMask))];
      };
      if (Elem<T>::kDtype == HEXKV_F16 && __ballot(far)) {
        // (a loop that is not unrolled: the detour costs the main path no registers)
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          u32x4 w[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const u32x4 v = x.w[s][t];
            w[t] = mx_bf16(j < 2 ? (j == 0 ? v[0] : v[1]) : (j == 2 ? v[2] : v[3]), mx_scale(x.byte[s][t]));
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            float f[8];
            Elem<_Float16>::to_float(tokens(0, m, j), f);
            u32x4 terms[2];
            terms8<2>(f, terms);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int n = 0; n < 2; ++n) acc[m][t] = mma32_bf16(w[t], terms[n], acc[m][t]);
          }
        }
        continue;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 b[PL][MT];
#pragma unroll
        for (int n = 0; n < PL; ++n)
#pragma unroll
          for (int m = 0; m < MT; ++m) b[n][m] = tokens(n, m, j);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (Elem<T>::kDtype == HEXKV_F16) {
            const u32x4 w = mx_f16(x.w[s][t][j], mx_scale(x.byte[s][t]));
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m][t] = mma32_f16(w, b[0][m], acc[m][t]);
          } else {
            const u32x4 w = mx_bf16(x.w[s][t][j], mx_scale(x.byte[s][t]));
#pragma unroll
            for (int n = 0; n < PL; ++n)
#pragma unroll
              for (int m = 0; m < MT; ++m) acc[m][t] = mma32_bf16(w, b[n][m], acc[m][t]);
          }
        }
      }
    }
  };

  if (k_first < k_last) {
    Weights now, next;
    fetch_x(k_first);
    fetch_w(k_first, now);
    store_x(0);
    __syncthreads();
    int buf = 0;
    for (int k0 = k_first; k0 < k_last; k0 += S::kStep) {
      const bool more = k0 + S::kStep < k_last;
      if (more) {
        fetch_x(k0 + S::kStep);
        fetch_w(k0 + S::kStep, next);
      }
      compute(buf, now);
      if (more) store_x(buf ^ 1);
      buf ^= 1;
      now = next;
      __syncthreads();
    }
  }

  // the waves that share the inner dimension join in the first of them
  if constexpr (S::WK > 1) {
    float *s_acc = reinterpret_cast<float *>(s_mem);
    const int piece = (wm * S::WN + wn) * MT * NT * 16 * 64 + lane;
    if (wk > 0) {
      float *p = s_acc + (wk - 1) * S::WM * S::WN * MT * NT * 16 * 64 + piece;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) p[((m * NT + t) * 16 + i) * 64] = acc[m][t][i];
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int w = 0; w < S::WK - 1; ++w) {
      const float *p = s_acc + w * S::WM * S::WN * MT * NT * 16 * 64 + piece;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[m][t][i] += p[((m * NT + t) * 16 + i) * 64];
    }
  }
  // acc: column c is the token, rows 8 i + 4 h + e the matrix's
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int token = m0 + (wm * MT + m) * 32 + c;
    if (token >= a.rows) continue;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = n0 + (wn * NT + t) * 32 + 8 * i + 4 * h;
        const f32x4 v = {acc[m][t][4 * i], acc[m][t][4 * i + 1], acc[m][t][4 * i + 2], acc[m][t][4 * i + 3]};
        if (n >= a.n) continue;
        if (a.splits > 1) {
          float *o = a.partial + (static_cast<int64_t>(split) * a.rows + token) * a.n + n;
          if (n + 4 <= a.n) store4(o, v);
          else for (int e = 0; e < a.n - n; ++e) o[e] = v[e];
        } else {
          T *o = static_cast<T *>(a.out) + static_cast<int64_t>(token) * a.n + n;
          if (n + 4 <= a.n) store4(o, v);
          else for (int e = 0; e < a.n - n; ++e) o[e] = Elem<T>::from_float(v[e]);
        }
      }
  }
}

// out = the sum of the splits' products, in their order.
template <typename T>
__global__ __launch_bounds__(kMxlThreads) void mx_sum_kernel(const MxLinearArgs a, int64_t total) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * kMxlThreads + threadIdx.x) * 4;
  if (i >= total) return;
  T *out = static_cast<T *>(a.out) + i;
  if (i + 4 <= total && total % 4 == 0) {
    f32x4 sum = *reinterpret_cast<const f32x4 *>(a.partial + i);
    for (int s = 1; s < a.splits; ++s) sum += *reinterpret_cast<const f32x4 *>(a.partial + s * total + i);
    store4(out, sum);
  } else {
    for (int e = 0; e < 4 && i + e < total; ++e) {
      float sum = a.partial[i + e];
      for (int s = 1; s < a.splits; ++s) sum += a.partial[s * total + i + e];
      out[e] = Elem<T>::from_float(sum);
    }
  }
}

// The tile a call runs: its tokens and matrix rows, and what a split of the
// inner dimension is a multiple of.
struct MxPlan {
  int kind;  // 0: few tokens
  int m_tiles, n_tiles, splits, split_k;
};

template <typename T> using TileDecode32 = MxTileShape<T, 1, 1, 1, 4, 2, sizeof(T) == 4 ? 1 : 2>;
template <typename T> using TileDecode64 = MxTileShape<T, 2, 1, 1, 4, 2, sizeof(T) == 4 ? 1 : 2>;
template <typename T> using TilePrompt = MxTileShape<T, 2, 2, 2, 2, 1, 1>;

template <typename S>
static void plan_tile(MxPlan *p, int rows, int n, int k) {
  p->m_tiles = (rows + S::kTokens - 1) / S::kTokens;
  p->n_tiles = (n + S::kRows - 1) / S::kRows;
  const int steps = (k + S::kStep - 1) / S::kStep;
  const int splits = std::max(1, std::min(steps / 4, 512 / std::max(1, p->m_tiles * p->n_tiles)));
  p->split_k = (steps + splits - 1) / splits * S::kStep;
  p->splits = (k + p->split_k - 1) / p->split_k;
}

template <typename T>
static MxPlan mx_plan(int rows, int n, int k) {
  MxPlan p = {};
  if (rows <= 16) return p;
  if (rows <= 32) { p.kind = 1; plan_tile<TileDecode32<T>>(&p, rows, n, k); }
  else if (rows <= 64) { p.kind = 2; plan_tile<TileDecode64<T>>(&p, rows, n, k); }
  else { p.kind = 3; plan_tile<TilePrompt<T>>(&p, rows, n, k); }
  return p;
}

static MxPlan mx_plan_of(int rows, int n, int k, int dtype) {
  return dtype == HEXKV_F32 ? mx_plan<float>(rows, n, k) : mx_plan<__bf16>(rows, n, k);
}

static size_t mx_partial_bytes(const MxPlan &p, int rows, int n) {
  return p.splits > 1 ? static_cast<size_t>(p.splits) * rows * n * sizeof(float) : 0;
}

template <typename T, typename S>
static void launch_tile_shape(const MxLinearArgs &a, hipStream_t s) {
  static_assert(S::kLds <= 160 * 1024, "LDS");
  const unsigned groups = static_cast<unsigned>(a.n_tiles * a.splits + 7) / 8 * 8;
  mx_tile_kernel<T, S><<<groups * a.m_tiles, S::kThreads, 0, s>>>(a);
}

template <typename T>
static void mx_linear_launch(MxLinearArgs a, const MxPlan &p, hipStream_t s) {
  a.m_tiles = p.m_tiles;
  a.n_tiles = p.n_tiles;
  a.splits = p.splits;
  a.split_k = p.split_k;
  switch (p.kind) {
    case 0: return mx_few_kernel<T><<<(a.n + 15) / 16, kMxlThreads, 0, s>>>(a);
    case 1: launch_tile_shape<T, TileDecode32<T>>(a, s); break;
    case 2: launch_tile_shape<T, TileDecode64<T>>(a, s); break;
    default: launch_tile_shape<T, TilePrompt<T>>(a, s);
  }
  if (a.splits > 1) {
    const int64_t total = static_cast<int64_t>(a.rows) * a.n;
    mx_sum_kernel<T><<<static_cast<unsigned>((total + 4 * kMxlThreads - 1) / (4 * kMxlThreads)), kMxlThreads, 0, s>>>(a, total);
  }
}

static int mx_linear_check(int rows, int n, int k, int dtype, const char *what) {
  if (dtype != HEXKV_F16 && dtype != HEXKV_BF16 && dtype != HEXKV_F32)
    return fail(HEXKV_EINVAL, "%s: unknown dtype %d", what, dtype);
  if (rows < 0 || n < 0 || k < 0) return fail(HEXKV_EINVAL, "%s: negative size", what);
  if (k == 0 || k % kMxBlock) return fail(HEXKV_EINVAL, "%s: k %d is not a positive multiple of %d", what, k, kMxBlock);
  if (rows > (1 << 20) || (static_cast<int64_t>(rows) + 63) / 64 * ((n + 15) / 16) >= INT64_C(1) << 24)
    return fail(HEXKV_ERANGE, "%s: over 2^20 tokens, or 2^24 workgroups or more; split the call", what);
  return HEXKV_OK;
}

}  // namespace hexkv

extern "C" size_t hexkv_mx_linear_workspace_bytes(int rows, int n, int k, int dtype) {
  using namespace hexkv;
  clear_error();
  if (mx_linear_check(rows, n, k, dtype, "hexkv_mx_linear_workspace_bytes") != HEXKV_OK) return 0;
  return mx_partial_bytes(mx_plan_of(rows, n, k, dtype), rows, n);
}

extern "C" int hexkv_mx_linear(const void *x, int64_t x_stride, const void *codes, const void *powers, void *out,
                               int rows, int n, int k, int dtype, void *workspace, size_t workspace_bytes,
                               hexkv_stream_t stream) {
  using namespace hexkv;
  const char *what = "hexkv_mx_linear";
  clear_error();
  const int rc = mx_linear_check(rows, n, k, dtype, what);
  if (rc != HEXKV_OK) return rc;
  if (rows == 0 || n == 0) return HEXKV_OK;
  if (!x || !codes || !powers || !out) return fail(HEXKV_EINVAL, "%s: null argument", what);
  const int elem = dtype == HEXKV_F32 ? 4 : 2;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & (elem - 1)) || !aligned16(codes))
    return fail(HEXKV_EINVAL, "%s: x/out misaligned, or codes not 16-byte aligned", what);
  const MxPlan plan = mx_plan_of(rows, n, k, dtype);
  const size_t need = mx_partial_bytes(plan, rows, n);
  if (need && (!workspace || workspace_bytes < need))
    return fail(HEXKV_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : 0, need);
  if (need && !aligned16(workspace)) return fail(HEXKV_EINVAL, "%s: workspace must be 16-byte aligned", what);
  MxLinearArgs a = {};
  a.x = x;
  a.x_stride = x_stride;
  a.codes = static_cast<const unsigned char *>(codes);
  a.powers = static_cast<const unsigned char *>(powers);
  a.out = out;
  a.rows = rows;
  a.n = n;
  a.k = k;
  a.partial = static_cast<float *>(workspace);
  a.vec = aligned16(x) && x_stride * elem % 16 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == HEXKV_BF16) mx_linear_launch<__bf16>(a, plan, s);
  else if (dtype == HEXKV_F16) mx_linear_launch<_Float16>(a, plan, s);
  else mx_linear_launch<float>(a, plan, s);
  return check_launch(what);
}
