// Products with 4-bit matrices: hexkv_mx_linear.
//
// What bounds it: reading the matrix while tokens are few, 17/32 byte an element
// (read-only streams reach 7.1 TB/s here), the matrix cores for a prompt.
// Everywhere a lane loads whole blocks of a row (16 bytes, 32 elements, one
// power) and converts them in registers; the matrix instructions' inner dimension is laid
// out to fit what a lane holds, the tokens' operand in the same order, so a
// converted block is an operand as it stands.  Four kernels, see mx_plan:
//   mx_rows_kernel  one or two tokens: a wave reads rows from end to end;
//   mx_few_kernel   up to 64: a wave holds the tokens' operands of its share of
//                   the inner dimension in registers and walks the matrix;
//   mx_prompt_kernel  more: tiles, with the tokens and the matrix's four bits in LDS;
//   mx_tile_kernel  fp32 above 16 tokens: tiles, with the tokens' three terms in LDS.
//
// bf16 activations meet the matrix as bf16, exact for every power.  fp16 ones
// meet it as fp16, exact for powers from 2^-23 to 2^13; blocks with another
// power are left out there and added afterwards in bf16, with each activation as two
// terms (fp32 in mx_rows_kernel).  Left out they are zeros, whose product with an
// infinite activation is a NaN: where the sum without them is not finite, all
// blocks are added up that way instead.  fp32 activations are three bf16 terms.  All sums
// are fp32.
#include "hexkv_mx.h"

#include <algorithm>

namespace hexkv {

constexpr int kMxlThreads = 256;

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

// x less its upper half; of an infinity nothing is left, of a NaN (whose payload
// may lie in the lower half alone, which leaves an infinity's upper half) a NaN.
__device__ __forceinline__ float first_rest(float x) {
  const float rest = x - __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  return __builtin_amdgcn_classf(x, 0x204) ? 0.f : rest;  // minus and plus infinity
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
      x0 = n == 0 ? first_rest(x0) : x0 - __uint_as_float(u0 & 0xffff0000u);
      x1 = n == 0 ? first_rest(x1) : x1 - __uint_as_float(u1 & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ f32x4 mma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma_f16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// fp16 activations: the scale a block enters the fp16 product with, 0 for a
// power that fp16 does not hold exactly (*far is raised), so that the block
// adds nothing there.
__device__ __forceinline__ float near_scale(unsigned int byte, bool *far) {
  const bool out = byte - kMxF16Low > kMxF16High - kMxF16Low;
  *far |= out;
  return out ? 0.f : mx_scale(byte);
}

// Such a block alone (with `all` any block), as bf16; the others are zero.
struct FarBlock {
  u32x4 w;
  float scale;
  bool any;
  __device__ __forceinline__ void read(const MxLinearArgs &a, int64_t row, int block, bool live, bool all) {
    const unsigned int byte = live ? a.powers[row * (a.k / kMxBlock) + block] : 127u;
    any = (all && live) || byte - kMxF16Low > kMxF16High - kMxF16Low;
    w = u32x4{};
    if (any) w = *reinterpret_cast<const u32x4 *>(a.codes + row * (a.k / 2) + block * 16);
    scale = any ? mx_scale(byte) : 1.f;
  }
  __device__ __forceinline__ unsigned int word(int j) const { return j < 2 ? (j == 0 ? w[0] : w[1]) : (j == 2 ? w[2] : w[3]); }
  __device__ __forceinline__ u32x4 operand(int j) const { return mx_bf16(word(j), scale); }
};
// The two bf16 terms of 8 fp16 activations.
__device__ __forceinline__ void far_terms(const _Float16 *p, bool live, u32x4 *terms) {
  float f[8] = {};
  if (live) mx_read8(p, false, f);
  terms8<2>(f, terms);
}

// acc + the dot product of one block of the matrix and 32 fp32 activations.
__device__ __forceinline__ float mx_dot(u32x4 w, unsigned int byte, const u32x4 *x, float acc) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float m[8], f[8];
    mx_f32(w[j], mx_scale(byte), m);
    Elem<float>::to_float(x[2 * j], f);
    Elem<float>::to_float(x[2 * j + 1], f + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = fmaf(m[i], f[i], acc);
  }
  return acc;
}

// One or two tokens: a wave takes ROWS rows of the matrix, its lanes the
// blocks of a row in turn (LOADS of them each), and the activations of those
// blocks stay in registers.  No load is conditional: loads inside branches
// waited for one another's latency (15.5 us where this takes 11, 1 x 22528 x 4096).
template <typename T, int TOKENS, int LOADS, int ROWS, bool VEC>
__global__ __launch_bounds__(kMxlThreads) void mx_rows_kernel(const MxLinearArgs a) {
  constexpr int XW = sizeof(T) * 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blocks = a.k / kMxBlock;
  const int n0 = (static_cast<int>(blockIdx.x) * (kMxlThreads / 64) + wave) * ROWS;
  if (n0 >= a.n) return;
  u32x4 w[ROWS][LOADS];
  unsigned int byte[ROWS][LOADS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t row = min(n0 + r, a.n - 1);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int block = min(i * 64 + lane, blocks - 1);  // past the end: the last one again
      w[r][i] = *reinterpret_cast<const u32x4 *>(a.codes + (row * blocks + block) * 16);
      byte[r][i] = a.powers[row * blocks + block];
    }
  }
  u32x4 x[TOKENS][LOADS][XW];
#pragma unroll
  for (int t = 0; t < TOKENS; ++t)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const T *p = static_cast<const T *>(a.x) + t * a.x_stride + min(i * 64 + lane, blocks - 1) * kMxBlock;
      if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < XW; ++j) x[t][i][j] = *reinterpret_cast<const u32x4 *>(p + j * 16 / sizeof(T));
      } else {
        T e[kMxBlock];
#pragma unroll
        for (int j = 0; j < kMxBlock; ++j) e[j] = p[j];
        __builtin_memcpy(x[t][i], e, sizeof(e));
      }
    }
  // the blocks past the end count as zero, in the matrix and in the tokens
#pragma unroll
  for (int i = 0; i < LOADS; ++i)
    if (i * 64 + 64 > blocks && i * 64 + lane >= blocks) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        w[r][i] = u32x4{};
        byte[r][i] = 127;
      }
#pragma unroll
      for (int t = 0; t < TOKENS; ++t)
#pragma unroll
        for (int j = 0; j < XW; ++j) x[t][i][j] = u32x4{};
    }
  float sum[TOKENS][ROWS];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int t = 0; t < TOKENS; ++t)
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        sum[t][r] = 0.f;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) sum[t][r] = mx_dot(w[r][i], byte[r][i], x[t][i], sum[t][r]);
      }
  } else {
    // The matrix instruction of what the lanes hold: entry (i, j) is the sum
    // over g of lane (i, g)'s elements times lane (j, g)'s activations, so its
    // diagonal adds up to the sum over all lanes.
    f32x4 acc[TOKENS][ROWS];
    bool far = false;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
#pragma unroll
      for (int t = 0; t < TOKENS; ++t) acc[t][r] = f32x4{};
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const float scale = Elem<T>::kDtype == HEXKV_F16 ? near_scale(byte[r][i], &far) : mx_scale(byte[r][i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 m = Elem<T>::kDtype == HEXKV_F16 ? mx_f16(w[r][i][j], scale) : mx_bf16(w[r][i][j], scale);
#pragma unroll
          for (int t = 0; t < TOKENS; ++t)
            acc[t][r] = Elem<T>::kDtype == HEXKV_F16 ? mma_f16(m, x[t][i][j], acc[t][r]) : mma_bf16(m, x[t][i][j], acc[t][r]);
        }
      }
    }
    const int c = lane & 15;
#pragma unroll
    for (int t = 0; t < TOKENS; ++t)
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const f32x4 v = acc[t][r];
        const float d = c & 2 ? (c & 1 ? v[3] : v[2]) : (c & 1 ? v[1] : v[0]);
        sum[t][r] = c >> 2 == lane >> 4 ? d : 0.f;
      }
    if (Elem<T>::kDtype == HEXKV_F16 && __ballot(far)) {
      float check = 0.f;
#pragma unroll
      for (int t = 0; t < TOKENS; ++t)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) check = fmaf(sum[t][r], 0.f, check);
      const bool all = __ballot(!(check == 0.f)) != 0;
      if (all) {
#pragma unroll
        for (int t = 0; t < TOKENS; ++t)
#pragma unroll
          for (int r = 0; r < ROWS; ++r) sum[t][r] = 0.f;
      }
#pragma unroll 1
      for (int b = lane; b < blocks; b += 64)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          FarBlock block;
          block.read(a, min(n0 + r, a.n - 1), b, true, all);
          if (!block.any) continue;
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            float m[8], f[8];
            mx_f32(block.word(j), block.scale, m);
#pragma unroll
            for (int t = 0; t < TOKENS; ++t) {
              mx_read8(static_cast<const T *>(a.x) + t * a.x_stride + b * kMxBlock + 8 * j, false, f);
#pragma unroll
              for (int i = 0; i < 8; ++i) sum[t][r] = fmaf(m[i], f[i], sum[t][r]);
            }
          }
        }
    }
  }
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    float mine = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float v = group_sum<64>(sum[t][r]);
      if (lane == r) mine = v;
    }
    if (lane < ROWS && n0 + lane < a.n)
      static_cast<T *>(a.out)[static_cast<int64_t>(t) * a.n + n0 + lane] = Elem<T>::from_float(mine);
  }
}

// Words of 16 bytes that hold 32 activations of T as operands (fp32: three terms).
template <typename T>
constexpr int kOperandWords = sizeof(T) == 4 ? 12 : 4;

// BL bytes at p.
template <int BL>
struct PowerBytes {
  unsigned int v[BL <= 4 ? 1 : 2];
  __device__ __forceinline__ void read(const unsigned char *p) {
    if constexpr (BL == 1) {
      v[0] = *p;
    } else if constexpr (BL == 2) {
      unsigned short u;
      __builtin_memcpy(&u, p, 2);
      v[0] = u;
    } else {
      __builtin_memcpy(v, p, BL);
    }
  }
  __device__ __forceinline__ unsigned int operator[](int i) const { return v[i / 4] >> 8 * (i % 4) & 255; }
};

__device__ __forceinline__ void lds_fence() {  // orders this wave's LDS accesses
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Up to 16 MT tokens over one split of the inner dimension (1024 BL of it): each
// of eight waves takes an eighth, its tokens' operands in registers (16 MT BL of
// them), and walks the matrix 16 rows at a time; the waves join through LDS.
// What bounded it were the address units, where a load's lanes read different
// rows: the matrix's words now change lanes after the load, the tokens go through
// LDS once (64 x 22528 x 4096 31 -> 25 us, 16 x 4096 x 4096 8 -> 6).  BL: consecutive
// blocks of a row that a lane holds; RING: matrix tiles a wave has loaded or in
// flight (one more cost 1 to 5%); VEC: the activations' rows are 16-byte aligned.
template <typename T, int MT, int BL, int RING, bool VEC>
__global__ __launch_bounds__(512) void mx_few_kernel(const MxLinearArgs a) {
  constexpr int XW = kOperandWords<T>, WAVES = 8;
  // the join's, and before it the tokens on their way to the lanes
  constexpr int kJoin = 2 * WAVES * MT * 64, kStage = sizeof(T) == 2 ? WAVES * 256 * BL : 0;
  __shared__ f32x4 s_mem[kJoin > kStage ? kJoin : kStage];
  auto *s_part = reinterpret_cast<f32x4(*)[WAVES][MT][64]>(s_mem);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int row_blocks = a.k / kMxBlock, n_tiles = (a.n + 15) / 16;
  const int split = static_cast<int>(blockIdx.y) % a.splits, m0 = static_cast<int>(blockIdx.y) / a.splits * 16 * MT;
  const int block0 = split * (a.split_k / kMxBlock), blocks = min(row_blocks, block0 + a.split_k / kMxBlock);
  const int first = block0 + (wave * 4 + g) * BL;  // this lane's blocks
  // of the whole wave: none of its blocks exists, or not all of them
  const bool idle = block0 + wave * 4 * BL >= blocks, ragged = block0 + (wave + 1) * 4 * BL > blocks;

  // No load is conditional (the launch has rows of at least BL blocks): a lane
  // whose blocks do not all exist reads BL before the end, and those
  // that are not its own count as zero.
  const auto nearest = [&](int block) { return max(0, min(block, blocks - BL)); };
  const int from = nearest(first);
  const auto foreign = [&](int s) { return from + s < first || from + s >= blocks; };
  struct Tile {
    u32x4 w[BL];
    PowerBytes<BL> power;
  };
  Tile ring[RING];
  // Loaded, lane 4 c + g has what lane (c, g) needs: four lanes read one row, and
  // a load touches 16 to 32 lines instead of 64.
  const int loads_from = nearest(block0 + (wave * 4 + (lane & 3)) * BL);
  const auto fetch = [&](int tile, Tile &t) {
    const int64_t row = min(tile * 16 + (lane >> 2), a.n - 1);
    const unsigned char *p = a.codes + (row * row_blocks + loads_from) * 16;
#pragma unroll
    for (int i = 0; i < BL; ++i) t.w[i] = *reinterpret_cast<const u32x4 *>(p + i * 16);
    t.power.read(a.powers + row * row_blocks + loads_from);
  };
  const auto exchange = [&](unsigned int v) {
    return static_cast<unsigned int>(__builtin_amdgcn_ds_bpermute(16 * c + 4 * g, static_cast<int>(v)));
  };
  const int stride = static_cast<int>(gridDim.x);
  const int tile0 = static_cast<int>(blockIdx.x);
  if (!idle) fetch(tile0, ring[0]);

  // The activations of the wave's share stay in registers.  Columns behind the
  // last token repeat it (they are not stored); past the inner dimension
  // they are zero, as the matrix is.
  u32x4 x[MT][BL][XW];
  const T *tokens[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
    tokens[m] = static_cast<const T *>(a.x) + static_cast<int64_t>(min(m0 + 16 * m + c, a.rows - 1)) * a.x_stride + from * kMxBlock;
  if constexpr (sizeof(T) == 2) {
    // (through LDS: lanes that load their own token's 16 bytes touch 64 lines a
    // load, 7 of the 25 us of 64 x 22528 x 4096)
    constexpr int CH = 16 * BL;  // chunks of 8 elements of a token's share
    u32x4 *stage = reinterpret_cast<u32x4 *>(s_mem) + wave * 256 * BL;
    const int share = block0 + wave * 4 * BL;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      u32x4 v[4 * BL];
#pragma unroll
      for (int i = 0; i < 4 * BL; ++i) {
        const int at = i * 64 + lane;
        const T *row = static_cast<const T *>(a.x) + static_cast<int64_t>(min(m0 + 16 * m + at / CH, a.rows - 1)) * a.x_stride;
        v[i] = raw8(row + min(share * kMxBlock + at % CH * 8, a.k - 8), VEC);
      }
#pragma unroll
      for (int i = 0; i < 4 * BL; ++i) {
        const int at = i * 64 + lane, token = at / CH;
        stage[token * CH + (at % CH ^ (token & 7))] = v[i];
      }
      lds_fence();
#pragma unroll
      for (int s = 0; s < BL; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int chunk = max(0, from + s - share) * 4 + j;  // (a foreign block: any)
          x[m][s][j] = stage[c * CH + (chunk ^ (c & 7))];
        }
      lds_fence();
    }
    __syncthreads();
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int s = 0; s < BL; ++s) {
      const T *p = tokens[m] + s * kMxBlock;
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float f[8];
          mx_read8(p + 8 * j, VEC, f);
          terms8<3>(f, &x[m][s][3 * j]);
        }
      }
    }
  if (ragged) {
#pragma unroll
    for (int s = 0; s < BL; ++s)
      if (foreign(s)) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < XW; ++j) x[m][s][j] = u32x4{};
      }
  }
#pragma unroll
  for (int r = 1; r < RING; ++r)
    if (!idle) fetch(tile0 + r * stride, ring[r]);

  for (int base = tile0, turn = 0; base < n_tiles; base += RING * stride) {
#pragma unroll
    for (int r = 0; r < RING; ++r, ++turn) {
      const int tile = base + r * stride;
      if (tile >= n_tiles) break;
      f32x4 acc[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m] = f32x4{};
      bool far = false;
      if (!idle) {
        Tile &t = ring[r];
        unsigned int byte[BL];
#pragma unroll
        for (int s = 0; s < BL; ++s) {
#pragma unroll
          for (int j = 0; j < 4; ++j) t.w[s][j] = exchange(t.w[s][j]);
        }
#pragma unroll
        for (int i = 0; i < (BL + 3) / 4; ++i) t.power.v[i] = exchange(t.power.v[i]);
#pragma unroll
        for (int s = 0; s < BL; ++s) byte[s] = t.power[s];
        if (ragged) {
#pragma unroll
          for (int s = 0; s < BL; ++s)
            if (foreign(s)) {
              t.w[s] = u32x4{};
              byte[s] = 127;
            }
        }
#pragma unroll
        for (int s = 0; s < BL; ++s) {
          const float scale = Elem<T>::kDtype == HEXKV_F16 ? near_scale(byte[s], &far) : mx_scale(byte[s]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) {
              const u32x4 w = mx_bf16(t.w[s][j], scale);
#pragma unroll
              for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < 3; ++n) acc[m] = mma_bf16(w, x[m][s][3 * j + n], acc[m]);
            } else if constexpr (Elem<T>::kDtype == HEXKV_BF16) {
              const u32x4 w = mx_bf16(t.w[s][j], scale);
#pragma unroll
              for (int m = 0; m < MT; ++m) acc[m] = mma_bf16(w, x[m][s][j], acc[m]);
            } else {
              const u32x4 w = mx_f16(t.w[s][j], scale);
#pragma unroll
              for (int m = 0; m < MT; ++m) acc[m] = mma_f16(w, x[m][s][j], acc[m]);
            }
          }
        }
        fetch(tile + RING * stride, t);  // (past the end the last row again)
      }
      if (Elem<T>::kDtype == HEXKV_F16 && __ballot(far)) {
        const int64_t row = min(tile * 16 + c, a.n - 1);
        float check = 0.f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) check = fmaf(acc[m][i], 0.f, check);
        const bool all = __ballot(!(check == 0.f)) != 0;
        if (all) {
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m] = f32x4{};
        }
#pragma unroll 1
        for (int s = 0; s < BL; ++s) {
          FarBlock block;
          block.read(a, row, from + s, !foreign(s), all);
          if (!__ballot(block.any)) continue;
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            const u32x4 w = block.operand(j);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              u32x4 terms[2];
              far_terms(reinterpret_cast<const _Float16 *>(tokens[m]) + s * kMxBlock + 8 * j, !foreign(s), terms);
              acc[m] = mma_bf16(w, terms[1], mma_bf16(w, terms[0], acc[m]));
            }
          }
        }
      }
      // Two halves of LDS in turn: a wave writes one again only after the
      // barrier that follows the reading of it.
#pragma unroll
      for (int m = 0; m < MT; ++m) s_part[turn & 1][wave][m][lane] = acc[m];
      __syncthreads();
      // acc: column c is the token, rows 4 g + i are the matrix's
      const int m = (wave + turn * MT) % WAVES;
      if (m < MT) {
        f32x4 sum = s_part[turn & 1][0][m][lane];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) sum += s_part[turn & 1][i][m][lane];
        const int token = m0 + 16 * m + c, n = tile * 16 + 4 * g;
        if (token < a.rows && n < a.n) {
          const int64_t at = static_cast<int64_t>(token) * a.n + n;
          const int count = min(4, a.n - n);
          if (a.splits > 1) {
            float *o = a.partial + static_cast<int64_t>(split) * a.rows * a.n + at;
            if (count == 4) store4(o, sum);
            else for (int i = 0; i < count; ++i) o[i] = sum[i];
          } else {
            T *o = static_cast<T *>(a.out) + at;
            if (count == 4) store4(o, sum);
            else for (int i = 0; i < count; ++i) o[i] = Elem<T>::from_float(sum[i]);
          }
        }
      }
    }
  }
}

// fp32 above 16 tokens: a workgroup takes 32 MT WM tokens by 32 NT WN rows of the matrix;
// its waves are WM x WN pieces of that, times WK that share the inner
// dimension.  A step is STEPS times 64 of the inner dimension for each of the
// WK: the tokens' piece of it lies in LDS (two of them, loaded through
// registers while the other is used), in 16-byte chunks permuted within a row so that
// a wave's reads of one chunk of 32 rows meet every bank equally; the matrix
// goes straight to the registers of the waves that convert it, one step
// ahead.  v_mfma_f32_32x32x16: lane (c, h) holds one block of row c, half h of 64,
// and the tokens' operand the same elements.
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int MT_, int NT_, int WM_, int WN_, int WK_, int STEPS_, int RING_, int XR_>
struct MxTileShape {
  static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, WK = WK_, STEPS = STEPS_, RING = RING_, XR = XR_;
  static_assert(RING % XR == 0 && RING % 2 == 0, "the loop is unrolled by the ring");
  static constexpr int kWaves = WM * WN * WK, kThreads = 64 * kWaves;
  static constexpr int kTokens = 32 * MT * WM, kRows = 32 * NT * WN;
  static constexpr int kStep = 64 * WK * STEPS;            // inner dimension of one step
  static constexpr int kPlanes = 3;                        // 16-bit terms of an activation in LDS
  static constexpr int kChunks = kStep / 8;                // 16-byte chunks of a token's row in LDS
  static constexpr int kPlane = kTokens * kChunks;         // chunks of a plane
  static constexpr int kLoads = kPlane / kThreads;         // chunks a thread stages
  static constexpr size_t kLds = size_t{16} * 2 * kPlanes * kPlane;
  static_assert(kPlane % kThreads == 0, "every thread stages as much");
  static_assert(static_cast<size_t>(WK / 2) * WM * WN * MT * NT * 16 * 64 * 4 <= kLds, "the join fits the stage");
};

__device__ __forceinline__ f32x16 mma32_bf16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32_f16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The blocks whose power fp16 does not hold, in bf16; all blocks, from zero,
// where the sum is not finite.
template <typename T, typename S>
__device__ __forceinline__ void tile_far(const MxLinearArgs &a, int m0, int n0, int k_first, int k_last, int wm, int wn,
                                         int c, int h, f32x16 (&acc)[S::MT][S::NT]) {
  constexpr int MT = S::MT, NT = S::NT;
  float check = 0.f;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) check = fmaf(acc[m][t][i], 0.f, check);
  const bool all = __ballot(!(check == 0.f)) != 0;
  if (all) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[m][t] = f32x16{};
  }
#pragma unroll 1
  for (int k0 = k_first; k0 < k_last; k0 += S::kStep)
#pragma unroll 1
    for (int s = 0; s < S::STEPS; ++s) {
      const int k = k0 + s * 64 + h * kMxBlock;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        FarBlock block;
        block.read(a, min(n0 + (wn * NT + t) * 32 + c, a.n - 1), k / kMxBlock, k < k_last, all);
        if (!__ballot(block.any)) continue;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int token = min(m0 + (wm * MT + m) * 32 + c, a.rows - 1);
          const _Float16 *p = static_cast<const _Float16 *>(a.x) + static_cast<int64_t>(token) * a.x_stride + k;
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            u32x4 terms[2];
            far_terms(p + 8 * j, k < k_last, terms);
            const u32x4 w = block.operand(j);
            acc[m][t] = mma32_bf16(w, terms[1], mma32_bf16(w, terms[0], acc[m][t]));
          }
        }
      }
    }
}

template <typename T, typename S>
__device__ __forceinline__ void tile_store(const MxLinearArgs &a, int m0, int n0, int split, int wm, int wn, int c, int h,
                                           const f32x16 (&acc)[S::MT][S::NT]) {
  constexpr int MT = S::MT, NT = S::NT;
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

template <typename S, bool VEC>
__global__ __launch_bounds__(S::kThreads) void mx_tile_kernel(const MxLinearArgs a) {
  using T = float;
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

  // Every load is a uniform base that moves along the inner dimension plus a
  // lane's constant 32-bit offset, and none is conditional: in the last step
  // what lies past the end is the split's last piece again, and counts as zero.
  const char *x_base = static_cast<const char *>(a.x) + static_cast<int64_t>(m0) * a.x_stride * sizeof(T);
  const unsigned char *w_base = a.codes + static_cast<int64_t>(n0) * (a.k / 2);
  const unsigned char *p_base = a.powers + static_cast<int64_t>(n0) * (a.k / kMxBlock);
  unsigned int x_off[S::kLoads], w_off[NT], p_off[NT];
#pragma unroll
  for (int i = 0; i < S::kLoads; ++i) {
    const int at = i * S::kThreads + tid, token = min(at / CH, a.rows - 1 - m0);
    x_off[i] = (static_cast<unsigned int>(token) * static_cast<unsigned int>(a.x_stride) + at % CH * 8) * sizeof(T);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const unsigned int row = min((wn * NT + t) * 32 + c, a.n - 1 - n0);
    w_off[t] = row * (a.k / 2) + wk * S::STEPS * 32 + h * 16;
    p_off[t] = row * (a.k / kMxBlock) + wk * S::STEPS * 2 + h;
  }

  struct Tokens {
    u32x4 v[2][S::kLoads];
  };
  const auto fetch_x = [&](int k0, Tokens &stage) {
    const char *base = x_base + static_cast<int64_t>(k0) * sizeof(T);
    const bool whole = k0 + S::kStep <= k_last;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      unsigned int off = x_off[i];
      if (!whole) off -= max(0, k0 + (i * S::kThreads + tid) % CH * 8 - (k_last - 8)) * sizeof(T);
      const T *p = reinterpret_cast<const T *>(base + off);
      u32x4 f[2];
      if constexpr (VEC) {
        f[0] = *reinterpret_cast<const u32x4 *>(p);
        f[1] = *reinterpret_cast<const u32x4 *>(p + 4);
      } else {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = p[j];
        __builtin_memcpy(f, e, sizeof(e));
      }
      stage.v[0][i] = f[0];
      stage.v[1][i] = f[1];
    }
  };
  // (Tokens past the last repeat it and are not stored.)
  const auto store_x = [&](int buf, int k0, const Tokens &stage) {
    const bool whole = k0 + S::kStep <= k_last;
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int at = i * S::kThreads + tid, token = at / CH, chunk = at % CH;
      u32x4 terms[PL];
      float f[8];
      Elem<float>::to_float(stage.v[0][i], f);
      Elem<float>::to_float(stage.v[1][i], f + 4);
      terms8<3>(f, terms);
      if (!whole && k0 + chunk * 8 >= k_last) {
#pragma unroll
        for (int n = 0; n < PL; ++n) terms[n] = u32x4{};
      }
#pragma unroll
      for (int n = 0; n < PL; ++n)
        s_x[(buf * PL + n) * S::kPlane + token * CH + (chunk ^ (token / kSpread & kMask))] = terms[n];
    }
  };
  struct Weights {
    u32x4 w[S::STEPS][NT];
    unsigned int byte[S::STEPS][NT];
  };
  const auto fetch_w = [&](int k0, Weights &x) {
    const unsigned char *w = w_base + k0 / 2, *p = p_base + k0 / kMxBlock;
    const bool whole = k0 + S::kStep <= k_last;
#pragma unroll
    for (int s = 0; s < S::STEPS; ++s) {
      // blocks this lane's lies past the last one
      const int past = whole ? 0 : max(0, k0 / kMxBlock + (wk * S::STEPS + s) * 2 + h - (k_last / kMxBlock - 1));
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        x.w[s][t] = *reinterpret_cast<const u32x4 *>(w + (w_off[t] + s * 32 - past * 16));
        x.byte[s][t] = p[p_off[t] + s * 2 - past];
      }
    }
  };

  f32x16 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x16{};

  const auto compute = [&](int buf, int k0, Weights &x) {
    if (k0 + S::kStep > k_last) {  // what lies past the end counts as zero
#pragma unroll
      for (int s = 0; s < S::STEPS; ++s)
        if (k0 + (wk * S::STEPS + s) * 64 + h * kMxBlock >= k_last) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            x.w[s][t] = u32x4{};
            x.byte[s][t] = 127;
          }
        }
    }
#pragma unroll
    for (int s = 0; s < S::STEPS; ++s) {
      float scale[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t)
        scale[t] = mx_scale(x.byte[s][t]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 b[PL][MT];
#pragma unroll
        for (int n = 0; n < PL; ++n)
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const int token = (wm * MT + m) * 32 + c, chunk = (wk * S::STEPS + s) * 8 + h * 4 + j;
            b[n][m] = s_x[(buf * PL + n) * S::kPlane + token * CH + (chunk ^ (token / kSpread & kMask))];
          }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const u32x4 w = mx_bf16(x.w[s][t][j], scale[t]);
#pragma unroll
          for (int n = 0; n < PL; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m][t] = mma32_bf16(w, b[n][m], acc[m][t]);
        }
      }
    }
  };

  Weights ring[S::RING];
  Tokens xs[S::XR];
  fetch_x(k_first, xs[0]);
  fetch_w(k_first, ring[0]);
#pragma unroll
  for (int r = 1; r < S::RING; ++r) {  // in the order of their use
    if (r < S::XR && k_first + r * S::kStep < k_last) fetch_x(k_first + r * S::kStep, xs[r]);
    if (r < S::RING - 1 && k_first + r * S::kStep < k_last) fetch_w(k_first + r * S::kStep, ring[r]);
  }
  store_x(0, k_first, xs[0]);
  __syncthreads();
  for (int base = k_first; base < k_last; base += S::RING * S::kStep) {
#pragma unroll
    for (int r = 0; r < S::RING; ++r) {
      const int k0 = base + r * S::kStep;
      if (k0 >= k_last) break;
      if (k0 + S::XR * S::kStep < k_last) fetch_x(k0 + S::XR * S::kStep, xs[r % S::XR]);
      if (k0 + (S::RING - 1) * S::kStep < k_last) fetch_w(k0 + (S::RING - 1) * S::kStep, ring[(r + S::RING - 1) % S::RING]);
      compute(r & 1, k0, ring[r]);
      if (k0 + S::kStep < k_last) store_x((r + 1) & 1, k0 + S::kStep, xs[(r + 1) % S::XR]);
      __syncthreads();
    }
  }

  // the waves that share the inner dimension join, half of them at a time
  if constexpr (S::WK > 1) {
    float *s_acc = reinterpret_cast<float *>(s_mem);
    constexpr int kPiece = MT * NT * 16 * 64;
#pragma unroll
    for (int half = S::WK / 2; half > 0; half /= 2) {
      if (wk >= half && wk < 2 * half) {
        float *p = s_acc + ((wk - half) * S::WM * S::WN + wm * S::WN + wn) * kPiece + lane;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) p[((m * NT + t) * 16 + i) * 64] = acc[m][t][i];
      }
      __syncthreads();
      if (wk < half) {
        const float *p = s_acc + (wk * S::WM * S::WN + wm * S::WN + wn) * kPiece + lane;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[m][t][i] += p[((m * NT + t) * 16 + i) * 64];
      }
      if (half > 1) __syncthreads();
    }
    if (wk > 0) return;
  }
  tile_store<T, S>(a, m0, n0, split, wm, wn, c, h, acc);
}

// A prompt's tile (16-bit data): as mx_tile_kernel, but the matrix reaches its
// waves through LDS as well, in four bits, so that a load's four lanes read one
// row (lanes of different rows each cost a line: the address units were
// the bound at 27% of the matrix cores), and each element is loaded once a workgroup.  A step is 128 of
// the inner dimension in one buffer, the next one's in registers; several
// workgroups a CU fill the barriers.
template <typename T, int MT_, int NT_, int WM_, int WN_>
struct MxPromptShape {
  static constexpr int MT = MT_, NT = NT_, WM = WM_, WN = WN_, STEPS = 2;
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int kTokens = 32 * MT * WM, kRows = 32 * NT * WN, kStep = 128;
  static constexpr int kChunks = kStep / 8;
  static constexpr int kLoads = kTokens * kChunks / kThreads;     // chunks of the tokens a thread stages
  static constexpr int kLoadsW = kRows * 4 / kThreads;            // blocks of the matrix
  static constexpr size_t kLds = size_t{16} * (kTokens * kChunks + kRows * 4) + size_t{4} * kRows;
  static_assert(kTokens * kChunks % kThreads == 0 && kRows * 4 % kThreads == 0, "every thread stages as much");
  static_assert(kThreads % kRows == 0 || kRows % kThreads == 0, "powers");
};

template <typename T, typename S, bool VEC>
__global__ __launch_bounds__(S::kThreads, 2) void mx_prompt_kernel(const MxLinearArgs a) {
  constexpr int MT = S::MT, NT = S::NT, CH = S::kChunks;
  constexpr int PR = S::kRows > S::kThreads ? S::kRows / S::kThreads : 1;  // rows' powers a thread stages
  __shared__ __attribute__((aligned(16))) char s_mem[S::kLds];
  u32x4 *s_x = reinterpret_cast<u32x4 *>(s_mem);           // [tokens][chunks], chunk c of token t at c ^ t % 16
  u32x4 *s_w = s_x + S::kTokens * CH;                       // [rows][4], block b of row r at b ^ r / 4 % 4
  unsigned int *s_p = reinterpret_cast<unsigned int *>(s_w + S::kRows * 4);  // [rows] the four blocks' powers
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5, wn = wave % S::WN, wm = wave / S::WN;

  // (XCDs and pieces as in mx_tile_kernel)
  const int local = static_cast<int>(blockIdx.x >> 3);
  const int group = local / a.m_tiles * 8 + static_cast<int>(blockIdx.x & 7);
  const int m0 = (local % a.m_tiles) * S::kTokens;
  if (group >= a.n_tiles * a.splits) return;
  const int n0 = group / a.splits * S::kRows, split = group % a.splits;
  const int k_first = split * a.split_k, k_last = min(a.k, k_first + a.split_k);
  const int blocks = a.k / kMxBlock;  // at least 4

  const char *x_base = static_cast<const char *>(a.x) + static_cast<int64_t>(m0) * a.x_stride * sizeof(T);
  const unsigned char *w_base = a.codes + static_cast<int64_t>(n0) * (a.k / 2);
  const unsigned char *p_base = a.powers + static_cast<int64_t>(n0) * blocks;
  unsigned int x_off[S::kLoads], w_off[S::kLoadsW], p_off[PR];
#pragma unroll
  for (int i = 0; i < S::kLoads; ++i) {
    const int at = i * S::kThreads + tid, token = min(at / CH, a.rows - 1 - m0);
    x_off[i] = (static_cast<unsigned int>(token) * static_cast<unsigned int>(a.x_stride) + at % CH * 8) * sizeof(T);
  }
#pragma unroll
  for (int i = 0; i < S::kLoadsW; ++i) {
    const int at = i * S::kThreads + tid;
    w_off[i] = static_cast<unsigned int>(min(at / 4, a.n - 1 - n0)) * (a.k / 2) + at % 4 * 16;
  }
#pragma unroll
  for (int i = 0; i < PR; ++i)
    p_off[i] = static_cast<unsigned int>(min((i * S::kThreads + tid) % S::kRows, a.n - 1 - n0)) * blocks;

  // In the last step what lies past the end is loaded from the last piece (the
  // powers from the row's last four) and counts as zero.
  u32x4 x[S::kLoads], w[S::kLoadsW];
  unsigned int pw[PR];
  const auto fetch = [&](int k0) {
    const bool whole = k0 + S::kStep <= k_last;
    const char *xp = x_base + static_cast<int64_t>(k0) * sizeof(T);
    const unsigned char *wp = w_base + k0 / 2, *pp = p_base + min(k0 / kMxBlock, blocks - 4);
#pragma unroll
    for (int i = 0; i < S::kLoadsW; ++i) {
      unsigned int off = w_off[i];
      if (!whole) off -= max(0, k0 / kMxBlock + tid % 4 - (k_last / kMxBlock - 1)) * 16;
      w[i] = *reinterpret_cast<const u32x4 *>(wp + off);
    }
#pragma unroll
    for (int i = 0; i < PR; ++i) __builtin_memcpy(&pw[i], pp + p_off[i], 4);
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      unsigned int off = x_off[i];
      if (!whole) off -= max(0, k0 + (i * S::kThreads + tid) % CH * 8 - (k_last - 8)) * sizeof(T);
      x[i] = raw8(reinterpret_cast<const T *>(xp + off), VEC);
    }
  };
  const auto store = [&](int k0) {
    if (k0 + S::kStep > k_last) {
      const int past = k0 / kMxBlock + 4 - k_last / kMxBlock;  // blocks of this step past the end, 1 to 3
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i)
        if (k0 + (i * S::kThreads + tid) % CH * 8 >= k_last) x[i] = u32x4{};
#pragma unroll
      for (int i = 0; i < S::kLoadsW; ++i)
        if (tid % 4 >= 4 - past) w[i] = u32x4{};
#pragma unroll
      for (int i = 0; i < PR; ++i) pw[i] = pw[i] >> (8 * past) | 0x7f7f7f7fu << (32 - 8 * past);
    }
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int at = i * S::kThreads + tid, token = at / CH;
      s_x[token * CH + (at % CH ^ (token & 15))] = x[i];
    }
#pragma unroll
    for (int i = 0; i < S::kLoadsW; ++i) {
      const int at = i * S::kThreads + tid, row = at / 4;
      s_w[row * 4 + (at % 4 ^ (row >> 2 & 3))] = w[i];
    }
#pragma unroll
    for (int i = 0; i < PR; ++i)
      if (PR > 1 || tid < S::kRows) s_p[i * S::kThreads + tid] = pw[i];
  };

  f32x16 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x16{};
  bool far = false;
  const auto compute = [&]() {
    unsigned int bytes[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) bytes[t] = s_p[(wn * NT + t) * 32 + c] >> (8 * h);
#pragma unroll
    for (int s = 0; s < S::STEPS; ++s) {
      float scale[NT];
      u32x4 block[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const unsigned int byte = bytes[t] >> (16 * s) & 255;
        scale[t] = Elem<T>::kDtype == HEXKV_F16 ? near_scale(byte, &far) : mx_scale(byte);
        const int row = (wn * NT + t) * 32 + c;
        block[t] = s_w[row * 4 + ((s * 2 + h) ^ (row >> 2 & 3))];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 b[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int token = (wm * MT + m) * 32 + c;
          b[m] = s_x[token * CH + ((s * 8 + h * 4 + j) ^ (token & 15))];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (Elem<T>::kDtype == HEXKV_F16) {
            const u32x4 e = mx_f16(block[t][j], scale[t]);
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m][t] = mma32_f16(e, b[m], acc[m][t]);
          } else {
            const u32x4 e = mx_bf16(block[t][j], scale[t]);
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m][t] = mma32_bf16(e, b[m], acc[m][t]);
          }
        }
      }
    }
  };

  fetch(k_first);
  for (int k0 = k_first; k0 < k_last; k0 += S::kStep) {
    store(k0);
    __syncthreads();
    fetch(min(k0 + S::kStep, k_last - kMxBlock));  // (after the last step: loaded, never used)
    compute();
    __syncthreads();
  }
  if (Elem<T>::kDtype == HEXKV_F16 && __ballot(far)) tile_far<T, S>(a, m0, n0, k_first, k_last, wm, wn, c, h, acc);
  tile_store<T, S>(a, m0, n0, split, wm, wn, c, h, acc);
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

// The kernels and tiles a call may run, by tokens (GPU time of a call on MI355X,
// weights from memory, bf16 unless said):
//   1, 2    kRows: 1 x 22528 x 4096 11 us (4.4 TB/s); kFew 14.
//   3-64    kFew, 16, 32 or 64 tokens a wave (16 x 22528 x 4096 15 us, 32 x 17, 64 x 25;
//           64 x 4096 x 4096 11.2, where a tile of the tokens in LDS took 14.8; 32 x
//           2560 x 2048 4.6 and 9.0; 32 x 4096 x 11264 18.7 and 17.8).
//           fp32: to 16, then tiles (three registers a token of each).
//   65-     16-bit: mx_prompt_kernel, by tiles of 64 tokens x 128 rows up to
//           kNarrowTokens (128 x 22528 x 4096 45 us, x 256 rows 49; 300 x 6144 x
//           4096 30.5 / 32.3), then 64 x 256 (611 x 4096 x 11264 76 us, x 128
//           rows over 82), and 128 x 256 where those make kLargeTiles (2048 x
//           22528 x 4096 355 us, 1.06 PFLOP/s; 64 x 256 over 369; 611 x 4096 x
//           11264 80 / 76).
//           Below 128 of the inner dimension, kFew 64 at a time.  fp32:
//           mx_tile_kernel, 64 tokens up to kWideTokens, 128 above.
enum MxKind { kRows, kFew16, kFew32, kFew64, kTile32, kTile64, kNarrow, kPrompt, kLarge, kWide32, kWider32 };
constexpr int kNarrowTokens = 320, kLargeTiles = 512, kWideTokens = 192;

struct MxPlan {
  int kind;
  int blocks;  // kRows: loads of a lane; kFew*: blocks of a lane
  int m_tiles, n_tiles, splits, split_k;
};

using Tile32 = MxTileShape<1, 1, 1, 2, 2, 1, 4, 4>;
using Tile64 = MxTileShape<2, 1, 1, 2, 2, 1, 4, 2>;
template <typename T> using Narrow = MxPromptShape<T, 1, 2, 2, 2>;
template <typename T> using Prompt = MxPromptShape<T, 2, 2, 1, 4>;
template <typename T> using Large = MxPromptShape<T, 2, 4, 2, 2>;
using Wide32 = MxTileShape<2, 2, 1, 2, 2, 1, 2, 2>;
using Wider32 = MxTileShape<2, 2, 2, 2, 1, 1, 2, 1>;

// Splits of the inner dimension: two workgroups a CU, at least four steps each.
template <typename S>
static void plan_tile(MxPlan *p, int kind, int rows, int n, int k) {
  p->kind = kind;
  p->m_tiles = (rows + S::kTokens - 1) / S::kTokens;
  p->n_tiles = (n + S::kRows - 1) / S::kRows;
  const int steps = (k + S::kStep - 1) / S::kStep;
  const int splits = std::max(1, std::min(steps / 4, 512 / std::max(1, p->m_tiles * p->n_tiles)));
  p->split_k = (steps + splits - 1) / splits * S::kStep;
  p->splits = (k + p->split_k - 1) / p->split_k;
}

// Blocks a lane holds of a row: a wave's share of eight, or as much of it as
// leaves the activations 128 registers; more is further splits.
static void plan_few(MxPlan *p, int kind, int most, int rows, int k) {
  p->kind = kind;
  p->blocks = 1;
  while (p->blocks < most && k > 1024 * p->blocks) p->blocks *= 2;
  p->m_tiles = kind == kFew16 ? 1 : (rows + 63) / 64;
  p->split_k = 1024 * p->blocks;
  p->splits = (k + p->split_k - 1) / p->split_k;
}

template <typename T>
static MxPlan mx_plan(int rows, int n, int k) {
  MxPlan p = {};
  p.splits = 1;
  // kRows: the registers hold 6 blocks a lane of one token, 4 of two (fp32: 4, 2)
  const int loads = (k + 2047) / 2048, most = (rows == 1 ? 6 : 4) - (sizeof(T) == 4 ? 2 : 0);
  if (rows <= 2 && loads <= most) {
    p.kind = kRows;
    p.blocks = loads <= 2 ? loads : loads <= 4 ? 4 : 6;
  } else if (rows <= 16) {
    plan_few(&p, kFew16, sizeof(T) == 4 ? 2 : 4, rows, k);
  } else if constexpr (sizeof(T) == 4) {
    if (rows <= 32) plan_tile<Tile32>(&p, kTile32, rows, n, k);
    else if (rows <= 64) plan_tile<Tile64>(&p, kTile64, rows, n, k);
    else if (rows <= kWideTokens) plan_tile<Wide32>(&p, kWide32, rows, n, k);
    else plan_tile<Wider32>(&p, kWider32, rows, n, k);
  } else if (rows <= 32) {
    plan_few(&p, kFew32, 4, rows, k);
  } else if (rows <= 64 || k < 128) {
    plan_few(&p, kFew64, 2, rows, k);
  } else if (rows <= kNarrowTokens) {
    plan_tile<Narrow<T>>(&p, kNarrow, rows, n, k);
  } else {
    plan_tile<Large<T>>(&p, kLarge, rows, n, k);
    if (p.m_tiles * p.n_tiles < kLargeTiles) plan_tile<Prompt<T>>(&p, kPrompt, rows, n, k);
  }
  return p;
}

static MxPlan mx_plan_of(int rows, int n, int k, int dtype) {
  return dtype == HEXKV_F32 ? mx_plan<float>(rows, n, k) : mx_plan<__bf16>(rows, n, k);
}

static size_t mx_partial_bytes(const MxPlan &p, int rows, int n) {
  return p.splits > 1 ? static_cast<size_t>(p.splits) * rows * n * sizeof(float) : 0;
}

template <typename S>
static void launch_tile(const MxLinearArgs &a, hipStream_t s) {
  static_assert(S::kLds <= 160 * 1024, "LDS");
  const unsigned groups = static_cast<unsigned>(a.n_tiles * a.splits + 7) / 8 * 8;
  if (a.vec) mx_tile_kernel<S, true><<<groups * a.m_tiles, S::kThreads, 0, s>>>(a);
  else mx_tile_kernel<S, false><<<groups * a.m_tiles, S::kThreads, 0, s>>>(a);
}

template <typename T, typename S>
static void launch_prompt(const MxLinearArgs &a, hipStream_t s) {
  static_assert(S::kLds <= 64 * 1024, "LDS");
  const unsigned groups = static_cast<unsigned>(a.n_tiles * a.splits + 7) / 8 * 8;
  if (a.vec) mx_prompt_kernel<T, S, true><<<groups * a.m_tiles, S::kThreads, 0, s>>>(a);
  else mx_prompt_kernel<T, S, false><<<groups * a.m_tiles, S::kThreads, 0, s>>>(a);
}

template <typename T, int TOKENS, int LOADS, int ROWS>
static void launch_rows(const MxLinearArgs &a, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>((a.n + 4 * ROWS - 1) / (4 * ROWS));
  if (a.vec) mx_rows_kernel<T, TOKENS, LOADS, ROWS, true><<<grid, kMxlThreads, 0, s>>>(a);
  else mx_rows_kernel<T, TOKENS, LOADS, ROWS, false><<<grid, kMxlThreads, 0, s>>>(a);
}

// Matrix rows a wave takes: as many as the registers hold beside the tokens
// (1 x 4096 x 4096 4.1 us with 4 and with 2, 1 x 8192 x 8192 8.4 with 4, 9.5 with 2).
template <typename T, int TOKENS>
static void launch_rows(const MxLinearArgs &a, int loads, hipStream_t s) {
  constexpr bool wide = sizeof(T) == 4;
  if (loads == 1) return launch_rows<T, TOKENS, 1, 4>(a, s);
  if (loads == 2) return launch_rows<T, TOKENS, 2, wide && TOKENS == 2 ? 2 : 4>(a, s);
  if constexpr (!wide || TOKENS == 1)
    if (loads == 4) return launch_rows<T, TOKENS, 4, wide || TOKENS == 2 ? 2 : 4>(a, s);
  if constexpr (!wide && TOKENS == 1)
    if (loads == 6) return launch_rows<T, TOKENS, 6, 2>(a, s);
}

// One workgroup of eight waves a CU, shared out among the splits.
template <typename T, int MT, int BL, int RING>
static void launch_few(const MxLinearArgs &a, hipStream_t s) {
  const int groups = a.splits * a.m_tiles;
  const dim3 grid(static_cast<unsigned>(std::min((a.n + 15) / 16, std::max(1, (256 + groups - 1) / groups))),
                  static_cast<unsigned>(groups));
  if (a.vec) mx_few_kernel<T, MT, BL, RING, true><<<grid, 512, 0, s>>>(a);
  else mx_few_kernel<T, MT, BL, RING, false><<<grid, 512, 0, s>>>(a);
}

template <typename T>
static void mx_linear_launch(MxLinearArgs a, const MxPlan &p, hipStream_t s) {
  a.m_tiles = p.m_tiles;
  a.n_tiles = p.n_tiles;
  a.splits = p.splits;
  a.split_k = p.split_k;
  switch (p.kind) {
    case kRows:
      if (a.rows == 1) launch_rows<T, 1>(a, p.blocks, s);
      else launch_rows<T, 2>(a, p.blocks, s);
      break;
    // more than one block a lane only where k > 512 times it: a row then has
    // more than 16 times as many
    case kFew16:
      if (p.blocks == 1) launch_few<T, 1, 1, 2>(a, s);
      else if (p.blocks == 2) launch_few<T, 1, 2, 1>(a, s);
      else if constexpr (sizeof(T) == 2) launch_few<T, 1, 4, 1>(a, s);
      break;
    case kFew32:
      if constexpr (sizeof(T) == 2) {
        if (p.blocks == 1) launch_few<T, 2, 1, 2>(a, s);
        else if (p.blocks == 2) launch_few<T, 2, 2, 1>(a, s);
        else launch_few<T, 2, 4, 1>(a, s);
      }
      break;
    case kFew64:
      if constexpr (sizeof(T) == 2) {
        if (p.blocks == 1) launch_few<T, 4, 1, 2>(a, s);
        else launch_few<T, 4, 2, 1>(a, s);
      }
      break;
    default:
      if constexpr (sizeof(T) == 4) {
        if (p.kind == kTile32) launch_tile<Tile32>(a, s);
        else if (p.kind == kTile64) launch_tile<Tile64>(a, s);
        else if (p.kind == kWide32) launch_tile<Wide32>(a, s);
        else launch_tile<Wider32>(a, s);
      } else {
        if (p.kind == kNarrow) launch_prompt<T, Narrow<T>>(a, s);
        else if (p.kind == kPrompt) launch_prompt<T, Prompt<T>>(a, s);
        else launch_prompt<T, Large<T>>(a, s);
      }
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
  if (k > (1 << 22)) return fail(HEXKV_ERANGE, "%s: k above 2^22", what);
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
  // a tile's tokens are addressed with 32-bit offsets from its first
  if (rows > 1 && (x_stride < 0 || x_stride > (1 << 22)))
    return fail(HEXKV_ERANGE, "%s: x_stride %lld outside [0, 2^22]", what, static_cast<long long>(x_stride));
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
