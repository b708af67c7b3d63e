// Attention over a 4-bit cache: hexkv_mx_attend.
//
// A workgroup takes up to 16 query rows that share a KV head (the heads of a
// group, and several positions' where there are) over one partition of the
// keys; its waves take 32 keys at a time in turn:
//   S^T = K Q^T    v_mfma_f32_16x16x32_bf16.  Lane (c, g) holds a quarter of
//                  key c's elements, the query's operand the same quarter in
//                  the same order, so a lane's vector of elements is its
//                  operand as it stands.  Loads go four lanes to a row (16
//                  lines a load and not 64: the address units were busy three
//                  quarters of the time), and the words change lanes in 4 bits.
//                  The conversion from 4 bits takes the power with it and is
//                  exact in bf16 for every power (fp16 would end at 2^15); the
//                  query enters as one (bf16), two (fp16) or three (fp32) bf16
//                  terms that add up to it exactly.
//   softmax        per lane (its query row), in the log2 domain; the running
//                  maximum moves only when a score exceeds it by 2^kSlack.
//   O^T += V^T P^T the scores' layout is the operand as it stands; V^T comes
//                  from row-major LDS (bf16, written by the lanes that
//                  converted it) by transposing reads.  Probabilities enter as two
//                  bf16 terms, each rounded (off by 2^-16 of the probability at
//                  most; three for fp32: exact), both products in fp32.
//                  Truncated terms (2^-14, all to one side) turned 3.4 in
//                  1000 bf16 outputs to a neighbour, rounded ones 0.5, three
//                  terms 0.3 at 3% more time (64 sequences of 128 to 8192).
// A lane's accumulators belong to its own row, so rescaling and the final
// division need no exchange.  The waves' sums meet in LDS; rows split over
// partitions leave (sum, maximum, unscaled output) in the workspace and a
// second kernel joins them.
//
// Measured (append included, bf16, head_dim 128, 32 query heads on 8 KV heads):
// 64 sequences of 128 to 8192 81 us, 3.2 TB/s; reading alone could reach 7.1 (36
// us).  What bounds it is a step's own instructions: VALU 41% and LDS 37% of the
// cycles (a third of the latter bank conflicts of V's stores), matrix cores
// 15%, at 2.6 waves per SIMD that wait for memory 30% of their time.  Few keys a
// wave are bound by a step's latency, about 1 us from LDS to the last product;
// loading two or three steps ahead instead of one cost 3 to 10%
// (registers), steps of one wave a partition 12% at 64 sequences and 20 to 60%
// at one to four.  16 x 90 rows over 2048 keys: 122 us, VALU 64% and LDS 58% busy
// (a tile of 16 rows converts every key for itself).
//
// A NaN block of V, or one with an element that fp32 does not hold (2^128 and
// above), is taken out of the product (0 times either is a NaN, which would reach
// rows that do not attend it); the rows that do get NaN there.
#include "hexkv_mx.h"

#include <algorithm>

namespace hexkv {

constexpr int kMxaMaxWaves = 8;
constexpr int kXcds = 8;
constexpr int kMxaRows = 16;  // query rows of a wave
constexpr int kMxaKeys = 32;  // keys of one step
constexpr float kMxaLowest = -3.4028234e38f;  // the running maximum's start: the lowest float, finite in differences
constexpr float kMxaSlack = 8.f;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

struct MxAttendArgs {
  const void *q;
  int64_t q_bs, q_rs;  // elements
  unsigned char *cache;
  int64_t c_bs, c_ps;  // bytes
  void *out;
  int64_t o_bs, o_rs;  // elements
  const int32_t *seqlens;
  int32_t batch, bias, max_seqlen, q_len, causal;
  int32_t q_heads, kv_heads, group, tiles;  // tiles: row tiles of one (sequence, KV head)
  int32_t part, max_parts;
  int32_t members; // of a group: workgroups that run on one XCD, each for a row tile and a KV head
  int64_t groups;
  int64_t rows;    // (sequence, position, query head)
  int32_t waves;   // of a workgroup, every one of them each `waves`-th step of its partition
  const void *kv_new;
  float scale_log2;
  float *ws_o, *ws_ml;
  unsigned int *status;
  bool q_vec;
};

// Terms whose sum is an element of T (query), and that hold a probability.
template <typename T>
struct MxTerms;
template <>
struct MxTerms<__bf16> { static constexpr int kQ = 1, kP = 2; };
template <>
struct MxTerms<_Float16> { static constexpr int kQ = 2, kP = 2; };
template <>
struct MxTerms<float> { static constexpr int kQ = 3, kP = 3; };

__device__ __forceinline__ f32x4 mx_mma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The bf16 terms of (x0, x1), each the truncated rest of those before: 8 bits
// of the significand a term, and never past the largest bf16.
template <int N>
__device__ __forceinline__ void mx_split(float x0, float x1, unsigned int *terms) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const unsigned int u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
    terms[n] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);  // the upper halves
    if (n + 1 < N) {
      const float r0 = x0 - __uint_as_float(u0 & 0xffff0000u), r1 = x1 - __uint_as_float(u1 & 0xffff0000u);
      x0 = r0 == r0 ? r0 : 0.f;  // an infinity is its first term alone
      x1 = r1 == r1 ? r1 : 0.f;
    }
  }
}

// The same of two probabilities (at most 2^kMxaSlack), each term the rounded
// rest of those before: N terms are off by 2^-8N of the probability at most.
template <int N>
__device__ __forceinline__ void mx_split_rounded(float x0, float x1, unsigned int *terms) {
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int n = 0; n < N; ++n) {
    terms[n] = __builtin_bit_cast(unsigned int, v2{static_cast<__bf16>(x0), static_cast<__bf16>(x1)});
    x0 -= __uint_as_float(terms[n] << 16);
    x1 -= __uint_as_float(terms[n] & 0xffff0000u);
  }
}

// Orders this wave's LDS writes before its later reads of other lanes' data.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A wave's LDS: V of a step (at the end its output), the new row, sums and maxima.
template <int D>
struct MxLds {
  static constexpr int VP = 2 * D + 32;  // bytes per V row: a transposed read's four rows over all banks
  static constexpr int NEW = 2 * (D / 8) + 2 * (D / 32);
  static constexpr int kNew = kMxaKeys * VP, kMl = kNew + NEW * 4, kWave = (kMl + kMxaRows * 8 + 15) / 16 * 16;
  static_assert(kNew >= D * kMxaRows * 4 && kMl % 8 == 0);
};

template <int D>
struct MxTile {
  static constexpr int NW = D / 32, NB = D < 128 ? 1 : D / 128;
  unsigned int k[2][NW], v[2][NW];
  unsigned char kp[2][NB], vp[2][NB];
};

template <int NW>
__device__ __forceinline__ void mx_read_words(const unsigned char *p, unsigned int *w) {
  if constexpr (NW >= 4) {
#pragma unroll
    for (int i = 0; i < NW; i += 4) {
      const u32x4 v = *reinterpret_cast<const u32x4 *>(p + 4 * i);
      w[i] = v[0], w[i + 1] = v[1], w[i + 2] = v[2], w[i + 3] = v[3];
    }
  } else if constexpr (NW == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const unsigned int *>(p);
  }
}

template <typename T, int D>
__global__ __launch_bounds__(64 * kMxaMaxWaves, 2) void mx_attend_kernel(const MxAttendArgs a) {
  constexpr int NQ = MxTerms<T>::kQ, NP = MxTerms<T>::kP;
  constexpr int NW = MxTile<D>::NW;  // words of elements a lane holds of a key, = products of a score
  constexpr int NB = MxTile<D>::NB;  // blocks they lie in
  constexpr int ND = D / 16;         // output tiles
  constexpr int VP = MxLds<D>::VP;
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  char *s_v = lds + wave * MxLds<D>::kWave;
  unsigned int *s_new = reinterpret_cast<unsigned int *>(s_v + MxLds<D>::kNew);

  // Workgroups that differ by a multiple of the XCDs run on one XCD: they take
  // the heads and row tiles of one (sequence, partition), which share its lines.
  // These count sequences first, and a sequence's partitions go to one XCD after
  // the other, so that neither empty partitions nor one long sequence leave XCDs
  // idle.
  const unsigned slot = blockIdx.x / kXcds, eight = slot / static_cast<unsigned>(a.members) * kXcds;
  unsigned rest = eight + (blockIdx.x + eight / static_cast<unsigned>(a.batch)) % kXcds;
  if (rest >= a.groups) return;
  const int64_t b = rest % static_cast<unsigned>(a.batch);
  rest /= static_cast<unsigned>(a.batch);
  const int part = static_cast<int>(rest % static_cast<unsigned>(a.max_parts));
  rest = rest / static_cast<unsigned>(a.max_parts) * a.members + slot % static_cast<unsigned>(a.members);
  const int tile = static_cast<int>(rest / static_cast<unsigned>(a.kv_heads));
  const int h = static_cast<int>(rest % static_cast<unsigned>(a.kv_heads));

  // Lengths: `base` keys as asked for, no more than max_seqlen of them.
  int64_t want = static_cast<int64_t>(a.bias) + (a.kv_new ? 1 : 0);
  if (a.seqlens) want += a.seqlens[b];
  const int len = static_cast<int>(want < 0 ? 0 : want > a.max_seqlen ? a.max_seqlen : want);
  if (want > a.max_seqlen && threadIdx.x == 0 && h == 0 && tile == 0 && part == 0)
    raise_status(a.status, HEXKV_STATUS_LENGTH_CLAMPED);
  const int fresh = a.kv_new && want > 0 && want <= a.max_seqlen ? len - 1 : -1;  // the new row's position
  const int nparts = len > 0 ? (len + a.part - 1) / a.part : 1;
  if (part >= nparts) return;
  const int p0 = part * a.part, p1 = min(len, p0 + a.part);

  // This lane's query row, and the tile's first and last.
  const int rows = a.q_len * a.group;
  const int row = tile * kMxaRows + c;
  const bool live = row < rows;
  const int own = min(row, rows - 1), t = own / a.group, qh = h * a.group + own - t * a.group;
  const auto keys_of = [&](int tt) {
    const int64_t n = a.causal ? want - a.q_len + tt + 1 : want;
    return static_cast<int>(n < 0 ? 0 : n > a.max_seqlen ? a.max_seqlen : n);
  };
  const int lim = keys_of(t);
  const int first_lim = keys_of(tile * kMxaRows / a.group);
  const int end = min(p1, keys_of((min(rows, (tile + 1) * kMxaRows) - 1) / a.group));

  const unsigned char *seq = a.cache + b * a.c_bs + static_cast<int64_t>(p0) * a.c_ps;
  // Loaded, a lane holds quarter lane % 4 of key lane / 4: four lanes read one
  // key's row, so that a load touches 16 lines and not 64.
  const int kr = lane >> 2, kq = lane & 3;
  const int blk = NB > 1 ? kq * NB : kq * D / 128;  // its first block within a head
  const unsigned char *k_base = seq + h * (D / 2);
  const unsigned char *v_base = k_base + static_cast<int64_t>(a.kv_heads) * (D / 2);
  const unsigned char *kp_base = seq + static_cast<int64_t>(a.kv_heads) * D + h * (D / 32);
  const unsigned char *vp_base = kp_base + a.kv_heads * (D / 32);
  const unsigned int pitch = static_cast<unsigned int>(a.c_ps);

  // The new row: converted once by the wave whose step has it, written to the
  // cache, and put in place of what that step has loaded for its position.
  const bool holds_new = fresh >= p0 && fresh < p1 && (fresh - p0) / kMxaKeys % a.waves == wave;
  if (holds_new) {
    const int half = lane / (D / 8), at = lane % (D / 8);
    if (half < 2) {
      float f[8];
      mx_read8(static_cast<const T *>(a.kv_new) + ((b * 2 + half) * a.kv_heads + h) * D + at * 8, true, f);
      const unsigned int byte = mx_power(mx_block_bits(mx_bits(f))), w = mx_encode(f, byte);
      unsigned char *dst = a.cache + b * a.c_bs + static_cast<int64_t>(fresh) * a.c_ps;
      const int64_t head = static_cast<int64_t>(half) * a.kv_heads + h;
      *reinterpret_cast<unsigned int *>(dst + head * (D / 2) + at * 4) = w;
      s_new[half * (D / 8) + at] = w;
      if (at % 4 == 0) {
        dst[static_cast<int64_t>(a.kv_heads) * D + head * (D / 32) + at / 4] = static_cast<unsigned char>(byte);
        s_new[2 * (D / 8) + half * (D / 32) + at / 4] = byte;
      }
    }
    wave_lds_fence();
  }

  // (Lanes behind the last row repeat it; they are not stored.)
  u32x4 q[NQ][NW];
  {
    const T *p = static_cast<const T *>(a.q) + b * a.q_bs + t * a.q_rs + static_cast<int64_t>(qh) * D + g * (D / 4);
    float f[NW][8];
    if (a.q_vec) {
#pragma unroll
      for (int j = 0; j < NW; ++j) mx_read8(p + 8 * j, true, f[j]);
    } else {
#pragma unroll
      for (int j = 0; j < NW; ++j) mx_read8(p + 8 * j, false, f[j]);
    }
#pragma unroll
    for (int j = 0; j < NW; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned int terms[NQ];
        mx_split<NQ>(f[j][2 * i], f[j][2 * i + 1], terms);
#pragma unroll
        for (int n = 0; n < NQ; ++n) q[n][j][i] = terms[n];
      }
  }

  float m = kMxaLowest, l = 0.f;
  f32x4 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x4{};
  unsigned int nan_blocks = 0;

  const auto fetch = [&](int k0, MxTile<D> &x) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const unsigned int at = static_cast<unsigned int>(min(k0 + s * 16 + kr, end - 1) - p0) * pitch;
      mx_read_words<NW>(k_base + (at + kq * (D / 8)), x.k[s]);
      mx_read_words<NW>(v_base + (at + kq * (D / 8)), x.v[s]);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        x.kp[s][n] = kp_base[at + blk + n];
        x.vp[s][n] = vp_base[at + blk + n];
      }
    }
  };

  const auto compute = [&](int k0, MxTile<D> &x) {
    const bool whole = k0 + kMxaKeys <= end;
    if (holds_new && fresh >= k0 && fresh < k0 + kMxaKeys) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (k0 + s * 16 + kr == fresh) {
#pragma unroll
          for (int i = 0; i < NW; ++i) {
            x.k[s][i] = s_new[kq * NW + i];
            x.v[s][i] = s_new[D / 8 + kq * NW + i];
          }
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            x.kp[s][n] = static_cast<unsigned char>(s_new[2 * (D / 8) + blk + n]);
            x.vp[s][n] = static_cast<unsigned char>(s_new[2 * (D / 8) + D / 32 + blk + n]);
          }
        }
    }
    if (!whole) {  // keys past the end repeat the last one: their values are zero, their scores masked
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (k0 + s * 16 + kr >= end) {
#pragma unroll
          for (int i = 0; i < NW; ++i) x.v[s][i] = 0;
#pragma unroll
          for (int n = 0; n < NB; ++n) x.vp[s][n] = 127;
        }
    }
    bool bad = false;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < NB; ++n) bad |= x.vp[s][n] >= kMxLastPower;
    if (__ballot(bad)) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        unsigned int bits = 0;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          bool past = false;
#pragma unroll
          for (int i = 0; i < NW / NB; ++i) past |= mx_past(x.v[s][n * (NW / NB) + i], x.vp[s][n]);
          if (past) {
            bits |= 1u << (blk + n);
            x.vp[s][n] = 127;
#pragma unroll
            for (int i = 0; i < NW / NB; ++i) x.v[s][n * (NW / NB) + i] = 0;
          }
        }
        uint64_t from = __ballot(bits != 0);
        while (from) {
          const int r = __builtin_ctzll(from);
          from &= from - 1;
          const unsigned int theirs = __shfl(bits, r);
          if (k0 + s * 16 + (r >> 2) < lim) nan_blocks |= theirs;
        }
      }
    }

    // V into LDS, as the transposed reads want it
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NW; ++i)
        *reinterpret_cast<u32x4 *>(&s_v[(s * 16 + kr) * VP + kq * (D / 2) + i * 16]) =
            mx_bf16(x.v[s][i], mx_scale(x.vp[s][i * NB / NW]));

    f32x4 sc[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      sc[s] = f32x4{};
      unsigned int kp[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) kp[n] = __builtin_amdgcn_ds_bpermute(16 * c + 4 * g, x.kp[s][n]);
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        const unsigned int kw = __builtin_amdgcn_ds_bpermute(16 * c + 4 * g, x.k[s][j]);
        const u32x4 k = mx_bf16(kw, mx_scale(kp[j * NB / NW]));
#pragma unroll
        for (int n = 0; n < NQ; ++n) sc[s] = mx_mma(k, q[n][j], sc[s]);
      }
    }
    float top = -INFINITY;
    if (__builtin_expect(!(k0 + kMxaKeys <= first_lim && whole), 0)) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (k0 + s * 16 + 4 * g + i >= min(lim, end)) sc[s][i] = -INFINITY;
      asm volatile("");  // a branch, not eight selections in every step
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        top = fmaxf(top, sc[s][i]);
      }
    top = max_from<16>(top) * a.scale_log2;
    if (__ballot(top > m + kMxaSlack)) {
      const float moved = top > m + kMxaSlack ? top : m;
      const float by = __builtin_amdgcn_exp2f(m - moved);
      m = moved;
      l *= by;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] *= by;
    }
    u32x4 p[NP];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[s][i], a.scale_log2, -m));
        const float e1 = __builtin_amdgcn_exp2f(fmaf(sc[s][i + 1], a.scale_log2, -m));
        l += e0 + e1;
        unsigned int terms[NP];
        mx_split_rounded<NP>(e0, e1, terms);
#pragma unroll
        for (int n = 0; n < NP; ++n) p[n][s * 2 + i / 2] = terms[n];
      }
    wave_lds_fence();
    const auto *shared = (const __attribute__((address_space(3))) char *)&s_v[0];
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const int at = (4 * g + c / 4) * VP + (c % 4) * 8 + d * 32;
      const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(shared + at));
      const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(shared + at + 16 * VP));
      const u32x4 v = __builtin_bit_cast(u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int n = 0; n < NP; ++n) acc[d] = mx_mma(v, p[n], acc[d]);
    }
    wave_lds_fence();
  };

  const int first = p0 + wave * kMxaKeys, stride = a.waves * kMxaKeys;
  if (end > first) {
    // The next step is always loaded (past the end the last key again): were it
    // conditional, a step would wait for the next one's loads as well.
    MxTile<D> now, next;
    fetch(first, now);
    for (int k0 = first;; k0 += 2 * stride) {
      fetch(k0 + stride, next);
      compute(k0, now);
      if (k0 + stride >= end) break;
      fetch(k0 + 2 * stride, now);
      compute(k0 + stride, next);
      if (k0 + 2 * stride >= end) break;
    }
  }

  l = sum_from<16>(l);
  nan_blocks |= __shfl_xor(nan_blocks, 16);
  nan_blocks |= __shfl_xor(nan_blocks, 32);
#pragma unroll
  for (int d = 0; d < ND; ++d)
    if (nan_blocks >> (d / 2) & 1) acc[d] = f32x4{} + NAN;

  // The waves' sums meet in LDS, each wave's in its own V region, and wave w
  // joins the output tiles w, w + waves, ...
  f32x4 *s_acc = reinterpret_cast<f32x4 *>(s_v);
#pragma unroll
  for (int d = 0; d < ND; ++d) s_acc[d * 64 + lane] = acc[d];
  float2 *s_ml = reinterpret_cast<float2 *>(s_v + MxLds<D>::kMl);
  if (g == 0) s_ml[c] = float2{m, l};
  __syncthreads();
  float2 ml[kMxaMaxWaves];
  m = kMxaLowest;
#pragma unroll
  for (int w = 0; w < kMxaMaxWaves; ++w)
    if (w < a.waves) {
      ml[w] = reinterpret_cast<const float2 *>(lds + w * MxLds<D>::kWave + MxLds<D>::kMl)[c];
      m = fmaxf(m, ml[w].x);
    }
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kMxaMaxWaves; ++w)
    if (w < a.waves) {
      ml[w].x = __builtin_amdgcn_exp2f(ml[w].x - m);
      l = fmaf(ml[w].x, ml[w].y, l);
    }
  if (!live) return;
  const int64_t out_slot = ((b * a.q_len + t) * a.q_heads + qh) * a.max_parts + part;
  const float inv = 1.f / l;
  for (int d = wave; d < ND; d += a.waves) {
    f32x4 sum = {};
#pragma unroll
    for (int w = 0; w < kMxaMaxWaves; ++w)
      if (w < a.waves) {
        const f32x4 v = reinterpret_cast<const f32x4 *>(lds + w * MxLds<D>::kWave)[d * 64 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = fmaf(ml[w].x, v[i], sum[i]);
      }
    if (nparts == 1) {
      // A row without keys is zero; one whose scores are all minus infinity has
      // no softmax (0 / 0).
      T *out = static_cast<T *>(a.out) + b * a.o_bs + t * a.o_rs + static_cast<int64_t>(qh) * D + 4 * g;
      store4(out + d * 16, lim > 0 ? sum * inv : f32x4{});
    } else {
      *reinterpret_cast<f32x4 *>(a.ws_o + out_slot * D + 4 * g + d * 16) = sum;
    }
  }
  if (nparts > 1 && threadIdx.x < kMxaRows) *reinterpret_cast<float2 *>(a.ws_ml + out_slot * 2) = float2{m, l};
}

// Joins a row's partitions, W waves of a workgroup per (sequence, position,
// query head), every one of them each W-th partition, eight loaded at a time.
constexpr int kJoinWaves = 8;

template <typename T, int D, int W>
__global__ __launch_bounds__(64 * kJoinWaves) void mx_join_kernel(const MxAttendArgs a) {
  constexpr int E = D < 64 ? 1 : D / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (kJoinWaves / W) + wave / W;
  if (r >= a.rows) return;  // (W == kJoinWaves: never)
  const unsigned qh = static_cast<unsigned>(r) % static_cast<unsigned>(a.q_heads);
  const unsigned bt = static_cast<unsigned>(r) / static_cast<unsigned>(a.q_heads);
  const int t = static_cast<int>(bt % static_cast<unsigned>(a.q_len));
  const int64_t b = bt / static_cast<unsigned>(a.q_len);
  int64_t want = static_cast<int64_t>(a.bias) + (a.kv_new ? 1 : 0);
  if (a.seqlens) want += a.seqlens[b];
  const int len = static_cast<int>(want < 0 ? 0 : want > a.max_seqlen ? a.max_seqlen : want);
  const int nparts = len > 0 ? (len + a.part - 1) / a.part : 1;
  if (nparts == 1) return;  // written by the attention kernel
  const bool empty = a.causal && want - a.q_len + t + 1 <= 0;
  const float *ml = a.ws_ml + r * a.max_parts * 2, *o = a.ws_o + r * a.max_parts * D + lane % (D / E) * E;
  float m = kMxaLowest, l = 0.f, sum[E] = {};
  constexpr int U = 8;
  for (int p0 = wave % W; p0 < nparts; p0 += W * U) {
    float v[U][E];
    float2 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (past the end the last one, with weight 0)
      const int p = min(p0 + u * W, nparts - 1);
#pragma unroll
      for (int e = 0; e < E; ++e) v[u][e] = o[static_cast<int64_t>(p) * D + e];
      w[u] = *reinterpret_cast<const float2 *>(ml + 2 * p);
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, w[u].x);
    const float by = __builtin_amdgcn_exp2f(m - top);
    m = top;
    l *= by;
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] *= by;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p0 + u * W >= nparts) break;
      const float f = __builtin_amdgcn_exp2f(w[u].x - m);
      l = fmaf(f, w[u].y, l);
#pragma unroll
      for (int e = 0; e < E; ++e) sum[e] = fmaf(f, v[u][e], sum[e]);
    }
  }
  if constexpr (W > 1) {
    __shared__ float s_sum[W][64 * E], s_l[W], s_m[W];
#pragma unroll
    for (int e = 0; e < E; ++e) s_sum[wave][lane * E + e] = sum[e];
    if (lane == 0) s_l[wave] = l, s_m[wave] = m;
    __syncthreads();
    if (wave > 0) return;
    m = kMxaLowest;
#pragma unroll
    for (int i = 0; i < W; ++i) m = fmaxf(m, s_m[i]);
    l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float f = __builtin_amdgcn_exp2f(s_m[i] - m);
      l = fmaf(f, s_l[i], l);
#pragma unroll
      for (int e = 0; e < E; ++e) sum[e] = fmaf(f, s_sum[i][lane * E + e], sum[e]);
    }
  }
  if (lane * E >= D) return;
  T *out = static_cast<T *>(a.out) + b * a.o_bs + t * a.o_rs + static_cast<int64_t>(qh) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = Elem<T>::from_float(empty ? 0.f : sum[e] / l);
}

static int elem_bytes(int dtype) { return dtype == HEXKV_F32 ? 4 : 2; }

static int mx_validate(const hexkv_mx_attend_params *p, const char *what) {
  if (!p) return fail(HEXKV_EINVAL, "%s: null params", what);
  if (p->dtype != HEXKV_F16 && p->dtype != HEXKV_BF16 && p->dtype != HEXKV_F32)
    return fail(HEXKV_EINVAL, "%s: unknown dtype %d", what, p->dtype);
  if (p->batch < 0 || p->q_len < 1 || p->q_heads < 1 || p->kv_heads < 1)
    return fail(HEXKV_EINVAL, "%s: bad batch/q_len/heads", what);
  if (p->q_heads % p->kv_heads)
    return fail(HEXKV_EINVAL, "%s: q_heads %d not a multiple of kv_heads %d", what, p->q_heads, p->kv_heads);
  if (p->q_heads > 65536) return fail(HEXKV_EINVAL, "%s: over 65536 heads", what);
  if (p->head_dim != 32 && p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
    return fail(HEXKV_EUNSUPPORTED, "%s: head_dim %d (compiled: 32, 64, 128, 256)", what, p->head_dim);
  if (p->kv_new && p->q_len != 1) return fail(HEXKV_EINVAL, "%s: fused append needs q_len 1", what);
  if (p->max_seqlen > INT32_MAX - (1 << 17))  // (steps are counted past the end, in 32 bits)
    return fail(HEXKV_ERANGE, "%s: max_seqlen %d too long", what, p->max_seqlen);
  if (p->max_seqlen < 0 || p->max_seqlen > p->capacity)
    return fail(HEXKV_ERANGE, "%s: max_seqlen %d outside [0, capacity %lld]", what, p->max_seqlen,
                static_cast<long long>(p->capacity));
  if (p->partition < 0 || p->partition % kMxaKeys || p->partition > 65536)
    return fail(HEXKV_EINVAL, "%s: partition must be 0 or a multiple of %d up to 65536", what, kMxaKeys);
  if (!(p->softmax_scale > 0.f) || p->softmax_scale > 3.0e38f)
    return fail(HEXKV_EINVAL, "%s: softmax_scale must be positive and finite", what);
  if (static_cast<int64_t>(p->q_len) * (p->q_heads / p->kv_heads) >= INT64_C(1) << 30 ||
      static_cast<int64_t>(p->batch) * p->q_len * p->q_heads >= INT64_C(1) << 31)
    return fail(HEXKV_ERANGE, "%s: 2^31 query rows or more", what);
  if (p->cache_row_bytes < mx_row_bytes(p->kv_heads, p->head_dim) || p->cache_row_bytes % 16 ||
      p->cache_batch_bytes % 16 || p->cache_row_bytes > (INT64_C(1) << 24) ||
      (p->batch > 1 && p->cache_batch_bytes < p->capacity * p->cache_row_bytes))
    return fail(HEXKV_EINVAL, "%s: cache rows must be multiples of 16 bytes, at least %lld apart (at most 2^24), and "
                              "sequences capacity rows apart", what,
                static_cast<long long>(mx_row_bytes(p->kv_heads, p->head_dim)));
  return HEXKV_OK;
}

static int64_t row_tiles(const hexkv_mx_attend_params *p) {
  return (static_cast<int64_t>(p->q_len) * (p->q_heads / p->kv_heads) + kMxaRows - 1) / kMxaRows;
}

static int64_t mx_units(const hexkv_mx_attend_params *p) {
  return static_cast<int64_t>(p->batch) * p->kv_heads * row_tiles(p);
}

// Positions per partition.  One partition where the join would cost more than
// it saves: to 1024 keys; where there is a unit for each of the 256 CUs to 2560;
// and for more than kFewTiles row tiles there whatever the length (their rows'
// lengths differ little).  Beyond, two workgroups a CU, of 256 to 1024 keys
// each (the upper end for ragged lengths).  us, one partition / 256 / 512 /
// 1024 keys each, bf16, head_dim 128, 32 query heads:
//   8 KV heads, B 1 of 1024     11.3 /  9.8 / 10.7 /  -     of 2048  14.4 / 11.2 / 11.1 / 14
//               B 1 of 8192     38.2 / 11.8 / 12.4 / 18.9
//               B 32 of 1024    13.0 / 21.2 / 17   /  -     of 2048  24.2 / 39   / 30   / 27.8
//               B 64 of 128..8192  86 / 99 / 83.2 / 80.7
//   (one / 1024 keys each)
//               B 32 of 2304  25.7 / 29.4, of 2816  29.7 / 34.4, of 4096  41 / 44
//               B 32 of n / 32..n, n 2560  23.9 / 24.0, 3000  24.6 / 28.2, 4096  33.6 / 31.9
//               B 64 of n / 32..n, n 2560  36.6 / 37.1, 3000  45.8 / 45.9, 4096  63.4 / 59.7
//   32 KV heads, B 8 of 256..2048 (fp16)  17.8 / 38 / 23 / 19.9
//   400 rows, B 2 of 4096, 8 heads on 1 (fp16)  45 / - / - / 51;  1600 rows, 32 on 8  385 / - / - / 571;
//   60 rows, B 16 of 1..8192, 8 on 1  71 / - / - / 62
constexpr int64_t kCus = 256, kFewTiles = 24;
static int mx_partition(const hexkv_mx_attend_params *p) {
  const int64_t units = std::max<int64_t>(1, mx_units(p)), n = std::max<int64_t>(1, p->max_seqlen);
  int64_t part = p->partition;
  if (!part && (n <= (units >= kCus ? 2560 : 1024) || (units >= kCus && row_tiles(p) > kFewTiles))) part = n;
  if (!part) {
    const int64_t parts = std::max<int64_t>(1, 2 * kCus / units);
    part = std::min<int64_t>(1024, std::max<int64_t>(256, n / parts / 128 * 128));
  }
  part = std::min<int64_t>((part + kMxaKeys - 1) / kMxaKeys * kMxaKeys, 65536);
  // a partition's rows are addressed with 32-bit offsets
  while (part > kMxaKeys && part * p->cache_row_bytes >= INT64_C(1) << 31) part = part / 2 / kMxaKeys * kMxaKeys;
  return static_cast<int>(part);
}

static int64_t mx_parts(const hexkv_mx_attend_params *p, int part) {
  return std::max<int64_t>(1, (static_cast<int64_t>(p->max_seqlen) + part - 1) / part);
}

static size_t mx_join_bytes(const hexkv_mx_attend_params *p) {
  const int64_t parts = mx_parts(p, mx_partition(p));
  if (parts == 1) return 0;
  return static_cast<size_t>(p->batch) * p->q_len * p->q_heads * parts * (p->head_dim + 2) * sizeof(float);
}

// Many bf16 query rows (a prompt's chunk): the rows' keys and values are taken
// out of the cache once, exactly, and attended by hexkv_attend's query tiles,
// where those are compiled.  To kFewTiles row tiles the keys are read in four
// bits (four bits / taken out, us, 4 query heads a KV head: 2 x 2048 keys, 5 tiles
// 16 / 28, 24 tiles 29 / 45; 16 x 2048 keys, 5 tiles 42 / 82, 24 tiles 120 / 129).
// fp16 queries always read them in four bits: fp16 holds neither a power
// above 2^13 (an fp16 value from 57344 up is stored as 2^16) nor all below
// 2^-23, so rows taken out as fp16 would not be the stored ones.  What that
// costs (four bits / taken out, 2 x 4096 keys, 32 heads on 8 of 128): 400 rows
// 133 / 134, 800 228 / 170, 1600 385 / 263; on 4 of 64: 84 / 101, 142 / 113, 240 / 160.
static bool mx_unpacks(const hexkv_mx_attend_params *p) {
  return p->dtype == HEXKV_BF16 && (p->head_dim == 64 || p->head_dim == 128) && p->q_len > 1 && p->partition == 0 &&
         row_tiles(p) > kFewTiles && static_cast<int64_t>(p->batch) * p->q_len <= 65535 && p->max_seqlen > 0 &&
         aligned16(p->q) && p->q_batch_stride % 8 == 0 && p->q_row_stride % 8 == 0 &&
         static_cast<int64_t>(p->max_seqlen) * 2 * p->kv_heads * p->head_dim * 2 < INT64_C(0xffff0000);
}

static hexkv_attend_params mx_unpacked(const hexkv_mx_attend_params *p, void *kv) {
  const int64_t row = static_cast<int64_t>(p->kv_heads) * p->head_dim;
  hexkv_attend_params t = {};
  t.dtype = p->dtype;
  t.batch = p->batch;
  t.q_len = p->q_len;
  t.q_heads = p->q_heads;
  t.kv_heads = p->kv_heads;
  t.head_dim = p->head_dim;
  t.causal = p->causal;
  t.softmax_scale = p->softmax_scale;
  t.q = p->q;
  t.q_batch_stride = p->q_batch_stride;
  t.q_row_stride = p->q_row_stride;
  t.cache = kv;
  t.cache_batch_stride = 2 * row * p->max_seqlen;
  t.cache_pos_stride = 2 * row;
  t.cache_kv_stride = row;
  t.capacity = p->max_seqlen;
  t.out = p->out;
  t.out_batch_stride = p->out_batch_stride;
  t.out_row_stride = p->out_row_stride;
  t.seqlens_dev = p->seqlens_dev;
  t.seqlen_bias = p->seqlen_bias;
  t.max_seqlen = p->max_seqlen;
  return t;
}

static size_t mx_unpacked_bytes(const hexkv_mx_attend_params *p) {
  const size_t n = static_cast<size_t>(p->batch) * p->max_seqlen * 2 * p->kv_heads * p->head_dim * 2;
  return (n + 255) / 256 * 256;
}

static size_t mx_workspace(const hexkv_mx_attend_params *p) {
  if (!mx_unpacks(p)) return mx_join_bytes(p);
  const hexkv_attend_params t = mx_unpacked(p, nullptr);
  return mx_unpacked_bytes(p) + hexkv_attend_workspace_bytes(&t);
}

// To kJoinAlone partitions a wave joins a row by itself: 17 of them 28 us
// instead of 20 in a call of 4 sequences, two 22.4 instead of 24.5 in one of 64.
constexpr int kJoinAlone = 16;
static int64_t mx_slots(const MxAttendArgs &a) { return (a.groups + kXcds - 1) / kXcds * kXcds * a.members; }
static int64_t mx_join_groups(const MxAttendArgs &a) {
  return a.max_parts > kJoinAlone ? a.rows : a.max_parts > 1 ? (a.rows + kJoinWaves - 1) / kJoinWaves : 0;
}

template <typename T, int D>
static void mx_launch(const MxAttendArgs &a, hipStream_t s) {
  mx_attend_kernel<T, D><<<static_cast<unsigned>(mx_slots(a)), 64 * a.waves, a.waves * MxLds<D>::kWave, s>>>(a);
  const unsigned join = static_cast<unsigned>(mx_join_groups(a));
  if (a.max_parts > kJoinAlone) mx_join_kernel<T, D, kJoinWaves><<<join, 64 * kJoinWaves, 0, s>>>(a);
  else if (join) mx_join_kernel<T, D, 1><<<join, 64 * kJoinWaves, 0, s>>>(a);
}

template <typename T>
static void mx_launch_dim(const MxAttendArgs &a, int head_dim, hipStream_t s) {
  switch (head_dim) {
    case 32: return mx_launch<T, 32>(a, s);
    case 64: return mx_launch<T, 64>(a, s);
    case 128: return mx_launch<T, 128>(a, s);
    default: return mx_launch<T, 256>(a, s);
  }
}

}  // namespace hexkv

extern "C" size_t hexkv_mx_attend_workspace_bytes(const hexkv_mx_attend_params *p) {
  using namespace hexkv;
  clear_error();
  return mx_validate(p, "hexkv_mx_attend_workspace_bytes") == HEXKV_OK && p->batch ? mx_workspace(p) : 0;
}

extern "C" int hexkv_mx_attend(const hexkv_mx_attend_params *p, void *workspace, size_t workspace_bytes,
                               hexkv_stream_t stream) {
  using namespace hexkv;
  const char *what = "hexkv_mx_attend";
  clear_error();
  int rc = mx_validate(p, what);
  if (rc != HEXKV_OK) return rc;
  if (p->batch == 0) return HEXKV_OK;
  if (!p->q || !p->cache || !p->out) return fail(HEXKV_EINVAL, "%s: null tensor", what);
  const int elem = elem_bytes(p->dtype);
  if (!aligned16(p->cache) || (p->kv_new && !aligned16(p->kv_new)))
    return fail(HEXKV_EINVAL, "%s: cache/kv_new must be 16-byte aligned", what);
  if ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out)) & (elem - 1))
    return fail(HEXKV_EINVAL, "%s: q/out misaligned", what);
  const size_t need = mx_workspace(p);
  if (need && (!workspace || workspace_bytes < need))
    return fail(HEXKV_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : 0, need);
  if (need && !aligned16(workspace)) return fail(HEXKV_EINVAL, "%s: workspace must be 16-byte aligned", what);

  if (mx_unpacks(p)) {
    const int64_t row = static_cast<int64_t>(p->kv_heads) * p->head_dim;
    rc = hexkv_mx_load(p->cache, p->cache_batch_bytes, p->cache_row_bytes, p->capacity, workspace,
                       2 * row * p->max_seqlen, 2 * row, row, p->batch, p->max_seqlen, p->kv_heads, p->head_dim, p->dtype,
                       nullptr, 0, stream);
    if (rc != HEXKV_OK) return rc;
    const hexkv_attend_params t = mx_unpacked(p, workspace);
    const size_t kv = mx_unpacked_bytes(p);
    return hexkv_attend(&t, static_cast<char *>(workspace) + kv, workspace_bytes - kv, stream);
  }

  MxAttendArgs a = {};
  a.q = p->q;
  a.q_bs = p->q_batch_stride;
  a.q_rs = p->q_row_stride;
  a.cache = static_cast<unsigned char *>(p->cache);
  a.c_bs = p->cache_batch_bytes;
  a.c_ps = p->cache_row_bytes;
  a.out = p->out;
  a.o_bs = p->out_batch_stride;
  a.o_rs = p->out_row_stride;
  a.seqlens = p->seqlens_dev;
  a.batch = static_cast<int32_t>(p->batch);
  a.bias = p->seqlen_bias;
  a.max_seqlen = p->max_seqlen;
  a.q_len = p->q_len;
  a.causal = p->causal && p->q_len > 1;
  a.q_heads = p->q_heads;
  a.kv_heads = p->kv_heads;
  a.group = p->q_heads / p->kv_heads;
  a.tiles = static_cast<int32_t>(row_tiles(p));
  a.part = mx_partition(p);
  a.max_parts = static_cast<int32_t>(mx_parts(p, a.part));
  const int64_t workgroups = mx_units(p) * a.max_parts;
  if (workgroups >= INT64_C(1) << 24)
    return fail(HEXKV_ERANGE, "%s: 2^24 workgroups or more; split the call", what);
  // (a call too small to give every XCD a group parts its tiles, then its heads)
  const int64_t pairs = static_cast<int64_t>(p->batch) * a.max_parts;
  a.members = pairs >= kXcds ? a.tiles * p->kv_heads : pairs * a.tiles >= kXcds ? p->kv_heads : 1;
  a.groups = workgroups / a.members;
  // Eight waves share a partition while there is no second workgroup for a CU
  // (8 / 4 waves: 577 keys of 4 KV heads 6.6 / 7.5 us, 17.8 / 19.4 for the 8 x
  // 32 heads above), four else (B 64 of 1024 keys, 32 KV heads: 86.6 / 85.7).
  a.waves = workgroups <= kCus ? kMxaMaxWaves : kMxaMaxWaves / 2;
  a.rows = static_cast<int64_t>(p->batch) * p->q_len * p->q_heads;
  if (mx_slots(a) * 64 * a.waves >= INT64_C(1) << 32 || mx_join_groups(a) * 64 * kJoinWaves >= INT64_C(1) << 32)
    return fail(HEXKV_ERANGE, "%s: 2^32 lanes or more in a launch; split the call", what);
  a.kv_new = p->kv_new;
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  if (a.max_parts > 1) {
    a.ws_o = static_cast<float *>(workspace);
    a.ws_ml = a.ws_o + a.rows * a.max_parts * p->head_dim;
  }
  const int vec = 16 / elem;
  a.q_vec = aligned16(p->q) && p->q_batch_stride % vec == 0 && p->q_row_stride % vec == 0;
  rc = status_word(stream, &a.status, what);
  if (rc != HEXKV_OK) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == HEXKV_BF16) mx_launch_dim<__bf16>(a, p->head_dim, s);
  else if (p->dtype == HEXKV_F16) mx_launch_dim<_Float16>(a, p->head_dim, s);
  else mx_launch_dim<float>(a, p->head_dim, s);
  return check_launch(what);
}
