// Attention over a paged cache: hexkv_paged_attend.
//
// A row is one query head of one new token; the rows of a sequence that share
// a KV head (tokens x group of them, in (token, head) order) read the same keys.
//
// Row kernel: 16 rows a workgroup, its waves taking steps of the keys in turn.
//   S^T = K Q^T    16 keys x 16 rows a matrix instruction; K's operand is
//                  loaded as it lies: lane (r, g) holds key r, dims of chunk g
//   softmax        a lane's scores are all its own row's; the other 3 lanes
//                  of a row are two exchanges away
//   O^T += V^T P^T the scores' layout is P's operand as it stands, with the contraction
//                  index of a step being key 4 g + i (16-bit: then 16 + 4 g + i);
//                  16-bit V goes through the wave's own LDS, row-major in and
//                  transposed out, fp32 V is loaded in place
// What bounds it: a decode row's K and V are read once, 4 D flops a key, so
// memory.  Steps are loaded one ahead into registers, page numbers two ahead.
#include "hexkv_paged.h"

#include <algorithm>
#include <type_traits>

namespace hexkv {

typedef short h4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) h4 lds_h4;

struct PagedAttendArgs {
  PageTables p;
  const void *q, *pages;
  void *out;
  int64_t q_stride, o_stride;
  int32_t q_heads, kv_heads, group, causal;
  int32_t max_tokens, max_seqlen;
  float scale_log2;
  int32_t row_tiles;        // 16-row tiles of a sequence and KV head
  int32_t part, max_parts;  // rows per partition, partitions of the longest row
  float *ws_o, *ws_ml;      // split rows: [pair][row][max_parts][D] sums, [..][2] maximum and sum
  unsigned int *status;
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// Tokens of sequence b as this call sees them, and the keys they attend.
struct Rows {
  int32_t first, count;  // tokens
  int64_t start;
  int32_t total;  // keys of the last token
  bool cut;

  __device__ __forceinline__ int keys(const PagedAttendArgs &a, int i) const {
    if (!a.causal) return total;
    return start < 0 ? 0 : static_cast<int>(min(start + i + 1, static_cast<int64_t>(a.max_seqlen)));
  }
};

__device__ __forceinline__ Rows rows_of(const PagedAttendArgs &a, int b) {
  const Sequence s = sequence_of(a.p, b);
  Rows r;
  r.first = s.first;
  r.count = min(s.count, a.max_tokens);
  r.start = s.start;
  const int64_t all = s.start < 0 ? 0 : static_cast<int64_t>(s.start) + s.count;
  r.total = static_cast<int>(min(all, static_cast<int64_t>(a.max_seqlen)));
  r.cut = s.count > a.max_tokens || all > a.max_seqlen;
  return r;
}

// The matrix products of one type.  A probability is held at 2^kShift of the
// running maximum, which moves when a score exceeds it by kSlack more (log2
// units), and enters P V as hi + lo, two 16-bit terms: what bounds the kernel
// is memory, and one term would double the error of a 16-bit output.  fp16
// ends at 2^-24, so that at scale 1 many small probabilities would be lost;
// 2^(11 + 4) still lies below its largest.
template <typename T>
struct Mma;

template <>
struct Mma<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static constexpr float kShift = 0.f, kSlack = 8.f;
  __device__ __forceinline__ static f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ static void split(float p0, float p1, unsigned int *hi, unsigned int *lo) {
    const v2 h = {static_cast<__bf16>(p0), static_cast<__bf16>(p1)};
    const v2 r = {static_cast<__bf16>(p0 - static_cast<float>(h[0])), static_cast<__bf16>(p1 - static_cast<float>(h[1]))};
    *hi = __builtin_bit_cast(unsigned int, h);
    *lo = __builtin_bit_cast(unsigned int, r);
  }
};

template <>
struct Mma<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static constexpr float kShift = 11.f, kSlack = 4.f;
  __device__ __forceinline__ static f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ static void split(float p0, float p1, unsigned int *hi, unsigned int *lo) {
    const v2 h = {static_cast<_Float16>(p0), static_cast<_Float16>(p1)};
    const v2 r = {static_cast<_Float16>(p0 - static_cast<float>(h[0])), static_cast<_Float16>(p1 - static_cast<float>(h[1]))};
    *hi = __builtin_bit_cast(unsigned int, h);
    *lo = __builtin_bit_cast(unsigned int, r);
  }
};

template <>
struct Mma<float> {
  static constexpr float kShift = 0.f, kSlack = 8.f;
};

// Row (token i, query head qh) of sequence b over keys [p0, end) by one wave, key by key
// in fp32: lanes hold a key each for the scores, D / 64 outputs each for the
// values.  For rows whose result is not finite: masked keys (and keys of pages outside the
// pool) enter the matrix products with probability 0, which an infinity or
// NaN among the values turns into NaN; here they are not touched.
template <typename T, int D>
__device__ void exact_row(const PagedAttendArgs &a, const T *q, int b, int hk, int p0, int end, float *m_out, float *l_out,
                          float *o) {
  using E = Elem<T>;
  constexpr int DPL = D >= 64 ? D / 64 : 1;
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  const int lane = threadIdx.x & 63;
  const int32_t *table = a.p.tables + b * a.p.table_stride;
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < DPL; ++e) o[e] = 0.f;
#pragma unroll 1
  for (int k0 = p0; k0 < end; k0 += 64) {
    const int pos = min(k0 + lane, end - 1);
    const int page = table[pos >> a.p.shift];
    const bool in_pool = static_cast<unsigned>(page) < static_cast<unsigned>(a.p.n_pages);
    const uint64_t seen = __ballot(k0 + lane < end && in_pool);
    const int64_t at = (in_pool ? page : 0) * a.p.page_stride + (pos & ((1 << a.p.shift) - 1)) * a.p.pos_stride +
                       hk * a.p.head_stride;
    const T *k = static_cast<const T *>(a.pages) + at;
    float s = 0.f;
#pragma unroll 1
    for (int c = 0; c < D; c += VEC)
      s = E::dot(*reinterpret_cast<const u32x4 *>(q + c), *reinterpret_cast<const u32x4 *>(k + c), s);
    const bool mine = seen >> lane & 1;
    if (!mine) s = -INFINITY;
    const float mt = wave_max(s) * a.scale_log2;
    if (mt > m) {
      const float c = exp2_of(m - mt);
      m = mt;
      l *= c;
#pragma unroll
      for (int e = 0; e < DPL; ++e) o[e] *= c;
    }
    const float p = mine ? exp2_of(fmaf(s, a.scale_log2, m == -INFINITY ? 0.f : -m)) : 0.f;
    l += p;
    uint64_t left = seen;
#pragma unroll 1
    while (left) {
      const int j = __builtin_ctzll(left);
      left &= left - 1;
      const float pj = __shfl(p, j);
      const int64_t vat = __shfl(at, j) + a.p.kv_stride;
      const T *v = static_cast<const T *>(a.pages) + vat + (D >= 64 ? lane * DPL : lane & (D - 1));
#pragma unroll
      for (int e = 0; e < DPL; ++e) o[e] = fmaf(pj, static_cast<float>(v[e]), o[e]);
    }
  }
  *m_out = m;
  *l_out = sum_from<1>(l);
}

template <typename T, int D, int W>
__global__ __launch_bounds__(W * 64) void paged_rows_kernel(const PagedAttendArgs a) {
  constexpr bool F32 = std::is_same<T, float>::value;
  using M = Mma<T>;
  constexpr int KEYS = F32 ? 16 : 32;       // keys of a step
  constexpr int NT = KEYS / 16;             // 16-key blocks of a step
  constexpr int NK = F32 ? D / 16 : (D >= 32 ? D / 32 : 1);  // K vectors of a lane and block
  constexpr int NV = D / 16;                // 16-bit: V vectors of a lane and step
  constexpr int VW = D >= 64 ? 4 : D / 16;  // fp32: V elements of a load
  constexpr int NB = D / (16 * VW);         // fp32: loads of a V row
  constexpr int ND = D / 16;                // output blocks
  constexpr int CH = D / 8;                 // 16-bit: 16-byte chunks of a V row
  constexpr int VP = 2 * D + 32;            // 16-bit: LDS bytes of a V row
  constexpr int OP = D + 4;                 // floats of a row in the join
  constexpr int kVBytes = F32 ? 0 : W * KEYS * VP, kOBytes = W * 16 * OP * 4;
  __shared__ __attribute__((aligned(16))) char s_mem[kVBytes > kOBytes ? kVBytes : kOBytes];
  __shared__ float s_m[W][16], s_l[W][16];
  __shared__ int s_bad;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int pairs = a.p.batch * a.kv_heads;
  int block = blockIdx.x;
  const int pair = block % pairs;
  block /= pairs;
  const int part = block % a.max_parts, tile = block / a.max_parts;
  const int b = pair / a.kv_heads, hk = pair - b * a.kv_heads;
  const Rows seq = rows_of(a, b);
  const int rows = seq.count * a.group, row0 = tile * 16;
  if (seq.cut && threadIdx.x == 0 && part == 0 && tile == 0) raise_status(a.status, HEXKV_STATUS_LENGTH_CLAMPED);
  if (row0 >= rows) return;
  const int p0 = part * a.part;
  const int live = min(16, rows - row0);
  const int t_first = row0 / a.group, t_last = (row0 + live - 1) / a.group;
  const int end = min(seq.keys(a, t_last), p0 + a.part);    // keys [p0, end) are the workgroup's
  if (part > 0 && end <= p0) return;
  const int full = min(seq.keys(a, t_first), end);          // all rows see the keys below

  // this lane's row; those past the last repeat it
  const int row = min(row0 + r, rows - 1), t = row / a.group, qh = hk * a.group + row - t * a.group;
  const int len = seq.keys(a, t), lim = min(len, p0 + a.part);
  const T *q_row = static_cast<const T *>(a.q) + (seq.first + t) * a.q_stride + static_cast<int64_t>(qh) * D;
  u32x4 qf[NK];
#pragma unroll
  for (int j = 0; j < NK; ++j) {
    if constexpr (F32) qf[j] = *reinterpret_cast<const u32x4 *>(q_row + 16 * j + 4 * g);
    else if constexpr (D >= 32) qf[j] = *reinterpret_cast<const u32x4 *>(q_row + 32 * j + 8 * g);
    else qf[j] = g < 2 ? *reinterpret_cast<const u32x4 *>(q_row + 8 * g) : u32x4{};
  }

  const T *head = static_cast<const T *>(a.pages) + hk * a.p.head_stride;
  const int32_t *table = a.p.tables + b * a.p.table_stride;
  const int last = (max(end, 1) - 1) & ~15;
  unsigned bad_pages = 0;

  // Where the 16-key block at position k lies (blocks past the end: the last one's place).
  auto place = [&](int k, bool *in_pool) {
    const int at = min(k, last);
    const int page = __builtin_amdgcn_readfirstlane(table[at >> a.p.shift]);
    *in_pool = static_cast<unsigned>(page) < static_cast<unsigned>(a.p.n_pages);
    return (*in_pool ? page : 0) * a.p.page_stride + (at & ((1 << a.p.shift) - 1)) * a.p.pos_stride;
  };
  const int64_t k_lane = F32 ? r * a.p.pos_stride + 4 * g : r * a.p.pos_stride + (D >= 32 ? 8 * g : 8 * (g & 1));
  auto load_k = [&](u32x4 (&k)[NT][NK], const int64_t *at) {
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
      for (int j = 0; j < NK; ++j)
        k[kt][j] = *reinterpret_cast<const u32x4 *>(head + at[kt] + k_lane + (F32 ? 16 : 32) * j);
  };
  // 16-bit: lane l loads chunk l % CH of row l / CH + i * 64 / CH.
  const int v_row = lane / CH, v_ch = lane % CH;
  auto load_v16 = [&](u32x4 (&v)[NV], const int64_t *at) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int kk = v_row + i * (64 / CH);
      const int64_t base = D == 16 ? (kk < 16 ? at[0] : at[NT - 1]) : at[(i * (64 / CH)) / 16];
      v[i] = *reinterpret_cast<const u32x4 *>(head + base + a.p.kv_stride + (kk & 15) * a.p.pos_stride + 8 * v_ch);
    }
  };
  // fp32: lane (r, g) loads dims VW r of key 4 g + i.
  typedef float vw __attribute__((ext_vector_type(VW)));
  auto load_v32 = [&](vw (&v)[4][NB], const int64_t *at) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < NB; ++n)
        v[i][n] = *reinterpret_cast<const vw *>(reinterpret_cast<const float *>(head) + at[0] + a.p.kv_stride +
                                                (4 * g + i) * a.p.pos_stride + n * 16 * VW + VW * r);
  };

  float m = -INFINITY, l = 0.f;  // m: the running maximum less kShift
  f32x4 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x4{};

  constexpr int STRIDE = W * KEYS;
  int k0 = p0 + wave * KEYS;
  if (k0 < end) {
    u32x4 kf[NT][NK];
    u32x4 v16[F32 ? 1 : NV];
    vw v32[F32 ? 4 : 1][F32 ? NB : 1];
    int64_t at[NT], at_next[NT];
    bool in[NT], in_next[NT];
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) at[kt] = place(k0 + 16 * kt, &in[kt]);
    load_k(kf, at);
    if constexpr (F32) load_v32(v32, at);
    else load_v16(v16, at);
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) at_next[kt] = place(k0 + STRIDE + 16 * kt, &in_next[kt]);
    char *s_v = s_mem + wave * KEYS * VP;
    for (; k0 < end; k0 += STRIDE) {
      f32x4 s[NT];
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        s[kt] = f32x4{};
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[kt][j][e]), __uint_as_float(qf[j][e]), s[kt], 0, 0, 0);
          } else {
            u32x4 kv = kf[kt][j];
            if constexpr (D == 16) kv = g < 2 ? kv : u32x4{};
            s[kt] = M::mma(kv, qf[j], s[kt]);
          }
        }
      }
      load_k(kf, at_next);
      bool masked = k0 + KEYS > full;
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) masked |= !in[kt];
      vw vf[F32 ? 4 : 1][F32 ? NB : 1];
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < NB; ++n) vf[i][n] = v32[i][n];
      }
      if (masked) {
        const int left = lim - k0;
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
          bad_pages |= !in[kt] && k0 + 16 * kt < end;
#pragma unroll
          for (int i = 0; i < 4; ++i) s[kt][i] = in[kt] && 16 * kt + 4 * g + i < left ? s[kt][i] : -INFINITY;
        }
        // keys that no row of the tile attends (rows of the page not yet
        // written, pages outside the pool) give zeros
        if constexpr (F32) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < NB; ++n)
              if (!in[0] || k0 + 4 * g + i >= end) vf[i][n] = vw{};
        } else {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int kk = v_row + i * (64 / CH);
            if (k0 + kk >= end || !(kk < 16 ? in[0] : in[NT - 1])) v16[i] = u32x4{};
          }
        }
      }
      if constexpr (F32) {
        load_v32(v32, at_next);
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          *reinterpret_cast<u32x4 *>(s_v + (v_row + i * (64 / CH)) * VP + v_ch * 16) = v16[i];
        load_v16(v16, at_next);
      }
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        in[kt] = in_next[kt];
        at_next[kt] = place(k0 + 2 * STRIDE + 16 * kt, &in_next[kt]);
      }

      float mt = s[0][0];
#pragma unroll
      for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mt = fmaxf(mt, s[kt][i]);
      mt = xor_step<32>(xor_step<16>(mt, MaxOp{}), MaxOp{}) * a.scale_log2;
      const bool up = mt > m + (M::kShift + M::kSlack);
      if (__any(up)) {
        const float mnew = up ? mt - M::kShift : m;
        const float f = up ? exp2_of(m - mnew) : 1.f;
        m = mnew;
        l *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= f;
      }
      const float base = m == -INFINITY ? 0.f : -m;
      float p[NT][4];
#pragma unroll
      for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[kt][i] = exp2_of(fmaf(s[kt][i], a.scale_log2, base));
          l += p[kt][i];
        }
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < VW; ++e)
              acc[n * VW + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[i][n][e], p[0][i], acc[n * VW + e], 0, 0, 0);
      } else {
        u32x4 hi, lo;
#pragma unroll
        for (int kt = 0; kt < NT; ++kt)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            unsigned int x, y;
            M::split(p[kt][i], p[kt][i + 1], &x, &y);
            hi[2 * kt + i / 2] = x;
            lo[2 * kt + i / 2] = y;
          }
        auto *shared = (__attribute__((address_space(3))) char *)s_v;
        const int s16 = lane & 15;
        const uint32_t v_read = static_cast<uint32_t>((4 * g + s16 / 4) * VP + (s16 % 4) * 8);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const h4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_h4 *)(shared + v_read + d * 32));
          const h4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_h4 *)(shared + v_read + d * 32 + 16 * VP));
          const u32x4 v = __builtin_bit_cast(u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
          acc[d] = M::mma(v, hi, acc[d]);
          acc[d] = M::mma(v, lo, acc[d]);
        }
      }
    }
  }
  if (bad_pages && lane == 0) raise_status(a.status, HEXKV_STATUS_PAGE);

  // The waves' sums, joined in LDS at the largest of their maxima.
  l = xor_step<32>(xor_step<16>(l, AddOp{}), AddOp{});
  if (g == 0) {
    s_m[wave][r] = m;
    s_l[wave][r] = l;
  }
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  float *s_o = reinterpret_cast<float *>(s_mem);
  {
    float top = s_m[0][r];
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, s_m[w][r]);
    const float f = m == -INFINITY ? 0.f : exp2_of(m - top);
    float *o = s_o + (wave * 16 + r) * OP;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      if constexpr (F32) {
        // block (n, e) holds dims 16 VW n + VW (4 g + i) + e
#pragma unroll
        for (int i = 0; i < 4; ++i) o[(d / VW) * 16 * VW + VW * (4 * g + i) + d % VW] = acc[d][i] * f;
      } else {
        *reinterpret_cast<f32x4 *>(o + 16 * d + 4 * g) = acc[d] * f;
      }
    }
  }
  __syncthreads();
  // Four outputs of a row a thread, D / 4 threads a row.
  constexpr int PER = D / 4, PASSES = (16 * PER + W * 64 - 1) / (W * 64);
  f32x4 o[PASSES];
  float top[PASSES], sum[PASSES];
  int bad = 0;
#pragma unroll
  for (int n = 0; n < PASSES; ++n) {
    const int u = static_cast<int>(threadIdx.x) + n * W * 64, rr = u / PER, c = u % PER;
    if (rr >= live) continue;
    top[n] = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) top[n] = fmaxf(top[n], s_m[w][rr]);
    sum[n] = 0.f;
    o[n] = f32x4{};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      sum[n] += s_m[w][rr] == -INFINITY ? 0.f : s_l[w][rr] * exp2_of(s_m[w][rr] - top[n]);
      o[n] += *reinterpret_cast<const f32x4 *>(s_o + (w * 16 + rr) * OP + 4 * c);
    }
    const float check = (o[n][0] + o[n][1] + o[n][2] + o[n][3] + sum[n]) * 0.f;
    if (!(check == 0.f)) bad |= 1 << rr;
  }
  if (bad) atomicOr(&s_bad, bad);
  __syncthreads();
  const int redo = s_bad;
#pragma unroll
  for (int n = 0; n < PASSES; ++n) {
    const int u = static_cast<int>(threadIdx.x) + n * W * 64, rr = u / PER, c = u % PER;
    if (rr >= live || redo >> rr & 1) continue;
    const int rrow = row0 + rr, tt = rrow / a.group, hh = hk * a.group + rrow - tt * a.group;
    const int rlen = seq.keys(a, tt);
    if (part > 0 && rlen <= p0) continue;
    if (rlen <= a.part) {
      if (rlen <= 0) o[n] = f32x4{};
      else o[n] *= 1.f / sum[n];
      store4(static_cast<T *>(a.out) + (seq.first + tt) * a.o_stride + static_cast<int64_t>(hh) * D + 4 * c, o[n]);
    } else {
      const int64_t slot = ((static_cast<int64_t>(pair) * a.row_tiles + tile) * 16 + rr) * a.max_parts + part;
      *reinterpret_cast<f32x4 *>(a.ws_o + slot * D + 4 * c) = o[n];
      if (c == 0) *reinterpret_cast<float2 *>(a.ws_ml + slot * 2) = float2{top[n], sum[n]};
    }
  }
  if (!redo || wave) return;
  for (int left = redo; left; left &= left - 1) {
    const int rr = __builtin_ctz(left), rrow = row0 + rr, tt = rrow / a.group, hh = hk * a.group + rrow - tt * a.group;
    const int rlen = seq.keys(a, tt), rend = min(rlen, p0 + a.part);
    if (part > 0 && rlen <= p0) continue;
    constexpr int DPL = D >= 64 ? D / 64 : 1;
    float em, el, eo[DPL];
    exact_row<T, D>(a, static_cast<const T *>(a.q) + (seq.first + tt) * a.q_stride + static_cast<int64_t>(hh) * D, b, hk, p0,
                    rend, &em, &el, eo);
    if (lane * DPL >= D) continue;
    const bool split = rlen > a.part;
    T *out = static_cast<T *>(a.out) + (seq.first + tt) * a.o_stride + static_cast<int64_t>(hh) * D + lane * DPL;
    const int64_t slot = ((static_cast<int64_t>(pair) * a.row_tiles + tile) * 16 + rr) * a.max_parts + part;
#pragma unroll
    for (int e = 0; e < DPL; ++e) {
      if (split) a.ws_o[slot * D + lane * DPL + e] = eo[e];
      else out[e] = Elem<T>::from_float(rlen <= 0 ? 0.f : eo[e] / el);
    }
    if (split && lane == 0) *reinterpret_cast<float2 *>(a.ws_ml + slot * 2) = float2{em, el};
  }
}

// The partitions of a split row, joined: a wave a row.
constexpr int kJoinThreads = 256;
constexpr int kMaxParts = 64;  // a lane each

template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(const PagedAttendArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (kJoinThreads / 64) + (threadIdx.x >> 6);
  const int per = a.row_tiles * 16;
  const int64_t pair = id / per;
  if (pair >= static_cast<int64_t>(a.p.batch) * a.kv_heads) return;
  const int row = static_cast<int>(id - pair * per);
  const int b = static_cast<int>(pair / a.kv_heads), hk = static_cast<int>(pair - static_cast<int64_t>(b) * a.kv_heads);
  const Rows seq = rows_of(a, b);
  if (row >= seq.count * a.group) return;
  const int t = row / a.group, qh = hk * a.group + row - t * a.group;
  const int len = seq.keys(a, t);
  if (len <= a.part) return;
  const int parts = (len + a.part - 1) / a.part;
  const int64_t slot = id * a.max_parts;
  float2 ml{-INFINITY, 0.f};
  if (lane < parts) ml = *reinterpret_cast<const float2 *>(a.ws_ml + (slot + lane) * 2);
  const float top = wave_max(ml.x);
  const float w = ml.x == -INFINITY ? 0.f : exp2_of(ml.x - top);
  const float sum = sum_from<1>(ml.y * w);
  constexpr int DPL = D >= 64 ? D / 64 : 1;
  if (lane * DPL >= D) return;
  float o[DPL] = {};
  const float *src = a.ws_o + slot * D + lane * DPL;
  for (int p = 0; p < parts; ++p) {
    const float wp = __shfl(w, p);
#pragma unroll
    for (int e = 0; e < DPL; ++e) o[e] = fmaf(src[static_cast<int64_t>(p) * D + e], wp, o[e]);
  }
  T *out = static_cast<T *>(a.out) + (seq.first + t) * a.o_stride + static_cast<int64_t>(qh) * D + lane * DPL;
#pragma unroll
  for (int e = 0; e < DPL; ++e) out[e] = Elem<T>::from_float(o[e] / sum);
}

// ------------------------------------------------------------------ host ---

static int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Checks a call and fills its arguments but for addresses.
static int fill_attend(const hexkv_paged_attend_params *params, PagedAttendArgs *a, const char *what) {
  if (!params) return fail(HEXKV_EINVAL, "%s: null argument", what);
  const hexkv_paged_attend_params &p = *params;
  int rc = fill_tables(p.pool, p.seqs, &a->p, what);
  if (rc != HEXKV_OK) return rc;
  const int d = p.pool.head_dim, vec = 16 / elem_bytes(p.pool.dtype);
  if (p.q_heads < 1 || p.q_heads > 1 << 16 || p.q_heads % p.pool.kv_heads)
    return fail(HEXKV_EINVAL, "%s: %d query heads on %d KV heads", what, p.q_heads, p.pool.kv_heads);
  if (!(p.softmax_scale > 0.f) || p.softmax_scale > 3e38f) return fail(HEXKV_EINVAL, "%s: softmax_scale is not positive", what);
  if (p.max_seqlen < 0 || p.max_seqlen > static_cast<int64_t>(p.seqs.table_width) * p.pool.page_size)
    return fail(HEXKV_ERANGE, "%s: max_seqlen %d outside the tables' [0, %lld]", what, p.max_seqlen,
                static_cast<long long>(p.seqs.table_width) * p.pool.page_size);
  const int64_t row = static_cast<int64_t>(p.q_heads) * d, tokens = p.seqs.tokens;
  if (tokens > 1 && (p.q_stride < row || p.q_stride % vec))
    return fail(HEXKV_EINVAL, "%s: q's rows overlap or are not 16-byte aligned", what);
  if (tokens > 1 && p.out_stride < row) return fail(HEXKV_EINVAL, "%s: out's rows overlap", what);
  if (p.partition < 0 || p.partition % 64) return fail(HEXKV_EINVAL, "%s: partition %d is not a multiple of 64", what, p.partition);
  if (p.seqs.cu_tokens && p.max_tokens < 0) return fail(HEXKV_EINVAL, "%s: negative max_tokens", what);
  a->q = p.q;
  a->pages = p.pages;
  a->out = p.out;
  a->q_stride = p.q_stride;
  a->o_stride = p.out_stride;
  a->q_heads = p.q_heads;
  a->kv_heads = p.pool.kv_heads;
  a->group = p.q_heads / p.pool.kv_heads;
  a->causal = p.causal ? 1 : 0;
  a->max_tokens = p.seqs.cu_tokens ? std::min(p.max_tokens, p.seqs.tokens) : a->p.each;
  a->max_seqlen = p.max_seqlen;
  a->scale_log2 = p.softmax_scale * 1.44269504f;
  const int64_t rows = static_cast<int64_t>(a->max_tokens) * a->group, pairs = static_cast<int64_t>(p.seqs.batch) * a->kv_heads;
  const int64_t tiles = (rows + 15) / 16;
  if (rows > INT32_MAX || pairs * tiles >= INT64_C(1) << 24)
    return fail(HEXKV_ERANGE, "%s: 2^24 tiles of rows or more", what);
  a->row_tiles = static_cast<int32_t>(tiles);
  int64_t part = p.partition;
  if (!part) {
    const int64_t want = pairs * tiles ? std::max<int64_t>(1, 768 / (pairs * tiles)) : 1;
    part = std::max<int64_t>(256, round_up((p.max_seqlen + want - 1) / want, 64));
  }
  while ((p.max_seqlen + part - 1) / part > kMaxParts) part = round_up((p.max_seqlen + kMaxParts - 1) / kMaxParts, 64);
  a->part = static_cast<int32_t>(part);
  a->max_parts = static_cast<int32_t>(std::max<int64_t>(1, (p.max_seqlen + part - 1) / part));
  if (pairs * tiles * a->max_parts >= INT64_C(1) << 24) return fail(HEXKV_ERANGE, "%s: 2^24 workgroups or more", what);
  return HEXKV_OK;
}

static size_t attend_workspace(const PagedAttendArgs &a, int head_dim) {
  if (a.max_parts <= 1) return 0;
  return static_cast<size_t>(a.p.batch) * a.kv_heads * a.row_tiles * 16 * a.max_parts * (head_dim + 2) * sizeof(float);
}

template <typename T, int D>
static void launch_rows(const PagedAttendArgs &a, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.p.batch) * a.kv_heads * a.row_tiles;
  constexpr int W = 4;
  paged_rows_kernel<T, D, W><<<dim3(static_cast<unsigned>(rows * a.max_parts)), W * 64, 0, s>>>(a);
  if (a.max_parts > 1) paged_join_kernel<T, D><<<dim3(static_cast<unsigned>(rows * 4)), kJoinThreads, 0, s>>>(a);
}

template <typename T>
static void launch_dims(const PagedAttendArgs &a, int head_dim, hipStream_t s) {
  switch (head_dim) {
    case 16: launch_rows<T, 16>(a, s); break;
    case 32: launch_rows<T, 32>(a, s); break;
    case 64: launch_rows<T, 64>(a, s); break;
    case 128: launch_rows<T, 128>(a, s); break;
    default: launch_rows<T, 256>(a, s); break;
  }
}

}  // namespace hexkv

extern "C" size_t hexkv_paged_attend_workspace_bytes(const hexkv_paged_attend_params *params) {
  using namespace hexkv;
  clear_error();
  PagedAttendArgs a;
  if (fill_attend(params, &a, "hexkv_paged_attend_workspace_bytes") != HEXKV_OK) return 0;
  return attend_workspace(a, params->pool.head_dim);
}

extern "C" int hexkv_paged_attend(const hexkv_paged_attend_params *params, void *workspace, size_t workspace_bytes,
                                  hexkv_stream_t stream) {
  using namespace hexkv;
  clear_error();
  const char *what = "hexkv_paged_attend";
  PagedAttendArgs a;
  int rc = fill_attend(params, &a, what);
  if (rc != HEXKV_OK) return rc;
  if (a.p.tokens == 0 || a.p.batch == 0 || a.max_tokens == 0) return HEXKV_OK;
  if (!a.q || !a.out || !a.pages) return fail(HEXKV_EINVAL, "%s: null tensor", what);
  if (!aligned16(a.q) || !aligned16(a.pages)) return fail(HEXKV_EINVAL, "%s: q or pages are not 16-byte aligned", what);
  const int d = params->pool.head_dim;
  const size_t need = attend_workspace(a, d);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(HEXKV_EWORKSPACE, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", what, need, workspace_bytes);
  a.ws_o = static_cast<float *>(workspace);
  a.ws_ml = need ? a.ws_o + static_cast<int64_t>(a.p.batch) * a.kv_heads * a.row_tiles * 16 * a.max_parts * d : nullptr;
  rc = status_word(stream, &a.status, what);
  if (rc != HEXKV_OK) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (params->pool.dtype) {
    case HEXKV_BF16: launch_dims<__bf16>(a, d, s); break;
    case HEXKV_F16: launch_dims<_Float16>(a, d, s); break;
    default: launch_dims<float>(a, d, s); break;
  }
  return check_launch(what);
}
