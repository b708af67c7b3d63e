// Attention over a paged cache: hexkv_paged_attend.
//
// A row is one query head of one new token; the rows of a sequence that share
// a KV head (tokens x group of them, in (token, head) order) read the same keys.
//
// Row path: 16 rows a workgroup, its waves taking steps of the keys in turn.
//   S^T = K Q^T    16 keys x 16 rows a matrix instruction: lane (r, g) holds key
//                  r, dims of chunk g
//   softmax        a lane's scores are all its own row's; the other 3 lanes
//                  of a row are two exchanges away
//   O^T += V^T P^T the scores' layout is P's operand as it stands, with the contraction
//                  index of a step being key 4 g + i (16-bit: then 16 + 4 g + i);
//                  V^T is read transposed from LDS, fp32 V loaded in place
// 16-bit rows are loaded whole, 16 lanes a row, and pass through the wave's own
// LDS (K, then V in the same place): loaded as K's operand takes it, in 64 bytes of
// each of 16 rows, a line was asked for twice, and the loads could not be
// nontemporal (Llama-3-8B decode batch 211 us, 224 nontemporal, against 185).
// What bounds it: a decode row's K and V are read once, 4 D flops a key, so
// memory (64 sequences of 128 to 8192, 8 KV heads of 128: 1.10 GB in 181 us, 6.1 TB/s).  Steps are loaded one ahead into registers, page numbers two ahead.
//
// Tile path (16-bit, head_dim from 64 on, sequences of more than kFewRows rows):
// 32 rows a wave, four or eight waves a workgroup (128 or 256 rows), which share tiles of
// 16 keys a wave in LDS; the same products on 32 x 32 x 16 matrix instructions.  What
// bounds it: the matrix cores, the LDS reads of their operands, and the softmax on the
// VALU beside them (2048 rows over 8192 keys, 32 heads of 128 on 8: 424 us, 729 TFLOP/s,
// the second terms' products not counted).  A probability enters P V as hi + lo here too:
// one rounded term takes 316 us, but its error is half a step of the type, as much as the
// output's own rounding.
#include "hexkv_paged.h"

#include <algorithm>
#include <type_traits>

namespace hexkv {

typedef short h4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) h4 lds_h4;

struct PagedAttendArgs {
  PageTables p;
  const void *q, *pages;
  void *out;
  int64_t q_stride, o_stride;
  int32_t q_heads, kv_heads, group, causal;
  int32_t max_tokens, max_seqlen;
  uint32_t page_bytes, pos_bytes;  // of the pool
  float scale_log2;
  int32_t few_rows;         // a sequence's rows per KV head up to which it takes the row path
  // row path: 16-row tiles of a sequence and KV head (at most), keys per partition,
  // partitions of the longest row, workgroups
  int32_t row_tiles, part, max_parts, row_blocks;
  // tile path: a bound on the tiles of all sequences, keys per partition and
  // partitions, and workgroups
  int32_t tiles, tile_part, tile_parts, tile_blocks, wide;
  // split rows: of the row path [sequence][KV head][pair_rows][max_parts], or where tokens times heads
  // are fewer (pair_rows 0) [token][head][max_parts], of the tile path [token][head][tile_parts]; each of D
  // sums, and of (maximum, sum)
  int32_t pair_rows;
  float *ws_o, *ws_ml, *ws_tile_o, *ws_tile_ml;
  unsigned int *status;
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// What a row's sums are multiplied by: its softmax's reciprocal sum, 0 where
// nothing was attended.
__device__ __forceinline__ float weight_of(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }

// Tokens of sequence b as this call sees them, and the keys they attend.
struct Rows {
  int32_t first, count;  // tokens
  int32_t start;
  int32_t total;  // keys of the last token
  bool cut;

  __device__ __forceinline__ int keys(const PagedAttendArgs &a, int i) const {
    if (!a.causal) return total;
    return start < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(start) + i + 1, static_cast<int64_t>(a.max_seqlen)));
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

// The place of the row path's split row `row` of sequence b and KV head hk (its token t and head qh), less
// its partitions.
__device__ __forceinline__ int64_t few_slot(const PagedAttendArgs &a, int b, int hk, int row, int first, int t, int qh) {
  return a.pair_rows ? (static_cast<int64_t>(b) * a.kv_heads + hk) * a.pair_rows + row
                     : static_cast<int64_t>(first + t) * a.q_heads + qh;
}

// Workgroups of either path are numbered by (tile, partition, KV head), the
// head fastest; a tile is one of those of all sequences, which the host bounds by
// the tokens' number: a launch over (sequence, most tiles) of 2 chunks beside 46 single tokens
// was 17000 workgroups, 200 us of them leaving at once.
struct Place {
  int b, tile, part, hk;
  Rows seq;
};

// The sequence that has the index-th of all tiles, and which of its own that is
// (b -1: none).  tiles(count): those of a sequence of so many tokens.
template <typename F>
__device__ __forceinline__ Place place_of(const PagedAttendArgs &a, int block, int parts, int reversed_from, F tiles) {
  Place p;
  const int rest = block / a.kv_heads;
  p.hk = block - rest * a.kv_heads;
  p.part = rest % parts;
  int index = rest / parts;
  if (reversed_from) index = reversed_from - 1 - index;
  if (!a.p.cu) {
    const int each = tiles(a.max_tokens);
    p.b = each ? index / each : a.p.batch;
    p.tile = index - p.b * each;
    if (p.b >= a.p.batch) p.b = -1;
    else p.seq = rows_of(a, p.b);
    return p;
  }
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < a.p.batch; b0 += 64) {
    const int b = b0 + lane;
    const Rows seq = rows_of(a, min(b, a.p.batch - 1));
    const int n = b < a.p.batch ? tiles(seq.count) : 0;
    int upto = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(upto, d);
      if (lane >= d) upto += x;
    }
    const uint64_t past = __ballot(upto > index);
    if (past) {
      const int j = __builtin_ctzll(past);
      p.b = __builtin_amdgcn_readfirstlane(b0 + j);
      p.tile = index - __builtin_amdgcn_readlane(upto - n, j);
      p.seq.first = __builtin_amdgcn_readlane(seq.first, j);
      p.seq.count = __builtin_amdgcn_readlane(seq.count, j);
      p.seq.start = __builtin_amdgcn_readlane(seq.start, j);
      p.seq.total = __builtin_amdgcn_readlane(seq.total, j);
      p.seq.cut = __builtin_amdgcn_readlane(static_cast<int>(seq.cut), j);
      return p;
    }
    index -= __builtin_amdgcn_readlane(upto, 63);
  }
  p.b = -1;
  p.tile = 0;
  return p;
}

// A sequence's table, read by scalar loads: a wave's lanes need the same page,
// and a vector load's number would be waited for behind the rows loaded before it
// (Llama-3-8B decode batch 217 us instead of 185).
typedef const __attribute__((address_space(4))) int32_t *ScalarTable;

__device__ __forceinline__ ScalarTable scalar_table(const PagedAttendArgs &a, int b) {
  return (ScalarTable)(a.p.tables + __builtin_amdgcn_readfirstlane(b) * a.p.table_stride);
}

// Bytes from the pool's base to position k's row in a page (in 64 bits: of a page's
// positions some may lie 2^32 bytes from its first).
__device__ __forceinline__ uint64_t block_offset(const PagedAttendArgs &a, int page, int k) {
  return static_cast<uint64_t>(static_cast<uint32_t>(page)) * a.page_bytes +
         static_cast<uint64_t>(static_cast<uint32_t>(k & ((1 << a.p.shift) - 1))) * a.pos_bytes;
}

// 16 rows of one head in a page, as a buffer that ends behind the last row that
// holds a key: rows past it (those of the page not yet written) and every row of
// a page outside the pool read as zeros, and blocks past the end, which the
// loads made ahead ask for, cost nothing.  (Addressed as memory the last block
// was loaded again in their place: 512 keys of a partition moved 25% more.)  Positions are up to
// 2^28 bytes apart, so that 15 of them and a row fit the buffer's 32 bits.
template <int ROW_BYTES>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t block_of(const char *at, int rows, uint32_t pos_bytes) {
  const uint32_t bytes = rows >= 16 ? 15 * pos_bytes + ROW_BYTES : rows > 0 ? (rows - 1) * pos_bytes + ROW_BYTES : 0;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(at), 0, __builtin_amdgcn_readfirstlane(bytes), 0x00027000);
}
constexpr int kNontemporal = 2;  // a buffer load's cache policy
template <int POLICY>
__device__ __forceinline__ u32x4 load_16(__amdgpu_buffer_rsrc_t block, uint32_t offset) {
  return __builtin_amdgcn_raw_buffer_load_b128(block, offset, 0, POLICY);
}

// The matrix products of one type.  A probability is held at 2^kShift of the
// running maximum, which moves when a score exceeds it by kSlack more (log2
// units), and enters P V as hi + lo, two 16-bit terms: one would double the
// error of a 16-bit output.  fp16
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
  __device__ __forceinline__ static f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
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
  __device__ __forceinline__ static f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
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

// LDS bytes of the row path: V as its waves turn it, then their sums.
template <typename T, int D, int W>
constexpr int rows_lds() {
  const int v = std::is_same<T, float>::value ? 0 : W * 32 * (2 * D + 32), o = W * 16 * (D + 4) * 4;
  return (v > o ? v : o) + 2 * W * 16 * 4 + 16;
}

template <typename T, int D, int W>
__device__ __forceinline__ void rows_path(const PagedAttendArgs &a, int block, char *s_mem) {
  constexpr bool F32 = std::is_same<T, float>::value;
  using M = Mma<T>;
  constexpr int KEYS = F32 ? 16 : 32;       // keys of a step
  constexpr int NT = KEYS / 16;             // 16-key blocks of a step
  constexpr int NK = F32 ? D / 16 : (D >= 32 ? D / 32 : 1);  // K vectors of a lane and block
  constexpr int NV = D >= 32 ? D / 16 : 2;  // 16-bit: vectors of a lane, of a step's K or V
  constexpr int VW = D >= 64 ? 4 : D / 16;  // fp32: V elements of a load
  constexpr int NB = D / (16 * VW);         // fp32: loads of a V row
  constexpr int ND = D / 16;                // output blocks
  constexpr int CH = D / 8;                 // 16-bit: 16-byte chunks of a V row
  constexpr int KP = 2 * D + 16;            // 16-bit: LDS bytes of a K row: 16 rows' chunks over all banks
  constexpr int VP = 2 * D + 32;            // of a V row: the 16 rows of a transposed read in two passes
  constexpr int OP = D + 4;                 // floats of a row in the join
  constexpr int kMl = rows_lds<T, D, W>() - 2 * W * 16 * 4 - 16;
  float(*s_m)[16] = reinterpret_cast<float(*)[16]>(s_mem + kMl), (*s_l)[16] = s_m + W;
  int &s_bad = *reinterpret_cast<int *>(s_mem + kMl + 2 * W * 16 * 4);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const Place mine = place_of(a, block, a.max_parts, 0, [&](int count) {
    return count * a.group <= a.few_rows ? (count * a.group + 15) / 16 : 0;
  });
  const int b = mine.b, hk = mine.hk, part = mine.part, tile = mine.tile;
  if (b < 0) return;
  const Rows seq = mine.seq;
  const int rows = seq.count * a.group, row0 = tile * 16;
  if (seq.cut && threadIdx.x == 0 && part == 0 && tile == 0) raise_status(a.status, HEXKV_STATUS_LENGTH_CLAMPED);
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

  // (addresses: a uniform base and a lane's 32-bit offset inside a block)
  constexpr int ES = static_cast<int>(sizeof(T));
  const char *head = static_cast<const char *>(a.pages) + hk * a.p.head_stride * ES;
  const ScalarTable table = scalar_table(a, b);
  const uint32_t pos_bytes = a.pos_bytes;
  const int64_t kv_bytes = a.p.kv_stride * ES;
  unsigned bad_pages = 0;

  // The page of the 16-key block at position k, and the block.
  struct Block {
    __amdgpu_buffer_rsrc_t k, v;
    bool in_pool;
  };
  auto page_of = [&](int k) { return table[min(k >> a.p.shift, a.p.width - 1)]; };
  auto block_at = [&](int k, int page) {
    Block x;
    x.in_pool = static_cast<unsigned>(page) < static_cast<unsigned>(a.p.n_pages);
    const char *at = head + block_offset(a, x.in_pool ? page : 0, k);
    x.k = block_of<D * ES>(at, x.in_pool ? end - k : 0, pos_bytes);
    x.v = block_of<D * ES>(at + kv_bytes, x.in_pool ? end - k : 0, pos_bytes);
    return x;
  };
  // 16-bit: lane l loads chunk l % CH of row l / CH + i * RPL, so that a load takes
  // whole rows, which nothing else reads (head_dim 16: by half of the lanes).
  constexpr int RPL = D >= 32 ? 64 / CH : 16;  // rows of a load
  const int v_row = lane / CH, v_ch = lane % CH;
  const bool loads = v_row < RPL;
  auto load16 = [&](u32x4 (&v)[NV], const Block *at, bool values) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t off = ((v_row + i * RPL) & 15) * pos_bytes + 16 * v_ch;
      v[i] = load_16<kNontemporal>(values ? at[i * RPL / 16].v : at[i * RPL / 16].k, loads ? off : ~0u);
    }
  };
  auto store16 = [&](const u32x4 (&v)[NV], char *to, int pitch) {
    if (!loads) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) *reinterpret_cast<u32x4 *>(to + (v_row + i * RPL) * pitch + v_ch * 16) = v[i];
  };
  const uint32_t k_lane = r * pos_bytes + 16 * g;
  auto load_k32 = [&](u32x4 (&k)[NK], const Block &at) {
#pragma unroll
    for (int j = 0; j < NK; ++j) k[j] = load_16<0>(at.k, k_lane + 64 * j);
  };
  // fp32: lane (r, g) loads dims VW r of key 4 g + i.
  typedef float vw __attribute__((ext_vector_type(VW)));
  auto load_v32 = [&](vw (&v)[4][NB], const Block &at) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const uint32_t off = (4 * g + i) * pos_bytes + 4 * (n * 16 * VW + VW * r);
        if constexpr (VW == 4) v[i][n] = __builtin_bit_cast(vw, load_16<0>(at.v, off));
        else if constexpr (VW == 2) v[i][n] = __builtin_bit_cast(vw, __builtin_amdgcn_raw_buffer_load_b64(at.v, off, 0, 0));
        else v[i][n] = vw{__uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(at.v, off, 0, 0))};
      }
  };

  float m = -INFINITY, l = 0.f;  // m: the running maximum less kShift
  f32x4 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x4{};

  constexpr int STRIDE = W * KEYS;
  int k0 = p0 + wave * KEYS;
  if (k0 < end) {
    u32x4 k32[F32 ? NK : 1];
    u32x4 k16[F32 ? 1 : NV], v16[F32 ? 1 : NV];
    vw v32[F32 ? 4 : 1][F32 ? NB : 1];
    Block at[NT];
    bool in[NT];
    int page[NT];
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) {
      at[kt] = block_at(k0 + 16 * kt, page_of(k0 + 16 * kt));
      in[kt] = at[kt].in_pool;
    }
    if constexpr (F32) load_k32(k32, at[0]);
    else load16(k16, at, false);
    __builtin_amdgcn_sched_barrier(0);  // (in this order here, too: the loop waits for K alone)
    if constexpr (F32) load_v32(v32, at[0]);
    else load16(v16, at, true);
#pragma unroll
    for (int kt = 0; kt < NT; ++kt) page[kt] = page_of(k0 + STRIDE + 16 * kt);
    char *s_v = s_mem + wave * KEYS * VP;
    for (; k0 < end; k0 += STRIDE) {
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) {
        at[kt] = block_at(k0 + STRIDE + 16 * kt, page[kt]);
        page[kt] = page_of(k0 + 2 * STRIDE + 16 * kt);
      }
      f32x4 s[NT];
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) s[kt] = f32x4{};
      if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k32[j][e]), __uint_as_float(qf[j][e]), s[0], 0, 0, 0);
        load_k32(k32, at[0]);
      } else {
        store16(k16, s_v, KP);
        load16(k16, at, false);
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
          for (int kt = 0; kt < NT; ++kt) {
            u32x4 k = *reinterpret_cast<const u32x4 *>(s_v + (16 * kt + r) * KP + (D >= 32 ? 64 * j + 16 * g : 16 * (g & 1)));
            if constexpr (D == 16) k = g < 2 ? k : u32x4{};
            s[kt] = M::mma(k, qf[j], s[kt]);
          }
      }
      bool masked = k0 + KEYS > full;
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) masked |= !in[kt];
      if (masked) {
        const int left = lim - k0;
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
          bad_pages |= !in[kt] && k0 + 16 * kt < end;
#pragma unroll
          for (int i = 0; i < 4; ++i) s[kt][i] = in[kt] && 16 * kt + 4 * g + i < left ? s[kt][i] : -INFINITY;
        }
      }
      vw vf[F32 ? 4 : 1][F32 ? NB : 1];
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < NB; ++n) vf[i][n] = v32[i][n];
        load_v32(v32, at[0]);
      } else {
        store16(v16, s_v, VP);
        load16(v16, at, true);
      }
#pragma unroll
      for (int kt = 0; kt < NT; ++kt) in[kt] = at[kt].in_pool;

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
      o[n] *= weight_of(sum[n]);
      store4(static_cast<T *>(a.out) + (seq.first + tt) * a.o_stride + static_cast<int64_t>(hh) * D + 4 * c, o[n]);
    } else {
      const int64_t slot = few_slot(a, b, hk, rrow, seq.first, tt, hh) * a.max_parts + part;
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
    const int64_t slot = few_slot(a, b, hk, rrow, seq.first, tt, hh) * a.max_parts + part;
#pragma unroll
    for (int e = 0; e < DPL; ++e) {
      if (split) a.ws_o[slot * D + lane * DPL + e] = eo[e];
      else out[e] = Elem<T>::from_float(eo[e] * weight_of(el));
    }
    if (split && lane == 0) *reinterpret_cast<float2 *>(a.ws_ml + slot * 2) = float2{em, el};
  }
}

// ------------------------------------------------------------ tile path ---

constexpr int kCus = 256;
// A sequence of so many rows per KV head, or fewer, takes the row path (16 sequences of
// 40 rows over 4000 keys of 128 dims 19.0 us on tiles, 29.5 on rows; one alone 15.5 and 12.5).
constexpr int kFewRows = 32;

// Rows a wave takes, and keys it computes at a time.
constexpr int kWaveRows = 32, kStepKeys = 64;

// W waves: 32 W rows, and tiles of 16 W keys, a block of 16 brought by each wave.
template <int D, int W>
struct TileLds {
  static constexpr int KT = 16 * W;      // keys of a tile
  static constexpr int KP = 2 * D + 16;  // bytes per K row: 16 rows' chunks over all banks
  static constexpr int VP = 2 * D + 64;  // per V row: the 4 rows of a transposed read over all banks
  static constexpr int kBytes = 2 * KT * (KP + VP) + 16;
};

// The order of a block's matrix products and LDS reads.  Left alone the compiler reads a
// product's operands just before it, into registers that the last product has freed,
// and the matrix cores wait for each read (a chunk of 2048 over 8192 keys, its waves in
// two phases as below, 447 us instead of 429).
template <int N>
__device__ __forceinline__ void order_reads() {
  __builtin_amdgcn_sched_group_barrier(0x100, N, 0);
}
template <int N>
__device__ __forceinline__ void order_products() {
  __builtin_amdgcn_sched_group_barrier(0x008, N, 0);
}
template <int N, typename F>
__device__ __forceinline__ void repeat(F f) {
  if constexpr (N > 0) {
    f();
    repeat<N - 1>(f);
  }
}

// A barrier that waits for this wave's LDS accesses and for nothing else.
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// A wave, 32 rows, one per lane and half h:
//   S^T = K Q^T: K (A) from LDS, Q (B) in registers; lane (c, h) gets row c's
//   scores of keys 8 i + 4 h + e.
//   O^T += V^T P^T: that layout is the B operand as it stands (the contraction
//   index of a 16-key step is key 4 h + e, then 8 + 4 h + e), V^T (A) comes from
//   row-major LDS by transposing reads in the same order.
// All of a lane's accumulators belong to its own row.
template <typename T, int D, int W>
__device__ __forceinline__ void tile_path(const PagedAttendArgs &a, int block, char *s_mem) {
  using M = Mma<T>;
  using L = TileLds<D, W>;
  constexpr int KT = L::KT, NKB = kStepKeys / 32, kTileRows = kWaveRows * W;
  constexpr int NJ = D / 16;   // score steps
  constexpr int ND = D / 32;   // output blocks
  constexpr int CH = D / 8;    // 16-byte chunks of a head's row
  static_assert(KT % kStepKeys == 0, "whole steps");
  constexpr int KP = L::KP, VP = L::VP;
  char *s_k = s_mem, *s_v = s_mem + 2 * KT * KP;
  int &s_bad = *reinterpret_cast<int *>(s_mem + 2 * KT * (KP + VP));

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  // (the last tiles first: theirs are the most keys)
  const Place mine = place_of(a, block, a.tile_parts, a.tiles, [&](int count) {
    return count * a.group > a.few_rows ? (count * a.group + kTileRows - 1) / kTileRows : 0;
  });
  const int b = mine.b, hk = mine.hk, part = mine.part, tile = mine.tile;
  if (b < 0) return;
  const Rows seq = mine.seq;
  const int total = seq.count * a.group, row0 = tile * kTileRows;
  const int p0 = part * a.tile_part;
  const int t_last = (min(row0 + kTileRows, total) - 1) / a.group;
  if (seq.cut && tid == 0 && part == 0 && tile == 0) raise_status(a.status, HEXKV_STATUS_LENGTH_CLAMPED);
  const int end = min(seq.keys(a, t_last), p0 + a.tile_part);
  if (part > 0 && end <= p0) return;

  // This wave's rows and this lane's; rows past the last repeat it.  A wave
  // without rows only stages.
  const int wrow0 = row0 + wave * kWaveRows;
  const bool idle = wrow0 >= total, live = wrow0 + c < total;
  const int row = min(wrow0 + c, total - 1), t = row / a.group, qh = hk * a.group + row - t * a.group;
  const int len = seq.keys(a, t), lim = min(len, p0 + a.tile_part);
  const int w_end = idle ? p0 : min(seq.keys(a, (min(wrow0 + 32, total) - 1) / a.group), p0 + a.tile_part);
  const int w_full = idle ? p0 : min(seq.keys(a, wrow0 / a.group), p0 + a.tile_part);
  const T *q_row = static_cast<const T *>(a.q) + (seq.first + t) * a.q_stride + static_cast<int64_t>(qh) * D;
  u32x4 qf[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) qf[j] = *reinterpret_cast<const u32x4 *>(q_row + h * 8 + j * 16);

  constexpr int ES = static_cast<int>(sizeof(T));
  const char *head = static_cast<const char *>(a.pages) + hk * a.p.head_stride * ES;
  const int64_t kv_bytes = a.p.kv_stride * ES;
  const ScalarTable table = scalar_table(a, b);
  int bad_pages = 0;
  // A wave moves the tile's block of 16 rows of its own, which lie in one page:
  // lane l chunk l % CH of rows l / CH + i * RPL.
  constexpr int RPL = 64 / CH, NL = 16 / RPL;
  const uint32_t pos_bytes = a.pos_bytes;
  const uint32_t lane_at = (lane / CH) * pos_bytes + 16 * (lane % CH);
  const int s_row = 16 * wave + lane / CH;
  const uint32_t k_write = s_row * KP + (lane % CH) * 16, v_write = s_row * VP + (lane % CH) * 16;
  u32x4 kr[NL], vr[NL];
  int page;
  auto find = [&](int k0) { page = table[min((k0 + 16 * wave) >> a.p.shift, a.p.width - 1)]; };
  auto fetch = [&](int k0) {
    const bool in_pool = static_cast<unsigned>(page) < static_cast<unsigned>(a.p.n_pages);
    const int k = k0 + 16 * wave;
    bad_pages |= !in_pool && k < end;
    const char *at = head + block_offset(a, in_pool ? page : 0, k);
    const __amdgpu_buffer_rsrc_t bk = block_of<D * ES>(at, end - k, pos_bytes), bv = block_of<D * ES>(at + kv_bytes, end - k, pos_bytes);
#pragma unroll
    for (int i = 0; i < NL; ++i) kr[i] = load_16<0>(bk, lane_at + i * RPL * pos_bytes);
#pragma unroll
    for (int i = 0; i < NL; ++i) vr[i] = load_16<0>(bv, lane_at + i * RPL * pos_bytes);
  };
  auto stage = [&](int buf) {
    char *to_k = s_k + (k_write + (buf ? KT * KP : 0)), *to_v = s_v + (v_write + (buf ? KT * VP : 0));
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4 *>(to_k + i * RPL * KP) = kr[i];
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<u32x4 *>(to_v + i * RPL * VP) = vr[i];
  };

  float m = -INFINITY, l = 0.f;  // m: the running maximum less kShift
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
  const uint32_t k_read = static_cast<uint32_t>(c * KP + h * 16);
  const int s16 = lane & 15;
  const uint32_t v_read = static_cast<uint32_t>((4 * h + s16 / 4) * VP + ((lane >> 4) & 1) * 32 + (s16 % 4) * 8);

  // A step, of the keys at k0, which are the LDS buffers' rows from `row` on: their
  // scores, their probabilities, the sums of V.
  f32x16 s[NKB];
  u32x4 hi[2 * NKB], lo[2 * NKB];
  auto scores = [&](int row) {
    const char *from_k = s_k + (k_read + row * KP);
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) s[kb] = f32x16{};
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
        s[kb] = M::mma32(*reinterpret_cast<const u32x4 *>(from_k + kb * 32 * KP + j * 32), qf[j], s[kb]);
  };
  auto weigh = [&](int k0) {
    if (k0 + kStepKeys > w_full) {
      const int left = lim - k0 - 4 * h;
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = kb * 32 + 8 * (i / 4) + i % 4 < left ? s[kb][i] : -INFINITY;
    }
    float mt = s[0][0];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[kb][i]);
    mt = xor_step<32>(mt, MaxOp{}) * a.scale_log2;
    const bool up = mt > m + (M::kShift + M::kSlack);
    if (__any(up)) {
      const float mnew = up ? mt - M::kShift : m;
      const float f = up ? exp2_of(m - mnew) : 1.f;
      m = mnew;
      l *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= f;
    }
    const float base = m == -INFINITY ? 0.f : -m;
    float l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float e0 = exp2_of(fmaf(s[kb][i], a.scale_log2, base)), e1 = exp2_of(fmaf(s[kb][i + 1], a.scale_log2, base));
        l0 += e0;
        l1 += e1;
        unsigned int x, y;
        M::split(e0, e1, &x, &y);
        hi[2 * kb + i / 8][i % 8 / 2] = x;
        lo[2 * kb + i / 8][i % 8 / 2] = y;
      }
    l += l0 + l1;
  };
  auto values = [&](int row) {
    auto *from_v = (__attribute__((address_space(3))) char *)s_v + (v_read + row * VP);
#pragma unroll
    for (int ks = 0; ks < 2 * NKB; ++ks)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const h4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_h4 *)(from_v + ks * 16 * VP + d * 64));
        const h4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_h4 *)(from_v + ks * 16 * VP + d * 64 + 8 * VP));
        const u32x4 v = __builtin_bit_cast(u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        acc[d] = M::mma32(v, hi[ks], acc[d]);
        acc[d] = M::mma32(v, lo[ks], acc[d]);
      }
  };

  if (tid == 0) s_bad = 0;
  if (end > p0) {
    find(p0);
    fetch(p0);
    find(p0 + KT);
    stage(0);
    __syncthreads();
    if constexpr (W == 4) {
      int buf = 0;
      for (int k0 = p0; k0 < end; k0 += KT) {
        const bool more = k0 + KT < end;
        if (more) {
          fetch(k0 + KT);
          find(k0 + 2 * KT);
        }
        if (k0 < w_end) {
          scores(buf * KT);
          order_reads<4>();
          repeat<NKB * NJ - 4>([] { order_products<1>(), order_reads<1>(); });
          order_products<4>();
          weigh(k0);
          values(buf * KT);
          order_reads<2 * ND>();
          repeat<(2 * NKB - 1) * ND>([] { order_products<2>(), order_reads<2>(); });
          order_products<2 * ND>();
        }
        if (more) stage(buf ^ 1);
        buf ^= 1;
        __syncthreads();
      }
    } else {
      // Waves w and w + 4 share a SIMD.  The second four run one phase behind, so that
      // one of the two is at its products while the other is at its softmax (429 us for
      // 495 with all in step):
      // phase 2 i: products of step i (the last step's V, this one's scores), 2 i + 1: its
      // softmax.  A tile is two steps; the next is staged with its second step's
      // products, by when both halves are done with the buffer's V (in phases 4 t and 4 t +
      // 1 of tile t), and before either reads it (from 4 t + 4 on).  All waves take all
      // steps, as keys past a row's last weigh nothing.
      const bool behind = wave >= W / 2;
      if (behind) meet();
      if (p0 + KT < end) {
        fetch(p0 + KT);
        find(p0 + 2 * KT);
      }
      scores(0);
      meet();
      weigh(p0);
      meet();
      int row = 0;
#pragma unroll 1
      for (int k0 = p0 + kStepKeys; k0 < end; k0 += kStepKeys) {
        const int last = row;
        row = row + kStepKeys == 2 * KT ? 0 : row + kStepKeys;
        const bool first = row % KT == 0;
        const int next = k0 - row % KT + KT;  // the next tile
        if (first && next < end) {
          fetch(next);
          find(next + KT);
        }
        values(last);
        scores(row);
        order_reads<2 * ND>();
        repeat<(2 * NKB - 1) * ND>([] { order_reads<2>(), order_products<2>(); });
        repeat<NKB * NJ>([] { order_reads<1>(), order_products<1>(); });
        order_products<2 * ND>();
        if (!first && next < end) stage(row < KT);
        meet();
        weigh(k0);
        meet();
      }
      values(row);
      if (!behind) meet();
    }
  }
  if (bad_pages && lane == 0) {
    s_bad = 1;
    raise_status(a.status, HEXKV_STATUS_PAGE);
  }
  __syncthreads();
  if (idle) return;

  l = xor_step<32>(l, AddOp{});
  const bool holds = live && (part == 0 || lim > p0);  // this lane's row has something to write
  float check = l * 0.f;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) check = fmaf(acc[d][i], 0.f, check);
  // Decided for the row, over both lanes that hold its outputs, before either
  // stores: out may be q, and exact_row reads the row's query again.
  uint64_t redo = __ballot(holds && lim > p0 && (s_bad || !(check == 0.f)));
  redo = (redo | redo >> 32) & 0xffffffffu;
  const bool split = len > a.tile_part;
  T *out = static_cast<T *>(a.out) + (seq.first + t) * a.o_stride + static_cast<int64_t>(qh) * D;
  const int64_t slot = (static_cast<int64_t>(seq.first + t) * a.q_heads + qh) * a.tile_parts + part;
  if (holds && !(redo >> c & 1)) {
    if (!split) {
      const float inv = weight_of(l);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 o = {acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
          store4(out + d * 32 + i * 8 + 4 * h, len > 0 ? o * inv : f32x4{});
        }
    } else {
      float *o = a.ws_tile_o + slot * D + 4 * h;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4 *>(o + d * 32 + i * 8) =
              f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
      if (h == 0) *reinterpret_cast<float2 *>(a.ws_tile_ml + slot * 2) = float2{m, l};
    }
  }
  while (redo) {
    const int r = __builtin_ctzll(redo);
    redo &= redo - 1;
    constexpr int DPL = D / 64;
    const int tr = __shfl(t, r), hr = __shfl(qh, r);
    const bool row_split = __shfl(static_cast<int>(split), r);
    float em, el, eo[DPL];
    exact_row<T, D>(a, static_cast<const T *>(a.q) + (seq.first + tr) * a.q_stride + static_cast<int64_t>(hr) * D, b, hk, p0,
                    __shfl(lim, r), &em, &el, eo);
    const int64_t to = (static_cast<int64_t>(seq.first + tr) * a.q_heads + hr) * a.tile_parts + part;
    T *row_out = static_cast<T *>(a.out) + (seq.first + tr) * a.o_stride + static_cast<int64_t>(hr) * D + lane * DPL;
#pragma unroll
    for (int e = 0; e < DPL; ++e) {
      if (row_split) a.ws_tile_o[to * D + lane * DPL + e] = eo[e];
      else row_out[e] = Elem<T>::from_float(eo[e] * weight_of(el));
    }
    if (row_split && lane == 0) *reinterpret_cast<float2 *>(a.ws_tile_ml + to * 2) = float2{em, el};
  }
}

template <typename T, int D>
constexpr bool has_tiles() {
  return !std::is_same<T, float>::value && D >= 64;
}

// (Three waves a SIMD, where the registers allow: fp32 heads of 128 spill at three, 105
// us for 11 sequences of up to 4200 keys on 8 KV heads, and take 40 at two.)
template <typename T, int D>
__global__ __launch_bounds__(256, D > 128 ? 1 : D * sizeof(T) > 256 ? 2 : 3) void paged_rows_kernel(const PagedAttendArgs a) {
  __shared__ __attribute__((aligned(16))) char s_mem[rows_lds<T, D, 4>()];
  rows_path<T, D, 4>(a, blockIdx.x, s_mem);
}

template <typename T, int D, int W>
__global__ __launch_bounds__(W * 64, D > 128 ? 1 : 2) void paged_tile_kernel(const PagedAttendArgs a) {
  __shared__ __attribute__((aligned(16))) char s_mem[TileLds<D, W>::kBytes];
  tile_path<T, D, W>(a, blockIdx.x, s_mem);
}

// A call that may hold sequences of either kind: tiles first (they take longest).
template <typename T, int D, int W>
__global__ __launch_bounds__(W * 64, D > 128 ? 1 : 2) void paged_mixed_kernel(const PagedAttendArgs a) {
  constexpr int kRows = rows_lds<T, D, W>(), kTiles = TileLds<D, W>::kBytes;
  __shared__ __attribute__((aligned(16))) char s_mem[kRows > kTiles ? kRows : kTiles];
  const int block = blockIdx.x;
  if (block < a.tile_blocks) tile_path<T, D, W>(a, block, s_mem);
  else rows_path<T, D, W>(a, block - a.tile_blocks, s_mem);
}

// The partitions of a split row, joined: a wave a row.
constexpr int kJoinThreads = 256;
constexpr int kMaxParts = 512;

// Sums are taken with the maximum as it rises, so that a row of up to kDepth
// partitions waits for memory once.
template <typename T, int D>
__device__ __forceinline__ void join_row(const float *o_parts, const float *ml_parts, int parts, T *out) {
  const int lane = threadIdx.x & 63;
  constexpr int DPL = D >= 64 ? D / 64 : 1;
  typedef float vd __attribute__((ext_vector_type(DPL)));
  const int at = D >= 64 ? lane * DPL : lane & (D - 1);
  vd o = {};
  float top = -INFINITY, sum = 0.f;
  constexpr int kDepth = 8;  // parts in flight
  for (int p0 = 0; p0 < parts; p0 += kDepth) {
    vd v[kDepth];
    float2 ml[kDepth];
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      const int p = min(p0 + k, parts - 1);
      v[k] = *reinterpret_cast<const vd *>(o_parts + p * D + at);
      ml[k] = *reinterpret_cast<const float2 *>(ml_parts + p * 2);
    }
    float now = top;
#pragma unroll
    for (int k = 0; k < kDepth; ++k) now = fmaxf(now, ml[k].x);
    const float before = top == -INFINITY ? 0.f : exp2_of(top - now);
    top = now;
    o *= before;
    sum *= before;
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      // (copies of the last are left out, not weighed by 0, which makes a NaN of an infinite sum)
      const bool part = p0 + k < parts;
      const float w = !part || ml[k].x == -INFINITY ? 0.f : exp2_of(ml[k].x - top);
      o += part ? v[k] * w : vd{};
      sum = part ? fmaf(ml[k].y, w, sum) : sum;
    }
  }
  const float inv = weight_of(sum);
  if (lane * DPL >= D) return;
#pragma unroll
  for (int e = 0; e < DPL; ++e) out[at + e] = Elem<T>::from_float(o[e] * inv);
}

// Rows that are numbered by sequence and KV head first (`few` of them), then those that are by token
// and head.
template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(const PagedAttendArgs a, int few) {
  int id = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x * (kJoinThreads / 64) + (threadIdx.x >> 6)));
  int b, hk, row, t, qh;
  Rows seq;
  if (id < few) {
    const int pair = id / a.pair_rows;
    row = id - pair * a.pair_rows;
    b = pair / a.kv_heads;
    hk = pair - b * a.kv_heads;
    seq = rows_of(a, b);
    t = row / a.group;
    qh = hk * a.group + row - t * a.group;
    if (seq.count * a.group > a.few_rows) return;
  } else {
    id -= few;
    const int token = id / a.q_heads;
    if (token >= a.p.tokens) return;
    qh = id - token * a.q_heads;
    b = a.p.cu ? token_sequence(a.p, token) : token / a.p.each;
    if (b < 0) return;
    seq = rows_of(a, b);
    t = token - seq.first;
    hk = qh / a.group;
    row = t * a.group + qh - hk * a.group;
    if (a.pair_rows && seq.count * a.group <= a.few_rows) return;
  }
  if (t >= seq.count) return;
  const bool tile = seq.count * a.group > a.few_rows;
  const int len = seq.keys(a, t), part = tile ? a.tile_part : a.part;
  if (len <= part) return;
  const int64_t slot = tile ? (static_cast<int64_t>(seq.first + t) * a.q_heads + qh) * a.tile_parts
                            : few_slot(a, b, hk, row, seq.first, t, qh) * a.max_parts;
  join_row<T, D>((tile ? a.ws_tile_o : a.ws_o) + slot * D, (tile ? a.ws_tile_ml : a.ws_ml) + slot * 2, (len + part - 1) / part,
                 static_cast<T *>(a.out) + (seq.first + t) * a.o_stride + static_cast<int64_t>(qh) * D);
}

// ------------------------------------------------------------------ host ---

static int64_t ceil_div(int64_t n, int64_t by) { return (n + by - 1) / by; }
static int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Keys of a tile's partition.  A split fills the CUs evenly, and costs sums that
// are written, read and joined.  A step of 64 keys (D = 128) takes a CU 1.89 us
// for a lone tile of 128 rows, 3.0 for two at once, 2.68 for one of 256; with D = 64 0.62 of
// that, with 256 (one at a time) 1.64; a partition's sums 0.026 us per 128 rows, the join 5.  With those, the least of
// whole rows and of partitions that fill all CUs once to eight times: 512 rows of
// 4 heads over 8192 keys on 8 KV heads 111 us in 4, 153 in 2, 120 in 8, 266 whole; 1100 rows
// over 31100 keys 793 for 986 whole; 1024 over 4096 111 in two, 138 whole; 250 rows of 8 heads on
// one over 1050 keys 18.7 in partitions of 256, 23.6 of 512, 32.9 whole.  From two
// tiles a CU on, causal rows' lengths even out by themselves (2500 rows over 4000
// keys 190 whole, in two 248).
static int64_t tile_partition(int64_t tiles, int64_t keys, int d, bool wide) {
  if (tiles >= 2 * kCus) return std::max<int64_t>(64, round_up(keys, 64));
  const auto time = [&](int64_t parts) {
    const int64_t steps = ceil_div(keys, 64 * parts) + 1, each = ceil_div(tiles * parts, kCus);
    return steps * (wide ? each * 268 : d > 128 ? each * 189 : each / 2 * 300 + each % 2 * 189) * (d + 64) / 192 +
           (parts > 1 ? 500 + tiles * parts * (wide ? 52 : 26) * d / 1280 : 0);
  };
  int64_t best = 1, least = time(1);
  for (int64_t fill = 1; fill <= 8; ++fill) {
    const int64_t parts = std::min(fill * kCus / std::max<int64_t>(tiles, 1), keys / 192);
    if (parts < 2) continue;
    const int64_t t = time(parts);
    if (t < least) least = t, best = parts;
  }
  return std::max<int64_t>(64, round_up(ceil_div(keys, best), 64));
}

// Rows of either path that may be split.
static int64_t split_few(const PagedAttendArgs &a) {
  if (a.max_parts <= 1) return 0;
  return a.pair_rows ? static_cast<int64_t>(a.p.batch) * a.kv_heads * a.pair_rows : static_cast<int64_t>(a.p.tokens) * a.q_heads;
}
static int64_t split_tiled(const PagedAttendArgs &a) {
  return a.tile_parts > 1 ? static_cast<int64_t>(a.p.tokens) * a.q_heads : 0;
}
// Waves of the join: those numbered by sequence, and those by token.
static int64_t joined_pairs(const PagedAttendArgs &a) { return a.pair_rows ? split_few(a) : 0; }
static int64_t joined_tokens(const PagedAttendArgs &a) { return a.pair_rows ? split_tiled(a) : std::max(split_few(a), split_tiled(a)); }

// Checks a call and fills its arguments but for addresses.
static int fill_attend(const hexkv_paged_attend_params *params, PagedAttendArgs *a, const char *what) {
  if (!params) return fail(HEXKV_EINVAL, "%s: null argument", what);
  const hexkv_paged_attend_params &p = *params;
  int rc = fill_tables(p.pool, p.seqs, &a->p, what);
  if (rc != HEXKV_OK) return rc;
  const int d = p.pool.head_dim, vec = 16 / elem_bytes(p.pool.dtype);
  if (p.q_heads < 1 || p.q_heads > 1 << 16 || p.q_heads % p.pool.kv_heads)
    return fail(HEXKV_EINVAL, "%s: %d query heads on %d KV heads", what, p.q_heads, p.pool.kv_heads);
  a->scale_log2 = p.softmax_scale * 1.44269504f;
  if (!(p.softmax_scale > 0.f) || a->scale_log2 > 3e38f)
    return fail(HEXKV_EINVAL, "%s: softmax_scale is not positive, or above 2e38", what);
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
  a->page_bytes = static_cast<uint32_t>(p.pool.page_stride * elem_bytes(p.pool.dtype));
  a->pos_bytes = static_cast<uint32_t>(p.pool.pos_stride * elem_bytes(p.pool.dtype));
  const int64_t rows = static_cast<int64_t>(a->max_tokens) * a->group;
  if (rows > INT32_MAX - 256) return fail(HEXKV_ERANGE, "%s: 2^31 rows or more", what);
  // Which paths can have work: without cu_tokens every sequence has as many rows.
  // Heads of 256 leave a CU one tile, of four waves (tokens of 8 heads on one, us on tiles and on rows): 2048 over
  // 8048 keys 220 and 743, 16 x 40 over 4000 94 and 130; at the border 16 x 40 over 240 24 and 27, 100 over 1300 28 and 28,
  // 150 over 950 28 and 21; 40 over 1040 26 and 16.
  const bool tiled = p.pool.dtype != HEXKV_F32 && rows > kFewRows &&
                     (d == 64 || d == 128 || (d == 256 && static_cast<double>(tokens) * p.q_heads * p.max_seqlen >= 1 << 20));
  // Tiles of 256 rows read LDS and pages half as often, but one alone has a CU to
  // itself from its first key to its last: chunks of 2048 over 8192 keys (32 heads
  // on 8) 429 us for 461 with 128, of 512 114 for 124, of 8192 from the first key on 736 for 777; at the
  // borders 128 tokens (512 rows of a KV head) over 8128 keys 43 for 42, 2048 over 3548 146 for 145 and
  // over 4108 170 for 172; yet 2048 from the first key on 80 for 71, 64 (256 rows) over 8064
  // 35 for 29.  Workgroups of few rows are then one a CU too, so a call of more
  // than four ragged sequences, which may be single tokens, keeps 128: a chunk of
  // 2000 and 64 single tokens 478 us, with 256 rows a tile 534; 500 of 8 heads and 20 single ones 42, 56
  // (and 3 single ones 41, 46; 2000 of 32 heads and 3 352, 336).
  a->wide = tiled && d == 128 && rows >= 512 && p.max_seqlen >= 4096 && (!p.seqs.cu_tokens || p.seqs.batch <= 4);
  const int64_t tile_rows = a->wide ? 256 : 128;
  const bool few = !tiled || p.seqs.cu_tokens;
  a->few_rows = tiled ? kFewRows : INT32_MAX;
  a->row_tiles = few ? static_cast<int32_t>((std::min<int64_t>(rows, a->few_rows) + 15) / 16) : 0;
  // Tiles of all sequences: without cu_tokens as they are, else at most one a
  // sequence more than full ones, of sequences with enough rows to have any.
  const int64_t batch = p.seqs.batch, all_rows = tokens * a->group;
  int64_t few_tiles = batch * a->row_tiles, tiles = tiled ? batch * ((rows + tile_rows - 1) / tile_rows) : 0;
  if (p.seqs.cu_tokens) {
    few_tiles = std::min(few_tiles, all_rows / 16 + std::min<int64_t>(batch, tokens));
    tiles = std::min(tiles, all_rows / tile_rows + std::min<int64_t>(batch, all_rows / (kFewRows + 1)));
  }
  if ((few_tiles + tiles) * a->kv_heads >= INT64_C(1) << 24) return fail(HEXKV_ERANGE, "%s: 2^24 workgroups or more", what);
  // Partitions.  A CU alone takes 55 GB/s whatever its waves, so a row's keys are spread
  // over CUs, but for those of up to 128 KB of K, which end before a second
  // launch would have joined them (a step of 128 keys of 128 16-bit dims takes 1.15 us, the
  // join 2.7): one workgroup a CU where that leaves it 2048 keys or fewer, else
  // partitions of 1024 keys, which even out ragged lengths (us, MI355X, 16-bit heads
  // of 128: 8 pairs of 1024 keys 8.5 split in 8, 12.9 whole, of 512 8.2 and 8.6; 32 pairs of 4096
  // keys 19.5, 17.0, 16.5, 18.2, 26.3 and 40 in partitions of 128, 256, 512, 1024, 2048 and
  // whole; 512 ragged ones of up to 8192 191, 181, 177, 193 and 200 from 256 on).  More than half a
  // workgroup a CU are not split for that: 144 pairs of 1100 keys 16.5 whole, 17.5 in
  // partitions of 256, 19.2 of 512, 21.6 of 640; of up to 2000, 24 whole, 22 to 27 split.
  const int64_t pairs = few_tiles * a->kv_heads;
  const int64_t each = 2 * pairs > kCus ? p.max_seqlen : std::max<int64_t>(128, round_up(ceil_div(pairs * p.max_seqlen, kCus), 128));
  int64_t part = p.partition ? p.partition : each <= 2048 ? std::max<int64_t>(each, 64) : 1024;
  if (!p.partition && part < p.max_seqlen) {
    // of one length, and where they save more than the join takes
    part = round_up(ceil_div(p.max_seqlen, ceil_div(p.max_seqlen, part)), 128);
    const int64_t key = static_cast<int64_t>(d) * elem_bytes(p.pool.dtype);
    if (p.max_seqlen * key <= 128 << 10 || (p.max_seqlen - part) * key <= 96 << 10) part = 1 << 30;
  }
  part = std::max(part, round_up((p.max_seqlen + kMaxParts - 1) / kMaxParts, 128));
  a->part = static_cast<int32_t>(std::min<int64_t>(part, 1 << 30));
  a->max_parts = static_cast<int32_t>(std::max<int64_t>(1, (p.max_seqlen + part - 1) / part));
  // Of ragged sequences, all but one taken for single tokens.
  const int64_t long_rows = p.seqs.cu_tokens ? (std::max(tokens - batch, INT64_C(0)) + 1) * a->group : 0;
  const int64_t full = (p.seqs.cu_tokens ? ceil_div(long_rows, tile_rows) : tiles) * a->kv_heads;
  part = p.partition ? p.partition : tile_partition(full, p.max_seqlen, d, a->wide);
  part = std::max(part, round_up((p.max_seqlen + kMaxParts - 1) / kMaxParts, 64));
  a->tile_part = static_cast<int32_t>(std::min<int64_t>(part, 1 << 30));
  a->tile_parts = static_cast<int32_t>(std::max<int64_t>(1, (p.max_seqlen + part - 1) / part));
  // Where the tokens are so many that each sequence is a long one, unless some
  // are left out, what few rows there may be are not split: no join is launched for
  // them (5 us).
  if (!few || (tiled && (tokens - (batch - 1) * a->max_tokens) * a->group > kFewRows)) {
    a->part = 1 << 30;
    a->max_parts = 1;
  }
  if (!tiled) a->tile_parts = 1;
  // The row path's split rows by sequence, with room for the longest of them, or by token,
  // with room for all: a chunk beside many single tokens (fp32, 32 heads on 8, 2048 tokens beside 63)
  // has 67 552 rows, which by sequence would take 4.2 million places.
  const int64_t by_token = tokens * p.q_heads, most = std::min<int64_t>(rows, a->few_rows);
  a->pair_rows = batch * p.pool.kv_heads <= by_token && batch * p.pool.kv_heads * most <= by_token ? static_cast<int32_t>(most) : 0;
  if (joined_pairs(*a) + joined_tokens(*a) >= INT64_C(1) << 26) return fail(HEXKV_ERANGE, "%s: 2^26 split rows or more", what);
  const int64_t row_blocks = few_tiles * a->kv_heads * a->max_parts, tile_blocks = tiles * a->kv_heads * a->tile_parts;
  if ((row_blocks + tile_blocks) * (a->wide ? 512 : 256) >= INT64_C(1) << 32)
    return fail(HEXKV_ERANGE, "%s: workgroups of 2^32 lanes or more", what);
  a->row_blocks = static_cast<int32_t>(row_blocks);
  a->tiles = static_cast<int32_t>(tiles);
  a->tile_blocks = static_cast<int32_t>(tile_blocks);
  return HEXKV_OK;
}

// ... each with its partitions' slots.
static int64_t few_slots(const PagedAttendArgs &a) { return split_few(a) * a.max_parts; }
static int64_t tile_slots(const PagedAttendArgs &a) { return split_tiled(a) * a.tile_parts; }

static size_t attend_workspace(const PagedAttendArgs &a, int head_dim) {
  return static_cast<size_t>(few_slots(a) + tile_slots(a)) * (head_dim + 2) * sizeof(float);
}

template <typename T, int D>
static void launch_attend(const PagedAttendArgs &a, hipStream_t s) {
  const unsigned rows = static_cast<unsigned>(a.row_blocks);
  const unsigned tiles = static_cast<unsigned>(a.tile_blocks);
  if constexpr (has_tiles<T, D>()) {
    if constexpr (D == 128) {
      if (a.wide && rows) paged_mixed_kernel<T, D, 8><<<dim3(rows + tiles), 512, 0, s>>>(a);
      else if (a.wide) paged_tile_kernel<T, D, 8><<<dim3(tiles), 512, 0, s>>>(a);
    }
    if (tiles && rows && !a.wide) paged_mixed_kernel<T, D, 4><<<dim3(rows + tiles), 256, 0, s>>>(a);
    else if (tiles && !a.wide) paged_tile_kernel<T, D, 4><<<dim3(tiles), 256, 0, s>>>(a);
  }
  if (!tiles) paged_rows_kernel<T, D><<<dim3(rows), 256, 0, s>>>(a);
  const int64_t few = joined_pairs(a), joined = few + joined_tokens(a);
  if (joined)
    paged_join_kernel<T, D><<<dim3(static_cast<unsigned>((joined + 3) / 4)), kJoinThreads, 0, s>>>(a, static_cast<int>(few));
}

template <typename T>
static void launch_dims(const PagedAttendArgs &a, int head_dim, hipStream_t s) {
  switch (head_dim) {
    case 16: launch_attend<T, 16>(a, s); break;
    case 32: launch_attend<T, 32>(a, s); break;
    case 64: launch_attend<T, 64>(a, s); break;
    case 128: launch_attend<T, 128>(a, s); break;
    default: launch_attend<T, 256>(a, s); break;
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
  const int d = params->pool.head_dim, es = elem_bytes(params->pool.dtype);
  // A workgroup reads its rows of q before it writes them: out may be q, or lie
  // beside it in the same rows, but not over other rows' q.
  const int64_t row = static_cast<int64_t>(a.q_heads) * d, last = a.p.tokens - 1;
  const int64_t q_bytes = (last * a.q_stride + row) * es, o_bytes = (last * a.o_stride + row) * es, pool = pool_bytes(params->pool);
  if (overlap(a.out, o_bytes, a.q, q_bytes) && (last || a.out != a.q)) {
    const int64_t step = a.q_stride * es, apart = static_cast<const char *>(a.out) - static_cast<const char *>(a.q);
    const int64_t shift = last ? (apart % step + step) % step : 0;
    if (!last || a.q_stride != a.o_stride || (apart && (shift < row * es || step - shift < row * es)))
      return fail(HEXKV_EINVAL, "%s: out overlaps other rows of q", what);
  }
  if (overlap(a.out, o_bytes, a.pages, pool)) return fail(HEXKV_EINVAL, "%s: out overlaps the pages", what);
  const size_t need = attend_workspace(a, d);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(HEXKV_EWORKSPACE, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", what, need, workspace_bytes);
  if (overlap(workspace, need, a.q, q_bytes) || overlap(workspace, need, a.out, o_bytes) || overlap(workspace, need, a.pages, pool))
    return fail(HEXKV_EINVAL, "%s: the workspace overlaps a tensor", what);
  if (need) {
    const int64_t few = few_slots(a), tile = tile_slots(a);
    a.ws_o = static_cast<float *>(workspace);
    a.ws_tile_o = a.ws_o + few * d;
    a.ws_ml = a.ws_tile_o + tile * d;
    a.ws_tile_ml = a.ws_ml + few * 2;
  } else {
    a.ws_o = a.ws_ml = a.ws_tile_o = a.ws_tile_ml = nullptr;
  }
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
