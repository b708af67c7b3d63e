// Rows into the 4-bit block format and back: hexkv_mx_store, hexkv_mx_load
// (K/V rows of a cache), hexkv_mx_quantize and hexkv_mx_dequantize (the rows of
// a matrix).
//
// What bounds them: memory, every element read once and written once, 2 or 4
// bytes on one side and 17/32 on the other.  A lane takes 8 elements (one or two
// 16-byte vectors) and four lanes a block, whose largest magnitude they
// exchange by DPP; a wave then reads 1 KB (16-bit data) and writes 256 bytes
// of elements in one piece, beside 16 powers.
#include "hexkv_mx.h"

namespace hexkv {

constexpr int kMxThreads = 256;

// Rows of `groups` groups of 8 elements: row r is position r % seqlen of
// sequence r / seqlen.  The first half of a row's groups starts at the row, the
// second `half_stride` elements behind it (K and V; a matrix row is one
// half).  On the 4-bit side a row holds 4 bytes a group, then a byte per
// four groups, at codes / powers + sequence and position strides.
struct MxRowsArgs {
  const void *x;
  int64_t x_bs, x_ps, x_hs;  // elements
  unsigned char *codes, *powers;
  int64_t c_bs, c_ps, p_bs, p_ps;  // bytes
  int32_t seqlen, groups, half;    // half: groups of the first half
  int64_t rows, capacity;
  const int32_t *positions;
  int32_t bias;
  int32_t rows_per_wg, chunks;  // one of them 1
  unsigned int *status;
};

struct MxPlace {
  int64_t b, s, at;
  int group;
  bool live;
};

// This lane's sequence, position within the call, cache position and group.
// Lanes of a block share a row (groups is a multiple of 4), so they are live
// together.
__device__ __forceinline__ MxPlace mx_place(const MxRowsArgs &a, unsigned int flag) {
  MxPlace p;
  int64_t row;
  if (a.chunks > 1) {
    row = blockIdx.x / static_cast<unsigned>(a.chunks);
    p.group = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.chunks)) * kMxThreads + static_cast<int>(threadIdx.x);
    p.live = p.group < a.groups;
  } else {
    const int r = static_cast<int>(threadIdx.x / static_cast<unsigned>(a.groups));
    row = static_cast<int64_t>(blockIdx.x) * a.rows_per_wg + r;
    p.group = static_cast<int>(threadIdx.x) - r * a.groups;
    p.live = r < a.rows_per_wg && row < a.rows;
  }
  if (!p.live) row = 0;
  p.b = static_cast<int64_t>(static_cast<unsigned>(row) / static_cast<unsigned>(a.seqlen));
  p.s = row - p.b * a.seqlen;
  p.at = p.s + a.bias;
  if (a.positions) p.at += a.positions[p.b];
  if (p.live && (p.at < 0 || p.at >= a.capacity)) {
    if (p.group == 0) raise_status(a.status, flag);
    p.at = -1;
  }
  return p;
}

template <typename T>
__device__ __forceinline__ int64_t mx_element(const MxRowsArgs &a, const MxPlace &p) {
  const bool second = p.group >= a.half;
  return p.b * a.x_bs + p.s * a.x_ps + (second ? a.x_hs : 0) + static_cast<int64_t>(p.group - (second ? a.half : 0)) * 8;
}

template <typename T>
__global__ __launch_bounds__(kMxThreads) void mx_store_kernel(const MxRowsArgs a, bool vec) {
  const MxPlace p = mx_place(a, HEXKV_STATUS_APPEND_SKIPPED);
  if (!p.live || p.at < 0) return;
  float f[8];
  mx_read8(static_cast<const T *>(a.x) + mx_element<T>(a, p), vec, f);
  const unsigned int byte = mx_power(mx_block_bits(mx_bits(f)));
  *reinterpret_cast<unsigned int *>(a.codes + p.b * a.c_bs + p.at * a.c_ps + p.group * 4) = mx_encode(f, byte);
  if (p.group % 4 == 0) a.powers[p.b * a.p_bs + p.at * a.p_ps + p.group / 4] = static_cast<unsigned char>(byte);
}

template <typename T>
__global__ __launch_bounds__(kMxThreads) void mx_load_kernel(const MxRowsArgs a, bool vec) {
  const MxPlace p = mx_place(a, HEXKV_STATUS_LOAD_SKIPPED);
  if (!p.live) return;
  float f[8] = {};
  if (p.at >= 0) {
    const unsigned int w = *reinterpret_cast<const unsigned int *>(a.codes + p.b * a.c_bs + p.at * a.c_ps + p.group * 4);
    mx_f32(w, mx_scale(a.powers[p.b * a.p_bs + p.at * a.p_ps + p.group / 4]), f);
  }
  mx_write8(static_cast<T *>(const_cast<void *>(a.x)) + mx_element<T>(a, p), vec, f);
}

template <bool STORE>
static int mx_rows(MxRowsArgs a, int dtype, hexkv_stream_t stream, const char *what) {
  if (a.rows == 0 || a.groups == 0) return HEXKV_OK;
  if (a.rows >= INT64_C(1) << 31) return fail(HEXKV_ERANGE, "%s: 2^31 rows or more", what);
  a.rows_per_wg = a.groups < kMxThreads ? kMxThreads / a.groups : 1;
  a.chunks = (a.groups + kMxThreads - 1) / kMxThreads;
  const int64_t wgs = a.chunks > 1 ? a.rows * a.chunks : (a.rows + a.rows_per_wg - 1) / a.rows_per_wg;
  if (wgs >= INT64_C(1) << 24) return fail(HEXKV_ERANGE, "%s: 2^24 workgroups or more; split the call", what);
  const int elem = dtype == HEXKV_F32 ? 4 : 2, per = 16 / elem;
  const bool vec = aligned16(a.x) && a.x_bs % per == 0 && a.x_ps % per == 0 && a.x_hs % per == 0;
  const dim3 grid(static_cast<unsigned>(wgs));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define HEXKV_MX_ROWS(T)                                                                   \
  if constexpr (STORE) mx_store_kernel<T><<<grid, kMxThreads, 0, s>>>(a, vec);             \
  else mx_load_kernel<T><<<grid, kMxThreads, 0, s>>>(a, vec);
  if (dtype == HEXKV_BF16) { HEXKV_MX_ROWS(__bf16) }
  else if (dtype == HEXKV_F16) { HEXKV_MX_ROWS(_Float16) }
  else { HEXKV_MX_ROWS(float) }
#undef HEXKV_MX_ROWS
  return check_launch(what);
}

template <bool STORE>
static int mx_cache_rows(const void *kv, int64_t kv_bs, int64_t kv_ps, int64_t kv_hs, const void *cache,
                         int64_t c_bs, int64_t c_ps, int64_t capacity, int batch, int seqlen, int heads,
                         int head_dim, int dtype, const int32_t *positions, int32_t bias, hexkv_stream_t stream,
                         const char *what) {
  clear_error();
  if (dtype != HEXKV_F16 && dtype != HEXKV_BF16 && dtype != HEXKV_F32)
    return fail(HEXKV_EINVAL, "%s: unknown dtype %d", what, dtype);
  if (batch < 0 || seqlen < 0 || heads < 1) return fail(HEXKV_EINVAL, "%s: bad batch/positions/heads", what);
  if (head_dim < 1 || head_dim % kMxBlock || head_dim > 1024)
    return fail(HEXKV_EUNSUPPORTED, "%s: head_dim %d is not a multiple of %d up to 1024", what, head_dim, kMxBlock);
  if (heads > 65536) return fail(HEXKV_EINVAL, "%s: over 65536 heads", what);
  if (batch == 0 || seqlen == 0) return HEXKV_OK;
  if (!kv || !cache) return fail(HEXKV_EINVAL, "%s: null argument", what);
  if (capacity < 1) return fail(HEXKV_EINVAL, "%s: bad capacity", what);
  if (c_ps < mx_row_bytes(heads, head_dim) || c_ps % 16 || c_bs % 16 || !aligned16(cache) ||
      (batch > 1 && c_bs < capacity * c_ps))
    return fail(HEXKV_EINVAL, "%s: cache rows must be 16-byte aligned, at least %lld bytes apart and sequences "
                              "capacity rows apart", what, static_cast<long long>(mx_row_bytes(heads, head_dim)));
  const int elem = dtype == HEXKV_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(kv) & (elem - 1)) return fail(HEXKV_EINVAL, "%s: kv misaligned", what);
  if (!positions && (bias < 0 || static_cast<int64_t>(bias) + seqlen > capacity))
    return fail(HEXKV_ERANGE, "%s: positions [%d, %lld) outside [0, %lld)", what, bias,
                static_cast<long long>(bias) + seqlen, static_cast<long long>(capacity));
  MxRowsArgs a = {};
  a.x = kv;
  a.x_bs = kv_bs;
  a.x_ps = kv_ps;
  a.x_hs = kv_hs;
  a.codes = static_cast<unsigned char *>(const_cast<void *>(cache));
  a.powers = a.codes + static_cast<int64_t>(heads) * head_dim;  // behind 2 * heads * head_dim / 2 bytes
  a.c_bs = a.p_bs = c_bs;
  a.c_ps = a.p_ps = c_ps;
  a.seqlen = seqlen;
  a.groups = 2 * heads * head_dim / 8;
  a.half = a.groups / 2;
  a.rows = static_cast<int64_t>(batch) * seqlen;
  a.capacity = capacity;
  a.positions = positions;
  a.bias = bias;
  if (positions) {
    const int rc = status_word(stream, &a.status, what);
    if (rc != HEXKV_OK) return rc;
  }
  return mx_rows<STORE>(a, dtype, stream, what);
}

template <bool STORE>
static int mx_matrix_rows(const void *x, int64_t x_stride, const void *codes, const void *powers, int64_t rows,
                          int width, int dtype, hexkv_stream_t stream, const char *what) {
  clear_error();
  if (dtype != HEXKV_F16 && dtype != HEXKV_BF16 && dtype != HEXKV_F32)
    return fail(HEXKV_EINVAL, "%s: unknown dtype %d", what, dtype);
  if (rows < 0 || width < 0) return fail(HEXKV_EINVAL, "%s: negative size", what);
  if (width % kMxBlock) return fail(HEXKV_EINVAL, "%s: rows of %d elements are not whole blocks of %d", what, width, kMxBlock);
  if (rows == 0 || width == 0) return HEXKV_OK;
  if (!x || !codes || !powers) return fail(HEXKV_EINVAL, "%s: null argument", what);
  const int elem = dtype == HEXKV_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x) & (elem - 1)) || (reinterpret_cast<uintptr_t>(codes) & 3))
    return fail(HEXKV_EINVAL, "%s: misaligned tensor", what);
  if (rows > INT32_MAX) return fail(HEXKV_ERANGE, "%s: 2^31 rows or more", what);
  MxRowsArgs a = {};
  a.x = x;
  a.x_ps = x_stride;
  a.codes = static_cast<unsigned char *>(const_cast<void *>(codes));
  a.powers = static_cast<unsigned char *>(const_cast<void *>(powers));
  a.c_ps = width / 2;
  a.p_ps = width / kMxBlock;
  a.seqlen = static_cast<int32_t>(rows);  // one sequence
  a.groups = a.half = width / 8;
  a.rows = a.capacity = rows;
  return mx_rows<STORE>(a, dtype, stream, what);
}

}  // namespace hexkv

extern "C" int hexkv_mx_store(const void *kv, int64_t kv_batch_stride, int64_t kv_pos_stride, int64_t kv_stride,
                              void *cache, int64_t cache_batch_bytes, int64_t cache_row_bytes, int64_t capacity,
                              int batch, int seqlen, int kv_heads, int head_dim, int dtype,
                              const int32_t *positions_dev, int32_t position_bias, hexkv_stream_t stream) {
  return hexkv::mx_cache_rows<true>(kv, kv_batch_stride, kv_pos_stride, kv_stride, cache, cache_batch_bytes,
                                    cache_row_bytes, capacity, batch, seqlen, kv_heads, head_dim, dtype, positions_dev,
                                    position_bias, stream, "hexkv_mx_store");
}

extern "C" int hexkv_mx_load(const void *cache, int64_t cache_batch_bytes, int64_t cache_row_bytes, int64_t capacity,
                             void *kv, int64_t kv_batch_stride, int64_t kv_pos_stride, int64_t kv_stride, int batch,
                             int seqlen, int kv_heads, int head_dim, int dtype, const int32_t *positions_dev,
                             int32_t position_bias, hexkv_stream_t stream) {
  return hexkv::mx_cache_rows<false>(kv, kv_batch_stride, kv_pos_stride, kv_stride, cache, cache_batch_bytes,
                                     cache_row_bytes, capacity, batch, seqlen, kv_heads, head_dim, dtype, positions_dev,
                                     position_bias, stream, "hexkv_mx_load");
}

extern "C" int hexkv_mx_quantize(const void *x, int64_t x_stride, void *codes, void *powers, int64_t rows, int width,
                                 int dtype, hexkv_stream_t stream) {
  return hexkv::mx_matrix_rows<true>(x, x_stride, codes, powers, rows, width, dtype, stream, "hexkv_mx_quantize");
}

extern "C" int hexkv_mx_dequantize(const void *codes, const void *powers, void *out, int64_t out_stride, int64_t rows,
                                   int width, int dtype, hexkv_stream_t stream) {
  return hexkv::mx_matrix_rows<false>(out, out_stride, codes, powers, rows, width, dtype, stream,
                                      "hexkv_mx_dequantize");
}
