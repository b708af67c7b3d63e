// Paged caches: the append that rotates on the way (hexkv_paged_append) and the
// handoff of their live rows (hexkv_paged_pack, hexkv_paged_unpack).
//
// What bounds them: memory.  Every element of a token's q, k and v is read
// once and written once, in 16-byte vectors where its strides allow; a decode
// step's few rows are a launch.  On one MI355X: 8192 tokens of 32 + 2 x 8 heads of 128
// in bf16 (201 MB) 37.6 us, 5.4 TB/s; 64 of them 3.8 us; 32 layers of 8 sequences, 8.2 GB
// gathered at 5.9 and scattered at 5.5 TB/s.
#include "hexkv_paged.h"

#include <algorithm>
#include <memory>
#include <new>

namespace hexkv {

int check_pool(const hexkv_pool &pool, const char *what) {
  if (pool.dtype != HEXKV_F16 && pool.dtype != HEXKV_BF16 && pool.dtype != HEXKV_F32)
    return fail(HEXKV_EINVAL, "%s: unknown dtype %d", what, pool.dtype);
  const int d = pool.head_dim;
  if (d != 16 && d != 32 && d != 64 && d != 128 && d != 256)
    return fail(HEXKV_EUNSUPPORTED, "%s: head_dim %d (16, 32, 64, 128 and 256 are compiled)", what, d);
  if (pool.kv_heads < 1 || pool.kv_heads > 1 << 16) return fail(HEXKV_EINVAL, "%s: %d KV heads", what, pool.kv_heads);
  if (pool.n_pages < 1) return fail(HEXKV_EINVAL, "%s: a pool needs a page", what);
  if (pool.page_size < 16 || pool.page_size > 1 << 20 || (pool.page_size & (pool.page_size - 1)))
    return fail(HEXKV_EINVAL, "%s: page_size %d is not a power of two from 16 to 2^20", what, pool.page_size);
  const int vec = 16 / elem_bytes(pool.dtype);
  for (const int64_t s : {pool.page_stride, pool.pos_stride, pool.kv_stride, pool.head_stride})
    if (s < 0 || s % vec || s > INT64_C(1) << 40)
      return fail(HEXKV_EINVAL, "%s: pool stride %lld is not a whole number of 16 bytes", what, static_cast<long long>(s));
  if (pool.page_stride >= 1 << 30) return fail(HEXKV_ERANGE, "%s: pages are 2^30 elements apart or more", what);
  if (pool.pos_stride < d || pool.pos_stride > 1 << 26)
    return fail(HEXKV_EINVAL, "%s: positions of a page are %lld elements apart, not %d to 2^26", what,
                static_cast<long long>(pool.pos_stride), d);
  return HEXKV_OK;
}

int64_t pool_bytes(const hexkv_pool &pool) {
  return ((pool.n_pages - 1) * pool.page_stride + (pool.page_size - 1) * pool.pos_stride + pool.kv_stride +
          (pool.kv_heads - 1) * pool.head_stride + pool.head_dim) * elem_bytes(pool.dtype);
}

static int check_table(const int32_t *tables, int64_t stride, int width, int batch, int page_size, const char *what) {
  if (batch < 0 || width < 0) return fail(HEXKV_EINVAL, "%s: negative batch or table width", what);
  if (batch && width && !tables) return fail(HEXKV_EINVAL, "%s: null tables", what);
  // (stride 0: one table for all)
  if (batch > 1 && stride != 0 && stride < width) return fail(HEXKV_EINVAL, "%s: table rows overlap", what);
  if (static_cast<int64_t>(width) * page_size > INT64_C(1) << 30)
    return fail(HEXKV_ERANGE, "%s: tables of more than 2^30 positions", what);
  return HEXKV_OK;
}

int fill_tables(const hexkv_pool &pool, const hexkv_paged_batch &seqs, PageTables *p, const char *what) {
  int rc = check_pool(pool, what);
  if (rc == HEXKV_OK) rc = check_table(seqs.tables, seqs.table_stride, seqs.table_width, seqs.batch, pool.page_size, what);
  if (rc != HEXKV_OK) return rc;
  if (seqs.tokens < 0) return fail(HEXKV_EINVAL, "%s: negative token count", what);
  if (seqs.batch && !seqs.starts) return fail(HEXKV_EINVAL, "%s: null starts", what);
  if (!seqs.cu_tokens && (seqs.batch ? seqs.tokens % seqs.batch : seqs.tokens))
    return fail(HEXKV_EINVAL, "%s: %d tokens are no equal shares of %d sequences", what, seqs.tokens, seqs.batch);
  p->tables = seqs.tables;
  p->table_stride = seqs.table_stride;
  p->starts = seqs.starts;
  p->cu = seqs.cu_tokens;
  p->width = seqs.table_width;
  p->batch = seqs.batch;
  p->tokens = seqs.tokens;
  p->each = seqs.cu_tokens || !seqs.batch ? 0 : seqs.tokens / seqs.batch;
  p->n_pages = pool.n_pages;
  p->shift = __builtin_ctz(static_cast<unsigned>(pool.page_size));
  p->page_stride = pool.page_stride;
  p->pos_stride = pool.pos_stride;
  p->kv_stride = pool.kv_stride;
  p->head_stride = pool.head_stride;
  return HEXKV_OK;
}

// ---------------------------------------------------------------- append ---

// (8192 tokens 38.0 us with 256 threads a token, 43.7 with 512, 40.2 with 128.)
constexpr int kAppendRowThreads = 256;

struct PagedAppendArgs {
  PageTables p;
  const void *qkv;
  void *q, *pages;
  int64_t qkv_stride, q_stride;
  const float *inv_freq;
  int32_t q_heads, kv_heads, head_dim, rotary;
  float scale;
  unsigned int *status;
};

// VEC consecutive elements of T as one load or store.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T e[VEC];
};

// One token a workgroup.  Its sines and cosines are made once, by one lane a pair,
// and shared by all heads through LDS.  The angle p f / 2 pi (in turns) is a
// product in 64 bits less its whole turns: 32 bits leave 2^-8 of a radian at
// position 100000.  A unit is what one thread turns or copies: two vectors
// half a rotation apart (halves), or one (interleaved, dims that do not turn, v).
template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(kAppendRowThreads) void paged_append_kernel(const PagedAppendArgs a) {
  using P = Vec<T, VEC>;
  __shared__ float2 s_turn[128];
  const int t = blockIdx.x;
  int b, i;
  if (a.p.cu) {
    b = token_sequence(a.p, t);
    if (b < 0) return;
    i = t - a.p.cu[b];
  } else {
    b = t / a.p.each;
    i = t - b * a.p.each;
  }
  const int start = a.p.starts[b];
  if (start < 0) return;
  const int64_t pos = static_cast<int64_t>(start) + i;
  const int64_t index = pos >> a.p.shift;
  int page = -1;
  unsigned flags = 0;
  if (index >= a.p.width) {
    flags = HEXKV_STATUS_APPEND_SKIPPED;
  } else {
    page = a.p.tables[b * a.p.table_stride + index];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.p.n_pages)) {
      flags = HEXKV_STATUS_PAGE;
      page = -1;
    }
  }
  if (flags && threadIdx.x == 0 && blockIdx.y == 0) raise_status(a.status, flags);
  const int D = a.head_dim, half = a.rotary / 2;
  if (static_cast<int>(threadIdx.x) < half) {
    double turns = static_cast<double>(pos) * static_cast<double>(a.inv_freq[threadIdx.x]) * 0.15915494309189533577;
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.f * static_cast<float>(turns), &sn, &cs);
    s_turn[threadIdx.x] = float2{cs * a.scale, sn * a.scale};
  }
  __syncthreads();
  const T *src = static_cast<const T *>(a.qkv) + t * a.qkv_stride;
  T *q = static_cast<T *>(a.q) + t * a.q_stride;
  T *row = page < 0 ? nullptr
                    : static_cast<T *>(a.pages) + page * a.p.page_stride + (pos & ((1 << a.p.shift) - 1)) * a.p.pos_stride;
  const int pairs = INTERLEAVED ? 0 : half / VEC;  // units of two vectors
  const int per = D / VEC - pairs, copies = D / VEC;
  const int turned = (a.q_heads + a.kv_heads) * per, units = turned + a.kv_heads * copies;
  for (int u = blockIdx.y * blockDim.x + threadIdx.x; u < units; u += gridDim.y * blockDim.x) {
    if (u < turned) {
      const int head = u / per, j = u - head * per;
      const T *x = src + head * D;
      T *y = head < a.q_heads ? q + head * D : row ? row + (head - a.q_heads) * a.p.head_stride : nullptr;
      if (!y) continue;
      if (j < pairs) {
        const P x0 = *reinterpret_cast<const P *>(x + j * VEC), x1 = *reinterpret_cast<const P *>(x + half + j * VEC);
        P y0, y1;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float2 w = s_turn[j * VEC + k];
          const float c = static_cast<float>(x0.e[k]), s = static_cast<float>(x1.e[k]);
          y0.e[k] = Elem<T>::from_float(c * w.x - s * w.y);
          y1.e[k] = Elem<T>::from_float(s * w.x + c * w.y);
        }
        *reinterpret_cast<P *>(y + j * VEC) = y0;
        *reinterpret_cast<P *>(y + half + j * VEC) = y1;
      } else {
        const int at = (j + pairs) * VEC;
        P v = *reinterpret_cast<const P *>(x + at);
        if constexpr (INTERLEAVED && VEC > 1) {
          if (at < a.rotary) {
#pragma unroll
            for (int k = 0; k < VEC; k += 2) {
              const float2 w = s_turn[(at + k) / 2];
              const float c = static_cast<float>(v.e[k]), s = static_cast<float>(v.e[k + 1]);
              v.e[k] = Elem<T>::from_float(c * w.x - s * w.y);
              v.e[k + 1] = Elem<T>::from_float(s * w.x + c * w.y);
            }
          }
        }
        *reinterpret_cast<P *>(y + at) = v;
      }
    } else if (row) {
      const int v = u - turned, head = v / copies, at = (v - head * copies) * VEC;
      *reinterpret_cast<P *>(row + a.p.kv_stride + head * a.p.head_stride + at) =
          *reinterpret_cast<const P *>(src + (a.q_heads + a.kv_heads + head) * D + at);
    }
  }
}

template <typename T, bool INTERLEAVED>
static void launch_append(const PagedAppendArgs &a, int vec, hipStream_t s) {
  // A wave, or two, where a token has no more units and pairs (22 000 tokens of 4 + 2 x 2 fp32
  // heads of 32 25.2 us with four, 13.8 with one).  Few tokens: their units over several
  // workgroups, a unit a thread.
  const int units = (a.q_heads + 2 * a.kv_heads) * (a.head_dim / vec);
  const int most = std::max(units, a.rotary / 2), threads = most <= 64 ? 64 : most <= 128 ? 128 : kAppendRowThreads;
  const int parts = a.p.tokens >= 512 ? 1 : (units + threads - 1) / threads;
  const dim3 grid(static_cast<unsigned>(a.p.tokens), static_cast<unsigned>(std::min(parts, 65535)));
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  if (vec == VEC) paged_append_kernel<T, VEC, INTERLEAVED><<<grid, threads, 0, s>>>(a);
  else paged_append_kernel<T, INTERLEAVED ? 2 : 1, INTERLEAVED><<<grid, threads, 0, s>>>(a);
}

// --------------------------------------------------------------- handoff ---

// One launch over L layers and S sequences at most, in its arguments (as the
// handoff of the other caches).
template <int L, int S>
struct PagedCopyArgs {
  const char *src[L];
  char *dst[L];
  const int32_t *tables;
  int64_t table_stride;
  int64_t page_bytes, pos_bytes, kv_bytes, head_bytes;  // of the pool
  int32_t n_pages, shift;
  int32_t heads2, chunk_shift;  // 2 x KV heads; 16-byte vectors of one head's row: 2^chunk_shift
  int32_t rows;             // rows per workgroup, a power of two that divides the page
  int32_t batch;
  int32_t cu[S + 1];        // packed row of each sequence's first
  int32_t blocks[S + 1];    // workgroup of each sequence's first rows
  unsigned int *status;
};
using WidePagedCopy = PagedCopyArgs<HEXKV_MAX_LAYERS_PER_LAUNCH, HEXKV_MAX_SEQS_PER_LAUNCH>;
using SmallPagedCopy = PagedCopyArgs<32, 16>;
static_assert(sizeof(WidePagedCopy) <= 4096, "kernel arguments above 4 KiB");

// Workgroups as for the handoff of the other caches: 1024 threads of eight
// vectors each, 128 KB, and 256 of four for copies below 128 MB.
constexpr int kCopyThreads = 1024, kCopyUnroll = 8;
constexpr int kSmallCopyThreads = 256, kSmallCopyUnroll = 4;

// A workgroup moves `rows` positions of one page of one layer.  Vectors are
// taken in the order of the side that is written: a row's heads one after another
// when packing, a head's rows, K then V, when unpacking.
template <bool PACK, typename A, int NT, int UN>
__global__ __launch_bounds__(NT) void paged_copy_kernel(const A a) {
  const int block = blockIdx.x;
  int lo = 0, hi = a.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.blocks[mid] <= block) lo = mid; else hi = mid;
  }
  const int p0 = (block - a.blocks[lo]) * a.rows;
  const int n = min(a.rows, a.cu[lo + 1] - a.cu[lo] - p0);
  const int page = a.tables[lo * a.table_stride + (p0 >> a.shift)];
  const bool bad = static_cast<unsigned>(page) >= static_cast<unsigned>(a.n_pages);
  if (bad && threadIdx.x == 0 && blockIdx.y == 0) raise_status(a.status, HEXKV_STATUS_PAGE);
  if (!PACK && bad) return;
  const int64_t in_page = (bad ? 0 : page) * a.page_bytes + (p0 & ((1 << a.shift) - 1)) * a.pos_bytes;
  const int64_t row_bytes = static_cast<int64_t>(a.heads2) << (a.chunk_shift + 4);
  const int64_t in_packed = (static_cast<int64_t>(a.cu[lo]) + p0) * row_bytes;
  const char *src = a.src[blockIdx.y] + (PACK ? in_page : in_packed);
  char *dst = a.dst[blockIdx.y] + (PACK ? in_packed : in_page);
  // Chunk c of unit u = outer * inner + i: a head of a row; a thread's next
  // unit is `step` further.
  const int heads = a.heads2 >> 1, total = n * a.heads2, inner = PACK ? a.heads2 : n;
  const int step = NT >> a.chunk_shift, d_outer = step / inner, d_i = step - d_outer * inner;
  const int64_t c = (threadIdx.x & ((1 << a.chunk_shift) - 1)) * 16;
  int u = static_cast<int>(threadIdx.x) >> a.chunk_shift, outer = u / inner, i = u - outer * inner;
  while (u < total) {
    u32x4 r[UN];
    int64_t to[UN];
    const int first = u;
#pragma unroll
    for (int k = 0; k < UN; ++k) {
      const int row = PACK ? outer : i, h2 = PACK ? i : outer;
      const int head = PACK ? (h2 >= heads ? h2 - heads : h2) : h2 >> 1, kv = PACK ? h2 >= heads : h2 & 1;
      const int64_t packed = row * row_bytes + ((static_cast<int64_t>(kv ? heads : 0) + head) << (a.chunk_shift + 4)) + c;
      const int64_t paged = row * a.pos_bytes + (kv ? a.kv_bytes : 0) + head * a.head_bytes + c;
      to[k] = PACK ? packed : paged;
      if (u < total) r[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src + (PACK ? paged : packed)));
      if (PACK && bad) r[k] = u32x4{};
      u += step;
      i += d_i;
      outer += d_outer;
      if (i >= inner) {
        i -= inner;
        ++outer;
      }
    }
#pragma unroll
    for (int k = 0; k < UN; ++k)
      if (first + k * step < total) __builtin_nontemporal_store(r[k], reinterpret_cast<u32x4 *>(dst + to[k]));
  }
}

template <typename A>
static int launch_paged_copy(bool pack, const hexkv_pool &pool, const void *const *src, void *const *dst, int l0, int nl,
                             const int32_t *tables, int64_t table_stride, int nb, const int64_t *lens, int64_t packed_off,
                             int rows, bool small, unsigned int *status, hipStream_t stream, const char *what) {
  A a;
  const int es = elem_bytes(pool.dtype);
  a.tables = tables;
  a.table_stride = table_stride;
  a.page_bytes = pool.page_stride * es;
  a.pos_bytes = pool.pos_stride * es;
  a.kv_bytes = pool.kv_stride * es;
  a.head_bytes = pool.head_stride * es;
  a.n_pages = pool.n_pages;
  a.shift = __builtin_ctz(static_cast<unsigned>(pool.page_size));
  a.heads2 = 2 * pool.kv_heads;
  a.chunk_shift = __builtin_ctz(static_cast<unsigned>(pool.head_dim * es / 16));
  a.rows = rows;
  a.batch = nb;
  a.status = status;
  a.cu[0] = a.blocks[0] = 0;
  for (int b = 0; b < nb; ++b) {
    a.cu[b + 1] = a.cu[b] + static_cast<int32_t>(lens[b]);
    a.blocks[b + 1] = a.blocks[b] + static_cast<int32_t>((lens[b] + rows - 1) / rows);
  }
  if (a.blocks[nb] == 0) return HEXKV_OK;
  for (int l = 0; l < nl; ++l) {
    a.src[l] = static_cast<const char *>(src[l0 + l]) + (pack ? 0 : packed_off);
    a.dst[l] = static_cast<char *>(dst[l0 + l]) + (pack ? packed_off : 0);
  }
  const dim3 grid(static_cast<unsigned>(a.blocks[nb]), static_cast<unsigned>(nl));
  if (small) {
    constexpr int NT = kSmallCopyThreads, UN = kSmallCopyUnroll;
    if (pack) paged_copy_kernel<true, A, NT, UN><<<grid, NT, 0, stream>>>(a);
    else paged_copy_kernel<false, A, NT, UN><<<grid, NT, 0, stream>>>(a);
  } else {
    constexpr int NT = kCopyThreads, UN = kCopyUnroll;
    if (pack) paged_copy_kernel<true, A, NT, UN><<<grid, NT, 0, stream>>>(a);
    else paged_copy_kernel<false, A, NT, UN><<<grid, NT, 0, stream>>>(a);
  }
  return check_launch(what);
}

// Whether layers of `read_bytes` from the addresses `read` and layers of `written_bytes` from those in
// `written` lie apart, and the written ones from each other (pools, whose pages may lie in turn: whether they
// start apart).  r, w: room for n addresses each.
static bool layers_apart(const void *const *read, int64_t read_bytes, void *const *written, int64_t written_bytes, int n, bool pack,
                         uintptr_t *r, uintptr_t *w) {
  for (int l = 0; l < n; ++l) {
    r[l] = reinterpret_cast<uintptr_t>(read[l]);
    w[l] = reinterpret_cast<uintptr_t>(written[l]);
  }
  std::sort(r, r + n);
  std::sort(w, w + n);
  for (int l = 1; l < n; ++l)
    if (w[l] - w[l - 1] < static_cast<uintptr_t>(pack ? written_bytes : 1)) return false;
  for (int i = 0, j = 0; i < n && j < n;) {
    if (r[i] + read_bytes <= w[j]) ++i;
    else if (w[j] + written_bytes <= r[i]) ++j;
    else return false;
  }
  return true;
}

static int paged_copy(bool pack, const hexkv_pool *pool, const void *const *src, void *const *dst, int n_layers,
                      const int32_t *tables, int64_t table_stride, int table_width, int batch, const int64_t *lens,
                      hexkv_stream_t stream) {
  clear_error();
  const char *what = pack ? "hexkv_paged_pack" : "hexkv_paged_unpack";
  if (!pool) return fail(HEXKV_EINVAL, "%s: null argument", what);
  int rc = check_pool(*pool, what);
  if (rc == HEXKV_OK) rc = check_table(tables, table_stride, table_width, batch, pool->page_size, what);
  if (rc != HEXKV_OK) return rc;
  if (n_layers < 0) return fail(HEXKV_EINVAL, "%s: negative layer count", what);
  if (n_layers == 0 || batch == 0) return HEXKV_OK;
  if (!src || !dst || !lens) return fail(HEXKV_EINVAL, "%s: null argument", what);
  int64_t total = 0;
  for (int b = 0; b < batch; ++b) {
    if (lens[b] < 0 || lens[b] > static_cast<int64_t>(table_width) * pool->page_size)
      return fail(HEXKV_ERANGE, "%s: length %lld of sequence %d outside [0, %lld]", what, static_cast<long long>(lens[b]),
                  b, static_cast<long long>(table_width) * pool->page_size);
    total += lens[b];
  }
  if (total > INT32_MAX) return fail(HEXKV_ERANGE, "%s: more than 2^31-1 live rows", what);
  if (total == 0) return HEXKV_OK;
  for (int l = 0; l < n_layers; ++l)
    if (!src[l] || !dst[l] || !aligned16(src[l]) || !aligned16(dst[l]))
      return fail(HEXKV_EINVAL, "%s: layer %d's address is null or not 16-byte aligned", what, l);
  const int64_t row_bytes = 2 * static_cast<int64_t>(pool->kv_heads) * pool->head_dim * elem_bytes(pool->dtype);
  if (row_bytes > INT64_C(1) << 26) return fail(HEXKV_ERANGE, "%s: rows of more than 2^26 bytes", what);
  const bool small = total * row_bytes * n_layers < 128 << 20;
  const int64_t share = small ? kSmallCopyThreads * kSmallCopyUnroll * 16 : kCopyThreads * kCopyUnroll * 16;
  int rows = pool->page_size;
  while (rows > 1 && rows * row_bytes > share) rows /= 2;
  if (total / rows + batch >= 1 << 22) return fail(HEXKV_ERANGE, "%s: 2^22 workgroups a layer or more", what);
  const int64_t pool_size = pool_bytes(*pool), packed_size = total * row_bytes;
  uintptr_t few[2 * HEXKV_MAX_LAYERS_PER_LAUNCH];
  std::unique_ptr<uintptr_t[]> many;
  if (n_layers > HEXKV_MAX_LAYERS_PER_LAUNCH) {
    many.reset(new (std::nothrow) uintptr_t[2 * static_cast<size_t>(n_layers)]);
    if (!many) return fail(HEXKV_ERANGE, "%s: no memory for the addresses of %d layers", what, n_layers);
  }
  uintptr_t *sorted = many ? many.get() : few;
  if (!layers_apart(src, pack ? pool_size : packed_size, dst, pack ? packed_size : pool_size, n_layers, pack, sorted,
                    sorted + n_layers))
    return fail(HEXKV_EINVAL, "%s: a layer that is written overlaps another, or one that is read", what);
  unsigned int *status = nullptr;
  rc = status_word(stream, &status, what);
  if (rc != HEXKV_OK) return rc;
  int64_t base = 0;
  for (int b0 = 0; b0 < batch; b0 += HEXKV_MAX_SEQS_PER_LAUNCH) {
    const int nb = std::min(batch - b0, HEXKV_MAX_SEQS_PER_LAUNCH);
    const int32_t *t = tables + b0 * table_stride;
    for (int l0 = 0; l0 < n_layers; l0 += HEXKV_MAX_LAYERS_PER_LAUNCH) {
      const int nl = std::min(n_layers - l0, HEXKV_MAX_LAYERS_PER_LAUNCH);
      hipStream_t s = static_cast<hipStream_t>(stream);
      rc = nl <= 32 && nb <= 16
          ? launch_paged_copy<SmallPagedCopy>(pack, *pool, src, dst, l0, nl, t, table_stride, nb, lens + b0, base * row_bytes,
                                              rows, small, status, s, what)
          : launch_paged_copy<WidePagedCopy>(pack, *pool, src, dst, l0, nl, t, table_stride, nb, lens + b0, base * row_bytes,
                                             rows, small, status, s, what);
      if (rc != HEXKV_OK) return rc;
    }
    for (int b = 0; b < nb; ++b) base += lens[b0 + b];
  }
  return HEXKV_OK;
}

}  // namespace hexkv

extern "C" int hexkv_paged_append(const hexkv_paged_append_params *params, hexkv_stream_t stream) {
  using namespace hexkv;
  clear_error();
  const char *what = "hexkv_paged_append";
  if (!params) return fail(HEXKV_EINVAL, "%s: null argument", what);
  const hexkv_paged_append_params &p = *params;
  PagedAppendArgs a;
  int rc = fill_tables(p.pool, p.seqs, &a.p, what);
  if (rc != HEXKV_OK) return rc;
  const int d = p.pool.head_dim, es = elem_bytes(p.pool.dtype), vec = 16 / es;
  if (p.q_heads < 0 || p.q_heads > 1 << 16) return fail(HEXKV_EINVAL, "%s: %d query heads", what, p.q_heads);
  if (p.rotary_dim < 0 || p.rotary_dim % 2 || p.rotary_dim > d)
    return fail(HEXKV_EINVAL, "%s: rotary_dim %d is not even or not in [0, %d]", what, p.rotary_dim, d);
  const int64_t q_row = static_cast<int64_t>(p.q_heads) * d, row = q_row + 2 * static_cast<int64_t>(p.pool.kv_heads) * d;
  const int64_t tokens = p.seqs.tokens;
  if (p.qkv_stride < row && tokens > 1) return fail(HEXKV_EINVAL, "%s: qkv's rows overlap", what);
  if (p.q_stride < q_row && tokens > 1) return fail(HEXKV_EINVAL, "%s: q's rows overlap", what);
  if (tokens >= 1 << 24) return fail(HEXKV_ERANGE, "%s: 2^24 tokens or more", what);
  if (tokens == 0 || p.seqs.batch == 0) return HEXKV_OK;
  if (!p.qkv || (p.q_heads && !p.q) || !p.pages || (p.rotary_dim && !p.inv_freq)) return fail(HEXKV_EINVAL, "%s: null tensor", what);
  if (!aligned16(p.pages)) return fail(HEXKV_EINVAL, "%s: pages are not 16-byte aligned", what);
  // A thread writes the q that it read, so q may stand where it was; over
  // other rows, or over the pages, it may not.
  const int64_t in_bytes = ((tokens - 1) * p.qkv_stride + row) * es, q_bytes = ((tokens - 1) * p.q_stride + q_row) * es;
  const bool in_place = p.q == p.qkv && (tokens == 1 || p.q_stride == p.qkv_stride);
  if (!in_place && overlap(p.q, q_bytes, p.qkv, in_bytes)) return fail(HEXKV_EINVAL, "%s: q overlaps qkv", what);
  const int64_t pool = pool_bytes(p.pool);
  if (overlap(p.pages, pool, p.qkv, in_bytes) || overlap(p.pages, pool, p.q, q_bytes))
    return fail(HEXKV_EINVAL, "%s: the pages overlap qkv or q", what);
  rc = status_word(stream, &a.status, what);
  if (rc != HEXKV_OK) return rc;
  a.qkv = p.qkv;
  a.q = p.q;
  a.pages = p.pages;
  a.qkv_stride = p.qkv_stride;
  a.q_stride = p.q_stride;
  a.inv_freq = p.inv_freq;
  a.q_heads = p.q_heads;
  a.kv_heads = p.pool.kv_heads;
  a.head_dim = d;
  a.rotary = p.rotary_dim;
  a.scale = p.rotary_scale;
  const bool aligned = aligned16(p.qkv) && aligned16(p.q) && (tokens == 1 || (p.qkv_stride % vec == 0 && p.q_stride % vec == 0));
  const bool whole = (p.interleaved ? p.rotary_dim : p.rotary_dim / 2) % vec == 0;
  const int unit = aligned && whole ? vec : p.interleaved ? 2 : 1;
  const uintptr_t pair = static_cast<uintptr_t>(2 * es - 1);
  if (unit == 2 && ((reinterpret_cast<uintptr_t>(p.qkv) | reinterpret_cast<uintptr_t>(p.q)) & pair ||
                    (tokens > 1 && (p.qkv_stride | p.q_stride) & 1)))
    return fail(HEXKV_EINVAL, "%s: interleaved pairs are not aligned to two elements", what);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (p.pool.dtype) {
    case HEXKV_BF16: p.interleaved ? launch_append<__bf16, true>(a, unit, s) : launch_append<__bf16, false>(a, unit, s); break;
    case HEXKV_F16: p.interleaved ? launch_append<_Float16, true>(a, unit, s) : launch_append<_Float16, false>(a, unit, s); break;
    default: p.interleaved ? launch_append<float, true>(a, unit, s) : launch_append<float, false>(a, unit, s); break;
  }
  return check_launch(what);
}

extern "C" int hexkv_paged_pack(const hexkv_pool *pool, const void *const *pages, void *const *packed, int n_layers,
                                const int32_t *tables_dev, int64_t table_stride, int table_width, int batch,
                                const int64_t *lens, hexkv_stream_t stream) {
  return hexkv::paged_copy(true, pool, pages, packed, n_layers, tables_dev, table_stride, table_width, batch, lens, stream);
}

extern "C" int hexkv_paged_unpack(const hexkv_pool *pool, const void *const *packed, void *const *pages, int n_layers,
                                  const int32_t *tables_dev, int64_t table_stride, int table_width, int batch,
                                  const int64_t *lens, hexkv_stream_t stream) {
  return hexkv::paged_copy(false, pool, packed, pages, n_layers, tables_dev, table_stride, table_width, batch, lens, stream);
}
