// Log-probabilities of given tokens, entropies and top alternatives of rows of
// logits: hexkv_token_logprobs.
//
// With m the row's largest logit, S = sum e^(x - m) and U = sum (x - m) e^(x - m):
//   log p(token) = x_token - m - log S,   entropy = log S - U / S.
// What bounds it: memory, every logit read once.  A workgroup walks a row (or,
// where rows are few, a part of one) 8192 logits at a time, 32 of them in each
// lane's registers; every lane keeps its own (m, S, U), rescaled when its
// maximum moves, and the lanes' are joined once at the end.
//
// The top alternatives are the largest keys, a key being the logit's order
// above the complement of its id, so that ties go to the lowest id and no
// two keys are equal.  The list of the best `top` so far sets the bar; logits above
// it are collected in LDS and the list is re-ranked by counting, which
// happens for few of them once a list is full.  Where too many pass the bar
// (a row's first logits, rising rows), it is raised to the top-th largest of
// 64 groups' maxima, below which no key can be among the best; where that
// does not suffice, the largest is taken out `top` times over.
#include "hexkv_common.h"

#include <algorithm>

namespace hexkv {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / 64;
constexpr int kLpEach = 32;  // logits a lane holds at a time
constexpr int kLpChunk = kLpThreads * kLpEach;
constexpr int kLpRoom = 512;  // keys collected at a time, beside the list
constexpr int kLpMaxParts = 32;

struct LogprobArgs {
  const void *logits;
  int64_t stride;  // elements
  const int64_t *tokens;
  float *logprob, *entropy, *top_logprobs;
  int64_t *top_ids;
  int32_t vocab, top, parts, span;  // span: logits of a part, a multiple of kLpChunk
  int64_t rows;
  float *ws_stats;              // [rows][parts][4]: m, S, U, -
  unsigned long long *ws_keys;  // [rows][parts][top]
};

typedef unsigned long long lp_key;

// Order of floats as unsigned integers; NaN above all, -0 as 0.
__device__ __forceinline__ lp_key lp_make_key(float x, unsigned int id) {
  unsigned int u = __float_as_uint(x + 0.f);
  u = x != x ? 0xffffffffu : u & 0x80000000u ? ~u : u | 0x80000000u;
  return static_cast<lp_key>(u) << 32 | (0xffffffffu - id);
}
__device__ __forceinline__ float lp_key_value(lp_key k) {
  const unsigned int u = static_cast<unsigned int>(k >> 32);
  if (u == 0xffffffffu) return NAN;
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int64_t lp_key_id(lp_key k) { return 0xffffffffu - static_cast<unsigned int>(k); }

__device__ __forceinline__ lp_key lp_shfl_xor(lp_key k, int off) {
  const unsigned int lo = __shfl_xor(static_cast<unsigned int>(k), off), hi = __shfl_xor(static_cast<unsigned int>(k >> 32), off);
  return static_cast<lp_key>(hi) << 32 | lo;
}

__device__ __forceinline__ float lp_exp(float u) { return __builtin_amdgcn_exp2f(u * 1.4426950408889634f); }

// (m, S, U) of two sets joined; a set without finite logits has S = 0.
struct LpStats {
  float m, s, u;
  __device__ __forceinline__ void shift(float to) {  // to >= m
    if (to == -INFINITY || m == to) return;
    const float d = m - to, w = lp_exp(d);  // 0 for m = -inf: then s = u = 0
    u = s > 0.f || s != s ? w * fmaf(d, s, u) : 0.f;
    s *= w;
    if (w == 0.f && s == s) s = u = 0.f;
    m = to;
  }
};

// What a row answers with, from its joined statistics.
__device__ __forceinline__ void lp_finish(const LogprobArgs &a, int64_t row, const LpStats &st, float token_logit,
                                          bool token_in) {
  const float log_s = logf(st.s);
  // a row of minus infinities has no probability to give
  const bool none = st.m == -INFINITY && st.s == 0.f;
  if (a.entropy) a.entropy[row] = none ? 0.f : log_s - st.u / st.s;
  if (a.tokens) {
    const int64_t t = a.tokens[row];
    float lp = none ? -INFINITY : token_logit - st.m - log_s;
    if (!token_in) lp = t < 0 ? 0.f : NAN;
    a.logprob[row] = lp;
  }
}

__device__ __forceinline__ void lp_write_top(const LogprobArgs &a, int64_t row, int rank, lp_key key, const LpStats &st) {
  const bool none = st.m == -INFINITY && st.s == 0.f;
  const float v = lp_key_value(key);
  a.top_ids[row * a.top + rank] = lp_key_id(key);
  a.top_logprobs[row * a.top + rank] = none ? -INFINITY : v - st.m - logf(st.s);
}

template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprob_kernel(const LogprobArgs a) {
  constexpr int VEC = 16 / sizeof(T), NV = kLpEach / VEC;
  __shared__ lp_key s_list[64 + kLpRoom];  // the best so far, then what was collected
  __shared__ lp_key s_best[64];
  __shared__ lp_key s_wave[kLpWaves];
  __shared__ int s_count;
  __shared__ lp_key s_bar;
  __shared__ float s_stats[kLpWaves][3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / static_cast<unsigned>(a.parts);
  const int part = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.parts));
  const T *x = static_cast<const T *>(a.logits) + row * a.stride;
  // vectors start at 16-byte boundaries: `skew` places before the row's first logit
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(x) / sizeof(T) % VEC);
  const int64_t first = static_cast<int64_t>(part) * a.span;
  const int64_t last = min(first + a.span, static_cast<int64_t>(a.vocab) + skew);
  const int top = a.top;
  LpStats st = {-INFINITY, 0.f, 0.f};
  int held = 0;  // keys in the list
  if (top) {
    if (tid < 64) s_list[tid] = 0;
    if (tid == 0) s_count = 0;
    __syncthreads();
  }

  for (int64_t base = first; base < last; base += kLpChunk) {
    float v[kLpEach];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t at = base + (i * kLpThreads + tid) * VEC - skew;
      if (at >= 0 && at + VEC <= a.vocab && at + skew + VEC <= last) {
        if constexpr (sizeof(T) == 2) Elem<T>::to_float(*reinterpret_cast<const u32x4 *>(x + at), v + i * VEC);
        else Elem<T>::to_float(*reinterpret_cast<const u32x4 *>(x + at), v + i * VEC);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int64_t id = at + e;
          v[i * VEC + e] = id >= 0 && id < a.vocab && id + skew < last ? static_cast<float>(x[id]) : -INFINITY;
        }
      }
    }
    // (A place outside the row counts as minus infinity, which adds nothing; it
    // is kept from the keys below.)
    float m = st.m;
#pragma unroll
    for (int i = 0; i < kLpEach; ++i) m = fmaxf(m, v[i]);
    st.shift(m);
#pragma unroll
    for (int i = 0; i < kLpEach; ++i) {
      const float d = v[i] - st.m, w = lp_exp(d);
      if (v[i] == -INFINITY) continue;
      st.s += w;
      st.u += w == 0.f ? 0.f : d * w;
    }
    if (!top) continue;

    const auto id_of = [&](int i) { return base + ((i / VEC) * kLpThreads + tid) * VEC + i % VEC - skew; };
    const auto key_of = [&](int i) -> lp_key {
      const int64_t id = id_of(i);
      return id >= 0 && id < a.vocab && id + skew < last ? lp_make_key(v[i], static_cast<unsigned int>(id)) : 0;
    };
    lp_key bar = held == top ? s_list[top - 1] : 0;  // keys have to exceed it
    bool raised = false;
    for (;;) {
      // collect what exceeds the bar
      bool over = false;
#pragma unroll
      for (int i = 0; i < kLpEach; ++i) {
        const lp_key k = key_of(i);
        if (k > bar && !over) {
          const int at = atomicAdd(&s_count, 1);
          if (at < kLpRoom) s_list[64 + at] = k;
          else over = true;
        }
      }
      __syncthreads();
      const int count = s_count;
      __syncthreads();  // read by all before anyone counts again
      if (count == 0) break;
      if (count <= kLpRoom) {
        // rank the list and what was collected by counting
        const int total = 64 + count;
        for (int i = tid; i < total; i += kLpThreads) {
          const lp_key k = s_list[i];
          int rank = 0;
          for (int j = 0; j < total; ++j) rank += s_list[j] > k;
          if (k && rank < 64) s_best[rank] = k;
        }
        __syncthreads();
        const int known = min(top, held + count);
        if (tid < 64) s_list[tid] = tid < known ? s_best[tid] : 0;
        if (tid == 0) s_count = 0;
        held = known;
        __syncthreads();
        break;
      }
      if (tid == 0) s_count = 0;
      if (!raised) {
        // the top-th largest of 64 groups' maxima
        raised = true;
        lp_key best = 0;
#pragma unroll
        for (int i = 0; i < kLpEach; ++i) best = max(best, key_of(i));
        best = max(best, lp_shfl_xor(best, 1));
        best = max(best, lp_shfl_xor(best, 2));
        if (lane % 4 == 0) s_best[wave * 16 + lane / 4] = best;
        __syncthreads();
        if (tid < 64) {
          const lp_key k = s_best[tid];
          int rank = 0;
          for (int j = 0; j < 64; ++j) rank += s_best[j] > k;
          const int groups = __popcll(__ballot(k != 0));  // (a group without a logit has key 0)
          if (groups < top ? tid == 0 : k && rank == top - 1) s_bar = groups < top ? 1 : k;
        }
        __syncthreads();
        bar = max(bar, s_bar - 1);
        __syncthreads();
        continue;
      }
      // take the largest out `top` times over, from the list and the lanes
      __syncthreads();
      lp_key below = ~static_cast<lp_key>(0);
      const lp_key mine = tid < 64 ? s_list[tid] : 0;
      int found = 0;
      for (; found < top; ++found) {
        lp_key best = mine < below ? mine : 0;
#pragma unroll
        for (int i = 0; i < kLpEach; ++i) {
          const lp_key k = key_of(i);
          if (k < below) best = max(best, k);
        }
        for (int off = 1; off < 64; off <<= 1) best = max(best, lp_shfl_xor(best, off));
        if (lane == 0) s_wave[wave] = best;
        __syncthreads();
        best = max(max(s_wave[0], s_wave[1]), max(s_wave[2], s_wave[3]));
        if (tid == 0) s_best[found] = best;
        __syncthreads();
        if (!best) break;
        below = best;
      }
      if (tid < 64) s_list[tid] = tid < found ? s_best[tid] : 0;
      held = found;
      __syncthreads();
      break;
    }
  }

  // join the lanes
  float m = wave_max(st.m);
  if (lane == 0) s_stats[wave][0] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_stats[0][0], s_stats[1][0]), fmaxf(s_stats[2][0], s_stats[3][0]));
  __syncthreads();
  st.shift(m);
  const float s_sum = sum_from<1>(st.s), u_sum = sum_from<1>(st.u);
  if (lane == 0) {
    s_stats[wave][1] = s_sum;
    s_stats[wave][2] = u_sum;
  }
  __syncthreads();
  LpStats all = {m, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    all.s += s_stats[w][1];
    all.u += s_stats[w][2];
  }
  if (a.parts > 1) {
    if (tid == 0) *reinterpret_cast<f32x4 *>(a.ws_stats + (row * a.parts + part) * 4) = f32x4{all.m, all.s, all.u, 0.f};
    if (tid < top) a.ws_keys[(row * a.parts + part) * top + tid] = s_list[tid];
    return;
  }
  if (tid == 0) {
    float logit = 0.f;
    bool in = false;
    if (a.tokens) {
      const int64_t t = a.tokens[row];
      in = t >= 0 && t < a.vocab;
      if (in) logit = static_cast<float>(x[t]);
    }
    lp_finish(a, row, all, logit, in);
  }
  if (tid < top) lp_write_top(a, row, tid, s_list[tid], all);
}

// Joins a row's parts.
template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprob_join_kernel(const LogprobArgs a) {
  __shared__ lp_key s_keys[kLpMaxParts * 64];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const float *stats = a.ws_stats + row * a.parts * 4;
  LpStats all = {-INFINITY, 0.f, 0.f};
  for (int p = 0; p < a.parts; ++p) all.m = fmaxf(all.m, stats[4 * p]);
  for (int p = 0; p < a.parts; ++p) {
    LpStats st = {stats[4 * p], stats[4 * p + 1], stats[4 * p + 2]};
    st.shift(all.m);
    all.s += st.s;
    all.u += st.u;
  }
  if (tid == 0) {
    float logit = 0.f;
    bool in = false;
    if (a.tokens) {
      const int64_t t = a.tokens[row];
      in = t >= 0 && t < a.vocab;
      if (in) logit = static_cast<float>(static_cast<const T *>(a.logits)[row * a.stride + t]);
    }
    lp_finish(a, row, all, logit, in);
  }
  if (!a.top) return;
  const int n = a.parts * a.top;
  for (int i = tid; i < n; i += kLpThreads) s_keys[i] = a.ws_keys[row * n + i];
  __syncthreads();
  for (int i = tid; i < n; i += kLpThreads) {
    const lp_key k = s_keys[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s_keys[j] > k;
    if (k && rank < a.top) lp_write_top(a, row, rank, k, all);
  }
}

// Parts a row is cut into: one where the rows alone give every CU several
// workgroups.
static int lp_parts(int64_t rows, int vocab, int64_t *span) {
  const int64_t chunks = (static_cast<int64_t>(vocab) + 7 + kLpChunk - 1) / kLpChunk;
  const int64_t wanted = std::max<int64_t>(1, std::min<int64_t>({chunks, kLpMaxParts, 1024 / std::max<int64_t>(rows, 1)}));
  const int64_t each = (chunks + wanted - 1) / wanted;
  *span = each * kLpChunk;
  return static_cast<int>((chunks + each - 1) / each);
}

static size_t lp_workspace(int64_t rows, int vocab, int top) {
  int64_t span;
  const int parts = lp_parts(rows, vocab, &span);
  return parts == 1 ? 0 : static_cast<size_t>(rows) * parts * (16 + 8 * static_cast<size_t>(top));
}

static int lp_check(int64_t rows, int vocab, int top, int dtype, const char *what) {
  if (dtype != HEXKV_F16 && dtype != HEXKV_BF16 && dtype != HEXKV_F32)
    return fail(HEXKV_EINVAL, "%s: unknown dtype %d", what, dtype);
  if (rows < 0 || vocab < 1 || vocab > (1 << 30)) return fail(HEXKV_EINVAL, "%s: bad rows/vocab", what);
  if (top < 0 || top > HEXKV_MAX_TOP || top > vocab)
    return fail(HEXKV_EINVAL, "%s: top %d outside [0, min(%d, vocab)]", what, top, HEXKV_MAX_TOP);
  if (rows >= INT64_C(1) << 19) return fail(HEXKV_ERANGE, "%s: 2^19 rows or more; split the call", what);
  return HEXKV_OK;
}

}  // namespace hexkv

extern "C" size_t hexkv_token_logprobs_workspace_bytes(int64_t rows, int vocab, int top) {
  using namespace hexkv;
  clear_error();
  if (lp_check(rows, vocab, top, HEXKV_F32, "hexkv_token_logprobs_workspace_bytes") != HEXKV_OK) return 0;
  return lp_workspace(rows, vocab, top);
}

extern "C" int hexkv_token_logprobs(const void *logits, int64_t row_stride, int64_t rows, int vocab, int dtype,
                                    const int64_t *tokens_dev, int top, float *logprob, float *entropy,
                                    float *top_logprobs, int64_t *top_ids, void *workspace, size_t workspace_bytes,
                                    hexkv_stream_t stream) {
  using namespace hexkv;
  const char *what = "hexkv_token_logprobs";
  clear_error();
  int rc = lp_check(rows, vocab, top, dtype, what);
  if (rc != HEXKV_OK) return rc;
  if (rows == 0) return HEXKV_OK;
  if (!logits || (tokens_dev && !logprob) || (top && (!top_logprobs || !top_ids)))
    return fail(HEXKV_EINVAL, "%s: null argument", what);
  const int elem = dtype == HEXKV_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(logits) & (elem - 1)) ||
      ((reinterpret_cast<uintptr_t>(tokens_dev) | reinterpret_cast<uintptr_t>(top_ids)) & 7))
    return fail(HEXKV_EINVAL, "%s: misaligned tensor", what);
  const size_t need = lp_workspace(rows, vocab, top);
  if (need && (!workspace || workspace_bytes < need))
    return fail(HEXKV_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : 0, need);
  if (need && !aligned16(workspace)) return fail(HEXKV_EINVAL, "%s: workspace must be 16-byte aligned", what);
  LogprobArgs a = {};
  a.logits = logits;
  a.stride = row_stride;
  a.tokens = tokens_dev;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_logprobs = top_logprobs;
  a.top_ids = top_ids;
  a.vocab = vocab;
  a.top = top;
  a.rows = rows;
  int64_t span;
  a.parts = lp_parts(rows, vocab, &span);
  a.span = static_cast<int32_t>(std::min<int64_t>(span, INT32_MAX));
  if (a.parts > 1) {
    a.ws_stats = static_cast<float *>(workspace);
    a.ws_keys = reinterpret_cast<unsigned long long *>(a.ws_stats + rows * a.parts * 4);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(rows * a.parts)), join(static_cast<unsigned>(rows));
#define HEXKV_LOGPROBS(T)                                            \
  logprob_kernel<T><<<grid, kLpThreads, 0, s>>>(a);                  \
  if (a.parts > 1) logprob_join_kernel<T><<<join, kLpThreads, 0, s>>>(a);
  if (dtype == HEXKV_BF16) { HEXKV_LOGPROBS(__bf16) }
  else if (dtype == HEXKV_F16) { HEXKV_LOGPROBS(_Float16) }
  else { HEXKV_LOGPROBS(float) }
#undef HEXKV_LOGPROBS
  return check_launch(what);
}
