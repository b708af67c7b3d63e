// Log-probabilities of given tokens, entropies and top alternatives of rows of
// logits: hexkv_token_logprobs.
//
// With m the row's largest logit, S = sum e^(x - m) and U = sum (x - m) e^(x - m):
//   log p(token) = x_token - m - log S,   entropy = log S - U / S.
// What bounds it: memory, every logit read once; beside that about 11 vector
// instructions a logit, one of them an exponential.  A workgroup walks a row
// (or, where rows are few, a part of one) 4096 logits at a time, 16 of them in each lane's
// registers and the next 16 in flight; every lane keeps its own (m, S, U),
// rescaled when its maximum moves, and the lanes' are joined once at the end.
//
// The top alternatives are the largest keys, a key being the logit's order
// above the complement of its id, so that ties go to the lowest id and no
// two keys are equal.  Every lane keeps the maximum of its logits too; the
// top-th largest of the lanes' is a bar that at least `top` logits reach, and,
// logits being spread over the lanes, little more do (21 of 32000 for the top 20).  The
// lanes whose maximum reaches it, as few, have their logits read again (from
// the caches) and what reaches the bar is ranked by counting.  Collecting during the walk
// instead, above the worst of the best so far, doubled a row's time (186 us
// against 97 without alternatives, 8191 x 32000 bf16): barriers and counting in
// every step.  A mask that leaves a few hundred neighbours makes all of them reach the bar
// (one lane in eight has any): up to 1024 are ranked (1 x 32000, 300 left, top 20: 21 us).
// Where more reach the bar (equal logits), those above it are ranked and the lowest ids
// equal to it follow; where more are above it (sorted logits), the top-th key is
// found by counting, eight bits at a time (1 x 32000 41 us; taking out the largest
// `top` times over took 474, and 370 for the mask).
//
// Measured on MI355X, bf16: 8191 x 32000 without alternatives 97 us (5.4 TB/s),
// with the top 20 126 us (4.2); one row of 32000 fp16, top 5, 10.2 us.
#include "hexkv_common.h"

#include <algorithm>

namespace hexkv {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / 64;
constexpr int kLpEach = 16;  // logits a lane holds at a time
constexpr int kLpChunk = kLpThreads * kLpEach;
constexpr int kLpRoom = 1024;  // keys that can be ranked
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
  // Neither a probability nor a logarithm to give: minus infinities alone.
  __device__ __forceinline__ bool none() const { return m == -INFINITY && s == 0.f; }
};

// What a row answers with, from its joined statistics.
template <typename T>
__device__ __forceinline__ void lp_finish(const LogprobArgs &a, int64_t row, const LpStats &st) {
  const float log_s = logf(st.s);
  if (a.entropy) a.entropy[row] = st.none() ? 0.f : log_s - st.u / st.s;
  if (a.tokens) {
    const int64_t t = a.tokens[row];
    float lp = t < 0 ? 0.f : NAN;
    if (t >= 0 && t < a.vocab) {
      const float x = static_cast<float>(static_cast<const T *>(a.logits)[row * a.stride + t]);
      lp = st.none() ? -INFINITY : x - st.m - log_s;
    }
    a.logprob[row] = lp;
  }
}

__device__ __forceinline__ void lp_write_top(const LogprobArgs &a, int64_t row, int rank, lp_key key, const LpStats &st) {
  const float v = lp_key_value(key);
  a.top_ids[row * a.top + rank] = lp_key_id(key);
  a.top_logprobs[row * a.top + rank] = st.none() ? -INFINITY : v - st.m - logf(st.s);
}

// One wave: the lowest ids in [first, last) of row x whose logit equals `value`,
// as keys at ranks from `held` to `top`; returns how many ranks are held then.
template <typename T>
__device__ __forceinline__ int lp_equal(const T *x, int64_t first, int64_t last, float value, int held, int top, lp_key *list) {
  constexpr int U = 8;  // loads in flight
  const int lane = threadIdx.x & 63;
  for (int64_t base = first; base < last && held < top; base += 64 * U) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = static_cast<float>(x[min(base + u * 64 + lane, last - 1)]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t id = base + u * 64 + lane;
      const bool out = id < last && v[u] == value;
      const uint64_t mask = __ballot(out);
      const int rank = held + __popcll(mask & ((uint64_t{1} << lane) - 1));
      if (out && rank < top) list[rank] = lp_make_key(value, static_cast<unsigned int>(id));
      held = min(top, held + __popcll(mask));
    }
  }
  return held;
}

template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprob_kernel(const LogprobArgs a) {
  constexpr int VEC = 16 / sizeof(T), NV = kLpEach / VEC;
  __shared__ lp_key s_list[kLpRoom], s_best[64];
  __shared__ float s_lane[kLpThreads], s_bar;
  __shared__ int s_active[kLpThreads], s_active_count, s_count[2], s_held, s_hist[256], s_pick[3];
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
  float best = -INFINITY;  // NaN where there is one

  u32x4 raw[NV];
  // Whether every place of a chunk is a logit of this part: then it is loaded ahead.
  const auto whole = [&](int64_t base) { return base >= skew && base + kLpChunk <= last; };
  const auto fetch = [&](int64_t base) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      raw[i] = *reinterpret_cast<const u32x4 *>(x + (base - skew) + (i * kLpThreads + tid) * VEC);
  };
  // The vector at place `at` of the row; a place outside the part counts as
  // minus infinity, which adds nothing and is never collected.
  const auto vector_at = [&](int64_t at, float *v) {
    if (at >= 0 && at + skew >= first && at + skew + VEC <= last) {
      Elem<T>::to_float(*reinterpret_cast<const u32x4 *>(x + at), v);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int64_t id = at + e;
        v[e] = id >= 0 && id + skew < last ? static_cast<float>(x[id]) : -INFINITY;
      }
    }
  };
  // A row of one chunk goes to the lanes logit by logit, so that every lane and
  // group has some however short the row or whatever a mask rules out: with
  // vectors, groups without any left no bar (709 x 825, part of it masked, top 20:
  // 36 us).
  const bool single = a.vocab + skew <= kLpChunk;
  const auto strided = [&](int i, int of) {
    const int id = i * kLpThreads + of;
    const float v = static_cast<float>(x[min(id, a.vocab - 1)]);
    return id < a.vocab ? v : -INFINITY;
  };
  if (!single && whole(first)) fetch(first);
  for (int64_t base = first; base < last; base += kLpChunk) {
    float v[kLpEach];
    if (single) {
#pragma unroll
      for (int i = 0; i < kLpEach; ++i) v[i] = strided(i, tid);
    } else if (whole(base)) {
#pragma unroll
      for (int i = 0; i < NV; ++i) Elem<T>::to_float(raw[i], v + i * VEC);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) vector_at(base + (i * kLpThreads + tid) * VEC - skew, v + i * VEC);
    }
    if (base + kLpChunk < last && whole(base + kLpChunk)) fetch(base + kLpChunk);
    float most = v[0];
#pragma unroll
    for (int i = 1; i < kLpEach; ++i) most = __builtin_elementwise_maximum(most, v[i]);
    best = __builtin_elementwise_maximum(best, most);
    st.shift(fmaxf(st.m, most));
    // Below -200 an exponential is 0 in any case; kept finite, it adds 0 to U too.
    const float m = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int i = 0; i < kLpEach; ++i) {
      const float d = __builtin_elementwise_maximum(v[i] - m, -200.f), w = lp_exp(d);
      st.s += w;
      st.u = fmaf(d, w, st.u);
    }
  }

  // join the lanes
  float m = wave_max(st.m);
  if (lane == 0) s_stats[wave][0] = m;
  if (best != best) best = INFINITY;  // a NaN is the largest there is
  s_lane[tid] = best;
  if (tid < 2) s_count[tid] = 0;
  if (tid == 0) s_active_count = 0;
  __syncthreads();
  m = fmaxf(fmaxf(s_stats[0][0], s_stats[1][0]), fmaxf(s_stats[2][0], s_stats[3][0]));
  st.shift(m);
  const float s_sum = sum_from<1>(st.s), u_sum = sum_from<1>(st.u);
  if (lane == 0) {
    s_stats[wave][1] = s_sum;
    s_stats[wave][2] = u_sum;
  }
  // The bar: the top-th largest of the lanes' maxima, of 64 groups of four while
  // those are several times as many as `top` (ranked by lane reads; 1 x 305, top 24, 6.3
  // us, by bits of all 256 7.4; top 32 by bits 7.6, ranking all 256 17).
  if (top && top <= 24) {
    if (wave == 0) {
      const f32x4 four = *reinterpret_cast<const f32x4 *>(s_lane + 4 * lane);
      const float mine = fmaxf(fmaxf(four[0], four[1]), fmaxf(four[2], four[3]));
      int rank = 0;
#pragma unroll
      for (int j = 0; j < 64; ++j) {
        const float other = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine), j));
        rank += other > mine || (other == mine && j < lane);
      }
      if (rank == top - 1) s_bar = mine;
    }
  } else if (top && wave == 0) {
    // all 256, bit by bit from the top: the largest order that `top` of them reach
    const f32x4 four = *reinterpret_cast<const f32x4 *>(s_lane + 4 * lane);
    unsigned int order[4], found = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) order[e] = static_cast<unsigned int>(lp_make_key(four[e], 0) >> 32);
#pragma unroll 4
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned int next = found | 1u << bit;
      int reach = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) reach += __popcll(__ballot(order[e] >= next));
      if (reach >= top) found = next;
    }
    if (lane == 0) s_bar = lp_key_value(static_cast<lp_key>(found) << 32);
  }
  __syncthreads();
  LpStats all = {m, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    all.s += s_stats[w][1];
    all.u += s_stats[w][2];
  }

  int held = 0;  // ranked keys in s_best
  if (top) {
    const float bar = s_bar;
    if (!(best < bar) && best > -INFINITY) s_active[atomicAdd(&s_active_count, 1)] = tid;
    __syncthreads();
    const int vectors = static_cast<int>((last - first + kLpChunk - 1) / kLpChunk) * NV, total = s_active_count * vectors;
    // the active lanes' vectors, shared out over all lanes (in any order: the ranks do not depend on it)
    const auto visit = [&](auto &&f) {
      if (single) {
        const int each = (a.vocab + kLpThreads - 1) / kLpThreads;
        for (int item = tid; item < s_active_count * each; item += kLpThreads) {
          const int of = item / each, i = item - of * each;
          f(strided(i, s_active[of]), static_cast<int64_t>(i) * kLpThreads + s_active[of]);
        }
        return;
      }
      for (int item = tid; item < total; item += kLpThreads) {
        const int of = item / vectors, j = item - of * vectors;
        const int64_t at = first + static_cast<int64_t>(j / NV) * kLpChunk + (j % NV * kLpThreads + s_active[of]) * VEC - skew;
        float v[VEC];
        vector_at(at, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f(v[e], at + e);
      }
    };
    const auto collect = [&](bool equal, int *counter) {
      visit([&](float v, int64_t id) {
        if ((equal ? !(v < bar) : !(v <= bar)) && v != -INFINITY) {
          const int place = atomicAdd(counter, 1);
          if (place < kLpRoom) s_list[place] = lp_make_key(v, static_cast<unsigned int>(id));
        }
      });
    };
    // Ranks by counting the larger keys: one wave by lane reads where a key
    // fits a lane each, as it nearly always does, else every lane over all in LDS.
    const auto rank_list = [&](int count) {
      if (count <= 64) {
        if (wave == 0) {
          const lp_key k = lane < count ? s_list[lane] : 0;
          const int lo = static_cast<int>(k), hi = static_cast<int>(k >> 32);
          int rank = 0;
          for (int j = 0; j < count; ++j) {
            const lp_key other = static_cast<lp_key>(static_cast<unsigned int>(__builtin_amdgcn_readlane(hi, j))) << 32 |
                                 static_cast<unsigned int>(__builtin_amdgcn_readlane(lo, j));
            rank += other > k;
          }
          if (lane < count && rank < top) s_best[rank] = k;
        }
      } else {
        for (int i = tid; i < count; i += kLpThreads) {
          const lp_key k = s_list[i];
          int rank = 0;
          for (int j = 0; j < count; ++j) rank += s_list[j] > k;
          if (rank < top) s_best[rank] = k;
        }
      }
      held = min(top, count);
      __syncthreads();
    };
    collect(true, &s_count[0]);
    __syncthreads();
    int count = s_count[0];
    if (count <= kLpRoom) {
      rank_list(count);
    } else {
      collect(false, &s_count[1]);
      __syncthreads();
      count = s_count[1];
      if (count <= kLpRoom) {
        rank_list(count);
        if (wave == 0 && held < top) {
          const int64_t from = max(first - skew, INT64_C(0));
          const int now = bar == -INFINITY ? held : lp_equal(x, from, last - skew, bar, held, top, s_best);
          if (lane == 0) s_held = now;
        } else if (tid == 0) {
          s_held = held;
        }
        __syncthreads();
        held = s_held;
      } else {
        // The top-th largest key, eight bits at a time from the top: the keys
        // at or above the bar that agree with it so far are counted by their next
        // eight, until all of a count are among the top.
        lp_key found = 0;
        int want = top;  // of the keys that agree with `found`
        for (int shift = 56;; shift -= 8) {
          s_hist[tid] = 0;
          __syncthreads();
          visit([&](float v, int64_t id) {
            if (v < bar || v == -INFINITY) return;
            const lp_key k = lp_make_key(v, static_cast<unsigned int>(id));
            if ((k ^ found) >> shift >> 8) return;
            const int bin = static_cast<int>(k >> shift) & 255, one = __builtin_amdgcn_readfirstlane(bin);
            const uint64_t same = __ballot(bin == one);  // mostly all of them: one addition
            if (bin != one) atomicAdd(&s_hist[bin], 1);
            else if (lane == __builtin_ctzll(same)) atomicAdd(&s_hist[one], __popcll(same));
          });
          __syncthreads();
          if (wave == 0) {  // four bins a lane, from the top down
            int n[4], own = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) own += n[e] = s_hist[255 - 4 * lane - e];
            int above = own;
            for (int off = 1; off < 64; off <<= 1) {
              const int other = __shfl_up(above, off);
              if (lane >= off) above += other;
            }
            above -= own;
            if (above < want && want <= above + own)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (above < want && want <= above + n[e]) {
                  s_pick[0] = 255 - 4 * lane - e;
                  s_pick[1] = want - above;
                  s_pick[2] = n[e];
                }
                above += n[e];
              }
          }
          if (tid == 0) s_count[0] = 0;
          __syncthreads();
          found |= static_cast<lp_key>(s_pick[0]) << shift;
          want = s_pick[1];
          if (want == s_pick[2] || shift == 0) break;
        }
        visit([&](float v, int64_t id) {
          const lp_key k = lp_make_key(v, static_cast<unsigned int>(id));
          if (v < bar || v == -INFINITY || k < found) return;
          const int place = atomicAdd(&s_count[0], 1);
          if (place < kLpRoom) s_list[place] = k;
        });
        __syncthreads();
        rank_list(min(s_count[0], kLpRoom));  // (`top` of them)
      }
    }
  }
  if (a.parts > 1) {
    if (tid == 0) *reinterpret_cast<f32x4 *>(a.ws_stats + (row * a.parts + part) * 4) = f32x4{all.m, all.s, all.u, 0.f};
    if (tid < top) a.ws_keys[(row * a.parts + part) * top + tid] = tid < held ? s_best[tid] : 0;
    return;
  }
  if (tid == 0) lp_finish<T>(a, row, all);
  // a list that ends short is filled with minus infinities, none of which was collected
  if (wave == 0) {
    if (held < top) lp_equal(x, 0, a.vocab, -INFINITY, held, top, s_best);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (lane < top) lp_write_top(a, row, lane, s_best[lane], all);
  }
}

// Joins a row's parts.
template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprob_join_kernel(const LogprobArgs a) {
  __shared__ lp_key s_keys[kLpMaxParts * 64], s_best[64];
  __shared__ int s_keyed;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int lane = tid & 63;
  // a part a lane (every wave for itself)
  LpStats all = {-INFINITY, 0.f, 0.f};
  if (lane < a.parts) {
    const f32x4 v = *reinterpret_cast<const f32x4 *>(a.ws_stats + (row * a.parts + lane) * 4);
    all = LpStats{v[0], v[1], v[2]};
  }
  all.shift(wave_max(all.m));
  all = LpStats{wave_max(all.m), sum_from<1>(all.s), sum_from<1>(all.u)};
  if (tid == 0) lp_finish<T>(a, row, all);
  if (!a.top) return;
  const int n = a.parts * a.top;
  if (tid == 0) s_keyed = 0;
  for (int i = tid; i < n; i += kLpThreads) s_keys[i] = a.ws_keys[row * n + i];
  __syncthreads();
  for (int i = tid; i < n; i += kLpThreads) {
    const lp_key k = s_keys[i];
    if (!k) continue;
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s_keys[j] > k;
    if (rank < a.top) {
      s_best[rank] = k;
      atomicAdd(&s_keyed, 1);
    }
  }
  __syncthreads();
  if (tid < 64) {
    if (s_keyed < a.top)
      lp_equal(static_cast<const T *>(a.logits) + row * a.stride, 0, a.vocab, -INFINITY, s_keyed, a.top, s_best);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (tid < a.top) lp_write_top(a, row, tid, s_best[tid], all);
  }
}

// Parts a row is cut into: one to kLpShort chunks, where the join's launch and
// the workspace cost more than the shorter walk saves (us a call, host included, one
// part / split, top 5 and 20: 1 x 32000 10.0 / 13.4 and 11.8 / 13.4; 40960 10.4 / 13.4
// and 12.1 / 13.3; 49145, the longest of 12 chunks, 12.0 / 13.3 and 14.2 / 13.2; 65536 13.4
// / 13.4 and 16.0 / 13.3; 16 x 49145 12.7 / 13.4 and 15.2 / 13.4); beyond, enough for a
// workgroup a CU, and for few rows of long vocabularies about twelve chunks
// each, but no more keys than a join ranks in passing, since it compares all of them (us
// in 1 / 4 / 8 / 32 parts: 1 x 128000, top 20 25.6 / 15.5 / 13 / 36, top 5 21 / 12.6 /
// 10.8 / 11.1; top 64 in 4 parts 23.5, in 32 over 200;
// 64 x 128000, top 20, 27.6 / 16.7 / 16.6 / 25.6; 300 x 128000 37.4 / 32.8 / 32.3).
constexpr int kLpShort = 12, kLpKeys = 160;
static int lp_parts(int64_t rows, int vocab, int top, int64_t *span) {
  const int64_t chunks = (static_cast<int64_t>(vocab) + 7 + kLpChunk - 1) / kLpChunk;
  const int64_t fill = 256 / std::max<int64_t>(rows, 1), long_rows = rows < 1024 ? chunks / 12 : 1;
  const int64_t most = top ? std::min(kLpMaxParts, std::max(4, kLpKeys / top)) : kLpMaxParts;
  const int64_t wanted = chunks <= kLpShort ? 1 : std::max<int64_t>(1, std::min<int64_t>({chunks, most, std::max(fill, long_rows)}));
  const int64_t each = (chunks + wanted - 1) / wanted;
  *span = each * kLpChunk;
  return static_cast<int>((chunks + each - 1) / each);
}

static size_t lp_workspace(int64_t rows, int vocab, int top) {
  int64_t span;
  const int parts = lp_parts(rows, vocab, top, &span);
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
  a.parts = lp_parts(rows, vocab, top, &span);
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
