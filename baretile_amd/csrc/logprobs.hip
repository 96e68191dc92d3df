// Log probabilities of given tokens, each row's entropy and its likeliest tokens, from rows of logits.
//
// With p = softmax(t x) of a row, m its largest logit, y_j = t (x_j - m), S = sum exp(y_j): log p_j = y_j - log S, and the entropy
// -sum p_j log p_j = log S - sum exp(y_j) y_j / S (no difference of large numbers: both terms are at most log(vocab)). Rows are cut
// into chunks, a block each, whose logits stay in registers: one read gives the chunk's maximum, then its sums against that, and
// its k largest. A second launch joins a row's chunks; rows of one chunk need none.
//
// The k largest of a chunk: at least k of its threads have a largest value of at least T, so all of the k largest are at least T,
// the largest such T found by halving over the threads' largest values (one wave's ballots), and few others are; these go to LDS
// and rank themselves by counting, equal values by their column, so the order in which they came doesn't matter. Where more
// threads tie at T than that is made for, only the columns up to the one that completes k threads count.
#include "common.h"
#include <algorithm>

namespace bt {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int PER = 16;     // logits a thread
constexpr int MOST_K = 64, MOST_VOCAB = 1 << 20;
constexpr float NONE = -__builtin_inff(), LARGEST = 3.4028234663852886e38f;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;
constexpr int NOWHERE = 0x7FFFFFFF;

struct ChunkSums {
  float m, s, e;  // the largest logit, sum w, sum w log2 w of its weights w = exp(t (x - m))
  int32_t at;     // where the largest first is (an infinite t's rows)
};
struct LogprobArgs {
  const float *logits, *t;
  const int32_t *ids;
  float *logprobs, *entropy, *values;
  int32_t *labels;
  ChunkSums *sums;               // [rows][chunks]
  float *top_values;             // [rows][chunks][k], -inf and column -1 where there are fewer
  int32_t *top_columns;
  int64_t logits_sr, t_sr;
  int32_t vocab, k, chunks;
};

// A logit as it counts: NaN as -inf, +inf as the largest finite.
__device__ __forceinline__ float logit(float x) { return x != x ? NONE : fminf(x, LARGEST); }

// A row's inverse temperature t, below 0 or NaN as 0. Differences of logits are taken halved, so that they don't pass the largest
// number, and t is at least the smallest number there is, so that a t of 0 weighs every logit over -inf alike.
struct Inverse {
  float log2, t;  // (log2: 2 t log2(e))
  bool greedy;  // an infinite t: the first of the largest alone
};
__device__ __forceinline__ Inverse inverse(const LogprobArgs &a, int row) {
  float t = a.t ? gload(a.t + row * a.t_sr) : 1.0f;
  t = t > 0.0f ? t : 0.0f;
  constexpr float least = 1.401298464e-45f;
  return {fmaxf(fminf(t * (2.0f * LOG2E), LARGEST), least), fmaxf(t, least), t > LARGEST};
}
__device__ __forceinline__ float half_less(float x, float m) { return __builtin_fmaf(x, 0.5f, -0.5f * m); }
// log2 of a weight, down to where it is 0. (-inf - -inf and NaN: 0 weight.)
__device__ __forceinline__ float log2_weight(float x, float m, float t2) { return fmaxf(half_less(x, m) * t2, -200.0f); }

__device__ __forceinline__ float wave_max(float x) {  // as wave_sum in common.h
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x128, 0xF, 0xF, false)));
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x141, 0xF, 0xF, false)));
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0x4E, 0xF, 0xF, false)));
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), 0xB1, 0xF, 0xF, false)));
}

// Values as whole numbers in their order (-0 as 0), and back.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t u) { return __uint_as_float(u ^ (u >> 31 ? 0x80000000u : 0xFFFFFFFFu)); }
constexpr uint32_t LEAST_ORDERED = 0x00800000u;  // the one above -inf

// The threads whose values may go on, k at least and so many at most.
__host__ __device__ constexpr int limit_of(int k) { return k + k / 2 + 8; }
template <int NT> struct TopLds {
  uint64_t found[PER * limit_of(MOST_K)];
  uint32_t tops[NT];
  int32_t first[NT];
  uint32_t least;
  int32_t upto, count;
};

// By the first wave: T, from the threads' largest values in LDS. Returns whether more than the limit tie at it.
template <int NT> __device__ __forceinline__ bool find_least(TopLds<NT> &lds, int k, uint32_t *least) {
  constexpr int N = NT / 64;
  const int lane = threadIdx.x & 63;
  uint32_t top[N];
#pragma unroll
  for (int i = 0; i < N; i++) top[i] = lds.tops[lane + 64 * i];
  const auto count = [&](uint32_t x) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; i++) n += __popcll(__ballot(top[i] >= x));
    return n;
  };
  uint32_t lo = LEAST_ORDERED, hi = 0xFF800000u;  // above every finite value
  int n = count(lo);
  if (n > k)
    while (n > limit_of(k) && hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const int m = count(mid);
      if (m >= k) lo = mid, n = m;
      else hi = mid;
    }
  *least = lo;
  return n > limit_of(k);
}
// By the first wave: the column up to which those that tie at T complete k threads.
template <int NT> __device__ __forceinline__ int find_upto(TopLds<NT> &lds, int k, uint32_t least) {
  constexpr int N = NT / 64;
  const int lane = threadIdx.x & 63;
  uint32_t top[N];
  int first[N];
#pragma unroll
  for (int i = 0; i < N; i++) top[i] = lds.tops[lane + 64 * i], first[i] = lds.first[lane + 64 * i];
  int lo = -1, hi = MOST_VOCAB;  // fewer than k up to lo, k up to hi
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; i++) n += __popcll(__ballot(top[i] > least || (top[i] == least && first[i] <= mid)));
    if (n >= k) hi = mid;
    else lo = mid;
  }
  return hi;
}

// The k largest of the block's values v (-inf: none), column(i) thread-wise theirs, by every thread: emit(rank, value, column), with
// -inf and -1 for the ranks there is nothing for. `between` runs beside the search for T.
template <int NT, class Column, class Between, class Emit>
__device__ __forceinline__ void select_top(TopLds<NT> &lds, const float (&v)[PER], int k, Column column, Between between, Emit emit) {
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  float top = v[0];
#pragma unroll
  for (int i = 1; i < PER; i++) top = fmaxf(top, v[i]);
  lds.tops[tid] = ordered(top);
  if (tid == 0) lds.count = 0;
  __syncthreads();
  if (wave == 0) {
    uint32_t least;
    const bool ties = find_least<NT>(lds, k, &least);
    if (tid == 0) lds.least = least, lds.upto = ties ? -1 : NOWHERE;
  }
  between();
  __syncthreads();
  const uint32_t least = lds.least;
  int upto = lds.upto;
  if (upto < 0) {
    int first = NOWHERE;
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (ordered(v[i]) == least) first = min(first, column(i));
    lds.first[tid] = first;
    __syncthreads();
    if (wave == 0) {
      upto = find_upto<NT>(lds, k, least);
      if (tid == 0) lds.upto = upto;
    }
    __syncthreads();
    upto = lds.upto;
  }
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const uint32_t u = ordered(v[i]);
    if (u >= least) {
      const int c = column(i);
      if (u > least || c <= upto) lds.found[atomicAdd(&lds.count, 1)] = (uint64_t)u << 32 | (uint32_t)~c;
    }
  }
  __syncthreads();
  const int n = lds.count;
  for (int i = tid; i < n; i += NT) {
    const uint64_t mine = lds.found[i];
    int rank = 0;
    for (int j = 0; j < n; j++) rank += lds.found[j] > mine;
    if (rank < k) emit(rank, value_of((uint32_t)(mine >> 32)), (int)~(uint32_t)mine);
  }
  for (int i = n + tid; i < k; i += NT) emit(i, NONE, -1);
}

// A row's largest logit and the logarithm of its sum, once they are known.
struct RowSums {
  float m, lse, entropy;
  int at;
};
__device__ __forceinline__ RowSums row_sums(float m, float s, float e, int at, bool greedy) {
  const float lse = logf(s);
  if (m == NONE || greedy) return {m, 0.0f, 0.0f, at};
  return {m, lse, lse - e / s * LN2, at};
}
__device__ __forceinline__ float logprob(float x, int column, const RowSums &r, const Inverse &t) {
  if (x == NONE || (t.greedy && column != r.at)) return NONE;
  return t.greedy ? 0.0f : half_less(x, r.m) * t.t * 2.0f - r.lse;
}
__device__ __forceinline__ void store_row(const LogprobArgs &a, int row, const RowSums &r, const Inverse &t) {
  const int id = gload(a.ids + row);
  const bool is = (uint32_t)id < (uint32_t)a.vocab;
  const float x = is ? logit(gload(a.logits + row * a.logits_sr + id)) : NONE;
  a.logprobs[row] = is ? logprob(x, id, r, t) : 0.0f;
  a.entropy[row] = r.entropy;
}

// A block: PER NT logits of a row.
template <int NT, bool WIDE> __global__ void __launch_bounds__(NT) logprobs_kernel(const LogprobArgs a) {
  constexpr int W = NT / 64;
  __shared__ TopLds<NT> lds;
  __shared__ float tops[W], ss[W], es[W];
  __shared__ int at;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, v0 = chunk * (PER * NT);
  const float *x = a.logits + row * a.logits_sr;
  const auto column = [&](int i) { return v0 + (WIDE ? i / 4 * (4 * NT) + 4 * tid + i % 4 : i * NT + tid); };
  float v[PER];
  if constexpr (WIDE) {  // rows end on 16 bytes too
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      f32x4 w = {NONE, NONE, NONE, NONE};
      if (column(i) < a.vocab) w = gload((const f32x4 *)(x + column(i)));
#pragma unroll
      for (int j = 0; j < 4; j++) v[i + j] = w[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = column(i) < a.vocab ? gload(x + column(i)) : NONE;
  }
  const Inverse t = inverse(a, row);
  float top = NONE;
#pragma unroll
  for (int i = 0; i < PER; i++) top = fmaxf(top, v[i] = logit(v[i]));
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  if (tid == 0) at = NOWHERE;
  float m = NONE;
  const auto sums = [&] {  // (behind a barrier)
#pragma unroll
    for (int i = 0; i < W; i++) m = fmaxf(m, tops[i]);
    float s = 0.0f, e = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const float y = log2_weight(v[i], m, t.log2), w = __builtin_amdgcn_exp2f(y);
      s += w, e = __builtin_fmaf(w, y, e);
    }
    s = wave_sum(s), e = wave_sum(e);
    if (lane == 0) ss[wave] = s, es[wave] = e;
    if (t.greedy)
#pragma unroll
      for (int i = 0; i < PER; i++)
        if (v[i] == m) atomicMin(&at, column(i));
  };
  const auto whole = [&] {  // (behind another)
    float s = 0.0f, e = 0.0f;
#pragma unroll
    for (int i = 0; i < W; i++) s += ss[i], e += es[i];
    return ChunkSums{m, s, e, at};
  };
  const int64_t unit = (int64_t)row * a.chunks + chunk;
  if (a.k) {
    RowSums r;
    bool known = false;
    select_top<NT>(lds, v, a.k, column, sums, [&](int rank, float value, int c) {
      if (a.chunks > 1) {
        a.top_values[unit * a.k + rank] = value, a.top_columns[unit * a.k + rank] = c;
        return;
      }
      if (!known) {
        const ChunkSums k = whole();
        r = row_sums(k.m, k.s, k.e, k.at, t.greedy), known = true;
      }
      a.values[(int64_t)row * a.k + rank] = logprob(value, c, r, t), a.labels[(int64_t)row * a.k + rank] = c;
    });
  } else {
    __syncthreads();
    sums();
    __syncthreads();
  }
  if (tid) return;
  const ChunkSums k = whole();
  if (a.chunks > 1) a.sums[unit] = k;
  else store_row(a, row, row_sums(k.m, k.s, k.e, k.at, t.greedy), t);
}

// A block: a row's chunks, up to 256, and their k largest, up to PER NT in all.
constexpr int JOIN = 256;
__global__ void __launch_bounds__(JOIN) logprobs_join_kernel(const LogprobArgs a) {
  constexpr int W = JOIN / 64;
  __shared__ TopLds<JOIN> lds;
  __shared__ float tops[W], ss[W], es[W];
  __shared__ int at;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.x;
  ChunkSums k = {NONE, 0.0f, 0.0f, NOWHERE};
  if (tid < a.chunks) k = a.sums[(int64_t)row * a.chunks + tid];
  const int n = a.chunks * a.k;
  float v[PER];
  int columns[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int e = tid + JOIN * i;
    v[i] = NONE, columns[i] = -1;
    if (e < n) v[i] = gload(a.top_values + (int64_t)row * n + e), columns[i] = gload(a.top_columns + (int64_t)row * n + e);
  }
  const Inverse t = inverse(a, row);
  const float top = wave_max(k.m);
  if (lane == 0) tops[wave] = top;
  if (tid == 0) at = NOWHERE;
  __syncthreads();
  float m = NONE;
#pragma unroll
  for (int i = 0; i < W; i++) m = fmaxf(m, tops[i]);
  const float y = log2_weight(k.m, m, t.log2), by = __builtin_amdgcn_exp2f(y);
  const float s = wave_sum(k.s * by), e = wave_sum(__builtin_fmaf(y, k.s, k.e) * by);
  if (lane == 0) ss[wave] = s, es[wave] = e;
  if (t.greedy && k.m == m) atomicMin(&at, k.at);
  __syncthreads();
  float s_all = 0.0f, e_all = 0.0f;
#pragma unroll
  for (int i = 0; i < W; i++) s_all += ss[i], e_all += es[i];
  const RowSums r = row_sums(m, s_all, e_all, at, t.greedy);
  if (tid == 0) store_row(a, row, r, t);
  if (a.k == 0) return;
  select_top<JOIN>(lds, v, a.k, [&](int i) { return columns[i]; }, [] {}, [&](int rank, float value, int c) {
    a.values[(int64_t)row * a.k + rank] = logprob(value, c, r, t), a.labels[(int64_t)row * a.k + rank] = c;
  });
}

static int logprobs_threads(const bt_logprobs_args *a) {
  return (int64_t)ceil_div(a->vocab, PER * 256) * std::max(a->k, 1) > PER * JOIN ? 1024 : 256;
}
static int logprobs_chunks(const bt_logprobs_args *a) { return ceil_div(a->vocab, PER * logprobs_threads(a)); }
static int check_logprobs(const bt_logprobs_args *a) {
  if (!a || !a->logits || !a->ids || !a->logprobs || !a->entropy || (a->k && (!a->values || !a->labels)))
    return fail(BT_EINVAL, "log probabilities need logits, ids and results");
  if ((a->logits | a->ids | a->t | a->logprobs | a->entropy | a->values | a->labels) % 4)
    return fail(BT_EINVAL, "log probabilities take tensors on 4-byte boundaries");
  if (a->rows < 1 || a->rows > 1 << 20 || a->vocab < 1 || a->vocab > MOST_VOCAB || a->k < 0 || a->k > MOST_K)
    return fail(BT_EINVAL, "log probabilities of %d rows of %d logits (each 1 to 2^20) with %d alternatives (0 to %d)", a->rows, a->vocab,
                a->k, MOST_K);
  if ((int64_t)a->rows * logprobs_chunks(a) * logprobs_threads(a) > 0xFFFFFFFFll)  // a grid counts its threads in 32 bits
    return fail(BT_EINVAL, "log probabilities of %d rows of %d logits are too large", a->rows, a->vocab);
  return BT_OK;
}
static uint64_t logprobs_bytes(const bt_logprobs_args *a) {
  const uint64_t chunks = logprobs_chunks(a);
  return chunks > 1 ? a->rows * chunks * (sizeof(ChunkSums) + 8 * (uint64_t)a->k) : 0;
}

}  // namespace bt

using namespace bt;

extern "C" {

int bt_logprobs_scratch(const bt_logprobs_args *a, uint64_t *bytes) {
  if (!bytes) return fail(BT_EINVAL, "no result pointer");
  if (int s = check_logprobs(a)) return s;
  *bytes = logprobs_bytes(a);
  return BT_OK;
}

int bt_logprobs(bt_runtime *rt, const bt_logprobs_args *a) {
  Runtime *r;
  if (int s = enter(rt, &r)) return s;
  if (int s = check_logprobs(a)) return s;
  const uint64_t need = logprobs_bytes(a);
  if (need && (!a->scratch || a->scratch % 16 || a->scratch_bytes < need))
    return fail(BT_EINVAL, "log probabilities need %llu bytes of 16-byte aligned scratch", (unsigned long long)need);
  LogprobArgs k;
  const auto f = [](uint64_t p) { return (float *)(uintptr_t)p; };
  k.logits = f(a->logits), k.t = f(a->t), k.ids = (const int32_t *)(uintptr_t)a->ids;
  k.logprobs = f(a->logprobs), k.entropy = f(a->entropy), k.values = f(a->values), k.labels = (int32_t *)(uintptr_t)a->labels;
  k.chunks = logprobs_chunks(a), k.vocab = a->vocab, k.k = a->k, k.logits_sr = a->logits_sr, k.t_sr = a->t_sr;
  const int64_t units = (int64_t)a->rows * k.chunks;
  k.sums = (ChunkSums *)(uintptr_t)a->scratch;
  k.top_values = (float *)(k.sums + units), k.top_columns = (int32_t *)(k.top_values + units * k.k);
  const bool wide = a->logits % 16 == 0 && a->logits_sr % 4 == 0 && a->vocab % 4 == 0;
  if (logprobs_threads(a) == 256) {
    if (wide) logprobs_kernel<256, true><<<(unsigned)units, 256, 0, r->stream>>>(k);
    else logprobs_kernel<256, false><<<(unsigned)units, 256, 0, r->stream>>>(k);
  } else {
    if (wide) logprobs_kernel<1024, true><<<(unsigned)units, 1024, 0, r->stream>>>(k);
    else logprobs_kernel<1024, false><<<(unsigned)units, 1024, 0, r->stream>>>(k);
  }
  BT_LAUNCHED("log probabilities");
  if (k.chunks > 1) {
    logprobs_join_kernel<<<(unsigned)a->rows, JOIN, 0, r->stream>>>(k);
    BT_LAUNCHED("log probabilities' join");
  }
  return BT_OK;
}

}  // extern "C"
