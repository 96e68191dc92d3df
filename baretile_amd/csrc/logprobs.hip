// Log probabilities of given tokens, each row's entropy and its likeliest tokens, from rows of logits.
//
// With p = softmax(t x) of a row, m its largest logit, y_j = t (x_j - m), S = sum exp(y_j): log p_j = y_j - log S, and the
// entropy -sum p_j log p_j = log S - sum exp(y_j) y_j / S (no difference of large numbers: both terms are at most
// log(vocab)). Rows are cut into segments, a block each, which walk through them a chunk at a time: a chunk's logits stay in
// registers while they are summed against a running maximum of the wave's and held against a bound. A second launch joins a row's
// segments; rows of one need none.
//
// The k largest: whatever is at least the bound goes to LDS, and where that gets full it ranks itself by counting, equal
// values by their column (so the order in which they came doesn't matter); the k first stay, and the last of them is the new
// bound. The first bound, and any that lets too much through, comes from a chunk's threads: where k of them have a largest
// value of T or more, so do the k largest of all, T found by halving over the threads' largest values (one wave's ballots).
// Where more threads tie at T than that is made for, only the columns up to the one that completes k threads count.
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
  int32_t vocab, k, chunks, turns;  // chunks: a row's segments of `turns` chunks
};

// A logit as it counts: NaN as -inf, +inf as the largest finite.
__device__ __forceinline__ float logit(float x) { return x != x ? NONE : fminf(x, LARGEST); }

// A row's inverse temperature t, below 0 or NaN as 0. Differences of logits are taken halved, so that they don't pass the
// largest number, and t is at least the smallest number there is, so that a t of 0 weighs every logit over -inf alike. Past FAR
// the factor 2 t log2(e) would pass the largest number: there it is a quarter of that, and the 4 comes after it.
constexpr float FAR = 0x1p126f;
struct Inverse {
  float log2, t;  // (log2: 2 t log2(e), or t log2(e) / 2 past FAR)
  bool greedy;  // an infinite t: the first of the largest alone
  __device__ __forceinline__ bool far() const { return t > FAR; }
};
__device__ __forceinline__ Inverse inverse(const LogprobArgs &a, int row) {
  float t = a.t ? gload(a.t + row * a.t_sr) : 1.0f;
  t = t > 0.0f ? t : 0.0f;
  constexpr float least = 1.401298464e-45f;
  return {fmaxf(fminf(t * (t > FAR ? 0.5f * LOG2E : 2.0f * LOG2E), LARGEST), least), fmaxf(t, least), t > LARGEST};
}
__device__ __forceinline__ float half_less(float x, float m) { return __builtin_fmaf(x, 0.5f, -0.5f * m); }
// log2 of a weight, down to where it is 0. (-inf - -inf and NaN: 0 weight.)
__device__ __forceinline__ float log2_near(float x, float m, const Inverse &t) { return fmaxf(half_less(x, m) * t.log2, -200.0f); }
__device__ __forceinline__ float log2_weight(float x, float m, const Inverse &t) {
  return t.far() ? fmaxf(half_less(x, m) * t.log2 * 4.0f, -200.0f) : log2_near(x, m, t);
}

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
// Values in LDS past which they are ranked: the k that stayed, and as many again.
__device__ __forceinline__ int full_of(int k) { return 2 * k + 16; }
constexpr int ROOM = 2 * MOST_K + 16 + PER * limit_of(MOST_K);  // what is there, and one chunk's within the limit
template <int NT> struct TopLds {
  uint64_t found[ROOM], best[MOST_K];
  uint32_t tops[NT];
  int32_t first[NT], counts[NT];
  float least;
  int32_t upto, came[3];  // (a chunk's count, while the last one's is read and the next one's cleared)
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

// The k largest of what the block's threads show it, by all of them together: chunks, then finish.
template <int NT> struct Top {
  TopLds<NT> &lds;
  int k, n = 0, turn = 0;  // values in LDS, by turns of the counts
  float least = NONE;      // what a value has to pass

  // Ahead of a chunk, where there are fewer than k yet: its bound, from the threads' largest values, by the first wave alone.
  __device__ __forceinline__ void begin(float top) {
    const int tid = threadIdx.x;
    lds.tops[tid] = ordered(top);
    __syncthreads();
    if (tid >= 64) return;
    uint32_t bound;
    const bool ties = find_least<NT>(lds, k, &bound);
    if (tid == 0) lds.least = value_of(bound), lds.upto = ties ? -1 : NOWHERE, lds.came[turn] = 0;
  }
  // A chunk's values v (-inf and NaN: none), the thread's largest among them, their columns (past every column before, or any order
  // in the first chunk), and whether another follows.
  template <class Column> __device__ __forceinline__ void chunk(const float (&v)[PER], float top, Column column, bool more) {
    if (n < k) {  // begun
      bounded(v, top, column);
    } else {
      push(v, top, column, [&](float x, int) { return x > least; });
      __syncthreads();
      const int came = lds.came[turn];
      if (n + came > ROOM) {  // all of it again, within the limit
        begin(top);
        bounded(v, top, column);
      } else {
        n += came;
        turn = turn == 2 ? 0 : turn + 1;
      }
    }
    if (more && (n > full_of(k) || (n >= k && least == NONE))) keep();
  }
  template <class Column, class In> __device__ __forceinline__ void push(const float (&v)[PER], float top, Column column, In in) {
    if (threadIdx.x == 0) lds.came[turn == 2 ? 0 : turn + 1] = 0;
    if (in(top, -1))  // (of most waves no thread, or a few)
#pragma unroll
      for (int i = 0; i < PER; i++)
        if (in(v[i], -1)) {
          const int c = column(i);
          if (in(v[i], c)) {
            const int at = n + atomicAdd(&lds.came[turn], 1);
            if (at < ROOM) lds.found[at] = (uint64_t)ordered(v[i]) << 32 | (uint32_t)~c;
          }
        }
  }
  // What of a chunk is at least its own bound (and passes the one there was).
  template <class Column> __device__ __forceinline__ void bounded(const float (&v)[PER], float top, Column column) {
    const int tid = threadIdx.x;
    __syncthreads();
    const float bound = lds.least;
    int upto = lds.upto;
    if (upto < 0) {
      int first = NOWHERE;
#pragma unroll
      for (int i = 0; i < PER; i++)
        if (v[i] == bound) first = min(first, column(i));
      lds.first[tid] = first;
      __syncthreads();
      if (tid < 64) {
        upto = find_upto<NT>(lds, k, ordered(bound));
        if (tid == 0) lds.upto = upto;
      }
      __syncthreads();
      upto = lds.upto;
    }
    push(v, top, column, [&](float x, int c) { return x > least && x >= bound && (c <= upto || x > bound); });
    __syncthreads();
    n += lds.came[turn], turn = turn == 2 ? 0 : turn + 1;
  }
  // to(rank, value in LDS) for the k first by rank; behind a barrier. More than a wave of them but no more than half the threads are
  // counted by several threads each, a slice of the others a thread (the join of 512 rows of 131072 with 64 alternatives 7.4 us, so 6.3).
  template <class To> __device__ __forceinline__ void ranked(To to) {
    const int span = n > 64 && n <= NT / 2 ? NT / 2 : NT, slices = NT / span, slice = threadIdx.x / span, i0 = threadIdx.x % span;
    const int each = (n + slices - 1) / slices, from = slice * each, end = min(from + each, n);
    for (int i = i0; i < n; i += span) {
      const uint64_t mine = lds.found[i];
      int rank = 0;
#pragma unroll 4
      for (int j = from; j < end; j++) rank += lds.found[j] > mine;
      if (slices == 1) {
        if (rank < k) to(rank, mine);
      } else {
        lds.counts[threadIdx.x] = rank;
      }
    }
    if (slices == 1) return;
    __syncthreads();
    if (slice || i0 >= n) return;
    int rank = 0;
    for (int l = 0; l < slices; l++) rank += lds.counts[l * span + i0];
    if (rank < k) to(rank, lds.found[i0]);
  }
  // Only the k first stay, and there is a bound from then on.
  __device__ __forceinline__ void keep() {
    ranked([&](int rank, uint64_t x) { lds.best[rank] = x; });
    __syncthreads();
    n = min(n, k);
    for (int i = threadIdx.x; i < n; i += NT) lds.found[i] = lds.best[i];
    if (n == k) least = value_of((uint32_t)(lds.best[k - 1] >> 32));
    __syncthreads();
  }
  // emit(rank, value, column), with -inf and -1 for the ranks there is nothing for.
  template <class Emit> __device__ __forceinline__ void finish(Emit emit) {
    ranked([&](int rank, uint64_t x) { emit(rank, value_of((uint32_t)(x >> 32)), (int)~(uint32_t)x); });
    for (int i = n + threadIdx.x; i < k; i += NT) emit(i, NONE, -1);
  }
};

// A row's largest logit and the logarithm of its sum, once they are known.
struct RowSums {
  float m, lse, entropy;
  int at;
};
__device__ __forceinline__ RowSums row_sums(const ChunkSums &r, bool greedy) {
  const float lse = logf(r.s);
  if (r.m == NONE || greedy) return {r.m, 0.0f, 0.0f, r.at};
  return {r.m, lse, lse - r.e / r.s * LN2, r.at};
}
// A block's waves' sums as one.
template <int W> __device__ __forceinline__ ChunkSums together(const ChunkSums (&waves)[W], const Inverse &t) {
  ChunkSums r = {NONE, 0.0f, 0.0f, NOWHERE};
#pragma unroll
  for (int i = 0; i < W; i++) r.m = fmaxf(r.m, waves[i].m);
#pragma unroll
  for (int i = 0; i < W; i++) {
    const ChunkSums w = waves[i];
    const float d = log2_weight(w.m, r.m, t), by = __builtin_amdgcn_exp2f(d);
    r.s = __builtin_fmaf(w.s, by, r.s), r.e = __builtin_fmaf(__builtin_fmaf(d, w.s, w.e), by, r.e);
    if (w.m == r.m) r.at = min(r.at, w.at);
  }
  return r;
}
__device__ __forceinline__ float logprob(float x, int column, const RowSums &r, const Inverse &t) {
  if (x == NONE || (t.greedy && column != r.at)) return NONE;
  return t.greedy ? 0.0f : half_less(x, r.m) * t.t * 2.0f - r.lse;
}
// The row's given token, requested ahead of the rest.
struct Given {
  int id;
  float x;
  bool is;
};
__device__ __forceinline__ Given given(const LogprobArgs &a, int row) {
  Given g;
  g.id = gload(a.ids + row), g.is = (uint32_t)g.id < (uint32_t)a.vocab;
  g.x = gload(a.logits + row * a.logits_sr + (g.is ? g.id : 0));
  return g;
}
__device__ __forceinline__ void store_row(const LogprobArgs &a, int row, const Given &g, const RowSums &r, const Inverse &t) {
  a.logprobs[row] = g.is ? logprob(logit(g.x), g.id, r, t) : 0.0f;
  a.entropy[row] = r.entropy;
}

// A wave's sums, from its lanes'.
__device__ __forceinline__ void store_sums(ChunkSums r, const Inverse &t, ChunkSums *to) {
  r.s = wave_sum(r.s), r.e = wave_sum(r.e);
  if (t.greedy)
    for (int d = 1; d < 64; d *= 2) r.at = min(r.at, __shfl_xor(r.at, d, 64));
  if ((threadIdx.x & 63) == 0) *to = r;
}

// A block: a segment of a row, `turns` chunks of PER NT logits. Sums are a thread's own, against a running maximum of its
// wave's; of the chunk that makes the bound they are made while the first wave looks for it. Memory bounds it where rows are many:
// 512 rows of 131072 with 20 alternatives (268 MB) 49 us where half of them are in the Infinity Cache, 59 where none is, 4.6
// TB/s, and a join of 5.8 and 6.4 (with 64 66 and 70, 6.3 and 7.0); 777 rows of 49152 without (153 MB) 24.3 and 27.2 us. One row of
// 49152 with 5 is latency: 5.9 us and a join of 4.5, 32 rows of 131072 with 20 9.2 and 11.2, and 6.2. Dropped: ranks counted over 4
// or 8 values at once (2 us more on the 49), a wave a chunk with no barrier (one row 5.4 us, but 32 13), the next chunk requested
// ahead of the one at work (three quarters of the blocks; alike).
template <int NT, bool WIDE> __global__ void __launch_bounds__(NT, NT == 256 ? 8 : 1) logprobs_kernel(const LogprobArgs a) {
  constexpr int W = NT / 64, CHUNK = PER * NT;
  __shared__ TopLds<NT> lds;
  __shared__ ChunkSums sums[W];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x / a.chunks, segment = blockIdx.x - row * a.chunks, from = segment * a.turns;
  const float *x = a.logits + row * a.logits_sr;
  const Inverse t = inverse(a, row);
  Given g = {};
  if (a.chunks == 1) g = given(a, row);
  Top<NT> largest{lds, a.k};
  ChunkSums r = {NONE, 0.0f, 0.0f, NOWHERE};
  // A chunk's 16 weights are summed in 32 bits, the thread's chunks in 64, so that the error doesn't grow with them (of equal
  // weights in 256 chunks 6 in 10^5, so 1 in 10^6; no case is slower). Weights are
  // against `ref`, which the wave's maximum passes by a factor of two before what was summed is moved to it: where it creeps up
  // from chunk to chunk the sums are rounded once a doubling.
  double s = 0.0, e = 0.0;
  float ref = NONE;
  const auto move = [&](float m) {
    const float d = log2_weight(ref, m, t), by = __builtin_amdgcn_exp2f(d);
    e = (e + d * s) * by, s *= by, ref = m;
  };
  const int end = min(from + a.turns, (a.vocab + CHUNK - 1) / CHUNK);
  for (int c = from; c < end; c++) {
    const int v0 = c * CHUNK;
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
    float top = NONE;  // NaNs count for nothing: not for a maximum, nor against a bound, nor as a weight
#pragma unroll
    for (int i = 0; i < PER; i++) top = fmaxf(top, v[i]);
    const float wave_top = wave_max(top);
    if (wave_top > LARGEST) {  // there are infinities
#pragma unroll
      for (int i = 0; i < PER; i++) v[i] = logit(v[i]);
      top = fminf(top, LARGEST);
    }
    if (a.k && largest.n < a.k) largest.begin(top);
    if (wave_top > r.m) {
      const float m = fminf(wave_top, LARGEST);
      if (m > r.m) r.at = NOWHERE;
      r.m = m;
      if (log2_weight(ref, m, t) < -1.0f) move(m);
    }
    if (t.greedy && r.at == NOWHERE)
#pragma unroll
      for (int i = PER - 1; i >= 0; i--)
        if (v[i] == r.m) r.at = column(i);  // the thread's first in this chunk: columns rise with i
    float chunk_s = 0.0f, chunk_e = 0.0f;
    const auto weigh = [&](auto log2) {
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const float y = log2(v[i], ref, t), w = __builtin_amdgcn_exp2f(y);
        chunk_s += w, chunk_e = __builtin_fmaf(w, y, chunk_e);
      }
    };
    if (__any(t.far())) weigh(log2_weight);  // (one t a row, so the wave's branch: a factor more for all of them costs 1 %)
    else weigh(log2_near);
    s += chunk_s, e += chunk_e;
    if (c + 1 == end) {
      if (ref != r.m) move(r.m);
      r.s = (float)s, r.e = (float)e;
      store_sums(r, t, &sums[wave]);
    }
    if (a.k) largest.chunk(v, top, column, c + 1 < end);
  }
  if (a.k == 0) __syncthreads();
  const int64_t unit = (int64_t)row * a.chunks + segment;
  if (a.chunks > 1) {
    if (tid == 0) a.sums[unit] = together(sums, t);
    if (a.k)
      largest.finish([&](int rank, float value, int c) {
        a.top_values[unit * a.k + rank] = value, a.top_columns[unit * a.k + rank] = c;
      });
    return;
  }
  const RowSums sum = row_sums(together(sums, t), t.greedy);
  if (tid == 0) store_row(a, row, g, sum, t);
  if (a.k)
    largest.finish([&](int rank, float value, int c) {
      a.values[(int64_t)row * a.k + rank] = logprob(value, c, sum, t), a.labels[(int64_t)row * a.k + rank] = c;
    });
}

// A block: a row's segments, up to 256, and their k largest, up to PER JOIN in all.
constexpr int JOIN = 256;
__global__ void __launch_bounds__(JOIN) logprobs_join_kernel(const LogprobArgs a) {
  constexpr int W = JOIN / 64;
  __shared__ TopLds<JOIN> lds;
  __shared__ ChunkSums sums[W];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.x;
  ChunkSums r = {NONE, 0.0f, 0.0f, NOWHERE};
  if (tid < a.chunks) r = a.sums[(int64_t)row * a.chunks + tid];
  const int n = a.chunks * a.k;
  float v[PER];
  int columns[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int e = tid + JOIN * i;
    v[i] = NONE, columns[i] = -1;
    if (JOIN * i < n && e < n) {
      // each segment's are in order: turned by another step each, so that no thread gets the largest of many (of 32 segments' 64, whose
      // largest would lie with four threads, the bound let 700 pass: 38 us)
      const int s = e / a.k, at = s * a.k + (e - s * a.k + (int)((uint32_t)s * 0x9E3779B1u >> 20)) % a.k;
      v[i] = gload(a.top_values + (int64_t)row * n + at), columns[i] = gload(a.top_columns + (int64_t)row * n + at);
    }
  }
  const Inverse t = inverse(a, row);
  const Given g = given(a, row);
  Top<JOIN> largest{lds, a.k};
  const float m = wave_max(r.m), d = log2_weight(r.m, m, t), by = __builtin_amdgcn_exp2f(d);
  if (r.m < m) r.at = NOWHERE;
  r.e = __builtin_fmaf(d, r.s, r.e) * by, r.s *= by, r.m = m;
  store_sums(r, t, &sums[wave]);
  if (a.k) {
    float top = NONE;
#pragma unroll
    for (int i = 0; i < PER; i++) top = fmaxf(top, v[i]);
    largest.begin(top);
    largest.chunk(v, top, [&](int i) { return columns[i]; }, false);
  } else {
    __syncthreads();
  }
  const RowSums sum = row_sums(together(sums, t), t.greedy);
  if (tid == 0) store_row(a, row, g, sum, t);
  if (a.k == 0) return;
  largest.finish([&](int rank, float value, int c) {
    a.values[(int64_t)row * a.k + rank] = logprob(value, c, sum, t), a.labels[(int64_t)row * a.k + rank] = c;
  });
}

// Blocks that fill the card: eight of 256 threads on each of the 256 CUs.
constexpr int BLOCKS = 2048;
// Threads of a block: more where a row's chunks' k largest would pass what the join takes. (512 rows of 131072 with 20
// alternatives, a chunk a block: 55 us by 256, 59 by 512, 100 by 1024, 83 by 128 and 136 by 64, whose chunks each bring k
// values to rank.)
static int logprobs_threads(const bt_logprobs_args *a) {
  return (int64_t)ceil_div(a->vocab, PER * 256) * std::max(a->k, 1) > PER * JOIN ? 1024 : 256;
}
// Chunks of a segment: one, until there are more than fill the card, which then pass a bound that most of their values
// don't: 512 rows of 131072 with 20 alternatives 61 us in 16384 segments, 47 in 2048, 55 in 4096, 52 in 1024. Without
// alternatives there is nothing to gain (777 rows of 49152 23.8 us, in segments of 4 chunks 26.8).
static int logprobs_turns(const bt_logprobs_args *a) {
  const int64_t chunks = ceil_div(a->vocab, PER * logprobs_threads(a));
  if (a->k == 0) return 1;
  return (int)std::max<int64_t>(1, std::min(chunks, a->rows * chunks / BLOCKS));
}
static int logprobs_chunks(const bt_logprobs_args *a) { return ceil_div(a->vocab, PER * logprobs_threads(a) * logprobs_turns(a)); }
static int check_logprobs(const bt_logprobs_args *a) {
  if (!a || !a->logits || !a->ids || !a->logprobs || !a->entropy || (a->k && (!a->values || !a->labels)))
    return fail(BT_EINVAL, "log probabilities need logits, ids and results");
  if ((a->logits | a->ids | a->t | a->logprobs | a->entropy | a->values | a->labels) % 4)
    return fail(BT_EINVAL, "log probabilities take tensors on 4-byte boundaries");
  if (a->rows < 1 || a->rows > 1 << 20 || a->vocab < 1 || a->vocab > MOST_VOCAB || a->k < 0 || a->k > MOST_K)
    return fail(BT_EINVAL, "log probabilities of %d rows of %d logits (each 1 to 2^20) with %d alternatives (0 to %d)", a->rows, a->vocab,
                a->k, MOST_K);
  // (a grid counts its threads in 32 bits)
  if ((int64_t)a->rows * a->vocab > 1ll << 36 || (int64_t)a->rows * logprobs_chunks(a) * logprobs_threads(a) > 0xFFFFFFFFll)
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
  k.chunks = logprobs_chunks(a), k.turns = logprobs_turns(a), k.vocab = a->vocab, k.k = a->k, k.logits_sr = a->logits_sr, k.t_sr = a->t_sr;
  const int64_t units = (int64_t)a->rows * k.chunks;
  k.sums = (ChunkSums *)(uintptr_t)a->scratch;
  k.top_values = (float *)(k.sums + units), k.top_columns = (int32_t *)(k.top_values + units * k.k);
  const bool wide = a->logits % 16 == 0 && a->logits_sr % 4 == 0 && a->vocab % 4 == 0;
  const auto launch = [&](auto kernel, int threads) { kernel<<<(unsigned)units, threads, 0, r->stream>>>(k); };
  if (logprobs_threads(a) == 256) wide ? launch(logprobs_kernel<256, true>, 256) : launch(logprobs_kernel<256, false>, 256);
  else wide ? launch(logprobs_kernel<1024, true>, 1024) : launch(logprobs_kernel<1024, false>, 1024);
  BT_LAUNCHED("log probabilities");
  if (k.chunks > 1) {
    logprobs_join_kernel<<<(unsigned)a->rows, JOIN, 0, r->stream>>>(k);
    BT_LAUNCHED("log probabilities' join");
  }
  return BT_OK;
}

}  // extern "C"
