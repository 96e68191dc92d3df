// Drafted tokens checked against the target's probabilities, from random numbers that the caller draws.
//
// For a request whose rows bring a token and then its drafts (behind a prompt's other rows, where `drafts` counts them), p_j =
// softmax(t_j x_j) of row j's logits is the target's choice of the token after row j, and q_j the distribution that the draft fed at row j was drawn from. Row j's draft d is
// accepted where u0_j q_j(d) < p_{j-1}(d). The first refusal, after row j, draws from max(p_j - q_{j+1}, 0); where every
// draft was accepted the last row draws from p: the first token whose running sum passes u1_j times the whole. Tokens
// so drawn are distributed as the target's own (speculative sampling: Leviathan, Kalman and Matias, 2023).
//
// A token depends on which side of a border a sum falls, so weights, sums and comparisons are in 64 bits throughout, and
// what is drawn from stays unnormalized, so that equal weights add without rounding. Three launches: every row's chunks, a wave
// each, give a maximum and a sum (each logit read once, weighed once against its chunk's maximum); each request's chunks find
// the first refusal from those and sum what is left (only where a draft was refused and its distribution given does that
// read the row again); then a wave a request picks the chunk and the token.
#include "common.h"
#include <algorithm>

namespace bt {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// A chunk's largest logit, where it first is, and the sum of exp(t (x - m)).
struct ChunkStat {
  double s;
  float m;
  int32_t at;
};
// Where a request draws: after `accepted` drafts, from that row, with its maximum and sum and its number in [0, 1).
struct Draw {
  double z, t2;
  float m, u;
  int32_t accepted, refused, without, token;  // without: the token that a certain draft takes out, or -1; token: where there
};                                            // is nothing to draw, the one to take (-1: none)
struct VerifyArgs {
  const float *logits, *probs, *t, *uniforms;
  const int32_t *ids, *starts;
  int32_t *tokens, *counts;
  ChunkStat *stats;  // [rows][chunks]
  Draw *draws;       // [requests]
  double *left;      // [requests][chunks]: what is left to draw from
  int64_t logits_sr, probs_sr, t_sr, uniforms_sr;
  int32_t requests, rows, vocab, chunks;
  const int32_t *drafts;  // or null: all of a request's rows but its first
};

constexpr int WAVES = 4;   // of a block; a chunk each
constexpr int KEPT = 64;   // rows of a request whose sums a block keeps
constexpr float NONE = -__builtin_inff();
constexpr int NOWHERE = 0x7FFFFFFF;

// A logit as it counts: NaN as -inf, +inf as the largest finite.
__device__ __forceinline__ float logit(float x) { return x != x ? NONE : fminf(x, 3.4028234663852886e38f); }
// An inverse temperature: at least 0 (a NaN is 0); infinity takes the first of the largest alone.
__device__ __forceinline__ float inverse(const VerifyArgs &a, int row) {
  const float t = a.t ? gload(a.t + row * a.t_sr) : 1.0f;
  return t > 0.0f ? t : 0.0f;
}
__device__ __forceinline__ bool greedy(float t) { return t > 3.4028234663852886e38f; }
// t log2(e), as weight() takes it.
__device__ __forceinline__ double in_log2(float t) { return (double)t * 1.4426950408889634074; }

// exp(t (x - m)) as 2^((x - m) t2), t2 = t log2(e): 2^n by the exponent and 2^f, |f| <= 1/2, by the polynomial of degree 9
// through it at the Chebyshev points, its constant set to 1 so that the largest weigh exactly that (3.8e-14 relative; a draw over
// 2^17 tokens falls on the other side of a border less than once in 10^8). 16 64-bit instructions, where exp() takes about 40
// and bounded the first launch. -inf and what is below 2^-1074 give 0.
__device__ __forceinline__ double weight(float x, float m, double t2) {
  const double y = fmax(((double)x - (double)m) * t2, -2000.0), n = rint(y), f = y - n;
  double p = 0x1.b6571e229927fp-24;
  p = fma(p, f, 0x1.63ef9699120e2p-20);
  p = fma(p, f, 0x1.ffcb767842e11p-17);
  p = fma(p, f, 0x1.43088e2580989p-13);
  p = fma(p, f, 0x1.5d87fe908fb19p-10);
  p = fma(p, f, 0x1.3b2ab72b175e1p-7);
  p = fma(p, f, 0x1.c6b08d7044117p-5);
  p = fma(p, f, 0x1.ebfbdff8149f2p-3);
  p = fma(p, f, 0x1.62e42fefa39f7p-1);
  p = fma(p, f, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}

// Reductions over a wave's lanes with no trip through LDS (as wave_sum in common.h): lane swaps by 32 and 16, then DPP moves
// within rows of 16, each step pairing lanes symmetrically, so every lane ends with the same bits.
template <int CTRL> __device__ __forceinline__ double moved(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)b, (int)b, CTRL, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(b >> 32), (int)(b >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double x) {
  const auto pair = [](uint32_t lo, uint32_t hi) { return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo); };
  uint64_t b = __builtin_bit_cast(uint64_t, x);
  auto lo = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
  auto hi = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
  x = pair(lo[0], hi[0]) + pair(lo[1], hi[1]);
  b = __builtin_bit_cast(uint64_t, x);
  lo = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
  hi = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
  x = pair(lo[0], hi[0]) + pair(lo[1], hi[1]);
  x += moved<0x128>(x);  // row_ror 8
  x += moved<0x141>(x);  // row_half_mirror
  x += moved<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  return x + moved<0xB1>(x);  // quad_perm [1, 0, 3, 2]
}
template <class F> __device__ __forceinline__ uint32_t wave_fold(uint32_t x, F f) {
  const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = f(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = f(b[0], b[1]);
  x = f(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x128, 0xF, 0xF, false));
  x = f(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x141, 0xF, 0xF, false));
  x = f(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x4E, 0xF, 0xF, false));
  return f(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0xB1, 0xF, 0xF, false));
}
__device__ __forceinline__ float wave_max(float x) {
  return __uint_as_float(wave_fold(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ int wave_min(int x) {
  return (int)wave_fold((uint32_t)x, [](uint32_t a, uint32_t b) { return (uint32_t)min((int)a, (int)b); });
}
// The sum over the lanes before this one: shifts within rows of 16, then each row's last sum to the rows after it.
template <int CTRL, int ROWS> __device__ __forceinline__ double shifted(double x) {  // 0 where no lane gives a value
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_before(double x) {
  double upto = x;
  upto += shifted<0x111, 0xF>(upto);  // row_shr 1, 2, 4, 8
  upto += shifted<0x112, 0xF>(upto);
  upto += shifted<0x114, 0xF>(upto);
  upto += shifted<0x118, 0xF>(upto);
  upto += shifted<0x142, 0xA>(upto);  // row_bcast 15 into rows 1 and 3
  upto += shifted<0x143, 0xC>(upto);  // row_bcast 31 into rows 2 and 3
  return upto - x;
}

// PER values of a chunk of 64 PER, four in a row a lane at a time where rows allow 16-byte loads (WIDE), else one; `none`
// past the row's end. place(i) is value i's.
template <int PER, bool WIDE> struct Chunk {
  static __device__ __forceinline__ int place(int lane, int i) { return WIDE ? i / 4 * 256 + 4 * lane + i % 4 : 64 * i + lane; }
  static __device__ __forceinline__ void load(float (&v)[PER], const float *row, int v0, int vocab, int lane, float none) {
    if constexpr (WIDE) {  // rows end on 16 bytes too
#pragma unroll
      for (int i = 0; i < PER; i += 4) {
        const int e = v0 + place(lane, i);
        f32x4 w = {none, none, none, none};
        if (e < vocab) w = gload((const f32x4 *)(row + e));
#pragma unroll
        for (int k = 0; k < 4; k++) v[i + k] = w[k];
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const int e = v0 + place(lane, i);
        v[i] = e < vocab ? gload(row + e) : none;
      }
    }
  }
};

// Wave (row, chunk): no LDS, no barrier.
template <int PER, bool WIDE> __global__ void __launch_bounds__(64 * WAVES) verify_stats_kernel(const VerifyArgs a) {
  const int lane = threadIdx.x & 63, at = blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = at / a.chunks, c = at - row * a.chunks, v0 = c * 64 * PER;
  if (row >= min(gload(a.starts + a.requests), a.rows)) return;
  float v[PER], top = NONE;
  Chunk<PER, WIDE>::load(v, a.logits + row * a.logits_sr, v0, a.vocab, lane, NONE);
  const float t = inverse(a, row);
#pragma unroll
  for (int i = 0; i < PER; i++) top = fmaxf(top, v[i] = logit(v[i]));
  top = wave_max(top);
  double s = 0.0;
  int first = NOWHERE;
  if (greedy(t)) {
#pragma unroll
    for (int i = PER - 1; i >= 0; i--)
      if (v[i] == top) first = v0 + Chunk<PER, WIDE>::place(lane, i);
    first = wave_min(first);
  } else if (top != NONE) {
    const double t2 = in_log2(t);
#pragma unroll
    for (int i = 0; i < PER; i++) s += weight(v[i], top, t2);
    s = wave_sum64(s);
  }
  if (lane == 0) a.stats[(int64_t)row * a.chunks + c] = ChunkStat{s, top, first};
}

// A row's maximum, its first place (greedy rows) and its sum, by a wave from the row's chunks.
struct RowStat {
  double z;
  float m, t;
  int at;
};
__device__ __forceinline__ RowStat row_stat(const VerifyArgs &a, int row, float t, int lane) {
  const ChunkStat *stats = a.stats + (int64_t)row * a.chunks;
  constexpr int G = 4;  // chunks a lane loads at once: all of up to 256
  RowStat r{0.0, NONE, t, NOWHERE};
  ChunkStat s[G];
#pragma unroll
  for (int i = 0; i < G; i++) {
    s[i] = stats[min(lane + 64 * i, a.chunks - 1)];  // past the last it is read again and left out
    if (lane + 64 * i < a.chunks) r.m = fmaxf(r.m, s[i].m);
  }
  for (int c = lane + 64 * G; c < a.chunks; c += 64) r.m = fmaxf(r.m, stats[c].m);
  r.m = wave_max(r.m);
  if (r.m == NONE) return r;
  const double t2 = in_log2(t);
  const auto add = [&](const ChunkStat &k) {
    if (greedy(t)) r.at = k.m == r.m ? min(r.at, k.at) : r.at;
    else r.z += k.s * weight(k.m, r.m, t2);
  };
#pragma unroll
  for (int i = 0; i < G; i++)
    if (lane + 64 * i < a.chunks) add(s[i]);
  for (int c = lane + 64 * G; c < a.chunks; c += 64) add(stats[c]);
  if (greedy(t)) r.at = wave_min(r.at);
  else r.z = wave_sum64(r.z);
  return r;
}

// What chunk c's tokens may still be drawn with, times z: p, or where a draft was refused what p has over q.
template <int PER, bool WIDE>
__device__ __forceinline__ void left_of(const VerifyArgs &a, const Draw &f, int row, int c, int lane, double (&out)[PER]) {
  float x[PER], q[PER];
  const int v0 = c * 64 * PER;
  const bool drawn = f.refused && a.probs;
  Chunk<PER, WIDE>::load(x, a.logits + row * a.logits_sr, v0, a.vocab, lane, NONE);
  if (drawn) Chunk<PER, WIDE>::load(q, a.probs + (row + 1) * a.probs_sr, v0, a.vocab, lane, 0.0f);
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const double p = weight(logit(x[i]), f.m, f.t2);
    if (drawn) out[i] = q[i] != q[i] ? p : fmax(fma(-(double)q[i], f.z, p), 0.0);
    else out[i] = v0 + Chunk<PER, WIDE>::place(lane, i) == f.without ? 0.0 : p;
  }
}
// The first row of request r that is verified, and how many are: all of its rows, or with drafts its last token's and that many
// drafts'. `ahead` rows of it lie before them. Within the rows there are, whatever starts and drafts hold.
__device__ __forceinline__ int request_rows(const VerifyArgs &a, int r, int *n, int *ahead) {
  const int s0 = gload(a.starts + r), s1 = gload(a.starts + r + 1), given = gload((a.drafts ? a.drafts : a.starts) + r);
  const int d = a.drafts ? given : NOWHERE;  // (a load either way: with a branch verify_draw_kernel took 5.7 us for 5.5)
  const int start = min(max(s0, 0), a.rows), rows = min(max(s1, start), a.rows) - start;
  *n = min(max(d, -1), rows - 1) + 1;
  *ahead = rows - *n;
  return start + *ahead;
}

// Block (request, 4 chunks): the first refused draft, found by every block for itself (so a request's drafts cost its chunks' number
// of searches, each as long as the drafts accepted), then what is left of a chunk a wave.
template <int PER, bool WIDE> __global__ void __launch_bounds__(64 * WAVES) verify_left_kernel(const VerifyArgs a) {
  __shared__ RowStat kept[KEPT];
  __shared__ int refusal;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (a.chunks + WAVES - 1) / WAVES, r = blockIdx.x / blocks, c = (blockIdx.x - r * blocks) * WAVES + w;
  int n, ahead;
  const int start = request_rows(a, r, &n, &ahead);
  if (n == 0) return;
  if (tid == 0) refusal = n;
  __syncthreads();
  for (int i = 1 + w; i <= n; i += WAVES) {  // draft i, against the row before it; past the last, that row's sums alone
    const int row = start + i - 1;
    const float t = inverse(a, row);
    int d = -1;
    float u = 0.0f, x = NONE, q = 1.0f;
    bool is = false;
    if (i < n) {
      d = gload(a.ids + row + 1), u = gload(a.uniforms + row + 1);
      is = (uint32_t)d < (uint32_t)a.vocab;
      const int at = is ? d : 0;
      x = logit(gload(a.logits + row * a.logits_sr + at));
      q = a.probs ? gload(a.probs + (row + 1) * a.probs_sr + at) : 1.0f;
    }
    const RowStat s = row_stat(a, row, t, lane);
    if (lane == 0 && i <= KEPT) kept[i - 1] = s;
    if (i < n && is && s.m != NONE && (greedy(t) ? d == s.at : (double)u * (double)q * s.z < weight(x, s.m, in_log2(t)))) continue;
    if (lane == 0) atomicMin(&refusal, i);
    break;
  }
  __syncthreads();
  Draw f;
  f.accepted = refusal - 1, f.refused = refusal < n;
  const int from = start + f.accepted;
  const RowStat s = refusal <= KEPT ? kept[refusal - 1] : row_stat(a, from, inverse(a, from), lane);
  const float t = s.t;
  f.u = c == 0 ? gload(a.uniforms + a.uniforms_sr + from) : 0.0f;
  f.z = s.z, f.m = s.m, f.t2 = in_log2(t), f.without = f.refused && !a.probs ? gload(a.ids + from + 1) : -1;
  const bool known = s.m == NONE || greedy(t);
  f.token = s.m == NONE ? -1 : greedy(t) ? s.at : NOWHERE;
  if (c == 0 && lane == 0) a.draws[r] = f;
  if (known || c >= a.chunks) return;
  double sum = 0.0;
  if ((f.refused && a.probs) || (f.without >= 0 && f.without / (64 * PER) == c)) {
    double v[PER];
    left_of<PER, WIDE>(a, f, from, c, lane, v);
#pragma unroll
    for (int i = 0; i < PER; i++) sum += v[i];
    sum = wave_sum64(sum);
  } else {  // p's share of the chunk is known
    const ChunkStat k = a.stats[(int64_t)from * a.chunks + c];
    sum = k.s * weight(k.m, f.m, f.t2);
  }
  if (lane == 0) a.left[(int64_t)r * a.chunks + c] = sum;
}

// Wave (request): the chunk, the token, and the request's rows of the result.
template <int PER, bool WIDE> __global__ void __launch_bounds__(64) verify_draw_kernel(const VerifyArgs a) {
  const int r = blockIdx.x, lane = threadIdx.x;
  if (r == a.requests) {  // rows of no request: ahead of the first's and behind the last's
    const int first = min(gload(a.starts), a.rows), last = min(max(gload(a.starts + a.requests), 0), a.rows);
    for (int j = lane; j < first; j += 64) a.tokens[j] = -1;
    for (int j = last + lane; j < a.rows; j += 64) a.tokens[j] = -1;
    return;
  }
  constexpr int KEEP = 4;  // sums a lane keeps: of up to 256 chunks all
  const double *left = a.left + (int64_t)r * a.chunks;
  const int each = (a.chunks + 63) / 64, c0 = lane * each, c1 = min(c0 + each, a.chunks);  // the lane's chunks
  Draw f = a.draws[r];
  double kept[KEEP];
#pragma unroll
  for (int i = 0; i < KEEP; i++) kept[i] = gload(left + min(c0 + i, a.chunks - 1));  // requested with the rest, used or not
  int n, ahead;
  const int start = request_rows(a, r, &n, &ahead);
  for (int i = lane; i < ahead; i += 64) a.tokens[start - ahead + i] = -1;
  if (n == 0) {
    if (lane == 0) a.counts[r] = 0;
    return;
  }
  if (f.token == NOWHERE) {
    const int row = start + f.accepted;
    const auto each_of = [&](auto value, auto step) {  // step(c, value(c, its kept sum)) for the lane's chunks in order
#pragma unroll
      for (int i = 0; i < KEEP; i++)
        if (c0 + i < c1) step(c0 + i, value(c0 + i, kept[i]));
      for (int c = c0 + KEEP; c < c1; c++) step(c, value(c, gload(left + c)));
    };
    double s = 0.0;
    const auto as_left = [](int, double l) { return l; };
    each_of(as_left, [&](int, double l) { s += l; });
    double all = wave_sum64(s);
    const bool none = !(all > 0.0);  // p nowhere over q, yet a draft refused (by rounding): all of p is drawn from
    const ChunkStat *stats = a.stats + (int64_t)row * a.chunks;
    const auto as_weighed = [&](int c, double) { return stats[c].s * weight(stats[c].m, f.m, f.t2); };
    if (none) {
      f.refused = 0, f.without = -1, s = 0.0;
      each_of(as_weighed, [&](int, double l) { s += l; });
      all = wave_sum64(s);
    }
    double goal = (double)f.u * all, upto = wave_before(s), from = 0.0;
    // the first chunk whose running sum passes the goal; by rounding none may, then the last with any weight
    int pick = NOWHERE, last = -1;
    const auto look = [&](int c, double l) {
      if (l > 0.0) last = c;
      if (pick == NOWHERE && l > 0.0 && upto + l > goal) pick = c, from = upto;
      upto += l;
    };
    if (none) each_of(as_weighed, look);
    else each_of(as_left, look);
    uint64_t who = __ballot(pick != NOWHERE);
    if (who) {
      const int l = __builtin_ctzll(who);
      pick = __shfl(pick, l, 64), goal -= __shfl(from, l, 64);
    } else {
      who = __ballot(last >= 0);
      pick = who ? __shfl(last, 63 - __builtin_clzll(who), 64) : 0, goal = __builtin_inf();
    }
    pick = __builtin_amdgcn_readfirstlane(pick);
    // the chunk's tokens in order: RUN in a row a lane, 64 RUN a turn
    constexpr int RUN = WIDE ? 4 : 1, TURNS = PER / RUN;
    double v[PER], before[TURNS], carry = 0.0;
    left_of<PER, WIDE>(a, f, row, pick, lane, v);
#pragma unroll
    for (int i = 0; i < TURNS; i++) {
      double mine = 0.0;
#pragma unroll
      for (int k = 0; k < RUN; k++) mine += v[RUN * i + k];
      before[i] = wave_before(mine);
      const double turn = __shfl(before[i] + mine, 63, 64);
      before[i] += carry, carry += turn;
    }
    int best = NOWHERE;
    last = -1;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int e = pick * 64 * PER + Chunk<PER, WIDE>::place(lane, i);
      before[i / RUN] += v[i];
      if (v[i] > 0.0) {
        last = e;
        if (best == NOWHERE && before[i / RUN] > goal) best = e;
      }
    }
    best = wave_min(best);
    f.token = best != NOWHERE ? best : -wave_min(-last);
  }
  for (int i = lane; i < n; i += 64)
    a.tokens[start + i] = i < f.accepted ? gload(a.ids + start + i + 1) : i == f.accepted ? f.token : -1;
  if (lane == 0) a.counts[r] = f.accepted + (f.token >= 0);
}

// Logits a lane of a chunk's 64: 8 up to 2^22 logits, where larger chunks would leave waves too few to fill the card (5 rows of
// 49152 12.3 us), else 16, which spreads a chunk's maximum and sums over more of them (112 rows of 131072 in 32 requests: the three
// launches 15.8, 9.3 and 5.5 us; with 32 a lane, whose draw is one wave's long run, 16.7, 10.6 and 8.8).
static int verify_per(const bt_verify_args *a) { return (int64_t)a->rows * a->vocab <= 1 << 22 ? 8 : 16; }
static int verify_chunks(const bt_verify_args *a) { return ceil_div(a->vocab, 64 * verify_per(a)); }
static int check_verify(const bt_verify_args *a) {
  if (!a || !a->logits || !a->ids || !a->starts || !a->uniforms || !a->tokens || !a->counts)
    return fail(BT_EINVAL, "verifying drafts needs logits, ids, starts, uniforms and results");
  if ((a->logits | a->probs | a->t | a->uniforms | a->ids | a->starts | a->tokens | a->counts | a->drafts) % 4)
    return fail(BT_EINVAL, "verifying drafts takes tensors on 4-byte boundaries");
  if (a->requests < 1 || a->rows < 1 || a->vocab < 1 || a->vocab > 1 << 20 || a->requests > 1 << 20 || a->rows > 1 << 20)
    return fail(BT_EINVAL, "verifying %d requests' %d rows of %d logits (each 1 to 2^20)", a->requests, a->rows, a->vocab);
  // a grid counts its threads in 32 bits: a wave a chunk of every row, and of every request, a block of 4 at least
  if ((int64_t)std::max(a->rows, a->requests) * (verify_chunks(a) + WAVES) * 64 > 0xFFFFFFFFll)
    return fail(BT_EINVAL, "verifying %d requests' %d rows of %d logits is too large", a->requests, a->rows, a->vocab);
  return BT_OK;
}
static uint64_t verify_bytes(const bt_verify_args *a) {
  return (uint64_t)a->rows * verify_chunks(a) * sizeof(ChunkStat) + (uint64_t)a->requests * (sizeof(Draw) + 8 * verify_chunks(a));
}

template <int PER, bool WIDE> static int launch_verify(const VerifyArgs &k, hipStream_t s) {
  verify_stats_kernel<PER, WIDE><<<(unsigned)ceil_div((int64_t)k.rows * k.chunks, WAVES), 64 * WAVES, 0, s>>>(k);
  BT_LAUNCHED("verifying drafts");
  verify_left_kernel<PER, WIDE><<<(unsigned)(k.requests * ceil_div(k.chunks, WAVES)), 64 * WAVES, 0, s>>>(k);
  BT_LAUNCHED("verifying drafts");
  verify_draw_kernel<PER, WIDE><<<(unsigned)(k.requests + 1), 64, 0, s>>>(k);
  BT_LAUNCHED("verifying drafts");
  return BT_OK;
}

}  // namespace bt

using namespace bt;

extern "C" {

int bt_verify_scratch(const bt_verify_args *a, uint64_t *bytes) {
  if (!bytes) return fail(BT_EINVAL, "no result pointer");
  if (int s = check_verify(a)) return s;
  *bytes = verify_bytes(a);
  return BT_OK;
}

int bt_verify(bt_runtime *rt, const bt_verify_args *a) {
  Runtime *r;
  if (int s = enter(rt, &r)) return s;
  if (int s = check_verify(a)) return s;
  if (!a->scratch || a->scratch % 16 || a->scratch_bytes < verify_bytes(a))
    return fail(BT_EINVAL, "verifying drafts needs %llu bytes of 16-byte aligned scratch", (unsigned long long)verify_bytes(a));
  VerifyArgs k;
  const auto f = [](uint64_t p) { return (const float *)(uintptr_t)p; };
  k.logits = f(a->logits), k.probs = f(a->probs), k.t = f(a->t), k.uniforms = f(a->uniforms);
  k.ids = (const int32_t *)(uintptr_t)a->ids, k.starts = (const int32_t *)(uintptr_t)a->starts;
  k.drafts = (const int32_t *)(uintptr_t)a->drafts;
  k.tokens = (int32_t *)(uintptr_t)a->tokens, k.counts = (int32_t *)(uintptr_t)a->counts;
  k.chunks = verify_chunks(a);
  k.stats = (ChunkStat *)(uintptr_t)a->scratch;
  k.draws = (Draw *)(k.stats + (int64_t)a->rows * k.chunks), k.left = (double *)(k.draws + a->requests);
  k.logits_sr = a->logits_sr, k.probs_sr = a->probs_sr, k.t_sr = a->t_sr, k.uniforms_sr = a->uniforms_sr;
  k.requests = a->requests, k.rows = a->rows, k.vocab = a->vocab;
  const bool wide = a->logits % 16 == 0 && a->logits_sr % 4 == 0 && a->probs % 16 == 0 && a->probs_sr % 4 == 0 && a->vocab % 4 == 0;
  if (verify_per(a) == 8) return wide ? launch_verify<8, true>(k, r->stream) : launch_verify<8, false>(k, r->stream);
  return wide ? launch_verify<16, true>(k, r->stream) : launch_verify<16, false>(k, r->stream);
}

}  // extern "C"
