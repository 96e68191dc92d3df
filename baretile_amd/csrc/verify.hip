// Drafted tokens checked against the target's probabilities, from random numbers that the caller draws.
//
// For a request whose rows bring a token and then its drafts, p_j = softmax(t_j x_j) of row j's logits is the target's choice
// of the token after row j, and q_j the distribution that the draft fed at row j was drawn from. Row j's draft d is
// accepted where u0_j q_j(d) < p_{j-1}(d). The first refusal, after row j, draws from max(p_j - q_{j+1}, 0); where every
// draft was accepted the last row draws from p: the first token whose running sum passes u1_j times the whole. Tokens
// so drawn are distributed as the target's own (speculative sampling, Leviathan, Kalman and Matias, 2023).
//
// A token depends on which side of a border a sum falls, so weights, sums and comparisons are in 64 bits throughout
// (matrix-free work that reads each logit once: HBM bounds it, then the 64-bit exponential). Three launches: each row's
// chunks give a maximum and a sum; each request's chunks find the first refusal from those and sum what is left to draw
// from; then one block a request finds the chunk and the token.
#include "common.h"
#include <algorithm>

namespace bt {

struct VerifyArgs {
  const float *logits, *probs, *t, *uniforms;
  const int32_t *ids, *starts;
  int32_t *tokens, *counts;
  int64_t logits_sr, probs_sr, t_sr, uniforms_sr;
  int32_t requests, rows, vocab, chunks, chunk;  // a row's chunks, and their tokens
  struct ChunkStat *stats;                       // [rows][chunks]
  double *left;                                  // [requests][chunks]
  struct Refusal *refusals;                      // [requests]
};
// A chunk's largest logit, where it first is, and the sum of exp(t (x - m)).
struct ChunkStat {
  double s;
  float m;
  int32_t at;
};
// Where a request draws: `accepted` drafts, row's maximum and sum of exp(t (x - m)), whether a draft was refused.
struct Refusal {
  double z;
  float m;
  int32_t accepted, refused, at;
};

constexpr int VT = 256;
constexpr float NONE = -__builtin_inff();

// A logit as it counts: NaN as -inf, +inf as the largest finite.
__device__ __forceinline__ float logit(float x) { return x != x ? NONE : fminf(x, 3.4028234663852886e38f); }
// An inverse temperature: at least 0 (a NaN is 0); infinity takes the first of the largest alone.
__device__ __forceinline__ float inverse(const VerifyArgs &a, int row) {
  const float t = a.t ? gload(a.t + row * a.t_sr) : 1.0f;
  return t > 0.0f ? t : 0.0f;
}
__device__ __forceinline__ bool greedy(float t) { return t > 3.4028234663852886e38f; }
// exp(t (x - m)), 0 for a logit that has no weight.
__device__ __forceinline__ double weight(float x, float m, float t) {
  return x == NONE ? 0.0 : exp((double)t * ((double)x - (double)m));
}

__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
  for (int d = 32; d; d /= 2) x += __shfl_xor(x, d, 64);
  return x;
}
__device__ __forceinline__ double block_sum64(double x, double *sums) {
  x = wave_sum64(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int i = 0; i < VT / 64; i++) all += sums[i];
  return all;
}

// Block (row, chunk): PER logits a thread, all loaded at once.
template <int PER> __global__ void __launch_bounds__(VT) verify_stats_kernel(const VerifyArgs a) {
  __shared__ double sums[VT / 64];
  __shared__ float tops[VT / 64];
  __shared__ int ats[VT / 64];
  const int row = blockIdx.x / a.chunks, c = blockIdx.x - row * a.chunks, tid = threadIdx.x;
  if (row >= gload(a.starts + a.requests)) return;  // row < rows by the grid
  const int v0 = c * a.chunk, end = min(a.vocab, v0 + a.chunk);
  const float *x = a.logits + row * a.logits_sr;
  const float t = inverse(a, row);
  float v[PER], top = NONE;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int e = v0 + tid + VT * i;
    v[i] = e < end ? gload(x + e) : NONE;
  }
#pragma unroll
  for (int i = 0; i < PER; i++) top = fmaxf(top, v[i] = logit(v[i]));
#pragma unroll
  for (int d = 32; d; d /= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  int at = 0x7FFFFFFF;
#pragma unroll
  for (int i = PER - 1; i >= 0; i--)
    if (v[i] == top) at = v0 + tid + VT * i;
#pragma unroll
  for (int d = 32; d; d /= 2) at = min(at, __shfl_xor(at, d, 64));
  if ((tid & 63) == 0) ats[tid >> 6] = at;
  double s = 0.0;
  if (!greedy(t))
#pragma unroll
    for (int i = 0; i < PER; i++) s += weight(v[i], top, t);
  s = block_sum64(s, sums);
  if (tid == 0) a.stats[(int64_t)row * a.chunks + c] = ChunkStat{s, top, min(min(ats[0], ats[1]), min(ats[2], ats[3]))};
}

// A row's maximum, its first place and its sum, from its chunks' (64 at most), by a wave; the chunk sums are added in order of lanes.
struct RowStat {
  double z;
  float m;
  int at;
};
__device__ __forceinline__ RowStat row_stat(const VerifyArgs &a, int row, float t, int lane) {
  ChunkStat s{0.0, NONE, 0x7FFFFFFF};
  if (lane < a.chunks) s = a.stats[(int64_t)row * a.chunks + lane];
  RowStat r;
  r.m = s.m;
#pragma unroll
  for (int d = 32; d; d /= 2) r.m = fmaxf(r.m, __shfl_xor(r.m, d, 64));
  r.at = s.m == r.m ? s.at : 0x7FFFFFFF;
#pragma unroll
  for (int d = 32; d; d /= 2) r.at = min(r.at, __shfl_xor(r.at, d, 64));
  r.z = wave_sum64(greedy(t) ? 0.0 : s.s * weight(s.m, r.m, t));
  return r;
}

// What the thread's PER tokens from e on, `step` apart, may still be drawn with: p, or where a draft was refused what p has
// over q. Every load is issued before the first is used.
template <int PER>
__device__ __forceinline__ void left_of(const VerifyArgs &a, const Refusal &f, int row, float t, int e, int step, int end,
                                        double (&out)[PER]) {
  float x[PER], q[PER];
  const double inv = 1.0 / f.z;
  const bool drawn = f.refused && a.probs;
  const float *logits = a.logits + row * a.logits_sr, *probs = drawn ? a.probs + (row + 1) * a.probs_sr : logits;
#pragma unroll
  for (int i = 0; i < PER; i++) x[i] = e + i * step < end ? gload(logits + e + i * step) : NONE;
  if (drawn) {
#pragma unroll
    for (int i = 0; i < PER; i++) q[i] = e + i * step < end ? gload(probs + e + i * step) : 0.0f;
  } else {
    const int d = f.refused ? gload(a.ids + row + 1) : -1;
#pragma unroll
    for (int i = 0; i < PER; i++) q[i] = e + i * step == d ? 1.0f : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const double p = weight(logit(x[i]), f.m, t) * inv;
    out[i] = q[i] != q[i] ? p : p > (double)q[i] ? p - (double)q[i] : 0.0;
  }
}
// The first row of request r, and its rows; within the rows there are, whatever starts holds.
__device__ __forceinline__ int request_rows(const VerifyArgs &a, int r, int *n) {
  const int s0 = gload(a.starts + r), s1 = gload(a.starts + r + 1), start = min(max(s0, 0), a.rows);
  *n = min(max(s1, start), a.rows) - start;
  return start;
}

// Block (request, chunk): the first refused draft, then the chunk's sum of what is left.
template <int PER> __global__ void __launch_bounds__(VT) verify_left_kernel(const VerifyArgs a) {
  __shared__ double sums[VT / 64];
  __shared__ int refused;
  __shared__ Refusal found;
  const int r = blockIdx.x / a.chunks, c = blockIdx.x - r * a.chunks, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int n;
  const int start = request_rows(a, r, &n);
  if (n <= 0) return;
  if (tid == 0) refused = n;
  __syncthreads();
  for (int i = 1 + w; i < n; i += VT / 64) {  // draft i, against the row before it
    const int row = start + i - 1, d = gload(a.ids + row + 1);
    const float t = inverse(a, row);
    const bool is = (uint32_t)d < (uint32_t)a.vocab;
    const float x = is ? logit(gload(a.logits + row * a.logits_sr + d)) : NONE;
    const double q = a.probs ? (is ? (double)gload(a.probs + (row + 1) * a.probs_sr + d) : 1.0) : 1.0;
    const double u = gload(a.uniforms + row + 1);
    const RowStat s = row_stat(a, row, t, lane);
    const bool ok = is && s.m != NONE && (greedy(t) ? d == s.at : u * q < weight(x, s.m, t) / s.z);
    if (!ok) {
      if (lane == 0) atomicMin(&refused, i);
      break;
    }
  }
  __syncthreads();
  if (w == 0) {
    const int accepted = refused - 1, row = start + accepted;
    const RowStat s = row_stat(a, row, inverse(a, row), lane);
    if (lane == 0) found = Refusal{s.z, s.m, accepted, refused < n, s.at};
  }
  __syncthreads();
  const Refusal f = found;
  if (tid == 0 && c == 0) a.refusals[r] = f;
  const int row = start + f.accepted;
  const float t = inverse(a, row);
  if (greedy(t) || f.m == NONE) return;
  const int v0 = c * a.chunk, end = min(a.vocab, v0 + a.chunk);
  if (!f.refused) {  // the chunk's share of p is known already
    const ChunkStat k = a.stats[(int64_t)row * a.chunks + c];
    if (tid == 0) a.left[(int64_t)r * a.chunks + c] = k.s * weight(k.m, f.m, t) / f.z;
    return;
  }
  double left[PER], s = 0.0;
  left_of<PER>(a, f, row, t, v0 + tid, VT, end, left);
#pragma unroll
  for (int i = 0; i < PER; i++) s += left[i];
  s = block_sum64(s, sums);
  if (tid == 0) a.left[(int64_t)r * a.chunks + c] = s;
}

// Block (request): the token, then the request's rows of the result.
template <int PER> __global__ void __launch_bounds__(VT) verify_draw_kernel(const VerifyArgs a) {
  __shared__ double sums[VT / 64], goal;
  __shared__ int chunk, token, other, lasts[VT / 64];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  int n;
  const int start = request_rows(a, r, &n);
  if (r == 0)  // rows behind the last request's
    for (int j = max(0, gload(a.starts + a.requests)) + tid; j < a.rows; j += VT) a.tokens[j] = -1;
  if (n <= 0) {
    if (tid == 0) a.counts[r] = 0;
    return;
  }
  Refusal f = a.refusals[r];
  const int row = start + f.accepted;
  const float t = inverse(a, row);
  if (f.m == NONE || greedy(t)) {
    if (tid == 0) token = f.m == NONE ? -1 : f.at;
  } else {
    if (tid < 64) {
      double s = lane < a.chunks ? a.left[(int64_t)r * a.chunks + lane] : 0.0;
      double all = wave_sum64(s);
      if (!(all > 0.0)) {  // p nowhere over q, yet a draft refused (by rounding): all of p is drawn from
        const ChunkStat k = lane < a.chunks ? a.stats[(int64_t)row * a.chunks + lane] : ChunkStat{0.0, NONE, 0};
        s = k.s * weight(k.m, f.m, t) / f.z, all = wave_sum64(s);
        if (lane == 0) other = 1;
      } else if (lane == 0) {
        other = 0;
      }
      double upto = s;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const double up = __shfl_up(upto, d, 64);
        if (lane >= d) upto += up;
      }
      const double aim = (double)gload(a.uniforms + a.uniforms_sr + row) * all;
      // the first chunk whose running sum passes the aim; by rounding none may, then the last with any weight
      const uint64_t past = __ballot(upto > aim && s > 0.0), any = __ballot(s > 0.0);
      const int pick = past ? __builtin_ctzll(past) : any ? 63 - __builtin_clzll(any) : 0;
      if (lane == pick) chunk = pick, goal = aim - (upto - s);
    }
    __syncthreads();
    if (other) f.refused = 0;
    // PER tokens in a row a thread; its running sum over the threads before it, as the block's order has it
    const int v0 = chunk * a.chunk + tid * PER, w = tid >> 6;
    double left[PER], s = 0.0;
    left_of<PER>(a, f, row, t, v0, 1, min(a.vocab, (chunk + 1) * a.chunk), left);
    int last = -1;
#pragma unroll
    for (int i = 0; i < PER; i++) s += left[i], last = left[i] > 0.0 ? v0 + i : last;
    double upto = s;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double up = __shfl_up(upto, d, 64);
      if (lane >= d) upto += up;
    }
#pragma unroll
    for (int d = 32; d; d /= 2) last = max(last, __shfl_xor(last, d, 64));
    if (lane == 63) sums[w] = upto, lasts[w] = last;
    if (tid == 0) token = 0x7FFFFFFF;
    __syncthreads();
    double before = 0.0;
#pragma unroll
    for (int i = 0; i < VT / 64; i++) before += i < w ? sums[i] : 0.0;
    before += upto - s;
    if (before + s > goal) {  // the first token past the goal is the lowest that any thread finds
      int pick = 0x7FFFFFFF;
      double sum = before;
#pragma unroll
      for (int i = 0; i < PER; i++) {
        sum += left[i];
        if (pick == 0x7FFFFFFF && left[i] > 0.0 && sum > goal) pick = v0 + i;
      }
      atomicMin(&token, pick);
    }
    __syncthreads();
    if (tid == 0 && token == 0x7FFFFFFF)  // by rounding none passes it: the last with any weight
      token = max(max(lasts[0], lasts[1]), max(lasts[2], lasts[3]));
  }
  __syncthreads();
  for (int i = tid; i < n; i += VT)
    a.tokens[start + i] = i < f.accepted ? gload(a.ids + start + i + 1) : i == f.accepted ? token : -1;
  if (tid == 0) a.counts[r] = f.accepted + (token >= 0);
}

// How a call's rows are cut: 64 chunks at most (a lane a chunk where they join).
static void verify_chunks(const bt_verify_args *a, int *chunk, int *chunks) {
  int per = 8;  // logits a thread
  while ((int64_t)per * VT * 64 < a->vocab) per *= 2;
  *chunk = per * VT;
  *chunks = ceil_div(a->vocab, *chunk);
}
static int check_verify(const bt_verify_args *a) {
  if (!a || !a->logits || !a->ids || !a->starts || !a->uniforms || !a->tokens || !a->counts)
    return fail(BT_EINVAL, "verifying drafts needs logits, ids, starts, uniforms and results");
  if ((a->logits | a->probs | a->t | a->uniforms | a->ids | a->starts | a->tokens | a->counts) % 4)
    return fail(BT_EINVAL, "verifying drafts takes tensors on 4-byte boundaries");
  if (a->requests < 1 || a->rows < 1 || a->vocab < 1 || a->vocab > 1 << 20 || a->requests > 1 << 20 || a->rows > 1 << 20)
    return fail(BT_EINVAL, "verifying %d requests' %d rows of %d logits (each 1 to 2^20)", a->requests, a->rows, a->vocab);
  return BT_OK;
}
static uint64_t verify_bytes(const bt_verify_args *a) {
  int chunk, chunks;
  verify_chunks(a, &chunk, &chunks);
  return (uint64_t)a->rows * chunks * sizeof(ChunkStat) + (uint64_t)a->requests * (chunks * 8 + sizeof(Refusal));
}

template <int PER> static int launch_verify(const VerifyArgs &k, hipStream_t s) {
  verify_stats_kernel<PER><<<(unsigned)(k.rows * k.chunks), VT, 0, s>>>(k);
  BT_LAUNCHED("verifying drafts");
  verify_left_kernel<PER><<<(unsigned)(k.requests * k.chunks), VT, 0, s>>>(k);
  BT_LAUNCHED("verifying drafts");
  verify_draw_kernel<PER><<<(unsigned)k.requests, VT, 0, s>>>(k);
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
  k.tokens = (int32_t *)(uintptr_t)a->tokens, k.counts = (int32_t *)(uintptr_t)a->counts;
  k.logits_sr = a->logits_sr, k.probs_sr = a->probs_sr, k.t_sr = a->t_sr, k.uniforms_sr = a->uniforms_sr;
  k.requests = a->requests, k.rows = a->rows, k.vocab = a->vocab;
  verify_chunks(a, &k.chunk, &k.chunks);
  k.stats = (ChunkStat *)(uintptr_t)a->scratch;
  k.refusals = (Refusal *)(k.stats + (int64_t)a->rows * k.chunks);
  k.left = (double *)(k.refusals + a->requests);
  const int64_t blocks = (int64_t)std::max(a->rows, a->requests) * k.chunks;
  if (blocks > 0x7FFFFFFF) return fail(BT_EINVAL, "verifying %d rows of %d logits is too large", a->rows, a->vocab);
  switch (k.chunk / VT) {
    case 8: return launch_verify<8>(k, r->stream);
    case 16: return launch_verify<16>(k, r->stream);
    case 32: return launch_verify<32>(k, r->stream);
    default: return launch_verify<64>(k, r->stream);
  }
}

}  // extern "C"
