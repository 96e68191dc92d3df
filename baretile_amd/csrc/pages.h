// What the paged caches of 8 and of 4 bits share: a batch's requests and their rows found on the device, attention's running
// softmax, its parts and tiles, and the plan of a call.
#pragma once
#include "common.h"
#include <algorithm>

namespace bt {

typedef short bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int KB = 64;          // keys of a block
constexpr int MOST_PARTS = 32;  // parts of one request (64: of 65536 keys 23.0 us and a join of 7.6, for 23.0 + 4.6)
constexpr int SHORT = 16 * KB;  // keys that tables of one part a request hold at most
// Waves that attention's parts are for, over all key heads: 8 on each of the 256 CUs, which is what their registers allow at once
// (8 requests of up to 8191 keys: 19.7 us; with half as many 23.4, with half as many again 22.5).
constexpr int WAVES = 2048;
constexpr int MOST_REQUESTS = 2048;

struct PoolArgs {
  uint8_t *values;
  float *scales;
  int32_t pages, page_log2, kv;
};
struct BatchArgs {
  const int32_t *tables, *starts, *lengths, *parts;
  int64_t tables_sr;
  int32_t requests, width, rows;
};

// What one request of a batch is: its first row, rows and length, and which of its pieces a block takes.
struct Piece {
  int r, k, row0, n, len;
};
// The request whose pieces `before(i, starts[i])` .. `before(i + 1, ..)` hold piece `at`, found by the wave's lanes
// together: of more than 64 requests first which of 64 equal runs, then which of the run's, a trip to memory each (64 at a time
// from the first on, a put over 2048 requests 135 us, so 90; a search by halves would be a trip a step). Starts count within
// the rows there are and lengths hold their rows, whatever they say.
template <class F> __device__ __forceinline__ bool find_piece(const BatchArgs &b, int at, int lane, F before, Piece *p) {
  const auto held = [&](int s) { return min(max(s, 0), b.rows); };
  int base = 0;
  if (b.requests > 64) {
    const int run = (b.requests + 63) >> 6, i = min(lane * run, b.requests - 1);  // at most 32 of MOST_REQUESTS
    const uint64_t from = __ballot(before(i, held(gload(b.starts + i))) <= at);
    base = from ? min((63 - __builtin_clzll(from)) * run, b.requests - 1) : 0;
  }
  const int i = min(base + lane, b.requests - 1);
  int f0 = gload(b.starts + i), f1 = gload(b.starts + i + 1), len = gload(b.lengths + i);
  int lo = before(i, held(f0)), hi = before(i + 1, held(f1));
  asm volatile("" : "+v"(f0), "+v"(f1), "+v"(len), "+v"(lo), "+v"(hi));  // all requested at once, not once the piece is found
  const int s0 = held(f0), s1 = max(held(f1), s0);
  const uint64_t hit = __ballot(base + lane < b.requests && lo <= at && at < hi);
  if (!hit) return false;
  const int l = __builtin_ctzll(hit);
  p->r = base + l;
  p->k = at - __builtin_amdgcn_readlane(lo, l);
  p->row0 = __builtin_amdgcn_readlane(s0, l);
  p->n = __builtin_amdgcn_readlane(s1, l) - p->row0;
  p->len = max(__builtin_amdgcn_readlane(len, l), p->n);
  return true;
}

// Request r whole, as one piece.
__device__ __forceinline__ Piece whole_piece(const BatchArgs &b, int r) {
  int f0 = gload(b.starts + r), f1 = gload(b.starts + r + 1), len = gload(b.lengths + r);
  asm volatile("" : "+v"(f0), "+v"(f1), "+v"(len));  // all requested at once
  Piece p{r, 0, __builtin_amdgcn_readfirstlane(min(max(f0, 0), b.rows)), 0, 0};
  p.n = __builtin_amdgcn_readfirstlane(min(max(f1, p.row0), b.rows)) - p.row0;
  p.len = max(__builtin_amdgcn_readfirstlane(len), p.n);
  return p;
}

// ---- attention over pages --------------------------------------------------------------------------------------------

struct AttendArgs {
  PoolArgs c;
  BatchArgs b;
  const uint16_t *q;
  uint16_t *out;
  float *scratch;
  int64_t q_sh, q_sr, o_sh, o_sr;
  FastDiv drep;
  int32_t rep, window;
  int32_t items, few, groups;  // the most parts there are, the most query pairs they are for, in groups of 32
  int32_t least;               // a part's least blocks of keys, beside the plan's; over 1: a part a request
  // from here on, past the three cache lines that pages_few_kernel reads (a fourth: 16 requests of 5 rows 15.2 us, so 14.7):
  uint32_t joins;         // waves that join parts
  int32_t tiles, splits;  // tiles of 128 pairs, and the pieces that each one's keys are cut into
  float *split_scratch;
};

// Rows behind the last request's are zeros: block `at` clears 16 of them, every head.
template <int HD> __device__ __forceinline__ void clear_rows(const AttendArgs &a, int at, int tid, int threads) {
  const int last = gload(a.b.starts + a.b.requests), heads = a.c.kv * a.rep;
  for (int j = max(16 * at, last); j < min(16 * at + 16, a.b.rows); j++)
    for (int e = tid; e < heads * (HD / 8); e += threads) {
      const int h = e / (HD / 8);
      *(uint4 *)(a.out + h * a.o_sh + j * a.o_sr + e % (HD / 8) * 8) = make_uint4(0, 0, 0, 0);
    }
}

__device__ __forceinline__ uint32_t pack_rne(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, bf16x2));
}
__device__ __forceinline__ float max_groups(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_groups(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// l plus both bf16 values of w.
__device__ __forceinline__ float sum_pair(uint32_t w, float l) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3F803F80u), l, false);
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr float INF = __builtin_inff();

// 16 query pairs' running softmax: the reference maximum of the lane's pair in log2 units (p = 2^(s log2 e - m)), the sum
// of the lane's own p, and O^T. The reference moves only where a block's maximum passes it by 2^8 (O / l is the same for
// any reference, and p stays below 256), so most blocks rescale nothing.
template <int HD> struct Running {
  float m, l;
  f32x4 o[HD / 16];
  __device__ __forceinline__ void clear() {
    m = -INF, l = 0.0f;
#pragma unroll
    for (int c = 0; c < HD / 16; c++) o[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // The reference that a block's scores s (hidden keys at -inf) are weighed against, in log2 units, moved where they pass it.
  __device__ __forceinline__ float reference(const f32x4 (&s)[4]) {
    float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
    for (int kt = 1; kt < 4; kt++) top = fmaxf(top, fmaxf(fmaxf(s[kt][0], s[kt][1]), fmaxf(s[kt][2], s[kt][3])));
    top = max_groups(top) * LOG2E;
    if (__any(top > m + 8.0f)) {
      const float now = fmaxf(m, top), by = m == -INF ? 0.0f : __builtin_amdgcn_exp2f(m - now);
      m = now, l *= by;
#pragma unroll
      for (int c = 0; c < HD / 16; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[c][i] *= by;
    }
    return m == -INF ? 0.0f : m;  // no key of the pair seen yet: every weight is 2^-inf = 0
  }
  // p: the lane's 16 weights as bf16, the second operand of the two 32-key steps of O^T. They are rounded to nearest, since the
  // operand is bf16; l sums them as rounded, in 32 bits, so that a row's weights still add up to 1.
  __device__ __forceinline__ void weigh(const f32x4 (&s)[4], bf16x8 (&p)[2]) {
    const float ref = reference(s);
    u32x4 w[2];
#pragma unroll
    for (int kt = 0; kt < 4; kt++) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; i++) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], LOG2E, -ref));
      const uint32_t p0 = pack_rne(e[0], e[1]), p1 = pack_rne(e[2], e[3]);
      l = sum_pair(p1, sum_pair(p0, l));
      w[kt / 2][kt % 2 * 2] = p0, w[kt / 2][kt % 2 * 2 + 1] = p1;
    }
    p[0] = __builtin_bit_cast(bf16x8, w[0]), p[1] = __builtin_bit_cast(bf16x8, w[1]);
  }
};

// The lane's query pair, its row of q in the operand's order, and the keys it sees. RUN: the dims in a row that a lane of a
// key's row holds, of every 4 RUN.
template <int HD, int RUN = 16> struct Query {
  bf16x8 f[HD / 32];
  int lo, hi;
  __device__ __forceinline__ void load(const AttendArgs &a, const Piece &p, int kvh, int pair, int g) {
    const bool real = pair < p.n * a.rep;
    const int pp = real ? pair : 0, i = (int)fdiv((uint32_t)pp, a.drep), h = kvh * a.rep + pp - i * a.rep;
    const uint16_t *q = a.q + h * a.q_sh + (p.row0 + i) * a.q_sr + RUN * g;
#pragma unroll
    for (int k = 0; k < HD / 32; k++) f[k] = gload((const bf16x8 *)(q + 8 * k / RUN * (4 * RUN) + 8 * k % RUN));
    hi = real ? p.len - p.n + i : -1;  // the row's place
    lo = a.window > 0 ? max(hi - a.window + 1, 0) : 0;
  }
};

// Where pair `pair`'s output row starts.
__device__ __forceinline__ uint16_t *out_row(const AttendArgs &a, const Piece &p, int kvh, int pair) {
  const int i = (int)fdiv((uint32_t)pair, a.drep), h = kvh * a.rep + pair - i * a.rep;
  return a.out + h * a.o_sh + (p.row0 + i) * a.o_sr;
}

// The finished rows of a tile: O / l in bf16, 4 dims a store. A row that sees no key is zeros; a NaN stays one.
template <int HD> __device__ __forceinline__ void store_rows(const AttendArgs &a, const Piece &p, int kvh, int pair, int g,
                                                             const Running<HD> &st, float l) {
  const float inv = l > 0.0f ? 1.0f / l : l;
  uint16_t *out = out_row(a, p, kvh, pair) + 4 * g;
#pragma unroll
  for (int c = 0; c < HD / 16; c++)
    *(uint2 *)(out + 16 * c) = make_uint2(pack_rne(st.o[c][0] * inv, st.o[c][1] * inv),
                                          pack_rne(st.o[c][2] * inv, st.o[c][3] * inv));
}

template <int HD, int QT, int NW> struct FewLds {
  f32x4 o[NW / 2][QT * (HD / 16)][64];
  float m[NW / 2][QT][64], l[NW / 2][QT][64];
};
// A part as its block takes it: the request, its key head, the block's first pair, and the blocks of keys of the wave.
struct Part : Piece {
  int kvh, pair0, pairs, parts, unit, b0, b1;
  bool real;
};
// `block` of the launch's parts, or 16 of the rows to clear behind the last request's; `b0` is the wave's own.
template <int HD, int QT, int NW>
__device__ __forceinline__ void take_part(const AttendArgs &a, const int block, const int tid, Part *to) {
  const int lane = tid & 63, lg = a.c.page_log2, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int units = a.items * a.c.kv, group = block / units, unit = block - group * units;
  const int item = unit / a.c.kv, kvh = unit - item * a.c.kv, pair0 = 16 * QT * group;
  const int per = gload(a.b.parts + a.b.requests + 1);
  Piece p{0, 0, 0, 0, 0};
  const int32_t *at = a.b.parts;
  if (group >= a.groups) clear_rows<HD>(a, block - a.groups * units, tid, 64 * NW);
  else if (a.least > 1) p = whole_piece(a.b, item);
  else if (!find_piece(a.b, item, lane, [&](int i, int) { return gload(at + i); }, &p)) p.n = 0;
  if (p.n * a.rep > a.few) p.n = 0;
  const int pairs = p.n * a.rep;
  const int room = min(p.len, a.b.width << lg), nb = (room + KB - 1) / KB;
  const int mine = max(max(per, a.least), (nb + MOST_PARTS - 1) / MOST_PARTS), parts = (nb + mine - 1) / mine;
  const bool real = pair0 < pairs && p.k < parts;
  int b0 = p.k * mine;
  const int b1 = real ? min(b0 + mine, nb) : 0;
  if (a.window > 0) b0 = max(b0, max(p.len - p.n - a.window + 1, 0) / KB);
  *to = Part{p, kvh, pair0, pairs, parts, unit, b0 + wave, b1, real};
}

// The waves of a part join by halves through LDS, lane by lane; then its rows, or its sums for the join of parts.
template <int HD, int QT, int NW>
__device__ __forceinline__ void finish_part(const AttendArgs &a, const Part &p, const int tid, Running<HD> (&st)[QT],
                                            FewLds<HD, QT, NW> &lds) {
  constexpr int C = HD / 16;
  const int lane = tid & 63, n = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
  for (int half = NW / 2; half; half /= 2) {
    if (p.real && wave >= half && wave < 2 * half) {
#pragma unroll
      for (int t = 0; t < QT; t++) {
        lds.m[wave - half][t][lane] = st[t].m, lds.l[wave - half][t][lane] = st[t].l;
#pragma unroll
        for (int c = 0; c < C; c++) lds.o[wave - half][t * C + c][lane] = st[t].o[c];
      }
    }
    __syncthreads();
    if (p.real && wave < half) {
#pragma unroll
      for (int t = 0; t < QT; t++) {
        const float m = lds.m[wave][t][lane], top = fmaxf(st[t].m, m);
        const float mine = st[t].m == -INF ? 0.0f : __builtin_amdgcn_exp2f(st[t].m - top);
        const float other = m == -INF ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        st[t].m = top, st[t].l = st[t].l * mine + lds.l[wave][t][lane] * other;
#pragma unroll
        for (int c = 0; c < C; c++) {
          const f32x4 o = lds.o[wave][t * C + c][lane];
#pragma unroll
          for (int i = 0; i < 4; i++) st[t].o[c][i] = st[t].o[c][i] * mine + o[i] * other;
        }
      }
    }
    __syncthreads();
  }
  if (wave || !p.real) return;
#pragma unroll
  for (int t = 0; t < QT; t++) {
    const int pair = p.pair0 + 16 * t + n;
    const float l = sum_groups(st[t].l);
    if (pair >= p.pairs) continue;
    if (p.parts == 1) {
      store_rows<HD>(a, p, p.kvh, pair, g, st[t], l);
    } else {  // the part's sums for the join: the pair's O, then its maximum and sum
      float *to = a.scratch + (int64_t)p.unit * a.few * (HD + 4) + pair * (HD + 4);
#pragma unroll
      for (int c = 0; c < C; c++) *(f32x4 *)(to + 16 * c + 4 * g) = st[t].o[c];
      if (g == 0) to[HD] = st[t].m, to[HD + 1] = l;
    }
  }
}

// A pair's output from `parts` parts' sums, `step` floats apart, by a wave: M = max m, L = sum 2^(m - M) l, out = sum
// 2^(m - M) O / L. 16 parts' are requested at once, so that the usual plan is one trip to memory.
template <int HD> __device__ __forceinline__ void join_parts(const float *from, int64_t step, int parts, uint16_t *out, int lane) {
  constexpr int V = HD / 64, TURN = 16;
  float M = -INF, L = 0.0f, O[V];
#pragma unroll
  for (int i = 0; i < V; i++) O[i] = 0.0f;
  for (int b = 0; b < parts; b += TURN) {
    float m[TURN], l[TURN], o[TURN][V];
#pragma unroll
    for (int j = 0; j < TURN; j++) {
      m[j] = -INF, l[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) o[j][i] = 0.0f;
      if (b + j < parts) {  // (the whole wave's branch)
        const float *s = from + (b + j) * step;
        m[j] = gload(s + HD), l[j] = gload(s + HD + 1);
#pragma unroll
        for (int i = 0; i < V; i++) o[j][i] = gload(s + V * lane + i);
      }
    }
    float top = M;
#pragma unroll
    for (int j = 0; j < TURN; j++) top = fmaxf(top, m[j]);
    const float keep = M == -INF ? 0.0f : __builtin_amdgcn_exp2f(M - top);
    L *= keep;
#pragma unroll
    for (int i = 0; i < V; i++) O[i] *= keep;
#pragma unroll
    for (int j = 0; j < TURN; j++) {
      const float by = m[j] == -INF ? 0.0f : __builtin_amdgcn_exp2f(m[j] - top);  // 0: nothing seen (0 of a NaN stays one)
      L += by * l[j];
#pragma unroll
      for (int i = 0; i < V; i++) O[i] += by * o[j][i];
    }
    M = top;
  }
  const float inv = L > 0.0f ? 1.0f / L : L;
  if constexpr (V == 2) *(uint32_t *)(out + 2 * lane) = pack_rne(O[0] * inv, O[1] * inv);
  else out[lane] = (uint16_t)pack_rne(O[0] * inv, 0.0f);
}

constexpr int TILE_LOG2 = 7, TILE = 1 << TILE_LOG2;  // pairs of a block
// The tile that `slot` is: 128 pairs of request p->r from pair 128 p->k on. Request r owns tiles starts[r] * rep / 128 + r and on:
// at least as many as its pairs fill. False where there are none, or few enough for pages_few_kernel.
__device__ __forceinline__ bool find_tile(const AttendArgs &a, int slot, int lane, Piece *p) {
  return find_piece(a.b, slot, lane, [&](int i, int s) { return (int)((uint32_t)s * (uint32_t)a.rep >> TILE_LOG2) + i; }, p) &&
         p->n * a.rep > a.few && TILE * p->k < p->n * a.rep;
}

// The two halves of a tile's block, 4 waves of 32 pairs each, join a tile of pairs at a time: `joined` holds every wave of the
// second half's O^T, `sums` its maxima and sums, where nothing is read any more. Then the rows, or the split's sums for the join.
// HALVES: 1 where the block's 4 waves are all.
struct TileAt {
  int slot, kvh, split;
};
template <int HD, int HALVES = 2>
__device__ __forceinline__ void finish_tile(const AttendArgs &a, const Piece &p, const TileAt at, const int half, const int wave,
                                            const int lane, Running<HD> (&st)[2], f32x4 *joined, float *sums) {
  constexpr int C = HD / 16;
  const int n = lane & 15, g = lane >> 4, pairs = p.n * a.rep, pair0 = TILE * p.k, mine0 = pair0 + 32 * wave;
  if constexpr (HALVES == 2) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
      if (half) {
#pragma unroll
        for (int c = 0; c < C; c++) joined[(wave * C + c) * 64 + lane] = st[t].o[c];
        sums[(2 * wave) * 64 + lane] = st[t].m, sums[(2 * wave + 1) * 64 + lane] = st[t].l;
      }
      __syncthreads();
      if (!half) {
        const float m = sums[(2 * wave) * 64 + lane], top = fmaxf(st[t].m, m);
        const float mine = st[t].m == -INF ? 0.0f : __builtin_amdgcn_exp2f(st[t].m - top);
        const float other = m == -INF ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        st[t].m = top, st[t].l = st[t].l * mine + sums[(2 * wave + 1) * 64 + lane] * other;
#pragma unroll
        for (int c = 0; c < C; c++) {
          const f32x4 o = joined[(wave * C + c) * 64 + lane];
#pragma unroll
          for (int i = 0; i < 4; i++) st[t].o[c][i] = st[t].o[c][i] * mine + o[i] * other;
        }
      }
      __syncthreads();
    }
    if (half) return;
  }
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const int pair = mine0 + 16 * t + n;
    const float l = sum_groups(st[t].l);
    if (pair >= pairs) continue;
    if (a.splits == 1) {
      store_rows<HD>(a, p, at.kvh, pair, g, st[t], l);
    } else {
      float *to = a.split_scratch + ((((int64_t)at.slot * a.c.kv + at.kvh) * a.splits + at.split) * TILE + pair - pair0) * (HD + 4);
#pragma unroll
      for (int c = 0; c < C; c++) *(f32x4 *)(to + 16 * c + 4 * g) = st[t].o[c];
      if (g == 0) to[HD] = st[t].m, to[HD + 1] = l;
    }
  }
}

// ---- a call's checks and plan ----------------------------------------------------------------------------------------

// A pool of 8 bits a value has its scales beside its values; one of 4 bits among them, and `scales` is not looked at.
inline int check_pool(const bt_pages *c, int bits, PoolArgs *out) {
  const uint64_t scales = c && bits == 8 ? c->scales : 0;
  if (!c || !c->values || (bits == 8 && !scales))
    return fail(BT_EINVAL, "a paged cache needs its %s", bits == 8 ? "values and scales" : "values");
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(BT_EINVAL, "a paged cache's heads are 64 or 128 wide, not %d", c->head_dim);
  int lg = 0;
  while (lg < 9 && (1 << lg) != c->page) lg++;
  if (lg < 4 || lg > 8) return fail(BT_EINVAL, "a page holds 16, 32, 64, 128 or 256 tokens, not %d", c->page);
  if (c->kv < 1 || c->kv > 1024 || c->pages < 1 || (int64_t)c->pages * c->page > 0x7FFFFFFFll)
    return fail(BT_EINVAL, "a paged cache of %d pages of %d tokens and %d key heads", c->pages, c->page, c->kv);
  if (c->values % 16 || scales % 4) return fail(BT_EINVAL, "a paged cache's values are 16-byte aligned, its scales 4-byte");
  if (out) *out = PoolArgs{(uint8_t *)(uintptr_t)c->values, (float *)(uintptr_t)scales, c->pages, lg, c->kv};
  return BT_OK;
}

constexpr int MOST_ROWS = 1 << 20, MOST_KEYS = 1 << 30;  // rows of a batch, tokens of a request's table

// A launch of `blocks` of `threads` fits the 32 bits that a grid counts threads in.
inline bool grid_fits(int64_t blocks, int threads) { return blocks > 0 && blocks * threads <= 0xFFFFFFFFll; }

// The parts that a plan aims at, and a part's least blocks: all of a short table's keys (a part a request, and no join), else a
// block for each of its 4 waves. 1000 keys in one part and in parts with their join: one request of 3 heads of 64 6.2 us and 4.4
// + 3.1, 32 of 8 heads of 128 14.6 and 14.2 + 4.2, drafts' 5 rows of 16 14.2 and 12.6 + 4.5; 2000 keys: 9.8 us and 4.7 + 3.8,
// 8 requests of 8 heads of 128 15.4 and 9.9 + 4.0.
inline int parts_target(int kv) { return std::max(1, WAVES / (4 * kv)); }
inline int parts_least(int64_t keys) { return keys <= SHORT ? SHORT / KB : 4; }

inline int check_batch(const bt_batch *b, BatchArgs *out) {
  if (!b || !b->tables || !b->starts || !b->lengths || !b->parts)
    return fail(BT_EINVAL, "a batch needs its tables, starts, lengths and parts");
  if ((b->tables | b->starts | b->lengths | b->parts) % 4) return fail(BT_EINVAL, "a batch's tensors are int32-aligned");
  if (b->requests < 1 || b->requests > MOST_REQUESTS || b->rows < 1 || b->rows > MOST_ROWS || b->width < 1 ||
      b->width > MOST_KEYS / 16 || b->most < 1)
    return fail(BT_EINVAL, "a batch of %d requests (1 to %d), %d rows (1 to %d), tables %d wide, %d rows a request at most",
                b->requests, MOST_REQUESTS, b->rows, MOST_ROWS, b->width, b->most);
  if (out)
    *out = BatchArgs{(const int32_t *)(uintptr_t)b->tables,  (const int32_t *)(uintptr_t)b->starts,
                     (const int32_t *)(uintptr_t)b->lengths, (const int32_t *)(uintptr_t)b->parts,
                     b->tables_sr, b->requests, b->width, b->rows};
  return BT_OK;
}

// How a call is cut: `few`, the most pairs of a request whose keys are cut into parts, in tiles of 16 (`tiles` a wave); `many`,
// whether requests may have more, whose rows then share blocks of 128 pairs, and then parts are for up to 32 pairs. Where no
// request can have more than 64 all go to parts, 32 pairs at a time, which reads keys twice but spreads them further: 48 pairs of
// one request over 65536 keys 46.9 + 4.9 us in parts, 85.3 + 4.0 in tiles; 64 pairs of 16 over 2048 34.4 + 8.5 and 30.2 + 11.2.
struct AttendPlan {
  int few, tiles, groups, items;
  int waves;             // of a part's block
  int many_tiles, splits;  // tiles of 128 pairs, and the pieces that each one's keys are cut into
  bool many, join;
  int least;
  int64_t joins;  // waves that join parts
  uint64_t scratch, split_scratch;
};
inline int plan_attend(const bt_pages *c, int bits, const bt_batch *b, int heads, int window, AttendPlan *p) {
  if (int s = check_pool(c, bits, nullptr)) return s;
  if (int s = check_batch(b, nullptr)) return s;
  if (heads < 1 || heads % c->kv || window < 0 || (int64_t)heads * b->rows > 0x3FFFFFFF)
    return fail(BT_EINVAL, "paged attention of %d heads over %d key heads, %d rows, window %d", heads, c->kv, b->rows, window);
  if ((int64_t)b->width * c->page > MOST_KEYS)
    return fail(BT_EINVAL, "tables %d wide of pages of %d tokens hold over 2^30", b->width, c->page);
  const int rep = heads / c->kv;
  const int64_t most = (int64_t)std::min(b->most, b->rows) * rep;
  p->many = most > 64;
  p->few = p->many ? 32 : (int)most;
  p->tiles = p->few <= 16 ? 1 : 2;
  p->groups = (p->few + 31) / 32;
  // keys: what a request's rows see between them. Where a window leaves few of a long table's, one part has them: 32 requests
  // of 8192 keys in a window of 128 5.7 us and a launch less, in the plan's parts 6.7 + 3.5; of 1000 17.8, 18.8 + 4.0
  const int64_t held = (int64_t)b->width * c->page, keys = window ? std::min<int64_t>(held, (int64_t)window + b->most) : held;
  p->join = keys > SHORT, p->least = !p->join ? MOST_KEYS / KB : 1;
  p->items = p->join ? parts_target(c->kv) + b->requests : b->requests;  // (least > 1: the requests themselves)
  // a block of 8 waves where a part a request leaves most CUs idle: one request of 3 heads of 64 and 1000 keys 6.4 us, with 4 waves
  // 6.8; 512 of 8 heads and 500 keys 121.4 and 88.7
  p->waves = p->many || (p->tiles == 1 && !p->join && (int64_t)b->requests * c->kv < 64) ? 8 : 4;
  const uint64_t bytes = (uint64_t)p->items * c->kv * p->few * (c->head_dim + 4) * 4;
  p->scratch = p->join ? bytes : 0;
  // tiles that leave CUs idle (of 256, a block each at a time) have their keys cut, while a cut keeps 8 blocks of keys at least:
  // 100 rows of 32 heads over 8192 keys 235 us whole, 32.4 + 5.0 in 8 splits, 38.5 + 7.1 in 16; 512 rows 161 whole, 95 + 11.7 in
  // 2 and 119.5 + 12.0 in 3; 32 rows over 65536 86.1 + 4.0 in 16, 62.8 + 5.7 in 32, 72.6 + 7.6 in 48. A request's last tile
  // counts by half, but for the first's.
  p->many_tiles = (int)((int64_t)b->rows * rep >> TILE_LOG2) + b->requests, p->splits = 1, p->split_scratch = 0;
  if (p->many) {
    const int64_t blocks = (int64_t)p->many_tiles * c->kv;
    const int64_t full = (ceil_div((int64_t)b->rows * rep, TILE) + (b->requests - 1) / 2) * c->kv;
    p->splits = (int)std::max<int64_t>(1, std::min<int64_t>({256 / full, keys / (8 * KB), 64}));
    if (p->splits > 1) p->split_scratch = (uint64_t)blocks * p->splits * TILE * (c->head_dim + 4) * 4;
  }
  p->joins = p->join ? (int64_t)b->requests * c->kv * p->few : 0;
  const int64_t tiles = p->many ? (int64_t)p->many_tiles * c->kv : 0;
  if (!grid_fits((int64_t)p->items * c->kv * p->groups + (b->rows + 15) / 16 + tiles * p->splits, 64 * p->waves) ||
      !grid_fits(std::max<int64_t>(p->joins, 1) + tiles * TILE, 64))
    return fail(BT_EINVAL, "paged attention of %d rows and %d requests over %d heads is too large", b->rows, b->requests, heads);
  return BT_OK;
}

// A call's plan and its kernels' arguments, checked.
inline int attend_args(const bt_pages *pool, int bits, const bt_batch *batch, uint64_t q, int64_t q_sh, int64_t q_sr, uint64_t out,
                       int64_t o_sh, int64_t o_sr, int32_t heads, int32_t window, uint64_t scratch, uint64_t scratch_bytes,
                       AttendPlan *plan, AttendArgs *args) {
  AttendPlan &p = *plan;
  AttendArgs &a = *args;
  if (int s = plan_attend(pool, bits, batch, heads, window, &p)) return s;
  check_pool(pool, bits, &a.c), check_batch(batch, &a.b);
  if (!q || !out || q % 16 || q_sh % 8 || q_sr % 8 || out % 16 || o_sh % 8 || o_sr % 8)
    return fail(BT_EINVAL, "paged attention needs q and out rows on 16-byte boundaries");
  const uint64_t need = p.scratch + p.split_scratch;
  if (need && (!scratch || scratch % 16 || scratch_bytes < need))
    return fail(BT_EINVAL, "paged attention needs %llu bytes of 16-byte aligned scratch", (unsigned long long)need);
  a.q = (const uint16_t *)(uintptr_t)q, a.out = (uint16_t *)(uintptr_t)out, a.scratch = (float *)(uintptr_t)scratch;
  a.split_scratch = (float *)(uintptr_t)(scratch + p.scratch), a.splits = p.splits;
  a.q_sh = q_sh, a.q_sr = q_sr, a.o_sh = o_sh, a.o_sr = o_sr;
  a.rep = heads / a.c.kv, a.window = window, a.items = p.items, a.few = p.few, a.groups = p.groups, a.least = p.least;
  a.tiles = p.many_tiles, a.joins = (uint32_t)p.joins;
  a.drep = make_fastdiv((uint32_t)a.rep);
  return BT_OK;
}
// Queues the join of what attention cut, where it cut anything.
int launch_pages_join(const AttendArgs &a, const AttendPlan &p, int head_dim, hipStream_t s);

}  // namespace bt
