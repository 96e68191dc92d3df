// The paged KV cache in 4 bits a value: rows put into their pages, attention over the pages, and the pages read back. Plans,
// batches, parts, tiles and joins are the 8-bit cache's (pages.h, pages.hip).
//
// A value is a code of one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign (e2m1) times a scale. v_cvt_scalef32_pk_bf16_fp4 turns a
// byte into two bf16 values times a power of two, so a key's scale, a power of two for 32 of its dims, costs nothing there.
// A value row has one scale for all of its dims, which the weights of its key are multiplied by before they meet it: O = sum
// (p_t s_t) c_t. That scale has two bits behind its leading one, since it costs the same (rows of uneven channels: their
// rounding's error 0.126 of their size for 0.150 under powers of two; 0.126 and 0.127 are a key's under one scale of full
// precision and under a power of two for each 32 dims). Every scale belongs to one row, so a row's codes are final when it
// is put: no page is rounded again as it fills, and what it holds doesn't depend on how its rows came.
//
// A page is one run of bytes, for every key head (`kv` of them) a record of
//   keys' codes    [page][HD / 2]              a row's dims in order, the even one in a byte's low half;
//   keys' scales   [page / 16][HD / 32][4][4]  the exponent (biased by 127) of token 16 a + 4 j + i at [a][dims][i][j];
//   values' codes  [page / 16][HD / 32][16][2][8]  16 tokens of dim 32 c + 16 j + n at [a][c][n][j], the even one in the low half;
//   values' scales [page]                      bf16.
// so that attention's operands lie as its lanes take them (pages.hip has the two products): lane (n, g) of a wave holds for
// tile kt of a block of 64 keys the key 16 (n / 4) + 4 kt + n % 4, dims HD / 4 g and on, which are the codes of all four
// contraction steps, in one load (the contraction takes dims in any order that both operands share), with the four tiles'
// exponents in a word; and for dims 32 c .. + 31 the codes of its keys 16 g .. + 15 for dims 32 c + n and 32 c + 16 + n in
// another.
#include "pages.h"

namespace bt {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Where the parts of a key head's record of a page start.
template <int HD> struct Record {
  static constexpr int ROW = HD / 2;  // bytes of a row's codes
  static __host__ __device__ constexpr int key_scales(int lg) { return ROW << lg; }
  static __host__ __device__ constexpr int values(int lg) { return (ROW + HD / 32) << lg; }
  static __host__ __device__ constexpr int value_scales(int lg) { return (HD + HD / 32) << lg; }
  static __host__ __device__ constexpr int bytes(int lg) { return (HD + HD / 32 + 2) << lg; }
};
template <int HD> __device__ __forceinline__ uint8_t *record_of(const PoolArgs &c, int id, int kvh) {
  return c.values + ((int64_t)id * c.kv + kvh) * Record<HD>::bytes(c.page_log2);
}

template <int SEL> __device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float s) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, SEL));
}
__device__ __forceinline__ bf16x8 fp4_to_bf16(uint32_t w, float s) {
  return __builtin_bit_cast(bf16x8, u32x4{fp4_pair<0>(w, s), fp4_pair<1>(w, s), fp4_pair<2>(w, s), fp4_pair<3>(w, s)});
}
// 8 values of at most 6 in size after their rounding as codes, nearest, ties to even.
__device__ __forceinline__ uint32_t fp4_codes(const float (&x)[8], float s) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
}
__device__ __forceinline__ float two(int e) { return __uint_as_float((uint32_t)e << 23); }  // 2^(e - 127)

constexpr int LEAST_E = 27, MOST_E = 227;  // the scales' exponents, biased: 2^-100 to 2^100

// The smallest power of two s with amax <= 7 s, so that no value is off by more than half the largest step, 2 s: its exponent.
__device__ __forceinline__ int key_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);  // 7 = 1.75 * 2^2
  return min(max((int)(b >> 23) - ((b & 0x7FFFFFu) > 0x600000u ? 1 : 2), LEAST_E), MOST_E);
}
// The smallest s = k / 4 * 2^e, k = 4 .. 7, with amax <= 7 s.
__device__ __forceinline__ float value_scale(float amax) {
  const float half = two(key_exponent(amax) - 1);
  float s = 2.0f * half;
#pragma unroll
  for (int k = 7; k >= 4; k--) s = amax <= 7.0f * (half * (0.25f * k)) ? half * (0.25f * k) : s;
  return fmaxf(s, two(LEAST_E));
}

// ---- rows into pages ------------------------------------------------------------------------------------------------

// A wave: the rows that one request puts into 16 tokens of one head, a block's waves runs of 16 in a row. Rows are loaded
// once, all at once, and each one's scale is made by its own lanes. Values turn by dimension in the wave's own LDS; tokens
// of the 16 that take no row keep their codes. Memory bounds it where there are many rows: 131072 of 16 heads of 128 (677
// MB) 156 us, 4.3 TB/s (160 where a block's waves take four heads of one run); a decode step's 32 rows are latency, 3.9 us,
// and 1500 rows of 3 requests 6.8 (the 8-bit cache's 5.2 and 9.1). A row put alone reads and writes its 16 tokens' codes of
// a value head, 1 KB.
template <int HD, int W>
__global__ void __launch_bounds__(64 * W) put_pages4_kernel(const PoolArgs c, const BatchArgs b, const uint16_t *x, int64_t x_sb,
                                                             int64_t x_sr, int each) {
  constexpr int U = HD / 8, RP = 64 / U, TURNS = 16 / RP;  // 16-byte units of a row, rows of a turn
  // bytes of a dim in LDS, 16 tokens and 4 more, every 8th dim's in a row: what the lanes write at once falls in distinct banks
  constexpr int LINE = 20;
  __shared__ __attribute__((aligned(16))) uint8_t turned[W][HD * LINE];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lg = c.page_log2;
  const int heads = 2 * c.kv, h = blockIdx.x % heads, at = blockIdx.x / heads * W + w;
  Piece p;
  if (each) {  // pieces of every request
    if (at / each >= b.requests) return;
    p = whole_piece(b, at / each);
    p.k = at - p.r * each;
  } else if (!find_piece(b, at, lane, [&](int i, int s) { return (s >> 4) + 2 * i; }, &p)) {
    return;  // request r owns pieces starts[r] / 16 + 2 r and on: at least as many as the 16 tokens its rows touch
  }
  const int cached = p.len - p.n, run = (cached >> 4) + p.k, on = run >> (lg - 4);
  if (on >= b.width) return;  // (before anything is counted in tokens, whatever lengths say)
  const int token0 = run << 4, in = token0 & ((1 << lg) - 1);
  const int from = max(cached, token0), count = min(p.len, token0 + 16) - from, held = from - token0;
  if (count <= 0) return;
  const int id = gload(b.tables + p.r * b.tables_sr + on);  // the rows are requested before it is looked at
  const int unit = lane % U, row0 = lane / U;
  const uint16_t *src = x + h * x_sb + (int64_t)(p.row0 + from - cached) * x_sr + 8 * unit;
  u32x4 v[TURNS];
#pragma unroll
  for (int i = 0; i < TURNS; i++)  // (past the last row it is read again, so that no load waits behind a lane's branch)
    if (RP * i < count) v[i] = gload((const u32x4 *)(src + min(row0 + RP * i, count - 1) * x_sr));
  if ((uint32_t)id >= (uint32_t)c.pages) return;
  const bool value = h >= c.kv;
  uint8_t *rec = record_of<HD>(c, id, value ? h - c.kv : h);
#pragma unroll
  for (int i = 0; i < TURNS; i++) {
    if (RP * i >= count) break;
    const int row = row0 + RP * i, token = held + row;
    float f[8], top = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      f[k] = __uint_as_float(k & 1 ? v[i][k / 2] & 0xFFFF0000u : v[i][k / 2] << 16);
      top = fmaxf(top, (__float_as_uint(f[k]) & 0x7FFFFFFFu) < 0x7F800000u ? fabsf(f[k]) : 0.0f);
    }
    top = fmaxf(top, __shfl_xor(top, 1, 64)), top = fmaxf(top, __shfl_xor(top, 2, 64));  // 32 dims
    if (!value) {
      const int e = key_exponent(top);
      const float s = two(e), most = 7.0f * s;
#pragma unroll
      for (int k = 0; k < 8; k++) f[k] = __builtin_copysignf(fminf(fabsf(f[k]), most), f[k]);  // (NaN: the most)
      if (row < count) {
        *(uint32_t *)(rec + (in + token) * Record<HD>::ROW + 4 * unit) = fp4_codes(f, s);
        if (unit % 4 == 0) rec[Record<HD>::key_scales(lg) + in * (HD / 32) + 4 * unit + 4 * (token & 3) + (token >> 2)] = (uint8_t)e;
      }
    } else {
#pragma unroll
      for (int d = 4; d < U; d *= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
      const float s = value_scale(top), inv = 1.0f / s;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        // x / s to 16 bits of precision: a quotient on the border between two codes comes out exactly there, and any other is
        // 1 / 255 of it away at least (x has 8 bits, s times a border 6)
        const float q = __uint_as_float((__float_as_uint(fminf(fabsf(f[k] * inv), 7.0f)) + 0x80u) & ~0xFFu);
        f[k] = __builtin_copysignf(q, f[k]);
      }
      if (row < count) {
        const uint32_t codes = fp4_codes(f, 1.0f);
        uint8_t *to = turned[w] + unit * LINE + token;
#pragma unroll
        for (int k = 0; k < 8; k++) to[k * U * LINE] = (uint8_t)(codes >> 4 * k & 15);
        if (unit == 0) ((uint16_t *)(rec + Record<HD>::value_scales(lg)))[in + token] = (uint16_t)(__float_as_uint(s) >> 16);
      }
    }
  }
  if (!value) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  uint64_t *to = (uint64_t *)(rec + Record<HD>::values(lg) + in * Record<HD>::ROW);
  const uint64_t upto = held + count == 16 ? ~0ull : (1ull << 4 * (held + count)) - 1, fresh = upto & ~((1ull << 4 * held) - 1);
#pragma unroll
  for (int i = 0; i < HD / 64; i++) {
    const int e = (HD / 64) * lane + i, dim = e >> 5 << 5 | (e & 1) << 4 | (e >> 1 & 15);
    const uint32_t *line = (const uint32_t *)(turned[w] + (dim % 8 * U + dim / 8) * LINE);
    uint32_t half[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {  // a byte a token to half a byte
      const uint32_t lo = line[2 * k] & 0x0F0F0F0Fu, hi = line[2 * k + 1] & 0x0F0F0F0Fu;  // (anything where no row is)
      half[k] = __builtin_amdgcn_perm(hi | hi >> 4, lo | lo >> 4, 0x06040200);
    }
    const uint64_t now = (uint64_t)half[1] << 32 | half[0];
    to[e] = fresh == ~0ull ? now : (now & fresh) | (to[e] & ~fresh);
  }
}

// A block: 64 tokens of a page (or all of a shorter one), keys' or values', of one key head as bf16 rows, 16 tokens a wave.
// Values turn back through the wave's LDS. 12.6 million values (32 MB read and written) 6.5 us, 270 million (680 MB) 127 us,
// 5.4 TB/s.
template <int HD>
__global__ void __launch_bounds__(256) read_pages4_kernel(const PoolArgs c, uint16_t *out, int runs) {
  constexpr int U = HD / 8, RP = 64 / U, LINE = HD + 8;  // (rows of LDS 16 bytes apart from a power of two)
  __shared__ __attribute__((aligned(16))) uint16_t turned[4][16 * LINE];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lg = c.page_log2, heads = 2 * c.kv;
  const int64_t unit = blockIdx.x / runs;
  const int in = 64 * (int)(blockIdx.x - unit * runs) + 16 * w, h = (int)(unit % heads);
  if (in >> lg) return;
  const bool value = h >= c.kv;
  const uint8_t *rec = record_of<HD>(c, (int)(unit / heads), value ? h - c.kv : h);
  uint16_t *to = out + ((unit << lg) + in) * HD;
  if (!value) {
#pragma unroll
    for (int i = 0; i < 16 / RP; i++) {
      const int row = lane / U + RP * i, u = lane % U;
      const uint32_t codes = gload((const uint32_t *)(rec + (in + row) * Record<HD>::ROW + 4 * u));
      const float s = two(gload(rec + Record<HD>::key_scales(lg) + in * (HD / 32) + 4 * (u & ~3) + 4 * (row & 3) + (row >> 2)));
      *(uint4 *)(to + row * HD + 8 * u) = __builtin_bit_cast(uint4, fp4_to_bf16(codes, s));
    }
    return;
  }
  const u32x2 *codes = (const u32x2 *)(rec + Record<HD>::values(lg) + in * Record<HD>::ROW);
  const uint16_t *scales = (const uint16_t *)(rec + Record<HD>::value_scales(lg)) + in;
  float s[16];
#pragma unroll
  for (int t = 0; t < 16; t++) s[t] = __uint_as_float((uint32_t)gload(scales + t) << 16);
#pragma unroll
  for (int i = 0; i < HD / 64; i++) {
    const int e = 64 * i + lane, dim = e >> 5 << 5 | (e & 1) << 4 | (e >> 1 & 15);
    const u32x2 x = gload(codes + e);
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const u32x4 v = __builtin_bit_cast(u32x4, fp4_to_bf16(x[k], 1.0f));
#pragma unroll
      for (int t = 0; t < 8; t++) {  // times its row's scale: 5 bits, exact
        const float f = __uint_as_float(t & 1 ? v[t / 2] & 0xFFFF0000u : v[t / 2] << 16) * s[8 * k + t];
        turned[w][(8 * k + t) * LINE + dim] = (uint16_t)(__float_as_uint(f) >> 16);
      }
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < 16 / RP; i++) {
    const int row = lane / U + RP * i, u = lane % U;
    *(uint4 *)(to + row * HD + 8 * u) = *(const uint4 *)(turned[w] + row * LINE + 8 * u);
  }
}

// ---- attention over pages --------------------------------------------------------------------------------------------

// 64 of a request's pages from page `p0` on, one a lane (-1: none, whose keys are hidden).
__device__ __forceinline__ int page_ids(const AttendArgs &a, int r, int p0, int lane) {
  const int p = p0 + lane, id = p < a.b.width ? gload(a.b.tables + r * a.b.tables_sr + p) : -1;
  return (uint32_t)id < (uint32_t)a.c.pages ? id : -1;
}
// The page that key `key` lies in. ONE: blocks of 64 keys lie in one page (of 64 tokens or more), so `key` is the wave's.
template <bool ONE> __device__ __forceinline__ int page_of(int ids, int p0, int key, int lg) {
  if constexpr (ONE) return __builtin_amdgcn_readlane(ids, (key >> lg) - p0);
  else return __shfl(ids, (key >> lg) - p0, 64);
}

// What a lane holds of a block of 64 keys: its codes, its keys' exponents for the four tiles, its 16 values' scales.
template <int HD> struct Block4 {
  static constexpr int KW = HD / 32;  // words of a key's codes
  uint32_t k[4][KW];
  uint32_t ks;
  u32x4 v[HD / 32], vs[2];
  bool seen;  // whether the values' page is one
};
// The weights of a block's 16 pairs, times the values' scales, as bf16: rounded to nearest, since the second product's
// operand is bf16. l sums them in 32 bits before either, so that a row's weights add up to 1 but for that rounding.
template <int HD>
__device__ __forceinline__ void weigh4(Running<HD> &st, const f32x4 (&s)[4], const u32x4 (&vs)[2], bf16x8 (&p)[2]) {
  const float ref = st.reference(s);
  u32x4 w[2];
#pragma unroll
  for (int kt = 0; kt < 4; kt++)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const uint32_t both = vs[kt / 2][kt % 2 * 2 + i / 2];
      const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], LOG2E, -ref));
      const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i + 1], LOG2E, -ref));
      st.l += e0 + e1;
      w[kt / 2][kt % 2 * 2 + i / 2] = pack_rne(e0 * __uint_as_float(both << 16), e1 * __uint_as_float(both & 0xFFFF0000u));
    }
  p[0] = __builtin_bit_cast(bf16x8, w[0]), p[1] = __builtin_bit_cast(bf16x8, w[1]);
}

// One block of 64 keys against QT tiles of pairs, as fold_block in pages.hip. key: the lane's first key, seen: whether their
// page is one; values(c): the lane's codes of dims 32 c ..; between: run once the scores are made.
template <int HD, int QT, class Keys, class Values, class Between>
__device__ __forceinline__ void fold4(const Query<HD, HD / 4> (&q)[QT], Running<HD> (&st)[QT], int key, bool seen, uint32_t ks,
                                      const u32x4 (&vs)[2], Keys keys, Values values, Between between) {
  constexpr int KW = HD / 32;
  f32x4 s[QT][4];
#pragma unroll
  for (int kp = 0; kp < 4; kp += 2) {
    bf16x8 kf[2][KW];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const float scale = two(ks >> 8 * (kp + i) & 255);
#pragma unroll
      for (int j = 0; j < KW; j++) kf[i][j] = fp4_to_bf16(keys(kp + i, j), scale);
    }
#pragma unroll
    for (int k = 0; k < KW; k++)
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int t = 0; t < QT; t++) {
          if (k == 0) s[t][kp + i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          s[t][kp + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i][k], q[t].f[k], s[t][kp + i], 0, 0, 0);
        }
  }
  between();
  bf16x8 w[QT][2];
#pragma unroll
  for (int t = 0; t < QT; t++) {
    const int lo = q[t].lo - key, hi = seen ? q[t].hi - key : -1;
    if (!__all(lo <= 0 && hi >= 15)) {
#pragma unroll
      for (int kt = 0; kt < 4; kt++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (4 * kt + i < lo || 4 * kt + i > hi) s[t][kt][i] = -INF;
    }
    weigh4<HD>(st[t], s[t], vs, w[t]);
  }
#pragma unroll
  for (int c = 0; c < HD / 32; c++) {
    const u32x4 x = values(c);
    bf16x8 v[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++) v[i][0] = fp4_to_bf16(x[2 * i], 1.0f), v[i][1] = fp4_to_bf16(x[2 * i + 1], 1.0f);
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int t = 0; t < QT; t++)
          st[t].o[2 * c + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[i][h], w[t][h], st[t].o[2 * c + i], 0, 0, 0);
  }
}

// The blocks b, b + step .. below b1 of request r's keys, by a wave: a block's keys are requested while the block before
// weighs its scores, its values while it multiplies. ONCE: nobody else reads them, so past the caches.
template <int HD, int QT, bool ONE, bool ONCE>
__device__ __forceinline__ void walk4(const AttendArgs &a, int r, int kvh, int b, int b1, int step, const int lane,
                                      const Query<HD, HD / 4> (&q)[QT], Running<HD> (&st)[QT]) {
  using R = Record<HD>;
  if (b >= b1) return;
  const int n = lane & 15, g = lane >> 4, lg = a.c.page_log2, mask = (1 << lg) - 1;
  int p0 = b * KB >> lg;
  int ids = page_ids(a, r, p0, lane);
  Block4<HD> x;
  const auto load = [](auto *p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    else return gload(p);
  };
  const uint32_t krow = ((ONE ? 16 * (n >> 2) : 0) + (n & 3)) * R::ROW + R::ROW / 4 * g;
  const uint32_t kscale = (ONE ? (n >> 2) * (HD / 2) : 0) + (HD == 128 ? g : g >> 1) * 16 + (n & 3) * 4;
  const uint32_t vrow = (ONE ? g * 16 * R::ROW : 0) + 16 * n, vscale = ONE ? 32 * g : 0;
  const auto fetch_keys = [&](int b) {
    const int key = b * KB + (ONE ? 0 : 16 * (n >> 2)), in = key & mask;
    const uint8_t *rec = record_of<HD>(a.c, max(page_of<ONE>(ids, p0, key, lg), 0), kvh), *k = rec + in * R::ROW;
#pragma unroll
    for (int kt = 0; kt < 4; kt++) {
      if constexpr (HD == 128) {
        const u32x4 w = load((const u32x4 *)(k + (krow + 4 * kt * R::ROW)));
#pragma unroll
        for (int j = 0; j < HD / 32; j++) x.k[kt][j] = w[j];
      } else {
        const u32x2 w = load((const u32x2 *)(k + (krow + 4 * kt * R::ROW)));
#pragma unroll
        for (int j = 0; j < HD / 32; j++) x.k[kt][j] = w[j];
      }
    }
    x.ks = load((const uint32_t *)(rec + R::key_scales(lg) + in * (HD / 32) + kscale));
  };
  const auto fetch_values = [&](int b) {
    const int key = b * KB + (ONE ? 0 : 16 * g), in = key & mask, id = page_of<ONE>(ids, p0, key, lg);
    const uint8_t *rec = record_of<HD>(a.c, max(id, 0), kvh), *v = rec + R::values(lg) + in * R::ROW;
    const u32x4 *vs = (const u32x4 *)(rec + R::value_scales(lg) + 2 * in + vscale);
    x.seen = id >= 0;
#pragma unroll
    for (int i = 0; i < 2; i++) x.vs[i] = load(vs + i);
#pragma unroll
    for (int c = 0; c < HD / 32; c++) x.v[c] = load((const u32x4 *)(v + 256 * c + vrow));
  };
  fetch_keys(b), fetch_values(b);
  for (; b < b1; b += step) {
    const int next = b + step;
    const bool more = next < b1;
    fold4<HD, QT>(q, st, b * KB + 16 * g, x.seen, x.ks, x.vs, [&](int kt, int j) { return x.k[kt][j]; },
                  [&](int c) { return x.v[c]; }, [&] {
                    if (!more) return;
                    // the 64 pages that its keys lie in, if they are not there yet
                    if (((next * KB + KB - 1) >> lg) - p0 >= 64) p0 = next * KB >> lg, ids = page_ids(a, r, p0, lane);
                    fetch_keys(next);
                  });
    if (more) fetch_values(next);
  }
}

// Few query pairs a request, a part a block of NW waves, as few_pairs in pages.hip. Memory bounds it, less a launch's start
// and end: 32 requests of 4096 keys of 8 heads of 128 (140 MB) 26.4 us, 5.3 TB/s (8 bits, 269 MB: 44.8), 8 of up to 16383
// (105 MB) 22.3. Dropped: two blocks of keys ahead of the one at work (27 % more registers; the 26.4 us 28.2); scores from
// 8-bit products of q in two parts with keys' codes as they are, which saves the keys' conversion (prompts 118 us for 122,
// but the 26.4 us 27.6, drafts 14.0 and 16.2, a token 5.0 and 5.3: q's parts cost more than a few blocks' keys, and the
// product's own sums are less exact, 2^-17).
template <int HD, int QT, int NW, bool ONE>
__device__ __forceinline__ void few_pairs4(const AttendArgs &a, const int block, const int tid, FewLds<HD, QT, NW> &lds) {
  const int lane = tid & 63;
  Part p;
  take_part<HD, QT, NW>(a, block, tid, &p);
  Query<HD, HD / 4> q[QT];
  Running<HD> st[QT];
#pragma unroll
  for (int t = 0; t < QT; t++) {
    if (p.real) q[t].load(a, p, p.kvh, p.pair0 + 16 * t + (lane & 15), lane >> 4);
    st[t].clear();
  }
  walk4<HD, QT, ONE, true>(a, p.r, p.kvh, p.b0, p.b1, NW, lane, q, st);
  finish_part<HD, QT, NW>(a, p, tid, st, lds);
}

template <int HD, int QT, int NW, bool ONE>
__global__ void __launch_bounds__(64 * NW, 2) pages4_few_kernel(const AttendArgs a) {
  __shared__ FewLds<HD, QT, NW> lds;
  few_pairs4<HD, QT, NW, ONE>(a, blockIdx.x, threadIdx.x, lds);
}

// Many query pairs a request, 128 of one key head a block: 8 waves, two halves of 4 that take every other block of keys,
// each wave 32 pairs. Every wave loads its keys as the parts' do, four of them the same, from the caches: 4 bits are few
// enough for that (a block of 64 keys and heads of 128 is 8.4 KB), and the waves keep no step with each other: two prompts
// of up to 2048 rows behind cached ones 122 us, through LDS with a barrier a block, as the 8-bit cache's, 138 (that one's
// are 129); in blocks of one half 106. The vector instructions beside the matrix ones bound it, at work 0.70 of the
// time, matrix ones 0.35: a prompt of 4096 rows of 32 heads of 128 (137 GF) 154 us, 0.89 PFLOP/s; of 8192 563, 0.98. Heads of 64 have
// half the products for the same weights, vector instructions 0.73 and matrix ones 0.23: 4096 rows of 32 118 us, 0.58, of 8192 389,
// 0.71. Dropped: queries in LDS and values requested a step later,
// for three waves a SIMD (27 registers spilled; the 153 us 258).
template <int HD> struct Many4Lds {
  f32x4 joined[4 * (HD / 16) * 64];
  float sums[8 * 64];
};
template <int HD, int HALVES, bool ONE>
__device__ __forceinline__ void many_pairs4(const AttendArgs &a, const int block, Many4Lds<HD> &lds) {
  const int tid = threadIdx.x & 255, lane = tid & 63, n = lane & 15, g = lane >> 4, lg = a.c.page_log2;
  const int half = HALVES == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = block % a.c.kv, unit = block / a.c.kv, split = unit % a.splits;
  const int slot = a.tiles - 1 - unit / a.splits;  // the longest rows first
  Piece p;
  if (!find_tile(a, slot, lane, &p)) return;
  const int pairs = p.n * a.rep, pair0 = TILE * p.k, mine0 = pair0 + 32 * wave;
  Query<HD, HD / 4> q[2];
  Running<HD> st[2];
#pragma unroll
  for (int t = 0; t < 2; t++) q[t].load(a, p, kvh, mine0 + 16 * t + n, g), st[t].clear();
  const int cached = p.len - p.n, room = min(p.len, a.b.width << lg);
  const auto place = [&](int pair) { return cached + (int)fdiv((uint32_t)min(pair, pairs - 1), a.drep); };
  const auto low = [&](int at) { return a.window > 0 ? max(at - a.window + 1, 0) : 0; };
  int b0 = low(place(pair0)) / KB, b1 = min(place(pair0 + TILE - 1), room - 1) / KB + 1;
  if (a.splits > 1) {
    const int each = (b1 - b0 + a.splits - 1) / a.splits;
    b0 += split * each, b1 = min(b0 + each, b1);
  }
  // the wave's own keys among them
  b0 = max(b0, low(place(mine0)) / KB), b1 = mine0 < pairs ? min(b1, place(mine0 + 32 - 1) / KB + 1) : 0;
  walk4<HD, 2, ONE, false>(a, p.r, kvh, b0 + half, b1, HALVES, lane, q, st);
  finish_tile<HD, HALVES>(a, p, {slot, kvh, split}, half, wave, lane, st, lds.joined, lds.sums);
}

// A batch that may hold both, as pages_mixed_kernel in pages.hip.
template <int HD, int HALVES, bool ONE> __global__ void __launch_bounds__(256 * HALVES, 2) pages4_mixed_kernel(const AttendArgs a) {
  __shared__ union {
    Many4Lds<HD> many;
    FewLds<HD, 2, 4> few[HALVES];
  } lds;
  const int tiles = a.tiles * a.c.kv * a.splits;
  if ((int)blockIdx.x < tiles) return many_pairs4<HD, HALVES, ONE>(a, blockIdx.x, lds.many);
  const int half = HALVES == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  few_pairs4<HD, 2, 4, ONE>(a, HALVES * (blockIdx.x - tiles) + half, threadIdx.x & 255, lds.few[half]);
}

// ---- entry points ----------------------------------------------------------------------------------------------------

// Blocks of tiles past which each is 4 waves, so that two share a CU and one's start and end lie beside the other's work; up
// to it, 8. Prompts of 32 heads of 128, as 8 and as 4 waves: 4096 rows (1032 blocks) 183 and 153 us, 8 of 300 (664) 71 and
// 62, 16 of 128 (640) 28 and 22, 2048 (520) 59 and 62, 1024 (264) 27.6 and 29.5; 16 of 5 rows beside one of 256 (216) 50 and
// 58. Every request counts as a block, also one with few rows, whose tile is empty: where they are many their parts are most of
// the work, and those go faster beside each other in blocks of their own. A prompt of 256 rows beside 128 of a row and 500 keys
// (1128 blocks, 64 of them tiles) 34.9 and 28.2 us, of 100 beside 200 (1680, 32) 49.5 and 38.9, beside 200 of 3000 keys 166 and
// 138, of 2000 beside 200 (2152, 504) 112 and 86; 16 rows of two requests each over 16384 keys, cut in 32 (768, 512) 43 and 33.
constexpr unsigned HALVED = 600;
template <int HD, bool ONE> static int launch_attend4(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  const unsigned parts = p.items * a.c.kv * p.groups + (a.b.rows + 15) / 16, tiles = p.many_tiles * a.c.kv;
  const unsigned blocks = tiles * p.splits;
  // Blocks of 8 waves where parts are long, by what tables can hold: for heads of 64 from where a request's most parts have a block of
  // keys for each wave, for heads of 128, whose registers leave a CU one such block, where the parts there can be are no more than
  // the CUs, and the longer the more they are. Times by 4 and by 8 waves, caches from memory:
  //   128, parts at most: 32 (one key head): 32768 keys 14.5 and 14.9 us, 65536 19.4 and 17.9, 524288 87 and 66; 128: 32768 15.2 and
  //        15.5, 49152 18.1 and 18.3, 65536 20.5 and 18.5, 262144 50 and 40; 192: 49152 18.8 and 18.2, 65536 21.1 and 20.2, 98304
  //        25.8 and 23.1; 256 (8 key heads): 32768 16.4 and 17.8, 65536 21.9 and 22.5, 98304 27.5 and 27.4, 131072 33.5 and
  //        32.6, 524288 100 and 94; 512: 16384 17.6 and 21.0, 131072 52 and 57, 524288 176 and 178
  //   64: 8192 keys 15.7 and 16.0 (one request of 3 key heads), 27.4 and 27.8 (32), 15.7 and 16.0 (one of 8); 16384 17.9 and 17.6, 41.8
  //        and 41.7, 17.8 and 17.0; 131072 33.1 and 28.2 (one of 3)
  // A recorded step whose tables hold more than its caches do is cut by its tables: 16384 keys of 8 heads of 128 14.8 and 15.3.
  const int64_t held = (int64_t)a.b.width << a.c.page_log2, most = (int64_t)MOST_PARTS * a.b.requests * a.c.kv;
  const bool long_parts = p.join && (HD == 64 ? held >= 8 * KB * MOST_PARTS : most <= 256 && held >= std::max<int64_t>(65536, 512 * most));
  if (p.many && blocks > HALVED) pages4_mixed_kernel<HD, 1, ONE><<<blocks + parts, 256, 0, s>>>(a);
  else if (p.many) pages4_mixed_kernel<HD, 2, ONE><<<blocks + (parts + 1) / 2, 512, 0, s>>>(a);
  else if (p.tiles == 2) pages4_few_kernel<HD, 2, 4, ONE><<<parts, 256, 0, s>>>(a);
  else if (p.waves == 8 || long_parts) pages4_few_kernel<HD, 1, 8, ONE><<<parts, 512, 0, s>>>(a);
  else pages4_few_kernel<HD, 1, 4, ONE><<<parts, 256, 0, s>>>(a);
  BT_LAUNCHED("paged attention");
  return launch_pages_join(a, p, HD, s);
}

template <int HD> static int launch_put4(const PoolArgs &c, const BatchArgs &b, const uint16_t *x, int64_t x_sb, int64_t x_sr, int most,
                                         hipStream_t s) {
  const int heads = 2 * c.kv, each = most == 1 ? 1 : most <= 16 ? 2 : 0;
  // A wave a block while there are few, so that they spread over the CUs; past that four runs of a head, whose codes lie in a row. By
  // 1 and by 4, pieces of all heads: 192 3.4 and 3.6 us, 768 3.3 and 3.5 (128 requests of a row), 1520 7.0 and 7.3 (1500 rows), 2080 6.6 and
  // 7.1, 3088 7.5 and 7.4, 4128 9.0 and 8.5, 8192 9.1 and 7.6 (256 requests of 5 rows), 16384 12.3 and 11.6, 132096 151 and 154.
  const int64_t pieces = each ? (int64_t)each * b.requests : (b.rows >> 4) + 2 * b.requests;
  const int waves = pieces * heads <= 2048 ? 1 : 4;
  const int64_t blocks = (pieces + waves - 1) / waves;
  if (!grid_fits(blocks * heads, 64 * waves)) return fail(BT_EINVAL, "a put of %d rows of %d heads is too large", b.rows, heads);
  if (waves == 1) put_pages4_kernel<HD, 1><<<(unsigned)(blocks * heads), 64, 0, s>>>(c, b, x, x_sb, x_sr, each);
  else put_pages4_kernel<HD, 4><<<(unsigned)(blocks * heads), 256, 0, s>>>(c, b, x, x_sb, x_sr, each);
  BT_LAUNCHED("a paged put");
  return BT_OK;
}

}  // namespace bt

using namespace bt;

extern "C" {

int bt_pages4_bytes(const bt_pages *pool, uint64_t *bytes) {
  if (!bytes) return fail(BT_EINVAL, "no result pointer");
  bt_pages c = pool ? *pool : bt_pages{};
  c.values = 16;  // the shape alone counts
  PoolArgs a;
  if (int s = check_pool(&c, 4, &a)) return s;
  *bytes = (uint64_t)c.pages * c.kv * (c.head_dim == 64 ? Record<64>::bytes(a.page_log2) : Record<128>::bytes(a.page_log2));
  return BT_OK;
}

int bt_pages4_put(bt_runtime *rt, const bt_pages *pool, const bt_batch *batch, uint64_t x, int64_t x_sb, int64_t x_sr) {
  Runtime *r;
  if (int s = enter(rt, &r)) return s;
  PoolArgs c;
  BatchArgs b;
  if (int s = check_pool(pool, 4, &c)) return s;
  if (int s = check_batch(batch, &b)) return s;
  if (!x || x % 16 || x_sb % 8 || x_sr % 8) return fail(BT_EINVAL, "a paged cache takes rows on 16-byte boundaries");
  if ((int64_t)b.width * pool->page > MOST_KEYS)
    return fail(BT_EINVAL, "tables %d wide of pages of %d tokens hold over 2^30", b.width, pool->page);
  const uint16_t *src = (const uint16_t *)(uintptr_t)x;
  const int most = std::min(batch->most, batch->rows);
  if (pool->head_dim == 64) return launch_put4<64>(c, b, src, x_sb, x_sr, most, r->stream);
  return launch_put4<128>(c, b, src, x_sb, x_sr, most, r->stream);
}

int bt_pages4_read(bt_runtime *rt, const bt_pages *pool, uint64_t out) {
  Runtime *r;
  if (int s = enter(rt, &r)) return s;
  PoolArgs c;
  if (int s = check_pool(pool, 4, &c)) return s;
  if (!out || out % 16) return fail(BT_EINVAL, "pages are read to a 16-byte aligned tensor");
  const int runs = (pool->page + 63) / 64;
  const int64_t blocks = (int64_t)c.pages * 2 * c.kv * runs;
  if (!grid_fits(blocks, 256)) return fail(BT_EINVAL, "%d pages of %d heads are too many to read at once", c.pages, 2 * c.kv);
  uint16_t *to = (uint16_t *)(uintptr_t)out;
  if (pool->head_dim == 64) read_pages4_kernel<64><<<(unsigned)blocks, 256, 0, r->stream>>>(c, to, runs);
  else read_pages4_kernel<128><<<(unsigned)blocks, 256, 0, r->stream>>>(c, to, runs);
  BT_LAUNCHED("reading pages");
  return BT_OK;
}

int bt_pages4_attend_scratch(const bt_pages *pool, const bt_batch *batch, int32_t heads, int32_t window, uint64_t *bytes) {
  if (!bytes) return fail(BT_EINVAL, "no result pointer");
  AttendPlan p;
  if (int s = plan_attend(pool, 4, batch, heads, window, &p)) return s;
  *bytes = p.scratch + p.split_scratch;
  return BT_OK;
}

int bt_pages4_attend(bt_runtime *rt, const bt_pages *pool, const bt_batch *batch, uint64_t q, int64_t q_sh, int64_t q_sr,
                     uint64_t out, int64_t o_sh, int64_t o_sr, int32_t heads, int32_t window, uint64_t scratch,
                     uint64_t scratch_bytes) {
  Runtime *r;
  if (int s = enter(rt, &r)) return s;
  AttendPlan p;
  AttendArgs a;
  if (int s = attend_args(pool, 4, batch, q, q_sh, q_sr, out, o_sh, o_sr, heads, window, scratch, scratch_bytes, &p, &a)) return s;
  const bool one = pool->page >= KB;
  if (pool->head_dim == 64) return one ? launch_attend4<64, true>(a, p, r->stream) : launch_attend4<64, false>(a, p, r->stream);
  return one ? launch_attend4<128, true>(a, p, r->stream) : launch_attend4<128, false>(a, p, r->stream);
}

}  // extern "C"
