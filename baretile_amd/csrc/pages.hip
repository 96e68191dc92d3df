// A paged 8-bit KV cache: the step's plan (block tables, row starts, places, slots) from request lengths, keys and values
// put into their pages, attention over the pages, and the pages read back.
//
// A page holds `page` tokens of every key and value head under one id. A head's values are e4m3 codes (4 exponent and 3
// mantissa bits, at most 448) times one power of two for the page and head, so each is exact in bf16 and the conversion
// v_cvt_scalef32_pk_bf16_fp8 applies the scale: half an instruction a value, where a block float's decoding takes 2.5.
// Keys are kept by row, 64 dims at a time, [head width / 64][page][64], and values by dimension, up to 64 tokens at a time,
// [page / 64][head width][64], so that both products of attention read their operands from memory as they lie, 16 bytes a
// lane, with no transposition and no trip through LDS, and each load of a wave covers whole lines (keys by rows of 128 dims,
// of which a load takes half a line each: 8 requests of up to 8191 keys 20.8 us, by halves 19.5; 32 of 4096 47.5 and 45.4):
//   S^T = K Q^T: lane (n, g) (n = l % 16, g = l / 16) holds for tile kt (of 4 in a block of 64 keys) the key
//     16 (n / 4) + 4 kt + n % 4, dims 64 j + 16 g .. + 15 (the contraction takes dims in any order that both operands share);
//   so in the result lane (n, g) holds keys 16 g + 4 kt + i, i < 4, against pair n: 16 keys in a row over the 4 tiles;
//   O^T = V^T P^T: the second operand is the lane's own P, the first 16 bytes of dim 16 c + n: keys 16 g .. + 15.
// O^T's column is the lane's pair as well, so the running maximum rescales it with no move between lanes.
#include "pages.h"
#include <type_traits>

namespace bt {

// ---- the plan ------------------------------------------------------------------------------------------------------

struct PlanArgs {
  int32_t *tables;
  const int32_t *cached, *fresh, *free_pages, *taken;
  int32_t *starts, *lengths, *places, *slots, *taken_out, *parts;
  int64_t tables_sr;
  int32_t requests, width, n_free, rows, page_log2, pages, most, target, least;
};

__device__ __forceinline__ int pages_of(int n, int lg) { return (n + (1 << lg) - 1) >> lg; }

// The sum of x over the lower threads of the block, and the block's total. `sums`: a word of LDS a wave.
template <int NT> __device__ __forceinline__ int block_exclusive(int x, int *sums, int *total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int inc = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int up = __shfl_up(inc, d, 64);
    if (lane >= d) inc += up;
  }
  __syncthreads();
  if (lane == 63) sums[w] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; i++) {
    const int s = sums[i];
    before += i < w ? s : 0, all += s;
  }
  *total = all;
  return before + inc - x;
}

// The request that owns row j: the last one that starts at or before it.
__device__ __forceinline__ int owner_of(const int *starts, int requests, int j) {
  int lo = 0, hi = requests;  // starts[lo] <= j < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= j) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The place and slot of row j (-1 past the last request's).
__device__ __forceinline__ void plan_row(const PlanArgs &a, int j, int start, int cached, int id_or_free, bool real) {
  const int place = cached + j - start, mask = (1 << a.page_log2) - 1;
  a.places[j] = real ? place : -1;
  a.slots[j] = real && id_or_free >= 0 ? (id_or_free << a.page_log2) + (place & mask) : -1;
}

// One block, of 64, 256 or 1024 threads by the larger of its requests and the rows it writes. Requests are scanned a thread
// each: first their rows, cut to `most` each and to the rows there are, and the pages they take; then, with the keys' blocks
// counted, the parts that attention cuts each request's keys into: as many parts over all requests as `target`, of whole blocks
// of 64 keys and `least` of them, so that uneven lengths make parts of even length.
// Latency bounds it: three scans of about a microsecond and two trips to memory. 32 requests of a row: 4.1 us (5.7 by 1024
// threads, whose scans pass 16 sums through LDS); 512 with 8500 rows: 6.2 and 4.1 us for the rows.
// LARGE: requests' blocks of keys may pass 2^30 in all (2048 of 2^24 would pass 32 bits), and are summed by their lower 12 bits
// and the rest. A kernel of its own: decided on the device, every plan took 0.1 us more (32 requests 4.2 us for 4.1).
// The block writes up to PLAN_ROWS rows itself, past that many blocks of plan_rows_kernel do: 2048 rows 6.8 us here, 3.5 + 3.2 us
// and a launch more there; 8192 12.4 us and 4.5 + 4.0.
constexpr int PLAN_ROWS = 2048;
template <int NT, bool LARGE> __global__ void __launch_bounds__(NT) plan_kernel(const PlanArgs a) {
  __shared__ int starts[MOST_REQUESTS + 1], first[MOST_REQUESTS], from[MOST_REQUESTS + 1], cache[MOST_REQUESTS];
  __shared__ int sums[NT / 64];
  const int lg = a.page_log2, room = (int)min((int64_t)a.width << lg, (int64_t)0x40000000);
  const int taken = a.taken ? gload(a.taken) : 0;
  int rows = 0, takes = 0;
  std::conditional_t<LARGE, int64_t, int> blocks = 0;
  for (int base = 0; base < a.requests; base += NT) {
    const int r = base + threadIdx.x;
    int c = 0, n = 0, total;
    if (r < a.requests) c = min(max(gload(a.cached + r), 0), room), n = min(max(gload(a.fresh + r), 0), a.most);
    // 2^20 rows at most, and so many a request: a sum over 1024 requests keeps to 31 bits
    const int s = rows + block_exclusive<NT>(n, sums, &total);
    const int s0 = min(s, a.rows), s1 = min(s + n, a.rows);
    rows = min(rows + total, a.rows);
    n = s1 - s0;
    int k = 0, need = 0;
    if (r < a.requests) {
      const int end = min(pages_of(c + n, lg), a.width);
      k = pages_of(c, lg);
      const int32_t *row = a.tables + r * a.tables_sr;
      while (k < end && (uint32_t)row[k] < (uint32_t)a.pages) k++;
      need = max(end - k, 0);
      starts[r] = s0, first[r] = k, cache[r] = c;
      a.starts[r] = s0, a.lengths[r] = c + n;
    }
    const int off = block_exclusive<NT>(need, sums, &total);
    if (r < a.requests) from[r] = takes + off;
    takes += total;
    const int nb = n > 0 ? (min(c + n, room) + KB - 1) / KB : 0;
    block_exclusive<NT>(LARGE ? nb & 4095 : nb, sums, &total);
    blocks += total;
    if constexpr (LARGE) block_exclusive<NT>(nb >> 12, sums, &total), blocks += (int64_t)total << 12;
  }
  const int last = rows;
  if (threadIdx.x == 0) {
    starts[a.requests] = last, from[a.requests] = takes;
    a.starts[a.requests] = last;
    a.taken_out[0] = taken + takes;
  }
  auto each = (blocks + a.target - 1) / a.target;
  if constexpr (LARGE) each = min(each, (int64_t)(0x40000000 / KB));  // a part holds one request's blocks, 2^24 at most
  const int per = max(a.least, ((int)each + 3) & ~3);
  int made = 0;
  __syncthreads();
  for (int base = 0; base < a.requests; base += NT) {
    const int r = base + threadIdx.x;
    int parts = 0, total;
    if (r < a.requests) {
      const int n = starts[r + 1] - starts[r], nb = n > 0 ? (min(cache[r] + n, room) + KB - 1) / KB : 0;
      const int mine = max(per, (nb + MOST_PARTS - 1) / MOST_PARTS);
      parts = (nb + mine - 1) / mine;
    }
    const int off = block_exclusive<NT>(parts, sums, &total);
    if (r < a.requests) a.parts[r] = made + off;
    made += total;
  }
  if (threadIdx.x == 0) a.parts[a.requests] = made, a.parts[a.requests + 1] = per;
  auto page_at = [&](int e) {  // the free list's page e, or -1
    if ((uint32_t)e >= (uint32_t)a.n_free) return -1;
    const int id = gload(a.free_pages + e);
    return (uint32_t)id < (uint32_t)a.pages ? id : -1;
  };
  for (int e = threadIdx.x; e < takes; e += NT) {
    const int r = owner_of(from, a.requests, e);
    a.tables[r * a.tables_sr + first[r] + e - from[r]] = page_at(taken + e);
  }
  if (a.rows > PLAN_ROWS) return;
  for (int j = threadIdx.x; j < a.rows; j += NT) {
    const bool real = j < last;
    const int r = real ? owner_of(starts, a.requests, j) : 0;
    const int on = (cache[r] + j - starts[r]) >> lg;
    int id = -1;
    if (real && on < a.width) {
      if (on >= first[r]) id = page_at(taken + from[r] + on - first[r]);
      else id = gload(a.tables + r * a.tables_sr + on);
      if ((uint32_t)id >= (uint32_t)a.pages) id = -1;
    }
    plan_row(a, j, starts[r], cache[r], id, real);
  }
}

// The rows' places and slots from the finished tables.
__global__ void __launch_bounds__(256) plan_rows_kernel(const PlanArgs a) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= a.rows) return;
  const bool real = j < gload(a.starts + a.requests);
  const int r = real ? owner_of(a.starts, a.requests, j) : 0;
  const int start = a.starts[r], cached = a.lengths[r] - (a.starts[r + 1] - start);
  const int on = (cached + j - start) >> a.page_log2;
  int id = real && on < a.width ? gload(a.tables + r * a.tables_sr + on) : -1;
  if ((uint32_t)id >= (uint32_t)a.pages) id = -1;
  plan_row(a, j, start, cached, id, real);
}

// ---- rows into pages ------------------------------------------------------------------------------------------------

// Where a value head's code of dimension `dim` and row `row` of a page lies.
template <int HD> __device__ __forceinline__ int value_at(int dim, int row, int lg) {
  const int run = min(lg, 6);
  return (row >> run) * (HD << run) + (dim << run) + (row & ((1 << run) - 1));
}
// Two codes of x0, x1 in the low half: nearest even, at most 448 in size (a NaN, which no code stands for in a cache, 448).
__device__ __forceinline__ uint32_t codes_of(float x0, float x1) {
  x0 = __builtin_copysignf(fminf(fabsf(x0), 448.0f), x0), x1 = __builtin_copysignf(fminf(fabsf(x1), 448.0f), x1);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false) & 0xFFFFu;
}
__device__ __forceinline__ uint32_t codes_of4(float x0, float x1, float x2, float x3) {
  return codes_of(x0, x1) | codes_of(x2, x3) << 16;
}
// Four codes under another scale: times `by`, a power of two of at most 1.
__device__ __forceinline__ uint32_t rescaled4(uint32_t w, float by) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  return codes_of4(lo[0] * by, lo[1] * by, hi[0] * by, hi[1] * by);
}

// The smallest power of two s with amax <= 448 s = 1.75 * 2^8 s, from 2^-100 to 2^119 (so that every value is a normal
// bf16). amax is finite.
__device__ __forceinline__ float scale_of(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - ((b & 0x7FFFFFu) > 0x600000u ? 7 : 8);  // biased by 127
  return __uint_as_float((uint32_t)min(max(e, 27), 246) << 23);
}

// A block: the rows that one request puts into one page of one head, PAGE of them at most. They are loaded once (up to 16 loads of
// 16 bytes a thread, all at once and before the page's id is there), their largest finite size gives the scale, and a page that
// already holds rows and whose scale grows has them rounded again. Values turn by dimension in LDS, so they are stored as
// whole words.
// Memory bounds it where there are many rows: 131072 of 16 heads of 128 (800 MB) 181 us, 4.4 TB/s; a decode step's 32 rows are
// latency, 5.3 us, and so are a few prompts' chunks: 3 requests' 1500 rows of 16 heads of 128 9.1 us for 9.2 MB, in 832 blocks,
// three or four a CU, whose waves wait 64% of their cycles (for a chain of trips to memory and two barriers; vector instructions
// are 16%, and of the LDS's 0.32 million cycles 0.19 are bank conflicts).
// Rows by the most that a request can put into one page, so that registers, LDS and threads fit them: up to 16 by one wave (512
// requests of one row 25.8 us, by four waves 48.4, of 8 rows 31.0 and 49.8, all with a search for the request), up to 64 with
// loads for 64 (32 requests of 48 rows 10.2 us, with loads for 256 11.1).
template <int HD, int NT, int PAGE>
__global__ void __launch_bounds__(NT) put_pages_kernel(const PoolArgs c, const BatchArgs b, const uint16_t *x, int64_t x_sb,
                                                        int64_t x_sr, int each) {
  constexpr int U = HD / 8, MOST = PAGE * U / NT;  // 16-byte units of a row, loads a thread for the most rows
  __shared__ float tops[NT / 64];
  __shared__ __attribute__((aligned(16))) uint8_t turned[HD * (PAGE + 4)];  // by dimension, from the new rows' first word on
  const int tid = threadIdx.x, lane = tid & 63, lg = c.page_log2, page = 1 << lg, heads = 2 * c.kv;
  const int at = blockIdx.x / heads, h = blockIdx.x - at * heads;
  Piece p;
  if (each) {  // pieces of every request
    p = whole_piece(b, at / each);
    p.k = at - p.r * each;
  } else if (!find_piece(b, at, lane, [&](int i, int s) { return (s >> lg) + 2 * i; }, &p)) {
    return;  // request r owns pieces starts[r] / page + 2 r and on: at least as many as the pages its rows touch
  }
  const int cached = p.len - p.n, on = (cached >> lg) + p.k;
  const int from = max(cached, on << lg), count = min(min(p.len, (on + 1) << lg) - from, PAGE);
  if (count <= 0 || on >= b.width) return;
  const int id = gload(b.tables + p.r * b.tables_sr + on);  // the rows are requested before it is looked at
  const int held = from & (page - 1), units = count * U;
  const uint16_t *src = x + h * x_sb + (int64_t)(p.row0 + from - cached) * x_sr;
  u32x4 v[MOST];
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < MOST; i++) {
    const int e = tid + NT * i;
    // (past the last row it is read again, so that no load waits behind a lane's branch)
    if (NT * i < units) v[i] = gload((const u32x4 *)(src + min(e / U, count - 1) * x_sr + e % U * 8));
  }
  if ((uint32_t)id >= (uint32_t)c.pages) return;
  float *scale_at = c.scales + (int64_t)id * heads + h;
  const float old = held ? gload(scale_at) : 0.0f;
#pragma unroll
  for (int i = 0; i < MOST; i++)
    if (NT * i < units)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const uint32_t lo = v[i][k] << 16 & 0x7FFFFFFFu, hi = v[i][k] & 0x7FFF0000u;
        top = fmaxf(top, lo < 0x7F800000u ? __uint_as_float(lo) : 0.0f);
        top = fmaxf(top, hi < 0x7F800000u ? __uint_as_float(hi) : 0.0f);
      }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
  if (lane == 0) tops[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; i++) top = fmaxf(top, tops[i]);
  const float s = fmaxf(scale_of(top), old), inv = __uint_as_float((254u << 23) - __float_as_uint(s));  // 1 / s, exact
  const float by = old * inv;
  uint8_t *to = c.values + (((int64_t)id * heads + h) << lg) * HD;
  if (h < c.kv) {  // keys: 64 dims of a row are 4 units of 16
    if (held && by != 1.0f)
      for (int e = tid; e < held * HD / 16; e += NT) {
        u32x4 *at = (u32x4 *)(to + (e / 4 / held << (lg + 6)) + e / 4 % held * 64 + e % 4 * 16), w = *at;
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = rescaled4(w[k], by);
        *at = w;
      }
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int e = tid + NT * i;
      if (NT * i < units && e < units) {
        uint2 w;
        const auto val = [&](int k) { return __uint_as_float(k & 1 ? v[i][k / 2] & 0xFFFF0000u : v[i][k / 2] << 16) * inv; };
        w.x = codes_of4(val(0), val(1), val(2), val(3)), w.y = codes_of4(val(4), val(5), val(6), val(7));
        *(uint2 *)(to + (e % U / 8 << (lg + 6)) + (held + e / U) * 64 + e % 8 * 8) = w;
      }
    }
  } else {  // values: each dimension's codes lie along the page
    constexpr int line = PAGE + 4;
    const int base = held & ~3;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
      const int e = tid + NT * i;
      if (NT * i < units && e < units) {
        const int row = held - base + e / U, dim = e % U * 8;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t w = codes_of(__uint_as_float(v[i][k] << 16) * inv, __uint_as_float(v[i][k] & 0xFFFF0000u) * inv);
          turned[(dim + 2 * k) * line + row] = (uint8_t)w, turned[(dim + 2 * k + 1) * line + row] = (uint8_t)(w >> 8);
        }
      }
    }
    __syncthreads();
    // whole words of 4 rows: from the page's start where its rows are rounded again, else from the word with the first new row
    const int w0 = held && by != 1.0f ? 0 : held / 4, w1 = (held + count + 3) / 4, words = w1 - w0;
    for (int e = tid; e < words * HD; e += NT) {
      const int dim = e / words, w = w0 + e - dim * words;
      uint32_t *word = (uint32_t *)(to + value_at<HD>(dim, 4 * w, lg));
      const uint32_t now = 4 * w >= base ? *(const uint32_t *)(turned + dim * line + 4 * w - base) : 0;
      const int kept = min(max(held - 4 * w, 0), 4), end = min(held + count - 4 * w, 4);
      if (kept == 0 && end == 4) {
        *word = now;
      } else {  // rows kept before the new ones, and what lies behind them
        const uint32_t was = *word, before = by != 1.0f && kept ? rescaled4(was, by) : was;
        const auto low = [](int n) { return n >= 4 ? 0xFFFFFFFFu : (1u << 8 * n) - 1; };
        const uint32_t fresh = low(end) & ~low(kept);
        *word = (now & fresh) | (before & low(kept)) | (was & ~low(end));
      }
    }
  }
  if (tid == 0) *scale_at = s;
}

// A block: one page of one head as bf16 rows. Values turn back through LDS, 4 x 4 codes a thread by byte permutes. PAGE: the
// longest page that LDS holds. 12.6 million values of pages of 64 (38 MB read and written): 7.7 us, 4.9 TB/s, and 9.9 with LDS for
// 256 (4 blocks a CU).
template <int HD, int PAGE>
__global__ void __launch_bounds__(256) read_pages_kernel(const PoolArgs c, uint16_t *out) {
  __shared__ __attribute__((aligned(16))) uint8_t turned[HD * (PAGE + 4)];
  const int tid = threadIdx.x, lg = c.page_log2, page = 1 << lg, heads = 2 * c.kv;
  const int64_t unit = blockIdx.x;
  const int h = (int)(unit % heads);
  const uint8_t *from = c.values + (unit << lg) * HD;
  uint16_t *to = out + (unit << lg) * HD;
  const float s = gload(c.scales + unit);
  const auto pair = [&](uint32_t w, bool up) {
    return up ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false));
  };
  if (h < c.kv) {
    for (int e = tid; e < page * HD / 8; e += 256) {  // e: 8 codes as they lie
      const uint2 w = gload((const uint2 *)(from + 8 * e));
      const int row = e / 8 & (page - 1), dim = (e >> (lg + 3)) * 64 + e % 8 * 8;
      *(uint4 *)(to + row * HD + dim) = make_uint4(pair(w.x, false), pair(w.x, true), pair(w.y, false), pair(w.y, true));
    }
    return;
  }
  const int line = page + 4, wl = lg - 2;
  for (int e = tid; e < HD << wl; e += 256) {
    const int dim = e >> wl, w = e & ((1 << wl) - 1);
    *(uint32_t *)(turned + dim * line + 4 * w) = gload((const uint32_t *)(from + value_at<HD>(dim, 4 * w, lg)));
  }
  __syncthreads();
  for (int e = tid; e < page * HD / 16; e += 256) {  // 4 dims of 4 rows, turned by byte permutes
    const int dim = e % (HD / 4) * 4, row = e / (HD / 4) * 4;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; k++) w[k] = *(const uint32_t *)(turned + (dim + k) * line + row);
    const uint32_t a01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400), b01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602);
    const uint32_t a23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400), b23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
    const uint32_t r[4] = {__builtin_amdgcn_perm(a23, a01, 0x05040100), __builtin_amdgcn_perm(a23, a01, 0x07060302),
                           __builtin_amdgcn_perm(b23, b01, 0x05040100), __builtin_amdgcn_perm(b23, b01, 0x07060302)};
#pragma unroll
    for (int k = 0; k < 4; k++) *(uint2 *)(to + (row + k) * HD + dim) = make_uint2(pair(r[k], false), pair(r[k], true));
  }
}

// ---- attention over pages --------------------------------------------------------------------------------------------

// 64 of a request's pages from page `p0` on, one a lane: its id (-1: none, whose keys are hidden) and the head's scales.
struct PageRun {
  int id;
  float ks, vs;
};
__device__ __forceinline__ PageRun page_run(const AttendArgs &a, int r, int kvh, int p0, int lane) {
  const int p = p0 + lane;
  PageRun w;
  w.id = p < a.b.width ? gload(a.b.tables + r * a.b.tables_sr + p) : -1;
  if ((uint32_t)w.id >= (uint32_t)a.c.pages) w.id = -1;
  const float *s = a.c.scales + (int64_t)max(w.id, 0) * (2 * a.c.kv) + kvh;
  w.ks = gload(s), w.vs = gload(s + a.c.kv);
  return w;
}

// Where key `key` lies: its page (0 where it is none, whose keys are hidden), its row there, the head's scales. ONE: blocks of
// 64 keys lie in one page (of 64 tokens or more), so `key` is the wave's and everything here is in scalar registers (a 2048-row
// prompt 64.3 us, without 68.3; decoding alike).
struct PageAt {
  int id, real, in;
  float ks, vs;
};
template <bool ONE> __device__ __forceinline__ PageAt page_at(const PageRun &run, int p0, int key, int lg) {
  PageAt p;
  const int from = (key >> lg) - p0;
  if constexpr (ONE) {
    p.id = __builtin_amdgcn_readlane(run.id, from);
    p.ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(run.ks), from));
    p.vs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(run.vs), from));
  } else {
    p.id = __shfl(run.id, from, 64), p.ks = __shfl(run.ks, from, 64), p.vs = __shfl(run.vs, from, 64);
  }
  p.real = p.id >= 0, p.id = max(p.id, 0), p.in = key & ((1 << lg) - 1);
  return p;
}

__device__ __forceinline__ bf16x8 fp8_to_bf16(uint32_t lo, uint32_t hi, float s) {
  u32x4 w;
  w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true));
  w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false));
  w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true));
  return __builtin_bit_cast(bf16x8, w);
}
// One block of 64 keys against QT tiles of pairs. key: the lane's first key (its 16 are in a row), seen: whether their page
// is one; keys(kt, j) and values(c): the lane's 16 codes of each piece; between: run once the scores are made. Matrix
// instructions on one accumulator are kept 2 QT apart: one that follows its like at once waits for it.
template <int HD, int QT, class Keys, class Values, class Between>
__device__ __forceinline__ void fold_block(const Query<HD> (&q)[QT], Running<HD> (&st)[QT], int key, bool seen, float ks, float vs,
                                           Keys keys, Values values, Between between) {
  constexpr int J = HD / 64, C = HD / 16;
  f32x4 s[QT][4];
#pragma unroll
  for (int kp = 0; kp < 4; kp += 2) {
    bf16x8 kf[2][2 * J];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < J; j++) {
        const u32x4 w = keys(kp + i, j);
        kf[i][2 * j] = fp8_to_bf16(w[0], w[1], ks), kf[i][2 * j + 1] = fp8_to_bf16(w[2], w[3], ks);
      }
#pragma unroll
    for (int k = 0; k < 2 * J; k++)
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
    st[t].weigh(s[t], w[t]);
  }
#pragma unroll
  for (int cp = 0; cp < C; cp += 2) {
    bf16x8 v[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const u32x4 x = values(cp + i);
      v[i][0] = fp8_to_bf16(x[0], x[1], vs), v[i][1] = fp8_to_bf16(x[2], x[3], vs);
    }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int t = 0; t < QT; t++)
          st[t].o[cp + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[i][h], w[t][h], st[t].o[cp + i], 0, 0, 0);
  }
}
// Few query pairs a request: a block of NW waves a part. A part is a run of whole blocks of 64 keys of one request, against QT
// tiles of 16 of its pairs, so every key and value is read and converted once for all of them; the waves take its
// blocks in turn and join by halves through LDS, lane by lane, since every wave's state lies in the same lanes. A block's keys
// are requested while the block before weighs its scores, its values while it multiplies, so 16 KB a wave (heads of 128) are
// always in flight. Two waves a SIMD: held to their registers (the compiler's own choice put O into accumulation registers as
// well, which left one of QT = 2: 16 requests of 5 rows of 4 heads over 2048 keys 20.1 us, 15.2 so).
// Memory bounds it once every CU has its waves: 32 requests of 4096 keys of 8 heads of 128 (269 MB) 44.8 us, 6.0 TB/s; one of
// 65536 23.1 us, 5.8. 8 requests of up to 8191 (101 MB) 19.7 us and 16 of 2048 in drafts (51 MB) 15 us are two or three blocks a
// wave, so the trips to memory before the first and the join in LDS are a third of it. Loads past the caches, since no key is
// read twice (through them, with caches of three steps in turn: 51.5 us for the 44.8). One tile of pairs where 16 will do: 8
// requests of 8191 keys 23.7, with a second one empty 25.9.
// tid: the thread among the part's, which pass every barrier, as other parts of their block may be at work.
template <int HD, int QT, int NW, bool ONE>
__device__ __forceinline__ void few_pairs(const AttendArgs &a, const int block, const int tid, FewLds<HD, QT, NW> &lds) {
  constexpr int J = HD / 64, C = HD / 16;
  const int lane = tid & 63, n = lane & 15, g = lane >> 4, lg = a.c.page_log2;
  Part p;
  take_part<HD, QT, NW>(a, block, tid, &p);
  const int kvh = p.kvh, b0 = p.b0, b1 = p.b1;
  Query<HD> q[QT];
  Running<HD> st[QT];
#pragma unroll
  for (int t = 0; t < QT; t++) {
    if (p.real) q[t].load(a, p, kvh, p.pair0 + 16 * t + n, g);
    st[t].clear();
  }
  if (b0 < b1) {
    const int64_t head = (int64_t)HD << lg;  // codes of one page of one head
    int p0 = b0 * KB >> lg;
    PageRun run = page_run(a, p.r, kvh, p0, lane);
    u32x4 kw[4][J], vw[C];
    const auto turn = [&](int b) {  // the 64 pages that block b's keys lie in, if they are not there yet
      if (((b * KB + KB - 1) >> lg) - p0 >= 64) p0 = b * KB >> lg, run = page_run(a, p.r, kvh, p0, lane);
    };
    const uint8_t *base = a.c.values + kvh * head;
    const int run6 = min(lg, 6);
    const uint32_t krow = ((ONE ? 16 * (n >> 2) : 0) + (n & 3)) * 64 + 16 * g, vrow = (n << run6) + (ONE ? 16 * g : 0);
    const auto fetch_keys = [&](int b) {
      const PageAt at = page_at<ONE>(run, p0, b * KB + (ONE ? 0 : 16 * (n >> 2)), lg);
      const uint8_t *k = base + (int64_t)at.id * (2 * a.c.kv) * head + at.in * 64;
#pragma unroll
      for (int j = 0; j < J; j++) {
        const uint8_t *kj = k + (j << (lg + 6));
#pragma unroll
        for (int kt = 0; kt < 4; kt++) kw[kt][j] = __builtin_nontemporal_load((const u32x4 *)(kj + (krow + 4 * kt * 64)));
      }
    };
    const auto fetch_values = [&](int b) {
      const PageAt at = page_at<ONE>(run, p0, b * KB + (ONE ? 0 : 16 * g), lg);
      const uint8_t *v = base + ((int64_t)at.id * (2 * a.c.kv) + a.c.kv) * head + value_at<HD>(0, at.in, lg);
#pragma unroll
      for (int c = 0; c < C; c++) vw[c] = __builtin_nontemporal_load((const u32x4 *)(v + (c << (run6 + 4)) + vrow));
    };
    fetch_keys(b0), fetch_values(b0);
    for (int b = b0; b < b1; b += NW) {
      const bool more = b + NW < b1;
      // the scales once the codes are requested, so that these don't wait for them
      const PageAt ka = page_at<ONE>(run, p0, b * KB + (ONE ? 0 : 16 * (n >> 2)), lg);
      const PageAt va = page_at<ONE>(run, p0, b * KB + (ONE ? 0 : 16 * g), lg);
      fold_block<HD, QT>(q, st, b * KB + 16 * g, va.real, ka.ks, va.vs, [&](int kt, int j) { return kw[kt][j]; },
                         [&](int c) { return vw[c]; }, [&] {
                           if (more) turn(b + NW), fetch_keys(b + NW);
                         });
      if (more) fetch_values(b + NW);
    }
  }
  finish_part<HD, QT, NW>(a, p, tid, st, lds);
}

template <int HD, int QT, int NW, bool ONE>
__global__ void __launch_bounds__(64 * NW, 2) pages_few_kernel(const AttendArgs a) {
  __shared__ FewLds<HD, QT, NW> lds;
  few_pairs<HD, QT, NW, ONE>(a, blockIdx.x, threadIdx.x, lds);
}

// Many query pairs a request (a prompt's rows): a block takes 128 pairs of one key head against a `splits`th of the blocks of
// keys that they see. Its 8 waves are two halves of 4 that take every other block of keys, each wave 32 pairs, so
// every fragment that a wave converts feeds two matrix instructions; the halves join through LDS at the end. Blocks of 64 keys
// and values pass through LDS as codes, one barrier a step, the next step's codes held in registers meanwhile. 16-byte units are
// placed so that the 16 lanes of a read meet distinct banks: keys' unit u of row r at u ^ (2 (r / 16) + (r / 2) % 2)
// (heads of 64: u ^ (r / 16)), values' unit u of dim d at u ^ (d / 4) % 4.
// The instructions beside the matrix ones bound it: a prompt of 2048 rows of 32 heads of 128 (34.4 GF) 65 us, 529 TFLOP/s; 4096
// rows 217 us, 633 (62 and 213 in a launch without parts, as which the steps below were timed). Vector instructions run 58 % of
// the time and matrix ones 28 %, hardly ever together, since the waves of a block keep step. Dropped: 4 waves of 64 pairs (118
// us for the 62) and 4 of 32 with no halves (78); codes converted once, into bf16 in LDS (63.5 and 226 us for the 62 and 213:
// twice the LDS traffic); scores from 8-bit products with q in two parts (no faster); the halves half a step apart, one at its
// products while the other weighs (68.5 us for the 65), with a barrier between the two as well (72); fences that interleave
// the two kinds, wave priorities and loads from LDS a tile ahead (no change).
template <int HD> struct ManyLds {
  __attribute__((aligned(16))) uint8_t k[2][2][KB * HD], v[2][2][KB * HD];  // [half][stage]
};
template <int HD, bool ONE> __device__ __forceinline__ void many_pairs(const AttendArgs &a, const int block, ManyLds<HD> &lds) {
  constexpr int C = HD / 16, UK = HD / 16, NU = HD * KB / 16 / 256;  // units of a key's row; units a thread
  const int tid = threadIdx.x & 255, lane = tid & 63, n = lane & 15, g = lane >> 4, lg = a.c.page_log2;
  const int half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = block % a.c.kv, unit = block / a.c.kv, split = unit % a.splits;
  const int slot = a.tiles - 1 - unit / a.splits;  // the longest rows first
  Piece p;
  if (!find_tile(a, slot, lane, &p)) return;
  const int pairs = p.n * a.rep, pair0 = TILE * p.k, mine0 = pair0 + 32 * wave;
  Query<HD> q[2];
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
  // the wave's own keys: blocks outside them it only helps to bring in
  const int wlo = low(place(mine0)), whi = mine0 < pairs ? place(mine0 + 32 - 1) : -1;
  const int64_t head = (int64_t)HD << lg;
  int p0 = b0 * KB >> lg;
  PageRun run = page_run(a, p.r, kvh, p0, lane);
  u32x4 kr[NU], vr[NU];
  const uint8_t *base = a.c.values + kvh * head;
  uint32_t kunit[NU], vunit[NU];  // the thread's units in a block of keys, and where each starts in it
#pragma unroll
  for (int i = 0; i < NU; i++) {
    const int u = tid + 256 * i;
    kunit[i] = (u % UK / 4 << (lg + 6)) + (ONE ? u / UK * 64 : u / UK % 16 * 64) + u % 4 * 16;
    vunit[i] = (u / 4 << min(lg, 6)) + (ONE ? 16 * (u & 3) : 0);
  }
  const auto fetch = [&](int b) {
    if (((b * KB + KB - 1) >> lg) - p0 >= 64) p0 = b * KB >> lg, run = page_run(a, p.r, kvh, p0, lane);
    if constexpr (ONE) {
      const PageAt at = page_at<true>(run, p0, b * KB, lg);
      const uint8_t *k = base + (int64_t)at.id * (2 * a.c.kv) * head + at.in * 64;
      const uint8_t *v = base + ((int64_t)at.id * (2 * a.c.kv) + a.c.kv) * head + value_at<HD>(0, at.in, lg);
#pragma unroll
      for (int i = 0; i < NU; i++) kr[i] = gload((const u32x4 *)(k + kunit[i])), vr[i] = gload((const u32x4 *)(v + vunit[i]));
    } else {
#pragma unroll
      for (int i = 0; i < NU; i++) {
        const int u = tid + 256 * i;
        const PageAt k = page_at<false>(run, p0, b * KB + (u / UK & ~15), lg);
        const PageAt v = page_at<false>(run, p0, b * KB + 16 * (u & 3), lg);
        kr[i] = gload((const u32x4 *)(base + (int64_t)k.id * (2 * a.c.kv) * head + k.in * 64 + kunit[i]));
        vr[i] = gload((const u32x4 *)(base + ((int64_t)v.id * (2 * a.c.kv) + a.c.kv) * head + v.in + vunit[i]));
      }
    }
  };
  const auto turned = [](int row) { return HD == 128 ? row >> 4 << 1 | (row >> 1 & 1) : row >> 4; };
  const auto store = [&](int to) {
#pragma unroll
    for (int i = 0; i < NU; i++) {
      const int u = tid + 256 * i, row = u / UK, dim = u / 4;
      *(u32x4 *)(lds.k[half][to] + row * HD + 16 * (u % UK ^ turned(row))) = kr[i];
      *(u32x4 *)(lds.v[half][to] + dim * KB + 16 * ((u & 3) ^ (dim >> 2 & 3))) = vr[i];
    }
  };
  if (b0 + half < b1) fetch(b0 + half), store(0);
  __syncthreads();
  for (int b = b0 + half, now = 0; b - half < b1; b += 2, now ^= 1) {
    const PageAt ka = page_at<ONE>(run, p0, b * KB + (ONE ? 0 : 16 * (n >> 2)), lg);
    const PageAt va = page_at<ONE>(run, p0, b * KB + (ONE ? 0 : 16 * g), lg);
    if (b + 2 < b1) fetch(b + 2);
    if (b < b1 && b * KB <= whi && b * KB + KB > wlo) {
      const uint8_t *k = lds.k[half][now], *v = lds.v[half][now];
      fold_block<HD, 2>(q, st, b * KB + 16 * g, va.real, ka.ks, va.vs,
                        [&](int kt, int j) {
                          const int row = 16 * (n >> 2) + 4 * kt + (n & 3);
                          return *(const u32x4 *)(k + row * HD + 16 * ((4 * j + g) ^ turned(row)));
                        },
                        [&](int c) { return *(const u32x4 *)(v + (16 * c + n) * KB + 16 * (g ^ (n >> 2))); }, [] {});
    }
    if (b + 2 < b1) store(now ^ 1);
    __syncthreads();
  }
  finish_tile<HD>(a, p, {slot, kvh, split}, half, wave, lane, st, (f32x4 *)lds.k, (float *)lds.v);
}

// A batch that may hold both: the tiles of many pairs, then the parts of few, two a block, which fill the CUs that the tiles
// leave. As two launches the parts cost 4.5 to 6 us even where every request has many pairs; 16 requests of 5 rows over 4096 keys
// beside one of 256 over 2048: 70.1 us as four launches, 60.0; 60 of a row over 2000 beside 2 of 512 over 1000: 81.3 and 86.3.
// Dropped: tiles and parts by eights in turn, 78.4 us for those 86.3, but a 2048-row prompt 105 for its 64.9 (idle parts shift
// the tiles); a part to a block of 8 waves, 200 requests of 500 keys beside 8 of 300 rows 101.5 us for 93.1.
template <int HD, bool ONE> __global__ void __launch_bounds__(512, 2) pages_mixed_kernel(const AttendArgs a) {
  __shared__ union {
    ManyLds<HD> many;
    FewLds<HD, 2, 4> few[2];
  } lds;
  const int tiles = a.tiles * a.c.kv * a.splits;
  if ((int)blockIdx.x < tiles) return many_pairs<HD, ONE>(a, blockIdx.x, lds.many);
  const int half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  few_pairs<HD, 2, 4, ONE>(a, 2 * (blockIdx.x - tiles) + half, threadIdx.x & 255, lds.few[half]);
}

// Joins what attention cut, a wave a pair, 4 a block: the parts of a request's keys (request, key head, pair), then the splits of
// the tiles' (tile, key head, pair). Latency: 4.0 to 4.6 us from one part a request to 32.
template <int HD>
__global__ void __launch_bounds__(256) pages_join_kernel(const AttendArgs a) {
  const int lane = threadIdx.x & 63;
  uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Piece p;
  if (unit < a.joins) {
    const uint32_t heads = unit / a.few;
    const int pair = unit - heads * a.few, r = heads / a.c.kv, kvh = heads - r * a.c.kv;
    int f0 = gload(a.b.starts + r), f1 = gload(a.b.starts + r + 1);
    int first = gload(a.b.parts + r), last = gload(a.b.parts + r + 1);
    asm volatile("" : "+v"(f0), "+v"(f1), "+v"(first), "+v"(last));  // all requested at once
    first = __builtin_amdgcn_readfirstlane(first);
    const int parts = __builtin_amdgcn_readfirstlane(last) - first;
    p = Piece{r, 0, __builtin_amdgcn_readfirstlane(min(max(f0, 0), a.b.rows)), 0, 0};
    p.n = __builtin_amdgcn_readfirstlane(min(max(f1, p.row0), a.b.rows)) - p.row0;
    if (parts <= 1 || first + parts > a.items || pair >= p.n * a.rep || p.n * a.rep > a.few) return;
    const int64_t step = (int64_t)a.c.kv * a.few * (HD + 4);
    const float *from = a.scratch + first * step + ((int64_t)kvh * a.few + pair) * (HD + 4);
    join_parts<HD>(from, step, parts, out_row(a, p, kvh, pair), lane);
    return;
  }
  unit -= a.joins;
  const int at = unit & (TILE - 1), kvh = (unit >> TILE_LOG2) % a.c.kv, slot = (unit >> TILE_LOG2) / a.c.kv;
  if (slot >= a.tiles || a.splits == 1 || !find_tile(a, slot, lane, &p)) return;
  const int pair = TILE * p.k + at;
  if (pair >= p.n * a.rep) return;
  join_parts<HD>(a.split_scratch + (((int64_t)slot * a.c.kv + kvh) * a.splits * TILE + at) * (HD + 4), TILE * (HD + 4), a.splits,
                 out_row(a, p, kvh, pair), lane);
}

// ---- entry points ----------------------------------------------------------------------------------------------------

int launch_pages_join(const AttendArgs &a, const AttendPlan &p, int head_dim, hipStream_t s) {
  const int64_t joins = p.joins + (p.splits > 1 ? (int64_t)p.many_tiles * a.c.kv * TILE : 0);
  if (!joins) return BT_OK;
  if (head_dim == 64) pages_join_kernel<64><<<(unsigned)ceil_div(joins, 4), 256, 0, s>>>(a);
  else pages_join_kernel<128><<<(unsigned)ceil_div(joins, 4), 256, 0, s>>>(a);
  BT_LAUNCHED("paged attention's join");
  return BT_OK;
}

template <int HD, bool ONE> static int launch_attend(const AttendArgs &a, const AttendPlan &p, hipStream_t s) {
  const unsigned parts = p.items * a.c.kv * p.groups + (a.b.rows + 15) / 16, tiles = p.many_tiles * a.c.kv;
  if (p.many) pages_mixed_kernel<HD, ONE><<<tiles * p.splits + (parts + 1) / 2, 512, 0, s>>>(a);
  else if (p.tiles == 2) pages_few_kernel<HD, 2, 4, ONE><<<parts, 256, 0, s>>>(a);
  else if (p.waves == 8) pages_few_kernel<HD, 1, 8, ONE><<<parts, 512, 0, s>>>(a);
  else pages_few_kernel<HD, 1, 4, ONE><<<parts, 256, 0, s>>>(a);
  BT_LAUNCHED("paged attention");
  return launch_pages_join(a, p, HD, s);
}

}  // namespace bt

using namespace bt;

extern "C" {

int bt_pages_plan(bt_runtime *rt, const bt_plan_args *a) {
  Runtime *r;
  if (int s = enter(rt, &r)) return s;
  if (!a || !a->tables || !a->cached || !a->fresh || !a->free_pages || !a->starts || !a->lengths || !a->places || !a->slots ||
      !a->taken_out || !a->parts)
    return fail(BT_EINVAL, "a plan needs its tables, lengths, free pages and results");
  if ((a->tables | a->cached | a->fresh | a->free_pages | a->taken | a->starts | a->lengths | a->places | a->slots | a->taken_out |
       a->parts) % 4)
    return fail(BT_EINVAL, "a plan's tensors are int32-aligned");
  int lg = 0;
  while (lg < 9 && (1 << lg) != a->page) lg++;
  if (lg < 4 || lg > 8) return fail(BT_EINVAL, "a page holds 16, 32, 64, 128 or 256 tokens, not %d", a->page);
  if (a->requests < 1 || a->requests > MOST_REQUESTS || a->width < 1 || a->n_free < 1 || a->rows < 1 || a->rows > MOST_ROWS ||
      (int64_t)a->width * a->page > MOST_KEYS || a->most < 1 || a->kv < 1 || a->kv > 1024 || a->pages < 1 ||
      (int64_t)a->pages * a->page > 0x7FFFFFFFll)
    return fail(BT_EINVAL,
                "a plan of %d requests (1 to %d), %d rows (1 to %d), %d a request at most, tables %d wide, %d free of %d pages",
                a->requests, MOST_REQUESTS, a->rows, MOST_ROWS, a->most, a->width, a->n_free, a->pages);
  const auto at = [](uint64_t p) { return (int32_t *)(uintptr_t)p; };
  const PlanArgs k{at(a->tables), at(a->cached), at(a->fresh), at(a->free_pages), at(a->taken), at(a->starts), at(a->lengths),
                   at(a->places), at(a->slots), at(a->taken_out), at(a->parts), a->tables_sr, a->requests, a->width, a->n_free,
                   a->rows, lg, a->pages, std::min(a->most, a->rows), parts_target(a->kv),
                   parts_least((int64_t)a->width * a->page)};
  const int most = std::max(a->requests, a->rows > PLAN_ROWS ? 1 : a->rows);
  const int64_t blocks = (int64_t)a->requests * ceil_div((int64_t)a->width * a->page, KB);  // of keys, at most
  if (blocks > 1 << 30) plan_kernel<1024, true><<<1, 1024, 0, r->stream>>>(k);
  else if (most <= 64) plan_kernel<64, false><<<1, 64, 0, r->stream>>>(k);
  else if (most <= 256) plan_kernel<256, false><<<1, 256, 0, r->stream>>>(k);
  else plan_kernel<1024, false><<<1, 1024, 0, r->stream>>>(k);
  BT_LAUNCHED("a plan");
  if (a->rows > PLAN_ROWS) {
    plan_rows_kernel<<<(unsigned)ceil_div(a->rows, 256), 256, 0, r->stream>>>(k);
    BT_LAUNCHED("a plan's rows");
  }
  return BT_OK;
}

int bt_pages_put(bt_runtime *rt, const bt_pages *pool, const bt_batch *batch, uint64_t x, int64_t x_sb, int64_t x_sr) {
  Runtime *r;
  if (int s = enter(rt, &r)) return s;
  PoolArgs c;
  BatchArgs b;
  if (int s = check_pool(pool, 8, &c)) return s;
  if (int s = check_batch(batch, &b)) return s;
  if (!x || x % 16 || x_sb % 8 || x_sr % 8) return fail(BT_EINVAL, "a paged cache takes rows on 16-byte boundaries");
  const int most = std::min(batch->most, batch->rows);
  // the pages that a request's rows can touch, where they are few; else pieces go by the rows there are, which takes a search
  // (2048 requests of a row: 73.5 us, by a search 89; 32 alike)
  const int each = most == 1 ? 1 : most <= pool->page ? 2 : 0;
  const int64_t blocks = (each ? (int64_t)each * b.requests : (b.rows >> c.page_log2) + 2 * b.requests) * 2 * c.kv;
  if ((int64_t)b.width * pool->page > MOST_KEYS)
    return fail(BT_EINVAL, "tables %d wide of pages of %d tokens hold over 2^30", b.width, pool->page);
  if (!grid_fits(blocks, 256)) return fail(BT_EINVAL, "a put of %d rows of %d heads is too large", b.rows, 2 * c.kv);
  const uint16_t *src = (const uint16_t *)(uintptr_t)x;
  const int top = std::min(most, pool->page);  // the most rows of a request in one page
  const auto launch = [&](auto kernel, int threads) {
    kernel<<<(unsigned)blocks, threads, 0, r->stream>>>(c, b, src, x_sb, x_sr, each);
  };
  if (pool->head_dim == 64) {
    if (top <= 16) launch(put_pages_kernel<64, 64, 16>, 64);
    else if (top <= 64) launch(put_pages_kernel<64, 256, 64>, 256);
    else launch(put_pages_kernel<64, 256, 256>, 256);
  } else {
    if (top <= 16) launch(put_pages_kernel<128, 64, 16>, 64);
    else if (top <= 64) launch(put_pages_kernel<128, 256, 64>, 256);
    else launch(put_pages_kernel<128, 256, 256>, 256);
  }
  BT_LAUNCHED("a paged put");
  return BT_OK;
}

int bt_pages_read(bt_runtime *rt, const bt_pages *pool, uint64_t out) {
  Runtime *r;
  if (int s = enter(rt, &r)) return s;
  PoolArgs c;
  if (int s = check_pool(pool, 8, &c)) return s;
  if (!out || out % 16) return fail(BT_EINVAL, "pages are read to a 16-byte aligned tensor");
  const int64_t blocks = (int64_t)c.pages * 2 * c.kv;
  if (!grid_fits(blocks, 256)) return fail(BT_EINVAL, "%d pages of %d heads are too many to read at once", c.pages, 2 * c.kv);
  const auto launch = [&](auto kernel) { kernel<<<(unsigned)blocks, 256, 0, r->stream>>>(c, (uint16_t *)(uintptr_t)out); };
  if (pool->head_dim == 64) pool->page <= 64 ? launch(read_pages_kernel<64, 64>) : launch(read_pages_kernel<64, 256>);
  else pool->page <= 64 ? launch(read_pages_kernel<128, 64>) : launch(read_pages_kernel<128, 256>);
  BT_LAUNCHED("reading pages");
  return BT_OK;
}

int bt_pages_attend_scratch(const bt_pages *pool, const bt_batch *batch, int32_t heads, int32_t window, uint64_t *bytes) {
  if (!bytes) return fail(BT_EINVAL, "no result pointer");
  AttendPlan p;
  if (int s = plan_attend(pool, 8, batch, heads, window, &p)) return s;
  *bytes = p.scratch + p.split_scratch;
  return BT_OK;
}

int bt_pages_attend(bt_runtime *rt, const bt_pages *pool, const bt_batch *batch, uint64_t q, int64_t q_sh, int64_t q_sr,
                    uint64_t out, int64_t o_sh, int64_t o_sr, int32_t heads, int32_t window, uint64_t scratch,
                    uint64_t scratch_bytes) {
  Runtime *r;
  if (int s = enter(rt, &r)) return s;
  AttendPlan p;
  AttendArgs a;
  if (int s = attend_args(pool, 8, batch, q, q_sh, q_sr, out, o_sh, o_sr, heads, window, scratch, scratch_bytes, &p, &a)) return s;
  const bool one = pool->page >= KB;
  if (pool->head_dim == 64) return one ? launch_attend<64, true>(a, p, r->stream) : launch_attend<64, false>(a, p, r->stream);
  return one ? launch_attend<128, true>(a, p, r->stream) : launch_attend<128, false>(a, p, r->stream);
}

}  // extern "C"
