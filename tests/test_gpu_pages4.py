"""The paged 4-bit cache on the GPU, against oracle/pages.py in 64 bits: puts exactly, attention within what its roundings allow.
Needs a GPU."""
import ctypes
import numpy as np
import pytest

from baretile_amd import _lib
from baretile_amd.pages import Pages
from baretile_amd.tensor import Recording, Storage, Tensor, jit
from oracle import bfp as B, pages as P
from test_gpu_pages import bf16_rows, ints, planned, row

pytestmark = pytest.mark.gpu


def pool4(rt, pages, kv, hd, page): return Pages(rt, pages, kv, hd, page, bits=4)


def whole(pool): return np.array(pool.values().tolist()).reshape(pool.pages, 2 * pool.kv, pool.page, pool.head)


# ---- puts

@pytest.mark.parametrize("hd, kv, page", [(64, 1, 16), (128, 2, 32), (64, 3, 64), (128, 1, 128), (128, 5, 256), (64, 2, 256)])
def test_put(rt, hd, kv, page):
  rng = np.random.default_rng(hd + kv + page)
  pool = pool4(rt, 24, kv, hd, page)
  assert pool.bits == 4 and not whole(pool).any()
  values = np.zeros((24, 2 * kv, page, hd))
  tables, lengths, taken = np.full((5, 6), -1), np.zeros(5, int), 0
  free = rng.permutation(24)
  for step, new in enumerate(([page + 3, 1, 0, 2 * page, 5], [1, 1, 1, 1, 1], [0, page - 1, 2, 1, 7], [1, 2, 0, 17, 3], [3, 1, 4, 1, 1])):
    rows = sum(new) + 2
    x = bf16_rows(rng, 2 * kv, rows, hd) * 4.0 ** (step % 3)
    b, (tables, starts, lengths, _, _, taken) = planned(rt, pool, tables, lengths, new, free, rows, taken)
    pool.put(b, Tensor.of(rt, x))
    P.put4(values, tables, starts, lengths, x)
    assert np.array_equal(whole(pool), values), step
  assert (values != 0).any(axis=(1, 2, 3)).sum() == taken  # pages of no request stay as they were


@pytest.mark.parametrize("most", [None, 1, 3, 16])
def test_put_of_many_requests(rt, most):
  # enough pieces that blocks take four heads each; a request's rows found by a search, or by its number
  rng = np.random.default_rng(most or 0)
  kv, hd, page, R = 3, 64, 32, 700
  pool = pool4(rt, 1500, kv, hd, page)
  cached, new = rng.integers(0, 40, R), rng.integers(0, 24, R)
  rows = int(np.minimum(new, most or 99).sum()) + 5
  x = bf16_rows(rng, 2 * kv, rows, hd)
  b, (tables, starts, lengths, *_) = planned(rt, pool, np.full((R, 3), -1), cached, new, rng.permutation(1500), rows, most=most)
  values = np.zeros((1500, 2 * kv, page, hd))
  pool.put(b, Tensor.of(rt, x))
  P.put4(values, tables, starts, lengths, x)
  assert np.array_equal(whole(pool), values)


def test_put_of_every_border(rt):
  # every quotient of a bf16 value and a scale that falls on a border between two codes, and its neighbours on both sides, for
  # each of a value's four leading digits and a key's one
  pool = pool4(rt, 1, 1, 128, 256)
  x = np.zeros((2, 200, 128), np.float32)
  borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
  r = 0
  for k in (4, 5, 6, 7):
    for e in (-90, -3, 0, 5, 95):
      s = k / 4 * 2.0 ** e
      at = B.bf16(borders * s)
      bits = B.bf16_bits(at).astype(np.int64)
      near = np.concatenate([((bits + d) << 16).astype(np.uint32).view(np.float32) for d in (-2, -1, 0, 1, 2)])
      for h in (0, 1):
        scale = 2.0 ** e if h == 0 else s
        x[h, r, :35], x[h, r, 35:70] = near, -near
        for g in range(0, 128, 32): x[h, r, g + 31] = 7 * scale  # what makes the scale, in each 32 dims of a key
        x[h, r][np.abs(x[h, r]) > 7 * scale] = 0
      r += 1
  x = B.bf16(x)
  b, (tables, starts, lengths, *_) = planned(rt, pool, np.full((1, 1), -1), [0], [200], [0], 200)
  pool.put(b, Tensor.of(rt, x))
  values = np.zeros((1, 2, 256, 128))
  P.put4(values, tables, starts, lengths, x)
  assert np.array_equal(whole(pool), values)


def test_put_of_odd_values(rt):
  pool = pool4(rt, 3, 1, 64, 16)
  x = np.zeros((2, 20, 64))
  x[:, 0, :8] = [np.inf, -np.inf, np.nan, 3.0, -1e-3, 448, -449, 1e-30]  # infinities and NaNs don't count for the scale
  x[:, 1, 0], x[:, 2, 0], x[:, 3, :2], x[:, 3, 40] = 3e38, 1e-38, [np.nan, -np.inf], 2.0
  x[:, 16] = B.bf16(2.0 ** -133 * np.arange(64))  # smaller than any scale's grid
  x[:, 17, :4] = [np.inf, np.inf, np.nan, 0]  # nothing finite but zeros
  x[:, 18, 1], x[:, 19, 1] = 7 * 2.0 ** 100, -7 * 2.0 ** -100
  bits = (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)
  x = (bits.astype(np.uint32) << 16).view(np.float32)
  b, (tables, starts, lengths, *_) = planned(rt, pool, np.full((1, 2), -1), [0], [20], np.arange(3), 20)
  values = np.zeros((3, 2, 16, 64))
  pool.put(b, Tensor.frombytes(rt, 20, 64, bits.tobytes(), 2))
  P.put4(values, tables, starts, lengths, x)
  assert np.array_equal(whole(pool), values)


def test_what_a_page_holds_does_not_depend_on_its_puts(rt):
  rng = np.random.default_rng(3)
  x = B.bf16(bf16_rows(rng, 4, 70, 128) * np.exp(rng.normal(0, 2, (1, 70, 1))))
  stored = []
  for runs in ([70], [1] * 70, [5, 1, 30, 2, 17, 15]):
    pool, tables, at, taken = pool4(rt, 4, 2, 128, 32), np.full((1, 4), -1), 0, 0
    for n in runs:
      b, (tables, *_, taken) = planned(rt, pool, tables, [at], [n], [2, 0, 3, 1], n, taken)
      pool.put(b, Tensor.of(rt, x[:, at:at + n]))
      at += n
    stored.append(rt.download(pool.storage.addr, pool.storage.nbytes))
  assert bytes(stored[0]) == bytes(stored[1]) == bytes(stored[2])


def test_put_drops_rows_without_a_page_and_takes_strided_rows(rt):
  rng = np.random.default_rng(4)
  pool = pool4(rt, 5, 1, 64, 16)
  tables = np.array([[2, -1, 7], [0, 1, -1]])
  cached, new = [10, 20], [30, 20]
  x = bf16_rows(rng, 2, 60, 192)  # wider rows, of which the middle is put
  b, (made, starts, lengths, *_) = planned(rt, pool, tables, cached, new, [9, 4], 60)
  values = np.zeros((5, 2, 16, 64))
  pool.put(b, Tensor.of(rt, x)[:, :, 64:128])
  P.put4(values, made, starts, lengths, x[:, :, 64:128])
  assert np.array_equal(whole(pool), values)


def test_refused_drafts_places_are_put_again(rt):
  rng = np.random.default_rng(5)
  pool, values, tables = pool4(rt, 3, 2, 128, 16), np.zeros((3, 4, 16, 128)), np.full((1, 3), -1)
  taken = 0
  for cached, new in ((0, 21), (13, 6), (13, 1), (14, 20)):
    x = B.bf16(bf16_rows(rng, 4, new, 128) * (100.0 if cached == 13 else 1.0))
    b, (tables, starts, lengths, _, _, taken) = planned(rt, pool, tables, [cached], [new], [1, 2, 0], new, taken)
    pool.put(b, Tensor.of(rt, x))
    P.put4(values, tables, starts, lengths, x)
    assert np.array_equal(whole(pool), values)


# ---- attention

def bound(q, values, weighed, out, keys):
  """How far an output may be from the oracle's: the weights' rounding to bf16 times their value's scale (2^-8 of the weighed |v|),
  the output's, the fp32 scores' (4 roundings of a sum of hd products, doubled for the weights' sum) and a rounding a key of the
  weights' sum."""
  size = np.linalg.norm(q, axis=-1).max() * np.linalg.norm(values, axis=-1).max()
  return weighed * (2.0 ** -8 + (8 * q.shape[-1] * (1 + size) + keys) * 2.0 ** -24) + 2.0 ** -8 * np.abs(out) + 1e-30


def filled(rt, rng, kv, hd, page, lengths, spare=3):
  """A pool with rows of every request in it, (pool, values, tables)."""
  width = max(1, -(-max(lengths) // page))
  pages = sum(-(-n // page) for n in lengths) + spare
  pool = pool4(rt, pages, kv, hd, page)
  values = np.zeros((pages, 2 * kv, page, hd))
  rows = max(1, sum(lengths))
  x = bf16_rows(rng, 2 * kv, rows, hd)
  b, (tables, starts, *_) = planned(rt, pool, np.full((len(lengths), width), -1), [0] * len(lengths), lengths, rng.permutation(pages), rows)
  pool.put(b, Tensor.of(rt, x))
  P.put4(values, tables, starts, lengths, x)
  return pool, values, tables


def attended(rt, rng, heads, kv, hd, page, lengths, new, window=0, spare=0, tables=None, merged=False, most=None):
  pool, values, made = filled(rt, rng, kv, hd, page, lengths)
  if tables is not None: made = tables(made)
  rows = sum(new) + spare
  q = B.bf16(rng.normal(0, 1, (heads, rows, hd)) * 1.5 / np.sqrt(hd))
  b, (made, starts, total, *_) = planned(rt, pool, made, [n - m for n, m in zip(lengths, new)], new, [-1], rows, most=most)
  out = pool.attend(Tensor.of(rt, q), b, window, merged)
  got = np.array(out.tolist())
  if merged: got = got.reshape(rows, heads, hd).transpose(1, 0, 2)
  got = got.reshape(heads, rows, hd)
  want, weighed = P.attend(q, values, made, starts, total, window)
  assert np.all(np.abs(got - want) <= bound(q, values, weighed, want, max(lengths))), np.abs(got - want).max()
  return got, want


@pytest.mark.parametrize("heads, kv, hd, page", [(8, 2, 64, 16), (4, 4, 128, 32), (32, 8, 128, 64), (9, 3, 64, 128), (7, 1, 128, 256), (20, 1, 64, 16),
                                                 (8, 2, 128, 16), (6, 2, 64, 32)])
@pytest.mark.parametrize("lengths, new", [([1], [1]), ([300], [1]), ([64, 0, 1, 65, 500], [1, 0, 1, 1, 1]), ([700, 63, 129], [5, 3, 0]),
                                          ([200, 90], [9, 7])])
def test_attend_few_rows(rt, heads, kv, hd, page, lengths, new):
  attended(rt, np.random.default_rng(heads + page + sum(lengths)), heads, kv, hd, page, lengths, new, spare=2, merged=page == 64)


@pytest.mark.parametrize("heads, kv, hd, page", [(8, 2, 64, 16), (4, 1, 128, 64), (6, 2, 128, 32), (3, 3, 64, 256), (4, 2, 64, 64), (4, 2, 128, 16)])
@pytest.mark.parametrize("lengths, new", [([130], [130]), ([333, 1, 200], [140, 1, 90]), ([520, 64], [71, 64])])
def test_attend_many_rows(rt, heads, kv, hd, page, lengths, new):
  attended(rt, np.random.default_rng(heads + page + sum(lengths)), heads, kv, hd, page, lengths, new, spare=17)


@pytest.mark.parametrize("new", [[1, 1, 0], [2, 1, 40]])
def test_attend_many_heads_to_one(rt, new):
  attended(rt, np.random.default_rng(12), 130, 1, 64, 32, [700, 90, 50], new)  # a token's pairs pass a tile


@pytest.mark.parametrize("requests", [65, 2048])
def test_many_requests(rt, requests):
  rng = np.random.default_rng(requests)
  lengths = rng.integers(0, 40, requests)
  new = np.minimum(lengths, rng.choice([0, 1, 3], requests))
  attended(rt, rng, 4, 2, 64, 16, lengths.tolist(), new.tolist(), spare=3, most=3)
  lengths[requests // 2], new[requests // 2] = 100, 50
  attended(rt, rng, 4, 2, 64, 16, lengths.tolist(), new.tolist())


@pytest.mark.parametrize("hd, page", [(64, 16), (64, 64), (128, 16), (128, 64)])
def test_many_requests_beside_prompts(rt, hd, page):
  # tiles enough that each is a block of 4 waves, most of them of requests with few rows, whose parts lie behind them
  rng = np.random.default_rng(hd + page)
  lengths = rng.integers(0, 70, 330)
  new = np.minimum(lengths, rng.choice([0, 1, 3], 330))
  lengths[[5, 200, 329]], new[[5, 200, 329]] = [150, 90, 300], [100, 70, 130]
  attended(rt, rng, 4, 2, hd, page, lengths.tolist(), new.tolist(), spare=3)


def test_puts_of_many_rows_of_wide_heads(rt):
  # blocks of four waves, for heads of 128
  rng = np.random.default_rng(21)
  filled_pool, values, _ = filled(rt, rng, 4, 128, 64, [5000, 17, 900, 1, 0, 333])
  assert np.array_equal(whole(filled_pool), values)


def test_a_long_cache_of_wide_heads(rt):
  # parts long enough for blocks of 8 waves
  attended(rt, np.random.default_rng(22), 4, 1, 128, 256, [140000, 5], [1, 1], most=1)
  attended(rt, np.random.default_rng(23), 2, 2, 64, 64, [9000, 70], [2, 1], most=2)


@pytest.mark.parametrize("window", [1, 7, 64, 100, 1000])
@pytest.mark.parametrize("lengths, new", [([300, 40], [1, 3]), ([400, 150], [100, 70])])
def test_attend_window(rt, window, lengths, new):
  attended(rt, np.random.default_rng(window), 8, 2, 64, 16, lengths, new, window)


@pytest.mark.parametrize("hd, page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("new, window", [([1, 1, 5], 0), ([4, 0, 1], 1019), ([3, 1, 70], 1020), ([1, 1, 1], 40)])
def test_attend_over_long_tables(rt, hd, page, new, window):
  # keys in parts or in one, by the window and the tables
  attended(rt, np.random.default_rng(window), 8, 2, hd, page, [5000, 90, 2001], new, window, most=max(new))


@pytest.mark.parametrize("new", [[1, 3, 1], [90, 80, 1]])
@pytest.mark.parametrize("hd, page", [(64, 16), (128, 64)])
def test_attend_hides_pages_that_are_none(rt, hd, page, new):
  def holes(t):
    t = t.copy()
    t[0, 1], t[0, 2], t[1, 0], t[2, :] = -1, 10 ** 6, -2 ** 31, -1
    return t
  got, want = attended(rt, np.random.default_rng(5), 8, 2, hd, page, [200, 120, 30], new, tables=holes)
  assert not want[:, -1].any()  # a request with no page at all: its row sees nothing


@pytest.mark.parametrize("new", [[1, 2], [40, 2], [17, 30]])
def test_attend_long(rt, new):
  attended(rt, np.random.default_rng(6), 4, 1, 64, 64, [40000, 100], new)  # parts, and a prompt's keys in splits


def test_a_long_cache(rt):
  # 300000 tokens, over 1172 pages that 19 loads of a wave's page table bring in
  attended(rt, np.random.default_rng(17), 4, 1, 64, 256, [300000, 5], [1, 1], most=1)
  attended(rt, np.random.default_rng(18), 4, 1, 64, 16, [90000, 5], [2, 1], window=30000)


@pytest.mark.parametrize("hd, page, window", [(64, 16, 0), (128, 32, 0), (64, 16, 1500), (128, 128, 700), (64, 256, 0)])
@pytest.mark.parametrize("new", [[1, 2], [4, 70]])
def test_attend_past_a_wave_of_pages(rt, hd, page, window, new):
  attended(rt, np.random.default_rng(hd + page), 4, 2, hd, page, [3100, 2500], new, window, spare=5)


def test_attend_weighs_rows_of_every_size(rt):
  # values of sizes from 2^-100 to 2^96, a request of each: a weight times its scale keeps its precision
  rng = np.random.default_rng(20)
  sizes = 2.0 ** np.array([-96, -40, 0, 40, 96])
  pool = pool4(rt, 10, 1, 64, 32)
  x = bf16_rows(rng, 2, 200, 64)
  x[1] = B.bf16(x[1] / np.abs(x[1]).max() * np.repeat(sizes, 40)[:, None])
  b, (tables, starts, total, *_) = planned(rt, pool, np.full((5, 2), -1), [0] * 5, [40] * 5, np.arange(10), 200)
  values = np.zeros((10, 2, 32, 64))
  pool.put(b, Tensor.of(rt, x))
  P.put4(values, tables, starts, total, x)
  q = B.bf16(rng.normal(0, 0.2, (4, 200, 64)))
  got = np.array(pool.attend(Tensor.of(rt, q), b).tolist())
  want, weighed = P.attend(q, values, tables, starts, total)
  size = np.linalg.norm(q, axis=-1).max() * np.linalg.norm(values[:, 0], axis=-1).max()
  allowed = weighed * (2.0 ** -8 + (8 * 64 * (1 + size) + 40) * 2.0 ** -24) + 2.0 ** -8 * np.abs(want)
  assert np.all(np.abs(got - want) <= allowed + weighed.max(-1, keepdims=True) * 2.0 ** -24)


def test_attend_a_row_that_is_not_a_number(rt):
  rng = np.random.default_rng(7)
  for new in ([2, 2], [40, 40]):
    pool, values, tables = filled(rt, rng, 2, 64, 16, [300, 90])
    rows = sum(new)
    q = B.bf16(rng.normal(0, 0.2, (4, rows, 64)))
    bits = B.bf16_bits(q)
    bits[1, 1, 3], bits[2, new[0], 0] = 0x7FC0, 0x7F80  # one row's head with a NaN, one with an infinity
    b, (tables, starts, total, *_) = planned(rt, pool, tables, [300 - new[0], 90 - new[1]], new, [-1], rows)
    got = np.array(pool.attend(Tensor.frombytes(rt, rows, 64, bits.tobytes(), 4), b).tolist())
    want, weighed = P.attend(q, values, tables, starts, total)
    ok = np.ones((4, rows), bool)
    ok[1, 1] = ok[2, new[0]] = False
    assert np.isnan(got[1, 1]).all() and np.isnan(got[2, new[0]]).all()
    assert np.all(np.abs(got - want)[ok] <= bound(q, values, weighed, want, 300)[ok])


def test_attend_masks_what_a_page_held_before(rt):
  rng = np.random.default_rng(8)
  pool, values, tables = filled(rt, rng, 2, 64, 16, [100])
  page = int(tables[0, 5])  # the request ends; another takes a page of it, whose other rows are the old request's
  b, (t, starts, total, *_) = planned(rt, pool, np.full((1, 1), -1), [0], [5], [page], 5)
  x = bf16_rows(rng, 4, 5, 64)
  pool.put(b, Tensor.of(rt, x))
  P.put4(values, t, starts, total, x)
  assert np.array_equal(whole(pool), values)
  q = B.bf16(rng.normal(0, 0.2, (5, 8 * 64)))
  got = np.array(pool.attend(Tensor.of(rt, q).split(8), b).tolist())
  q = q.reshape(5, 8, 64).transpose(1, 0, 2)
  want, weighed = P.attend(q, values, t, starts, total)
  assert np.all(np.abs(got - want) <= bound(q, values, weighed, want, 5))


def test_attend_repeats_itself(rt):
  rng = np.random.default_rng(9)
  pool, _, tables = filled(rt, rng, 2, 128, 64, [3000, 50, 900])
  q = Tensor.of(rt, B.bf16(rng.normal(0, 0.2, (8, 12, 128))))
  b, _ = planned(rt, pool, tables, [2996, 46, 896], [4, 4, 4], [-1], 12)
  first = pool.attend(q, b).tobytes()
  for _ in range(5): assert pool.attend(q, b).tobytes() == first


# ---- together

def test_a_recorded_step_follows_its_lengths(rt):
  # plan, put and attention recorded once, over a pool of 4 bits and one of 8 that share the plan; each replay takes lengths and
  # rows of its own
  rng = np.random.default_rng(10)
  heads, kv, hd, page, R, rows = 8, 2, 64, 16, 3, 9
  pool, other = pool4(rt, 40, kv, hd, page), Pages(rt, 40, kv, hd, page)
  free = rng.permutation(40)
  tables, fr = Tensor.of(rt, np.full((R, 10), -1), "int32"), row(rt, free)
  cached, new, taken = row(rt, [0] * R), row(rt, [0] * R), row(rt, [0])
  x, q = Tensor.zeros(rt, rows, hd, 2 * kv), Tensor.zeros(rt, rows, hd, heads)
  def step():
    b = pool.plan(tables, cached, new, fr, rows, taken, most=4)
    pool.put(b, x)
    other.put(b, x)
    o = pool.attend(q, b)
    taken.assign(b.taken)
    cached.assign(b.lengths - 0)
    return b, o, other.attend(q, b), pool.values()
  step()
  rt.wait()
  for t, v in ((tables, np.full((R, 10), -1)), (cached, [[0] * R]), (taken, [[0]])): t.assign(Tensor.of(rt, np.array(v), "int32"))
  rec = Recording(rt)
  with rec: out = step()
  values, values8, s8 = np.zeros((40, 2 * kv, page, hd)), np.zeros((40, 2 * kv, page, hd)), np.full((40, 2 * kv), 2.0 ** -100)
  want_tables, want_cached, want_taken = np.full((R, 10), -1), np.zeros(R, int), 0
  for i in range(8):
    n = rng.integers(0, 6, R)  # some past `most`
    xs, qs = bf16_rows(rng, 2 * kv, rows, hd) * 2.0 ** i, B.bf16(rng.normal(0, 0.2 / 2.0 ** i, (heads, rows, hd)))
    new.assign(row(rt, n))
    x.assign(Tensor.of(rt, xs))
    q.assign(Tensor.of(rt, qs))
    rec.send()
    rt.wait()
    want_tables, starts, total, places, slots, want_taken = P.plan(want_tables, want_cached, n, free, rows, page, 40, want_taken, 4)
    P.put4(values, want_tables, starts, total, xs)
    P.put(values8, s8, want_tables, starts, total, xs)
    b, o, o8, v = out
    assert np.array_equal(np.array(tables.tolist()), want_tables) and np.array_equal(ints(b.slots), slots)
    assert np.array_equal(whole(pool), values) and np.array_equal(np.array(v.tolist()).reshape(values.shape), values)
    for got, held in ((o, values), (o8, values8)):
      want, weighed = P.attend(qs, held, want_tables, starts, total)
      assert np.all(np.abs(np.array(got.tolist()) - want) <= bound(qs, held, weighed, want, 64)), i
    want_cached = total


def test_a_jit_step_takes_its_tables_and_rows(rt):
  rng = np.random.default_rng(14)
  pool = pool4(rt, 12, 2, 64, 16)
  free = rng.permutation(12)
  fr = row(rt, free)
  def step(tables, cached, new, taken, x, q):
    b = pool.plan(tables, cached, new, fr, 30, taken)
    pool.put(b, x)
    return pool.attend(q, b)
  f = jit(step)
  values = np.zeros((12, 4, 16, 64))
  tables, want_tables, cached, used = Tensor.of(rt, np.full((2, 6), -1), "int32"), np.full((2, 6), -1), np.zeros(2, int), 0
  for new in ([20, 3], [1, 4], [0, 12], [5, 1]):
    x, q = bf16_rows(rng, 4, 30, 64), B.bf16(rng.normal(0, 0.2, (8, 30, 64)))
    got = np.array(f(tables, row(rt, cached), row(rt, new), row(rt, [used]), Tensor.of(rt, x), Tensor.of(rt, q)).tolist())
    want_tables, starts, total, _, _, used = P.plan(want_tables, cached, new, free, 30, 16, 12, used)
    P.put4(values, want_tables, starts, total, x)
    want, weighed = P.attend(q, values, want_tables, starts, total)
    assert np.array_equal(np.array(tables.tolist()), want_tables) and np.array_equal(whole(pool), values)
    assert np.all(np.abs(got - want) <= bound(q, values, weighed, want, 64))
    cached = total


def test_rows_that_are_views(rt):
  rng = np.random.default_rng(15)
  pool, lengths, rows, free = pool4(rt, 20, 2, 64, 16), [40, 0, 17], 60, rng.permutation(20)
  x, q = bf16_rows(rng, 4, 2 * rows, 64), B.bf16(rng.normal(0, 0.2, (8, rows, 64)))
  b, (tables, starts, total, *_) = planned(rt, pool, np.full((3, 6), -1), [0, 0, 0], lengths, free, rows)
  pool.put(b, Tensor.of(rt, x)[:, rows // 2:rows // 2 + rows, :])
  values = np.zeros((20, 4, 16, 64))
  P.put4(values, tables, starts, total, x[:, rows // 2:rows // 2 + rows])
  assert np.array_equal(whole(pool), values)
  got = np.array(pool.attend(Tensor.of(rt, np.concatenate([q[:, :3], q], 1))[:, 3:, :], b).tolist())
  want, weighed = P.attend(q, values, tables, starts, total)
  assert np.all(np.abs(got - want) <= bound(q, values, weighed, want, 40))


def test_pages_past_32_bits(rt):
  # the last pages of a pool of 5.5 GB hold what the first of a small one do, bit for bit
  rng = np.random.default_rng(16)
  kv, hd, page, n = 2, 128, 256, 80000
  lengths = [700, 300]
  x, q = Tensor.of(rt, bf16_rows(rng, 2 * kv, 1000, hd)), Tensor.of(rt, B.bf16(rng.normal(0, 0.2, (8, 1000, hd))))
  outs = []
  for pages in (5, n):
    pool = pool4(rt, pages, kv, hd, page)
    b = pool.plan(Tensor.of(rt, np.full((2, 3), -1), "int32"), row(rt, [0, 0]), row(rt, lengths), row(rt, range(pages - 5, pages)), 1000)
    pool.put(b, x)
    step = pool.plan(b.tables, row(rt, [699, 298]), row(rt, [1, 2]), row(rt, [-1]), 3)
    size = pool.storage.nbytes // pages
    outs.append([pool.attend(q, b).tobytes(), pool.attend(q[:, :3, :], step).tobytes(),
                 bytes(rt.download(pool.storage.addr + (pages - 5) * size, 5 * size)),
                 pool.values()[(pages - 5) * 2 * kv:, :, :].contiguous().tobytes()])
    del pool, b, step
  assert outs[0] == outs[1]


def test_a_closed_runtime(chip):
  from baretile_amd.runtime import Runtime
  first = Runtime(chip)
  pool = pool4(first, 4, 2, 64, 16)
  b = pool.plan(Tensor.of(first, [[-1]], "int32"), row(first, [0]), row(first, [1]), row(first, [0]), 1)
  x, q = Tensor.zeros(first, 1, 64, 4), Tensor.zeros(first, 1, 64, 4)
  second = Runtime(chip)
  try:
    for f in (lambda: pool.put(b, x), lambda: pool.attend(q, b), pool.values, lambda: pool4(first, 4, 2, 64, 16)):
      with pytest.raises(RuntimeError): f()
    other = pool4(second, 4, 2, 64, 16)
    with pytest.raises(ValueError, match="batch must be planned"): other.put(b, Tensor.zeros(second, 1, 64, 4))
  finally: second.close()


@pytest.mark.parametrize("hd, page, lengths, new, window", [(128, 16, [700, 30, 65], [1, 2, 1], 0), (64, 64, [3000, 90, 1], [5, 5, 1], 0),
                                                            (128, 64, [500, 200, 40], [100, 1, 40], 0), (64, 16, [2000, 90, 40], [70, 2, 40], 300)])
def test_stays_within_its_memory(rt, hd, page, lengths, new, window):
  # put, attend and read between guards: what lies before and behind the pool and the results keeps its bits
  rng = np.random.default_rng(hd + page)
  kv, heads, rows = 2, 8, sum(new) + 3
  pages = sum(-(-n // page) for n in lengths)
  need, guard = ctypes.c_uint64(), 4096
  args = _lib.PagesArgs(0, 0, pages, page, kv, hd)
  _lib.call("pages4_bytes", ctypes.byref(args), ctypes.byref(need))
  pool = pool4(rt, pages, kv, hd, page)
  def guarded(nbytes):
    s = Storage(rt, nbytes + 2 * guard)
    rt.fill32(s.addr, 0xA5A5A5A5, s.nbytes // 4)
    return s
  def kept(s, nbytes):
    got = bytes(rt.download(s.addr, s.nbytes))
    assert got[:guard] == b"\xa5" * guard and got[guard + nbytes:] == b"\xa5" * (len(got) - guard - nbytes)
  store = guarded(need.value)
  rt.fill32(store.addr + guard, 0, need.value // 4)
  args.values = store.addr + guard
  b, _ = planned(rt, pool, np.full((3, max(-(-n // page) for n in lengths)), -1), [0] * 3, lengths, rng.permutation(pages), sum(lengths))
  x = Tensor.of(rt, bf16_rows(rng, 2 * kv, sum(lengths), hd))
  pool.put(b, x)
  rt.run("put", "pages4_put", ctypes.byref(args), ctypes.byref(b.args), x.addr, x.sb, x.sr)
  kept(store, need.value)
  assert bytes(rt.download(args.values, need.value)) == bytes(rt.download(pool.storage.addr, need.value))
  out = guarded(pages * 2 * kv * page * hd * 2)
  rt.run("read", "pages4_read", ctypes.byref(args), out.addr + guard)
  kept(out, pages * 2 * kv * page * hd * 2)
  step, _ = planned(rt, pool, np.array(b.tables.tolist()), [n - m for n, m in zip(lengths, new)], new, [-1], rows)
  q = Tensor.of(rt, B.bf16(rng.normal(0, 0.2, (heads, rows, hd))))
  _lib.call("pages4_attend_scratch", ctypes.byref(args), ctypes.byref(step.args), heads, window, ctypes.byref(need))
  scratch, o = guarded(need.value), guarded(heads * rows * hd * 2)
  rt.run("attend", "pages4_attend", ctypes.byref(args), ctypes.byref(step.args), q.addr, q.sb, q.sr, o.addr + guard, rows * hd, hd, heads, window,
         scratch.addr + guard, need.value)
  kept(scratch, need.value)
  kept(o, heads * rows * hd * 2)
  assert bytes(rt.download(o.addr + guard, heads * rows * hd * 2)) == pool.attend(q, step, window).tobytes()
  kept(store, args.pages * kv * page * (hd + hd // 32 + 2))


@pytest.mark.parametrize("new, most", [([1, 1, 1], 1), ([3, 9, 2], 9), ([40, 3, 20], None)])
@pytest.mark.parametrize("hd, page", [(64, 16), (128, 64)])
def test_stray_starts_and_lengths_touch_nothing_else(rt, hd, page, new, most):
  # starts and lengths that no plan makes: any rows and places, but nothing outside the pool's and the results' memory
  rng = np.random.default_rng(hd + sum(new))
  kv, heads, rows, guard = 2, 4, sum(new) + 2, 1 << 16
  pool, width = pool4(rt, 12, kv, hd, page), 4
  store = Storage(rt, pool.storage.nbytes + 2 * guard)
  rt.fill32(store.addr, 0xA5A5A5A5, store.nbytes // 4)
  rt.fill32(store.addr + guard, 0, pool.storage.nbytes // 4)
  args = _lib.PagesArgs(store.addr + guard, 0, 12, page, kv, hd)
  tables = rng.permutation(12).reshape(3, 4)
  b, _ = planned(rt, pool, tables, [5, 0, 7], new, [-1], rows, most=most)
  x, q = Tensor.of(rt, bf16_rows(rng, 2 * kv, rows, hd)), Tensor.of(rt, B.bf16(rng.normal(0, 0.2, (heads, rows, hd))))
  n = heads * rows * hd * 2
  out = Storage(rt, n + 2 * guard)
  rt.fill32(out.addr, 0xA5A5A5A5, out.nbytes // 4)
  need = ctypes.c_uint64()
  _lib.call("pages4_attend_scratch", ctypes.byref(args), ctypes.byref(b.args), heads, 0, ctypes.byref(need))
  scratch = Storage(rt, max(need.value, 16))
  big = 2 ** 31 - 1
  for starts, lengths in (([0, 10, 9000, 9001], [5, 6, 7]), ([-5, 1, 2, 3], [0, -9, 40]), ([3, 1, 0, 2], [big, big - 3, -big]), ([0, 1, 2, 3], [big, big, big]),
                          ([0, rows, rows, rows], [big, 0, 0]), ([big, -big, big, 0], [-1, big, 12]), ([0, 1, 2, 3], [width * page, width * page + 1, 1 << 30])):
    b.starts.assign(row(rt, starts))
    b.lengths.assign(row(rt, lengths))
    rt.run("put", "pages4_put", ctypes.byref(args), ctypes.byref(b.args), x.addr, x.sb, x.sr)
    rt.run("attend", "pages4_attend", ctypes.byref(args), ctypes.byref(b.args), q.addr, q.sb, q.sr, out.addr + guard, rows * hd, hd, heads, 0,
           scratch.addr, need.value)
    rt.wait()
  for s, size in ((store, pool.storage.nbytes), (out, n)):
    got = bytes(rt.download(s.addr, s.nbytes))
    assert got[:guard] == b"\xa5" * guard and got[guard + size:] == b"\xa5" * (len(got) - guard - size)


def numpy_step(L, ids, w, c, caches, plan, places):
  """Logits of every row as paged_forward gives them, over NumPy pages of 4 bits."""
  tables, starts, lengths = plan
  x = w["embed"][ids].astype(np.float32)
  nh = c.heads + 2 * c.kv
  rot = [L.split(w[t][np.maximum(places, 0)], nh) for t in ("cos", "sin")]
  for l in range(c.layers):
    p = L.block(w, l)
    heads = L.rope(L.split(L.rms(x, p["input_layernorm"], c.eps) @ p["qkv_proj"], nh), *rot, w["turn"])
    P.put4(caches[l], tables, starts, lengths, B.bf16(heads[c.heads:]))
    o, _ = P.attend(heads[:c.heads], caches[l], tables, starts, lengths)
    x = x + L.merge(o) @ p["o_proj"]
    x = x + L.mlp(L.rms(x, p["post_attention_layernorm"], c.eps), p)
  return L.rms(x, w["norm"], c.eps) @ w["embed.T"]


@pytest.mark.parametrize("page, spare", [(16, 3), (64, 0)])
def test_paged_llama_matches_numpy(rt, page, spare):
  # prompts of three requests in one step, then tokens and drafts, some given up, over pages of 4 bits: every row's logits within
  # 3% of the largest (test_models.py:849), as for the other caches
  from baretile_amd.models import llama
  from oracle import llama_ref as L
  rng = np.random.default_rng(41)
  c, w = L.smol(rng, 2, vocab=256, places=96)
  dc = llama.model(dim=576, heads=9, kv=3, layers=2, eps=1e-5, theta=10000.0, vocab=256, ffn=1536)
  dw = llama.upload(rt, {k: v for k, v in w.items() if k not in ("cos", "sin", "turn", "embed.T")}, dc, places=96)
  pages, width = 24, 96 // page
  caches = llama.paged_cache(rt, dc, pages, page, bits=4)
  values = [np.zeros((pages, 6, page, 64)) for _ in range(2)]
  tables, cached, taken, free = np.full((3, width), -1), np.zeros(3, int), 0, rng.permutation(pages)
  for new, kept in (([20, 7, 33], [20, 7, 33]), ([1, 4, 3], [1, 2, 3]), ([5, 3, 0], [1, 3, 0]), ([1, 1, 1], [1, 1, 1])):
    rows = sum(new) + spare
    ids = rng.integers(0, 256, rows)
    b, (tables, starts, lengths, places, _, taken) = planned(rt, caches[0], tables, cached, new, free, rows, taken)
    got = np.array(llama.paged_forward(row(rt, ids), b, dw, dc, caches).tolist()).reshape(rows, -1)[:starts[-1]]
    want = numpy_step(L, ids, w, c, values, (tables, starts, lengths), places)[:starts[-1]]
    assert np.abs(got - want).max() <= 0.03 * np.abs(want).max(), np.abs(got - want).max() / np.abs(want).max()
    cached = cached + kept


def test_refusals(rt):
  pool = pool4(rt, 10, 2, 64, 16)
  tables, r = Tensor.of(rt, np.full((2, 4), -1), "int32"), lambda *v: row(rt, v)
  b = pool.plan(tables, r(0, 0), r(1, 1), r(*range(10)), 4)
  x, q = Tensor.zeros(rt, 4, 64, 4), Tensor.zeros(rt, 4, 64, 8)
  for bad in (dict(page=24), dict(head=32), dict(kv=0), dict(pages=0), dict(pages=1 << 28), dict(bits=3)):
    with pytest.raises(ValueError): Pages(rt, **(dict(pages=10, kv=2, head=64, page=16, bits=4) | bad))
  for bad in (Tensor.zeros(rt, 4, 64, 2), Tensor.zeros(rt, 3, 64, 4), Tensor.zeros(rt, 4, 128, 4), Tensor.zeros(rt, 4, 64, 4, "fp32"), None):
    with pytest.raises(ValueError, match="put needs"): pool.put(b, bad)
  for bad in (Tensor.zeros(rt, 4, 64, 7), Tensor.zeros(rt, 3, 64, 8), Tensor.zeros(rt, 4, 64, 8, "fp32"), None):
    with pytest.raises(ValueError, match="attend needs"): pool.attend(bad, b)
  with pytest.raises(ValueError, match="window"): pool.attend(q, b, -1)
  other = pool4(rt, 10, 2, 64, 32)
  for f in (lambda: other.put(b, x), lambda: other.attend(q, b), lambda: pool.put(None, x)):
    with pytest.raises(ValueError, match="batch must be planned"): f()
  args, need = (ctypes.byref(pool.args), ctypes.byref(b.args)), ctypes.c_uint64()
  for name, rest in (("pages4_put", (0, 0, 64)), ("pages4_put", (x.addr + 2, x.sb, x.sr)), ("pages4_put", (x.addr, x.sb, 60)),
                     ("pages4_attend", (0, 0, 64, q.addr, q.sb, q.sr, 8, 0, 0, 0)), ("pages4_attend", (q.addr, q.sb, q.sr, q.addr + 2, q.sb, q.sr, 8, 0, 0, 0))):
    with pytest.raises(ValueError): rt.run("refused", name, *args, *rest)
  with pytest.raises(ValueError): rt.run("refused", "pages4_read", args[0], 0)
  none = _lib.PagesArgs(0, 0, 10, 16, 2, 64)
  with pytest.raises(ValueError, match="values"): rt.run("refused", "pages4_put", ctypes.byref(none), args[1], x.addr, x.sb, x.sr)


@pytest.mark.parametrize("hd, page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("new", [[15, 17], [28, 4]])
def test_tiles_of_4_waves_whose_keys_are_cut(rt, hd, page, new):
  # a tile of pairs and a block for each request, times 8 heads and 32 pieces of the keys
  attended(rt, np.random.default_rng(24), 32, 8, hd, page, [16400, 40], new)


def test_parts_of_4_and_of_8_waves(rt):
  # on both sides of the lengths from which a part is a block of 8 waves, by the most parts there can be
  for i, (heads, kv, hd, page, length, requests) in enumerate([(2, 1, 128, 64, 65535 - 64, 1), (2, 1, 128, 64, 65536, 1), (2, 1, 128, 256, 65530, 5),
                                                               (2, 1, 128, 128, 81920, 5), (4, 1, 64, 64, 16383 - 64, 2), (4, 1, 64, 64, 16384, 2)]):
    attended(rt, np.random.default_rng(30 + i), heads, kv, hd, page, [length] + [9] * (requests - 1), [1] * requests, most=1)
