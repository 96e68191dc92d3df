"""The paged 8-bit cache and the verification of drafts on the GPU, against oracle/pages.py in 64 bits: plans, puts and tokens
exactly, attention within what its roundings allow. Needs a GPU."""
import ctypes
import numpy as np
import pytest

from baretile_amd import _lib
from baretile_amd.models import serve
from baretile_amd.pages import Pages
from baretile_amd.tensor import Recording, Storage, Tensor, jit
from oracle import bfp as B, pages as P

pytestmark = pytest.mark.gpu


def row(rt, a): return Tensor.of(rt, [[int(v) for v in a]], "int32")


def ints(t): return np.array(t.tolist()).reshape(t.shape[-2:]).squeeze(0) if t.rows == 1 else np.array(t.tolist())


def planned(rt, pool, tables, cached, new, free, rows, taken=None, most=None):
  """A plan made on the device and checked against the oracle's: (batch, the oracle's results)."""
  t = Tensor.of(rt, np.asarray(tables), "int32")
  b = pool.plan(t, row(rt, cached), row(rt, new), row(rt, free), rows, row(rt, [taken]) if taken is not None else None, most)
  want = P.plan(tables, cached, new, free, rows, pool.page, pool.pages, taken or 0, most)
  got = [ints(t).reshape(np.shape(tables)), *(ints(v) for v in (b.starts, b.lengths, b.places, b.slots)), int(ints(b.taken)[0])]
  for g, w, name in zip(got, want, ("tables", "starts", "lengths", "places", "slots", "taken")):
    assert np.array_equal(g, w), (name, g, w)
  return b, want


def bf16_rows(rng, *shape):
  x = rng.normal(0, 1, shape) * np.exp(rng.normal(0, 0.7, (*shape[:-1], 1)))
  return B.bf16(x)


# ---- plans

@pytest.mark.parametrize("requests, page, most, rows", [(1, 16, None, 1), (1, 64, None, 40), (5, 16, None, 33), (7, 32, 3, 50), (64, 64, None, 64),
                                                        (65, 16, 2, 300), (300, 128, None, 900), (1100, 16, 4, 2048), (2048, 16, None, 4100),
                                                        (3, 256, None, 2500)])
def test_plan(rt, requests, page, most, rows):
  rng = np.random.default_rng(requests + rows)
  pool = Pages(rt, 5000, 1, 64, page)
  width = 12
  cached, new = rng.integers(0, page * 6, requests), rng.integers(0, max(2, 2 * rows // requests), requests)
  free = rng.permutation(5000)
  # every request's pages for what it has cached, some with a spare page behind, some with a hole
  tables, at = np.full((requests, width), -1), 0
  for r in range(requests):
    n = min(-(-int(cached[r]) // page) + int(rng.integers(0, 3) == 0), width)
    tables[r, :n] = rng.integers(0, 5000, n)
    if n and rng.integers(0, 5) == 0: tables[r, rng.integers(0, n)] = rng.choice([-1, 5000, 2 ** 31 - 1, -2 ** 31])
  planned(rt, pool, tables, cached, new, free, rows, most=most)
  planned(rt, pool, tables, cached, new, free[:3], rows, taken=2, most=most)  # the free list runs out


def test_plan_with_odd_lengths(rt):
  pool = Pages(rt, 20, 1, 64, 16)
  none = np.full((4, 3), -1)
  free = np.arange(20)
  planned(rt, pool, none, [0, 0, 0, 0], [0, 0, 0, 0], free, 5)  # nothing to do
  planned(rt, pool, none, [-5, 0, 2 ** 31 - 1, 48], [3, -2, 4, 1], free, 20)  # below 0, and past the tables' width
  planned(rt, pool, none, [0, 0, 0, 0], [2 ** 31 - 1] * 4, free, 40)  # more than the rows
  planned(rt, pool, none, [0, 15, 16, 17], [1, 1, 1, 1], [99, -1, 3, 20], 4)  # free pages that are none
  planned(rt, pool, none, [0, 0, 0, 0], [5, 5, 5, 5], free, 20, taken=-3)
  planned(rt, pool, none, [0, 0, 0, 0], [40, 1, 1, 1], free, 20, taken=19)


def test_plan_leaves_refused_drafts_their_pages(rt):
  pool = Pages(rt, 20, 1, 64, 16)
  b, want = planned(rt, pool, np.full((2, 4), -1), [0, 0], [30, 20], np.arange(20), 50)
  assert want[5] == 4
  planned(rt, pool, want[0], [14, 20], [5, 5], np.arange(20), 10, taken=4)  # the first request's second page is its own still


# ---- puts

def whole(pool): return np.array(pool.values().tolist()).reshape(pool.pages, 2 * pool.kv, pool.page, pool.head)


def scales(pool): return np.array(pool.scales.tolist())


@pytest.mark.parametrize("hd, kv, page", [(64, 1, 16), (128, 2, 32), (64, 3, 64), (128, 1, 128), (128, 2, 256), (64, 2, 256)])
def test_put(rt, hd, kv, page):
  rng = np.random.default_rng(hd + kv + page)
  pool = Pages(rt, 24, kv, hd, page)
  values, s = np.zeros((24, 2 * kv, page, hd)), np.full((24, 2 * kv), 2.0 ** -100)
  tables, lengths, taken = np.full((5, 6), -1), np.zeros(5, int), 0
  free = rng.permutation(24)
  for step, new in enumerate(([page + 3, 1, 0, 2 * page, 5], [1, 1, 1, 1, 1], [0, page - 1, 2, 1, 7], [1, 2, 0, 17, 3], [3, 1, 4, 1, 1])):
    rows = sum(new) + 2
    x = bf16_rows(rng, 2 * kv, rows, hd) * 4.0 ** (step % 3)  # later rows larger, then smaller: scales that grow and stay
    b, (tables, starts, lengths, _, _, taken) = planned(rt, pool, tables, lengths, new, free, rows, taken)
    pool.put(b, Tensor.of(rt, x))
    P.put(values, s, tables, starts, lengths, x)
    assert np.array_equal(whole(pool), values), step
    assert np.array_equal(scales(pool), s), step
  assert (values != 0).any(axis=(1, 2, 3)).sum() == taken  # pages of no request stay as they were


def test_put_of_odd_values(rt):
  pool = Pages(rt, 3, 1, 64, 16)
  x = np.zeros((2, 20, 64))
  x[0, 0, :8] = [np.inf, -np.inf, np.nan, 3.0, -1e-3, 448, -449, 1e-30]  # infinities and NaNs don't count for the scale
  x[1, 1, 0], x[1, 2, 0], x[1, 3, :2] = 3e38, 1e-38, [np.nan, -np.inf]
  x[0, 16] = B.bf16(2.0 ** -133 * np.arange(64))  # smaller than any scale's grid
  x[1, 17, :4] = [np.inf, np.inf, np.nan, 0]  # nothing finite but zeros
  bits = (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)
  x = (bits.astype(np.uint32) << 16).view(np.float32)
  b, (tables, starts, lengths, *_) = planned(rt, pool, np.full((1, 2), -1), [0], [20], np.arange(3), 20)
  values, s = np.zeros((3, 2, 16, 64)), np.full((3, 2), 2.0 ** -100)
  pool.put(b, Tensor.frombytes(rt, 20, 64, bits.tobytes(), 2))
  P.put(values, s, tables, starts, lengths, x)
  assert np.array_equal(whole(pool), values) and np.array_equal(scales(pool), s)


def test_put_a_token_at_a_time(rt):
  rng = np.random.default_rng(3)
  pool = Pages(rt, 4, 2, 128, 32)
  values, s = np.zeros((4, 4, 32, 128)), np.full((4, 4), 2.0 ** -100)
  tables = np.full((1, 4), -1)
  x = bf16_rows(rng, 4, 70, 128) * np.exp(rng.normal(0, 2, (1, 70, 1)))  # sizes all over: scales that grow often
  x = B.bf16(x)
  taken = 0
  for i in range(70):
    b, (tables, starts, lengths, _, _, taken) = planned(rt, pool, tables, [i], [1], [2, 0, 3, 1], 1, taken)
    pool.put(b, Tensor.of(rt, x[:, i:i + 1]))
    P.put(values, s, tables, starts, lengths, x[:, i:i + 1])
  assert np.array_equal(whole(pool), values) and np.array_equal(scales(pool), s)


def test_put_drops_rows_without_a_page_and_takes_strided_rows(rt):
  rng = np.random.default_rng(4)
  pool = Pages(rt, 5, 1, 64, 16)
  tables = np.array([[2, -1, 7], [0, 1, -1]])
  cached, new = [10, 20], [30, 20]
  x = bf16_rows(rng, 2, 60, 192)  # wider rows, of which the middle is put
  b, (made, starts, lengths, *_) = planned(rt, pool, tables, cached, new, [9, 4], 60)
  values, s = np.zeros((5, 2, 16, 64)), np.full((5, 2), 2.0 ** -100)
  pool.put(b, Tensor.of(rt, x)[:, :, 64:128])
  P.put(values, s, made, starts, lengths, x[:, :, 64:128])
  assert np.array_equal(whole(pool), values) and np.array_equal(scales(pool), s)


# ---- attention

def bound(q, values, weighed, out):
  """How far an output may be from the oracle's: the weights' rounding to bf16 (2^-8 of the weighed |v|), the output's, and the fp32
  scores' (4 roundings of a sum of hd products, doubled for the weights' sum)."""
  size = np.linalg.norm(q, axis=-1).max() * np.linalg.norm(values, axis=-1).max()
  return weighed * (2.0 ** -8 + 8 * q.shape[-1] * 2.0 ** -24 * (1 + size)) + 2.0 ** -8 * np.abs(out) + 1e-30


def filled(rt, rng, heads, kv, hd, page, lengths, width=None, spare=3):
  """A pool with rows of every request in it, (pool, values, tables)."""
  width = width or max(1, -(-max(lengths) // page))
  pages = sum(-(-n // page) for n in lengths) + spare
  pool = Pages(rt, pages, kv, hd, page)
  values, s = np.zeros((pages, 2 * kv, page, hd)), np.full((pages, 2 * kv), 2.0 ** -100)
  rows = max(1, sum(lengths))
  x = bf16_rows(rng, 2 * kv, rows, hd)
  b, (tables, starts, _, _, _, taken) = planned(rt, pool, np.full((len(lengths), width), -1), [0] * len(lengths), lengths, rng.permutation(pages), rows)
  pool.put(b, Tensor.of(rt, x))
  P.put(values, s, tables, starts, lengths, x)
  return pool, values, tables, taken


def attended(rt, rng, heads, kv, hd, page, lengths, new, window=0, spare=0, tables=None, merged=False, most=None):
  pool, values, made, taken = filled(rt, rng, heads, kv, hd, page, lengths)
  if tables is not None: made = tables(made)
  rows = sum(new) + spare
  q = B.bf16(rng.normal(0, 1, (heads, rows, hd)) * 1.5 / np.sqrt(hd))
  b, (made, starts, total, *_) = planned(rt, pool, made, [n - m for n, m in zip(lengths, new)], new, [-1], rows, most=most)
  out = pool.attend(Tensor.of(rt, q), b, window, merged)
  got = np.array(out.tolist())
  if merged: got = got.reshape(rows, heads, hd).transpose(1, 0, 2)
  got = got.reshape(heads, rows, hd)
  want, weighed = P.attend(q, values, made, starts, total, window)
  assert np.all(np.abs(got - want) <= bound(q, values, weighed, want)), np.abs(got - want).max()
  return got, want


@pytest.mark.parametrize("heads, kv, hd, page", [(8, 2, 64, 16), (4, 4, 128, 32), (32, 8, 128, 64), (9, 3, 64, 128), (7, 1, 128, 256), (20, 1, 64, 16)])
@pytest.mark.parametrize("lengths, new", [([1], [1]), ([300], [1]), ([64, 0, 1, 65, 500], [1, 0, 1, 1, 1]), ([700, 63, 129], [5, 3, 0]),
                                          ([200, 90], [9, 7])])
def test_attend_few_rows(rt, heads, kv, hd, page, lengths, new):
  attended(rt, np.random.default_rng(heads + page + sum(lengths)), heads, kv, hd, page, lengths, new, spare=2, merged=page == 64)


@pytest.mark.parametrize("heads, kv, hd, page", [(8, 2, 64, 16), (4, 1, 128, 64), (6, 2, 128, 32), (3, 3, 64, 256)])
@pytest.mark.parametrize("lengths, new", [([130], [130]), ([333, 1, 200], [140, 1, 90]), ([520, 64], [71, 64])])
def test_attend_many_rows(rt, heads, kv, hd, page, lengths, new):
  attended(rt, np.random.default_rng(heads + page + sum(lengths)), heads, kv, hd, page, lengths, new, spare=17)


@pytest.mark.parametrize("new", [[1, 1, 0], [2, 1, 40]])
def test_attend_many_heads_to_one(rt, new):
  attended(rt, np.random.default_rng(12), 130, 1, 64, 32, [700, 90, 50], new)  # a token's pairs pass a tile


@pytest.mark.parametrize("requests", [64, 65, 300, 2048])
def test_many_requests(rt, requests):
  # some without rows or tokens; decoding steps, drafts and a prompt among them
  rng = np.random.default_rng(requests)
  lengths = rng.integers(0, 40, requests)
  new = np.minimum(lengths, rng.choice([0, 1, 3], requests))
  attended(rt, rng, 4, 2, 64, 16, lengths.tolist(), new.tolist(), spare=3, most=3)
  lengths[requests // 2], new[requests // 2] = 100, 50
  attended(rt, rng, 4, 2, 64, 16, lengths.tolist(), new.tolist())


@pytest.mark.parametrize("window", [1, 7, 64, 100, 1000])
@pytest.mark.parametrize("lengths, new", [([300, 40], [1, 3]), ([400, 150], [100, 70])])
def test_attend_window(rt, window, lengths, new):
  attended(rt, np.random.default_rng(window), 8, 2, 64, 16, lengths, new, window)


@pytest.mark.parametrize("window", [1, 40, 1000, 1019, 1020, 1100])
@pytest.mark.parametrize("new", [[1, 1, 5], [4, 0, 1], [3, 1, 70]])
def test_attend_window_over_long_tables(rt, window, new):
  # windows that leave a part's keys of tables that hold many more, and one key too many for that
  attended(rt, np.random.default_rng(window), 8, 2, 64, 32, [5000, 90, 2001], new, window, most=max(new))


@pytest.mark.parametrize("hd, page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("lengths, window", [([1024, 3], 0), ([5000, 300], 954), ([5000, 300], 955)])
def test_attend_prompts_keys_in_splits_and_one_part(rt, hd, page, lengths, window):
  # 1024 keys to see: a prompt's are cut in two, and joined, while the other request's are one part; of one more both join
  attended(rt, np.random.default_rng(hd + window), 4, 2, hd, page, lengths, [70, 3], window, most=70)


@pytest.mark.parametrize("new", [[1, 3, 1], [90, 80, 1]])
def test_attend_hides_pages_that_are_none(rt, new):
  def holes(t):
    t = t.copy()
    t[0, 1], t[0, 4], t[1, 0], t[2, :] = -1, 10 ** 6, -2 ** 31, -1
    return t
  got, want = attended(rt, np.random.default_rng(5), 8, 2, 64, 16, [200, 120, 30], new, tables=holes)
  assert not want[:, -1].any()  # a request with no page at all: its row sees nothing


def test_attend_long(rt):
  attended(rt, np.random.default_rng(6), 4, 1, 64, 64, [40000, 100], [1, 2])


@pytest.mark.parametrize("new", [[40, 2], [17, 30]])
def test_attend_long_behind_a_prompt(rt, new):
  attended(rt, np.random.default_rng(11), 4, 1, 64, 64, [40000, 100], new)  # keys cut into as many splits as there are


@pytest.mark.parametrize("hd, page", [(64, 16), (128, 64), (128, 256)])
@pytest.mark.parametrize("lengths", [[1024, 3], [1025, 1024], [1008, 961]])
@pytest.mark.parametrize("new", [[1, 1], [6, 2]])
def test_attend_at_a_short_tables_end(rt, hd, page, lengths, new):
  # tables of 1024 keys are one part a request; of one page more, several and a join
  attended(rt, np.random.default_rng(hd + page), 8, 2, hd, page, lengths, new, spare=1)


@pytest.mark.parametrize("hd, page, window", [(64, 16, 0), (128, 32, 0), (64, 16, 1500), (128, 128, 700), (64, 256, 0)])
@pytest.mark.parametrize("new", [[1, 2], [4, 70]])
def test_attend_past_a_wave_of_pages(rt, hd, page, window, new):
  # over 64 pages of 16 or 32 tokens, which a wave's lanes hold at a time, and prompts whose keys are cut into splits
  attended(rt, np.random.default_rng(hd + page), 4, 2, hd, page, [3100, 2500], new, window, spare=5)


def test_attend_a_row_that_is_not_a_number(rt):
  rng = np.random.default_rng(7)
  for new in ([2, 2], [40, 40]):
    pool, values, tables, _ = filled(rt, rng, 4, 2, 64, 16, [300, 90])
    rows = sum(new)
    q = B.bf16(rng.normal(0, 0.2, (4, rows, 64)))
    bits = B.bf16_bits(q)
    bits[1, 1, 3], bits[2, new[0], 0] = 0x7FC0, 0x7F80  # one row's head with a NaN, one with an infinity
    b, (tables, starts, total, *_) = planned(rt, pool, tables, [300 - new[0], 90 - new[1]], new, [-1], rows)
    got = np.array(pool.attend(Tensor.frombytes(rt, rows, 64, bits.tobytes(), 4), b).tolist())
    want, weighed = P.attend(q, values, tables, starts, total)
    ok = np.ones((4, rows), bool)
    ok[1, 1] = ok[2, new[0]] = False
    assert np.isnan(got[~ok]).all()
    assert np.all(np.abs(got - want)[ok] <= bound(q, values, weighed, want)[ok])


def test_attend_takes_strided_queries_and_masks_what_a_page_held_before(rt):
  rng = np.random.default_rng(8)
  pool, values, tables, _ = filled(rt, rng, 8, 2, 64, 16, [100])
  # the request ends; another takes its last page and half fills it: the rows behind it are the old request's
  page = int(tables[0, 6])
  b, (t, starts, total, *_) = planned(rt, pool, np.full((1, 1), -1), [0], [5], [page], 5)
  x = bf16_rows(rng, 4, 5, 64)
  pool.put(b, Tensor.of(rt, x))
  s = scales(pool)
  values[page] = 0
  P.put(values, s, t, starts, total, x)
  q = B.bf16(rng.normal(0, 0.2, (5, 8 * 64)))
  got = np.array(pool.attend(Tensor.of(rt, q).split(8), b).tolist())
  q = q.reshape(5, 8, 64).transpose(1, 0, 2)
  want, weighed = P.attend(q, values, t, starts, total)
  assert np.all(np.abs(got - want) <= bound(q, values, weighed, want))


def test_attend_repeats_itself(rt):
  rng = np.random.default_rng(9)
  pool, _, tables, _ = filled(rt, rng, 8, 2, 128, 64, [3000, 50, 900])
  q = Tensor.of(rt, B.bf16(rng.normal(0, 0.2, (8, 12, 128))))
  b, _ = planned(rt, pool, tables, [2996, 46, 896], [4, 4, 4], [-1], 12)
  first = pool.attend(q, b).tobytes()
  for _ in range(5): assert pool.attend(q, b).tobytes() == first


# ---- verification

def verified(rt, logits, ids, starts, uniforms, probs=None, t=None):
  of = lambda a: Tensor.of(rt, np.asarray(a, np.float32), "fp32")
  tokens, counts = serve.verify(of(logits), row(rt, ids), row(rt, starts), of(uniforms), of(probs) if probs is not None else None,
                                of(np.reshape(t, (-1, 1))) if t is not None else None)
  as32 = lambda a: np.asarray(a, np.float32)
  want = P.verify(as32(logits), ids, starts, as32(uniforms), None if probs is None else as32(probs), None if t is None else as32(t))
  got = ints(tokens), ints(counts)
  assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (got, want)
  return got


def soft(x): return np.exp(x - x.max(-1, keepdims=True)) / np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)


def near(rng, logits):  # draft probabilities near the row before's
  return soft(np.roll(logits, 1, 0) + 0.7 * rng.normal(0, 1, logits.shape)).astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 2048, 2049, 49152, 131072, 200001])
@pytest.mark.parametrize("drawn", [True, False])
def test_verify(rt, vocab, drawn):
  rng = np.random.default_rng(vocab)
  starts = [0, 5, 5, 6, 14]
  rows = 16
  logits = 3 * rng.normal(0, 1, (rows, vocab)).astype(np.float32)
  probs = near(rng, logits)
  ids = [int(np.searchsorted(np.cumsum(p.astype(np.float64)), rng.random() * 0.999)) for p in probs] if drawn else np.roll(logits, 1, 0).argmax(1)
  for _ in range(3):
    verified(rt, logits, np.minimum(ids, vocab - 1), starts, rng.random((2, rows)).astype(np.float32), probs if drawn else None,
             rng.uniform(0.5, 2, rows).astype(np.float32))


def test_verify_many_requests(rt):
  rng = np.random.default_rng(1)
  starts = np.concatenate([[0], np.cumsum(rng.integers(0, 5, 150))])
  rows = int(starts[-1]) + 3
  logits = 2 * rng.normal(0, 1, (rows, 3001)).astype(np.float32)
  probs = near(rng, logits)
  ids = [int(rng.choice(3001, p=p.astype(np.float64) / p.sum(dtype=np.float64))) for p in probs]
  verified(rt, logits, ids, starts, rng.random((2, rows)).astype(np.float32), probs)


def test_verify_draws_from_all_of_the_distribution(rt):
  # one request a uniform, over a grid of them: the drawn tokens' counts are the distribution's, to the grid's step
  n = 1 << 11
  p = np.array([0.5, 0.0, 0.25, 0.125, 0.125])
  logits = np.tile(np.where(p > 0, np.log(np.maximum(p, 1e-9)), -np.inf), (n, 1))
  u = np.stack([np.zeros(n), (np.arange(n) + 0.5) / n])
  tokens, _ = verified(rt, logits, [0] * n, range(n + 1), u)
  assert np.array_equal(np.bincount(tokens, minlength=5), p * n)


def test_verify_at_its_edges(rt):
  rng = np.random.default_rng(2)
  inf, nan = np.inf, np.nan
  low = np.finfo(np.float32).min
  v = 300
  logits = rng.normal(0, 1, (24, v)).astype(np.float32)
  logits[0], logits[1], logits[2] = -inf, low, nan  # nothing; everything alike; nothing
  logits[3, 7], logits[4, [3, 9]] = inf, inf
  logits[5, 100:], logits[6, :] = -inf, -inf
  logits[6, 250] = -1e30  # one token left
  logits[7, 5] = nan
  for u0 in (0.0, 0.5, 1 - 2.0 ** -24):
    for u1 in (0.0, 0.5, 1 - 2.0 ** -24):
      u = np.array([[u0] * 24, [u1] * 24], np.float32)
      verified(rt, logits, [7] * 24, range(25), u)  # every row on its own
      verified(rt, logits, [7] * 24, range(0, 25, 2), u)  # drafts against odd rows
      verified(rt, logits, [7] * 24, range(0, 25, 3), u, soft(rng.normal(0, 1, (24, v))))
  ids = [0, -1, v, 2 ** 31 - 1, -2 ** 31, 5] * 4  # drafts that are no tokens
  verified(rt, logits, ids, [0, 12, 24], rng.random((2, 24)), soft(rng.normal(0, 1, (24, v))))
  # inverse temperatures: 0 takes any token with a weight, infinity the largest, the first of equals; below 0 and NaN are 0
  logits[10, 20], logits[10, 30] = 50, 50
  verified(rt, logits, logits.argmax(1), [0, 12, 24], rng.random((2, 24)), None, [0, inf, 1, -1, nan, inf, 0, 1e30, inf, 1e-30, inf, 3] * 2)
  # the same distribution on both sides: refused by rounding or not at all, something is drawn
  q = np.roll(soft(logits[12:].astype(np.float64)), 1, 0)
  verified(rt, logits[12:], [9] * 12, [0, 12], np.full((2, 12), 1 - 2.0 ** -24), q)


def test_verify_reads_starts_within_its_rows(rt):
  logits = Tensor.of(rt, np.zeros((4, 10)), "fp32")
  u = Tensor.of(rt, np.full((2, 4), 0.55), "fp32")
  for starts in ([0, 9], [-5, 2], [3, 1], [2 ** 31 - 1, -2 ** 31]):
    tokens, counts = serve.verify(logits, row(rt, [1, 2, 3, 4]), row(rt, starts), u)
    assert len(ints(tokens)) == 4 and len(ints(counts)) == 1  # (starts that no plan makes: any tokens, but nothing outside)


def test_a_batch_reads_starts_within_its_rows(rt):
  rng = np.random.default_rng(13)
  pool, values, tables, _ = filled(rt, rng, 4, 2, 64, 16, [30, 50])
  b, _ = planned(rt, pool, tables, [20, 10], [10, 40], [-1], 50)
  x, q = Tensor.of(rt, bf16_rows(rng, 4, 50, 64)), Tensor.of(rt, B.bf16(rng.normal(0, 0.2, (4, 50, 64))))
  for starts in ([0, 10, 9000], [-5, 20, 30], [40, 3, 50], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]):
    b.starts.assign(row(rt, starts))  # (starts that no plan makes: any rows, but nothing outside)
    pool.put(b, x)
    assert np.array(pool.attend(q, b).tolist()).shape == (4, 50, 64)


# ---- together

def test_a_recorded_step_follows_its_lengths(rt):
  # plan, put, attention and verification recorded once; each replay takes the lengths, rows and numbers of its own
  rng = np.random.default_rng(10)
  heads, kv, hd, page, R, rows, vocab = 8, 2, 64, 16, 3, 9, 500
  pool = Pages(rt, 40, kv, hd, page)
  free = rng.permutation(40)
  tables, fr = Tensor.of(rt, np.full((R, 10), -1), "int32"), row(rt, free)
  cached, new, taken = row(rt, [0] * R), row(rt, [0] * R), row(rt, [0])
  x, q = Tensor.zeros(rt, rows, hd, 2 * kv), Tensor.zeros(rt, rows, hd, heads)
  logits, ids, u = Tensor.zeros(rt, rows, vocab, dtype="fp32"), row(rt, [0] * rows), Tensor.zeros(rt, 2, rows, dtype="fp32")
  def step():
    b = pool.plan(tables, cached, new, fr, rows, taken, most=4)
    pool.put(b, x)
    o = pool.attend(q, b)
    tokens, counts = serve.verify(logits, ids, b.starts, u)
    taken.assign(b.taken)
    cached.assign(b.lengths - 0)
    return b, o, tokens, counts
  step()
  rt.wait()
  for t, v in ((tables, np.full((R, 10), -1)), (cached, [[0] * R]), (taken, [[0]])): t.assign(Tensor.of(rt, np.array(v), "int32"))
  rec = Recording(rt)
  with rec: out = step()
  values, s = np.zeros((40, 2 * kv, page, hd)), np.full((40, 2 * kv), 2.0 ** -100)
  want_tables, want_cached, want_taken = np.full((R, 10), -1), np.zeros(R, int), 0
  for i in range(8):
    n = rng.integers(0, 6, R)  # some past `most`
    xs, qs = bf16_rows(rng, 2 * kv, rows, hd) * 2.0 ** i, B.bf16(rng.normal(0, 0.2 / 2.0 ** i, (heads, rows, hd)))
    ls, ds, us = rng.normal(0, 2, (rows, vocab)).astype(np.float32), rng.integers(0, vocab, rows), rng.random((2, rows)).astype(np.float32)
    new.assign(row(rt, n))
    x.assign(Tensor.of(rt, xs))
    q.assign(Tensor.of(rt, qs))
    logits.assign(Tensor.of(rt, ls, "fp32"))
    ids.assign(row(rt, ds))
    u.assign(Tensor.of(rt, us, "fp32"))
    rec.send()
    rt.wait()
    want_tables, starts, total, places, slots, want_taken = P.plan(want_tables, want_cached, n, free, rows, page, 40, want_taken, 4)
    P.put(values, s, want_tables, starts, total, xs)
    want, weighed = P.attend(qs, values, want_tables, starts, total)
    b, o, tokens, counts = out
    assert np.array_equal(np.array(tables.tolist()), want_tables) and np.array_equal(ints(b.slots), slots)
    assert np.array_equal(whole(pool), values)
    assert np.all(np.abs(np.array(o.tolist()) - want) <= bound(qs, values, weighed, want)), i
    vt, vc = P.verify(ls, ds, starts, us)
    assert np.array_equal(ints(tokens), vt) and np.array_equal(ints(counts), vc)
    want_cached = total


def test_a_jit_step_takes_its_tables_and_rows(rt):
  # plan, put and attention under jit: its inputs are copied in, and the tables that the plan fills come back
  rng = np.random.default_rng(14)
  pool = Pages(rt, 12, 2, 64, 16)
  free = rng.permutation(12)
  fr = row(rt, free)
  def step(tables, cached, new, taken, x, q):
    b = pool.plan(tables, cached, new, fr, 30, taken)
    pool.put(b, x)
    return pool.attend(q, b)
  f = jit(step)
  values, s = np.zeros((12, 4, 16, 64)), np.full((12, 4), 2.0 ** -100)
  tables, want_tables, cached, used = Tensor.of(rt, np.full((2, 6), -1), "int32"), np.full((2, 6), -1), np.zeros(2, int), 0
  for new in ([20, 3], [1, 4], [0, 12], [5, 1]):
    x, q = bf16_rows(rng, 4, 30, 64), B.bf16(rng.normal(0, 0.2, (8, 30, 64)))
    got = np.array(f(tables, row(rt, cached), row(rt, new), row(rt, [used]), Tensor.of(rt, x), Tensor.of(rt, q)).tolist())
    want_tables, starts, total, _, _, used = P.plan(want_tables, cached, new, free, 30, 16, 12, used)
    P.put(values, s, want_tables, starts, total, x)
    want, weighed = P.attend(q, values, want_tables, starts, total)
    assert np.array_equal(np.array(tables.tolist()), want_tables) and np.array_equal(whole(pool), values)
    assert np.all(np.abs(got - want) <= bound(q, values, weighed, want))
    cached = total


def test_tables_and_rows_that_are_views(rt):
  rng = np.random.default_rng(15)
  pool = Pages(rt, 20, 2, 64, 16)
  all_tables = np.full((5, 9), 7)
  all_tables[1:4, 2:8] = -1
  t = Tensor.of(rt, all_tables, "int32")
  lengths, rows = [40, 0, 17], 60
  wide = Tensor.of(rt, np.stack([np.arange(20), rng.permutation(20)]), "int32")
  free = np.array(wide.tolist(), int)[1]
  x, q = bf16_rows(rng, 4, 2 * rows, 64), B.bf16(rng.normal(0, 0.2, (8, 2 * rows, 64)))
  b = pool.plan(t[1:4, 2:8], row(rt, [0, 0, 0]), row(rt, [9, *lengths, 9])[:, 1:4], wide[1:2, :], rows)
  want_tables, starts, total, *_ = P.plan(all_tables[1:4, 2:8], [0, 0, 0], lengths, free, rows, 16, 20)
  all_tables[1:4, 2:8] = want_tables
  assert np.array_equal(np.array(t.tolist()), all_tables)
  pool.put(b, Tensor.of(rt, x)[:, rows // 2:rows // 2 + rows, :])
  values, s = np.zeros((20, 4, 16, 64)), np.full((20, 4), 2.0 ** -100)
  P.put(values, s, want_tables, starts, total, x[:, rows // 2:rows // 2 + rows])
  assert np.array_equal(whole(pool), values)
  q = q[:, 5:5 + rows]
  got = np.array(pool.attend(Tensor.of(rt, np.concatenate([q[:, :3], q], 1))[:, 3:, :], b).tolist())
  want, weighed = P.attend(q, values, want_tables, starts, total)
  assert np.all(np.abs(got - want) <= bound(q, values, weighed, want))


def test_pages_past_32_bits(rt):
  # the last pages of a pool of 5 GB hold what the first of a small one do, bit for bit
  rng = np.random.default_rng(16)
  kv, hd, page, n = 2, 128, 256, 40000
  lengths = [700, 300]
  x, q = Tensor.of(rt, bf16_rows(rng, 2 * kv, 1000, hd)), Tensor.of(rt, B.bf16(rng.normal(0, 0.2, (8, 1000, hd))))
  outs = []
  for pages in (5, n):
    pool = Pages(rt, pages, kv, hd, page)
    b = pool.plan(Tensor.of(rt, np.full((2, 3), -1), "int32"), row(rt, [0, 0]), row(rt, lengths), row(rt, range(pages - 5, pages)), 1000)
    pool.put(b, x)
    step = pool.plan(b.tables, row(rt, [699, 298]), row(rt, [1, 2]), row(rt, [-1]), 3)
    outs.append([pool.attend(q, b).tobytes(), pool.attend(q[:, :3, :], step).tobytes(),
                 pool.values()[(pages - 5) * 2 * kv:, :, :].contiguous().tobytes()])
    del pool, b, step
  assert outs[0] == outs[1]


def test_a_long_cache(rt):
  # 300000 tokens, over 1172 pages that 19 loads of a wave's page table bring in
  attended(rt, np.random.default_rng(17), 4, 1, 64, 256, [300000, 5], [1, 1], most=1)
  attended(rt, np.random.default_rng(18), 4, 1, 64, 256, [300000, 5], [2, 1], window=100000)


def test_a_closed_runtime(chip):
  from baretile_amd.runtime import Runtime
  first = Runtime(chip)
  pool = Pages(first, 4, 2, 64, 16)
  b = pool.plan(Tensor.of(first, [[-1]], "int32"), row(first, [0]), row(first, [1]), row(first, [0]), 1)
  x, q = Tensor.zeros(first, 1, 64, 4), Tensor.zeros(first, 1, 64, 4)
  second = Runtime(chip)
  try:
    for f in (lambda: pool.put(b, x), lambda: pool.attend(q, b), pool.values, lambda: Pages(first, 4, 2, 64, 16)):
      with pytest.raises(RuntimeError): f()
    other = Pages(second, 4, 2, 64, 16)
    with pytest.raises(ValueError, match="batch must be planned"): other.put(b, Tensor.zeros(second, 1, 64, 4))
  finally: second.close()


def numpy_step(L, ids, w, c, caches, scales, plan, places):
  """Logits of every row as paged_forward gives them, over NumPy pages (caches, scales: one of each a block)."""
  tables, starts, lengths = plan
  x = w["embed"][ids].astype(np.float32)
  nh, hd = c.heads + 2 * c.kv, L.head(c)
  at = np.maximum(places, 0)
  rot = [L.split(w[t][at], nh) for t in ("cos", "sin")]
  for l in range(c.layers):
    p = L.block(w, l)
    heads = L.rope(L.split(L.rms(x, p["input_layernorm"], c.eps) @ p["qkv_proj"], nh), *rot, w["turn"])
    P.put(caches[l], scales[l], tables, starts, lengths, B.bf16(heads[c.heads:]))
    o, _ = P.attend(heads[:c.heads], caches[l], tables, starts, lengths)
    x = x + L.merge(o) @ p["o_proj"]
    x = x + L.mlp(L.rms(x, p["post_attention_layernorm"], c.eps), p)
  return L.rms(x, w["norm"], c.eps) @ w["embed.T"]


@pytest.mark.parametrize("page, spare", [(16, 3), (64, 0)])
def test_paged_llama_matches_numpy(rt, page, spare):
  # prompts of three requests in one step, then a token and drafts each, one request's drafts given up in between and its
  # places taken again, over pages: every row's logits within 3% of the largest (test_models.py:849), as for the other
  # caches, and the picks that serve.verify makes of them the oracle's
  from baretile_amd.models import llama
  from oracle import llama_ref as L
  rng = np.random.default_rng(41)
  c, w = L.smol(rng, 2, vocab=256, places=96)
  dc = llama.model(dim=576, heads=9, kv=3, layers=2, eps=1e-5, theta=10000.0, vocab=256, ffn=1536)
  dw = llama.upload(rt, {k: v for k, v in w.items() if k not in ("cos", "sin", "turn", "embed.T")}, dc, places=96)
  pages, width = 24, 96 // page
  caches = llama.paged_cache(rt, dc, pages, page)
  values, scales = ([np.zeros((pages, 6, page, 64)) for _ in range(2)], [np.full((pages, 6), 2.0 ** -100) for _ in range(2)])
  tables, cached, taken, free = np.full((3, width), -1), np.zeros(3, int), 0, rng.permutation(pages)
  for new, kept in (([20, 7, 33], [20, 7, 33]), ([1, 4, 3], [1, 2, 3]), ([5, 3, 0], [1, 3, 0]), ([1, 1, 1], [1, 1, 1])):
    rows = sum(new) + spare
    ids = rng.integers(0, 256, rows)
    b, (tables, starts, lengths, places, _, taken) = planned(rt, caches[0], tables, cached, new, free, rows, taken)
    logits = llama.paged_forward(row(rt, ids), b, dw, dc, caches).realize()
    got = np.array(logits.tolist()).reshape(rows, -1)[:starts[-1]]
    want = numpy_step(L, ids, w, c, values, scales, (tables, starts, lengths), places)[:starts[-1]]
    assert np.abs(got - want).max() <= 0.03 * np.abs(want).max(), np.abs(got - want).max()
    u = rng.random((2, rows)).astype(np.float32)
    tokens, counts = serve.verify(logits.reshape(rows, 256), row(rt, ids), b.starts, Tensor.of(rt, u, "fp32"))
    vt, vc = P.verify(np.array(logits.tolist(), np.float32).reshape(rows, -1), ids, starts, u)
    assert np.array_equal(ints(tokens), vt) and np.array_equal(ints(counts), vc)
    again, _ = serve.verify(llama.paged_forward(row(rt, ids), b, dw, dc, caches), row(rt, ids), b.starts, Tensor.of(rt, u, "fp32"))
    assert np.array_equal(ints(again), vt)  # the step again, its rows put over themselves, its logits taken as they come
    cached = cached + kept
  with pytest.raises(ValueError, match="paged_forward"): llama.paged_forward(row(rt, [1]), b, dw, dc, caches)
  with pytest.raises(ValueError, match="paged_forward"): llama.paged_forward(row(rt, [1] * rows), b, dw, dc, caches[:1])


def test_refusals(rt):
  pool = Pages(rt, 10, 2, 64, 16)
  tables, r = Tensor.of(rt, np.full((2, 4), -1), "int32"), lambda *v: row(rt, v)
  b = pool.plan(tables, r(0, 0), r(1, 1), r(*range(10)), 4)
  x, q = Tensor.zeros(rt, 4, 64, 4), Tensor.zeros(rt, 4, 64, 8)
  for bad in (dict(page=24), dict(head=32), dict(kv=0), dict(pages=0), dict(pages=1 << 28)):
    with pytest.raises(ValueError): Pages(rt, **(dict(pages=10, kv=2, head=64, page=16) | bad))
  for args in ((Tensor.zeros(rt, 2, 4), r(0, 0), r(1, 1), r(1), 4), (tables, r(0), r(1, 1), r(1), 4), (tables, r(0, 0), r(1, 1, 1), r(1), 4),
               (tables, r(0, 0), r(1, 1), tables, 4), (tables, r(0, 0), r(1, 1), r(1), 0), (tables, r(0, 0), r(1, 1), r(1), (1 << 20) + 1),
               (tables, r(0, 0), r(1, 1), r(1), 4, r(0, 0)), (tables, r(0, 0), r(1, 1), r(1), 4, None, 0), (tables.T, r(0, 0, 0, 0), r(1, 1, 1, 1), r(1), 4),
               ([[1]], r(0), r(1), r(1), 4), (Tensor.zeros(rt, 2049, 1, dtype="int32"), Tensor.zeros(rt, 1, 2049, dtype="int32"),
                                              Tensor.zeros(rt, 1, 2049, dtype="int32"), r(1), 4)):
    with pytest.raises(ValueError): pool.plan(*args)
  for bad in (Tensor.zeros(rt, 4, 64, 2), Tensor.zeros(rt, 3, 64, 4), Tensor.zeros(rt, 4, 128, 4), Tensor.zeros(rt, 4, 64, 4, "fp32"), None):
    with pytest.raises(ValueError, match="put needs"): pool.put(b, bad)
  for bad in (Tensor.zeros(rt, 4, 64, 7), Tensor.zeros(rt, 3, 64, 8), Tensor.zeros(rt, 4, 64, 8, "fp32"), None):
    with pytest.raises(ValueError, match="attend needs"): pool.attend(bad, b)
  with pytest.raises(ValueError, match="window"): pool.attend(q, b, -1)
  other = Pages(rt, 10, 2, 64, 32)
  for f in (lambda: other.put(b, x), lambda: other.attend(q, b), lambda: pool.put(None, x)):
    with pytest.raises(ValueError, match="batch must be planned"): f()
  logits, ids, starts, u = Tensor.zeros(rt, 4, 50, dtype="fp32"), r(1, 2, 3, 4), r(0, 4), Tensor.zeros(rt, 2, 4, dtype="fp32")
  for args in ((Tensor.zeros(rt, 4, 50), ids, starts, u), (logits, r(1), starts, u), (logits, ids, r(0), u), (logits, ids, starts, logits),
               (logits, ids, starts, u, u), (logits, ids, starts, u, None, u), (logits, ids, None, u)):
    with pytest.raises((ValueError, AttributeError)): serve.verify(*args)


def verified_behind(rt, logits, ids, starts, uniforms, drafts, probs=None, t=None):
  """verified() with a count of drafts a request: the rows ahead are not looked at."""
  of = lambda a: Tensor.of(rt, np.asarray(a, np.float32), "fp32")
  tokens, counts = serve.verify(of(logits), row(rt, ids), row(rt, starts), of(uniforms), of(probs) if probs is not None else None,
                                of(np.reshape(t, (-1, 1))) if t is not None else None, row(rt, drafts))
  want = P.verify(logits, ids, starts, uniforms, probs, None if t is None else np.asarray(t, np.float32), drafts)
  assert np.array_equal(ints(tokens), want[0]) and np.array_equal(ints(counts), want[1]), (ints(tokens), ints(counts), want)


@pytest.mark.parametrize("vocab", [300, 3001])
@pytest.mark.parametrize("drawn", [True, False])
def test_verify_behind_a_prompts_rows(rt, vocab, drawn):
  rng = np.random.default_rng(vocab)
  starts = [0, 90, 91, 91, 96, 170, 180]
  rows = 183
  logits = 3 * rng.normal(0, 1, (rows, vocab)).astype(np.float32)
  probs = near(rng, logits) if drawn else None
  ids = np.roll(logits, 1, 0).argmax(1)
  ids[::7] = rng.integers(0, vocab, len(ids[::7]))
  for drafts in ([0] * 6, [0, 0, -1, 4, -1, 3], [-1] * 6, [89, 90, 0, 2, 73, 2 ** 31 - 1], [-2 ** 31, 5, 5, 5, 70, 1]):
    u = rng.random((2, rows)).astype(np.float32)
    verified_behind(rt, logits, ids, starts, u, drafts, probs)
    verified_behind(rt, logits, ids, starts, u, drafts, probs, [np.inf] * rows)
    verified_behind(rt, logits, ids, starts, u, drafts, probs, rng.uniform(0.5, 2, rows))


def test_a_prompts_next_token_follows_its_last_row(rt):
  # one step with a prompt's last chunk, a chunk that does not end its prompt, a token and its drafts, and a request without
  # rows: greedily, the prompt's token is what its last row's logits give, and as good as llama.forward's over a bf16 cache
  # (whose logits the paged ones keep to within 3% of the largest, on either side)
  from baretile_amd.models import llama
  from oracle import llama_ref as L
  rng = np.random.default_rng(43)
  c, w = L.smol(rng, 2, vocab=256, places=96)
  dc = llama.model(dim=576, heads=9, kv=3, layers=2, eps=1e-5, theta=10000.0, vocab=256, ffn=1536)
  dw = llama.upload(rt, {k: v for k, v in w.items() if k not in ("cos", "sin", "turn", "embed.T")}, dc, places=96)
  caches = llama.paged_cache(rt, dc, 30, 16)
  prompts = [rng.integers(0, 256, n) for n in (37, 20, 9)]
  b, (tables, *_, taken) = planned(rt, caches[0], np.full((4, 6), -1), [0] * 4, [0, 0, 9, 0], rng.permutation(30), 9)
  llama.paged_forward(row(rt, prompts[2]), b, dw, dc, caches).realize()
  ids, drafts = np.concatenate([prompts[0], prompts[1], [5, 6, 7], [0]]), [0, -1, 2, -1]
  b, (_, starts, *_) = planned(rt, caches[0], tables, [0, 0, 9, 0], [37, 20, 3, 0], rng.permutation(30), 61, taken)
  logits = llama.paged_forward(row(rt, ids), b, dw, dc, caches).realize()
  u, t = rng.random((2, 61)).astype(np.float32), np.full((61, 1), np.inf)
  tokens, counts = serve.verify(logits.reshape(61, 256), row(rt, ids), b.starts, Tensor.of(rt, u, "fp32"), t=Tensor.of(rt, t, "fp32"),
                                drafts=row(rt, drafts))
  got = np.array(logits.tolist(), np.float32).reshape(61, 256)
  want = P.verify(got, ids, starts, u, t=t, drafts=drafts)
  assert np.array_equal(ints(tokens), want[0]) and np.array_equal(ints(counts), want[1])
  token = ints(tokens)[36]
  assert token == got[36].argmax() and (ints(tokens)[:36] == -1).all() and ints(counts)[:2].tolist() == [1, 0]
  plain = llama.forward(row(rt, prompts[0]), row(rt, range(37)), dw, dc, llama.kv_cache(rt, dc, 96))
  plain = np.array(plain.tolist()).reshape(-1)
  assert plain[token] >= plain.max() - 0.06 * np.abs(plain).max()
  with pytest.raises(ValueError, match="drafts"): serve.verify(logits.reshape(61, 256), row(rt, ids), b.starts, Tensor.of(rt, u, "fp32"),
                                                               drafts=row(rt, drafts[:3]))


def test_verify_writes_the_rows_ahead_of_its_first_request(rt):
  # a run of a longer batch's requests: the rows of the requests before it have no token either
  rng = np.random.default_rng(44)
  logits, u = rng.normal(0, 2, (70, 100)).astype(np.float32), rng.random((2, 70)).astype(np.float32)
  ids, starts = logits.argmax(1), Tensor.of(rt, [[0, 4, 66, 68, 69]], "int32")
  old = Tensor.of(rt, np.full((1, 70), 7), "int32")  # what the result's memory may hold
  del old
  tokens, counts = serve.verify(Tensor.of(rt, logits, "fp32"), row(rt, ids), starts[:, 2:], Tensor.of(rt, u, "fp32"))
  want = P.verify(logits, ids, [66, 68, 69], u)
  assert np.array_equal(ints(tokens), want[0]) and np.array_equal(ints(counts), want[1])


def test_plan_counts_blocks_past_32_bits(rt):
  # 160 requests of 2^30 tokens: 2^24 blocks of keys each, 2.7 billion in all. As many parts as attention launches, 512 and one
  # a request for one key head, and a run of at most 2^24 blocks to each.
  pool, requests = Pages(rt, 4, 1, 64, 256), 160
  tables = Tensor(rt, requests, 1 << 22, dtype="int32")
  rt.fill32(tables.addr, -1, requests << 22)
  b = pool.plan(tables, row(rt, [2 ** 30 - 1] * requests), row(rt, [1] * requests), row(rt, [0]), requests)
  *parts, per = ints(b.parts).tolist()
  blocks = 1 << 24
  assert per == (-(-requests * blocks // 512) + 3) // 4 * 4 <= blocks
  assert parts == [i * -(-blocks // per) for i in range(requests + 1)] and parts[-1] <= 512 + requests
  assert ints(b.lengths).tolist() == [2 ** 30] * requests and ints(b.starts).tolist() == list(range(requests + 1))


# ---- attention past the 64 pages of a request that a wave's lanes hold at a time. Every row's head has one key, at a place of its
# own, that outweighs all others (score 24; the others', of rows of hd unit normals, keep within 6 24 / hd^0.5, at most 18, and mostly
# within half of that), so a page that is read in another's place is another result altogether.

def shared(rt, rng, kv, hd, page, tokens):
  """A pool of one request's tokens: (pool, values, its pages). Requests that only read may share them."""
  pages = tokens // page
  pool, values, s = Pages(rt, pages, kv, hd, page), np.zeros((pages, 2 * kv, page, hd)), np.full((pages, 2 * kv), 2.0 ** -100)
  x = B.bf16(rng.normal(0, 1, (2 * kv, tokens, hd)))
  b, (tables, starts, lengths, *_) = planned(rt, pool, np.full((1, pages), -1), [0], [tokens], rng.permutation(pages), tokens)
  pool.put(b, Tensor.of(rt, x))
  P.put(values, s, tables, starts, lengths, x)
  return pool, values, tables[0]


def pointed(rng, heads, values, tables, starts, lengths, window=0):
  """Queries that each point at one of the keys that their row sees, one row's heads at places all over: (q, the places)."""
  pages, kv2, page, hd = values.shape
  q, at = np.zeros((heads, starts[-1], hd)), np.zeros((heads, starts[-1]), int)
  for r, length in enumerate(lengths):
    for i in range(starts[r], starts[r + 1]):
      place = length - starts[r + 1] + i
      for h in range(heads):
        at[h, i] = t = rng.integers(max(0, place + 1 - window) if window else 0, place + 1)
        k = values[tables[r, t // page], h // (heads // (kv2 // 2)), t % page]
        q[h, i] = 24 * k / (k @ k)
  return B.bf16(q), at


def attend_by_head(q, values, tables, starts, lengths, window=0):
  """oracle.pages.attend, a request's head at a time."""
  pages, kv2, page, hd = values.shape
  rep = q.shape[0] // (kv2 // 2)
  out, weighed = np.zeros(q.shape), np.zeros(q.shape)
  for r, length in enumerate(lengths):
    rows = slice(starts[r], starts[r + 1])
    place = np.arange(length - (starts[r + 1] - starts[r]), length)[:, None]
    held = values[tables[r, :-(-length // page)]]
    key = np.arange(held.shape[0] * page)
    hidden = (key > place) | ((key <= place - window) if window else False)
    for h in range(q.shape[0]):
      k, v = (held[:, i].reshape(-1, hd) for i in (h // rep, kv2 // 2 + h // rep))
      s = np.where(hidden, -np.inf, q[h, rows].astype(np.float64) @ k.T)
      p = np.exp(s - s.max(1, keepdims=True))
      p /= p.sum(1, keepdims=True)
      out[h, rows], weighed[h, rows] = p @ v, p @ np.abs(v)
  return out, weighed


def points_found(rt, rng, pool, values, heads, tables, lengths, new, window=0, most=None):
  """Attention with pointed queries against the 64-bit form, and the batch: what it found is near the value pointed at."""
  rows, kv, rep = sum(new), pool.kv, heads // pool.kv
  b, (made, starts, total, *_) = planned(rt, pool, tables, [n - m for n, m in zip(lengths, new)], new, [-1], rows, most=most)
  q, at = pointed(rng, heads, values, made, starts, total, window)
  got = np.array(pool.attend(Tensor.of(rt, q), b, window).tolist()).reshape(q.shape)
  want, weighed = attend_by_head(q, values, made, starts, total, window)
  owner = np.repeat(np.arange(len(new)), new)
  v = np.stack([values[made[owner, at[h] // pool.page], kv + h // rep, at[h] % pool.page] for h in range(heads)])
  assert (np.abs(want - v).max(-1) < 0.1).mean() > 0.95  # (the queries do point)
  assert np.all(np.abs(got - want) <= bound(q, values, weighed, want)), np.abs(got - want).max()
  return b


def pages_of_a_part(b, lengths):
  """The most pages of a part of the batch's, from the plan's least blocks of keys a part."""
  per, blocks = int(ints(b.parts)[-1]), -(-max(lengths) // 64)
  return max(per, -(-blocks // 32)) * 64 // b.page


@pytest.mark.parametrize("hd, page, requests, new", [(64, 16, 32, 1), (128, 16, 32, 1), (64, 32, 48, 1), (64, 16, 32, 5), (64, 16, 32, 17)])
def test_attend_parts_of_more_pages_than_a_wave_holds(rt, hd, page, requests, new):
  rng = np.random.default_rng(hd + page + new)
  pool, values, pages = shared(rt, rng, 8, hd, page, 4000)
  tables = np.stack([rng.permutation(pages) for _ in range(requests)])
  lengths = rng.integers(3900, 4001, requests).tolist()
  b = points_found(rt, rng, pool, values, 16, tables, lengths, [new] * requests, most=new)
  assert pages_of_a_part(b, lengths) > 64
  # with a window that leaves a part's first blocks out, and a part's last
  points_found(rt, rng, pool, values, 16, tables, lengths, [new] * requests, window=3333, most=new)


@pytest.mark.parametrize("new", [1, 6])
def test_attend_a_long_cache_of_short_pages(rt, new):
  # one request of 65536 keys is cut into 32 parts of 128 pages of 16; of 2^18 keys, of 256 pages of 32
  rng = np.random.default_rng(new)
  for page, tokens in ((16, 1 << 16), (32, 1 << 18)):
    pool, values, pages = shared(rt, rng, 1, 64, page, tokens)
    b = points_found(rt, rng, pool, values, 8, pages[None], [tokens], [new], most=new)
    assert pages_of_a_part(b, [tokens]) > 64
  pool, values, pages = shared(rt, rng, 1, 64, 256, 300032)  # and one whose parts' pages are loaded once each, 38 at most
  assert pages_of_a_part(points_found(rt, rng, pool, values, 8, pages[None], [300000], [new], most=new), [300000]) <= 64


@pytest.mark.parametrize("hd, page, tokens, window", [(64, 16, 2608, 0), (128, 16, 1600, 0), (64, 32, 3008, 0), (64, 64, 4608, 0),
                                                      (64, 16, 2608, 1500)])
def test_attend_tiles_of_more_pages_than_a_wave_holds(rt, hd, page, tokens, window):
  # a prompt of 520 rows of 32 heads over 8, which are tiles enough that none has its keys cut
  rng = np.random.default_rng(hd + page + window)
  pool, values, pages = shared(rt, rng, 8, hd, page, tokens)
  b = points_found(rt, rng, pool, values, 32, pages[None], [tokens - 3], [520], window)
  need = ctypes.c_uint64()
  _lib.call("pages_attend_scratch", ctypes.byref(pool.args), ctypes.byref(b.args), 32, window, ctypes.byref(need))
  items = 2048 // (4 * 8) + 1
  assert need.value == items * 8 * 32 * (hd + 4) * 4  # the parts' alone: no splits
  assert min(tokens, window + 520 if window else tokens) > 64 * page


def test_attend_parts_of_many_pages_beside_tiles(rt):
  rng = np.random.default_rng(45)
  pool, values, pages = shared(rt, rng, 8, 64, 16, 4000)
  tables = np.stack([rng.permutation(pages) for _ in range(33)])
  lengths = [4000] * 16 + [2100] + [3990] * 16
  b = points_found(rt, rng, pool, values, 16, tables, lengths, [1] * 16 + [300] + [2] * 16)
  assert pages_of_a_part(b, lengths) > 64


# ---- verification, 16 logits a lane (past 2^22 logits) and requests of more rows than a block keeps sums of (64)

@pytest.mark.parametrize("rows, vocab", [(40, 131072), (40, 131073), (23, 200001), (15, 300004), (15, 300001), (4200, 1000), (66000, 64)])
@pytest.mark.parametrize("drawn", [True, False])
def test_verify_of_more_logits(rt, rows, vocab, drawn):
  assert rows * vocab > 1 << 22
  rng = np.random.default_rng(vocab)
  lengths = rng.integers(0, 8, 2 * rows)
  starts = np.concatenate([[0], np.cumsum(lengths)])
  starts = starts[starts <= rows - 2].tolist()
  logits = 3 * rng.normal(0, 1, (rows, vocab)).astype(np.float32)
  logits[rng.random((rows, vocab)) < 0.1] = -np.inf
  logits[:, 0] = 0  # (a weight in every row)
  p = soft(logits)
  probs = soft(np.roll(np.where(np.isfinite(logits), logits, -9), 1, 0) + 0.7 * rng.normal(0, 1, logits.shape)).astype(np.float32)
  upto = np.cumsum(probs, 1, dtype=np.float64)
  ids = np.minimum((upto < rng.random((rows, 1)) * 0.999).sum(1), vocab - 1) if drawn else np.roll(p, 1, 0).argmax(1)
  t = rng.uniform(0.5, 2, rows)
  t[::9] = np.inf
  for i in range(2):
    verified(rt, logits, ids, starts, rng.random((2, rows)).astype(np.float32), probs if drawn else None, t.astype(np.float32) if i else None)


@pytest.mark.parametrize("vocab", [1000, 1001, 20000])
@pytest.mark.parametrize("drawn", [True, False])
def test_verify_of_long_runs_of_drafts(rt, vocab, drawn):
  # refused at their first draft, the last whose sums are kept, the first whose are not, far behind, or not at all
  rng = np.random.default_rng(vocab)
  starts, at = list(range(0, 1051, 150)), (1, 63, 64, 65, 149, None, 100)
  rows = starts[-1] + 3
  logits = 3 * rng.normal(0, 1, (rows, vocab)).astype(np.float32)
  probs = near(rng, logits) if drawn else None
  ids = np.roll(logits, 1, 0).argmax(1)
  for t in (None, np.full(rows, np.inf, np.float32), rng.uniform(0.5, 2, rows).astype(np.float32)):
    u = rng.random((2, rows)).astype(np.float32)
    u[0] = 0  # any draft that has a weight is accepted
    refused = ids.copy()
    odd = logits.copy()
    for s, k in zip(starts, at):
      if k is not None: odd[s + k - 1, refused[s + k]] = -np.inf  # the draft at row s + k has none
    got = verified(rt, odd, refused, starts, u, probs, t)
    for s, k, n in zip(starts, at, got[1]): assert n == (150 if k is None else k)


# ---- nothing outside: results and scratch between guards, pages of no request

class Guarded:
  """Device memory of exactly nbytes between guards, all of it a pattern at first."""
  AHEAD, FILL = 1024, 0x5A5A5A5A

  def __init__(self, rt, nbytes):
    self.rt, self.nbytes, self.storage = rt, nbytes, Storage(rt, nbytes + 2 * self.AHEAD)
    assert nbytes % 4 == 0
    rt.fill32(self.storage.addr, self.FILL, (nbytes + 2 * self.AHEAD) // 4)
    self.addr = self.storage.addr + self.AHEAD

  def values(self, dtype):
    """What lies between the guards, which have to be as they were."""
    a = np.frombuffer(bytes(self.rt.download(self.storage.addr, self.nbytes + 2 * self.AHEAD)), np.uint32)
    ahead = self.AHEAD // 4
    assert (a[:ahead] == self.FILL).all() and (a[ahead + self.nbytes // 4:] == self.FILL).all()
    return a[ahead:ahead + self.nbytes // 4].view(dtype)


def attend_guarded(rt, pool, b, q, window=0):
  """Pages.attend's call with its result and exactly the scratch that it asks for between guards: the result's bits."""
  heads, rows, hd = q.batch, q.rows, q.cols
  need = ctypes.c_uint64()
  pair = ctypes.byref(pool.args), ctypes.byref(b.args)
  _lib.call("pages_attend_scratch", *pair, heads, window, ctypes.byref(need))
  out, scratch = Guarded(rt, 2 * heads * rows * hd), Guarded(rt, need.value)
  rt.run("pages_attend", "pages_attend", *pair, q.addr, q.sb, q.sr, out.addr, rows * hd, hd, heads, window, scratch.addr if need.value else 0,
         need.value)
  scratch.values(np.uint32)
  return out.values(np.uint16)


STRAY = ([0, 10, 9000], [-5, 20, 30], [40, 3, 50], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [50, 50, 50], [-1, -1, -1], [0, 50, 0])


@pytest.mark.parametrize("vocab, probs", [(1000, True), (1001, False), (100000, True)])
def test_verify_stays_within_its_memory(rt, vocab, probs):
  rng = np.random.default_rng(vocab)
  rows, R = 50, 2
  logits, ids, u = rng.normal(0, 2, (rows, vocab)).astype(np.float32), rng.integers(-3, vocab + 3, rows), rng.random((2, rows)).astype(np.float32)
  p = near(rng, logits) if probs else None
  of = lambda a: Tensor.of(rt, a, "fp32")
  held = [of(logits), row(rt, ids), of(u), of(p) if probs else None]
  for starts, drafts in ([([0, 20, 47], None), ([0, 20, 47], [3, 0])] + [(s, None) for s in STRAY] +
                         [(s, [2 ** 31 - 1, -2 ** 31]) for s in STRAY] + [(s, [7, 1]) for s in STRAY]):
    s, d = row(rt, starts), row(rt, drafts) if drafts else None
    tokens, counts = Guarded(rt, 4 * rows), Guarded(rt, 4 * R)
    args = _lib.VerifyArgs(logits=held[0].addr, probs=held[3].addr if probs else 0, uniforms=held[2].addr, ids=held[1].addr, starts=s.addr,
                           tokens=tokens.addr, counts=counts.addr, logits_sr=vocab, probs_sr=vocab, uniforms_sr=rows, requests=R, rows=rows,
                           vocab=vocab, drafts=d.addr if drafts else 0)
    need = ctypes.c_uint64()
    _lib.call("verify_scratch", ctypes.byref(args), ctypes.byref(need))
    scratch = Guarded(rt, need.value)
    args.scratch, args.scratch_bytes = scratch.addr, need.value
    rt.run("verify", "verify", ctypes.byref(args))
    scratch.values(np.uint32)
    got = tokens.values(np.int32), counts.values(np.int32)
    if starts == [0, 20, 47]:
      want = P.verify(logits, ids, starts, u, p, drafts=drafts)
      assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("new, most, width", [([10, 40], None, 5), ([3, 2], 3, 5), ([3, 2], 1, 5), ([3, 2], 3, 80)])
def test_stray_starts_touch_nothing_else(rt, new, most, width):
  # starts that no plan makes: any rows of the batch's own, but no page of another request or of one that is left without rows, no
  # guard, and no row past the last
  rng = np.random.default_rng(13)
  pool, _, tables, _ = filled(rt, rng, 4, 2, 64, 16, [60, 80, 50], width, spare=4)
  own = np.array(tables)[:2]
  b, _ = planned(rt, pool, own, [60 - max(new), 80 - max(new)], new, [-1], 50, most=most)
  x, q = Tensor.of(rt, bf16_rows(rng, 4, 50, 64)), Tensor.of(rt, B.bf16(rng.normal(0, 0.2, (4, 50, 64))))
  for starts in STRAY:
    first, last = (np.clip(v, 0, 50) for v in (starts[:-1], starts[1:]))
    others = np.setdiff1d(np.arange(pool.pages), own[last > first])
    before = whole(pool)[others], scales(pool)[others]
    b.starts.assign(row(rt, starts))
    pool.put(b, x)
    attend_guarded(rt, pool, b, q)
    assert np.array_equal(whole(pool)[others], before[0]) and np.array_equal(scales(pool)[others], before[1])


@pytest.mark.parametrize("hd, page, lengths, new, window", [
  (64, 16, [300, 40, 0, 77], [1, 3, 0, 2], 0), (64, 16, [3000, 40, 2000], [1, 3, 5], 0), (128, 64, [3000, 40, 2000], [5, 1, 9], 0),
  (64, 32, [3000, 400, 2000], [1, 90, 5], 0), (128, 16, [700, 400], [333, 40], 0), (64, 16, [3000, 2000], [2, 70], 300), (64, 256, [5000, 9], [16, 9], 0)])
def test_attend_stays_within_its_memory(rt, hd, page, lengths, new, window):
  rng = np.random.default_rng(hd + page + sum(new))
  pool, _, tables, _ = filled(rt, rng, 8, 2, hd, page, lengths)
  rows = sum(new) + 5
  b, _ = planned(rt, pool, tables, [n - m for n, m in zip(lengths, new)], new, [-1], rows)
  q = Tensor.of(rt, B.bf16(rng.normal(0, 0.2, (8, rows, hd))))
  assert attend_guarded(rt, pool, b, q, window).tobytes() == pool.attend(q, b, window).tobytes()


@pytest.mark.parametrize("requests, rows", [(1, 1), (5, 33), (300, 900), (3, 2500)])
def test_plan_stays_within_its_memory(rt, requests, rows):
  rng = np.random.default_rng(requests)
  page, width, pages = 16, 40, 3000
  tables = np.full((requests, width), -1)
  cached, new, free = rng.integers(0, 300, requests), rng.integers(0, 2 * rows // requests + 2, requests), rng.permutation(pages)
  t = Guarded(rt, 4 * tables.size)
  rt.upload(t.addr, tables.astype(np.int32).tobytes())
  given = [row(rt, v) for v in (cached, new, free)]
  made = [Guarded(rt, 4 * n) for n in (requests + 1, requests, rows, rows, 1, requests + 2)]  # starts, lengths, places, slots, taken, parts
  args = _lib.PlanArgs(t.addr, *(g.addr for g in given), 0, *(m.addr for m in made), width, requests, width, pages, rows, page, pages, rows, 2)
  rt.run("plan", "pages_plan", ctypes.byref(args))
  want = P.plan(tables, cached, new, free, rows, page, pages)
  assert np.array_equal(t.values(np.int32).reshape(tables.shape), want[0])
  got = [m.values(np.int32) for m in made]
  for g, w in zip(got, want[1:5]): assert np.array_equal(g, w)
  assert got[4][0] == want[5]


def test_plan_counts_blocks_of_many_requests(rt):
  # 1100 requests of up to 2^28 tokens, over 2 billion blocks of keys in all, scanned in two turns; some bring no row
  rng = np.random.default_rng(46)
  pool, requests = Pages(rt, 4, 8, 64, 256), 1100
  tables = Tensor(rt, requests, 1 << 20, dtype="int32")
  rt.fill32(tables.addr, -1, requests << 20)
  cached, new = rng.integers(2 ** 27, 2 ** 28 - 3, requests), rng.integers(0, 3, requests)
  cached[5], new[5] = 0, 2
  b = pool.plan(tables, row(rt, cached), row(rt, new), row(rt, [0]), 2200)
  *parts, per = ints(b.parts).tolist()
  blocks = np.where(new > 0, -(-(cached + new) // 64), 0)
  assert blocks.sum() > 1 << 31
  assert per == min((-(-int(blocks.sum()) // 64) + 3) // 4 * 4, 1 << 24)  # (a part holds one request's, so never more than 2^24)
  assert parts == [0, *np.cumsum(-(-blocks // np.maximum(per, -(-blocks // 32)))).tolist()] and parts[-1] <= 64 + requests
  assert np.array_equal(ints(b.lengths), cached + new) and np.array_equal(ints(b.starts), [0, *np.cumsum(new)])


def test_missing_tensors_are_refused(rt):
  from baretile_amd.models import llama
  r = lambda *v: row(rt, v)
  logits, ids, starts, u = Tensor.zeros(rt, 4, 50, dtype="fp32"), r(1, 2, 3, 4), r(0, 4), Tensor.zeros(rt, 2, 4, dtype="fp32")
  for i in range(4):
    args = [logits, ids, starts, u]
    args[i] = None
    with pytest.raises(ValueError, match="verify needs"): serve.verify(*args)
  with pytest.raises(ValueError, match="verify needs"): serve.verify(logits, ids, starts, u, drafts=u)
  dc = llama.smol(layers=1)
  for bad in ((ids, None), (ids, starts), ([1, 2], None)):
    with pytest.raises(ValueError, match="paged_forward needs"): llama.paged_forward(*bad, {}, dc, [None])



def test_attend_scores_below_every_number(rt):
  # a row that sees only scores of -inf is zeros, as one that sees no key; beside keys with others they weigh nothing
  rng = np.random.default_rng(47)
  for lengths, new in (([90, 40], [2, 1]), ([90, 40], [2, 40]), ([2000, 40], [2, 1]), ([2000, 200], [2, 90])):
    rows = sum(new)
    pool = Pages(rt, 200, 2, 64, 16)
    x = np.abs(bf16_rows(rng, 4, sum(lengths), 64)) + 0.5
    x[0, lengths[0] - 5, 1] = x[1, lengths[0] - 5, 1] = 0  # one key of the first request scores 0 * -inf at dim 1: not a number
    b, (tables, *_, taken) = planned(rt, pool, np.full((2, 130), -1), [0, 0], lengths, rng.permutation(200), sum(lengths))
    pool.put(b, Tensor.of(rt, B.bf16(x)))
    values, s = np.zeros((200, 4, 16, 64)), np.full((200, 4), 2.0 ** -100)
    P.put(values, s, tables, [0, lengths[0], sum(lengths)], lengths, B.bf16(x))
    q = np.abs(B.bf16(rng.normal(0, 0.02, (4, rows, 64))))
    q[0, 0, 0] = q[2, rows - 1, 0] = -np.inf
    q[3, 1, 1] = -np.inf  # with a key that this row's head scores NaN
    b, (tables, starts, total, *_) = planned(rt, pool, tables, [n - m for n, m in zip(lengths, new)], new, [-1], rows, taken)
    got = np.array(pool.attend(Tensor.of(rt, q), b).tolist())
    odd = np.zeros((4, rows), bool)
    odd[0, 0] = odd[2, rows - 1] = odd[3, 1] = True
    assert (got[0, 0] == 0).all() and (got[2, rows - 1] == 0).all() and np.isnan(got[3, 1]).all()
    q[odd] = 0
    want, weighed = P.attend(q, values, tables, starts, total)
    assert np.all(np.abs(got - want)[~odd] <= bound(q, values, weighed, want)[~odd])


def test_a_recorded_verification_follows_its_drafts(rt):
  rng = np.random.default_rng(48)
  rows, R, vocab = 40, 4, 700
  logits, ids, starts = Tensor.zeros(rt, rows, vocab, dtype="fp32"), row(rt, [0] * rows), row(rt, [0] * (R + 1))
  u, drafts = Tensor.zeros(rt, 2, rows, dtype="fp32"), row(rt, [0] * R)
  step = lambda: serve.verify(logits, ids, starts, u, drafts=drafts)
  step()
  rt.wait()
  rec = Recording(rt)
  with rec: tokens, counts = step()
  for i in range(5):
    ls, us = rng.normal(0, 3, (rows, vocab)).astype(np.float32), rng.random((2, rows)).astype(np.float32)
    ds = np.roll(ls, 1, 0).argmax(1)
    at, n = np.sort(rng.choice(rows + 1, R + 1)), rng.integers(-1, 9, R)
    for t, v, kind in ((logits, ls, "fp32"), (ids, ds[None], "int32"), (starts, at[None], "int32"), (u, us, "fp32"), (drafts, n[None], "int32")):
      t.assign(Tensor.of(rt, v, kind))
    rec.send()
    rt.wait()
    want = P.verify(ls, ds, at, us, drafts=n)
    assert np.array_equal(ints(tokens), want[0]) and np.array_equal(ints(counts), want[1]), i
