"""serve.logprobs on the GPU against oracle/logprobs.py in 64 bits: labels exactly, the rest within what fp32's roundings allow. Needs a
GPU."""
import ctypes
import numpy as np
import pytest

from baretile_amd import _lib
from baretile_amd.models import serve
from baretile_amd.pages import Pages
from baretile_amd.tensor import Recording, Storage, Tensor
from oracle import logprobs as L

pytestmark = pytest.mark.gpu

INF = np.inf


def fp32(rt, a): return Tensor.frombytes(rt, *np.shape(a), np.ascontiguousarray(a, np.float32).tobytes(), 1, "fp32")


def row(rt, a): return Tensor.of(rt, [[int(v) for v in a]], "int32")


def back(t, dtype=np.float32): return np.frombuffer(t.tobytes(), dtype).reshape(t.shape[-2:])


def near(got, want, off):
  with np.errstate(over="ignore"): same = got == np.float32(want)  # (infinities, too, and what is past the largest number of 32 bits)
  with np.errstate(invalid="ignore"): return np.all(same | (np.abs(got - want) <= off))


def same_as_oracle(got, logits, ids, k, t):
  want = L.logprobs(logits, ids, k, t)
  lp, h = back(got[0])[0], back(got[1])[0]
  assert near(lp, want[0], want[4]), (lp, want[0])
  assert near(h, want[1], want[5]), (h, want[1], want[5])
  assert len(got) == (4 if k else 2)
  if k:
    assert np.array_equal(back(got[3], np.int32), want[3])
    assert near(back(got[2]), want[2], want[6])


def checked(rt, logits, ids, k=0, t=None):
  got = serve.logprobs(fp32(rt, logits), row(rt, ids), k, None if t is None else fp32(rt, np.reshape(t, (-1, 1))))
  same_as_oracle(got, logits, ids, k, t)


@pytest.mark.parametrize("k", [0, 1, 2, 5, 20, 64])
@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 256, 1000, 4095, 4096, 4097, 4100, 16390, 49152, 131072, 200001])
def test_logprobs(rt, vocab, k):
  rng = np.random.default_rng(vocab + k)
  rows = 1 if vocab > 100000 else 5
  logits = (3 * rng.normal(0, 1, (rows, vocab))).astype(np.float32)
  ids = rng.integers(0, vocab, rows)
  checked(rt, logits, ids, k)
  checked(rt, logits, ids, k, rng.uniform(0.3, 3, rows))


@pytest.mark.parametrize("k", [0, 3, 64])
def test_the_largest_vocabulary(rt, k):
  rng = np.random.default_rng(k)
  logits = (4 * rng.normal(0, 1, (2, 1 << 20))).astype(np.float32)
  checked(rt, logits, [5, (1 << 20) - 1], k)


def test_many_rows(rt):
  rng = np.random.default_rng(1)
  logits = (3 * rng.normal(0, 1, (700, 5000))).astype(np.float32)
  ids = rng.integers(-3, 5010, 700)  # some that are none
  checked(rt, logits, ids, 4)
  checked(rt, logits[:, :777], ids, 0, rng.uniform(0.5, 2, 700))


@pytest.mark.parametrize("vocab", [64, 300, 4096, 9000, 70001])
@pytest.mark.parametrize("k", [1, 7, 64])
def test_ties_go_to_the_lowest_column(rt, vocab, k):
  rng = np.random.default_rng(vocab)
  coarse = np.round(2 * rng.normal(0, 1, vocab)) / 2
  zeros = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
  peaks = np.where(np.arange(vocab) % 17 == 3, 5.0, rng.normal(0, 1, vocab))
  few = np.full(vocab, 1.0)
  few[rng.integers(0, vocab, 3)] = 2.0
  late = np.where(np.arange(vocab) >= vocab - 40, 3.0, -1.0)
  checked(rt, np.stack([coarse, zeros, peaks, few, late, np.full(vocab, -7.5)]), [0, 1, 3, 4, vocab - 1, 9], k)


@pytest.mark.parametrize("vocab", [500, 4096, 20000])
@pytest.mark.parametrize("k", [1, 20, 64])
def test_rows_in_order(rt, vocab, k):
  # where the largest lie in one thread's run, or in one chunk
  up = np.arange(vocab) / vocab
  blocks = np.arange(vocab) // 4 % 256 == 7  # one thread's columns in each chunk
  checked(rt, np.stack([up, -up, up % 0.1, np.where(blocks, 10 + up, up), np.where(np.arange(vocab) < 300, up + 3, up)]), [0, 1, 2, 3, 4], k)


@pytest.mark.parametrize("rows, vocab", [(2100, 9002), (1100, 33000), (5000, 5000), (700, 70001)])
@pytest.mark.parametrize("k", [0, 1, 20, 64])
def test_rows_walked_a_chunk_at_a_time(rt, rows, vocab, k):
  # rows enough that a block takes several chunks of one: rows whose every chunk passes the bound of the one before, rows that begin
  # with nothing, or with fewer than k, ties within and across chunks, infinities and NaNs, among random ones
  rng = np.random.default_rng(rows + k)
  x = rng.normal(0, 2, (rows, vocab)).astype(np.float32)
  at = np.arange(vocab)
  some = [at / 64.0, -at / 64.0, np.where(at < vocab - 70, -INF, at / 8.0), np.where(at % 1000 == 5, 1.0, -INF), np.zeros(vocab), np.full(vocab, -INF),
          np.where(at // 4096 % 2 == 1, 3.0, -INF), np.floor(at / 300.0), np.where(at >= vocab // 2, INF, at), np.where(at % 3 == 0, np.nan, at % 977),
          np.where(at < 30, 50.0 - at, -at / 64.0), np.where(at == vocab - 1, 0.0, -INF)]
  for i, a in enumerate(some): x[i::rows // 4][:4] = a
  t = rng.uniform(0.3, 2, rows).astype(np.float32)
  t[::7], t[1::50] = 1, INF
  ids = rng.integers(-1, vocab, rows)
  got = serve.logprobs(fp32(rt, x), row(rt, ids), k, fp32(rt, t[:, None]))
  looked = np.unique(np.concatenate([np.arange(i, rows, rows // 4)[:4] for i in range(20)] + [np.arange(rows - 5, rows)]))
  part = [back(v, np.int32 if v.dtype == "int32" else np.float32) for v in got]
  want = L.logprobs(x[looked], ids[looked], k, t[looked])
  assert near(part[0][0][looked], want[0], want[4]) and near(part[1][0][looked], want[1], want[5])
  if k: assert np.array_equal(part[3][looked], want[3]) and near(part[2][looked], want[2], want[6])


@pytest.mark.parametrize("vocab", [100, 4096, 30000])
@pytest.mark.parametrize("k", [0, 1, 8, 64])
def test_masked_rows(rt, vocab, k):
  rng = np.random.default_rng(vocab + k)
  x = rng.normal(0, 2, (8, vocab)).astype(np.float32)
  x[0, 1:] = -INF  # one token alone
  x[1] = -INF  # none
  x[2, rng.random(vocab) < 0.95] = -INF
  x[3, :] = -INF
  x[3, [vocab - 1, 7, 50]] = 1, 2, 1  # fewer than k
  x[4, :] = np.finfo(np.float32).min  # a mask of the lowest number
  x[4, 11] = 3
  x[5] = np.nan
  x[6, ::3], x[6, 1] = np.nan, -INF
  x[7, 40] = INF
  ids = [0, 3, int(np.argmax(x[2])), 50, 11, 0, 2, 40]
  checked(rt, x, ids, k)
  checked(rt, x, [1, 3, 5, 51, 12, 4, 3, 41], k, [0.5, 1, 2, 0.1, 1, 1, 3, 1])


@pytest.mark.parametrize("vocab", [50, 9000])
def test_temperatures(rt, vocab):
  rng = np.random.default_rng(vocab)
  x = rng.normal(0, 3, (10, vocab)).astype(np.float32)
  x[0, 5] = x[0, 9] = 40  # the first of two largest
  x[1, 3:] = -INF
  x[2] = -INF
  t = [INF, INF, INF, 0, 0, -1, np.nan, 1e-30, 1e30, 3e38]
  x[4, ::2] = -INF
  for ids in ([5, 0, 0, 7, 1, 0, 0, 1, int(x[8].argmax()), 0], [9, int(x[1].argmax()), 1, 2, 2, 3, 4, 5, 6, int(x[9].argmax())]):
    for k in (0, 6): checked(rt, x, ids, k, t)


def test_large_logits(rt):
  big = np.finfo(np.float32).max
  x = np.zeros((4, 300), np.float32)
  x[0], x[0, 3] = -big, big
  x[1], x[1, 3] = big, -big
  x[2] = 1e4 + np.arange(300) / 32
  x[3, 1], x[3, 2] = 3e38, 3e38
  checked(rt, x, [3, 4, 299, 1], 5)
  checked(rt, x, [2, 3, 0, 0], 5, [0, 0, 0.01, 0])


def test_views(rt):
  rng = np.random.default_rng(3)
  x = rng.normal(0, 2, (9, 5000)).astype(np.float32)
  whole, ids = fp32(rt, x), rng.integers(0, 900, (1, 9))
  t = rng.uniform(0.5, 2, (9, 3)).astype(np.float32)
  columns, ts = Tensor.of(rt, np.repeat(ids, 2, 0), "int32"), fp32(rt, t)
  for a, b, rows in ((0, 4096, slice(0, 9)), (1, 4001, slice(2, 7)), (4, 4999, slice(1, 9)), (100, 101 + 900, slice(3, 4))):
    got = serve.logprobs(whole[rows, a:b], columns[1:2, rows], 6, ts[rows, 1:2])
    same_as_oracle(got, x[rows, a:b], ids[0, rows], 6, t[rows, 1])


def test_repeats_itself(rt):
  rng = np.random.default_rng(4)
  x, ids = fp32(rt, np.round(8 * rng.normal(0, 1, (50, 20000))) / 8), row(rt, rng.integers(0, 20000, 50))
  first = [v.tobytes() for v in serve.logprobs(x, ids, 20)]
  for _ in range(5): assert [v.tobytes() for v in serve.logprobs(x, ids, 20)] == first


def test_a_recorded_call_follows_its_inputs(rt):
  rng = np.random.default_rng(5)
  rows, vocab = 6, 9001
  logits, ids, t = Tensor.zeros(rt, rows, vocab, dtype="fp32"), row(rt, [0] * rows), Tensor.zeros(rt, rows, 1, dtype="fp32")
  step = lambda: (serve.logprobs(logits, ids, 10, t), serve.logprobs(logits, ids, 0), serve.logprobs(logits[:, :3000], ids, 2, t))
  step()
  rt.wait()
  rec = Recording(rt)
  with rec: out = step()
  for i in range(5):
    x, at, ts = (rng.normal(0, 2, (rows, vocab))).astype(np.float32), rng.integers(0, 3000, rows), rng.uniform(0.5, 2, (rows, 1)).astype(np.float32)
    x[i % rows, 100:] = -INF
    logits.assign(fp32(rt, x))
    ids.assign(row(rt, at))
    t.assign(fp32(rt, ts))
    rec.send()
    rt.wait()
    same_as_oracle(out[0], x, at, 10, ts)
    same_as_oracle(out[1], x, at, 0, None)
    same_as_oracle(out[2], x[:, :3000], at, 2, ts)


@pytest.mark.parametrize("rows, vocab, k", [(3, 4097, 5), (1, 300, 64), (2, 100000, 0), (4, 70000, 64)])
def test_stays_within_its_memory(rt, rows, vocab, k):
  rng = np.random.default_rng(vocab)
  guard = 4096
  def guarded(nbytes):
    s = Storage(rt, nbytes + 2 * guard)
    rt.fill32(s.addr, 0xA5A5A5A5, s.nbytes // 4)
    return s, nbytes
  x, ids = rng.normal(0, 2, (rows, vocab)).astype(np.float32), rng.integers(0, vocab, rows)
  logits, given = fp32(rt, x), row(rt, ids)
  outs = [guarded(4 * rows), guarded(4 * rows), guarded(4 * rows * k), guarded(4 * rows * k)]
  args = _lib.LogprobsArgs(logits.addr, given.addr, 0, *(s.addr + guard for s, _ in outs), 0, 0, logits.sr, 0, rows, vocab, k, 0)
  need = ctypes.c_uint64()
  _lib.call("logprobs_scratch", ctypes.byref(args), ctypes.byref(need))
  outs.append(guarded(need.value))
  args.scratch, args.scratch_bytes = outs[-1][0].addr + guard, need.value
  rt.run("logprobs", "logprobs", ctypes.byref(args))
  for s, n in outs:
    got = bytes(rt.download(s.addr, s.nbytes))
    assert got[:guard] == b"\xa5" * guard and got[guard + n:] == b"\xa5" * (len(got) - guard - n)
  for (s, n), v in zip(outs, serve.logprobs(logits, given, k)): assert bytes(rt.download(s.addr + guard, n)) == v.tobytes()


def test_what_a_step_over_4_bit_pages_says_of_its_tokens(rt):
  # a prompt's own tokens through a small model over pages of 8 and of 4 bits: log probabilities of the tokens that follow, whose mean
  # the two caches agree on to within what their logits may differ (3% of the largest for each, on either side)
  from baretile_amd.models import llama
  from oracle import llama_ref as R
  rng = np.random.default_rng(6)
  c, w = R.smol(rng, 2, vocab=256, places=96)
  dc = llama.model(dim=576, heads=9, kv=3, layers=2, eps=1e-5, theta=10000.0, vocab=256, ffn=1536)
  dw = llama.upload(rt, {n: v for n, v in w.items() if n not in ("cos", "sin", "turn", "embed.T")}, dc, places=96)
  prompt = rng.integers(0, 256, 50)
  given = np.append(prompt[1:], -1)
  means, largest = [], 0
  for bits in (8, 4):
    caches = llama.paged_cache(rt, dc, 4, 16, bits=bits)
    b = caches[0].plan(Tensor.of(rt, np.full((1, 4), -1), "int32"), row(rt, [0]), row(rt, [50]), row(rt, range(4)), 50)
    logits = llama.paged_forward(row(rt, prompt), b, dw, dc, caches)
    got = serve.logprobs(logits, row(rt, given), 5)
    x = np.frombuffer(logits.tobytes(), np.float32).reshape(50, 256)
    same_as_oracle(got, x, given, 5, None)
    means.append(back(got[0])[0].mean())
    largest = max(largest, np.abs(x).max())
  assert abs(means[0] - means[1]) <= 2 * 2 * 0.03 * largest  # a log probability moves by twice what the logits do


def test_refusals(rt):
  x, ids, t = Tensor.zeros(rt, 4, 50, dtype="fp32"), row(rt, [1, 2, 3, 4]), Tensor.zeros(rt, 4, 1, dtype="fp32")
  for args in ((Tensor.zeros(rt, 4, 50), ids), (x, row(rt, [1])), (x, t), (x, ids, 65), (x, ids, -1), (x, ids, 3, x), (x, ids, 3, ids), (x, None),
               (None, ids), (Tensor.zeros(rt, 4, 50, 2, "fp32"), ids), (x, [1, 2, 3, 4])):
    with pytest.raises(ValueError): serve.logprobs(*args)
  with pytest.raises(TypeError): serve.logprobs(x, ids, 2.5)
  ok = lambda **kw: _lib.LogprobsArgs(**(dict(logits=x.addr, ids=ids.addr, logprobs=t.addr, entropy=t.addr, logits_sr=50, rows=4, vocab=50) | kw))
  for kw in (dict(logits=0), dict(ids=0), dict(logprobs=0), dict(entropy=0), dict(k=3), dict(k=65, values=t.addr, labels=t.addr), dict(rows=0),
             dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(rows=(1 << 20) + 1), dict(k=-1), dict(logits=x.addr + 2), dict(vocab=9000),
             dict(vocab=9000, scratch=x.addr, scratch_bytes=16), dict(vocab=9000, scratch=x.addr + 8, scratch_bytes=1 << 20),
             dict(rows=1 << 20, vocab=1 << 20)):
    with pytest.raises(ValueError): rt.run("refused", "logprobs", ctypes.byref(ok(**kw)))


@pytest.mark.parametrize("vocab", [131072, 1 << 20])
@pytest.mark.parametrize("k", [1, 20, 64])
def test_sums_of_many_chunks(rt, vocab, k):
  # rows enough that a block takes 32 to 256 chunks of one, all of them the same row in memory: equal weights whose sum rounds the same
  # way again and again, nearly equal ones, and largest logits that creep up from chunk to chunk
  rng = np.random.default_rng(vocab + k)
  rows, at = 2048, np.arange(vocab)
  def flat(x):  # with a largest logit that each wave meets in its first chunk
    return np.where((at < 16384) & (at % 64 == 0), 0.0, x)
  ids = np.resize([7, vocab // 2, vocab - 1, -1], rows)
  given, many = row(rt, ids), (rows, k)
  for x in (flat(-0.58), flat(-0.75), flat(-1.49), np.where(at == vocab - 1, 0.0, -1.2), flat(-1.2 + 1e-3 * rng.normal(0, 1, vocab)),
            at * (0.02 / 4096), at * (1e-4 / 4096)):
    x = x.astype(np.float32)
    logits = fp32(rt, x[None])
    out = [Tensor(rt, 1, rows, dtype="fp32"), Tensor(rt, 1, rows, dtype="fp32"), Tensor(rt, *many, dtype="fp32"), Tensor(rt, *many, dtype="int32")]
    args = _lib.LogprobsArgs(logits.addr, given.addr, 0, *(t.addr for t in out), 0, 0, 0, 0, rows, vocab, k, 0)
    need = ctypes.c_uint64()
    _lib.call("logprobs_scratch", ctypes.byref(args), ctypes.byref(need))
    scratch = Storage(rt, max(need.value, 16))
    args.scratch, args.scratch_bytes = scratch.addr, need.value
    rt.run("logprobs", "logprobs", ctypes.byref(args))
    lp, h, values, labels = back(out[0])[0], back(out[1])[0], back(out[2]), back(out[3], np.int32)
    want = L.logprobs(np.repeat(x[None], 4, 0), ids[:4], k)
    assert near(lp[:4], want[0], want[4]), (lp[:4], want[0], want[4])
    assert near(h[:4], want[1], want[5]), (h[:4], want[1], want[5])
    assert near(values[:4], want[2], want[6]) and np.array_equal(labels[:4], want[3])
    assert np.array_equal(lp, np.resize(lp[:4], rows)) and np.all(h == h[0]) and np.all(values == values[0]) and np.all(labels == labels[0])


@pytest.mark.parametrize("vocab", [50, 9000])
def test_the_largest_temperatures(rt, vocab):
  # inverse temperatures up to the largest number, over logits so close that they still tell them apart
  rng = np.random.default_rng(vocab)
  t = np.array([5e37, 1e38, 1.2e38, 2e38, 3e38, np.finfo(np.float32).max, 3e38], np.float32)
  x = (rng.normal(0, 1, (len(t), vocab)) / t[:, None]).astype(np.float32)
  x[-1, ::2] = -3e38
  for ids in (np.argmax(x, 1), rng.integers(0, vocab, len(t))):
    for k in (0, 6): checked(rt, x, ids, k, t)


@pytest.mark.parametrize("bits", [8, 4])
def test_each_tokens_log_probability_over_pages(rt, bits):
  # a prompt through a model whose logits its cache decides: every token's log probability against the oracle's over a cache of the same
  # width, within what a broken cache, or the other width's, is past twice over (test_cache_cost.py)
  import test_cache_cost as M
  from baretile_amd.models import llama
  c, w, prompt, ids = M.model()
  dc = llama.model(**M.CONFIG)
  dw = llama.upload(rt, {n: v for n, v in w.items() if n not in ("cos", "sin", "turn", "embed.T")}, dc, places=96)
  caches = llama.paged_cache(rt, dc, 5, M.PAGE, bits=bits)
  want = M.logits(c, w, prompt, bits)
  for steps in ([M.ROWS], [30, 1, 1, 5, 13]):  # whole, and in pieces, some of one token
    tables, at, taken, got = Tensor.of(rt, np.full((1, 4), -1), "int32"), 0, None, []
    for n in steps:
      b = caches[0].plan(tables, row(rt, [at]), row(rt, [n]), row(rt, [3, 0, 4, 1]), n, taken)
      x = llama.paged_forward(row(rt, prompt[at:at + n]), b, dw, dc, caches)
      out = serve.logprobs(x, row(rt, ids[at:at + n]), 5)
      same_as_oracle(out, np.frombuffer(x.tobytes(), np.float32).reshape(n, 256), ids[at:at + n], 5, None)
      got.append(back(out[0])[0])
      at, taken = at + n, b.taken
    assert np.abs(np.concatenate(got)[:-1] - M.given(want, ids)).max() <= M.allowed(want)
