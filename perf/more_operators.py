"""The operators of a serving step over a paged 4-bit cache, and what its logits say of given tokens, as cases to time and to
compare.

Kinds:
  put       a step's keys and values into their pages, rounded to 4 bits (Pages.put of a pool of 4 bits), and the cache's
            values read back (Pages.values);
  attend    attention over the pages, one row a request, several (drafts) or a prompt's (Pages.attend), for the caches of
            one or more layers;
  logprobs  the log probability of a given token after each row of logits, the row's entropy and its likeliest tokens
            (serve.logprobs).

Steps of few rows are recorded and replayed, as a serving loop runs them; prompts run eagerly. Head counts and widths are
the ones of models.llama.smol and of the benchmark's large block.

A value of the cache is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign, times a scale: for a key, the power of two of its 32
dims, for a value, its row's own, a quarter of 4, 5, 6 or 7 times a power of two; in both the smallest that is at least a
seventh of the largest.
"""
import math

import torch

own = False

LARGE = {"heads": 32, "kv": 8, "head": 128}
SMOL = {"heads": 9, "kv": 3, "head": 64}


def listed():
  return [
    # a decode step's rows into a small cache
    {"name": "put_decode", "kind": "put", **LARGE, "requests": 32, "new": 1, "ragged": False, "cached": 128, "page": 64, "spare": 0},
    # chunks of prompts behind cached rows: pages begun, ended and filled whole
    {"name": "put_prompts", "kind": "put", **LARGE, "requests": 3, "new": 1000, "ragged": True, "cached": 500, "page": 64, "spare": 7},
    # a chat's next token on the small model, 8 layers' caches one after another
    {"name": "attend_token", "kind": "attend", **SMOL, "requests": 1, "new": 1, "ragged": False, "keys": 301, "page": 16,
     "layers": 8, "window": 0, "spare": 0},
    # a batch of streams of uneven, long contexts, two layers
    {"name": "attend_decode_8", "kind": "attend", **LARGE, "requests": 8, "new": 1, "ragged": True, "keys": 16383, "page": 64,
     "layers": 2, "window": 0, "spare": 0},
    # a large batch, 4096 cached rows each
    {"name": "attend_decode_32", "kind": "attend", **LARGE, "requests": 32, "new": 1, "ragged": False, "keys": 4096, "page": 64,
     "layers": 1, "window": 0, "spare": 0},
    # four drafts a stream and the token before them, four layers
    {"name": "attend_drafts", "kind": "attend", **LARGE, "requests": 16, "new": 5, "ragged": True, "keys": 2048, "page": 32,
     "layers": 4, "window": 0, "spare": 3},
    # one stream's long context
    {"name": "attend_long", "kind": "attend", **LARGE, "requests": 1, "new": 1, "ragged": False, "keys": 131072, "page": 128,
     "layers": 1, "window": 0, "spare": 0},
    # two prompts' chunks behind cached rows
    {"name": "attend_prompts", "kind": "attend", **LARGE, "requests": 2, "new": 2048, "ragged": True, "keys": 2560, "page": 64,
     "layers": 1, "window": 0, "spare": 0},
    # one stream's token with its five alternatives, the small model's vocabulary
    {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": 49152, "k": 5, "t": True, "masked": 0.0},
    # a batch of streams, part of the vocabulary masked
    {"name": "logprobs_32", "kind": "logprobs", "rows": 32, "vocab": 131072, "k": 20, "t": True, "masked": 0.1},
    # a prompt's own tokens on the small model, for its perplexity
    {"name": "logprobs_prompt", "kind": "logprobs", "rows": 777, "vocab": 49152, "k": 0, "t": False, "masked": 0.0},
    # a prompt's tokens with their alternatives over a large vocabulary
    {"name": "logprobs_wide", "kind": "logprobs", "rows": 512, "vocab": 131072, "k": 20, "t": False, "masked": 0.0},
  ]


def _log_int(rng, lo, hi):
  """An integer from lo to hi, spread over its logarithm."""
  return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
  kind = rng.choice(("put", "attend", "attend", "logprobs"))
  if kind == "logprobs":
    vocab = _log_int(rng, 1000, 131072)
    return {"kind": "logprobs", "rows": _log_int(rng, 1, min(2048, 2 ** 26 // vocab)), "vocab": vocab, "k": rng.choice((0, 1, 5, rng.randint(2, 64))),
            "t": rng.random() < 0.5, "masked": rng.choice((0.0, 0.1, 0.9))}
  page, spare = rng.choice((16, 32, 64, 128)), rng.choice((0, rng.randint(1, 40)))
  kv, rep, hd = rng.choice(((8, 4, 128), (3, 3, 64), (8, 8, 128), (4, 7, 64), (8, 1, 64), (2, 4, 128)))
  shape = {"heads": kv * rep, "kv": kv, "head": hd}
  if kind == "put":
    if rng.random() < 0.5:
      return {"kind": "put", **shape, "requests": _log_int(rng, 1, 64), "new": _log_int(rng, 1, 8), "ragged": rng.random() < 0.5,
              "cached": _log_int(rng, 1, 200), "page": page, "spare": spare}
    return {"kind": "put", **shape, "requests": rng.randint(1, 4), "new": _log_int(rng, 9, 1024), "ragged": rng.random() < 0.5,
            "cached": _log_int(rng, 1, 600), "page": page, "spare": spare}
  if rng.random() < 0.7:
    requests, keys, new = _log_int(rng, 1, 32), _log_int(rng, 16, 32768), rng.choice((1, 1, rng.randint(2, 9)))
    keys = max(new, min(keys, 2 ** 27 // (requests * kv * hd)))
    return {"kind": "attend", **shape, "requests": requests, "new": new, "ragged": rng.random() < 0.5, "keys": keys, "page": page,
            "layers": rng.randint(1, min(4, 1 + 2 ** 25 // (requests * kv * keys * hd))), "window": rng.choice((0, 0, 0, _log_int(rng, 8, 2000))),
            "spare": spare}
  new = _log_int(rng, 65, 1500)
  return {"kind": "attend", **shape, "requests": rng.randint(1, 2), "new": new, "ragged": rng.random() < 0.5,
          "keys": new + rng.choice((0, _log_int(rng, 1, 1000))), "page": page, "layers": 1, "window": rng.choice((0, 0, _log_int(rng, 8, 600))),
          "spare": spare}


# ---- inputs, made on the GPU from the seed alone

def _generator(seed): return torch.Generator("cuda").manual_seed(int(seed))


def _ints(g, lo, hi, n): return torch.randint(lo, hi + 1, (n,), generator=g, device="cuda", dtype=torch.int32)


def _rows(g, kv, n, hd):
  """Keys and values of n tokens, (2 kv, n, hd) bf16: channels and tokens of uneven size, as a model's are."""
  x = torch.randn(2 * kv, n, hd, generator=g, device="cuda")
  x *= torch.exp(0.5 * torch.randn(2 * kv, 1, hd, generator=g, device="cuda"))
  x *= torch.exp(0.3 * torch.randn(1, n, 1, generator=g, device="cuda"))
  return x.bfloat16()


def _exclusive(n):
  return torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cumsum(n, 0)])


def _inputs(case, seed):
  """The step's lengths and, by kind, its rows. new: each request's rows; free: the pages in the order they are taken."""
  g, s, kind = _generator(seed), {"case": case}, case["kind"]
  if kind == "logprobs":
    n, V = case["rows"], case["vocab"]
    x = 3 * torch.randn(n, V, generator=g, device="cuda")
    if case["masked"]: x.masked_fill_(torch.rand(n, V, generator=g, device="cuda") < case["masked"], -math.inf)
    s["t"] = 0.7 + torch.rand(n, 1, generator=g, device="cuda") if case["t"] else None
    # the given token: one drawn from the row (the largest of it with Gumbel noise), -1 in a row that has none
    s["ids"] = torch.stack([(r - torch.log(-torch.log(torch.rand(V, generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))).argmax() for r in x])
    s["ids"] = torch.where(_ints(g, 0, 19, n) > 0, s["ids"], -1).to(torch.int32)
    s["logits"] = x
    return s
  R = case["requests"]
  s["new"] = _ints(g, 1, case["new"], R) if case["ragged"] else torch.full((R,), case["new"], device="cuda", dtype=torch.int32)
  rows = R * case["new"] + case["spare"]  # room for the most; rows behind the last request's stay empty
  s["rows"], page = rows, case["page"]
  if kind == "attend":
    total = _ints(g, max(case["new"], case["keys"] // 2), case["keys"], R) if case["ragged"] else \
      torch.full((R,), case["keys"], device="cuda", dtype=torch.int32)
    s["cached"] = total - s["new"]
  else:
    s["cached"] = _ints(g, case["cached"] // 2, case["cached"], R)
    total = s["cached"] + s["new"]
  s["wide"] = -(-(case["keys"] if kind == "attend" else case["cached"] + case["new"]) // page)
  s["pages"] = R * s["wide"] + 3
  s["free"] = torch.randperm(s["pages"], generator=g, device="cuda").to(torch.int32)
  kv, hd = case["kv"], case["head"]
  if kind == "put":
    s["filled"] = s["cached"]
    s["old"] = [_rows(g, kv, int(s["cached"].sum()), hd)]
    s["x"] = _rows(g, kv, rows, hd)
  else:
    s["filled"] = total
    s["old"] = [_rows(g, kv, int(total.sum()), hd) for _ in range(case["layers"])]
    s["q"] = [(torch.randn(case["heads"], rows, hd, generator=g, device="cuda") * 0.5 * hd ** -0.5).bfloat16() for _ in range(case["layers"])]
  s["total"] = total
  return s


# ---- the plain forms

def _tables(s):
  """Each request's pages, the free ones in order, for all of its tokens; -1 past them."""
  page = s["case"]["page"]
  held = (s["total"].long() + page - 1) // page
  at = _exclusive(held)[:-1, None] + torch.arange(s["wide"], device="cuda")
  full = torch.arange(s["wide"], device="cuda") < held[:, None]
  return torch.where(full, s["free"].long()[at.clamp(max=s["pages"] - 1)], -1)


def _slots(table, cached, new, rows, page):
  """Where each of `rows` rows goes in a flat cache of pages * page rows, -1 behind the last request's."""
  starts = _exclusive(new)
  row = torch.arange(rows, device="cuda")
  owner = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=new.numel() - 1)
  place = cached.long()[owner] + row - starts[owner]
  real = row < starts[-1]
  slot = table[owner, (place // page).clamp(max=table.shape[1] - 1)] * page + place % page
  return torch.where(real, slot, -1)


def _two(e):
  """2^e in 32 bits, made of the exponent's bits."""
  return (e.to(torch.int32) + 127 << 23).view(torch.float32)


def _scales(x, value):
  """The scale of the last axis: the smallest power of two s with amax <= 7 s, for values with a quarter of 4 to 7 before it."""
  amax = x.abs().amax(-1)
  m, e = torch.frexp(amax)  # 7 = 0.875 * 8
  e = torch.where(amax > 0, torch.where(m <= 0.875, e - 3, e - 2), -100).clamp(-100, 100)
  s = _two(e)
  if not value: return s
  half = s / 2  # the steps between the power of two below and s
  for k in (7, 6, 5): s = torch.where(amax <= 7 * half * k / 4, half * k / 4, s)
  return torch.where(e > -100, s, _two(torch.full_like(e, -100)))


def _codes(x):
  """The 4-bit codes of x by size: 0, 1/2, 1, 3/2, 2, 3, 4, 6, ties to the even code, and the sign above."""
  a = x.abs()
  c = (a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() + (a > 5).int()
  return (c + 8 * (x < 0).int()).to(torch.uint8)


_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _packed(codes): return codes[..., 0::2] | codes[..., 1::2] << 4


def _unpacked(packed):
  grid = torch.tensor(_GRID + tuple(-v for v in _GRID), device="cuda")
  c = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
  return grid[c.int()]


def _stored(x, value):
  """Rows (..., hd) as packed codes and scales (..., 1) or, of keys, (..., hd / 32)."""
  x = x.float()
  if value:
    s = _scales(x, True)[..., None]
    return _packed(_codes(x / s)), s
  x = x.unflatten(-1, (-1, 32))
  s = _scales(x, False)
  return _packed(_codes(x / s[..., None]).flatten(-2)), s


def _restored(codes, scales):
  v = _unpacked(codes)
  return (v.unflatten(-1, (scales.shape[-1], -1)) * scales[..., None]).flatten(-2)


class _Cache:
  """Keys' and values' packed codes and scales by slot: (kv, slots, ..)."""
  def __init__(self, kv, hd, slots):
    self.parts = [(torch.zeros(kv, slots, hd // 2, dtype=torch.uint8, device="cuda"),
                   torch.full((kv, slots, 1 if value else hd // 32), 2.0 ** -100, device="cuda")) for value in (False, True)]

  def put(self, slots, x):
    real = slots >= 0
    to, kv = slots[real], x.shape[0] // 2
    for value, (codes, scales) in enumerate(self.parts):
      c, s = _stored(x[value * kv:(value + 1) * kv, real], bool(value))
      codes[:, to], scales[:, to] = c, s

  def values(self, page):
    both = torch.cat([_restored(*p) for p in self.parts]).bfloat16()  # (2 kv, slots, hd)
    kv2, slots, hd = both.shape
    return both.reshape(kv2, slots // page, page, hd).transpose(0, 1).reshape(-1, page, hd)


def _attend(q, cache, table, starts, lengths, page, window):
  """q (heads, rows, hd) against a cache: (rows, heads * hd)."""
  heads, rows, hd = q.shape
  R, wide = table.shape
  slot = (table.clamp(min=0)[:, :, None] * page + torch.arange(page, device="cuda")).reshape(R, -1)
  keys, values = (_restored(c[:, slot], s[:, slot]).transpose(0, 1) for c, s in cache.parts)  # (R, kv, wide * page, hd)
  kv = keys.shape[1]
  rep = heads // kv
  n = starts[1:] - starts[:-1]
  most = int(n.max())
  i = torch.arange(most, device="cuda")
  row = (starts[:-1, None] + i).clamp(max=rows - 1)
  place = (lengths - n)[:, None] + i
  x = q.float()[:, row].reshape(kv, rep, R, most, hd).permute(2, 0, 1, 3, 4).reshape(R, kv, rep * most, hd)
  score = torch.matmul(x, keys.transpose(-1, -2).contiguous())
  key = torch.arange(wide * page, device="cuda")
  seen = (key <= place[..., None]) & (table >= 0).repeat_interleave(page, 1)[:, None]
  if window: seen &= key > place[..., None] - window
  seen = seen[:, None, None].expand(R, kv, rep, most, wide * page).reshape(score.shape)
  score.masked_fill_(~seen, -math.inf)
  top = score.amax(-1, keepdim=True)
  score = torch.exp_(score.sub_(torch.where(top == -math.inf, 0, top)))
  total = score.sum(-1, keepdim=True)
  o = torch.matmul(score, values.contiguous()) / torch.where(total > 0, total, 1)
  o = o.reshape(R, kv, rep, most, hd).permute(0, 3, 1, 2, 4).reshape(R, most, heads * hd).bfloat16()
  out = torch.zeros(rows, heads * hd, dtype=torch.bfloat16, device="cuda")
  real = i < n[:, None]
  out[row[real]] = o[real]
  return out


def _logprobs(x, ids, t, k):
  """(log probabilities of ids, entropies[, the k likeliest tokens' log probabilities, their columns])."""
  y = x if t is None else torch.where(x > -math.inf, x * t, -math.inf)
  y = y - y.amax(1, keepdim=True)
  e = torch.exp(y)
  total = e.sum(1)
  lse = torch.log(total)
  entropy = lse - torch.where(e > 0, e * y, 0).sum(1) / total
  given = y.gather(1, ids.long().clamp(min=0)[:, None])[:, 0] - lse
  out = [torch.where(ids >= 0, given, 0).reshape(1, 1, -1), entropy.reshape(1, 1, -1)]
  if not k: return out
  bits = (x + 0.0).view(torch.int32).long()  # (-0 + 0 is 0)
  order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)  # as the values are ordered
  key = order << 32 | 0x7FFFFFFF - torch.arange(x.shape[1], device="cuda")  # unique, the lowest column first among equals
  at = key.topk(k, 1, largest=True, sorted=True)[1]
  return out + [(y.gather(1, at) - lse[:, None])[None], at.to(torch.int32)[None]]


# ---- tensors between torch and the runtime

_rt = None


def _runtime():
  from baretile_amd.runtime import Runtime
  global _rt
  if _rt is None or _rt.closed: _rt = Runtime()
  return _rt


def _tensor(t):
  """A torch tensor of up to three dimensions as a Tensor, copied on the device."""
  from baretile_amd.tensor import Tensor
  rt, t = _runtime(), t.contiguous()
  shape = (1,) * (3 - t.dim()) + tuple(t.shape)
  out = Tensor(rt, shape[1], shape[2], batch=shape[0], dtype={torch.bfloat16: "bf16", torch.float32: "fp32", torch.int32: "int32"}[t.dtype])
  torch.cuda.synchronize()
  rt.copy(out.addr, t.data_ptr(), t.numel() * t.element_size())
  rt.wait()
  return out


class _Shared:
  """A realized, contiguous Tensor's memory for torch to read in place; it keeps the tensor."""
  KINDS = {"bf16": "<i2", "fp32": "<f4", "int32": "<i4"}

  def __init__(self, t):
    self.tensor = t
    self.__cuda_array_interface__ = {"shape": t.shape, "typestr": self.KINDS[t.dtype], "data": (t.addr, False), "version": 2}


def _torch(t):
  v = torch.as_tensor(_Shared(t), device="cuda")
  return v.view(torch.bfloat16) if t.dtype == "bf16" else v


def _replayed(fn):
  """fn, run once, then recorded: the recording and what it writes, as torch tensors."""
  from baretile_amd.tensor import Recording
  rt = _runtime()
  fn()
  rt.wait()
  rec = Recording(rt)
  with rec: out = fn()
  return rec, [_torch(t) for t in out]


def _prepare_own(s):
  """The framework's tensors for the inputs: caches filled, the step's plan, or its recording."""
  from baretile_amd.models import serve
  from baretile_amd.pages import Pages
  case, rt, kind, o = s["case"], _runtime(), s["case"]["kind"], {"case": s["case"]}
  row = lambda t: _tensor(t.to(torch.int32).reshape(1, -1))
  if kind == "logprobs":
    rows, x, ids, t, k = case["rows"], _tensor(s["logits"]), row(s["ids"]), _tensor(s["t"]) if s["t"] is not None else None, case["k"]
    step = lambda: serve.logprobs(x, ids, k=k, t=t)
    o["keep"] = (x, ids, t)
  else:
    page, rows = case["page"], s["rows"]
    cached, new, free = row(s["cached"]), row(s["new"]), row(s["free"])
    pools = [Pages(rt, s["pages"], case["kv"], case["head"], page, bits=4) for _ in s["old"]]
    table = _tensor(_tables(s).to(torch.int32))  # every page the step needs is its request's already
    filled = int(s["filled"].sum())
    if filled:  # (a plan takes a row at least)
      first = pools[0].plan(table, row(torch.zeros_like(s["cached"])), row(s["filled"]), free, filled)
      for pool, x in zip(pools, s["old"]): pool.put(first, _tensor(x))
    batch = pools[0].plan(table, cached, new, free, rows, most=case["new"])
    if kind == "put":
      x = _tensor(s["x"])
      def step():
        pools[0].put(batch, x)
        return [pools[0].values()]
    else:
      qs = [_tensor(q) for q in s["q"]]
      def step(): return [pool.attend(q, batch, window=case["window"], merged=True) for pool, q in zip(pools, qs)]
    o["keep"] = (pools, table, batch, cached, new, free, step)  # (step: its queries or rows)
  rt.wait()
  if rows <= 512: o["rec"], o["out"] = _replayed(step)
  else: o["step"] = step
  return o


def prepare(case, seed):
  s = _inputs(case, seed)
  if own: s = _prepare_own(s)
  elif case["kind"] != "logprobs":
    page, table = case["page"], _tables(s)
    filled = int(s["filled"].sum())
    at = _slots(table, torch.zeros_like(s["filled"]), s["filled"], filled, page)
    s["caches"] = []
    for x in s["old"]:
      cache = _Cache(case["kv"], case["head"], s["pages"] * page)
      cache.put(at, x)
      s["caches"].append(cache)
    s["table"], s["starts"], s["lengths"] = table, _exclusive(s["new"]), s["total"].long()
    s["slots"] = _slots(table, s["cached"], s["new"], s["rows"], page)
    del s["old"]
  torch.cuda.synchronize()
  return s


def run(s):
  if own:
    if "step" in s: return [_torch(t) for t in s["step"]()]
    s["rec"].send()
    return s["out"]
  case, kind = s["case"], s["case"]["kind"]
  if kind == "logprobs": return _logprobs(s["logits"], s["ids"], s["t"], case["k"])
  if kind == "put":
    s["caches"][0].put(s["slots"], s["x"])
    return [s["caches"][0].values(case["page"])]
  return [_attend(q, c, s["table"], s["starts"], s["lengths"], case["page"], case["window"])[None] for q, c in zip(s["q"], s["caches"])]


# ---- what a pass cannot do without

def work(case):
  kind = case["kind"]
  if kind == "logprobs":
    return {"bytes": 4.0 * case["rows"] * (case["vocab"] + 4 + 2 * case["k"]), "flops": 0}
  R = case["requests"]
  rows = R * (case["new"] + 1) / 2 if case["ragged"] else R * case["new"]
  values = 2 * case["kv"] * case["head"]  # of a token
  held = case["kv"] * (case["head"] + case["head"] // 32 + 2)  # its bytes: codes, a scale for 32 dims of a key and for a value
  if kind == "put":
    pages = R * -(-(case["cached"] + case["new"]) // case["page"]) + 3
    return {"bytes": rows * (2.0 * values + held) + pages * case["page"] * (2.0 * values + held), "flops": 0}
  n = case["new"] if not case["ragged"] else (case["new"] + 1) / 2
  keys = case["keys"] * 0.75 if case["ragged"] else case["keys"]
  pairs, seen = n * (keys - (n - 1) / 2), keys
  if case["window"]:
    w = min(case["window"], keys)
    pairs, seen = min(pairs, n * w), min(keys, w + n)
  heads = case["heads"] * case["head"]
  return {"bytes": case["layers"] * (R * seen * held + 4.0 * rows * heads), "flops": case["layers"] * 4.0 * R * pairs * heads}


# ---- the same in 64 bits

def _nearest(v, s):
  """v on the grid of 4-bit floats times s: the nearest of its list, of two as near the one of even place."""
  grid = torch.tensor(_GRID, dtype=torch.float64, device="cuda")
  a = (v / s).abs().contiguous()
  hi = torch.searchsorted(grid, a).clamp(max=7)
  lo = (hi - 1).clamp(min=0)
  up, down = (grid[hi] - a).abs(), (a - grid[lo]).abs()
  pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
  return torch.sign(v) * grid[pick] * s


def _held64(x, value):
  """What a cache holds of rows x (.., n, hd)."""
  x = x.double()
  e = torch.arange(-100, 101, device="cuda")
  scales = (e + 1023 << 52).view(torch.float64)
  if value: scales = torch.cat([(scales[:-1, None] * torch.tensor([1.0, 1.25, 1.5, 1.75], dtype=torch.float64, device="cuda")).flatten(), scales[-1:]])
  groups = x if value else x.unflatten(-1, (-1, 32))
  s = scales[torch.searchsorted(7 * scales, groups.abs().amax(-1)).clamp(max=scales.numel() - 1)][..., None]
  return _nearest(groups, s).reshape(x.shape)


def exact(case, seed):
  s, kind = _inputs(case, seed), case["kind"]
  if kind == "logprobs":
    given, entropy, values, labels = [], [], [], []
    for r, x in enumerate(s["logits"]):
      x = x.double()
      if s["t"] is not None: x = x * s["t"][r].double()
      p = torch.log_softmax(x, 0)
      given.append(p[s["ids"][r]] if s["ids"][r] >= 0 else p[0] * 0)
      entropy.append(torch.special.entr(p.exp()).sum())
      if case["k"]: values.append(p.topk(case["k"])[0])
    out = [torch.stack(given).reshape(1, 1, -1), torch.stack(entropy).reshape(1, 1, -1)]
    return out + ([torch.stack(values)[None], None] if case["k"] else [])
  page, kv, hd = case["page"], case["kv"], case["head"]
  cached, new, total = s["cached"].tolist(), s["new"].tolist(), s["total"].tolist()
  hold = lambda x: torch.cat([_held64(x[:kv], False), _held64(x[kv:], True)])
  if kind == "put":
    out = torch.zeros(s["pages"], 2 * kv, page, hd, dtype=torch.float64, device="cuda")
    free, taken, old, fresh = s["free"].tolist(), 0, 0, 0
    for c, n in zip(cached, new):
      rows = hold(torch.cat([s["old"][0][:, old:old + c], s["x"][:, fresh:fresh + n]], 1))
      old, fresh = old + c, fresh + n
      for at in range(0, c + n, page):
        part = rows[:, at:at + page]
        out[free[taken], :, :part.shape[1]] = part
        taken += 1
    return [out.reshape(-1, page, hd)]
  outs = []
  for q, x in zip(s["q"], s["old"]):
    out = torch.zeros(1, s["rows"], case["heads"], hd, dtype=torch.float64, device="cuda")
    row, at, rep = 0, 0, case["heads"] // kv
    for r, n in enumerate(new):
      v = hold(x[:, at:at + total[r]])
      key, place = torch.arange(total[r], device="cuda"), torch.arange(cached[r], cached[r] + n, device="cuda")[:, None]
      hidden = key > place
      if case["window"]: hidden |= key <= place - case["window"]
      for h in range(case["heads"]):
        score = (q[h, row:row + n].double() @ v[h // rep].T).masked_fill_(hidden, -math.inf)
        out[0, row:row + n, h] = score.softmax(-1) @ v[kv + h // rep]
      row, at = row + n, at + total[r]
    outs.append(out.reshape(1, s["rows"], -1))
  return outs
