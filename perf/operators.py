"""The operators of a serving step over a paged 8-bit cache, as cases to time and to compare.

Kinds:
  plan    a step's block tables, row starts, places and slots from request lengths (Pages.plan);
  put     the step's keys and values into their pages, rounded to 8 bits under a power of two for each page and head
          (Pages.put), and the cache's values read back (Pages.values);
  attend  attention over the pages, one row a request, several (drafts) or a prompt's (Pages.attend), for the caches of
          one or more layers;
  verify  drafted tokens against the target's probabilities, from given random numbers (serve.verify).

Steps of few rows are recorded and replayed, as a serving loop runs them; prompts run eagerly. Head counts and widths are
the ones of models.llama.smol and of the benchmark's large block.
"""
import math

import torch

own = False

LARGE = {"heads": 32, "kv": 8, "head": 128}
SMOL = {"heads": 9, "kv": 3, "head": 64}


def listed():
  return [
    # a decode step's tables: 32 streams, one new token each, every page's boundary crossed by some
    {"name": "plan_32", "kind": "plan", "requests": 32, "new": 1, "ragged": False, "cached": 4000, "page": 64, "spare": 0},
    # a busy step: many streams with drafts and chunks of prompts, small pages, rows left over
    {"name": "plan_512", "kind": "plan", "requests": 512, "new": 33, "ragged": True, "cached": 2000, "page": 16, "spare": 100},
    # a decode step's rows into a small cache
    {"name": "put_decode", "kind": "put", **LARGE, "requests": 32, "new": 1, "ragged": False, "cached": 128, "page": 64, "spare": 0},
    # chunks of prompts behind cached rows: pages begun, ended and filled whole
    {"name": "put_prompts", "kind": "put", **LARGE, "requests": 3, "new": 1000, "ragged": True, "cached": 500, "page": 64, "spare": 7},
    # a chat's next token on the small model, 8 layers' caches one after another
    {"name": "attend_token", "kind": "attend", **SMOL, "requests": 1, "new": 1, "ragged": False, "keys": 301, "page": 16,
     "layers": 8, "window": 0, "spare": 0},
    # a batch of streams of uneven lengths, two layers
    {"name": "attend_decode_8", "kind": "attend", **LARGE, "requests": 8, "new": 1, "ragged": True, "keys": 8191, "page": 64,
     "layers": 2, "window": 0, "spare": 0},
    # a large batch, 4096 cached rows each
    {"name": "attend_decode_32", "kind": "attend", **LARGE, "requests": 32, "new": 1, "ragged": False, "keys": 4096, "page": 64,
     "layers": 1, "window": 0, "spare": 0},
    # four drafts a stream and the token before them, four layers
    {"name": "attend_drafts", "kind": "attend", **LARGE, "requests": 16, "new": 5, "ragged": True, "keys": 2048, "page": 32,
     "layers": 4, "window": 0, "spare": 3},
    # one stream's long context
    {"name": "attend_long", "kind": "attend", **LARGE, "requests": 1, "new": 1, "ragged": False, "keys": 65536, "page": 128,
     "layers": 1, "window": 0, "spare": 0},
    # two prompts' chunks behind cached rows
    {"name": "attend_prompts", "kind": "attend", **LARGE, "requests": 2, "new": 2048, "ragged": True, "keys": 2560, "page": 64,
     "layers": 1, "window": 0, "spare": 0},
    # one stream's four drafts on the small model's vocabulary
    {"name": "verify_1", "kind": "verify", "requests": 1, "new": 5, "ragged": False, "vocab": 49152, "drawn": True, "masked": 0.0, "spare": 0},
    # a batch of streams with up to five drafts each, part of the vocabulary masked
    {"name": "verify_32", "kind": "verify", "requests": 32, "new": 6, "ragged": True, "vocab": 131072, "drawn": True, "masked": 0.1, "spare": 2},
  ]


def _log_int(rng, lo, hi):
  """An integer from lo to hi, spread over its logarithm."""
  return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
  kind = rng.choice(("plan", "put", "attend", "attend", "attend", "verify"))
  page, spare = rng.choice((16, 32, 64, 128)), rng.choice((0, rng.randint(1, 40)))
  if kind == "plan":
    return {"kind": "plan", "requests": _log_int(rng, 1, 1024), "new": _log_int(rng, 1, 64), "ragged": rng.random() < 0.5,
            "cached": _log_int(rng, 1, 4000), "page": page, "spare": spare}
  kv, rep, hd = rng.choice(((8, 4, 128), (3, 3, 64), (8, 8, 128), (4, 7, 64), (8, 1, 64), (2, 4, 128)))
  shape = {"heads": kv * rep, "kv": kv, "head": hd}
  if kind == "put":
    if rng.random() < 0.5:
      return {"kind": "put", **shape, "requests": _log_int(rng, 1, 64), "new": _log_int(rng, 1, 8), "ragged": rng.random() < 0.5,
              "cached": _log_int(rng, 1, 200), "page": page, "spare": spare}
    return {"kind": "put", **shape, "requests": rng.randint(1, 4), "new": _log_int(rng, 9, 1024), "ragged": rng.random() < 0.5,
            "cached": _log_int(rng, 1, 600), "page": page, "spare": spare}
  if kind == "verify":
    return {"kind": "verify", "requests": _log_int(rng, 1, 32), "new": rng.randint(1, 6), "ragged": rng.random() < 0.5,
            "vocab": _log_int(rng, 1000, 131072), "drawn": rng.random() < 0.7, "masked": rng.choice((0.0, 0.1, 0.9)), "spare": rng.randint(0, 3)}
  if rng.random() < 0.7:
    requests, keys, new = _log_int(rng, 1, 32), _log_int(rng, 16, 16384), rng.choice((1, 1, rng.randint(2, 9)))
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
  g, s = _generator(seed), {"case": case}
  R, kind = case["requests"], case["kind"]
  s["new"] = _ints(g, 1, case["new"], R) if case["ragged"] else torch.full((R,), case["new"], device="cuda", dtype=torch.int32)
  rows = R * case["new"] + case["spare"]  # room for the most; rows behind the last request's stay empty
  s["rows"] = rows
  if kind == "verify":
    V = case["vocab"]
    logits = 3 * torch.randn(rows, V, generator=g, device="cuda")
    if case["masked"]:
      logits.masked_fill_(torch.rand(rows, V, generator=g, device="cuda") < case["masked"], -math.inf)
    s["t"] = 0.7 + torch.rand(rows, 1, generator=g, device="cuda")
    near = torch.cat([logits[:1], logits[:-1]]) + 0.7 * torch.randn(rows, V, generator=g, device="cuda")
    near = torch.softmax(near * torch.cat([s["t"][:1], s["t"][:-1]]), 1)
    s["ids"] = torch.multinomial(near, 1, generator=g)[:, 0].to(torch.int32)
    s["logits"], s["probs"] = logits, near if case["drawn"] else None
    s["uniforms"] = torch.rand(2, rows, generator=g, device="cuda")
    s["starts"] = _exclusive(s["new"]).to(torch.int32)
    return s
  page = case["page"]
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
  kv, hd = case.get("kv"), case.get("head")
  if kind == "put":
    s["filled"] = s["cached"]
    s["old"] = [_rows(g, kv, int(s["cached"].sum()), hd)]
    s["x"] = _rows(g, kv, rows, hd)
  elif kind == "attend":
    s["filled"] = total
    s["old"] = [_rows(g, kv, int(total.sum()), hd) for _ in range(case["layers"])]
    s["q"] = [(torch.randn(case["heads"], rows, hd, generator=g, device="cuda") * 0.5 * hd ** -0.5).bfloat16() for _ in range(case["layers"])]
  else:
    s["filled"] = s["cached"]
  s["taken"] = ((s["filled"] + page - 1) // page).sum().to(torch.int32).reshape(1)
  return s


# ---- the plain forms

def _table(s, filled, wide, page):
  """Tables that hold `filled` rows of each request: the free pages in order, -1 past them."""
  held = (filled.long() + page - 1) // page
  at = _exclusive(held)[:-1, None] + torch.arange(wide, device="cuda")
  full = torch.arange(wide, device="cuda") < held[:, None]
  return torch.where(full, s["free"].long()[at.clamp(max=s["pages"] - 1)], -1)


def _plan(table, cached, new, free, taken, rows, page):
  """(tables, starts, lengths, places, slots, taken) of a step, whole numbers of 64 bits. A table's entries are kept up to
  the first that holds no page; those after it up to the request's new length are taken from the free pages in order."""
  wide = table.shape[1]
  cached, new = cached.long().clamp(0, wide * page), new.long().clamp(0, rows)
  starts = _exclusive(new).clamp(max=rows)
  new = starts[1:] - starts[:-1]
  lengths = cached + new
  entry = torch.arange(wide, device="cuda")
  first, last = (cached + page - 1) // page, (lengths + page - 1) // page
  touched = (entry >= first[:, None]) & (entry < last[:, None])
  empty = touched & (table < 0)
  taking = touched & (torch.cumsum(empty, 1) > 0)
  order = torch.cumsum(taking.reshape(-1), 0).reshape(taking.shape) - 1 + taken.long()
  got = torch.where(order < free.numel(), free.long()[order.clamp(0, free.numel() - 1)], -1)
  table = torch.where(taking, got, table)
  row = torch.arange(rows, device="cuda")
  owner = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=new.numel() - 1)
  real = row < starts[-1]
  place = cached[owner] + row - starts[owner]
  on = place // page
  held = torch.where(on < wide, table[owner, on.clamp(max=wide - 1)], -1)
  slots = torch.where(real & (held >= 0), held * page + place % page, -1)
  return table, starts, lengths, torch.where(real, place, -1), slots, taken.long() + taking.sum()


def _two(e):
  """2^e in 32 bits, made of the exponent's bits."""
  return (e.to(torch.int32) + 127 << 23).view(torch.float32)


def _powers(amax):
  """The smallest power of two s with amax <= 448 s, from 2^-100 to 2^119."""
  m, e = torch.frexp(amax)
  e = torch.where(m <= 0.875, e - 9, e - 8)
  return _two(torch.where(amax > 0, e, -100).clamp(-100, 119))


def _e4m3(x):
  """The nearest values of 4 exponent and 3 mantissa bits, ties to even, at most 448 in size."""
  _, e = torch.frexp(x)
  step = _two((e - 1).clamp(min=-6) - 3)
  return (torch.round(x / step) * step).clamp(-448, 448)


def _put(codes, scales, table, cached, new, x, page):
  """x (2 kv, rows, hd) into codes (pages, 2 kv, page, hd), 8-bit floats, under scales (pages, 2 kv): in place."""
  starts = _exclusive(new)
  most = int(((cached + new + page - 1) // page - cached // page).max())
  R, wide = table.shape
  entry = cached.long()[:, None] // page + torch.arange(most, device="cuda")
  ids = torch.where(entry < wide, table.gather(1, entry.clamp(max=wide - 1)), -1)
  place = entry[:, :, None] * page + torch.arange(page, device="cuda")
  fresh = (place >= cached[:, None, None]) & (place < (cached + new)[:, None, None])
  touched = fresh.any(2) & (ids >= 0)
  ids, place, fresh = ids[touched], place[touched], fresh[touched]
  owner = torch.arange(R, device="cuda")[:, None].expand(R, most)[touched]
  row = (starts[:-1][owner] - cached[owner])[:, None] + place
  rows = x.float()[:, row.clamp(0, x.shape[1] - 1)].transpose(0, 1)  # (touched, 2 kv, page, hd)
  fresh = fresh[:, None, :, None]
  amax = torch.where(fresh, rows.abs(), 0).amax((2, 3))
  begun = (place[:, 0] < cached[owner])[:, None]
  old = scales[ids]
  scale = torch.maximum(_powers(amax), torch.where(begun, old, 0))
  kept = codes[ids].float() * (old / scale)[:, :, None, None]
  mixed = _e4m3(torch.where(fresh, rows / scale[:, :, None, None], torch.where(begun[:, :, None, None], kept, codes[ids].float())))
  codes.view(torch.uint8)[ids] = mixed.to(torch.float8_e4m3fn).view(torch.uint8)
  scales[ids] = scale


def _values(codes, scales):
  v = codes.float() * scales[:, :, None, None]
  return v.bfloat16().reshape(-1, *codes.shape[2:])


def _attend(q, codes, scales, table, starts, lengths, page, window):
  """q (layers, heads, rows, hd) against codes (layers, pages, 2 kv, page, hd): (layers, rows, heads * hd)."""
  L, heads, rows, hd = q.shape
  R, wide = table.shape
  kv = codes.shape[2] // 2
  rep, ids = heads // kv, table.clamp(min=0)
  kept = codes.view(torch.uint8)[:, ids].view(torch.float8_e4m3fn).float() * scales[:, ids][..., None, None]
  kept = kept.permute(0, 1, 3, 2, 4, 5).reshape(L, R, 2 * kv, wide * page, hd)
  n = starts[1:] - starts[:-1]
  most = int(n.max())
  i = torch.arange(most, device="cuda")
  row = (starts[:-1, None] + i).clamp(max=rows - 1)
  place = (lengths - n)[:, None] + i
  x = q.float()[:, :, row].reshape(L, kv, rep, R, most, hd).permute(0, 3, 1, 2, 4, 5).reshape(L, R, kv, rep * most, hd)
  score = torch.matmul(x, kept[:, :, :kv].transpose(-1, -2))
  key = torch.arange(wide * page, device="cuda")
  seen = (key <= place[..., None]) & (table >= 0).repeat_interleave(page, 1)[:, None]
  if window: seen &= key > place[..., None] - window
  seen = seen[None, :, None, None].expand(L, R, kv, rep, most, wide * page).reshape(score.shape)
  score.masked_fill_(~seen, -math.inf)
  top = score.amax(-1, keepdim=True)
  score = torch.exp_(score.sub_(torch.where(top == -math.inf, 0, top)))
  total = score.sum(-1, keepdim=True)
  o = torch.matmul(score, kept[:, :, kv:]) / torch.where(total > 0, total, 1)
  o = o.reshape(L, R, kv, rep, most, hd).permute(0, 1, 4, 2, 3, 5).reshape(L, R, most, heads * hd).bfloat16()
  out = torch.zeros(L, rows, heads * hd, dtype=torch.bfloat16, device="cuda")
  real = i < n[:, None]
  out[:, row[real]] = o[:, real]
  return out


def _verify(logits, ids, starts, uniforms, probs, t):
  """(tokens, counts): each request's accepted drafts, then the token drawn where the first was refused, or after the last."""
  rows, V = logits.shape
  starts, ids = starts.long(), ids.long()
  p = torch.softmax(t.double() * logits.double(), 1)
  n = starts[1:] - starts[:-1]
  most = int(n.max())
  row = torch.arange(rows, device="cuda")
  mine = p[(row - 1).clamp(min=0), ids]
  theirs = probs.double()[row, ids] if probs is not None else torch.ones_like(mine)
  taken = uniforms[0].double() * theirs < mine
  i = torch.arange(1, most + 1, device="cuda")
  run = torch.where(i < n[:, None], taken[(starts[:-1, None] + i).clamp(max=rows - 1)], False)
  accepted = torch.cumprod(run.long(), 1).sum(1)
  at = starts[:-1] + accepted
  refused = accepted < n - 1
  after = (at + 1).clamp(max=rows - 1)
  if probs is not None: less = probs.double()[after]
  else: less = torch.nn.functional.one_hot(ids[after], V) * p[at]
  left = torch.where(refused[:, None], (p[at] - less).clamp(min=0), p[at])
  left = torch.where(left.sum(1, keepdim=True) > 0, left, p[at])
  upto = torch.cumsum(left, 1)
  drawn = (upto <= uniforms[1].double()[at, None] * upto[:, -1:]).sum(1).clamp(max=V - 1)
  tokens = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
  j = torch.arange(most, device="cuda")
  keep = j < accepted[:, None]
  tokens[(starts[:-1, None] + j)[keep]] = ids[(starts[:-1, None] + j + 1).clamp(max=rows - 1)[keep]]
  tokens[at] = drawn
  return tokens.to(torch.int32).reshape(1, 1, -1), (accepted + 1).to(torch.int32).reshape(1, 1, -1)


def _filled(s, x):
  """A cache of its own with x's rows in it: (codes, scales)."""
  case = s["case"]
  kv, hd, page = case["kv"], case["head"], case["page"]
  codes = torch.zeros(s["pages"], 2 * kv, page, hd, dtype=torch.float8_e4m3fn, device="cuda")
  scales = torch.full((s["pages"], 2 * kv), 2.0 ** -100, device="cuda")
  _put(codes, scales, s["base"], torch.zeros_like(s["filled"]), s["filled"], x, page)
  return codes, scales


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
  if kind == "verify":
    args = [_tensor(s["logits"]), row(s["ids"]), row(s["starts"]), _tensor(s["uniforms"])]
    probs, t = _tensor(s["probs"]) if s["probs"] is not None else None, _tensor(s["t"])
    o["rec"], o["out"] = _replayed(lambda: serve.verify(*args, probs=probs, t=t))
    o["keep"] = (args, probs, t)
    return o
  page, rows = case["page"], s["rows"]
  cached, new, free, taken = row(s["cached"]), row(s["new"]), row(s["free"]), row(s["taken"])
  if kind == "plan":
    pool, base = Pages(rt, s["pages"], 1, 64, page), _tensor(s["base"].to(torch.int32))
    table = _tensor(s["base"].to(torch.int32))
    def plan():
      table.assign(base)
      b = pool.plan(table, cached, new, free, rows, taken=taken)
      return [table, b.starts, b.lengths, b.places, b.slots, b.taken]
    o["rec"], o["out"] = _replayed(plan)
    o["keep"] = (pool, table, base, cached, new, free, taken)
    return o
  pools = [Pages(rt, s["pages"], case["kv"], case["head"], page) for _ in s["old"]]
  table = _tensor(torch.full_like(s["base"], -1).to(torch.int32))
  filled = int(s["filled"].sum())
  if filled:  # (a plan takes a row at least)
    first = pools[0].plan(table, row(torch.zeros_like(s["cached"])), row(s["filled"]), free, filled)
    for pool, x in zip(pools, s["old"]): pool.put(first, _tensor(x))
  batch = pools[0].plan(table, cached, new, free, rows, taken=taken, most=case["new"])
  if kind == "put":
    x = _tensor(s["x"])
    def step():
      pools[0].put(batch, x)
      return [pools[0].values()]
  else:
    qs = [_tensor(q) for q in s["q"]]
    def step(): return [pool.attend(q, batch, window=case["window"], merged=True) for pool, q in zip(pools, qs)]
  o["keep"] = (pools, table, batch, cached, new, free, taken, step)  # (step: its queries or rows)
  rt.wait()
  if rows <= 512: o["rec"], o["out"] = _replayed(step)
  else: o["step"] = step
  return o


def prepare(case, seed):
  s = _inputs(case, seed)
  if case["kind"] != "verify": s["base"] = _table(s, s["filled"], s["wide"], case["page"])
  if own: s = _prepare_own(s)
  elif case["kind"] in ("put", "attend"):
    pools = [_filled(s, x) for x in s["old"]]
    s["codes"], s["scales"] = torch.stack([c.view(torch.uint8) for c, _ in pools]).view(torch.float8_e4m3fn), torch.stack([c for _, c in pools])
    s["table"], s["starts"], s["lengths"] = _plan(s["base"], s["cached"], s["new"], s["free"], s["taken"], s["rows"], case["page"])[:3]
    if case["kind"] == "attend": s["q"] = torch.stack(s["q"])
    del s["old"]
  torch.cuda.synchronize()
  return s


def run(s):
  if own:
    if "step" in s: return [_torch(t) for t in s["step"]()]
    s["rec"].send()
    return s["out"]
  case = s["case"]
  kind, page = case["kind"], case.get("page")
  if kind == "plan":
    out = _plan(s["base"], s["cached"], s["new"], s["free"], s["taken"], s["rows"], page)
    return [out[0].to(torch.int32)[None], *(t.to(torch.int32).reshape(1, 1, -1) for t in out[1:])]
  if kind == "put":
    _put(s["codes"][0], s["scales"][0], s["table"], s["cached"], s["new"], s["x"], page)
    return [_values(s["codes"][0], s["scales"][0])]
  if kind == "attend":
    return [t[None] for t in _attend(s["q"], s["codes"], s["scales"], s["table"], s["starts"], s["lengths"], page, case["window"])]
  return list(_verify(s["logits"], s["ids"], s["starts"], s["uniforms"], s["probs"], s["t"]))


# ---- what a pass cannot do without

def work(case):
  kind, R = case["kind"], case["requests"]
  rows = R * (case["new"] + 1) / 2 if case["ragged"] else R * case["new"]
  if kind == "plan":
    wide = -(-(case["cached"] + case["new"]) // case["page"])
    return {"bytes": 4.0 * (2 * R * wide + 4 * R + 2 * (R * case["new"] + case["spare"])), "flops": 0}
  if kind == "verify":
    V = case["vocab"]
    return {"bytes": 4.0 * V * (rows + (R if case["drawn"] else 0)), "flops": 0}
  values = 2 * case["kv"] * case["head"]
  if kind == "put":
    pages = R * -(-(case["cached"] + case["new"]) // case["page"]) + 3
    return {"bytes": values * (2.0 * rows + 3 * pages * case["page"]), "flops": 0}
  n = case["new"] if not case["ragged"] else (case["new"] + 1) / 2
  keys = case["keys"] * 0.75 if case["ragged"] else case["keys"]
  pairs, seen = n * (keys - (n - 1) / 2), keys
  if case["window"]:
    w = min(case["window"], keys)
    pairs, seen = min(pairs, n * w), min(keys, w + n)
  heads = case["heads"] * case["head"]
  return {"bytes": case["layers"] * (R * seen * values + 4.0 * rows * heads), "flops": case["layers"] * 4.0 * R * pairs * heads}


# ---- the same in 64 bits

def _two64(e): return (e + 1023 << 52).view(torch.float64)


def _grid(v, s):
  """v / s on the grid of 8-bit floats, times s: by the grid's own list of magnitudes."""
  m = torch.arange(127, device="cuda")
  list64 = torch.where(m < 8, m.double() * 2.0 ** -9, (8 + m % 8).double() * _two64(m // 8 - 10))
  a = (v / s).abs().clamp(max=448.0)
  hi = torch.searchsorted(list64, a.contiguous()).clamp(max=126)
  lo = (hi - 1).clamp(min=0)
  up, down = list64[hi] - a, a - list64[lo]
  pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
  return torch.sign(v) * list64[pick] * s


def _scale64(amax):
  powers = _two64(torch.arange(-100, 120, device="cuda"))
  return powers[torch.searchsorted(448.0 * powers, amax).clamp(max=219)]


def exact(case, seed):
  s, kind = _inputs(case, seed), case["kind"]
  if kind in ("plan", "verify"): return None
  page, kv, hd = case["page"], case["kv"], case["head"]
  held, free = ((s["filled"] + page - 1) // page).tolist(), s["free"].tolist()
  tables, at = [], 0
  for n in held:
    tables.append(free[at:at + n])
    at += n
  filled, cached, new = s["filled"].tolist(), s["cached"].tolist(), s["new"].tolist()

  def paged(x):  # one layer's cache, by request and page
    pool, top = {}, {}
    at = 0
    for r, n in enumerate(filled):
      for k, p in enumerate(tables[r]):
        part = x[:, at + k * page:at + min((k + 1) * page, n)].double()
        top[p] = _scale64(part.abs().amax((1, 2), keepdim=True))
        pool[p] = _grid(part, top[p])
      at += n
    return pool, top
  if kind == "put":
    pool, top = paged(s["old"][0])
    row = 0
    for r, n in enumerate(new):
      k = cached[r] // page
      done = 0
      while done < n:
        here = (cached[r] + done) % page
        m = min(n - done, page - here)
        part = s["x"][:, row + done:row + done + m].double()
        scale = _scale64(part.abs().amax((1, 2), keepdim=True))
        if k == len(tables[r]):
          tables[r].append(free[at])
          at += 1
        p = tables[r][k]
        if here:
          scale = torch.maximum(scale, top[p])
          part = torch.cat([_grid(pool[p], scale), _grid(part, scale)], 1)
        else: part = _grid(part, scale)
        pool[p], done, k = part, done + m, k + 1
      row += n
    out = torch.zeros(s["pages"], 2 * kv, page, hd, dtype=torch.float64, device="cuda")
    for p, v in pool.items(): out[p, :, :v.shape[1]] = v
    return [out.reshape(-1, page, hd)]
  outs = []
  for q, x in zip(s["q"], s["old"]):
    pool, _ = paged(x)
    out = torch.zeros(1, s["rows"], case["heads"], hd, dtype=torch.float64, device="cuda")
    row, rep = 0, case["heads"] // kv
    for r, n in enumerate(new):
      v = torch.cat([pool[p] for p in tables[r]], 1)
      key, place = torch.arange(v.shape[1], device="cuda"), torch.arange(cached[r], cached[r] + n, device="cuda")[:, None]
      hidden = key > place
      if case["window"]: hidden |= key <= place - case["window"]
      for h in range(case["heads"]):
        score = (q[h, row:row + n].double() @ v[h // rep].T).masked_fill_(hidden, -math.inf)
        out[0, row:row + n, h] = score.softmax(-1) @ v[kv + h // rep]
      row += n
    outs.append(out.reshape(1, s["rows"], -1))
  return outs
