"""Paged caches of 8 and 4 bits and drafted tokens' verification in NumPy, in 64 bits and whole numbers, request by request: what
bt_pages_plan, bt_pages_put, bt_pages4_put, bt_pages_attend and bt_verify (include/baretile_amd.h) define."""
import numpy as np

LEAST, LARGEST = -100, 119  # exponents of the scales


def plan(tables, cached, new, free, rows, page, pages, taken=0, most=None):
  """(tables, starts, lengths, places, slots, taken) as Pages.plan gives them."""
  tables = np.array(tables)
  width = tables.shape[1]
  most = rows if most is None else min(most, rows)
  starts, lengths, places, slots = [0], [], np.full(rows, -1), np.full(rows, -1)
  real = lambda p: 0 <= p < pages
  for r, (c, n) in enumerate(zip(cached, new)):
    c, n = min(max(int(c), 0), width * page), min(max(int(n), 0), most, rows - starts[-1])
    k, end = -(-c // page), min(-(-(c + n) // page), width)
    while k < end and real(tables[r, k]): k += 1
    for k in range(k, end):
      tables[r, k] = free[taken] if 0 <= taken < len(free) and real(free[taken]) else -1
      taken += 1
    for i in range(n):
      place = c + i
      places[starts[-1] + i] = place
      if place // page < width and real(tables[r, place // page]):
        slots[starts[-1] + i] = tables[r, place // page] * page + place % page
    starts.append(starts[-1] + n)
    lengths.append(c + n)
  return tables, np.array(starts), np.array(lengths), places, slots, taken


def grid(x):
  """The nearest 8-bit floats (4 exponent and 3 mantissa bits), ties to even, at most 448 in size."""
  x = np.asarray(x, np.float64)
  with np.errstate(invalid="ignore"): x = np.where(np.isfinite(x), x, np.copysign(448.0, x))
  x = np.clip(x, -448.0, 448.0)
  step = np.exp2(np.maximum(np.frexp(x)[1] - 1, -6) - 3.0)
  return np.rint(x / step) * step


def scale(x):
  """The smallest power of two s with every finite |x| <= 448 s, over the last two axes."""
  top = np.where(np.isfinite(x), np.abs(x), 0).max((-2, -1))
  m, e = np.frexp(top)
  return np.exp2(np.clip(np.where(top > 0, np.where(m <= 0.875, e - 9, e - 8), LEAST), LEAST, LARGEST).astype(np.float64))


def put(values, scales, tables, starts, lengths, x):
  """x (2 kv, rows, head) into values (pages, 2 kv, page, head) under scales (pages, 2 kv), in place."""
  pages, _, page, _ = values.shape
  for r, length in enumerate(lengths):
    n = starts[r + 1] - starts[r]
    at = length - n
    while at < length:
      k, held = divmod(at, page)
      count = min(length - at, page - held)
      id = tables[r, k] if k < tables.shape[1] else -1
      if 0 <= id < pages:
        part = x[:, starts[r] + at - (length - n):][:, :count].astype(np.float64)
        s = scale(part)
        if held:
          s = np.maximum(s, scales[id])
          if (s != scales[id]).any():
            grown = (s != scales[id])[:, None, None]
            values[id, :, :held] = np.where(grown, grid(values[id, :, :held] / s[:, None, None]) * s[:, None, None],
                                            values[id, :, :held])
        values[id, :, held:held + count] = grid(part / s[:, None, None]) * s[:, None, None]
        scales[id] = s
      at += count


GRID4 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
LEAST4, LARGEST4 = -100, 100  # exponents of the 4-bit cache's scales


def grid4(x):
  """The nearest 4-bit floats (2 exponent bits, 1 mantissa bit), of two as near the one with the even code, at most 6 in size."""
  x = np.asarray(x, np.float64)
  with np.errstate(invalid="ignore"): a = np.minimum(np.where(np.isfinite(x), np.abs(x), 7.0), 7.0)
  far = np.abs(a[..., None] - GRID4)
  near = far == far.min(-1, keepdims=True)
  pick = np.where(near & (np.arange(8) % 2 == 0), np.arange(8), -1).max(-1)  # the even code, where it is among the nearest
  pick = np.where(pick >= 0, pick, np.argmax(near, -1))
  return np.copysign(GRID4[pick], x) + 0.0


def held4(x, value):
  """Rows x (.., n, head) as the 4-bit cache holds them, the smallest scales s with every finite |x| <= 7 s: for a key (value
  false) a power of two for each 32 dims, for a value k / 4 of one (k = 4 .. 7) for the row."""
  x = np.asarray(x, np.float64)
  scales = np.exp2(np.arange(LEAST4, LARGEST4 + 1, dtype=np.float64))
  if value: scales = np.append(np.outer(scales[:-1], [1, 1.25, 1.5, 1.75]), scales[-1])
  groups = x if value else x.reshape(*x.shape[:-1], -1, 32)
  top = np.where(np.isfinite(groups), np.abs(groups), 0).max(-1)
  s = scales[np.minimum(np.searchsorted(7 * scales, top), len(scales) - 1)][..., None]
  return (grid4(groups / s) * s).reshape(x.shape)


def put4(values, tables, starts, lengths, x):
  """x (2 kv, rows, head) into values (pages, 2 kv, page, head) of the 4-bit cache, in place."""
  pages, kv2, page, _ = values.shape
  held = np.concatenate([held4(x[:kv2 // 2], False), held4(x[kv2 // 2:], True)])
  for r, length in enumerate(lengths):
    n = starts[r + 1] - starts[r]
    for i in range(n):
      k, at = divmod(length - n + i, page)
      id = tables[r, k] if k < tables.shape[1] else -1
      if 0 <= id < pages: values[id, :, at] = held[:, starts[r] + i]


def attend(q, values, tables, starts, lengths, window=0):
  """(out, weighed): q (heads, rows, head) over the pages, and the weights' mean of |v|, which bounds an error of the weights."""
  heads, rows, hd = q.shape
  pages, kv2, page, _ = values.shape
  rep = heads // (kv2 // 2)
  out, weighed = np.zeros(q.shape), np.zeros(q.shape)
  for r, length in enumerate(lengths):
    n = starts[r + 1] - starts[r]
    if n == 0: continue
    ids = tables[r, :-(-min(length, tables.shape[1] * page) // page)]
    held = np.concatenate([values[i] if 0 <= i < pages else np.zeros(values.shape[1:]) for i in ids], 1)
    on = np.repeat([0 <= i < pages for i in ids], page)
    key = np.arange(held.shape[1])
    for i in range(n):
      place, j = length - n + i, starts[r] + i
      seen = on & (key <= place) & (key > place - window if window else True)
      if not seen.any(): continue
      for h in range(heads):
        k, v = held[h // rep][seen], held[kv2 // 2 + h // rep][seen]
        s = k @ q[h, j].astype(np.float64)
        p = np.exp(s - s.max())
        out[h, j], weighed[h, j] = p @ v / p.sum(), p @ np.abs(v) / p.sum()
  return out, weighed


def verify(logits, ids, starts, uniforms, probs=None, t=None, drafts=None):
  """(tokens, counts) as serve.verify gives them. What is drawn from is not normalized, in extended precision, so that equal weights
  add exactly and a number on the border between two falls where it should."""
  rows, vocab = logits.shape
  x = np.where(np.isnan(logits), -np.inf, np.minimum(logits.astype(np.float64), np.finfo(np.float32).max))
  tokens, counts = np.full(rows, -1), []
  t = np.ones(rows) if t is None else np.asarray(t, np.float64).reshape(rows)
  t = np.where(t > 0, t, 0)

  def choice(j):  # (weights of row j, their sum: p times it), or (None, 0) where it has no token
    if not (x[j] > -np.inf).any(): return None, 0
    if t[j] == np.inf: return np.eye(1, vocab, np.argmax(x[j]))[0], 1
    with np.errstate(invalid="ignore"):
      e = np.where(x[j] > -np.inf, np.exp(np.longdouble(t[j]) * (x[j] - x[j].max())), 0)
    return e, e.sum()

  def draw(w, u):
    upto = np.cumsum(w)
    past = np.flatnonzero((upto > u * upto[-1]) & (w > 0))
    return past[0] if len(past) else np.flatnonzero(w > 0)[-1]
  for r, (s, e) in enumerate(zip(starts[:-1], starts[1:])):
    if drafts is not None: s = max(s, e - max(int(drafts[r]) + 1, 0))  # what lies ahead is not looked at
    a, n, made = 0, e - s, -1
    while n > 0:
      p, z = choice(s + a)
      if a == n - 1:
        if p is not None: made = draw(p, uniforms[1, s + a])
        break
      d = ids[s + a + 1]
      q = probs[s + a + 1].astype(np.longdouble) if probs is not None else np.zeros(vocab)
      inside = 0 <= d < vocab
      if probs is None and inside: q[d] = 1
      if p is not None and inside and uniforms[0, s + a + 1] * q[d] * z < p[d]:
        tokens[s + a] = d
        a += 1
        continue
      if p is not None:
        left = p if t[s + a] == np.inf else np.maximum(p - q * z, 0) if probs is not None else np.where(q > 0, 0, p)
        made = draw(left if left.sum() > 0 else p, uniforms[1, s + a])
      break
    if n > 0: tokens[s + a] = made
    counts.append(a + (made >= 0) if n > 0 else 0)
  return tokens, np.array(counts)
