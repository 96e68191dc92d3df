"""A paged KV cache of 8 or 4 bits a value: requests share a pool of pages through block tables, and a step's tables, row
starts, places and slots are made on the device from request lengths, so the whole step can be recorded and replayed.

The reference keeps a fixed region a slot (llama.py:293-373), as models.serve.Engine does; here a request holds the pages
its tokens fill. A page holds the tokens of every key and value head, a head's as 8-bit floats (4 exponent and 3 mantissa bits)
under one power of two, which makes each value exact in bf16: half of a bf16 cache's memory, and decoded in one
instruction for two values where a bfp8 cache takes five. A pool of 4 bits halves that again: 4-bit floats (2 exponent bits and 1
mantissa bit) under scales of each token's own, a power of two for 32 dims of a key, one for a value's whole row.

A step over several requests, each with any number of new tokens (a token, a token and its drafts, a prompt's chunk), of which
the last drafts[r] of request r are drafts (0: none; -1: no token follows yet, as behind a chunk that does not end its prompt,
or the request brings no row):

  batch = pool.plan(tables, cached, new, free, rows)   # once a step; every block's pool of its shape shares it, of either width
  pool.put(batch, x)                                   # each block's keys and values
  o = pool.attend(q, batch)                            # and its attention
  tokens, counts = serve.verify(logits, ids, batch.starts, uniforms, drafts=drafts)
"""
import ctypes, operator
from baretile_amd import _lib
from baretile_amd.tensor import Storage, Tensor, _written

PAGES = (16, 32, 64, 128, 256)
REQUESTS, ROWS = 2048, 1 << 20


def _int32(t, rt, what, rows=None, cols=None):
  """t, realized: a whole int32 matrix of a batch of one, with these rows and columns where they are given."""
  if not isinstance(t, Tensor) or t.rt is not rt: raise ValueError(f"{what} must be a tensor on the pool's runtime")
  if not (t.dtype == "int32" and t.batch == 1 and (rows is None or t.rows == rows) and (cols is None or t.cols == cols)):
    raise ValueError(f"{what} must be int32, ({'any' if rows is None else rows}, {'any' if cols is None else cols}): "
                     f"{t.dtype} {t.shape}")
  return t.realize()


def _row(t, rt, what, cols=None):
  t = _int32(t, rt, what, 1, cols)
  return t if t._contiguous() else t.contiguous()


class Batch:
  """One step's plan (Pages.plan): `tables` as it was given, with the step's new pages in it, and int32 rows made here.
  starts (requests + 1): each request's first row, then the rows in use; lengths: each request's tokens with the new ones;
  places: each row's place in its request, -1 behind the last request's rows; slots: the row of a flat cache of
  pages * page rows that the token takes, -1 where there is no page; taken: how many of the free list's pages are
  used so far (more than it has: that many less were missing)."""
  def __init__(self, tables, starts, lengths, places, slots, taken, parts, rows, most, page, pages, kv):
    self.tables, self.starts, self.lengths, self.places, self.slots = tables, starts, lengths, places, slots
    self.taken, self.parts, self.rows, self.most = taken, parts, rows, most
    self.page, self.pages, self.kv, self.requests = page, pages, kv, tables.rows
    self.args = _lib.BatchArgs(tables.addr, starts.addr, lengths.addr, parts.addr, tables.sr, tables.rows, tables.cols,
                               rows, most)


class Pages:
  """A pool of `pages` pages of `page` tokens (16, 32, 64, 128 or 256) for kv key heads, 64 or 128 wide: one block's cache, of 8 or
  4 bits a value. Pages start as zeros. Which pages are free, and which a request gives back, is the caller's to keep."""
  def __init__(self, rt, pages, kv, head, page=64, bits=8):
    pages, kv, head, page, bits = (operator.index(v) for v in (pages, kv, head, page, bits))
    if bits not in (4, 8): raise ValueError(f"a paged cache has 8 or 4 bits a value, not {bits}")
    if page not in PAGES: raise ValueError(f"a page holds {', '.join(map(str, PAGES))} tokens, not {page}")
    if head not in (64, 128): raise ValueError(f"a paged cache's heads are 64 or 128 wide, not {head}")
    if not (0 < kv <= 1024 and pages > 0 and pages * page < 1 << 31):
      raise ValueError(f"a paged cache of {pages} pages of {page} tokens and {kv} key heads")
    rt.check()
    self.rt, self.pages, self.kv, self.head, self.page, self.bits = rt, pages, kv, head, page, bits
    if bits == 4:
      self.scales, need = None, ctypes.c_uint64()  # (they lie among the codes)
      self.args = _lib.PagesArgs(0, 0, pages, page, kv, head)
      _lib.call("pages4_bytes", ctypes.byref(self.args), ctypes.byref(need))
      self.storage = Storage(rt, need.value)
      self.args.values = self.storage.addr
    else:
      self.storage = Storage(rt, pages * 2 * kv * page * head)
      self.scales = Tensor(rt, pages, 2 * kv, dtype="fp32")
      rt.fill32(self.scales.addr, 127 - 100 << 23, pages * 2 * kv)  # 2^-100, the smallest scale
      self.args = _lib.PagesArgs(self.storage.addr, self.scales.addr, pages, page, kv, head)
    rt.fill32(self.storage.addr, 0, self.storage.nbytes // 4)

  def _call(self, name): return f"pages{'4' if self.bits == 4 else ''}_{name}"

  def plan(self, tables, cached, new, free, rows, taken=None, most=None):
    """The Batch of a step, made on the device (bt_pages_plan). tables (requests, width) int32: each request's pages in order,
    -1 where it has none; cached, new: int32 rows, each request's tokens in the cache and those that the step brings, at
    most `most` each (any more are cut off) and together at most `rows`; free: an int32 row of free pages, taken from the
    front, after the first `taken` (an int32 (1, 1), as an earlier Batch has it). A request's pages are kept up to its first
    empty entry, so that drafts that were refused leave theirs to the next step; the pages it needs from there on go into
    `tables`."""
    rows, most = operator.index(rows), rows if most is None else operator.index(most)
    if not (1 <= rows <= ROWS and most >= 1):
      raise ValueError(f"a plan takes 1 to {ROWS} rows, and one a request at least: {rows}, {most}")
    t = _int32(tables, self.rt, "a plan's tables")
    if not (t.rows <= REQUESTS and t.cols * self.page <= 1 << 30 and t.sc == 1 and t.rep == 1 and not t.cyc and t.op is None and
            (t.sr >= t.cols or t.rows == 1)):
      raise ValueError(f"a plan's tables are at most {REQUESTS} rows of pages of 2^30 tokens in all, each contiguous and "
                       f"apart from the others: {t.shape}")
    n = t.rows
    cached, new, free = _row(cached, self.rt, "cached", n), _row(new, self.rt, "new", n), _row(free, self.rt, "free")
    if taken is not None: taken = _row(taken, self.rt, "taken", 1)
    most = min(most, rows)
    made = lambda cols: Tensor(self.rt, 1, cols, dtype="int32")
    starts, lengths, places, slots, used, parts = (made(c) for c in (n + 1, n, rows, rows, 1, n + 2))
    _written(t.storage)
    args = _lib.PlanArgs(t.addr, cached.addr, new.addr, free.addr, taken.addr if taken is not None else 0, starts.addr,
                         lengths.addr, places.addr, slots.addr, used.addr, parts.addr, t.sr, n, t.cols, free.cols, rows,
                         self.page, self.pages, most, self.kv)
    self.rt.run("plan", "pages_plan", ctypes.byref(args))
    return Batch(t, starts, lengths, places, slots, used, parts, rows, most, self.page, self.pages, self.kv)

  def _fits(self, batch):
    if not (isinstance(batch, Batch) and batch.tables.rt is self.rt and (batch.page, batch.pages, batch.kv) ==
            (self.page, self.pages, self.kv)):
      raise ValueError(f"the batch must be planned by a pool of {self.pages} pages of {self.page} tokens and {self.kv} key "
                       f"heads on this runtime")

  def put(self, batch, x):
    """Puts the batch's rows into their pages (bt_pages_put, bt_pages4_put): x (2 kv, rows, head) bf16, key heads then value heads,
    as rope_put gives them. In 8 bits each page and head takes the smallest power of two under which its largest value is at most
    448; where a page that holds rows needs a larger one, those are rounded again under it. It stays so until the page is begun
    again, also where it was a refused draft's value that needed it. In 4 bits each row has scales of its own, the smallest under
    which its largest value is at most 7 (a power of two for 32 dims of a key, one of 4 to 7 quarters of one for a value), and
    what a page holds doesn't depend on the puts that its rows came in. Rows without a page are dropped. Requests may share pages
    that they only read; a page that takes rows is one request's."""
    self._fits(batch)
    if not (isinstance(x, Tensor) and x.rt is self.rt and x.dtype == "bf16" and
            (x.batch, x.rows, x.cols) == (2 * self.kv, batch.rows, self.head)):
      raise ValueError(f"put needs bf16 rows ({2 * self.kv}, {batch.rows}, {self.head}): {getattr(x, 'dtype', type(x))} "
                       f"{getattr(x, 'shape', '')}")
    x = x.realize()
    if x.sc != 1 or x.rep != 1 or x.cyc or x.sb % 8 or x.sr % 8 or x.addr % 16: x = x.contiguous()
    if self.scales is not None: _written(self.scales.storage)
    name = self._call("put")
    self.rt.run(name, name, ctypes.byref(self.args), ctypes.byref(batch.args), x.addr, x.sb, x.sr,
                reads=4 * self.kv * batch.rows * self.head)

  def attend(self, q, batch, window=0, merged=False):
    """softmax(q @ k^T + mask) @ v over each row's request (bt_pages_attend, bt_pages4_attend): q (heads, rows, head) bf16, heads a
    multiple of kv; a row sees its request's keys up to its own place and, with window, the last `window` of them. RoPE scales q
    beforehand. Rows behind the last request's come back as zeros. merged gives the result as merge() of it, (rows, heads * head)."""
    self._fits(batch)
    window = operator.index(window)
    if not 0 <= window < 1 << 31: raise ValueError(f"attention needs a nonnegative window of less than 2^31, not {window}")
    if not (isinstance(q, Tensor) and q.rt is self.rt and q.dtype == "bf16" and q.batch % self.kv == 0 and len(q.shape) <= 3 and
            (q.rows, q.cols) == (batch.rows, self.head)):
      raise ValueError(f"attend needs bf16 queries of a multiple of {self.kv} heads, ({batch.rows}, {self.head}) each: "
                       f"{getattr(q, 'dtype', type(q))} {getattr(q, 'shape', '')}")
    q = q.realize()
    if q.sc != 1 or q.rep != 1 or q.cyc or q.sb % 8 or q.sr % 8 or q.addr % 16: q = q.contiguous()
    if merged:
      out = Tensor(self.rt, q.rows, q.batch * q.cols)
      osh, osr = q.cols, out.sr
    else:
      out = Tensor(self.rt, q.rows, q.cols, batch=q.batch)
      osh, osr = out.sb, out.sr
    need, scratch = ctypes.c_uint64(), None
    name = self._call("attend")
    _lib.call(name + "_scratch", ctypes.byref(self.args), ctypes.byref(batch.args), q.batch, window, ctypes.byref(need))
    if need.value: scratch = Storage(self.rt, need.value)  # freed (stream-ordered) once the launches that use it are queued
    self.rt.run(name, name, ctypes.byref(self.args), ctypes.byref(batch.args), q.addr, q.sb, q.sr, out.addr,
                osh, osr, q.batch, window, scratch.addr if scratch else 0, need.value)
    del scratch
    return out

  def values(self):
    """Every page's values as bf16, exactly: (pages * 2 kv, page, head), key heads then value heads of each page."""
    out = Tensor(self.rt, self.page, self.head, batch=self.pages * 2 * self.kv)
    name = self._call("read")
    self.rt.run(name, name, ctypes.byref(self.args), out.addr, reads=self.storage.nbytes)
    return out
