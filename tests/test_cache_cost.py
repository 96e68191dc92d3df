"""What a paged cache's rounding costs a model, in log probabilities of given tokens, without a GPU: a small model whose logits its cache
decides, and that a cache with anything wrong in it shows. test_gpu_logprobs.py holds the device against the same model."""
import numpy as np
import pytest

from oracle import bfp as B, llama_ref as L, logprobs as LP, pages as P

ROWS, PAGE = 50, 16
CONFIG = dict(dim=576, heads=9, kv=3, layers=1, eps=1e-5, theta=10000.0, vocab=256, ffn=1536)


def model():
  """(config, weights, a prompt, the token given after each row): one block, whose attention's output is most of the residual and whose
  scores are wide enough that keys matter as much as values."""
  rng = np.random.default_rng(6)
  c, w = L.smol(rng, 1, vocab=256, places=96)
  w["layers.0.o_proj"] = B.bf16(10 * w["layers.0.o_proj"])
  w["layers.0.qkv_proj"][:, :12 * 64] *= 3  # queries and keys
  w["layers.0.qkv_proj"] = B.bf16(w["layers.0.qkv_proj"])
  w["embed"], w["norm"] = B.bf16(0.3 * w["embed"]), B.bf16(w["norm"] / 3)
  w["embed.T"] = np.ascontiguousarray(w["embed"].T)
  prompt = rng.integers(0, 256, ROWS)
  return c, w, prompt, np.append(prompt[1:], -1)


def logits(c, w, prompt, bits, broken=lambda v: v, rounded=lambda a: a):
  """The prompt's logits over a cache of 8 or 4 bits (None: values as they are). broken: what the cache's values (pages, 2 kv, page, head) are
  read as; rounded: what becomes of each operation's result."""
  nh, tables = c.heads + 2 * c.kv, np.arange(4)[None]
  x, p = w["embed"][prompt].astype(np.float32), L.block(w, 0)
  rot = [L.split(w[t][:ROWS], nh) for t in ("cos", "sin")]
  h = rounded(L.rms(x, p["input_layernorm"], c.eps))
  heads = rounded(L.rope(rounded(L.split(h @ p["qkv_proj"], nh)), *rot, w["turn"]))
  new, values = B.bf16(heads[c.heads:]), np.zeros((4, 2 * c.kv, PAGE, 64))
  if bits == 8: P.put(values, np.full((4, 2 * c.kv), 2.0 ** P.LEAST), tables, [0, ROWS], [ROWS], new)
  elif bits == 4: P.put4(values, tables, [0, ROWS], [ROWS], new)
  else:
    for i in range(ROWS): values[i // PAGE, :, i % PAGE] = new[:, i]
  o, _ = P.attend(heads[:c.heads], broken(values), tables, [0, ROWS], [ROWS])
  x = x + rounded(rounded(L.merge(o)) @ p["o_proj"])
  h = rounded(L.rms(x, p["post_attention_layernorm"], c.eps))
  gate, up = np.split(rounded(h @ p["gate_up_proj"]), 2, -1)
  x = x + rounded(rounded(gate / (1 + np.exp(-gate)) * up) @ p["down_proj"])
  return rounded(L.rms(x, w["norm"], c.eps)) @ w["embed.T"]


def given(x, ids): return LP.logprobs(np.float32(x), ids)[0][:-1]


def allowed(x):
  """How far a log probability may be off: logits by 3% of the largest, which the model's other tests allow, and it by twice that."""
  return 2 * 0.03 * np.abs(x).max()


@pytest.mark.parametrize("bits", [8, 4])
def test_a_broken_cache_shows(bits):
  c, w, prompt, ids = model()
  x = logits(c, w, prompt, bits)
  want = given(x, ids)
  off = lambda *a: np.abs(given(logits(c, w, prompt, *a), ids) - want).max()
  assert off(bits, lambda v: v, B.bf16) < allowed(x) / 3  # every result rounded to bf16, as the device does
  rng = np.random.default_rng(1)
  def some(at, f):
    def broken(v):
      v = v.copy()
      v[at] = f(v[at])
      return v
    return broken
  kv = c.kv
  for name, broken in {"zeros": lambda v: 0 * v, "signs": lambda v: -v, "noise": lambda v: rng.normal(0, v.std(), v.shape),
                       "keys' zeros": some(np.s_[:, :kv], lambda v: 0 * v), "values' zeros": some(np.s_[:, kv:], lambda v: 0 * v),
                       "keys' signs": some(np.s_[:, :kv], lambda v: -v), "values' signs": some(np.s_[:, kv:], lambda v: -v),
                       "a page turned by a token": some(np.s_[:1], lambda v: np.roll(v, 1, 2)),
                       "dims in pairs": lambda v: v.reshape(*v.shape[:-1], -1, 2)[..., ::-1].reshape(v.shape)}.items():
    assert off(bits, broken) > 2 * allowed(x), name  # so a device as far from it as is allowed is still caught
  assert off(12 - bits) > 2 * allowed(x)  # the other width's


def test_what_the_widths_cost():
  # log probabilities against those over values as they are: the root of the mean square over the prompt
  c, w, prompt, ids = model()
  want = given(logits(c, w, prompt, None), ids)
  cost = {bits: np.sqrt(np.mean((given(logits(c, w, prompt, bits), ids) - want) ** 2)) for bits in (8, 4)}
  assert 3 * cost[8] < cost[4] < 0.1 * np.abs(want).mean(), cost
