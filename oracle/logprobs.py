"""Log probabilities of given tokens, entropies and likeliest tokens in NumPy, in 64 bits: what bt_logprobs (include/baretile_amd.h)
defines, and how far fp32 may be from it."""
import numpy as np


def logprobs(logits, ids, k=0, t=None):
  """(log p, entropy, values, labels, how far each of the first three may be off in fp32), rows each."""
  logits = np.asarray(logits, np.float32)
  rows, vocab = logits.shape
  x = np.where(np.isnan(logits), -np.inf, np.minimum(logits, np.finfo(np.float32).max)).astype(np.float64)
  t = np.ones(rows) if t is None else np.asarray(t, np.float32).astype(np.float64).reshape(rows)
  t = np.where(t > 0, t, 0)
  given, entropy, values, labels = np.zeros(rows), np.zeros(rows), np.full((rows, k), -np.inf), np.full((rows, k), -1)
  off, off_entropy, off_values = np.zeros(rows), np.zeros(rows), np.zeros((rows, k))
  eps = 2.0 ** -24
  for r in range(rows):
    real = x[r] > -np.inf
    y = np.full(vocab, -np.inf)
    lse, logs, slack = 0.0, np.full(vocab, -np.inf), 0.0
    if real.any():
      if t[r] == np.inf:
        logs[np.argmax(x[r])] = 0
      else:
        y[real] = t[r] * (x[r][real] - x[r].max())
        w = np.exp(y)
        lse = np.log(w.sum())
        logs = y - lse
        p, size = w / w.sum(), np.where(real, -y, 0)
        p = np.where(real, p, 0)
        entropy[r] = lse + (p * size).sum()
        # Roundings of half a unit, eps: a weight's exponent four (relative to it), its power two; a chunk's 16 weights 15, the sum of a
        # thread's chunks one (it is of 64 bits), its move to the wave's largest logit two; 64 lanes' six, up to 16 waves' by a power each
        # 18, then the segments' likewise three, six and six: 59. A sum against a reference is moved to another only where that is twice
        # as far at least, two roundings each time: at most 2 / log(2) a unit of the weight's own distance from the largest, and
        # two, as the reference may lie a factor of two below. Then the logarithm's two units. The entropy's products have four more, its
        # quotient and the change of the logarithm's base three, and against a reference that is passed by two a chunk's 16 products may
        # be that much larger.
        with np.errstate(invalid="ignore"):
          mean = (p * size).sum()
          slack = eps * (7 * mean + 61 + 4 * lse)
          off_entropy[r] = slack + eps * (np.nansum(p * size * (7 * size + 68)) + 16 + 4 * entropy[r])
    def allowed(at): return 0.0 if logs[at] == -np.inf or t[r] == np.inf else slack + eps * (3 * -y[at] + 2 * abs(logs[at]))
    if 0 <= ids[r] < vocab: given[r], off[r] = logs[ids[r]], allowed(ids[r])
    order = [c for c in np.argsort(-(x[r] + 0.0), kind="stable")[:k] if real[c]]
    for j, c in enumerate(order): values[r, j], labels[r, j], off_values[r, j] = logs[c], c, allowed(c)
  return given, entropy, values, labels, off, off_entropy, off_values
