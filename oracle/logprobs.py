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
        # a weight's exponent has three roundings and its power two units, a sum of 16, 6 of a wave's lanes, up to 16 waves' and the
        # chunks' likewise about 50; then the logarithm's two units
        with np.errstate(invalid="ignore"):
          mean = (p * size).sum()
          slack = eps * (3 * mean + 54 + 4 * lse)
          off_entropy[r] = slack + eps * (np.nansum(p * size * (3 * size + 58)) + 4 * entropy[r])
    def allowed(at): return 0.0 if logs[at] == -np.inf or t[r] == np.inf else slack + eps * (3 * -y[at] + 2 * abs(logs[at]))
    if 0 <= ids[r] < vocab: given[r], off[r] = logs[ids[r]], allowed(ids[r])
    order = [c for c in np.argsort(-(x[r] + 0.0), kind="stable")[:k] if real[c]]
    for j, c in enumerate(order): values[r, j], labels[r, j], off_values[r, j] = logs[c], c, allowed(c)
  return given, entropy, values, labels, off, off_entropy, off_values
