"""Log probabilities without a GPU: the oracle by hand and by torch, and what the library refuses."""
import ctypes
import numpy as np
import pytest
import torch

from baretile_amd import _lib
from oracle import logprobs as L


def test_by_hand():
  x = np.log(np.array([[1, 2, 1, 4]], np.float32))
  given, entropy, values, labels, *_ = L.logprobs(x, [1], 6)
  assert abs(given[0] - np.log(1 / 4)) < 1e-6 and abs(entropy[0] - 1.75 * np.log(2)) < 1e-6
  assert labels[0].tolist() == [3, 1, 0, 2, -1, -1] and np.all(values[0, 4:] == -np.inf)
  given, entropy, values, labels, *_ = L.logprobs(x, [3], 2, [np.inf])
  assert given[0] == 0 and entropy[0] == 0 and values[0].tolist() == [0, -np.inf] and labels[0].tolist() == [3, 1]
  given, entropy, *_ = L.logprobs(x, [-1], 0, [0.0])
  assert given[0] == 0 and abs(entropy[0] - np.log(4)) < 1e-12
  given, entropy, values, labels, *_ = L.logprobs(np.full((1, 3), -np.inf), [1], 2)
  assert given[0] == -np.inf and entropy[0] == 0 and labels[0].tolist() == [-1, -1]


def test_by_torch():
  rng = np.random.default_rng(0)
  x, t, ids = rng.normal(0, 3, (20, 300)).astype(np.float32), rng.uniform(0.5, 2, 20).astype(np.float32), rng.integers(0, 300, 20)
  given, entropy, values, labels, *_ = L.logprobs(x, ids, 9, t)
  d = torch.distributions.Categorical(logits=torch.tensor(x).double() * torch.tensor(t).double()[:, None])
  assert np.allclose(given, d.log_prob(torch.tensor(ids)).numpy(), atol=1e-12) and np.allclose(entropy, d.entropy().numpy(), atol=1e-12)
  top = d.logits.topk(9)
  assert np.allclose(values, top[0].numpy(), atol=1e-12) and np.array_equal(labels, top[1].numpy())


@pytest.mark.parametrize("kw", [dict(logits=0), dict(ids=0), dict(logprobs=0), dict(entropy=0), dict(k=3), dict(k=65), dict(k=-1), dict(rows=0),
                                dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(rows=(1 << 20) + 1), dict(t=2), dict(rows=1 << 20, vocab=1 << 20), dict(rows=1 << 20, vocab=61441)])
def test_refused(kw):
  args = _lib.LogprobsArgs(**(dict(logits=16, ids=16, logprobs=16, entropy=16, rows=4, vocab=50) | kw))
  with pytest.raises(ValueError): _lib.call("logprobs_scratch", ctypes.byref(args), ctypes.byref(ctypes.c_uint64()))
  with pytest.raises(ValueError): _lib.call("logprobs_scratch", ctypes.byref(args), None)


def test_scratch():
  need = ctypes.c_uint64()
  for rows, vocab, k in ((1, 50, 0), (3, 4096, 64), (1, 4097, 0), (7, 1 << 20, 64), (1 << 10, 131072, 20)):
    args = _lib.LogprobsArgs(logits=16, ids=16, logprobs=16, entropy=16, values=16, labels=16, rows=rows, vocab=vocab, k=k)
    _lib.call("logprobs_scratch", ctypes.byref(args), ctypes.byref(need))
    assert (need.value == 0) == (vocab <= 4096)
