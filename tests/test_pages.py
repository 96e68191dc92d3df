"""The paged cache's and verification's host side, on the CPU: the oracle against other arithmetic, argument structs against the
header, and what the library refuses before it touches a GPU."""
import ctypes, os, shutil, subprocess
import numpy as np
import pytest
import torch

from baretile_amd import _lib
from oracle import pages as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_grid_is_the_8_bit_float_rounding():
  rng = np.random.default_rng(0)
  x = np.concatenate([rng.normal(0, 1, 5000), rng.normal(0, 1e-2, 5000), rng.uniform(-448, 448, 5000)]).astype(np.float32)
  codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
  codes = np.sort(codes[torch.isfinite(codes)].numpy())
  x = np.concatenate([x, codes, (codes[1:] + codes[:-1]) / 2]).astype(np.float32)  # and every tie
  assert np.array_equal(P.grid(x), torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy())


def test_scale_is_the_smallest_power_of_two():
  for top in (1e-3, 1.0, 1.75, 1.7578125, 1.99, 447.0, 448.0, 450.0, 1e30):
    s = P.scale(np.array([[-top, 0.0, np.inf, np.nan]]))
    assert np.log2(s) % 1 == 0 and top <= 448 * s and top > 448 * s / 2
  assert P.scale(np.zeros((2, 2))) == 2.0 ** -100 and P.scale(np.full((1, 1), 3e38)) == 2.0 ** 119


def test_structs_match_the_header(tmp_path):
  cc = shutil.which("gcc") or shutil.which("cc")
  if cc is None: pytest.skip("no C compiler")
  structs = {"bt_pages": _lib.PagesArgs, "bt_plan_args": _lib.PlanArgs, "bt_batch": _lib.BatchArgs, "bt_verify_args": _lib.VerifyArgs}
  lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "baretile_amd.h"', "int main(void) {"]
  for name, cls in structs.items():
    lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
    lines += [f'  printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, *_ in cls._fields_]
  src, exe = tmp_path / "sizes.c", tmp_path / "sizes"
  src.write_text("\n".join(lines + ["  return 0; }"]) + "\n")
  subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
  got = dict(l.split() for l in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
  for name, cls in structs.items():
    assert int(got[name]) == ctypes.sizeof(cls), name
    for f, *_ in cls._fields_: assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, (name, f)


def need(pool=None, batch=None, heads=8, window=0):
  c = _lib.PagesArgs(**({"values": 4096, "scales": 4096, "pages": 10, "page": 64, "kv": 2, "head_dim": 64} | (pool or {})))
  b = _lib.BatchArgs(**({"tables": 4096, "starts": 4096, "lengths": 4096, "parts": 4096, "tables_sr": 8, "requests": 3, "width": 20,
                         "rows": 6, "most": 2} | (batch or {})))
  n = ctypes.c_uint64()
  _lib.call("pages_attend_scratch", ctypes.byref(c), ctypes.byref(b), heads, window, ctypes.byref(n))
  return n.value


def test_attention_scratch():
  # two heads, 256 + 3 parts at most, 8 pairs (2 rows of 4 heads) of 64 dims, a maximum and a sum in 4 words
  assert need() == 259 * 2 * 8 * 68 * 4
  assert need(batch={"width": 8}) == 0  # 512 keys at most: a part a request, nothing to join


@pytest.mark.parametrize("bad, why", [
  (dict(pool={"page": 48}), "a page holds"), (dict(pool={"page": 8}), "a page holds"), (dict(pool={"page": 512}), "a page holds"),
  (dict(pool={"head_dim": 96}), "64 or 128"), (dict(pool={"kv": 0}), "pages of"), (dict(pool={"pages": 1 << 27}), "pages of"),
  (dict(pool={"values": 0}), "values and scales"), (dict(pool={"values": 4104}), "aligned"),
  (dict(batch={"tables": 0}), "needs its tables"), (dict(batch={"starts": 4098}), "aligned"), (dict(batch={"requests": 0}), "a batch of"),
  (dict(batch={"requests": 2049}), "a batch of"), (dict(batch={"rows": (1 << 20) + 1}), "a batch of"), (dict(batch={"width": 0}), "a batch of"),
  (dict(batch={"most": 0}), "a batch of"), (dict(batch={"width": 1 << 27}), "a batch of"),
  (dict(batch={"width": 1 << 25}), "over 2"), (dict(batch={"requests": 2048, "most": 12, "rows": 12}, pool={"kv": 1024}, heads=4096), "too large"),
  (dict(batch={"rows": 1 << 20, "most": 1 << 20}, heads=512), "too large"), (dict(heads=1 << 20, batch={"rows": 1 << 12}), "heads over"), (dict(heads=7), "7 heads"), (dict(heads=0), "0 heads"),
  (dict(window=-1), "window")])
def test_attention_refuses(bad, why):
  with pytest.raises(ValueError, match=why): need(**bad)


@pytest.mark.parametrize("bad", [{"logits": 0}, {"ids": 0}, {"uniforms": 0}, {"counts": 0}, {"logits": 4098}, {"vocab": 0},
                                 {"vocab": (1 << 20) + 1}, {"rows": 0}, {"requests": 0},
                                 {"vocab": 1 << 20, "rows": 1 << 17}, {"requests": 1 << 20, "vocab": 1 << 17}])
def test_verify_refuses(bad):
  fields = {"logits": 4096, "uniforms": 4096, "ids": 4096, "starts": 4096, "tokens": 4096, "counts": 4096, "rows": 5, "requests": 1,
            "vocab": 1000}
  n = ctypes.c_uint64()
  _lib.call("verify_scratch", ctypes.byref(_lib.VerifyArgs(**fields)), ctypes.byref(n))
  assert n.value == 5 * 2 * 16 + 40 + 2 * 8  # 1000 logits are two chunks of 512
  with pytest.raises(ValueError, match="verifying"):
    _lib.call("verify_scratch", ctypes.byref(_lib.VerifyArgs(**(fields | bad))), ctypes.byref(n))


def test_a_prompts_rows_are_no_drafts():
  # with drafts, each request is verified as if its last rows were all it had
  rng = np.random.default_rng(1)
  logits, ids = rng.normal(0, 2, (40, 500)).astype(np.float32), rng.integers(0, 500, 40)
  ids[31:40] = logits[30:39].argmax(1)  # drafts that greedy rows take
  u, greedy = rng.random((2, 40)).astype(np.float32), np.full(40, np.inf)
  tokens, counts = P.verify(logits, ids, [0, 25, 30, 30, 40], u, t=greedy, drafts=[0, -1, 0, 4])
  assert counts.tolist() == [1, 0, 0, 5]
  assert tokens[24] == logits[24].argmax() and (tokens[:24] == -1).all() and (tokens[25:35] == -1).all()
  assert np.array_equal(tokens[35:], logits[35:].argmax(1))
  for t in (None, greedy):
    tokens, counts = P.verify(logits, ids, [0, 40], u, t=t, drafts=[6])
    alone = P.verify(logits[33:], ids[33:], [0, 7], u[:, 33:], t=None if t is None else t[33:])
    assert np.array_equal(tokens[33:], alone[0]) and np.array_equal(counts, alone[1]) and (tokens[:33] == -1).all()


def test_verify_refuses_drafts_off_their_boundary():
  fields = {"logits": 4096, "uniforms": 4096, "ids": 4096, "starts": 4096, "tokens": 4096, "counts": 4096, "rows": 5, "requests": 1,
            "vocab": 1000}
  n = ctypes.c_uint64()
  _lib.call("verify_scratch", ctypes.byref(_lib.VerifyArgs(**fields, drafts=4096)), ctypes.byref(n))
  with pytest.raises(ValueError, match="4-byte"): _lib.call("verify_scratch", ctypes.byref(_lib.VerifyArgs(**fields, drafts=4098)), ctypes.byref(n))


def test_no_runtime():
  for name, args in (("pages_plan", (None,)), ("pages_put", (None, None, 0, 0, 0)), ("pages_read", (None, 0)), ("verify", (None,)),
                     ("pages_attend", (None, None, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0))):
    with pytest.raises(ValueError, match="no runtime"): _lib.call(name, None, *args)
