"""The 4-bit paged cache without a GPU: what its oracle rounds to, what the pools and the library refuse, and the layout's size."""
import ctypes
import numpy as np
import pytest

from baretile_amd import _lib
from baretile_amd.models import llama
from baretile_amd.pages import Pages
from oracle import pages as P


def test_grid():
  borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
  even = np.array([0, 1, 1, 2, 2, 4, 4.0])  # ties go to the even code: of 0, 1, 2, 4 to 0, 2, 4, 6 of the list
  assert np.array_equal(P.grid4(borders), even) and np.array_equal(P.grid4(-borders), -even)
  up = np.nextafter(borders, 9)
  assert np.array_equal(P.grid4(up), P.GRID4[1:]) and np.array_equal(P.grid4(np.nextafter(borders, 0)), P.GRID4[:-1])
  assert np.array_equal(P.grid4(P.GRID4), P.GRID4)
  assert np.array_equal(P.grid4([6.9, 7, 100, np.inf, -np.inf]), [6, 6, 6, 6, -6])
  assert abs(P.grid4(np.nan)) == 6


@pytest.mark.parametrize("value", [False, True])
def test_held_rows_by_hand(value):
  x = np.zeros((1, 64))
  x[0, 0], x[0, 1], x[0, 40] = 7.0, 0.25, 14.5
  got = P.held4(x, value)
  if value:  # 14.5 <= 7 s: s = 2.5 (of 2.5, 3, 3.5, 4): 7 / 2.5 = 2.8 -> 3, 0.1 -> 0, 5.8 -> 6
    assert got[0, 0] == 7.5 and got[0, 1] == 0 and got[0, 40] == 15
  else:  # s = 1 for the first 32 dims (0.25 ties to 0), 4 for the others: 14.5 / 4 = 3.625 -> 4
    assert got[0, 0] == 6 and got[0, 1] == 0 and got[0, 40] == 16


@pytest.mark.parametrize("value", [False, True])
def test_held_rows_are_within_half_the_largest_step(value):
  rng = np.random.default_rng(0)
  x = rng.normal(0, 1, (500, 128)) * np.exp2(rng.integers(-30, 30, (500, 1)))
  got = P.held4(x, value)
  top = np.abs(x if value else x.reshape(500, 4, 32)).max(-1, keepdims=True)
  s = 2 * top / 7 if not value else 1.25 * top / 7  # the scale is at most the next one above the largest / 7
  assert np.all(np.abs(got - x).reshape(500, -1, 128 if value else 32) <= np.reshape(s, (500, -1, 1)) * (1 + 1e-12))


def test_what_a_pool_of_4_bits_holds():
  need = ctypes.c_uint64()
  for hd, row in ((64, 68), (128, 134)):  # codes of both, an exponent for 32 dims of a key, a bf16 scale for a value
    for page in (16, 32, 64, 128, 256):
      _lib.call("pages4_bytes", ctypes.byref(_lib.PagesArgs(0, 0, 3, page, 5, hd)), ctypes.byref(need))
      assert need.value == 3 * 5 * page * row


@pytest.mark.parametrize("args", [(0, 0, 3, 64, 1, 96), (0, 0, 3, 48, 1, 64), (0, 0, 0, 64, 1, 64), (0, 0, 3, 64, 0, 64), (0, 0, 3, 64, 1025, 64),
                                  (0, 0, 1 << 25, 64, 1, 64)])
def test_pools_refused(args):
  with pytest.raises(ValueError): _lib.call("pages4_bytes", ctypes.byref(_lib.PagesArgs(*args)), ctypes.byref(ctypes.c_uint64()))


def test_bytes_refuses_no_pool():
  with pytest.raises(ValueError): _lib.call("pages4_bytes", None, ctypes.byref(ctypes.c_uint64()))
  with pytest.raises(ValueError): _lib.call("pages4_bytes", ctypes.byref(_lib.PagesArgs(0, 0, 3, 64, 1, 64)), None)


@pytest.mark.parametrize("bits", [0, 2, 5, 16])
def test_bits_refused(bits):
  with pytest.raises(ValueError): Pages(None, 3, 1, 64, bits=bits)
  with pytest.raises(ValueError): llama.paged_cache(None, llama.smol(1), 3, bits=bits)


def test_scratch_is_the_8_bit_caches():
  batch = _lib.BatchArgs(16, 16, 16, 16, 40, 5, 40, 9, 3)
  for hd, heads, page in ((64, 8, 16), (128, 32, 64)):
    a, b = ctypes.c_uint64(), ctypes.c_uint64()
    _lib.call("pages_attend_scratch", ctypes.byref(_lib.PagesArgs(16, 16, 9, page, 4, hd)), ctypes.byref(batch), heads, 0, ctypes.byref(a))
    _lib.call("pages4_attend_scratch", ctypes.byref(_lib.PagesArgs(16, 0, 9, page, 4, hd)), ctypes.byref(batch), heads, 0, ctypes.byref(b))
    assert a.value == b.value
    for bad in (6, 0, -4):
      with pytest.raises(ValueError):
        _lib.call("pages4_attend_scratch", ctypes.byref(_lib.PagesArgs(16, 0, 9, page, 4, hd)), ctypes.byref(batch), bad, 0, ctypes.byref(a))
    with pytest.raises(ValueError):
      _lib.call("pages4_attend_scratch", ctypes.byref(_lib.PagesArgs(16, 0, 9, page, 4, hd)), ctypes.byref(batch), heads, -1, ctypes.byref(a))


@pytest.mark.parametrize("scales", [0, 1, 2, 16, 2 ** 64 - 1])
def test_scales_of_a_pool_of_4_bits_are_not_looked_at(scales):
  need = ctypes.c_uint64()
  pool, batch = _lib.PagesArgs(16, scales, 9, 64, 4, 64), _lib.BatchArgs(16, 16, 16, 16, 40, 5, 40, 9, 3)
  _lib.call("pages4_bytes", ctypes.byref(pool), ctypes.byref(need))
  assert need.value == 9 * 4 * 64 * 68
  _lib.call("pages4_attend_scratch", ctypes.byref(pool), ctypes.byref(batch), 8, 0, ctypes.byref(need))
  with pytest.raises(ValueError): _lib.call("pages4_attend_scratch", ctypes.byref(_lib.PagesArgs(8, scales, 9, 64, 4, 64)), ctypes.byref(batch), 8, 0, ctypes.byref(need))
  if scales % 4:  # in 8 bits they are
    with pytest.raises(ValueError): _lib.call("pages_attend_scratch", ctypes.byref(pool), ctypes.byref(batch), 8, 0, ctypes.byref(need))
