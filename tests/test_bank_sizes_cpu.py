"""Bank sizes whose products leave 64 bits, or that no device holds, are refused before anything is computed from them."""
import ctypes

import pytest

from audiolazy_amd import _ffi


@pytest.mark.parametrize("n_sets,n_inputs,mode", [(1, 1 << 62, _ffi.BANK_DIAGONAL), (1, (1 << 40) + 1, _ffi.BANK_DIAGONAL), (1, 1 << 62, _ffi.BANK_OUTER),
                                                  (4, 1 << 62, _ffi.BANK_OUTER), (3, 1 << 40, _ffi.BANK_OUTER), (4, (1 << 62) + 1, _ffi.BANK_OUTER)])
def test_too_many_channels(n_sets, n_inputs, mode):
  L = _ffi.load()
  one = (ctypes.c_int * 1)(1)
  coefs = (ctypes.c_double * n_sets)(*[1.] * n_sets)
  handle = ctypes.c_void_p()
  assert L.alz_bank_create(n_sets, n_inputs, mode, 1, one, one, coefs, coefs, 0, ctypes.byref(handle)) == _ffi.E_ARG and not handle


@pytest.mark.parametrize("side", ["b", "a"])
def test_a_state_larger_than_any_device(side):
  L = _ffi.load()
  taps = 1 << 20
  counts = {"b": [1], "a": [1]}
  counts[side] = [taps]
  nb, na = ((ctypes.c_int * 1)(*counts[k]) for k in "ba")
  b, a = ((ctypes.c_double * counts[k][0])(1.) for k in "ba")
  handle = ctypes.c_void_p()
  assert L.alz_bank_create(1, 1 << 30, _ffi.BANK_DIAGONAL, 1, nb, na, b, a, 0, ctypes.byref(handle)) == _ffi.E_NOMEM and not handle
