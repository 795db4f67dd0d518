"""alz_tv_process_dev takes the pitches of alz_bank_process_dev (include/alz.h) and refuses the same ones: rows that overlap would be
written over by each other."""
import ctypes

import pytest

from audiolazy_amd import _ffi


@pytest.mark.parametrize("layout,ldx,ldy", [(_ffi.TIME_MAJOR, 7, 8), (_ffi.TIME_MAJOR, 8, 7), (_ffi.TIME_MAJOR, 0, 0), (_ffi.CHAN_MAJOR, 99, 100),
                                            (_ffi.CHAN_MAJOR, 100, 99), (_ffi.CHAN_MAJOR, 8, 8), (_ffi.TIME_MAJOR, -8, 8)])
def test_rows_that_overlap(layout, ldx, ldy):
  L = _ffi.load()
  tap, p = (_ffi.TvTap * 1)(_ffi.TvTap(1.0, None, 0, 0, 0)), ctypes.c_void_p(4096)     # (never looked at: the call is refused)
  taps = ctypes.cast(tap, ctypes.c_void_p)
  assert L.alz_tv_process_dev(1, taps, 1, taps, 8, p, p, 100, layout, ldx, ldy, None, None, 0.0, 0, None) == _ffi.E_ARG
