"""The frame geometry of the LPC entry points (include/alz.h) is refused before anything is launched or divided by: negative counts,
hops and orders, frames without a sample."""
import ctypes

import numpy as np
import pytest

from audiolazy_amd import _ffi
from audiolazy_amd.lpc import acorr_frames, kautocor_frames, lag_matrix_frames

P = ctypes.c_void_p(4096)          # (never looked at: the call is refused)
BAD = [(-1, 480, 240, 8), (3, 0, 240, 8), (3, -5, 240, 8), (3, 480, -2, 8), (3, 480, 240, -1), (20000, 480, 240, -1), (20000, 0, 240, 8)]


@pytest.mark.parametrize("frames,frame_len,hop,order", BAD)
@pytest.mark.parametrize("flags", [0, _ffi.LPC_FUSED, _ffi.LPC_DENSE])
def test_kautocor(frames, frame_len, hop, order, flags):
  L = _ffi.load()
  assert L.alz_lpc_kautocor_dev_ex(P, frames, frame_len, hop, order, P, P, P, flags, 0, None) == _ffi.E_ARG
  assert L.alz_lpc_kautocor_dev(P, frames, frame_len, hop, order, P, P, P, 0, None) == _ffi.E_ARG


@pytest.mark.parametrize("frames,frame_len,hop,order", BAD)
def test_acorr_and_lag_matrix(frames, frame_len, hop, order):
  L = _ffi.load()
  assert L.alz_acorr_dev(P, frames, frame_len, hop, order, P, 0, None) == _ffi.E_ARG
  assert L.alz_lag_matrix_dev(P, frames, frame_len, hop, order, P, 0, None) == _ffi.E_ARG


@pytest.mark.parametrize("call", [kautocor_frames, acorr_frames, lag_matrix_frames])
@pytest.mark.parametrize("hop", [-1, -480, -1000])
def test_hops_that_go_back(call, hop):
  with pytest.raises(ValueError):
    call(np.zeros(960), 480, 8, hop=hop)
