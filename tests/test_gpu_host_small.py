"""alz_bank_process_host below its pipelined path: every shape of rows the caller can have -- one channel, odd channel counts (whose
device rows are one double longer), rows with gaps on either side, single rows, blocks that grow and shrink from call to call."""
import ctypes

import numpy as np
import pytest

from oracle import oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def alz():
  import audiolazy_amd
  audiolazy_amd.load_library()
  assert audiolazy_amd.device_count() >= 1, "no HIP device: the engine has no CPU path"
  return audiolazy_amd


def same_bits(a, b):
  return a.shape == b.shape and bool(np.array_equal(a.view(np.uint64), b.view(np.uint64)))


@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("gap_x,gap_y", [(0, 0), (1, 0), (0, 1), (1, 1), (5, 2)])
@pytest.mark.parametrize("C", [1, 2, 3, 64, 101])
def test_blocks_of_one_stream(alz, C, gap_x, gap_y, layout):
  import bench
  from audiolazy_amd import _ffi
  b, a = bench.resonator_coefs(C)
  lens = [1, 2, 500, 33, 1, 1000, 64]
  rng = np.random.default_rng(C)
  x = rng.uniform(-1, 1, (sum(lens), C))
  ref = oracle.bank([3], [3], b, a, x, layout="time")
  bank = alz.FilterBank([(b, a)], n_inputs=C)
  bank.reset()
  dp, at = ctypes.POINTER(ctypes.c_double), 0
  for n in lens:
    turn = (lambda v: v) if layout == "time" else (lambda v: v.T)
    blk = turn(x[at:at + n])
    rows, cols = blk.shape
    xw, yw = np.full((rows, cols + gap_x), np.nan), np.full((rows, cols + gap_y), -7.5)
    xw[:, :cols] = blk
    _ffi.check(bank._L.alz_bank_process_host(bank._h, xw.ctypes.data_as(dp), yw.ctypes.data_as(dp), n,
                                             _ffi.TIME_MAJOR if layout == "time" else _ffi.CHAN_MAJOR, cols + gap_x, cols + gap_y))
    assert same_bits(np.ascontiguousarray(turn(yw[:, :cols])), ref[at:at + n]) and (yw[:, cols:] == -7.5).all(), n
    at += n


@pytest.mark.parametrize("layout", ["time", "chan"])
def test_outer_bank_with_an_odd_number_of_outputs(alz, layout):
  import bench
  sets, N = 5, 700
  b, a = bench.resonator_coefs(sets)
  x = np.random.default_rng(4).uniform(-1, 1, (N, 1))
  bank = alz.FilterBank([(b, a)], n_inputs=1, mode="outer")
  bank.reset()
  y = bank.process(x if layout == "time" else np.ascontiguousarray(x.T), layout=layout)
  ref = oracle.bank([3], [3], b, a, np.repeat(x, sets, axis=1), layout="time")
  assert same_bits(np.ascontiguousarray(y if layout == "time" else y.T), ref)
