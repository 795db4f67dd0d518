"""alz_bank_process_host on blocks of its pipelined path (64 MiB of traffic and more) whose pieces do not fall together with rows:
a row longer than a page-locked buffer, rows with gaps, odd channel counts, banks with more outputs than inputs.  The doubles are
the oracle's, and what lies between the caller's rows is left alone."""
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


def resonators(n):
  import bench
  return bench.resonator_coefs(n)


def test_one_channel_longer_than_a_buffer(alz):
  N = 5000011                                 # 40 MB in, 40 MB out: two chunks, each one row of 20 MB
  b, a = resonators(1)
  x = np.random.default_rng(1).uniform(-1, 1, (1, N))
  bank = alz.FilterBank([(b, a)], n_inputs=1)
  bank.reset()
  assert same_bits(bank.process(x, layout="chan"), oracle.bank([3], [3], b, a, x, layout="chan"))


@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("gap", [0, 7])
def test_rows_with_gaps(alz, layout, gap):
  C, N = 101, 60003                           # 48 MB in, 48 MB out
  b, a = resonators(C)
  rng = np.random.default_rng(2)
  rows, cols = (N, C) if layout == "time" else (C, N)
  xw, yw = rng.uniform(-1, 1, (rows, cols + gap)), np.full((rows, cols + 2 * gap), -7.5)
  bank = alz.FilterBank([(b, a)], n_inputs=C)
  bank.reset()
  dp = ctypes.POINTER(ctypes.c_double)
  from audiolazy_amd import _ffi
  _ffi.check(bank._L.alz_bank_process_host(bank._h, xw.ctypes.data_as(dp), yw.ctypes.data_as(dp), N,
                                           _ffi.TIME_MAJOR if layout == "time" else _ffi.CHAN_MAJOR, cols + gap, cols + 2 * gap))
  ref = oracle.bank([3], [3], b, a, np.ascontiguousarray(xw[:, :cols]), layout=layout)
  assert same_bits(np.ascontiguousarray(yw[:, :cols]), ref) and (yw[:, cols:] == -7.5).all()


@pytest.mark.parametrize("layout", ["time", "chan"])
def test_more_outputs_than_inputs_and_in_place(alz, layout):
  sets, N = 33, 300001                        # 2.4 MB in, 79 MB out
  b, a = resonators(sets)
  x = np.random.default_rng(3).uniform(-1, 1, (N, 1) if layout == "time" else (1, N))
  bank = alz.FilterBank([(b, a)], n_inputs=1, mode="outer")
  bank.reset()
  y = bank.process(x, layout=layout)
  wide = np.repeat(x, sets, axis=1 if layout == "time" else 0)
  assert same_bits(y, oracle.bank([3], [3], b, a, np.ascontiguousarray(wide), layout=layout))
  # the block as its own result: a diagonal bank over the outputs
  twin = alz.FilterBank([(b, a)], n_inputs=sets)
  twin.reset()
  ref = oracle.bank([3], [3], b, a, y, layout=layout)
  assert twin.process(y, layout=layout, out=y) is y and same_bits(y, ref)
