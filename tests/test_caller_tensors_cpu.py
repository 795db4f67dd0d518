"""The torch entry points take a caller's tensors by address, so what the kernels assume about them -- place, item type, extent,
order -- is checked on the host before any library call.  The library is a stub here that records its calls: a refusal must come
before the first of them.  ``dev`` makes a host tensor that says it lies on a device."""
import ctypes
import types

import numpy as np
import pytest
import torch

from audiolazy_amd import _ffi, timevar
from audiolazy_amd.bank import FilterBank, mix_sets
from audiolazy_amd.lpc import kautocor_frames


class _Dev(torch.Tensor):
  is_cuda = True


_Dev.__module__ = "torch"      # (the entry points tell tensors from arrays by the type's module)


def dev(shape, dtype=torch.float64):
  return torch.zeros(shape, dtype=dtype).as_subclass(_Dev)


class _Lib(object):
  def __init__(self):
    self.calls = []

  def __getattr__(self, name):
    def entry(*args):
      self.calls.append((name, args))
      return 0
    return entry


@pytest.fixture
def lib(monkeypatch):
  stub = _Lib()
  monkeypatch.setattr(_ffi, "load", lambda: stub)
  monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=0))
  return stub


# ---- lpc.kautocor_frames ------------------------------------------------------------------------
@pytest.mark.parametrize("sig", [torch.zeros(960, dtype=torch.float64), torch.zeros((2, 480), dtype=torch.float64),
                                 dev(960, torch.float32), dev(960, torch.int64), dev(960, torch.bfloat16)],
                         ids=["host", "host-2d", "float32", "int64", "bfloat16"])
@pytest.mark.parametrize("with_out", [False, True])
def test_kautocor_frames_refuses_other_signals(lib, sig, with_out):
  out = (dev((2, 9)), dev(2), dev(2, torch.int32)) if with_out else None
  with pytest.raises(ValueError):
    kautocor_frames(sig, 480, 8, out=out)
  assert not lib.calls


def test_kautocor_frames_hands_over_the_signal(lib):
  sig = dev(960)
  coefs, err, status = kautocor_frames(sig, 480, 8)
  (name, args), = lib.calls
  assert name == "alz_lpc_kautocor_dev_ex" and args[:5] == (sig.data_ptr(), 2, 480, 480, 8)
  assert args[5:8] == (coefs.data_ptr(), err.data_ptr(), status.data_ptr())


# ---- mix_sets / FilterBank.mixdown --------------------------------------------------------------
# 3 sets of 4 inputs, 10 samples: the mix is 40 doubles
@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("kind", ["short", "long", "flat", "transposed", "float32", "strided", "host", "array"])
def test_mix_sets_refuses_other_results(lib, layout, kind):
  shape = (10, 4) if layout == "time" else (4, 10)
  y = dev((10, 12) if layout == "time" else (12, 10))
  out = {"short": lambda: dev((shape[0] - 1, shape[1])), "long": lambda: dev((shape[0] + 1, shape[1])), "flat": lambda: dev(40),
         "transposed": lambda: dev(shape[::-1]), "float32": lambda: dev(shape, torch.float32),
         "strided": lambda: dev((shape[0], 2 * shape[1]))[:, ::2], "host": lambda: torch.zeros(shape, dtype=torch.float64),
         "array": lambda: np.zeros(shape)}[kind]()
  with pytest.raises(ValueError):
    mix_sets(y, 3, 4, layout=layout, out=out)
  assert not lib.calls


@pytest.mark.parametrize("layout", ["time", "chan"])
def test_mix_sets_writes_the_callers_result(lib, layout):
  out = dev((10, 4) if layout == "time" else (4, 10))
  assert mix_sets(dev((10, 12) if layout == "time" else (12, 10)), 3, 4, layout=layout, out=out) is out
  (name, args), = lib.calls
  assert name == "alz_mix_dev" and args[7] == out.data_ptr()


# ---- timevar.process_block ----------------------------------------------------------------------
# 3 numerator and 2 denominator taps, 10 samples of 4 channels: xh is [2, 4], yh is [1, 4]
@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("side", ["xh", "yh"])
@pytest.mark.parametrize("kind", ["rows", "columns", "flat", "transposed", "float32", "strided", "host", "array"])
def test_process_block_refuses_other_histories(lib, layout, side, kind):
  rows = {"xh": 2, "yh": 1}[side]
  bad = {"rows": lambda: dev((rows - 1, 4)), "columns": lambda: dev((rows, 3)), "flat": lambda: dev(rows * 4),
         "transposed": lambda: dev((4, rows)), "float32": lambda: dev((rows, 4), torch.float32),
         "strided": lambda: dev((rows, 8))[:, ::2], "host": lambda: torch.zeros((rows, 4), dtype=torch.float64),
         "array": lambda: np.zeros((rows, 4))}[kind]()
  with pytest.raises(ValueError):
    timevar.process_block([1., .5, .25], [1., .5], dev((10, 4) if layout == "time" else (4, 10)), layout=layout, **{side: bad})
  assert not lib.calls


@pytest.mark.parametrize("nb,na", [(1, 1), (1, 3), (3, 1), (3, 2)])
@pytest.mark.parametrize("spare", [0, 1])        # (a side without history: no row, or the one row of the default)
def test_process_block_takes_the_callers_histories(lib, nb, na, spare):
  xh, yh = dev((max(nb - 1, spare), 4)), dev((max(na - 1, spare), 4))
  timevar.process_block([1.] * nb, [1.] * na, dev((10, 4)), xh=xh, yh=yh)
  (name, args), = lib.calls
  assert name == "alz_tv_process_dev" and args[11:13] == (xh.data_ptr(), yh.data_ptr())


# ---- FilterBank.process on arrays ---------------------------------------------------------------
@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("kind", ["short", "transposed", "flat", "float32", "strided", "fortran", "read-only", "tensor", "list"])
def test_process_refuses_other_results(lib, layout, kind):
  bank = FilterBank([([1.], [1., .5])], n_inputs=4)
  del lib.calls[:]
  shape = (10, 4) if layout == "time" else (4, 10)
  out = {"short": lambda: np.zeros((shape[0] - 1, shape[1])), "transposed": lambda: np.zeros(shape[::-1]), "flat": lambda: np.zeros(40),
         "float32": lambda: np.zeros(shape, np.float32), "strided": lambda: np.zeros((shape[0], 2 * shape[1]))[:, ::2],
         "fortran": lambda: np.zeros(shape, order="F"), "read-only": lambda: np.broadcast_to(np.zeros(shape[1]), shape),
         "tensor": lambda: torch.zeros(shape, dtype=torch.float64), "list": lambda: [[0.] * shape[1]] * shape[0]}[kind]()
  with pytest.raises(ValueError):
    bank.process(np.zeros(shape), layout=layout, out=out)
  assert not lib.calls


@pytest.mark.parametrize("layout", ["time", "chan"])
def test_process_writes_the_callers_result(lib, layout):
  def written(bank, x, out):
    del lib.calls[:]
    assert bank.process(x, layout=layout, out=out) is out
    (name, args), = lib.calls
    return name == "alz_bank_process_host" and ctypes.cast(args[2], ctypes.c_void_p).value == out.ctypes.data
  shape = (10, 4) if layout == "time" else (4, 10)
  assert written(FilterBank([([1.], [1., .5])], n_inputs=4), np.zeros(shape), np.zeros(shape))
  one = FilterBank([([1.], [1., .5])], n_inputs=1)
  assert written(one, np.zeros(10), np.zeros((10, 1) if layout == "time" else (1, 10)))
  assert written(one, np.zeros(10), np.zeros(10))        # (a flat block and its flat result)


# ---- one device for the tensors of a call -------------------------------------------------------
class _Elsewhere(_Dev):
  device = torch.device("cuda", 1)


_Elsewhere.__module__ = "torch"


def elsewhere(*args, **kw):
  return dev(*args, **kw).as_subclass(_Elsewhere)


def test_tensors_of_another_device_are_refused(lib):
  from audiolazy_amd import sharding
  from audiolazy_amd.bank import mix_tracks
  from audiolazy_amd.maps import map_block
  bank = FilterBank([([1.], [1., .5])], n_inputs=4)            # (a bank of device 0)
  comm = sharding.DirectComm(0, 1, bytes(128), device=0)
  del lib.calls[:]
  for call in (lambda: bank.process(elsewhere((10, 4))), lambda: bank.process(dev((10, 4)), out=elsewhere((10, 4))),
               lambda: map_block("add2", dev(10), other=elsewhere(10)), lambda: map_block("abs", dev(10), out=elsewhere(10)),
               lambda: mix_tracks([dev(10), elsewhere(10)], [0, 3]), lambda: mix_sets(dev((10, 12)), 3, 4, out=elsewhere((10, 4))),
               lambda: timevar.process_block([elsewhere(10)], [1., .5], dev((10, 4))),
               lambda: timevar.process_block([1.], [1., elsewhere((10, 4))], dev((10, 4))),
               lambda: timevar.process_block([1., .5], [1.], dev((10, 4)), xh=elsewhere((1, 4))),
               lambda: kautocor_frames(dev(960), 480, 8, out=(elsewhere((2, 9)), dev(2), dev(2, torch.int32))),
               lambda: comm.gather(elsewhere(10)), lambda: comm.sum(elsewhere(10))):
    with pytest.raises(ValueError):
      call()
    assert not lib.calls


def test_tensors_of_the_banks_device_are_taken(lib):
  from audiolazy_amd.bank import mix_tracks
  from audiolazy_amd.maps import map_block
  bank = FilterBank([([1.], [1., .5])], n_inputs=4)
  del lib.calls[:]
  bank.process(dev((10, 4)), out=dev((10, 4)))
  map_block("add2", dev(10), other=dev(10), out=dev(10))
  mix_tracks([dev(10), dev(7), dev(0)], [0, 3, 2])
  timevar.process_block([dev(10)], [1., dev((10, 4))], dev((10, 4)))
  assert [name for name, _ in lib.calls] == ["alz_bank_process_dev", "alz_map_dev", "alz_mix_tracks_dev", "alz_tv_process_dev"]


# ---- nothing to do ------------------------------------------------------------------------------
def test_empty_blocks(lib):
  """A stream that ends on a block boundary hands over an empty last block: an empty result, like the array forms give."""
  from audiolazy_amd.bank import mix_tracks
  from audiolazy_amd.maps import map_block
  from audiolazy_amd.pcm import decode_pcm, encode_pcm
  assert tuple(map_block("abs", dev((0, 4))).shape) == (0, 4)
  assert tuple(map_block("sqrt", dev(0)).shape) == (0,)
  assert tuple(map_block("add2", dev((4, 0)), other=dev((4, 0))).shape) == (4, 0)
  out = dev((0, 4))
  assert map_block("neg", dev((0, 4)), out=out) is out
  assert tuple(mix_sets(dev((0, 12)), 3, 4).shape) == (0, 4) and tuple(mix_sets(dev((12, 0)), 3, 4, layout="chan").shape) == (4, 0)
  assert mix_sets(dev((0, 12)), 3, 4, out=out) is out
  out = np.zeros((0, 4))
  assert mix_sets(np.zeros((0, 12)), 3, 4, out=out) is out
  assert tuple(mix_tracks([dev(0)], [0]).shape) == (0,) and tuple(mix_tracks([dev(0), dev(0)], [0, 0]).shape) == (0,)
  assert tuple(timevar.process_block([1., dev(0)], [1., .5], dev((0, 4))).shape) == (0, 4)
  assert tuple(timevar.process_block([1.], [1., dev(0)], dev((4, 0)), layout="chan").shape) == (4, 0)
  raw = decode_pcm(dev(0, torch.uint8), 16)
  assert tuple(raw.shape) == (0,) and raw.dtype == torch.float64
  packed = encode_pcm(dev(0), "h")
  assert tuple(packed.shape) == (0,) and packed.dtype == torch.uint8
  coefs, err, status = kautocor_frames(dev(479), 480, 8)
  assert (tuple(coefs.shape), tuple(err.shape), tuple(status.shape)) == ((0, 9), (0,), (0,))
  assert not lib.calls


@pytest.mark.parametrize("shift", [-3, -1, 0, 1, 3])
def test_process_on_arrays_that_overlap(lib, shift):
  """The result may be the input itself; a result that lies across it must not be written while the input is still read."""
  bank = FilterBank([([1.], [1., .5])], n_inputs=4)
  base = np.arange(80.).reshape(20, 4)
  x, out = base[5:15], base[5 + shift:15 + shift]
  del lib.calls[:]
  bank.process(x, out=out)
  (name, args), = lib.calls
  read = np.ctypeslib.as_array(args[1], (10, 4))
  assert np.array_equal(read, x) and ctypes.cast(args[2], ctypes.c_void_p).value == out.ctypes.data
  assert np.shares_memory(read, out) == (shift == 0)


def test_process_on_a_larger_result_that_begins_with_the_input(lib):
  bank = FilterBank([([1.], np.array([[1., .5], [1., .25], [1., .125]]))], n_inputs=1, mode="outer")
  base = np.arange(30.)
  del lib.calls[:]
  bank.process(base[:10].reshape(10, 1), out=base.reshape(10, 3))
  (name, args), = lib.calls
  assert not np.shares_memory(np.ctypeslib.as_array(args[1], (10, 1)), base)
