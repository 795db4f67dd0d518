"""One stream of blocks through one bank, some of them torch tensors on a stream of the caller's and some NumPy arrays: a host block
continues from the state that the device block before it leaves, however late that one runs."""
import ctypes
import os

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


@pytest.fixture(scope="module")
def hold():
  """hold(ms, stream): keeps ``stream`` busy (a few workgroups that wait for the clock) for a while"""
  lib = ctypes.CDLL(os.path.join(os.path.dirname(os.path.abspath(__file__)), "helpers", "libhog.so"))
  lib.hog_launch.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p]

  def run(ms, stream):
    assert lib.hog_launch(4, 1024, ms * 1000, stream.cuda_stream) == 0
  return run


def same_bits(a, b):
  return a.shape == b.shape and bool(np.array_equal(a.view(np.uint64), b.view(np.uint64)))


@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("C,N", [(64, 500), (512, 10000)])          # (the synchronous path; the pipelined one)
def test_host_block_after_a_device_block(alz, hold, C, N, layout):
  import bench
  import torch
  b, a = bench.resonator_coefs(C)
  x = np.random.default_rng(C).uniform(-1, 1, (3 * N, C))
  ref = oracle.bank([3], [3], b, a, x, layout="time")
  part = lambda v, k: np.ascontiguousarray(v[k * N:(k + 1) * N] if layout == "time" else v[k * N:(k + 1) * N].T)
  bank = alz.FilterBank([(b, a)], n_inputs=C)
  bank.process(part(x, 0), layout=layout)          # (streams, buffers and kernels are there before anything is held)
  side = torch.cuda.Stream()
  bank.reset()
  x0, x2 = (torch.from_numpy(part(x, k)).cuda() for k in (0, 2))
  torch.cuda.synchronize()
  with torch.cuda.stream(side):
    hold(150, side)
    y0 = bank.process(x0, layout=layout)
  y1 = bank.process(part(x, 1), layout=layout)
  with torch.cuda.stream(side):
    y2 = bank.process(x2, layout=layout)
  torch.cuda.synchronize()
  assert same_bits(y0.cpu().numpy(), part(ref, 0)) and same_bits(y1, part(ref, 1)) and same_bits(y2.cpu().numpy(), part(ref, 2))
