"""Result and state tensors that the caller brings, on the device: the calls that the host checks let through write exactly those
buffers -- the doubles beside them stay as they were -- and give the doubles of the call without them."""
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
  a, b = np.asarray(a), np.asarray(b)
  return a.shape == b.shape and bool(np.array_equal(a.view(np.uint64), b.view(np.uint64)))


def guarded(shape):
  """(tensor of ``shape`` inside a larger buffer, check that the buffer around it is untouched)"""
  import torch
  n = int(np.prod(shape))
  base = torch.full((n + 256,), -7.5, dtype=torch.float64, device="cuda")

  def untouched():
    return bool((base[:128] == -7.5).all()) and bool((base[128 + n:] == -7.5).all())
  return base[128:128 + n].view(shape), untouched


@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("n_sets,n_inputs,n", [(1, 5, 33), (3, 1, 1000), (9, 7, 257), (20, 64, 512)])
def test_mix_sets_into_the_callers_result(alz, layout, n_sets, n_inputs, n):
  import torch
  from audiolazy_amd.bank import mix_sets
  y = np.random.default_rng(n).uniform(-1, 1, (n, n_sets * n_inputs) if layout == "time" else (n_sets * n_inputs, n))
  out, untouched = guarded((n, n_inputs) if layout == "time" else (n_inputs, n))
  assert mix_sets(torch.from_numpy(y).cuda(), n_sets, n_inputs, layout=layout, out=out) is out
  assert same_bits(out.cpu().numpy(), oracle.mix(y, n_sets, n_inputs, layout=layout)) and untouched()
