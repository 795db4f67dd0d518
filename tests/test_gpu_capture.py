"""A process call of a long feedback-free section captured into a graph before the bank has its pacing slab (include/alz.h): the launch
runs free, every replay continues the stream with the eager call's doubles, and the bank is usable eagerly in between and behind."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def alz():
  import audiolazy_amd
  audiolazy_amd.load_library()
  assert audiolazy_amd.device_count() >= 1, "no HIP device: the engine has no CPU path"
  return audiolazy_amd


def test_fir_chains_captured_before_the_first_eager_call(alz):
  import torch
  C, N, nb = 8192, 98304, 256                      # (the fewest rows that take chains of waves with pacing)
  taps = np.random.default_rng(9).uniform(-1, 1, nb)
  make = lambda: alz.FilterBank([(taps, np.array([1.0]))], n_inputs=C)
  gen = torch.Generator(device="cuda")
  gen.manual_seed(3)
  noise = lambda: torch.rand((N, C), dtype=torch.float64, device="cuda", generator=gen) - .5
  eager, bank = make(), make()
  eager.reset(zero=.25)
  bank.reset(zero=.25)
  x, y, ref = noise(), torch.zeros((N, C), dtype=torch.float64, device="cuda"), torch.empty((N, C), dtype=torch.float64, device="cuda")
  eager.process(x, out=ref)
  assert "chains" in eager.last_kernel, eager.last_kernel
  eager.reset(zero=.25)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    bank.process(x, out=y)
  assert "chains" in bank.last_kernel, bank.last_kernel
  for k in range(3):
    if k:
      x.copy_(noise())
    graph.replay()
    eager.process(x, out=ref)
    torch.cuda.synchronize()
    assert torch.equal(y, ref), k
    y.zero_()
  for k in range(2):                               # (these make the slab and use it)
    x.copy_(noise())
    assert torch.equal(bank.process(x), eager.process(x, out=ref)), k
  x.copy_(noise())
  graph.replay()
  assert torch.equal(y, eager.process(x, out=ref))
  a, b = bank.get_state(), eager.get_state()
  assert np.array_equal(a[0].view(np.uint64), b[0].view(np.uint64))
