"""Process calls captured into a graph: every replay continues the stream like the eager call, and the bank is usable eagerly in
between and behind -- with other block lengths, whose scratch and tables are not those of the graph.  What a capture cannot allocate
is refused; the one-pass time-parallel kernel, whose launches need a key of their own, leaves a captured block to the three-launch
form."""
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


def noise(shape, seed):
  import torch
  gen = torch.Generator(device="cuda")
  gen.manual_seed(seed)
  return torch.rand(shape, dtype=torch.float64, device="cuda", generator=gen) - .5


def play(make, shape, layout, close, other=None, warm=True):
  """A bank captured at one block shape and its twin that makes every call eagerly, side by side: replays, eager calls of the same
  shape and of ``other`` (larger, then smaller) in turn."""
  import torch
  eager, bank = make(), make()
  x = noise(shape, 1)
  ref = eager.process(x, layout=layout)
  y = torch.zeros_like(ref)
  if warm:
    bank.process(x, layout=layout, out=y)
  eager.reset(zero=.125)
  bank.reset(zero=.125)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    bank.process(x, layout=layout, out=y)
  assert bank.last_kernel
  turn = 2
  for step in ["replay", "replay", "eager", "replay", "large", "replay", "small", "replay", "replay"]:
    if step in ("large", "small") and other is None:
      continue
    if step == "replay":
      x.copy_(noise(shape, turn))
      y.zero_()
      graph.replay()
      got, want = y, eager.process(x, layout=layout)
    else:
      blk = noise({"eager": shape, "large": other and other[0], "small": other and other[1]}[step], turn)
      got, want = bank.process(blk, layout=layout), eager.process(blk, layout=layout)
    torch.cuda.synchronize()
    close(got, want, step)
    turn += 1
  torch.cuda.synchronize()
  for a, b in zip(bank.get_state(), eager.get_state()):
    close(a, b, "state")
  return bank, eager


def bits(got, want, what):
  got, want = (v.cpu().numpy() if hasattr(v, "cpu") else v for v in (got, want))
  assert np.array_equal(got.view(np.uint64), want.view(np.uint64)), what


def near(got, want, what):
  got, want = (v.cpu().numpy() if hasattr(v, "cpu") else v for v in (got, want))
  assert np.abs(got - want).max() <= 1e-9 * np.abs(want).max(), what      # (the mode's own bar in the tests of its kernels)


def biquads(alz, C, **kw):
  import bench
  b, a = bench.resonator_coefs(C)
  return alz.FilterBank([(b, a)], n_inputs=C, **kw)


@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("C,N", [(1, 3001), (70, 5000), (4096, 4096), (4096, 65536)])
def test_biquad_banks(alz, C, N, layout):
  shapes = [(n, C) if layout == "time" else (C, n) for n in (N, N + 700, 333)]
  play(lambda: biquads(alz, C), shapes[0], layout, bits, shapes[1:], warm=False)


def test_input_map_and_scratch(alz):
  """A map as a pass of its own (its block is scratch of the bank) and a second section that cannot run in place (so is its copy)."""
  rng = np.random.default_rng(5)
  C, taps = 96, rng.uniform(-1, 1, 40)

  def make():
    return alz.FilterBank([([1., .5], [1., -.5]), (taps, [1.])], n_inputs=C).set_input_map("square")
  play(make, (2000, C), "time", bits, [(9000, C), (100, C)])


def test_scratch_is_refused_in_a_capture(alz):
  import torch
  C = 96
  make = lambda: alz.FilterBank([([1., .5], [1., -.5])], n_inputs=C).set_input_map("square")
  bank, twin = make(), make()
  x = noise((500, C), 3)
  want = twin.process(x)
  y = torch.zeros_like(x)
  torch.cuda.synchronize()
  with pytest.raises(NotImplementedError, match="before the capture"):
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
      y.add_(1.)
      bank.process(x, out=y)
  torch.cuda.synchronize()
  bits(bank.process(x), want, "after the refusal")


def test_section_pipeline(alz):
  """A narrow cascade whose sections run on streams of the bank, chunk by chunk."""
  import bench
  C, N = 64, 4 * 16384 + 100
  b, a = bench.resonator_coefs(C)
  bank, _ = play(lambda: alz.FilterBank([(b, a)] * 3, n_inputs=C), (N, C), "time", bits, [(N + 20000, C), (70000, C)])
  assert "section pipeline" in bank.last_kernel


@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("C,mode", [(256, 1024), (64, True)])          # (both the three-launch form)
def test_time_parallel_bank(alz, layout, C, mode):
  N = 1 << 16
  shapes = [(n, C) if layout == "time" else (C, n) for n in (N, 2 * N + 64, 4096)]
  bank, _ = play(lambda: biquads(alz, C).set_time_parallel(mode), shapes[0], layout, near, shapes[1:])
  assert "k_scan(k_" in bank.last_kernel and "k_look" not in bank.last_kernel, bank.last_kernel


@pytest.mark.parametrize("mode", [True, "one-pass"])
def test_the_one_pass_form_refuses_a_capture(alz, mode):
  import torch
  make = lambda: biquads(alz, 256).set_time_parallel(mode)
  bank, eager = make(), make()
  x = noise((1 << 16, 256), 1)
  y = torch.zeros_like(x)
  near(bank.process(x), eager.process(x), "before")
  assert "k_look" in bank.last_kernel, bank.last_kernel
  torch.cuda.synchronize()
  with pytest.raises(NotImplementedError, match="chunk length"):
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
      y.add_(1.)
      bank.process(x, out=y)
  torch.cuda.synchronize()
  near(bank.process(x), eager.process(x), "after the refusal")


@pytest.mark.parametrize("layout", ["time", "chan"])
def test_time_parallel_cascade(alz, layout):
  s, Hz = alz.sHz(48000)
  fcs = [f * Hz for f in alz.erb_space(100., 8000., 64)]
  N = 1 << 18
  shapes = [(n, 1) if layout == "time" else (1, n) for n in (N, 2 * N, N // 2)]
  bank, _ = play(lambda: alz.gammatone_bank(fcs, 1, strategy="slaney", Hz=Hz).set_time_parallel(True), shapes[0], layout, near, shapes[1:])
  assert "k_cscan" in bank.last_kernel, bank.last_kernel


def test_operations_beside_the_bank(alz):
  """A time-varying block, elementwise stages, a mix and an LPC batch in one graph."""
  import torch
  from audiolazy_amd import maps, timevar
  from audiolazy_amd.bank import mix_sets
  from audiolazy_amd.lpc import kautocor_frames
  N, C = 4800, 64
  x, b0 = noise((N, C), 1), noise(N, 2)
  yh = torch.zeros((1, C), dtype=torch.float64, device="cuda")

  def run():
    y = timevar.process_block([b0], [1., .5], maps.map_block("abs", x), yh=yh)
    m = mix_sets(maps.add_blocks(y, x), 4, 16)
    return [y, m] + list(kautocor_frames(m, 480, 16)) + list(kautocor_frames(m, 480, 16, exact=True))
  run()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  yh.zero_()
  with torch.cuda.graph(graph):
    outs = run()
  for k in range(3):
    x.copy_(noise((N, C), 10 + k))
    yh.fill_(.5)
    want = [v.clone() for v in run()]
    state = yh.clone()
    yh.fill_(.5)
    for v in outs:
      v.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(yh, state) and all(torch.equal(a, b) for a, b in zip(outs, want)), k
