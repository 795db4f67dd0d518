"""Blocks of more than 2^32 samples (a filterbank over some minutes of sound): one launch has at most 2^32 work-items, so the passes that
take one sample each go in slices.  Checked around the places where a 32-bit index would wrap."""
import numpy as np
import pytest

from oracle import oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def alz():
  import torch
  import audiolazy_amd
  audiolazy_amd.load_library()
  assert audiolazy_amd.device_count() >= 1, "no HIP device: the engine has no CPU path"
  yield audiolazy_amd
  torch.cuda.empty_cache()


def same_bits(a, b):
  return a.shape == b.shape and bool(np.array_equal(a.view(np.uint64), b.view(np.uint64)))


@pytest.mark.parametrize("layout", ["time", "chan"])
def test_bank_of_bands_on_one_stream(alz, layout):
  import bench
  import torch
  B, N = 256, (1 << 24) + 37
  b, a = bench.resonator_coefs(B)
  x = np.random.default_rng(1).uniform(-1, 1, N)
  bank = alz.FilterBank([(b, a)], n_inputs=1, mode="outer")
  bank.reset()
  xd = torch.from_numpy(x).cuda().view((N, 1) if layout == "time" else (1, N))
  y = bank.process(xd, layout=layout)
  for band in (0, 1, 127, 254, 255):
    ref = oracle.bank([3], [3], b[band], a[band], x[None, :], layout="chan")[0]
    got = (y[:, band] if layout == "time" else y[band]).contiguous().cpu().numpy()
    assert same_bits(got, ref), band
  del y, bank
  torch.cuda.empty_cache()


def test_mix_and_tracks(alz):
  import torch
  from audiolazy_amd.bank import mix_sets, mix_tracks
  n, c = (1 << 22) + 3, 1024
  y = torch.empty((2, n, c), dtype=torch.float64, device="cuda").uniform_(-1, 1)
  ends = [0, 5, (1 << 22) - 1, 1 << 22, n - 1]
  out = mix_sets(y.view(2 * n, c), 2, n, layout="chan")          # (channel-major: a set is n rows of c samples)
  assert tuple(out.shape) == (n, c)
  for r in ends:
    assert torch.equal(out[r], y[0, r] + y[1, r]), r
  late = torch.ones(1000, dtype=torch.float64, device="cuda")
  start = (1 << 32) + 100
  flat = out.view(-1)
  total = mix_tracks([flat, late], [0, start], zero=.5)
  want = torch.full((2000,), .5, dtype=torch.float64, device="cuda") + flat[start - 500:start + 1500]
  want[500:1500] += 1.
  assert torch.equal(total[start - 500:start + 1500], want) and torch.equal(total[:1000], .5 + flat[:1000])
  assert float(total[-1]) == .5 + float(flat[-1])
  del y, out, total, flat, want
  torch.cuda.empty_cache()


@pytest.mark.parametrize("order", [9, 8])                        # (lags by (frame, lag) pairs; by frames)
def test_frames(alz, order):
  import torch
  from audiolazy_amd.lpc import kautocor_frames
  L, F = 32, ((1 << 32) + 1000) // (order + 1)
  sig = torch.empty(F - 1 + L, dtype=torch.float64, device="cuda").uniform_(-1, 1)
  coefs, err, status = kautocor_frames(sig, L, order, hop=1)
  torch.cuda.synchronize()
  for f in [0, 1, F // 2, F - 1000, F - 64, F - 1, (1 << 25) - 1, 1 << 25, (1 << 28) + 5]:
    rc, re, rst = oracle.kautocor_frames(sig[f:f + L].cpu().numpy(), 1, L, L, order)
    c, e = coefs[f].cpu().numpy(), float(err[f])
    assert int(status[f]) == rst[0] == 0 and np.abs(c - rc[0]).max() <= 1e-9 * np.abs(rc[0]).max() and abs(e - re[0]) <= 1e-9 * re[0], f
  del sig, coefs, err, status
  torch.cuda.empty_cache()
