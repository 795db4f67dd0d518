"""Frames of odd length in batches large enough for the one-launch kernel (16 384 frames and more, an even hop): the last sample of
such a frame belongs to the sums like every other one."""
import numpy as np
import pytest

from oracle import oracle

pytestmark = pytest.mark.gpu

F = 16400


@pytest.fixture(scope="module")
def lpc():
  import importlib
  import audiolazy_amd
  assert audiolazy_amd.device_count() >= 1, "no HIP device: the engine has no CPU path"
  return importlib.import_module("audiolazy_amd.lpc")


def same_bits(a, b):
  a, b = np.asarray(a, dtype=np.float64), np.asarray(b, dtype=np.float64)
  return a.shape == b.shape and bool(np.array_equal(a.view(np.uint64), b.view(np.uint64)))


def signal(frame_len, hop):
  return np.random.default_rng(frame_len * 1000 + hop).uniform(-1, 1, (F - 1) * hop + frame_len)


@pytest.mark.parametrize("order", [8, 16, 24, 32])
@pytest.mark.parametrize("frame_len,hop", [(33, 32), (35, 2), (63, 64), (65, 32), (479, 240), (481, 240), (480, 240), (66, 32)])
def test_lags(lpc, frame_len, hop, order):
  sig = signal(frame_len, hop)
  r = lpc.acorr_frames(sig, frame_len, order, hop=hop)
  for f in [0, 1, 63, 64, F // 2, F - 2, F - 1]:
    assert same_bits(r[f], oracle.acorr(sig[f * hop:f * hop + frame_len], order)), f


@pytest.mark.parametrize("exact,fused", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("frame_len,hop,order", [(33, 32, 8), (65, 32, 16), (481, 240, 16), (479, 240, 10), (480, 240, 16), (65, 64, 32)])
def test_coefficients(lpc, frame_len, hop, order, exact, fused):
  import torch
  sig = signal(frame_len, hop)
  rc, re, rst = oracle.kautocor_frames(sig, F, frame_len, hop, order)
  for s in (sig, torch.from_numpy(sig).cuda()):
    c, e, st = lpc.kautocor_frames(s, frame_len, order, hop=hop, exact=exact, fused=fused)
    c, e, st = (np.asarray(v.cpu() if hasattr(v, "cpu") else v) for v in (c, e, st))
    assert np.array_equal(st, rst)
    if exact:
      assert same_bits(c, rc) and same_bits(e, re)
    else:
      # the recursion's own bar against the reference's dense form
      assert np.abs(c - rc).max() / np.abs(rc).max() <= 1e-9 and np.abs(e - re).max() / np.abs(re).max() <= 1e-9
