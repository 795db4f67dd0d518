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


@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("nb,na", [(1, 1), (1, 3), (3, 1), (3, 2), (6, 4)])
def test_process_block_updates_the_callers_histories(alz, layout, nb, na):
  import torch
  from audiolazy_amd import timevar
  C, N, cut = 70, 300, 113
  rng = np.random.default_rng(10 * nb + na)
  x, s = rng.uniform(-1, 1, (N, C)), rng.uniform(.1, .4, N)
  b, a = [.5] * (nb - 1), [1.] + [.1] * (na - 1)
  xh, xh_ok = guarded((nb - 1, C))
  yh, yh_ok = guarded((na - 1, C))
  xh.fill_(.25)
  yh.fill_(.25)

  def part(lo, hi):
    blk = x[lo:hi] if layout == "time" else x[lo:hi].T
    y = timevar.process_block([torch.from_numpy(s[lo:hi].copy()).cuda()] + b, a, torch.from_numpy(np.ascontiguousarray(blk)).cuda(),
                              xh=xh, yh=yh, zero=.25, layout=layout).cpu().numpy()
    assert xh_ok() and yh_ok()
    return y if layout == "time" else y.T
  y = np.concatenate([part(0, cut), part(cut, N)])
  for ch in (0, 1, 33, 69):
    assert same_bits(y[:, ch], oracle.tv_df1([s] + b, a, x[:, ch], zero=.25)), ch
  assert same_bits(xh.cpu().numpy(), x[N - nb + 1:][::-1]) and same_bits(yh.cpu().numpy(), y[N - na + 1:][::-1])


def test_empty_blocks(alz):
  """An empty block through every torch entry point: an empty result, and the state of the stream as it was."""
  import torch
  from audiolazy_amd import maps, pcm, timevar
  from audiolazy_amd.bank import mix_sets, mix_tracks
  from audiolazy_amd.lpc import kautocor_frames
  f64 = lambda *shape: torch.empty(shape, dtype=torch.float64, device="cuda")
  bank = alz.FilterBank([([1.], [1., .5])], n_inputs=4)
  bank.reset(zero=.25)
  assert tuple(bank.process(f64(0, 4)).shape) == (0, 4) and (bank.get_state()[1] == .25).all()
  assert tuple(maps.map_block("abs", f64(0, 4)).shape) == (0, 4)
  assert tuple(mix_sets(f64(0, 12), 3, 4).shape) == (0, 4)
  assert tuple(mix_tracks([f64(0), f64(0)], [0, 0]).shape) == (0,)
  assert mix_tracks([f64(0), f64(0)], [0, 3], zero=.5).tolist() == [.5] * 3
  yh = torch.full((1, 4), .25, dtype=torch.float64, device="cuda")
  assert tuple(timevar.process_block([1., f64(0)], [1., .5], f64(0, 4), yh=yh).shape) == (0, 4) and bool((yh == .25).all())
  assert tuple(pcm.encode_pcm(f64(0), "h").shape) == (0,)
  assert tuple(pcm.decode_pcm(torch.empty(0, dtype=torch.uint8, device="cuda"), 24).shape) == (0,)
  assert tuple(kautocor_frames(f64(479), 480, 8)[0].shape) == (0, 9)
