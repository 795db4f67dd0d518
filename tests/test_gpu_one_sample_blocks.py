"""Blocks of a single sample, whose rows of one item lie at a pitch of one: a channel-major block then has the strides of a time-major
one.  A stream cut into such blocks and longer ones gives the doubles of the whole stream."""
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


KINDS = {"fir17": ([17], [1]), "fir40": ([40], [1]), "fir129": ([129], [1]), "biquad": ([3], [3]), "cascade": ([2, 2, 2, 2], [3, 3, 3, 3]),
         "order6": ([7], [7]), "order12": ([5], [13]), "fir and poles": ([20, 1], [1, 3])}


@pytest.mark.parametrize("layout", ["time", "chan"])
@pytest.mark.parametrize("source", ["tensor", "in place", "array"])
@pytest.mark.parametrize("C", [1, 3, 48, 64, 130, 512])
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_blocks(alz, kind, C, source, layout):
  import torch
  nbs, nas = KINDS[kind]
  rng = np.random.default_rng(C + len(kind))
  secs = [(rng.uniform(-1, 1, nb), np.r_[1., rng.uniform(-.8, .8, na - 1) / max(na - 1, 1)]) for nb, na in zip(nbs, nas)]
  bank = alz.FilterBank(secs, n_inputs=C)
  bank.reset()
  lens = [1, 127, 1, 1, 15, 1, 2]
  x = rng.uniform(-1, 1, (sum(lens), C))
  ref = oracle.bank(nbs, nas, np.concatenate([s[0] for s in secs]), np.concatenate([s[1] for s in secs]), x, layout="time")
  at = 0
  for n in lens:
    blk = np.ascontiguousarray(x[at:at + n] if layout == "time" else x[at:at + n].T)
    if source == "array":
      y = bank.process(blk, layout=layout)
    else:
      xd = torch.from_numpy(blk).cuda()
      y = bank.process(xd, layout=layout, out=xd if source == "in place" else None).cpu().numpy()
    y = np.ascontiguousarray(y if layout == "time" else y.T)
    assert np.array_equal(y.view(np.uint64), ref[at:at + n].view(np.uint64)), (n, at, bank.last_kernel)
    at += n
