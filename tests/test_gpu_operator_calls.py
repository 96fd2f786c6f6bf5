"""Calls of the token scores and the weight update as a user makes them that the
other files leave out."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
  assert torch.cuda.is_available()
  from mdlm_amd import ops as _ops
  return _ops


def test_muon_update_refuses_an_empty_norm(ops):
  """An empty sumsq has no address: it would have passed as 'do not clip'."""
  p, g, m = (torch.ones(8, 8, device='cuda') for _ in range(3))
  with pytest.raises(RuntimeError, match='sumsq'):
    ops.muon_update(p, g, m, 1e-3, sumsq=torch.zeros(0, device='cuda'), max_norm=1.0)
  assert (p == 1).all() and (m == 1).all()
