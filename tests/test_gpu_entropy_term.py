"""The entropy that Trainer reports beside the loss (training.entropy_weight)."""
import pytest
import torch

from test_gpu_train import _batch, _make_trainer

pytestmark = pytest.mark.gpu


def test_last_entropy_is_of_this_batch():
  model, cfg, p, tr = _make_trainer(0.0, extra=['training.entropy_weight=0.5'])
  x0, attn, t, u = (a.cuda() for a in _batch(4, cfg.model.length, seed=3))
  assert tr.last_entropy is None
  tr.forward_backward(x0, attn, t=t, u_xt=u)
  assert tr.last_entropy.item() > 0
  tr.forward_backward(x0, attn, t=t, u_xt=torch.full_like(u, 2.0))        # nothing is masked
  assert tr.last_entropy.item() == 0
  tr.forward_backward(x0, attn, t=t, u_xt=u)
  # masked positions, none of them attended
  tr.forward_backward(x0, torch.zeros_like(attn).index_fill_(1, torch.zeros(1, dtype=torch.long, device='cuda'), 1.0),
                      t=t, u_xt=torch.where(torch.arange(u.shape[1], device='cuda') > 0, u, torch.full_like(u, 2.0)))
  assert tr.last_entropy.item() == 0
  tr.forward_backward(x0, attn, t=t, u_xt=u)
  assert tr.last_entropy.item() > 0
  tr.entropy_weight = 0.0
  tr.forward_backward(x0, attn, t=t, u_xt=u)
  assert tr.last_entropy is None
