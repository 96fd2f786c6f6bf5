"""The token scores and the orthogonalised update as a training run uses them
(Trainer with an entropy term and optimizer 'muon'), and Diffusion.score_tokens."""
import math

import pytest
import torch

import mdlm_oracle as orc
from test_gpu_muon import oracle as orthogonal, tol_factor
from test_gpu_train import MASK_T, V_T, _batch, _make_trainer, _rel

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
  assert torch.cuda.is_available()
  from mdlm_amd import ops as _ops
  return _ops


def _loss_and_grads(p, x0, attn, t, u, m, w):
  """The oracle's loss with the entropy term, by autograd in fp32."""
  leaves = {k: v.detach().clone().requires_grad_(True) for k, v in p.items()}
  sigma, dsigma = orc.loglinear_noise(t)
  xt = orc.q_xt(x0, 1 - torch.exp(-sigma[:, None]), u, MASK_T)
  logits = orc.dit_forward(leaves, xt, torch.zeros_like(sigma), m.n_heads, m.n_blocks, None, 0.0)
  keep = torch.arange(V_T) != MASK_T
  l = torch.log_softmax(logits[..., keep], -1)
  ent = -(l.exp() * l).sum(-1) * (xt == MASK_T) * attn
  lp = orc.subs_parameterization(logits, xt, MASK_T)
  nll = -torch.gather(lp, -1, x0[..., None])[..., 0] * (dsigma / torch.expm1(sigma))[:, None] * attn
  token_nll = nll.sum() / attn.sum()
  loss = token_nll - w * ent.sum() / attn.sum()
  g = torch.autograd.grad(loss, list(leaves.values()), allow_unused=True)
  mean = ent.sum() / ((xt == MASK_T) * attn).sum()
  return token_nll.detach(), mean.detach(), {k: torch.zeros_like(p[k]) if d is None else d for k, d in zip(leaves, g)}


@pytest.mark.parametrize('weight', [0.3, -1.0])
def test_entropy_term_gradients(ops, weight):
  """The bounds are those of the training step without the term (bf16 backbone)."""
  model, cfg, p, tr = _make_trainer(0.0, extra=[f'training.entropy_weight={weight}'])
  assert tr.entropy_weight == weight
  m = cfg.model
  x0, attn, t, u = _batch(4, m.length, seed=3)
  loss, nlls = tr.forward_backward(x0.cuda(), attn.cuda(), t=t.cuda(), u_xt=u.cuda())
  ref_loss, ref_ent, ref = _loss_and_grads(p, x0, attn, t, u, m, weight)
  assert abs(loss.item() - ref_loss.item()) < 2e-2 * abs(ref_loss.item())
  assert abs(tr.last_entropy.item() - ref_ent.item()) < 2e-2 * ref_ent.item()
  g = tr.grads()
  flat = torch.cat([g[k].reshape(-1).cpu() for k in ref]).double()
  flat_ref = torch.cat([ref[k].reshape(-1) for k in ref]).double()
  assert ((flat @ flat_ref) / (flat.norm() * flat_ref.norm())).item() > 0.999
  assert max(_rel(g[k], ref[k]) for k in ref) < 6e-2
  # the term is there: without it the gradients differ
  plain = _loss_and_grads(p, x0, attn, t, u, m, 0.0)[2]
  flat0 = torch.cat([plain[k].reshape(-1) for k in ref]).double()
  assert (flat - flat_ref).norm() < 0.5 * (flat - flat0).norm()


def test_entropy_term_with_no_masked_token(ops):
  model, cfg, p, tr = _make_trainer(0.0, extra=['training.entropy_weight=0.5'])
  x0, attn, t, u = _batch(4, cfg.model.length)
  loss, _ = tr.forward_backward(x0.cuda(), attn.cuda(), t=t.cuda(), u_xt=torch.full_like(u, 2.0).cuda())
  assert loss.item() == 0 and all((v == 0).all() for k, v in tr.grads().items() if 'output_layer' in k)


def test_muon_training_steps(ops):
  """Two optimizer steps, each from the gradients that the trainer itself computed:
  the blocks' matrices move by orthogonalised momentum, the rest as under AdamW,
  both clipped by the one norm; EMA and bf16 copies follow."""
  model, cfg, p, tr = _make_trainer(0.0, extra=['optim.name=muon', 'optim.weight_decay=0.05',
                                                'training.entropy_weight=0.1'])
  muon = [n for n in tr.names if n.endswith(tr.MUON_NAMES) and n.startswith('blocks.')]
  assert len(muon) == 4 * cfg.model.n_blocks
  assert sum(b - a for a, b in tr.adamw_ranges) + sum(tr.offsets[n][1] for n in muon) == tr.n_flat
  P = {n: tr._view(tr.P, n).double().cpu() for n in tr.names}
  M = {n: torch.zeros_like(P[n]) for n in tr.names}
  V = {n: torch.zeros_like(P[n]) for n in tr.names}
  E = {n: v.clone() for n, v in P.items()}
  moved = {n: 0.0 for n in tr.names}
  start = {n: v.clone() for n, v in P.items()}
  for step in (1, 2):
    x0, attn, t, u = _batch(4, cfg.model.length, seed=step)
    tr.forward_backward(x0.cuda(), attn.cuda(), t=t.cuda(), u_xt=u.cuda())
    G = {n: g.double().cpu() for n, g in tr.grads().items()}
    norm = math.sqrt(sum(float(g.square().sum()) for g in G.values()))
    coef = min(1.0, 1.0 / (norm + 1e-6))
    lr = orc.constant_warmup_lr(3e-3, step - 1, 2)
    assert tr.optimizer_step() == lr
    omd = 1 - orc.ema_decay(0.9999, step)
    for n in tr.names:
      g = G[n] * coef
      if n in muon:
        M[n] += (g - M[n]) * 0.05
        o = orthogonal((g + 0.95 * (M[n] - g))[None])[0]
        move = lr * 0.2 * math.sqrt(max(o.shape)) * o
      else:
        M[n] += (g - M[n]) * 0.1
        V[n] = 0.999 * V[n] + 0.001 * g * g
        move = lr / (1 - 0.9 ** step) * M[n] / (V[n].sqrt() / math.sqrt(1 - 0.999 ** step) + 1e-8)
      P[n] = P[n] * (1 - lr * 0.05) - move
      E[n] -= omd * (E[n] - P[n])
      moved[n] += float(move.norm())
  sd = model.backbone.state_dict()
  ema = dict(zip(tr.names, tr.ema_state_dict()['shadow_params']))
  for n in tr.names:
    # orthogonal factor: its tolerance on the way moved; AdamW as the plain trainer's test
    tol = tol_factor(5) * moved[n] + 2.0 ** -22 * float(P[n].norm()) if n in muon else 2e-6 * math.sqrt(P[n].numel())
    assert (sd[n].cpu().double() - P[n]).norm() <= tol, n
    assert (ema[n].cpu().double() - E[n]).norm() <= tol + 2.0 ** -22 * float(E[n].norm()), n
    assert torch.equal(tr._w16(n), tr._view(tr.P, n).to(torch.bfloat16)), n
    if n in muon:
      assert (sd[n].cpu().double() - start[n]).norm() > 0.5 * moved[n]
  # forward on the new weights
  x0, attn, t, u = _batch(4, cfg.model.length, seed=9)
  lg = model.backbone(x0.cuda(), torch.zeros(4, device='cuda')).float().cpu()
  ref = orc.dit_forward({n: v.float() for n, v in P.items()}, x0, torch.zeros(4), cfg.model.n_heads, cfg.model.n_blocks)
  assert _rel(lg, ref) < 2e-2


@pytest.mark.parametrize('bad', ['optim.name=sgd', 'optim.momentum=1.0', 'optim.ns_steps=0', 'optim.ns_steps=33',
                                 'training.entropy_weight=.nan'])
def test_trainer_refuses(ops, bad):
  with pytest.raises(ValueError, match=bad.split('=')[0].split('.')[1] if 'name' not in bad else 'sgd'):
    _make_trainer(0.0, extra=['optim.name=muon', bad])


def test_muon_accumulates(ops):
  """Two micro-batches and one step: the momentum moves by the mean of their gradients."""
  model, cfg, p, tr = _make_trainer(0.0, extra=['optim.name=muon', 'training.entropy_weight=0.1'])
  tr.max_norm = 0.0
  total = None
  for seed in (1, 2):
    x0, attn, t, u = (a.cuda() for a in _batch(4, cfg.model.length, seed=seed))
    tr.forward_backward(x0, attn, t=t, u_xt=u)
    g = tr.G.double()
    total = g if total is None else total + g
  for i, seed in enumerate((1, 2)):
    x0, attn, t, u = (a.cuda() for a in _batch(4, cfg.model.length, seed=seed))
    tr.forward_backward(x0, attn, t=t, u_xt=u, accumulate=i > 0, last=i == 1)
  tr.optimizer_step()
  for name in ('blocks.0.attn_qkv.weight', 'blocks.1.mlp.2.weight'):
    o, n, _ = tr.offsets[name]
    want = total[o:o + n] / 2 * 0.05
    assert _rel(tr.M1[o:o + n].cpu(), want.cpu()) < 1e-3, name      # atomics order two backward passes


def test_muon_checkpoint_resume(ops, tmp_path):
  extra = ['optim.name=muon', 'training.ema=0.999']
  model, cfg, p, tr = _make_trainer(0.0, extra=extra)
  batches = [_batch(4, cfg.model.length, seed=s) for s in range(3)]

  def step(tr_, b):
    x0, attn, t, u = b
    tr_.forward_backward(x0.cuda(), attn.cuda(), t=t.cuda(), u_xt=u.cuda())
    tr_.optimizer_step()
  for b in batches[:2]:
    step(tr, b)
  path = str(tmp_path / 'last.ckpt')
  tr.save_checkpoint(path)
  step(tr, batches[2])
  _, _, _, tr2 = _make_trainer(0.0, seed=11, extra=extra)
  assert tr2.load_checkpoint(path) == 2
  step(tr2, batches[2])
  for name in ('P', 'M1', 'M2', 'E', 'W16'):
    a, b = getattr(tr, name).float(), getattr(tr2, name).float()
    assert torch.allclose(a, b, rtol=1e-2, atol=2e-5), (name, (a - b).abs().max().item())
  # the moments of one optimizer are refused by the other
  _, _, _, tr3 = _make_trainer(0.0, extra=['training.ema=0.999'])
  with pytest.raises(ValueError, match='optimizer'):
    tr3.load_checkpoint(path)


def test_score_tokens(ops):
  model, cfg, p, tr = _make_trainer(0.0)
  m = cfg.model
  x0, attn, t, u = _batch(4, m.length, seed=5)
  xt = torch.where(u < 0.6, torch.full_like(x0, MASK_T), x0)
  s = model.score_tokens(x0.cuda(), xt.cuda(), top_k=3)
  assert s.logp.shape == x0.shape and s.top_ids.shape == (*x0.shape, 3)
  table = model.forward(xt.cuda(), torch.zeros(4, device='cuda')).float()
  # the table is bf16: half a step of its values
  assert ((s.logp - table.gather(2, x0.cuda()[..., None])[..., 0]).abs() <= 2.0 ** -8 * (s.logp.abs() + 1e-3)).all()
  known = (xt != MASK_T).cuda()
  assert (s.logp[known] == 0).all() and (s.entropy[known] == 0).all()
  assert torch.equal(s.top_ids[known][:, 0], xt.cuda()[known])
  ref = orc.subs_parameterization(orc.dit_forward(p, xt, torch.zeros(4), m.n_heads, m.n_blocks), xt, MASK_T)
  want = torch.gather(ref, -1, x0[..., None])[..., 0]
  assert (s.logp.cpu() - want)[~known.cpu()].abs().max() < 6e-2
  assert (s.entropy >= 0).all() and (s.entropy <= math.log(V_T - 1) + 1e-4).all()
  with pytest.raises(ValueError, match='alike'):
    model.score_tokens(x0[:, :5].cuda(), xt.cuda())
  with pytest.raises(IndexError):
    model.score_tokens(x0.cuda() + V_T, xt.cuda())
