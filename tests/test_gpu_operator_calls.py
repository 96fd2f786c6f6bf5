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


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_one_position_of_each_sequence(ops, dtype):
  """logits[:, i:i + 1] has rows at a constant distance, that of the sequences."""
  B, L, V, mask = 3, 5, 1000, 999
  gen = torch.Generator(device='cuda').manual_seed(0)
  full = ops.alloc_logits(B, L, V, dtype)
  full.copy_(torch.randn(B, L, V, generator=gen, device='cuda'))
  one = full[:, 2:3]
  x0 = torch.randint(0, V - 1, (B, 1), generator=gen, device='cuda')
  xt = torch.full_like(x0, mask)
  s = ops.subs_scores(one, xt, x0, mask, top_k=4)
  want = ops.subs_scores(one.contiguous(), xt, x0, mask, top_k=4)
  for got, ref in zip(s, want):
    assert got.shape[:2] == (B, 1) and torch.equal(got, ref)
  g = torch.rand(B, 1, generator=gen, device='cuda')
  keep = full.clone()
  d = ops.subs_scores_bwd(one, xt, x0, mask, s.lse, s.entropy, g_logp=g, g_entropy=g)
  assert torch.equal(d, ops.subs_scores_bwd(one.contiguous(), xt, x0, mask, s.lse, s.entropy, g_logp=g, g_entropy=g))
  ops.subs_scores_bwd(one, xt, x0, mask, s.lse, s.entropy, g_logp=g, g_entropy=g, dlogits=one)
  assert torch.equal(one, d)
  others = [i for i in range(L) if i != 2]
  assert torch.equal(full[:, others], keep[:, others])


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('rows,V', [(200, 9000), (3000, 500), (7, 3)])
def test_scores_of_certain_tokens(ops, rows, V, dtype):
  """One token has (nearly) all the weight: its log-probability is not above 0, nor the
  entropy below it, whatever the logits' size."""
  gen = torch.Generator(device='cuda').manual_seed(V)
  mask = V - 1
  x = torch.randn(rows, V, generator=gen, device='cuda')
  top = torch.randint(0, mask, (rows,), generator=gen, device='cuda')
  x[torch.arange(rows, device='cuda'), top] += 10 + 2000 * torch.rand(rows, generator=gen, device='cuda') ** 3
  x += 3000 * torch.rand(rows, 1, generator=gen, device='cuda') ** 2
  xt = torch.full_like(top, mask)
  s = ops.subs_scores(x.to(dtype), xt, top, mask, top_k=2)
  assert (s.logp <= 0).all() and (s.top_logp <= 0).all() and (s.entropy >= 0).all()


def test_matrices_side_by_side(ops):
  """Column blocks of one wide matrix as a stack: they do not overlap."""
  n, r, c = 3, 70, 132
  gen = torch.Generator(device='cuda').manual_seed(5)
  flat = {k: torch.randn(r, 20 + n * c, generator=gen, device='cuda') * 0.1 for k in 'pgme'}
  flat['w'] = flat['p'].bfloat16()
  keep = {k: t.clone() for k, t in flat.items()}
  side = {k: t[:, 20:].view(r, n, c).transpose(0, 1) for k, t in flat.items()}
  apart = {k: t.contiguous() for k, t in side.items()}
  assert torch.equal(ops.orthogonalize(side['g']), ops.orthogonalize(apart['g']))
  out = torch.zeros(r, n * c, dtype=torch.bfloat16, device='cuda')
  ops.orthogonalize(apart['g'], out=out.view(r, n, c).transpose(0, 1))
  assert torch.equal(out.view(r, n, c).transpose(0, 1), ops.orthogonalize(apart['g']))
  for v in (side, apart):
    ops.muon_update(v['p'], v['g'], v['m'], 1e-2, ema=v['e'], w16=v['w'], ema_one_minus_decay=0.1)
  assert all(torch.equal(side[k], apart[k]) for k in side)
  assert all(torch.equal(flat[k][:, :20], keep[k][:, :20]) for k in flat) and not torch.equal(side['p'][2], keep['p'][:, -c:])
  for stride in (c - 1, 0):        # these do
    with pytest.raises(RuntimeError, match='overlapping'):
      ops.orthogonalize(flat['g'].as_strided((2, r, c), (stride, 20 + n * c, 1)))
