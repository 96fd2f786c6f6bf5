"""Token scores (ops.subs_scores) and their gradient against a plain form in 64
bits on the CPU.

Tolerances, with u = 2^-24 (half a step of fp32): a term exp2(t) is off by u |t|
from its argument (|t| <= 64 wherever the term matters) and by 2 u from the
instruction; a thread adds at most V / 256 terms one after another and the tree
behind it 16 more, so a row's sums are off by at most N = 82 + V / 256 units u,
relative.  A logarithm or a difference adds a few units of its own size: values
are held to 4 N u (1 + |value|), and gradients to 4 N u of the sum of their
terms' sizes plus half a step of their type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NEG = -1e6


@pytest.fixture(scope='module')
def ops():
  assert torch.cuda.is_available()
  from mdlm_amd import ops as _ops
  return _ops


def _units(V):
  return 4 * (82 + V / 256) * U


def make_logits(rows, V, dtype, layout, seed, scale=2.0):
  """layout: padded (rows 16-byte aligned), tight (rows V elements apart), odd (a
  view that starts one element into wider rows)."""
  gen = torch.Generator().manual_seed(seed)
  x = (torch.randn(rows, V, generator=gen) * scale).to(dtype)
  if layout == 'tight':
    return x.cuda()
  ld = (V + 127) // 128 * 128 if layout == 'padded' else V + 5
  buf = torch.full((rows, ld), float('nan'), dtype=dtype, device='cuda')   # never read as a score
  off = 0 if layout == 'padded' else 1
  view = buf[:, off:off + V]
  view.copy_(x)
  return view


def make_ids(rows, V, mask, seed, known=0.3):
  gen = torch.Generator().manual_seed(seed + 1)
  x0 = torch.randint(0, V, (rows,), generator=gen)
  xt = torch.where(torch.rand(rows, generator=gen) < known, x0, torch.full_like(x0, mask))
  return xt, x0


def oracle(logits, xt, x0, mask, k):
  """(logp, entropy, lse, top_logp, top_ids) in 64 bits."""
  x = logits.detach().cpu().double()
  rows, V = x.shape
  y = x.clone()
  y[:, mask] = -math.inf
  lse = torch.logsumexp(y, 1)
  l = torch.log_softmax(y, 1)      # lse of lowest values does not hold log Z even in 64 bits
  p = l.exp()
  ent = -torch.where(p > 0, p * l, torch.where(p.isnan(), p, 0.0)).sum(1)
  table = l.clone()
  table[:, mask] = x[:, mask] + NEG - lse
  ok = (x0 >= 0) & (x0 < V)
  at = x0.clamp(0, V - 1)
  logp = torch.where(ok, table.gather(1, at[:, None])[:, 0], 0.0)
  # order: logit, NaN first, then index; the mask column last
  key = torch.nan_to_num(y, nan=math.inf, posinf=torch.finfo(torch.float64).max, neginf=-1e300)
  key[:, mask] = -math.inf
  ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
  top = l.gather(1, ids)
  for r in range(rows):
    t = int(xt[r])
    if t == mask:
      continue
    logp[r] = 0.0 if int(x0[r]) == t or not ok[r] else NEG
    ent[r] = lse[r] = 0.0
    if k:
      ids[r] = torch.tensor(([t] + [v for v in range(V) if v not in (t, mask)])[:k])
      top[r] = torch.tensor([0.0] + [NEG] * (k - 1), dtype=torch.float64)
  return logp, ent, lse, top, ids


def close(got, want, V, what):
  got, want = got.detach().cpu().double(), want.double()
  assert got.shape == want.shape, what
  fin = want.isfinite()
  assert torch.equal(got.isnan(), want.isnan()), what
  assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()]), what
  err = (got[fin] - want[fin]).abs()
  tol = _units(V) * (1 + want[fin].abs())
  assert (err <= tol).all(), f'{what}: {(err / tol).max().item():.3g} times the tolerance'


def check(ops, logits, xt, x0, mask, k):
  V = logits.shape[1]
  s = ops.subs_scores(logits, xt.cuda(), x0.cuda(), mask, top_k=k)
  logp, ent, lse, top, ids = oracle(logits, xt, x0, mask, k)
  close(s.logp, logp, V, 'logp')
  # the entropy's two terms are of the size of the log-sum-exp's range, log V
  close(s.entropy, ent, V * 2, 'entropy')
  close(s.lse, lse, V, 'lse')
  if k:
    assert torch.equal(s.top_ids.cpu(), ids)
    close(s.top_logp, top, V, 'top_logp')
  else:
    assert s.top_ids is None and s.top_logp is None
  return s


SHAPES = [(1, 2, 1), (1, 3, 2), (5, 7, 6), (3, 8, 1), (4, 9, 3), (2, 64, 5), (3, 255, 64), (7, 300, 16), (2, 1031, 64),
          (3, 2049, 8), (2, 4099, 33), (130, 1000, 4), (3, 30522, 5), (2, 50258, 8), (1, 131075, 64)]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('layout', ['padded', 'tight', 'odd'])
@pytest.mark.parametrize('rows,V,k', SHAPES)
def test_scores(ops, rows, V, k, layout, dtype):
  for j, mask in enumerate((V - 1, 0, V // 2)):
    logits = make_logits(rows, V, dtype, layout, seed=V + j)
    xt, x0 = make_ids(rows, V, mask, seed=V + j, known=0.3 if j else 0.0)
    check(ops, logits, xt, x0, mask, min(k, V - 1))
  check(ops, logits, xt, x0, mask, 0)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_scores_of_every_kind_of_row(ops, dtype):
  V, mask, k = 777, 5, 20
  x = make_logits(14, V, dtype, 'padded', seed=3)
  x[0] = 1.5                                  # every logit equal: the lowest ids
  x[1] = -math.inf                            # no distribution
  x[2, 40:] = -math.inf                       # few tokens allowed
  x[3, :] = -math.inf
  x[3, 700] = 2.0                             # one token allowed: entropy 0
  x[4, 12] = float('nan')
  x[5, 12] = math.inf
  x[6, mask] = float('nan')                   # the mask column takes no part
  x[7, mask] = math.inf
  x[8] = torch.finfo(dtype).min               # the type's lowest value everywhere
  x[9, 100:200] = torch.finfo(dtype).min
  x[10, 3] = 80.0                             # all the mass on one token
  x[11] = 0.0
  x[11, ::2] = -0.0                           # equal to +0: by index
  x[12, :] = -math.inf
  x[12, mask] = 1.0                           # only the mask column is left
  xt = torch.full((14,), mask)
  x0 = torch.arange(14) * 50
  x0[3], x0[13] = 700, mask
  want = oracle(x, xt, x0, mask, k)
  s = ops.subs_scores(x, xt.cuda(), x0.cuda(), mask, top_k=k)
  # a row with a NaN or +inf has NaN scores throughout
  bad = torch.tensor([4, 5])
  good = torch.tensor([r for r in range(14) if r not in (4, 5)])
  for got in (s.logp, s.entropy, s.lse, s.top_logp):
    assert got[bad.cuda()].isnan().all()
  assert s.top_ids[4, 0] == 12 and s.top_ids[5, 0] == 12
  assert torch.equal(s.top_ids.cpu()[good], want[4][good])
  for got, w, name in ((s.logp, want[0], 'logp'), (s.entropy, want[1], 'entropy'), (s.lse, want[2], 'lse'),
                       (s.top_logp, want[3], 'top')):
    close(got[good.cuda()], w[good], V * 2, name)
  assert s.entropy[3] == 0 and s.logp[3] == 0
  assert s.lse[1] == -math.inf and s.lse[12] == -math.inf


def test_scores_of_one_column_and_of_the_mask_token(ops):
  """V = 1 is the mask column alone: a masked position has no distribution; in a row
  that has one, the mask token scores its logit - 1e6 - lse."""
  x = torch.zeros(2, 1, device='cuda')
  s = ops.subs_scores(x, torch.tensor([0, 5], device='cuda'), torch.tensor([0, 5], device='cuda'), 0)
  assert s.logp[0].isnan() and s.entropy[0].isnan() and s.lse[0] == -math.inf
  assert s.logp[1] == 0 and s.entropy[1] == 0
  V, mask = 50, 3
  x = make_logits(2, V, torch.float32, 'tight', seed=1)
  x[1] = -math.inf
  s = ops.subs_scores(x, torch.full((2,), mask, device='cuda'), torch.full((2,), mask, device='cuda'), mask, top_k=49)
  assert abs(s.logp[0].item() - (x[0, mask].item() + NEG - s.lse[0].item())) <= 1
  assert s.logp[1].isnan() and (s.top_ids != mask).all()


def test_scores_targets_that_are_no_tokens(ops):
  V, mask = 300, 299
  x = make_logits(4, V, torch.float32, 'tight', seed=9)
  xt = torch.full((4,), mask)
  s = check(ops, x, xt, torch.tensor([-1, V, -100, 2 ** 40]), mask, 3)
  assert (s.logp == 0).all()
  s = check(ops, x, torch.tensor([mask, 7, 0, mask]), torch.tensor([-100, -100, V, 2 ** 40]), mask, 3)   # known rows too
  assert (s.logp == 0).all()


def test_scores_batched_and_in_agreement_with_the_table(ops):
  B, L, V, mask = 3, 37, 501, 500
  lg = ops.alloc_logits(B, L, V)
  lg.copy_(torch.randn(B, L, V, generator=torch.Generator().manual_seed(2)).cuda() * 3)
  x0 = torch.randint(0, V - 1, (B, L), device='cuda')
  xt = torch.where(torch.rand(B, L, device='cuda') < 0.5, x0, mask)
  s = ops.subs_scores(lg, xt, x0, mask, top_k=4)
  assert s.logp.shape == (B, L) and s.top_ids.shape == (B, L, 4)
  table = ops.subs_logprobs(lg, xt, mask, out_dtype=torch.float32)
  want = table.gather(2, x0[..., None])[..., 0]
  assert torch.allclose(s.logp, want, rtol=0, atol=1e-5)
  assert torch.allclose(s.top_logp, table.gather(2, s.top_ids), rtol=1e-7, atol=1e-5)
  best = ops.subs_argmax(lg, xt, mask)
  assert torch.equal(s.top_ids[..., 0], best)


def oracle_grad(logits, xt, x0, mask, g_logp, g_ent, top_ids, g_top):
  """(gradient, sum of the sizes of its terms) in 64 bits, from the formula."""
  x = logits.detach().cpu().double()
  rows, V = x.shape
  x[:, mask] = -math.inf
  l = torch.log_softmax(x, 1)
  p = l.exp()
  lz = torch.where(p > 0, l, 0.0)
  H = -(p * lz).sum(1, keepdim=True)
  gl = torch.zeros(rows) if g_logp is None else g_logp.double()
  gh = torch.zeros(rows) if g_ent is None else g_ent.double()
  ok = ((x0 >= 0) & (x0 < V)).double()
  up = torch.zeros(rows, V, dtype=torch.float64)
  up.scatter_add_(1, x0.clamp(0, V - 1)[:, None], (gl * ok)[:, None])
  if g_top is not None:
    up.scatter_add_(1, top_ids, g_top.double())
  tot = up.sum(1, keepdim=True)
  size = (gl * ok).abs()[:, None] + (0 if g_top is None else g_top.double().abs().sum(1, keepdim=True))
  d = up - p * tot - gh[:, None] * p * (lz + H)
  mag = up.abs() + p * size + gh.abs()[:, None] * p * (lz.abs() + H)
  live = (xt == mask)[:, None] & (torch.arange(V) != mask)[None]
  return d * live, mag * live


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('layout', ['padded', 'tight', 'odd'])
@pytest.mark.parametrize('rows,V,k', SHAPES)
def test_scores_bwd(ops, rows, V, k, layout, dtype):
  mask, k = V // 2, min(k, V - 1)
  logits = make_logits(rows, V, dtype, layout, seed=V)
  xt, x0 = make_ids(rows, V, mask, seed=V)
  gen = torch.Generator().manual_seed(V)
  gl, gh = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen)
  gt = torch.randn(rows, k, generator=gen)
  s = ops.subs_scores(logits, xt.cuda(), x0.cuda(), mask, top_k=k)
  ids = s.top_ids.cpu()
  for use in ('logp', 'entropy', 'all'):
    a = gl if use != 'entropy' else None
    b = gh if use != 'logp' else None
    c = gt if use == 'all' else None
    dev = lambda t: None if t is None else t.cuda()
    d = ops.subs_scores_bwd(logits, xt.cuda(), x0.cuda(), mask, s.lse, s.entropy, dev(a), dev(b),
                            None if c is None else s.top_ids, dev(c))
    assert d.dtype == dtype and d.shape == logits.shape
    want, mag = oracle_grad(logits, xt, x0, mask, a, b, ids, c)
    tol = 4 * _units(V) * mag + torch.finfo(dtype).eps / 2 * want.abs() + 1e-37
    err = (d.cpu().double() - want).abs()
    assert (err <= tol).all(), (use, (err / tol).max().item())


def test_scores_bwd_against_differences(ops):
  """The gradient of  sum_r a logp + b entropy + c . top_logp  against central
  differences of the 64-bit scores.  Step h: the third derivative's term is h^2 / 6
  times a few units, the rounding 1e-16 / h: 1e-4 leaves 1e-8, fp32 dominates."""
  V, mask, rows, k = 23, 4, 3, 3
  x = make_logits(rows, V, torch.float32, 'tight', seed=1)
  xt, x0 = torch.full((rows,), mask), torch.tensor([1, 22, 9])
  gl, gh, gt = torch.tensor([0.7, -1.0, 0.3]), torch.tensor([0.5, 0.2, -1.0]), torch.randn(rows, k)
  s = ops.subs_scores(x, xt.cuda(), x0.cuda(), mask, top_k=k)
  d = ops.subs_scores_bwd(x, xt.cuda(), x0.cuda(), mask, s.lse, s.entropy, gl.cuda(), gh.cuda(), s.top_ids, gt.cuda()).cpu()
  ids = s.top_ids.cpu()

  def f(z):
    y = z.clone()
    y[:, mask] = -math.inf
    l = torch.log_softmax(y, 1)
    p = l.exp()
    H = -(p * torch.where(p > 0, l, 0.0)).sum(1)
    return (gl * l.gather(1, x0[:, None])[:, 0] + gh * H + (gt * l.gather(1, ids)).sum(1)).sum()
  z, h = x.cpu().double(), 1e-4
  for r in range(rows):
    for v in range(V):
      e = torch.zeros_like(z)
      e[r, v] = h
      assert abs((f(z + e) - f(z - e)).item() / (2 * h) - d[r, v].item()) < 1e-5


def test_scores_bwd_rows_without_gradient_and_repeated_ids(ops):
  V, mask, rows = 1003, 1002, 6
  x = make_logits(rows, V, torch.bfloat16, 'padded', seed=4)
  x[0] = float('nan')                       # nothing comes in: zero whatever it holds
  x[1] = -math.inf
  xt, x0 = torch.full((rows,), mask), torch.tensor([3, 4, 7, 7, -1, mask])
  lse, ent = (t.cuda() for t in oracle(x, xt, x0, mask, 0)[2:0:-1])
  lse, ent = lse.float(), ent.float()
  gl = torch.tensor([0.0, 0.0, 1.0, 1.0, 1.0, 1.0])
  ids = torch.tensor([[7, 7, 9], [1, 2, 3], [7, 7, 9], [9, 7, 7], [0, V - 2, 5], [mask, -5, V]])
  gt = torch.zeros(rows, 3)
  gt[2:] = torch.randn(4, 3)
  d = ops.subs_scores_bwd(x, xt.cuda(), x0.cuda(), mask, lse, ent, gl.cuda(), None, ids.cuda(), gt.cuda()).cpu()
  assert (d[:2] == 0).all()
  okid = (ids >= 0) & (ids < V)
  want, mag = oracle_grad(x[2:], xt[2:], x0[2:], mask, gl[2:], None, ids[2:].clamp(0, V - 1), (gt * okid)[2:])
  err = (d[2:].double() - want).abs()
  assert (err <= 4 * _units(V) * mag + 2.0 ** -8 * want.abs() + 1e-37).all()


def test_scores_bwd_of_large_logits(ops):
  """Rows whose log-sum-exp cannot hold log Z beside it: a common offset, or the
  type's lowest value everywhere (the uniform distribution)."""
  V, mask = 600, 599
  for dtype in (torch.bfloat16, torch.float32):
    x = make_logits(4, V, dtype, 'tight', seed=11)
    x[0] = torch.finfo(dtype).min
    x[1] = (x[1].float() + 2.0 ** 20).to(dtype)
    x[2] -= 300
    x[3, ::2] = torch.finfo(dtype).min
    xt, x0 = torch.full((4,), mask), torch.tensor([5, 6, 7, 9])
    s = check(ops, x, xt, x0, mask, 7)
    g = torch.tensor([1.0, -2.0, 3.0, 1.0])
    d = ops.subs_scores_bwd(x, xt.cuda(), x0.cuda(), mask, s.lse, s.entropy, g.cuda(), g.cuda())
    want, mag = oracle_grad(x, xt, x0, mask, g, g, None, None)
    err = (d.cpu().double() - want).abs()
    # the saved log-sum-exp is within half a step of 128 (2^-18)
    assert (err <= (4 * _units(V) + 2.0 ** -17) * mag + torch.finfo(dtype).eps / 2 * want.abs() + 1e-37).all()


def test_scores_bwd_in_place_and_padding_untouched(ops):
  rows, V, mask = 9, 1001, 0
  x = make_logits(rows, V, torch.bfloat16, 'padded', seed=5)
  xt, x0 = make_ids(rows, V, mask, seed=5)
  xt, x0 = xt.cuda(), x0.cuda()
  s = ops.subs_scores(x, xt, x0, mask)
  g = torch.randn(rows, device='cuda')
  d = ops.subs_scores_bwd(x, xt, x0, mask, s.lse, s.entropy, g, g)
  buf = torch.full((rows, 1024), 7.0, dtype=torch.bfloat16, device='cuda')
  ops.subs_scores_bwd(x, xt, x0, mask, s.lse, s.entropy, g, g, dlogits=buf[:, :V])
  assert torch.equal(buf[:, :V], d) and (buf[:, V:] == 7).all()
  odd = torch.full((rows, 1024), 7.0, dtype=torch.bfloat16, device='cuda')   # alignments that differ
  ops.subs_scores_bwd(x, xt, x0, mask, s.lse, s.entropy, g, g, dlogits=odd[:, 3:3 + V])
  assert torch.equal(odd[:, 3:3 + V], d) and (odd[:, :3] == 7).all() and (odd[:, 3 + V:] == 7).all()
  y = x.clone()
  ops.subs_scores_bwd(y, xt, x0, mask, s.lse, s.entropy, g, g, dlogits=y)
  assert torch.equal(y, d)


def test_scores_repeatable_other_stream_and_captured(ops):
  rows, V, mask, k = 40, 5003, 17, 12
  x = make_logits(rows, V, torch.bfloat16, 'odd', seed=6)
  xt, x0 = (t.cuda() for t in make_ids(rows, V, mask, seed=6))
  g = torch.randn(rows, device='cuda')
  gt = torch.randn(rows, k, device='cuda')

  def both():
    s = ops.subs_scores(x, xt, x0, mask, top_k=k)
    return list(s) + [ops.subs_scores_bwd(x, xt, x0, mask, s.lse, s.entropy, g, g, s.top_ids, gt)]
  ref = both()
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    got = both()
  side.synchronize()
  assert all(torch.equal(a, b) for a, b in zip(ref, got))
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = both()
  for i in range(4):
    x.copy_(make_logits(rows, V, torch.bfloat16, 'odd', seed=60 + i))
    for t in out:
      t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(both(), out)), i


def test_scores_of_no_rows(ops):
  x = torch.empty(0, 100, dtype=torch.bfloat16, device='cuda')
  ids = torch.empty(0, dtype=torch.int64, device='cuda')
  s = ops.subs_scores(x, ids, ids, 99, top_k=2)
  assert s.logp.shape == (0,) and s.top_ids.shape == (0, 2)
  f = torch.empty(0, device='cuda')
  assert ops.subs_scores_bwd(x, ids, ids, 99, f, f, f).shape == (0, 100)


def test_scores_past_32_bit_offsets(ops):
  """Rows whose elements lie past 2^31: the last rows score as they do alone."""
  V, rows = 50258, 43000
  ld = 50304
  buf = torch.zeros(rows, ld, dtype=torch.bfloat16, device='cuda')
  tail = make_logits(3, V, torch.bfloat16, 'tight', seed=8)
  buf[-3:, :V] = tail
  ids = torch.full((rows,), V - 1, device='cuda')
  x0 = torch.arange(rows, device='cuda') % (V - 1)
  s = ops.subs_scores(buf[:, :V], ids, x0, V - 1, top_k=3)
  t = ops.subs_scores(tail, ids[-3:], x0[-3:].contiguous(), V - 1, top_k=3)
  for a, b in zip(s, t):
    assert torch.allclose(a[-3:].double(), b.double(), rtol=1e-6, atol=1e-6)
  g = torch.ones(rows, device='cuda')
  d = ops.subs_scores_bwd(buf[:, :V], ids, x0, V - 1, s.lse, s.entropy, g)
  e = ops.subs_scores_bwd(tail, ids[-3:], x0[-3:].contiguous(), V - 1, s.lse[-3:].contiguous(),
                          s.entropy[-3:].contiguous(), g[-3:].contiguous())
  assert torch.equal(d[-3:], e)
