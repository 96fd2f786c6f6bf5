"""Orthogonalised matrices and the weight update built on them against plain
products in 64 bits.

Tolerance of the orthogonal factor (2-norm of the difference over the norm of the
result).  Operands are rounded to fp16 (half a step 2^-11, relative): per step the
correction P - mu I and the X it meets (each at most 0.5 .. 1 of the result's
size near convergence, where nothing later shrinks the error) and D, twice (2 c
|D| |dD| <= 0.8 of it): at most 2 x 2^-11 per step, or 5 x 2 x 2^-11 = 4.9e-3 over
five steps if all add up, plus half a step of bf16, 2^-8, for the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

COEFFS = (3.4445, -4.7750, 2.0315)


def tol_factor(steps):
  return 2 * steps * 2.0 ** -11


@pytest.fixture(scope='module')
def ops():
  assert torch.cuda.is_available()
  from mdlm_amd import ops as _ops
  return _ops


def oracle(g, steps=5, coeffs=COEFFS, eps=1e-7):
  a, b, c = coeffs
  x = g.detach().cpu().double()
  x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
  for _ in range(steps):
    A = x @ x.mT
    x = a * x + (b * A + c * (A @ A)) @ x
  return x


def rel(got, want):
  return ((got.detach().cpu().double() - want).norm() / want.norm()).item()


def gradient(n, r, c, seed, decay=0.0):
  gen = torch.Generator().manual_seed(seed)
  g = torch.randn(n, r, c, generator=gen)
  if decay:
    rk = max(1, min(r, c) // 8)
    amp = torch.arange(1, rk + 1).float() ** -decay
    g = 0.3 * g + torch.randn(n, r, rk, generator=gen) * amp @ torch.randn(n, rk, c, generator=gen)
  return g


SHAPES = [(1, 1, 1), (1, 1, 7), (1, 5, 1), (2, 3, 3), (1, 16, 200), (1, 127, 129), (1, 128, 128), (2, 129, 64),
          (3, 200, 333), (1, 517, 130), (2, 384, 128), (1, 1000, 300), (1, 640, 1291), (3, 128, 512), (2, 512, 100),
          (2, 129, 512),
          (1, 100, 513), (5, 33, 250), (2, 257, 17), (1, 129, 129)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n,r,c', SHAPES)
def test_orthogonalize(ops, n, r, c, dtype):
  for decay in (0.0, 1.0):
    g = gradient(n, r, c, seed=r + c, decay=decay).to(dtype)
    got = ops.orthogonalize(g.cuda())
    assert got.dtype == torch.bfloat16 and got.shape == g.shape
    want = oracle(g)
    for i in range(n):
      assert rel(got[i], want[i]) < tol_factor(5) + 2.0 ** -8, (i, decay)


@pytest.mark.parametrize('n,r,c', [(1, 1, 6000), (1, 64, 513), (1, 30, 4100), (1, 128, 5000), (2, 100, 1025),
                                   (1, 9000, 65), (3, 2100, 128), (40, 70, 2000), (5, 16, 20000), (9, 128, 8200),
                                   (600, 128, 66)])
def test_orthogonalize_short_sides(ops, n, r, c):
  """Short sides of up to 128 rows: A summed in parts of the long side, and workgroups
  that go through several tiles of X, the last ones fewer."""
  g = gradient(n, r, c, seed=r)
  got = ops.orthogonalize(g.cuda())
  for i in {0, n // 2, n - 1}:
    assert rel(got[i], oracle(g[i])) < tol_factor(5) + 2.0 ** -8, i
    assert torch.equal(got[i], ops.orthogonalize(g[i].cuda())), i


@pytest.mark.parametrize('n,r,c', [(300, 100, 140), (40, 560, 600), (25, 1000, 990), (30, 1100, 300), (20, 450, 500)])
def test_orthogonalize_many_matrices(ops, n, r, c):
  """Stacks large enough for the larger tiles.  Every tile adds the same products in the
  same order, so a matrix's result does not depend on the company it is in."""
  g = gradient(n, r, c, seed=n).to(torch.bfloat16).cuda()
  got = ops.orthogonalize(g)
  for i in (0, n // 2, n - 1):
    assert torch.equal(got[i], ops.orthogonalize(g[i])), i
  assert rel(got[n - 1], oracle(g[n - 1])) < tol_factor(5) + 2.0 ** -8


@pytest.mark.parametrize('coeffs', [COEFFS, (1.875, -1.25, 0.375), (2.0, -1.5, 0.5)])
@pytest.mark.parametrize('steps', [1, 2, 3, 7])
def test_orthogonalize_steps_and_coefficients(ops, steps, coeffs):
  g = gradient(1, 150, 260, seed=steps)
  got = ops.orthogonalize(g.cuda(), steps=steps, coeffs=coeffs)
  assert rel(got, oracle(g, steps, coeffs)) < tol_factor(steps) + 2.0 ** -8


def test_orthogonalize_singular_values(ops):
  """What it is for: singular values near 1 (0.6 .. 1.3 for these coefficients), the
  result's product with G symmetric and positive."""
  g = gradient(1, 256, 512, seed=0)[0]
  o = ops.orthogonalize(g.cuda()).float().cpu()
  sv = torch.linalg.svdvals(o)
  assert sv.min() > 0.6 and sv.max() < 1.3
  s = o.double() @ g.double().T
  assert (s - s.T).norm() < 2e-2 * s.norm() and torch.linalg.eigvalsh((s + s.T) / 2).min() > 0


def test_orthogonalize_zero_tiny_huge_and_bad(ops):
  g = gradient(6, 140, 90, seed=5)
  g[1] = 0
  g[2] *= 1e-3
  g[3] *= 1e18
  g[4, 3, 5] = float('nan')
  o = ops.orthogonalize(g.cuda(), eps=1e-30).cpu()
  assert (o[1] == 0).all()
  assert o[4].isnan().any()
  want = oracle(g[[0, 2, 3, 5]], eps=1e-30)
  for k, i in enumerate((0, 2, 3, 5)):       # a bad matrix leaves its neighbours alone
    assert rel(o[i], want[k]) < tol_factor(5) + 2.0 ** -8
  tiny = gradient(1, 40, 40, seed=6) * 1e-25  # squares below the fp32 range
  assert rel(ops.orthogonalize(tiny.cuda(), eps=1e-40), oracle(tiny, eps=1e-40)) < tol_factor(5) + 2.0 ** -8
  for eps in (1e-40, 1e-300):
    assert (ops.orthogonalize(torch.zeros(70, 20, device='cuda'), eps=eps) == 0).all()


def test_orthogonalize_strides_out_and_workspace(ops):
  n, r, c = 3, 70, 133
  g = gradient(n, r, c, seed=7)
  buf = torch.full((n, 5 + r, 150), float('nan'), device='cuda')
  view = buf[:, 2:2 + r, 9:9 + c]
  view.copy_(g)
  out = torch.full((n, r + 4, 200), 7.0, dtype=torch.bfloat16, device='cuda')
  ws = ops.workspace('orthogonalize', n, r, c, device='cuda')
  ws.fill_(float('nan'))                       # what it held before has no effect
  ops.orthogonalize(view, out=out[:, 1:1 + r, 11:11 + c], ws=ws)
  assert torch.equal(out[:, 1:1 + r, 11:11 + c], ops.orthogonalize(g.cuda()))
  out[:, 1:1 + r, 11:11 + c] = 7
  assert (out == 7).all()
  one = ops.orthogonalize(g.cuda()[1])
  assert torch.equal(one, ops.orthogonalize(g.cuda())[1])     # a stack's matrices are independent


def test_orthogonalize_repeatable_other_stream_and_captured(ops):
  g = gradient(2, 200, 300, seed=8).cuda()
  ref = ops.orthogonalize(g)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    got = ops.orthogonalize(g)
  side.synchronize()
  assert torch.equal(ref, got)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = ops.orthogonalize(g)
  for i in range(4):
    g.copy_(gradient(2, 200, 300, seed=80 + i))
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.orthogonalize(g)), i


def test_orthogonalize_on_two_streams_at_once(ops):
  """Calls that overlap in time, each with its own workspace."""
  g = [gradient(2, 300, 700, seed=90 + i).cuda() for i in range(2)]
  ref = [ops.orthogonalize(x) for x in g]
  ws = [torch.empty(ops.workspace_bytes('orthogonalize', 2, 300, 700), dtype=torch.uint8, device='cuda') for _ in g]
  out = [[torch.empty(2, 300, 700, dtype=torch.bfloat16, device='cuda') for _ in range(6)] for _ in g]
  side = [torch.cuda.Stream() for _ in g]
  torch.cuda.synchronize()
  for k in range(6):
    for i, s in enumerate(side):
      with torch.cuda.stream(s):
        ops.orthogonalize(g[i], out=out[i][k], ws=ws[i])
  torch.cuda.synchronize()
  assert all(torch.equal(o, ref[i]) for i in range(2) for o in out[i])


def test_orthogonalize_in_place(ops):
  for shape in ((2, 200, 90), (1, 64, 640)):
    g = gradient(*shape, seed=4).cuda().bfloat16()
    ref = ops.orthogonalize(g)
    assert ops.orthogonalize(g, out=g) is g
    assert torch.equal(g, ref)


def update_oracle(p, g, m, lr, ema, momentum, wd, scale, sumsq, max_norm, grad_scale, omd):
  p, g, m, ema = (t.double() for t in (p, g, m, ema))
  coef = grad_scale
  if sumsq is not None and max_norm > 0:
    coef *= min(1.0, max_norm / (math.sqrt(sumsq) * grad_scale + 1e-6))
  g = g * coef
  m = m + (1 - momentum) * (g - m)
  o = oracle(g + momentum * (m - g))
  scale = 0.2 * math.sqrt(max(p.shape[-2:])) if scale is None else scale
  move = lr * scale * o
  p = p * (1 - lr * wd) - move
  return p, m, ema - omd * (ema - p), move


@pytest.mark.parametrize('n,r,c', [(1, 1, 1), (1, 3, 50), (2, 384, 128), (3, 100, 257), (1, 515, 129)])
@pytest.mark.parametrize('variant', ['full', 'plain', 'clipped', 'scaled'])
def test_muon_update(ops, n, r, c, variant):
  gen = torch.Generator().manual_seed(r * c)
  p, m, e = (torch.randn(n, r, c, generator=gen) * 0.04 for _ in range(3))
  g = gradient(n, r, c, seed=r)
  kw = dict(lr=0.02, momentum=0.95, wd=0.1, scale=None, sumsq=None, max_norm=0.0, grad_scale=1.0, omd=0.01)
  if variant == 'plain':
    kw.update(wd=0.0, momentum=0.0)
  if variant == 'clipped':
    kw.update(sumsq=float((3 * g).double().square().sum()), max_norm=0.5, grad_scale=0.25)
  if variant == 'scaled':
    kw.update(scale=0.7, sumsq=1e-6, max_norm=1.0)          # below the limit: not clipped
  P, G, M = p.cuda(), g.cuda(), m.cuda()
  E = None if variant == 'plain' else e.cuda()
  W = None if variant == 'plain' else torch.zeros(n, r, c, dtype=torch.bfloat16, device='cuda')
  ops.muon_update(P, G, M, kw['lr'], ema=E, w16=W, momentum=kw['momentum'], weight_decay=kw['wd'], scale=kw['scale'],
                  sumsq=None if kw['sumsq'] is None else torch.tensor([kw['sumsq']], device='cuda'),
                  max_norm=kw['max_norm'], grad_scale=kw['grad_scale'], ema_one_minus_decay=kw['omd'])
  wp, wm, we, move = update_oracle(p, g, m, ema=e, **kw)
  u = 2.0 ** -24
  assert torch.equal(G.cpu(), g)
  # the momentum: four fp32 roundings of values no larger than |g| and |m|
  assert ((M.cpu().double() - wm).abs() <= 8 * u * (g.abs().double() * kw['grad_scale'] + m.abs().double())).all()
  # the weights: the factor's tolerance on the move, and the roundings of p
  assert (P.cpu().double() - wp).norm() <= tol_factor(5) * move.norm() + 4 * u * (p.double().norm() + move.norm())
  if E is not None:
    new = P.cpu().double()
    want = e.double() - kw['omd'] * (e.double() - new)
    assert ((E.cpu().double() - want).abs() <= 4 * u * (e.abs().double() + new.abs())).all()
    assert torch.equal(W, P.to(torch.bfloat16))


def test_muon_update_in_flat_buffers(ops):
  """Matrices at a constant stride inside flat buffers, as the trainer holds them:
  nothing between them is written, and each is moved as it is alone."""
  n, r, c, stride, off = 3, 96, 64, 96 * 64 + 640, 128
  gen = torch.Generator().manual_seed(0)
  flat = {k: torch.randn(off + n * stride, generator=gen).cuda() * 0.1 for k in 'pgme'}
  flat['w'] = flat['p'].to(torch.bfloat16)
  before = {k: v.clone() for k, v in flat.items()}
  v = {k: t[off:off + n * stride].view(n, stride)[:, :r * c].view(n, r, c) for k, t in flat.items()}
  alone = {k: v[k][1].clone() for k in 'pgme'}
  wal = torch.zeros(r, c, dtype=torch.bfloat16, device='cuda')
  ops.muon_update(v['p'], v['g'], v['m'], 1e-2, ema=v['e'], w16=v['w'], ema_one_minus_decay=0.1)
  ops.muon_update(alone['p'], alone['g'], alone['m'], 1e-2, ema=alone['e'], w16=wal, ema_one_minus_decay=0.1)
  for k in 'pme':
    assert torch.equal(v[k][1], alone[k])
    assert not torch.equal(flat[k], before[k])
  assert torch.equal(v['w'][1], wal) and torch.equal(flat['g'], before['g'])
  for k, t in flat.items():
    inside = torch.zeros_like(t, dtype=torch.bool)
    inside[off:off + n * stride].view(n, stride)[:, :r * c] = True
    assert torch.equal(t[~inside], before[k][~inside]), k


def test_muon_update_captured(ops):
  n, r, c = 2, 130, 200
  gen = torch.Generator().manual_seed(1)
  p, m = (torch.randn(n, r, c, generator=gen).cuda() * 0.1 for _ in range(2))
  g = gradient(n, r, c, seed=1).cuda()
  ss = torch.tensor([4.0], device='cuda')
  q, k = p.clone(), m.clone()
  step = lambda a, b: ops.muon_update(a, g, b, 1e-2, sumsq=ss, max_norm=1.0)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    step(p, m)
  for i in range(4):
    g.copy_(gradient(n, r, c, seed=10 + i))
    graph.replay()
    torch.cuda.synchronize()
    step(q, k)
    assert torch.equal(p, q) and torch.equal(m, k), i


def test_past_32_bit_offsets(ops):
  """Matrices, and rows of one, more than 2^31 elements apart: moved as they are side by side."""
  n, r, c, far = 2, 70, 140, 2 ** 31 + 64
  flat = {k: torch.empty(far + 70 * 200, dtype=torch.bfloat16 if k == 'w' else torch.float32, device='cuda')
          for k in 'pgmew'}
  gen = torch.Generator().manual_seed(3)
  near = {k: (torch.randn(n, r, c, generator=gen) * 0.1).cuda() for k in 'pgme'}
  near['w'] = near['p'].to(torch.bfloat16)
  away = {k: t.as_strided((n, r, c), (far, 200, 1)) for k, t in flat.items()}
  for k in away:
    away[k].copy_(near[k])
  assert torch.equal(ops.orthogonalize(away['g']), ops.orthogonalize(near['g']))
  for v in (away, near):
    ops.muon_update(v['p'], v['g'], v['m'], 1e-2, ema=v['e'], w16=v['w'], ema_one_minus_decay=0.1)
  assert all(torch.equal(away[k], near[k]) for k in near)
  rows = flat['p'].as_strided((2, 50), (far, 1))
  assert torch.equal(ops.orthogonalize(rows), ops.orthogonalize(rows.contiguous()))
  wide = ops.orthogonalize(away['g'], out=away['w'])
  assert wide is away['w'] and torch.equal(wide, ops.orthogonalize(near['g']))
