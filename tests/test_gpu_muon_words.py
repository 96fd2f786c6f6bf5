"""The two words (fp16 and e4m3) in which the orthogonalised update keeps X between
its products, element by element against 64 bits.

With the coefficients (a, 0, 1e-6) a step is X <- a X but for 1e-6 of X, and what is
left of the error is the words'.  Per step and element, in units of the element:
  the second word is rounded to e4m3, half a step 2^-4 of what it holds, itself at
    most half a step of fp16, 2^-11:                              2^-15
  P - mu I = a - 1 = 2^-7 (or nothing) meets the first word alone:  2^-18
  the step's own c A^2, c = 1e-6, A^2 at most 1:                   2^-20
  fp32 operations, ten at most:                                  10 x 2^-24
and 2^-25 for a second word below the range of e4m3 (half its smallest step 2^-9 over
the scales, 16 or more and 2048).  A first word that its second was not taken from costs
2^-11 .. 2^-10 of the element."""
import pytest
import torch

pytestmark = pytest.mark.gpu

A = 1 + 2.0 ** -7
REL = 2.0 ** -15 + 2.0 ** -18 + 2.0 ** -20 + 10 * 2.0 ** -24


@pytest.fixture(scope='module')
def ops():
  assert torch.cuda.is_available()
  from mdlm_amd import ops as _ops
  return _ops


def move(ops, g, **kw):
  """The orthogonalised matrix in fp32: the step of weights at zero."""
  p = torch.zeros_like(g)
  ops.muon_update(p, g, torch.zeros_like(g), 1.0, momentum=0.0, scale=1.0, **kw)
  return -p


def x0(g):
  x = g.double()
  return x / (torch.linalg.matrix_norm(x, keepdim=True) + 1e-7)


@pytest.mark.parametrize('steps', [1, 2, 4])
@pytest.mark.parametrize('n,r,c', [(1, 64, 4096), (3, 500, 128), (1, 384, 700), (2, 700, 390), (1, 1024, 1100)])
def test_two_words(ops, n, r, c, steps):
  gen = torch.Generator(device='cuda').manual_seed(r + c)
  g = torch.randn(n, r, c, generator=gen, device='cuda')
  got = move(ops, g, steps=steps, coeffs=(A, 0.0, 1e-6)).double()
  want = A ** steps * x0(g)
  err, tol = (got - want).abs(), steps * (REL * want.abs() + 2.0 ** -25)
  assert (err <= tol).all(), f'{int((err > tol).sum())} elements, up to {(err / tol).max().item():.3g} times the bound'


@pytest.mark.parametrize('n,r,c', [(1, 4096, 8192), (1, 1500, 20000), (1, 6000, 3001)])
def test_two_words_of_large_matrices(ops, n, r, c):
  """Their entries are small, and the second word is still there: half its smallest
  step is 2^-10 / (256 x 2048) = 2^-29."""
  gen = torch.Generator(device='cuda').manual_seed(r + c)
  g = torch.randn(n, r, c, generator=gen, device='cuda')
  got = move(ops, g, steps=2, coeffs=(A, 0.0, 1e-6)).double()
  want = A ** 2 * x0(g)
  err, tol = (got - want).abs(), 2 * (REL * want.abs() + 2.0 ** -29)
  assert (err <= tol).all(), f'{int((err > tol).sum())} elements, up to {(err / tol).max().item():.3g} times the bound'


def test_two_words_of_large_entries(ops):
  """A single entry is X_0 = 1, the largest there is.  With a = 2.4 it is 5.76 before the third
  step, where what the first word leaves, 3.5 of 11796, times 256 is past the largest e4m3:
  cut off there, no NaN, and no more lost than the first words' half steps (and those
  of P), 2^-11 each; c A^2 adds 1e-7 x 5.76^4."""
  g = torch.zeros(2, 70, 90, device='cuda')
  g[0, 3, 5] = 0.7
  g[1, 69, 89] = -4e-3
  o = move(ops, g, steps=3, coeffs=(2.4, 0.0, 1e-7))
  for got, want in ((o[0, 3, 5], 2.4 ** 3), (o[1, 69, 89], -2.4 ** 3)):
    assert abs(got.item() / want - 1) <= 3 * 2 * 2.0 ** -11 + 1.2e-4
  o[0, 3, 5] = o[1, 69, 89] = 0
  assert (o == 0).all()


@pytest.mark.parametrize('coeffs,steps', [
  ((3.4445, -4.7750, 2.0315), 32), ((2.0, -0.045, 1e-4), 5), ((3.9, 0.0, 1e-6), 3), ((8.3, -23.6, 17.3), 2),
  ((-2.0, -1.5, 0.5), 1)])
def test_coefficients_that_fp16_holds(ops, coeffs, steps):
  """Those near the limits are accepted, and nothing overflows: a rank-one matrix has
  the singular value 1, the largest there is, here all of it in one entry x.  A step's own
  error, of P = p(x^2): P - mu I and the first word of X are rounded to fp16 (mu between
  1 and a), D's diagonal to second order, X to two words.  What the entry was off by
  before grows by x (x p)' / (x p)."""
  a, b, c = coeffs
  x, off = 1.0, 2.0 ** -15
  for _ in range(steps):
    t = x * x
    p, grows = a + b * t + c * t * t, a + 3 * b * t + 5 * c * t * t
    own = 2 * 2.0 ** -11 * max(abs(p - a), abs(p - 1)) + abs(c) * ((t + b / (2 * c)) * 2.0 ** -11) ** 2
    off = off * abs(grows / p) * (1 + 20 * off) + own / abs(p) + 2.0 ** -15
    x *= p
  g = torch.zeros(1, 140, 150, device='cuda')
  g[0, 139, 7] = 5.0
  o = move(ops, g, steps=steps, coeffs=coeffs)
  assert o.isfinite().all() and (o != 0).sum() == 1
  if steps < 8:      # the usual coefficients do not converge: 32 steps have no digit left
    assert abs(o[0, 139, 7].item() / x - 1) <= off
  full = ops.orthogonalize(torch.randn(1, 140, 150, device='cuda'), steps=steps, coeffs=coeffs)
  assert full.isfinite().all()
