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
