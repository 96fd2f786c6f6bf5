"""How far the orthogonalised update is from 64 bits, on matrices whose small singular
values a rounding of X would drown.

Bound (2-norm of the difference over that of the result).  In a step P - mu I, the X
that it meets and D (twice) are rounded to fp16, together at most 2 x 2^-11 of the result if
all are at their largest.  In matrices of hundreds of rows they are independent and spread
evenly over their half steps, 1/sqrt(3) of the largest on average, and five steps add in squares:
sqrt(5) x 2 x 2^-11 / sqrt(3) = 1.26e-3.  X itself is held in two words, 2^-15 of an
entry at most (half a step of e4m3, 2^-4, of half a step of fp16), again over sqrt(3) on
average, of norm 1 at the start; a step makes a difference at most a = 3.4445 times as large,
484 in all: 484 x 2^-15 / sqrt(3) / |result|.  With the second word lost that is 16 times as much.
"""
import math

import pytest
import torch

from test_gpu_muon_words import move

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315


@pytest.fixture(scope='module')
def ops():
  assert torch.cuda.is_available()
  from mdlm_amd import ops as _ops
  return _ops


def exact(g, steps=5):
  x = g.double()
  if x.shape[0] > x.shape[1]:
    return exact(g.T.contiguous(), steps).T
  x = x / (x.norm() + 1e-7)
  for _ in range(steps):
    q = x @ x.T.contiguous()
    x = A * x + (B * q + C * (q @ q)) @ x
  return x


def bound(want):
  words = A ** 5 * 2.0 ** -15 / math.sqrt(3) / want.norm().item()
  return math.hypot(math.sqrt(5) * 2 * 2.0 ** -11 / math.sqrt(3), words)


def decaying(r, c, seed=0):
  """Singular values that fall off as i^-1.5."""
  gen = torch.Generator(device='cuda').manual_seed(seed)
  s = min(r, c)
  sv = torch.arange(1, s + 1, device='cuda').float() ** -1.5
  return (torch.randn(r, s, generator=gen, device='cuda') * sv) @ torch.randn(s, c, generator=gen, device='cuda')


def check(ops, g):
  want = exact(g)
  err = ((move(ops, g).double() - want).norm() / want.norm()).item()
  assert err < bound(want), (err, bound(want))


@pytest.mark.parametrize('r,c', [(256, 512), (128, 1024), (640, 1291), (4096, 1024), (2048, 8192), (4096, 8192)])
def test_decaying_spectrum(ops, r, c):
  check(ops, decaying(r, c))


def low_rank(r, c, seed=0):
  """A signal of rank min/16 and noise of 2 % of its size."""
  gen = torch.Generator(device='cuda').manual_seed(seed)
  k = min(r, c) // 16
  signal = torch.randn(r, k, generator=gen, device='cuda') @ torch.randn(k, c, generator=gen, device='cuda')
  return signal / math.sqrt(k) + 0.02 * torch.randn(r, c, generator=gen, device='cuda')


@pytest.mark.parametrize('r,c', [(256, 512), (128, 1024), (1024, 4096), (8192, 2048), (4096, 8192)])
def test_low_rank_and_noise(ops, r, c):
  check(ops, low_rank(r, c))


@pytest.mark.parametrize('steps', [1, 2, 3, 5])
@pytest.mark.parametrize('n,r,k', [(2, 24, 7), (1, 128, 3), (1, 300, 4), (3, 150, 64)])
def test_equal_singular_values(ops, n, r, k, steps):
  """Rows that do not meet, each k columns of its own, all of one length: every product
  is diagonal, and an element x sees what is lost on the diagonals.  D's rounding enters to
  second order, X is held in two words, and P is exact but for fp32; in steps before the last
  three the first word of X alone meets P - a.  A is made of the first words alone: of a sum of
  squares t each term is off by at most 2 x 2^-11, and P = a + b t + c t^2 by |b t + 2 c t^2| times
  that.  What a row was off by before grows by x (x p)' / (x p).  With P - mu I rounded to
  fp16 one step loses up to 7e-4, and one or two steps more than the bound in all of these
  shapes."""
  gen = torch.Generator(device='cuda').manual_seed(r)
  rows = torch.randn(n, r, k, generator=gen, device='cuda').double()
  rows = rows / rows.norm(dim=2, keepdim=True)
  g = torch.zeros(n, r, r, k, device='cuda')
  g[:, range(r), range(r)] = rows.float()
  s, off, floor = r ** -0.5, 2.0 ** -15, 2.0 ** -29
  for it in range(steps):
    t = s * s
    p, grows = A + B * t + C * t * t, A + 3 * B * t + 5 * C * t * t
    own = C * ((t + B / (2 * C)) * 2.0 ** -11) ** 2 + 16 * 2.0 ** -24 * A
    own += 2 * 2.0 ** -11 * abs(B * t + 2 * C * t * t)
    if it + 3 < steps:
      own += 2.0 ** -11 * abs(p - A)
    off = off * max(1.0, abs(grows / p)) * (1 + 10 * off) + own / abs(p) + 2.0 ** -15
    floor = floor * max(abs(p), abs(grows)) + 2.0 ** -29
    s *= p
  want = torch.zeros(n, r, r, k, dtype=torch.float64, device='cuda')
  want[:, range(r), range(r)] = rows * s
  for got in (move(ops, g.view(n, r, r * k), steps=steps),
              move(ops, g.view(n, r, r * k).transpose(1, 2).contiguous(), steps=steps).transpose(1, 2)):
    err = (got.reshape(n, r, r, k).double() - want).abs()
    assert (err <= off * want.abs() + floor).all(), ((err - floor) / want.abs()).nan_to_num(0).max().item() / off
