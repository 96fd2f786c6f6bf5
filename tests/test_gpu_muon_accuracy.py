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
