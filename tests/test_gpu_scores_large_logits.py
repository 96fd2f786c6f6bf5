"""Token scores of logits whose size is far above their differences, in 64 bits.

Log-probabilities and entropies depend on differences of logits alone, which fp32
holds exactly here, so the tolerance is that of small logits (test_gpu_scores):
4 (82 + V / 256) units 2^-24 of 1 + |value|."""
import pytest
import torch

from test_gpu_scores import check, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size', [300.0, 1e4, -1e4, 2e6])
@pytest.mark.parametrize('rows,V', [(79, 33), (40, 700), (300, 5000), (2, 60000)])
def test_large_logits(ops, rows, V, size, dtype):  # noqa: F811
  gen = torch.Generator().manual_seed(V)
  mask = V - 1
  x = (torch.randn(rows, V, generator=gen) * 2 + size).to(dtype)
  # chunks of one row that begin low: the running maximum moves
  low = torch.rand(rows, V, generator=gen) < 0.5
  x = torch.where(low, torch.where(torch.rand(rows, V, generator=gen) < 0.5, torch.finfo(dtype).min, size - 40.0), x).to(dtype)
  x0 = torch.randint(0, mask, (rows,), generator=gen)
  check(ops, x.cuda(), torch.full_like(x0, mask), x0, mask, 2)
