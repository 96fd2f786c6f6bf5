"""CPU-only checks of the orthogonalised update beyond test_operators_host.py."""
import pytest

from mdlm_amd import ops
from test_operators_host import _muon, _ortho


@pytest.mark.parametrize('coeffs,steps', [
  ((2.0, -0.07, 1e-4), 1),          # b / 2c = -350: D's diagonal, times 256, is past 65504
  ((2.0, 0.07, 1e-4), 1),
  ((3.9, 0.0, 1e-6), 5),            # 3.9^4 = 231 before the last step: X, times 2048
  ((-3.9, 0.0, 1e-6), 5),
  ((8.3, -23.6, 17.3), 3),          # 2.0 after one step and 370 after two
  ((2.0, 0.0, 32.0), 2),            # 34 after one
  ((1.0, 3.0, 30.0), 3),
  ((16.0, 0.0, 1e-3), 2),           # 16 after one: D = 256, and 256 x 256 = 65536 is past 65504
  ((2.0, 11.0, 2.0), 2)])           # 15 after one step, then p = 105000
def test_coefficients_past_fp16_are_refused(coeffs, steps):
  for call in (_ortho, _muon):
    with pytest.raises(RuntimeError, match='coefficients .* fp16'):
      call(steps=steps, **dict(zip('abc', coeffs)))


def test_workspace_query_refuses_what_the_call_refuses():
  """No workspace of many gigabytes for a call that would not run."""
  assert ops.workspace_bytes('orthogonalize', 1, 32768, 40000) > 0
  for rows, cols in ((32769, 40000), (131072, 32769)):
    with pytest.raises(RuntimeError, match='bad shape'):
      ops.workspace_bytes('orthogonalize', 1, rows, cols)
    with pytest.raises(RuntimeError, match='smaller side'):
      _ortho(n=1, rows=rows, cols=cols, ldg=cols, ldo=cols)
