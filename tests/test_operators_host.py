"""CPU-only checks of the token scores' and the orthogonalised update's entry
points: refusals (before any launch) and workspace arithmetic."""
import math

import pytest
import torch

from mdlm_amd import _lib, ops


def _scores(**kw):
  a = dict(logits=16, ld=100, dtype=0, xt=16, x0=16, logp=16, ent=16, lse=16, tl=16, ti=16, rows=1, V=100, mask=99,
           k=2, st=0)
  a.update(kw)
  _lib.call('mdlm_subs_scores', *a.values())


@pytest.mark.parametrize('bad,text', [
  (dict(logits=0), 'null pointer'), (dict(xt=0), 'null pointer'), (dict(lse=0), 'null pointer'),
  (dict(tl=0), 'alternatives'), (dict(ti=0), 'alternatives'), (dict(V=0), 'bad shape'), (dict(ld=99), 'bad shape'),
  (dict(rows=-1), 'bad shape'), (dict(rows=1 << 31), 'bad shape'), (dict(mask=100), 'mask index'),
  (dict(mask=-1), 'mask index'), (dict(k=65), 'top_k'), (dict(k=-1), 'top_k'), (dict(V=2, mask=1, k=2), 'top_k'),
  (dict(dtype=7), 'dtype')])
def test_scores_refusals(bad, text):
  with pytest.raises(RuntimeError, match=text):
    _scores(**bad)


def _scores_bwd(**kw):
  a = dict(logits=16, ld=100, dtype=0, xt=16, x0=16, lse=16, ent=16, gl=0, gh=0, ti=16, gt=16, k=2, dl=16, ldo=100,
           rows=1, V=100, mask=99, st=0)
  a.update(kw)
  _lib.call('mdlm_subs_scores_bwd', *a.values())


@pytest.mark.parametrize('bad,text', [
  (dict(logits=0), 'null pointer'), (dict(lse=0), 'null pointer'), (dict(dl=0), 'null pointer'),
  (dict(ti=0), 'alternatives'), (dict(gt=0), 'alternatives'), (dict(ldo=99), 'bad shape'), (dict(ld=99), 'bad shape'),
  (dict(ldo=101, rows=2), 'in place'),
  (dict(mask=100), 'mask index'), (dict(k=65), 'top_k'), (dict(dtype=7), 'dtype')])
def test_scores_bwd_refusals(bad, text):
  with pytest.raises(RuntimeError, match=text):
    _scores_bwd(**bad)


def _ortho(**kw):
  a = dict(g=256, ldg=64, gs=4096, dtype=0, out=256, ldo=64, os=4096, n=2, rows=64, cols=64, steps=5, a=3.4445,
           b=-4.775, c=2.0315, eps=1e-7, ws=256, st=0)
  a.update(kw)
  _lib.call('mdlm_orthogonalize', *a.values())


@pytest.mark.parametrize('bad,text', [
  (dict(g=0), 'null pointer'), (dict(out=0), 'null pointer'), (dict(ws=0), 'null pointer'), (dict(dtype=5), 'dtype'),
  (dict(n=-1), 'bad shape'), (dict(rows=-4), 'bad shape'), (dict(cols=1 << 18), 'bad shape'),
  (dict(ldg=63), 'overlapping'), (dict(gs=4095), 'overlapping'), (dict(ldo=63), 'overlapping'),
  (dict(os=0), 'overlapping'), (dict(steps=0), 'steps'), (dict(steps=33), 'steps'), (dict(c=0.0), 'coefficients'),
  (dict(a=math.nan), 'coefficients'), (dict(a=17.0), 'coefficients'), (dict(b=40.0), 'coefficients'),
  (dict(eps=0.0), 'eps'), (dict(eps=math.inf), 'eps'), (dict(ws=128), 'aligned')])
def test_orthogonalize_refusals(bad, text):
  with pytest.raises(RuntimeError, match=text):
    _ortho(**bad)


def _muon(**kw):
  a = dict(p=256, g=512, m=768, ema=0, w=0, ld=64, stride=4096, n=2, rows=64, cols=64, lr=1e-3, momentum=0.95, wd=0.0,
           scale=1.0, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, omd=0.0, sumsq=0, max_norm=0.0, gs=1.0, ws=256,
           st=0)
  a.update(kw)
  _lib.call('mdlm_muon_update', *a.values())


@pytest.mark.parametrize('bad,text', [
  (dict(p=0), 'null pointer'), (dict(m=0), 'null pointer'), (dict(ws=0), 'null pointer'), (dict(ld=60), 'overlapping'),
  (dict(stride=100), 'overlapping'), (dict(momentum=1.0), 'momentum'), (dict(momentum=-0.1), 'momentum'),
  (dict(momentum=math.nan), 'momentum'), (dict(steps=0), 'steps'), (dict(ws=16), 'aligned'),
  (dict(g=256), 'different'), (dict(m=256), 'different'), (dict(m=512), 'different'), (dict(ema=256), 'different'),
  (dict(ema=768), 'different'), (dict(ema=512), 'different'), (dict(w=256), 'different'), (dict(w=512), 'different'),
  (dict(ema=1024, w=1024), 'different')])
def test_muon_update_refusals(bad, text):
  with pytest.raises(RuntimeError, match=text):
    _muon(**bad)


def test_empty_calls_need_no_gpu():
  _scores(rows=0)
  _scores_bwd(rows=0)
  _ortho(n=0)
  _ortho(rows=0)
  _muon(cols=0)


def test_workspaces():
  one = ops.workspace_bytes('orthogonalize', 1, 100, 300)
  assert one >= 100 * 300 * 5 + 2 * 100 * 100 * 2
  assert ops.workspace_bytes('orthogonalize', 1, 300, 100) == one       # worked on the short side
  assert one < ops.workspace_bytes('orthogonalize', 4, 100, 300) <= 4 * one + 8192
  # past 2^31 bytes without wrapping
  assert ops.workspace_bytes('orthogonalize', 16, 8192, 65536) > 16 * 8192 * 65536 * 5
  for bad in ((0, 4, 4), (1, 0, 4), (1, 4, -1), (1, 1 << 18, 4)):
    with pytest.raises(RuntimeError, match='bad shape'):
      ops.workspace_bytes('orthogonalize', *bad)


def test_wrappers_refuse_cpu_tensors():
  x, i = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
  f = torch.zeros(2)
  for call in (lambda: ops.subs_scores(x, i, i, 7), lambda: ops.subs_scores_bwd(x, i, i, 7, f, f, f),
               lambda: ops.orthogonalize(x), lambda: ops.muon_update(x, x, x, 1e-3)):
    with pytest.raises(RuntimeError, match='no CPU fallback'):
      call()


def test_config_keys():
  from mdlm_amd.config import load_config
  cfg = load_config([])
  assert cfg.optim.name == 'adamw' and cfg.training.entropy_weight == 0.0
  cfg = load_config(['optim.name=muon', 'optim.momentum=0.9', 'training.entropy_weight=0.1'])
  assert cfg.optim.name == 'muon' and cfg.optim.momentum == 0.9 and cfg.training.entropy_weight == 0.1


def test_muon_stacks_cover_the_blocks():
  """The flat layout that the optimizer splits: stacks at a constant stride, AdamW's
  ranges and the stacks together every element once."""
  from types import SimpleNamespace

  from mdlm_amd.shadow import flat_layout
  from mdlm_amd.train import Trainer
  shapes = {'vocab_embed.embedding': (30, 16)}
  for i in range(3):
    shapes.update({f'blocks.{i}.norm1.weight': (16,), f'blocks.{i}.attn_qkv.weight': (48, 16),
                   f'blocks.{i}.attn_out.weight': (16, 16), f'blocks.{i}.norm2.weight': (16,),
                   f'blocks.{i}.mlp.0.weight': (64, 16), f'blocks.{i}.mlp.0.bias': (64,),
                   f'blocks.{i}.mlp.2.weight': (16, 64), f'blocks.{i}.mlp.2.bias': (16,),
                   f'blocks.{i}.adaLN_modulation.weight': (96, 8)})
  shapes['output_layer.linear.weight'] = (30, 16)
  table, n_flat = flat_layout(list(shapes.values()))
  t = SimpleNamespace(optimizer='muon', n_flat=n_flat, offsets=dict(zip(shapes, table)), bb=SimpleNamespace(n_blocks=3),
                      MUON_NAMES=Trainer.MUON_NAMES, dev='cpu')
  Trainer._split_parameters(t)
  seen = torch.zeros(n_flat, dtype=torch.int32)
  for a, b in t.adamw_ranges:
    seen[a:b] += 1
  for s in t.muon_stacks:
    Trainer._stack(t, seen, *s).add_(1)
  assert (seen == 1).all()
  assert len(t.muon_stacks) == 4 and len(t.adamw_ranges) == 3 * 3 + 1
  t.optimizer = 'adamw'
  Trainer._split_parameters(t)
  assert t.adamw_ranges == [(0, n_flat)] and t.muon_stacks == []
