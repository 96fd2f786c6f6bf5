"""CPU-only: what the library's makefile rebuilds."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, 'mdlm_amd', 'csrc')


@pytest.fixture
def tree(tmp_path):
  """The sources as empty files, built before them all an hour ago (nothing to do)."""
  csrc = tmp_path / 'mdlm_amd' / 'csrc'
  csrc.mkdir(parents=True)
  (tmp_path / 'include').mkdir()
  shutil.copy(os.path.join(CSRC, 'Makefile'), csrc)
  old, new = 1_000_000_000, 1_000_003_600
  files = {csrc / 'Makefile': old, tmp_path / 'include' / 'mdlm_hip.h': old,
           tmp_path / 'mdlm_amd' / 'libmdlm_hip.so': new + 10}
  for f in os.listdir(CSRC):
    if f.endswith(('.hip', '.h')):
      files[csrc / f] = old
    if f.endswith('.hip'):
      files[csrc / (f[:-4] + '.o')] = new
  for f, t in files.items():
    f.touch()
    os.utime(f, (t, t))
  return csrc, [f for f in os.listdir(CSRC) if f.endswith('.hip')]


def _commands(csrc):
  out = subprocess.run(['make', '-n', '-C', str(csrc)], capture_output=True, text=True, check=True).stdout
  return [line for line in out.splitlines() if 'hipcc' in line]


def test_nothing_changed(tree):
  assert _commands(tree[0]) == []


@pytest.mark.parametrize('changed', ['Makefile', 'common.h', '../../include/mdlm_hip.h'])
def test_flags_and_headers_rebuild_every_object(tree, changed):
  csrc, sources = tree
  os.utime(csrc / changed)
  lines = _commands(csrc)
  for src in sources:
    assert any(f'-c {src} ' in line for line in lines), src
  assert any('-shared' in line for line in lines)


def test_one_source_rebuilds_its_own_object(tree):
  csrc, _ = tree
  os.utime(csrc / 'muon.hip')
  assert [line.count('-c muon.hip') + line.count('-shared') for line in _commands(csrc)] == [1, 1]
