"""libkfac_torch.so belongs to the torch that it was built with: it is rebuilt for
another one, not loaded by another one, and where it is missing the layer norm is
torch's, as before there was a kernel for it."""
import importlib.util
import os
import shutil
import subprocess
import warnings

import pytest
import torch
import torch.nn.functional as F

from distributed_kfac_pytorch_amd.modules import LayerNorm
from distributed_kfac_pytorch_amd.ops import _lib, ln, vocab

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

needs_build = pytest.mark.skipif(not os.path.exists(_lib.TORCH_LIB_PATH), reason='not built here')


def without(monkeypatch, path):
    monkeypatch.setattr(_lib, 'TORCH_LIB_PATH', str(path))
    monkeypatch.setattr(_lib, '_torch_ops', None)
    monkeypatch.setattr(_lib, '_torch_ops_found', None)


def other_torch(tmp_path):
    """The built library, as another torch's."""
    path = tmp_path / 'libkfac_torch.so'
    shutil.copy(_lib.TORCH_LIB_PATH, str(path))
    (tmp_path / 'libkfac_torch.so.sources').write_text('1.2.3')
    return path


def builder():
    spec = importlib.util.spec_from_file_location('kfac_csrc_build',
                                                  os.path.join(ROOT, 'csrc', 'build.py'))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    return b


@needs_build
def test_missing_or_foreign_library_is_named_once(monkeypatch, tmp_path):
    for path, text in ((tmp_path / 'none.so', 'not built'),
                       (other_torch(tmp_path), 'built with torch 1.2.3')):
        without(monkeypatch, path)
        with pytest.raises(RuntimeError, match=text):
            _lib.torch_ops()
        with pytest.warns(UserWarning, match=text):
            assert not _lib.has_torch_ops()
        with warnings.catch_warnings():
            warnings.simplefilter('error')
            assert not _lib.has_torch_ops()


@needs_build
def test_a_file_that_does_not_load(monkeypatch, tmp_path):
    (tmp_path / 'bad.so').write_text('no library')
    without(monkeypatch, tmp_path / 'bad.so')
    with pytest.raises(RuntimeError, match='not loaded'):
        _lib.torch_ops()


@pytest.mark.skipif(not os.path.exists(_lib.TORCH_LIB_PATH + '.sources'), reason='not built here')
def test_the_built_library_is_this_torchs():
    with open(_lib.TORCH_LIB_PATH + '.sources') as f:
        assert f.read() == torch.__version__
    assert _lib.has_torch_ops() and _lib.torch_ops() is torch.ops.kfac_hip


@pytest.mark.parametrize('stamp,rebuilds', [('1.2.3', True), (None, True), ('same', False)])
def test_another_torch_rebuilds(monkeypatch, tmp_path, stamp, rebuilds):
    b = builder()
    lib = tmp_path / 'libkfac_torch.so'
    lib.write_text('')                                   # newer than every source
    monkeypatch.setattr(b, 'TORCH_LIB', str(lib))
    monkeypatch.setattr(torch.version, 'hip', '7.0')
    if stamp:
        (tmp_path / 'libkfac_torch.so.sources').write_text(
            torch.__version__ if stamp == 'same' else stamp)
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        open(cmd[cmd.index('-o') + 1], 'w').close()
        return subprocess.CompletedProcess(cmd, 0, '', '')
    monkeypatch.setattr(b.subprocess, 'run', run)
    assert b.build_torch_ops(verbose=False) == str(lib)
    assert bool(ran) == rebuilds
    assert (tmp_path / 'libkfac_torch.so.sources').read_text() == torch.__version__


def test_a_torch_without_rocm_builds_the_kernels_alone(monkeypatch, capsys):
    b = builder()
    monkeypatch.setattr(torch.version, 'hip', None)
    monkeypatch.setattr(b.subprocess, 'run', lambda *a, **k: pytest.fail('compiled'))
    assert b.build_torch_ops(force=True) is None
    assert 'no torch for ROCm' in capsys.readouterr().out


@pytest.mark.gpu
def test_the_norm_runs_without_the_library(monkeypatch, tmp_path):
    m = LayerNorm(32, device='cuda')
    x = torch.randn(4, 32, device='cuda', requires_grad=True)
    want = m(x)
    without(monkeypatch, tmp_path / 'none.so')
    with pytest.warns(UserWarning, match='not built'):
        y = m(x)
    assert torch.equal(y, F.layer_norm(x, (32,), m.weight, m.bias))
    assert not ln.eligible(x, (32,)) and torch.allclose(y, want, atol=1e-5)
    y, s = m(x, x)
    assert torch.equal(s, x + x)
    with pytest.raises(RuntimeError, match='not built'):      # nothing else runs these
        vocab.token_logprobs(x, top_k=1)
