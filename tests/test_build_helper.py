"""The library builds where torch is not installed or its headers do not compile: the torch binding's
helper is the only part that needs them. One small source stands for the kernels here."""
import importlib.util
import os
import sys

import pytest

from conftest import ROOT


@pytest.fixture
def builder(tmp_path, monkeypatch):
    path = os.path.join(ROOT, 'colabfold-legacy-kernels_b200', 'build.py')
    spec = importlib.util.spec_from_file_location('library_build', path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    monkeypatch.setattr(m, 'BUILD', str(tmp_path / 'objects'))
    monkeypatch.setattr(m, 'OUT_DIR', str(tmp_path))
    monkeypatch.setattr(m, 'LIB', str(tmp_path / 'lib.so'))
    monkeypatch.setattr(m, 'TABLE', str(tmp_path / 'table.so'))
    monkeypatch.setattr(m, 'sources', lambda: ['capi.cpp'])
    return m


def test_without_torch(builder, monkeypatch):
    monkeypatch.setitem(sys.modules, 'torch', None)  # as if it were not installed
    assert builder.build() == builder.LIB and os.path.exists(builder.LIB)
    assert not os.path.exists(builder.TABLE)


def test_helper_that_does_not_compile(builder, monkeypatch, tmp_path):
    bad = tmp_path / 'bad.cpp'
    bad.write_text('#error no\n')
    monkeypatch.setattr(builder, 'TABLE_SRC', str(bad))
    with pytest.raises(RuntimeError, match='g\\+\\+ failed'):
        builder.build()
    assert os.path.exists(builder.LIB)  # linked all the same


def test_clipping_says_what_is_missing(monkeypatch, tmp_path):
    from colabfold_legacy_kernels import b200
    monkeypatch.setattr(b200, '_table', None)
    monkeypatch.setattr(b200, 'library_path', lambda *a: str(tmp_path / 'lib.so'))
    for text in (None, 'no library'):
        if text:
            (tmp_path / '_cflk_table.so').write_text(text)
        with pytest.raises(RuntimeError, match='grad_clip: .*_cflk_table.so'):
            b200.clip_grad_norm([], 1.0)
