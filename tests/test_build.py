"""What build.py takes as out of date: the library and its PyTorch binding each for itself, and a binding that was built for
another torch or Python. Nothing is compiled here."""
from __future__ import annotations

import os

import pytest

import build


@pytest.fixture
def products(tmp_path, monkeypatch):
    """The present library and binding as files of their own, newer than every source, and a compiler that fails."""
    build.build()
    for name in ('OUT', 'OPS'):
        here = tmp_path / getattr(build, name).name
        here.write_bytes(getattr(build, name).read_bytes() if name == 'OPS' else b'')
        monkeypatch.setattr(build, name, here)
    monkeypatch.setattr(build, 'NVCC', str(tmp_path / 'no-compiler'))
    monkeypatch.setattr(build, 'BUILD', tmp_path)
    made = []

    def build_ops():
        made.append('ops')
        (tmp_path / 'ops.tmp').write_bytes(b'again')
        return tmp_path / 'ops.tmp'

    monkeypatch.setattr(build, 'build_ops', build_ops)
    return made


def test_present_products_are_kept(products):
    assert not build.stale() and build.build() == build.OUT and not products


@pytest.mark.parametrize('mine, other', [(b'torch 2.', b'torch 1.'), (b', cpython-3', b', cpython-2')])
def test_a_binding_for_another_torch_or_python(products, mine, other):
    """It is built again, and the library is not."""
    data = build.OPS.read_bytes()
    assert mine in data
    build.OPS.write_bytes(data.replace(mine, other))
    assert build.stale()
    build.build()
    assert products == ['ops'] and build.OPS.read_bytes() == b'again'


def test_a_newer_source_of_the_binding(products, tmp_path, monkeypatch):
    src = tmp_path / 'csrc'
    src.mkdir()
    for name in ('policy_ops.cpp', 'norm.cu'):
        (src / name).write_text('')
        os.utime(src / name, (1, 1))
    monkeypatch.setattr(build, 'CSRC', src)
    assert not build.stale()
    later = build.OPS.stat().st_mtime + 10
    os.utime(src / 'policy_ops.cpp', (later, later))
    build.build()   # with no nvcc
    assert products == ['ops']
    os.utime(src / 'norm.cu', (later, later))
    with pytest.raises(Exception):
        build.build()


def test_without_torch_the_library_alone(products, monkeypatch):
    """A missing binding is not built, and the library is not taken for out of date for want of it."""
    import sys
    monkeypatch.setitem(sys.modules, 'torch', None)   # import torch raises ImportError
    build.OPS.unlink()
    assert not build.stale() and build.build() == build.OUT and not products
