"""When the native parts are compiled again: the extension also when the torch or
Python it was made for is not the one that runs, and never in the library's way.
The compilers are stand-ins."""
import os
import types

import pytest
import torch

from gc_moe_b200 import build


@pytest.fixture
def tree(monkeypatch, tmp_path):
    """A package directory of its own; ``ran`` names the parts that were compiled."""
    state = types.SimpleNamespace(ran=[], fail=None)
    (tmp_path / 'csrc').mkdir()
    (tmp_path / 'include').mkdir()
    for name in ('csrc/gcmoe.cu', 'csrc/torch_binding.cpp', 'include/gcmoe.h'):
        (tmp_path / name).write_text('')
    monkeypatch.setattr(build, 'PACKAGE_DIR', str(tmp_path))
    monkeypatch.setattr(build, 'SOURCE', str(tmp_path / 'csrc/gcmoe.cu'))
    monkeypatch.setattr(build, 'BINDING_SOURCE', str(tmp_path / 'csrc/torch_binding.cpp'))
    monkeypatch.setattr(build, 'HEADER', str(tmp_path / 'include/gcmoe.h'))
    monkeypatch.setattr(build, 'LIBRARY', str(tmp_path / 'libgcmoe_sm100.so'))
    monkeypatch.setattr(build, 'BINDING', str(tmp_path / '_torch_binding.so'))
    monkeypatch.setattr(build, '_newest_source_mtime', lambda: os.path.getmtime(build.SOURCE))

    def run(cmd, **kwargs):
        part = os.path.basename(cmd[cmd.index('-o') + 1])
        state.ran.append(part)
        if part == state.fail:
            return types.SimpleNamespace(returncode=1, stdout='', stderr='no such header')
        with open(cmd[cmd.index('-o') + 1], 'w') as f:
            f.write('')
        return types.SimpleNamespace(returncode=0, stdout='', stderr='')

    monkeypatch.setattr(build.subprocess, 'run', run)
    return state


def test_nothing_is_compiled_twice(tree):
    build.build()
    assert sorted(tree.ran) == ['_torch_binding.so', 'libgcmoe_sm100.so']
    build.build()
    assert len(tree.ran) == 2
    build.build(force=True)
    assert len(tree.ran) == 4


def test_another_torch_compiles_the_extension_again(tree, monkeypatch):
    build.build()
    monkeypatch.setattr(torch, '__version__', '99.0.0')
    build.build()
    assert tree.ran[2:] == ['_torch_binding.so']
    build.build()
    assert len(tree.ran) == 3


def test_an_extension_of_unknown_origin_is_compiled_again(tree):
    """Its file is newer than its sources, but nothing says what it was made for."""
    open(build.BINDING, 'w').close()
    build.build()
    assert '_torch_binding.so' in tree.ran


def test_the_library_does_not_wait_for_the_extension(tree):
    tree.fail = '_torch_binding.so'
    with pytest.raises(RuntimeError, match='no such header'):
        build.build()
    assert os.path.exists(build.LIBRARY)
    tree.fail = None
    build.build()                                           # a failed compilation counts as none
    assert tree.ran == ['libgcmoe_sm100.so', '_torch_binding.so', '_torch_binding.so']
