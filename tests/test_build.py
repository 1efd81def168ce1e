"""The Makefile's rules for the _fast extension, with stand-ins for the
compilers and the interpreter, and the check of a built one: no GPU, no nvcc."""
import shutil
import subprocess
import sys
import types
import warnings
from pathlib import Path

import pytest
import torch

import ferry_b200
from ferry_b200 import _lib

ROOT = Path(__file__).resolve().parents[1]


def _script(path, body):
    path.write_text('#!/bin/sh\n' + body)
    path.chmod(0o755)
    return path


@pytest.fixture
def tree(tmp_path):
    """A copy of the build's files without kernels; nvcc and c++ that only make
    their output; an interpreter whose torch has the version in `torch`."""
    csrc = tmp_path / 'ferry_b200' / 'csrc'
    csrc.mkdir(parents=True)
    for name in ('Makefile', 'torch_flags.py', 'expert_ops_fast.cpp'):
        shutil.copy(ROOT / 'ferry_b200' / 'csrc' / name, csrc)
    shutil.copytree(ROOT / 'include', tmp_path / 'include')
    out = f'while [ "$1" != -o ]; do shift; done; echo built > "$2"; basename "$2" >> {tmp_path / "log"}\n'
    _script(tmp_path / 'nvcc', out)
    _script(tmp_path / 'c++', out)
    (tmp_path / 'torch').write_text('2.0.0\n')
    _script(tmp_path / 'python', f'cat {tmp_path / "torch"}\n')
    return tmp_path


def _make(tree, **tools):
    tools = dict(dict(NVCC=tree / 'nvcc', CXX=tree / 'c++', PYTHON=tree / 'python'), **tools)
    run = subprocess.run(['make', '-C', str(tree / 'ferry_b200' / 'csrc')] + [f'{k}={v}' for k, v in tools.items()],
                         capture_output=True, text=True)
    return run.returncode, run.stdout + run.stderr


def test_builds_both_once(tree):
    lib, fast = tree / 'ferry_b200' / 'libferryb.so', tree / 'ferry_b200' / '_fast.so'
    for _ in range(2):  # the second time there is nothing to do
        status, out = _make(tree)
        assert status == 0, out
        assert lib.exists() and fast.exists()
        assert sorted((tree / 'log').read_text().split()) == ['_fast.so', 'libferryb.so']


@pytest.mark.parametrize('tool', ['CXX', 'PYTHON'])
def test_library_alone_where_the_extension_cannot_be_built(tree, tool):
    """A compiler that fails (no headers, no CUDA libraries in torch), an interpreter without torch."""
    lib, fast = tree / 'ferry_b200' / 'libferryb.so', tree / 'ferry_b200' / '_fast.so'
    broken = _script(tree / 'broken', 'echo the reason >&2; exit 1\n')
    status, out = _make(tree, **{tool: broken})
    assert status == 0, out
    assert lib.exists() and not fast.exists()
    assert 'the reason' in out and '_fast.so is not built' in out
    status, out = _make(tree)  # and again once it can
    assert status == 0 and fast.exists()


def test_extension_is_rebuilt_for_another_torch(tree):
    fast = tree / 'ferry_b200' / '_fast.so'
    assert _make(tree)[0] == 0
    (tree / 'torch').write_text('2.1.0\n')
    assert _make(tree)[0] == 0
    assert fast.exists() and (tree / 'log').read_text().split().count('_fast.so') == 2
    # one that can no longer be built does not stay from before
    (tree / 'torch').write_text('2.2.0\n')
    status, out = _make(tree, CXX=_script(tree / 'broken', 'exit 1\n'))
    assert status == 0 and not fast.exists()


def _flags(tmp_path, torch_source, include=None):
    """torch_flags.py with a stand-in for torch."""
    (tmp_path / 'torch' / 'utils').mkdir(parents=True)
    (tmp_path / 'torch' / '__init__.py').write_text(torch_source)
    (tmp_path / 'torch' / 'utils' / '__init__.py').write_text('')
    (tmp_path / 'torch' / 'utils' / 'cpp_extension.py').write_text(
        'def include_paths(kind): return ["/inc"]\ndef library_paths(kind): return ["/lib"]\n')
    code = f'import sys, sysconfig, runpy\nsys.path.insert(0, {str(tmp_path)!r})\n'
    if include is not None:
        code += f'sysconfig.get_paths = lambda: dict(include={str(include)!r})\n'
    code += f'runpy.run_path({str(ROOT / "ferry_b200" / "csrc" / "torch_flags.py")!r}, run_name="__main__")\n'
    return subprocess.run([sys.executable, '-c', code], capture_output=True, text=True)


STUB = """
__version__ = '2.0.0+x'
class version: cuda = {cuda!r}
class _C: _GLIBCXX_USE_CXX11_ABI = True
"""


def test_flags_name_the_reason(tmp_path):
    (tmp_path / 'Python.h').write_text('')
    run = _flags(tmp_path / 'a', STUB.format(cuda='12.8'), include=tmp_path)
    assert run.returncode == 0 and '-ltorch_cuda' in run.stdout and '2.0.0+x' in run.stdout, run.stderr
    run = _flags(tmp_path / 'b', STUB.format(cuda=None), include=tmp_path)
    assert run.returncode != 0 and 'CUDA' in run.stderr and not run.stdout
    run = _flags(tmp_path / 'c', STUB.format(cuda='12.8'), include=tmp_path / 'a')
    assert run.returncode != 0 and 'Python.h' in run.stderr and not run.stdout
    run = _flags(tmp_path / 'd', 'raise ImportError("none here")\n', include=tmp_path)
    assert run.returncode != 0 and 'none here' in run.stderr and not run.stdout


def _load(monkeypatch, **attributes):
    module = types.ModuleType('ferry_b200._fast')
    module.__dict__.update(attributes, init=lambda *entries: None)
    monkeypatch.setitem(sys.modules, 'ferry_b200._fast', module)
    monkeypatch.setattr(ferry_b200, '_fast', module, raising=False)
    monkeypatch.setattr(_lib, '_fast', None)
    return module, _lib.fast


def test_an_extension_of_another_torch_or_python_is_not_used(monkeypatch):
    python = f'{sys.version_info[0]}.{sys.version_info[1]}.99'  # the last number does not matter
    module, fast = _load(monkeypatch, torch_version=torch.__version__, python_version=python)
    with warnings.catch_warnings():
        warnings.simplefilter('error')
        assert fast() is module
    for stale in (dict(torch_version='1.0', python_version=python), dict(),
                  dict(torch_version=torch.__version__, python_version='2.7.1')):
        _, fast = _load(monkeypatch, **stale)
        with pytest.warns(RuntimeWarning, match='another'):
            assert fast() is _lib._NoFast


def test_the_built_extension_is_this_one():
    assert _lib.fast() is not _lib._NoFast
    assert _lib.fast().torch_version == torch.__version__
