"""Compiler and linker flags of an extension of this interpreter's torch, or an
error that says why there can be none."""
import sys
import sysconfig
from pathlib import Path


def flags():
    include = sysconfig.get_paths()['include']
    if not (Path(include) / 'Python.h').exists():
        sys.exit(f'there is no Python.h in {include}')
    try:
        import torch
        from torch.utils import cpp_extension as ext
    except ImportError as e:
        sys.exit(f'{sys.executable} cannot import torch: {e}')
    if torch.version.cuda is None:
        sys.exit(f'torch {torch.__version__} is built without CUDA')
    out = [f'-I{p}' for p in ext.include_paths('cuda') + [include]]
    out.append(f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}')
    out += [f'-L{p}' for p in ext.library_paths('cuda')]
    return ' '.join(out + ['-lc10', '-lc10_cuda', '-ltorch_cpu', '-ltorch_cuda', '-ltorch', '-ltorch_python'])


if __name__ == '__main__':
    print(flags())
