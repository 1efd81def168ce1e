"""Compiler and linker flags of an extension of this interpreter's torch, or an
error that says why there can be none; with --stamp what identifies the two,
without importing torch."""
import sys
import sysconfig
from importlib import metadata
from pathlib import Path


def stamp():
    torch = metadata.distribution('torch')
    return f'{sys.executable} {sys.version.split()[0]} torch {torch.version} {torch.locate_file("torch")}'


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
    out += [f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}',
            f'-DFERRYB_TORCH_VERSION="{torch.__version__}"']
    out += [f'-L{p}' for p in ext.library_paths('cuda')]
    return ' '.join(out + ['-lc10', '-lc10_cuda', '-ltorch_cpu', '-ltorch_cuda', '-ltorch', '-ltorch_python'])


if __name__ == '__main__':
    print(stamp() if '--stamp' in sys.argv[1:] else flags())
