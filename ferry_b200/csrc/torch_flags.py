"""Compiler and linker flags of an extension of this interpreter's torch."""
import sysconfig

import torch
from torch.utils import cpp_extension as ext

flags = [f'-I{p}' for p in ext.include_paths('cuda') + [sysconfig.get_paths()['include']]]
flags.append(f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}')
flags += [f'-L{p}' for p in ext.library_paths('cuda')]
print(' '.join(flags + ['-lc10', '-lc10_cuda', '-ltorch_cpu', '-ltorch_cuda', '-ltorch', '-ltorch_python']))
