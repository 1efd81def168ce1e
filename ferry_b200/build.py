"""Build libferryb.so (sm_100a) and, where this interpreter's torch allows it, _fast.so
in-tree: python -m ferry_b200.build"""
import os
import subprocess
import sys
from pathlib import Path

CSRC = Path(__file__).resolve().parent / 'csrc'


def build(jobs=None, verbose=False):
    jobs = jobs or max(1, min(16, os.cpu_count() or 4))
    out = subprocess.run(['make', '-C', str(CSRC), f'-j{jobs}', f'PYTHON={sys.executable}'], capture_output=not verbose, text=True)
    if out.returncode != 0:
        raise RuntimeError('libferryb build failed:\n' + (out.stdout or '') + (out.stderr or ''))
    if not verbose and not (CSRC.parent / '_fast.so').exists():  # make has said why
        print((out.stderr or '') + out.stdout[-1000:], file=sys.stderr)
    return CSRC.parent / 'libferryb.so'


if __name__ == '__main__':
    print(build(verbose=True))
