"""Build the in-tree shared library ``noise_b200/libnoise_b200.so`` (sm_100a) with nvcc.

The library has no PyTorch dependency: it exports the C ABI of ``include/noise_b200.h`` and links the CUDA runtime
statically. ``noise_b200/_decode_ext.so`` is the Python extension of ``noise_b200.decode`` (argument checks, torch
allocation, the C calls), built with g++ against torch. ``python -m noise_b200.build`` (or ``__graft_entry__.build()``)
rebuilds either when a source is newer.
"""
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / 'csrc'
LIB = PKG / 'libnoise_b200.so'
SOURCES = sorted(CSRC.glob('*.cu'))
EXT = PKG / '_decode_ext.so'
EXT_SOURCE = CSRC / 'binding.cpp'
HEADERS = sorted(CSRC.glob('*.cuh')) + sorted((ROOT / 'include').glob('*.h'))
ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']


def nvcc():
    for cand in (os.environ.get('NVCC'), shutil.which('nvcc'), '/usr/local/cuda/bin/nvcc'):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError('nvcc not found')


def stale():
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    return any(p.stat().st_mtime > t for p in SOURCES + HEADERS + [Path(__file__)])


def build_ext(force=False):
    """The extension of noise_b200.decode (g++ against the installed torch)."""
    if not force and EXT.exists() and all(p.stat().st_mtime <= EXT.stat().st_mtime
                                          for p in [EXT_SOURCE, ROOT / 'include' / 'noise_b200.h', Path(__file__)]):
        return EXT
    import torch
    home, cuda = Path(torch.__file__).resolve().parent, Path(nvcc()).resolve().parents[1]
    tmp = EXT.with_suffix('.so.tmp')
    subprocess.run([os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-shared', '-fPIC',
                    f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}',
                    '-I', str(ROOT / 'include'), '-I', str(home / 'include'),
                    '-I', str(home / 'include' / 'torch' / 'csrc' / 'api' / 'include'),
                    '-I', sysconfig.get_paths()['include'], '-I', str(cuda / 'include'), '-o', str(tmp),
                    str(EXT_SOURCE), '-L', str(home / 'lib'), '-ltorch_python', '-ltorch_cpu', '-lc10', '-lc10_cuda',
                    '-ldl'], check=True)
    os.replace(tmp, EXT)
    return EXT


def build(force=False, verbose=False):
    build_ext(force)
    if not force and not stale():
        return LIB
    tmp = LIB.with_suffix('.so.tmp')
    cmd = [nvcc(), *ARCH, '-O3', '-lineinfo', '-std=c++17', '-DNOISE_B200_BUILD',
           '-I', str(ROOT / 'include'), '-I', str(CSRC), '-Xcompiler', '-fPIC,-O3', '-shared', '-cudart', 'static',
           '-o', str(tmp), *map(str, SOURCES)]
    if verbose:
        cmd.insert(1, '-Xptxas=-v')
        print(' '.join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == '__main__':
    build(force='--force' in sys.argv, verbose='-v' in sys.argv)
    print(LIB)
