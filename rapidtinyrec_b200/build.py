"""Build the native engine: ``csrc/*.cu`` -> ``librtr_b200.so`` for sm_100a.

``python -m rapidtinyrec_b200.build`` (or ``__graft_entry__.build()``) compiles
each translation unit with nvcc in parallel and links one shared library next
to this file, and with g++ the Python module of the 8-bit KV cache's calls
(``kv_call.cpp`` -> ``_kv_call.so``, against torch's headers and libraries).  nvcc cross-compiles, so no GPU is needed.  Objects are rebuilt
only when a source or header is newer than the library.
"""
from __future__ import annotations

import concurrent.futures
import os
import subprocess
import sys
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / 'csrc'
INCLUDE = HERE.parent / 'include'
LIB = HERE / 'librtr_b200.so'
CALLS = HERE / '_kv_call.so'
BUILD_DIR = HERE.parent / '_build'

ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']
NVCC_FLAGS = ['-O3', '-lineinfo', '-std=c++17', '-Xcompiler', '-fPIC', '--expt-relaxed-constexpr',
              '-Xptxas', '-warn-spills', f'-I{INCLUDE}', f'-I{CSRC}']


def nvcc() -> str:
    for cand in (os.environ.get('NVCC'), '/usr/local/cuda/bin/nvcc', 'nvcc'):
        if cand and (Path(cand).exists() or cand == 'nvcc'):
            return cand
    raise RuntimeError('nvcc not found')


def sources():
    return sorted(CSRC.glob('*.cu'))


def _stale() -> bool:
    if not LIB.exists() or not CALLS.exists():
        return True
    newest = max(p.stat().st_mtime for p in list(CSRC.iterdir()) + list(INCLUDE.iterdir()) + [Path(__file__)])
    return newest > min(LIB.stat().st_mtime, CALLS.stat().st_mtime)


def _compile_calls() -> None:
    import torch
    root = Path(torch.__file__).parent
    include = [root / 'include', root / 'include' / 'torch' / 'csrc' / 'api' / 'include',
               sysconfig.get_paths()['include'], Path(nvcc()).parent.parent / 'include', INCLUDE]
    tmp = CALLS.with_suffix('.so.tmp')
    cmd = [os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-fPIC', '-shared', '-w',
           f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}', *[f'-I{p}' for p in include],
           str(CSRC / 'kv_call.cpp'), '-o', str(tmp), f"-L{root / 'lib'}", '-lc10', '-lc10_cuda', '-ltorch_cpu',
           '-ltorch_cuda', '-ltorch_python']
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f'compiling kv_call.cpp failed:\n{res.stdout}\n{res.stderr}')
    tmp.replace(CALLS)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not _stale():
        return LIB
    BUILD_DIR.mkdir(exist_ok=True)
    cc = nvcc()

    def compile_one(src: Path) -> Path:
        obj = BUILD_DIR / (src.stem + '.o')
        cmd = [cc, *ARCH, *NVCC_FLAGS, '-c', str(src), '-o', str(obj)]
        if verbose:
            print(' '.join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f'nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}')
        if verbose and (res.stdout or res.stderr):
            print(res.stdout + res.stderr, flush=True)
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as pool:
        calls = pool.submit(_compile_calls)
        objs = list(pool.map(compile_one, sources()))
        calls.result()
    tmp = LIB.with_suffix('.so.tmp')
    cmd = [cc, *ARCH, '-shared', '-o', str(tmp), *map(str, objs), '-lcudart']
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f'link failed:\n{res.stdout}\n{res.stderr}')
    tmp.replace(LIB)
    return LIB


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose='-v' in sys.argv))
