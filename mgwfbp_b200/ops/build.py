# -*- coding: utf-8 -*-
"""Build ``libmgwfbp_b200.so`` in-tree with nvcc for sm_100a.

``python -m mgwfbp_b200.ops.build [--verbose] [--force] [--checked]``.  Every ``.cu`` under ``csrc/`` is compiled to
an object (only when stale) and linked into ``mgwfbp_b200/lib/libmgwfbp_b200.so``.  The CUDA runtime
is linked statically, so the library only needs the driver at load time and can be loaded in a
process that also runs PyTorch.  ``csrc/torch_binding.cpp`` (the autograd nodes and launches of the language-model
operators) is compiled with the host compiler against the installed PyTorch into ``lib/_torch_binding.so``.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from typing import List

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC_DIR = os.path.join(PKG_DIR, 'csrc')
LIB_DIR = os.path.join(PKG_DIR, 'lib')
OBJ_DIR = os.path.join(LIB_DIR, 'obj')
LIB_PATH = os.path.join(LIB_DIR, 'libmgwfbp_b200.so')
# the same sources with -DMGW_CHECKED: index checks inside the table-driven kernels (csrc/common.cuh)
CHECKED_OBJ_DIR = os.path.join(LIB_DIR, 'obj_checked')
CHECKED_LIB_PATH = os.path.join(LIB_DIR, 'libmgwfbp_b200_checked.so')

BINDING_SRC = os.path.join(SRC_DIR, 'torch_binding.cpp')
BINDING_PATH = os.path.join(LIB_DIR, '_torch_binding.so')

ARCH_FLAGS = ['-gencode', 'arch=compute_100a,code=sm_100a']
COMMON = ['-O3', '-std=c++17', '-lineinfo', '-Xcompiler', '-fPIC', '--expt-relaxed-constexpr']


def nvcc_path() -> str:
    cand = os.environ.get('NVCC') or shutil.which('nvcc') or '/usr/local/cuda/bin/nvcc'
    if not os.path.isfile(cand):
        raise RuntimeError('nvcc not found (set NVCC=/path/to/nvcc)')
    return cand


def sources() -> List[str]:
    return sorted(os.path.join(SRC_DIR, f) for f in os.listdir(SRC_DIR) if f.endswith('.cu'))


def _stale(target: str, deps: List[str]) -> bool:
    if not os.path.isfile(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose: bool = False, force: bool = False, checked: bool = False) -> str:
    obj_dir, lib_path = (CHECKED_OBJ_DIR, CHECKED_LIB_PATH) if checked else (OBJ_DIR, LIB_PATH)
    extra = ['-DMGW_CHECKED=1'] if checked else []
    os.makedirs(obj_dir, exist_ok=True)
    nvcc = nvcc_path()
    headers = [os.path.join(SRC_DIR, f) for f in os.listdir(SRC_DIR) if f.endswith(('.h', '.cuh'))]
    objs, rebuilt = [], False
    for src in sources():
        obj = os.path.join(obj_dir, os.path.basename(src)[:-3] + '.o')
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            cmd = [nvcc] + ARCH_FLAGS + COMMON + extra + (['-Xptxas', '-v'] if verbose else []) + ['-I', SRC_DIR, '-c', src, '-o', obj]
            if verbose:
                print(' '.join(cmd), flush=True)
            res = subprocess.run(cmd, capture_output=True, text=True)
            if verbose or res.returncode != 0:
                sys.stderr.write(res.stdout + res.stderr)
            if res.returncode != 0:
                raise RuntimeError('nvcc failed on %s' % src)
            rebuilt = True
    if rebuilt or force or _stale(lib_path, objs):
        cmd = [nvcc] + ARCH_FLAGS + ['-shared', '-cudart', 'static', '-o', lib_path] + objs
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError('link failed')
    return lib_path


def build_binding(verbose: bool = False, force: bool = False) -> str:
    """Compile ``csrc/torch_binding.cpp`` when it, its header or the installed PyTorch has changed."""
    import torch
    root = os.path.dirname(torch.__file__)
    stamp = os.path.join(OBJ_DIR, 'torch_binding.version')
    built_for = ''
    if os.path.isfile(stamp):
        with open(stamp) as f:
            built_for = f.read()
    if not force and built_for == torch.__version__ and not _stale(BINDING_PATH, [BINDING_SRC, os.path.join(SRC_DIR, 'lm_api.h')]):
        return BINDING_PATH
    os.makedirs(OBJ_DIR, exist_ok=True)
    cuda = os.path.dirname(os.path.dirname(nvcc_path()))
    system = [os.path.join(root, 'include'), os.path.join(root, 'include', 'torch', 'csrc', 'api', 'include'),
              sysconfig.get_paths()['include'], os.path.join(cuda, 'include')]
    cmd = [os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-fPIC', '-shared', '-fvisibility=hidden',
           '-D_GLIBCXX_USE_CXX11_ABI=%d' % torch._C._GLIBCXX_USE_CXX11_ABI, '-DTORCH_EXTENSION_NAME=_torch_binding',
           '-DMGW_TORCH_VERSION="%s"' % torch.__version__, '-I', SRC_DIR]
    for d in system:
        cmd += ['-isystem', d]
    cmd += [BINDING_SRC, '-L' + os.path.join(root, 'lib'), '-lc10', '-lc10_cuda', '-ltorch_cpu', '-ltorch_python', '-o', BINDING_PATH]
    if verbose:
        print(' '.join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError('%s failed on %s' % (cmd[0], BINDING_SRC))
    with open(stamp, 'w') as f:
        f.write(torch.__version__)
    return BINDING_PATH


if __name__ == '__main__':
    ap = argparse.ArgumentParser()
    ap.add_argument('--verbose', action='store_true')
    ap.add_argument('--force', action='store_true')
    ap.add_argument('--checked', action='store_true', help='build libmgwfbp_b200_checked.so (kernels verify their indices)')
    a = ap.parse_args()
    print(build(a.verbose, a.force, a.checked))
    print(build_binding(a.verbose, a.force))
