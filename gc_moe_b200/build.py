"""Build the package's native parts in-tree.

    python -m gc_moe_b200.build

``libgcmoe_sm100.so`` (nvcc, sm_100a) holds the kernels and the C ABI and is
loaded with ctypes by ``gc_moe_b200._native``; ``_torch_binding.so`` (g++, torch's
headers) takes the small calls in front of the layer from tensors to that ABI.
Neither is ever rebuilt implicitly at import.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

PACKAGE_DIR = os.path.dirname(os.path.abspath(__file__))
SOURCE = os.path.join(PACKAGE_DIR, 'csrc', 'gcmoe.cu')
LIBRARY = os.path.join(PACKAGE_DIR, 'libgcmoe_sm100.so')
BINDING_SOURCE = os.path.join(PACKAGE_DIR, 'csrc', 'torch_binding.cpp')
BINDING = os.path.join(PACKAGE_DIR, '_torch_binding.so')
HEADER = os.path.join(PACKAGE_DIR, '..', 'include', 'gcmoe.h')


def _newest_source_mtime() -> float:
    roots = [os.path.join(PACKAGE_DIR, 'csrc'), os.path.join(PACKAGE_DIR, '..', 'include')]
    return max(os.path.getmtime(os.path.join(r, f)) for r in roots for f in os.listdir(r))


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile what is missing, older than its sources or (the binding) made for
    another torch or Python; the library's path."""
    library = _build_library(force, verbose)
    _build_binding(force)
    return library


def _build_binding(force: bool) -> None:
    import sysconfig
    import torch
    # An extension works with the torch and the Python it was made for; a note beside it says which.
    made_for = f'torch {torch.__version__}, {sysconfig.get_config_var("SOABI")}'
    note = os.path.splitext(BINDING)[0] + '.made_for'
    if (not force and os.path.exists(BINDING) and os.path.exists(note) and open(note).read() == made_for
            and os.path.getmtime(BINDING) >= max(os.path.getmtime(f) for f in (BINDING_SOURCE, HEADER))):
        return
    if os.path.exists(note):
        os.remove(note)
    torch_dir = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(shutil.which('nvcc') or '/usr/local/cuda/bin/nvcc'))
    include = [os.path.join(torch_dir, 'include'), os.path.join(torch_dir, 'include', 'torch', 'csrc', 'api', 'include'),
               sysconfig.get_paths()['include'], os.path.join(cuda, 'include')]
    if shutil.which('g++') is None:
        raise RuntimeError('g++ not found; _torch_binding.so cannot be built')
    cmd = ['g++', '-O2', '-std=c++17', '-shared', '-fPIC',
           f'-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}', *(f'-isystem{i}' for i in include),
           BINDING_SOURCE, '-o', BINDING, f'-L{os.path.join(torch_dir, "lib")}',
           '-ltorch_python', '-ltorch_cuda', '-ltorch_cpu', '-lc10_cuda', '-lc10']
    result = subprocess.run(cmd, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError('g++ failed:\n' + result.stdout + result.stderr)
    with open(note, 'w') as f:
        f.write(made_for)


def _build_library(force: bool, verbose: bool) -> str:
    if (not force and os.path.exists(LIBRARY)
            and os.path.getmtime(LIBRARY) >= _newest_source_mtime()):
        return LIBRARY
    nvcc = shutil.which('nvcc') or '/usr/local/cuda/bin/nvcc'
    if not os.path.exists(nvcc):
        raise RuntimeError('nvcc not found; libgcmoe_sm100.so cannot be built')
    cmd = [nvcc, '-gencode', 'arch=compute_100a,code=sm_100a', '-O3', '-std=c++17',
           '-lineinfo', '--shared', '-Xcompiler', '-fPIC', '-Xptxas', '-v' if verbose else '-O3',
           '-cudart', 'shared', '-o', LIBRARY, SOURCE]
    result = subprocess.run(cmd, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError('nvcc failed:\n' + result.stdout + result.stderr)
    if verbose:
        print(result.stderr)
    return LIBRARY


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose='-v' in sys.argv))
