"""Build the sm_100a library: every .cu/.cpp under csrc/ into one shared object, and, where torch is
installed, the torch binding's host helper (torch_ext/tensor_table.cpp) into a Python extension
beside it.

  python colabfold-legacy-kernels_b200/build.py [--jobs N] [--verbose]

Output: src/colabfold_legacy_kernels/kernels/sm100/libcflk_sm100.so (in-tree, git-ignored).
nvcc links cudart statically; libstdc++ and libgcc are linked statically too, so the library
needs only libc and the CUDA driver at run time, as the reference's own libraries do.
"""
import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
OUT_DIR = os.path.join(HERE, 'src', 'colabfold_legacy_kernels', 'kernels', 'sm100')
LIB = os.path.join(OUT_DIR, 'libcflk_sm100.so')
BUILD = os.path.join(HERE, '_build')
TABLE_SRC = os.path.join(HERE, 'torch_ext', 'tensor_table.cpp')
TABLE = os.path.join(OUT_DIR, '_cflk_table.so')

ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']
NVCC_FLAGS = ARCH + ['-O3', '-std=c++17', '-lineinfo', '-Xcompiler', '-fPIC',
                     '-Xcompiler', '-fvisibility=hidden', '-Xptxas', '-warn-spills',
                     '--expt-relaxed-constexpr', '-I', CSRC, '-I', os.path.join(HERE, '..', 'include')]


def nvcc():
    path = shutil.which('nvcc') or '/usr/local/cuda/bin/nvcc'
    if not os.path.exists(path):
        raise RuntimeError('nvcc not found')
    return path


def sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(('.cu', '.cpp')))


def compile_one(src, verbose):
    obj = os.path.join(BUILD, src + '.o')
    cmd = [nvcc()] + NVCC_FLAGS + ['-c', os.path.join(CSRC, src), '-o', obj]
    if verbose:
        cmd += ['-Xptxas', '-v']
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError('nvcc failed on %s:\n%s%s' % (src, r.stdout, r.stderr))
    return obj, r.stderr


def build_table():
    """The extension that reads lists of torch tensors (no run path: torch's libraries are those the
    importing process has loaded). None where torch is not installed: only the torch binding wants it."""
    import sysconfig

    try:
        import torch
    except ImportError:
        return None
    from torch.utils import cpp_extension
    tmp = TABLE + '.tmp'
    cmd = ['g++', '-O2', '-std=c++17', '-shared', '-fPIC', '-fvisibility=hidden',
           '-D_GLIBCXX_USE_CXX11_ABI=%d' % torch._C._GLIBCXX_USE_CXX11_ABI,
           '-I', sysconfig.get_paths()['include']]
    for path in cpp_extension.include_paths():
        cmd += ['-isystem', path]
    cmd += [TABLE_SRC, '-o', tmp]
    for path in cpp_extension.library_paths():
        cmd += ['-L', path]
    cmd += ['-ltorch_python', '-ltorch_cpu', '-ltorch', '-lc10']
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError('g++ failed on %s:\n%s%s' % (TABLE_SRC, r.stdout, r.stderr))
    os.replace(tmp, TABLE)
    return TABLE


def build(jobs=None, verbose=False):
    """Compile and link; returns the library path. Raises on any compiler error; one in the torch
    binding's helper only after the library is linked."""
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(OUT_DIR, exist_ok=True)
    srcs = sources()
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs or os.cpu_count()) as ex:
        table = ex.submit(build_table)
        results = list(ex.map(lambda s: compile_one(s, verbose), srcs))
    for _, log in results:
        if verbose or 'spill' in log:
            sys.stderr.write(log)
    objs = [o for o, _ in results]
    tmp = LIB + '.tmp'
    cmd = [nvcc()] + ARCH + ['-shared', '-o', tmp] + objs + [
        '-Xcompiler', '-static-libstdc++', '-Xcompiler', '-static-libgcc']
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError('link failed:\n%s%s' % (r.stdout, r.stderr))
    os.replace(tmp, LIB)
    table.result()
    return LIB


if __name__ == '__main__':
    ap = argparse.ArgumentParser()
    ap.add_argument('--jobs', type=int, default=None)
    ap.add_argument('--verbose', action='store_true')
    a = ap.parse_args()
    print(build(a.jobs, a.verbose))
