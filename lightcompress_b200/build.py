"""Builds the C-ABI shared library (liblc_b200.so) in-tree with nvcc for sm_100a, and beside it the compiled front of
the W8A8 operators (_calls.so, a Python module over torch's C++ interface and that library) with g++.

    python __graft_entry__.py            (from the repository root; loads this file by path)
    python lightcompress_b200/build.py [--force]

One translation unit per kernel family; objects go to build/, the library next to this file.
"""
import concurrent.futures
import importlib.util
import os
import runpy
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, 'csrc')
LIB = os.path.join(HERE, 'liblc_b200.so')
CALLS_SRC = os.path.join(CSRC, 'host', 'calls.cpp')
CALLS = os.path.join(HERE, '_calls.so')
OBJ_DIR = os.path.join(ROOT, 'build', 'lc_b200')
CALLS_NOTE = os.path.join(OBJ_DIR, '_calls.built_for')

NVCC_FLAGS = ['-gencode', 'arch=compute_100a,code=sm_100a', '-lineinfo', '-O3', '-std=c++17',
              '-Xcompiler', '-fPIC', '-Xcompiler', '-fvisibility=hidden', '--fmad=true']


def _nvcc():
    exe = shutil.which('nvcc') or '/usr/local/cuda/bin/nvcc'
    if not os.path.exists(exe):
        raise RuntimeError('nvcc not found; the CUDA extension cannot be built')
    return exe


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.cu'))


def _deps_mtime():
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(('.cuh', '.h'))]
    hdrs.append(os.path.join(ROOT, 'include', 'lc_b200.h'))
    return max(os.path.getmtime(h) for h in hdrs)


def front_for(torch_dir):
    """What a compiled front is good for: the torch in torch_dir and this interpreter.  torch is found, not imported."""
    version = runpy.run_path(os.path.join(torch_dir, 'version.py'))['__version__']
    return f'torch {version}, {sysconfig.get_config_var("SOABI")}'


def _built_for():
    """The same of the front that lies there, from the note beside it; None where it has none."""
    try:
        with open(CALLS_NOTE) as f:
            return f.read().strip()
    except OSError:
        return None


def _front_is_stale(wanted):
    if not os.path.exists(CALLS) or _built_for() != wanted:
        return True
    header = os.path.join(ROOT, 'include', 'lc_b200.h')
    return os.path.getmtime(CALLS) < max(map(os.path.getmtime, (CALLS_SRC, header)))


def build(force=False, verbose=False):
    os.makedirs(OBJ_DIR, exist_ok=True)
    nvcc = _nvcc()
    hdr_m = _deps_mtime()
    jobs = []
    objs = []
    for src in sources():
        obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + '.o')
        objs.append(obj)
        stale = force or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(src), hdr_m)
        if stale:
            jobs.append([nvcc] + NVCC_FLAGS + ['-c', src, '-o', obj])

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError('nvcc failed: ' + ' '.join(cmd) + '\n' + r.stdout + r.stderr)
        if verbose and (r.stdout or r.stderr):
            print(r.stdout, r.stderr)

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        list(ex.map(run, jobs))
    if jobs or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        run([nvcc, '-shared', '-o', LIB] + objs + ['-gencode', 'arch=compute_100a,code=sm_100a'])
    torch = os.path.dirname(importlib.util.find_spec('torch').origin)
    wanted = front_for(torch)
    if force or _front_is_stale(wanted):
        cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), 'include')
        run(['g++', '-O2', '-std=c++17', '-fPIC', '-shared', '-fvisibility=hidden', '-Wall', f'-DLC_BUILT_FOR="{wanted}"',
             '-I' + sysconfig.get_path('include'), '-I' + os.path.join(torch, 'include'),
             '-I' + os.path.join(torch, 'include', 'torch', 'csrc', 'api', 'include'), '-I' + cuda, CALLS_SRC, '-o', CALLS,
             '-L' + os.path.join(torch, 'lib'), '-ltorch_python', '-ltorch_cpu', '-ltorch_cuda', '-ltorch', '-lc10', '-lc10_cuda',
             '-L' + HERE, '-l:' + os.path.basename(LIB), '-Wl,-rpath,$ORIGIN'])
        with open(CALLS_NOTE, 'w') as f:
            f.write(wanted + '\n')
    return LIB


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose=True))
