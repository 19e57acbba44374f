"""Build the C-ABI library libtcq_b200.so in-tree with nvcc for sm_100a, and its PyTorch binding _bind.so (no GPU needed).

    python -m yanlongvla_b200.build [--force] [--verbose]

Every .cu under csrc/ is compiled to an object with
    nvcc -gencode arch=compute_100a,code=sm_100a -lineinfo -O3 -std=c++17 -fmad=false -Xcompiler -fPIC
(-fmad=false: no FMA contraction, the FP32 arithmetic must match the reference definition bit for bit) and linked into
yanlongvla_b200/libtcq_b200.so. Objects are rebuilt only when a source or header is newer. csrc/bind.cpp (host code only) is
compiled by g++ against the installed PyTorch's headers.
"""
import argparse
import os
import re
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / 'csrc'
OBJ = PKG / '_build'
LIB = PKG / 'libtcq_b200.so'
BIND = PKG / '_bind.so'
NVCC = os.environ.get('NVCC', 'nvcc')
ARCH = ['-gencode', 'arch=compute_100a,code=sm_100a']
FLAGS = ['-lineinfo', '-O3', '-std=c++17', '-fmad=false', '-Xcompiler', '-fPIC', '--expt-relaxed-constexpr',
         f'-I{ROOT / "include"}', f'-I{CSRC}', '-Xptxas', '-v']
# Kernels whose warps divide the launch's registers among themselves (setmaxnreg), and the registers a thread that their shares are written
# down for (LAUNCH_REGS in the source). The library does not launch one that was compiled with another number.
LAUNCH_REGS = {r'k_cross_tiles': 168, r'k_attention_many\w*Li2EE': 80}


def _headers():
    return list(CSRC.glob('*.cuh')) + list((ROOT / 'include').glob('*.h'))


def registers(log):
    """(kernel, registers a thread, what its shares are written down for) of the kernels of LAUNCH_REGS in what `ptxas -v` has printed."""
    found = re.findall(r"Compiling entry function '(\w+)'.*?Used (\d+) registers", log, re.S)
    return [(name, int(n), want) for name, n in found for pattern, want in LAUNCH_REGS.items() if re.search(pattern, name)]


def wrong_registers(log):
    return [x for x in registers(log) if x[1] != x[2]]


def _compile(src, verbose=False, extra=()):
    obj = OBJ / (src.stem + '.o')
    newest = max(p.stat().st_mtime for p in [src] + _headers())
    log = OBJ / (src.stem + '.ptxas')
    if obj.exists() and log.exists() and obj.stat().st_mtime >= newest:
        return obj, None
    cmd = [NVCC, *ARCH, *FLAGS, *extra, '-c', str(src), '-o', str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or r.returncode:
        sys.stderr.write(' '.join(cmd) + '\n' + r.stdout + r.stderr)
    if r.returncode:
        raise RuntimeError(f'nvcc failed on {src.name}')
    log.write_text(r.stdout + r.stderr)
    for name, n, want in wrong_registers(r.stdout + r.stderr):
        sys.stderr.write(f'warning: {src.name}: {name} has {n} registers a thread, its warps divide {want}: it will not be launched\n')
    return obj, r.stderr


def build_bind(force=False, verbose=False):
    """The binding of the streaming-memory entry points (csrc/bind.cpp) for the running Python and PyTorch."""
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    src = CSRC / 'bind.cpp'
    stamp = OBJ / 'bind.stamp'
    made_for = f'{sys.version} {torch.__version__}'
    newest = max(p.stat().st_mtime for p in (src, ROOT / 'include' / 'tcq_b200.h', Path(__file__)))
    if not force and BIND.exists() and BIND.stat().st_mtime >= newest and stamp.exists() and stamp.read_text() == made_for:
        return BIND
    cuda = Path(os.environ.get('CUDA_HOME', '/usr/local/cuda'))
    libs = cpp_extension.library_paths()
    cmd = [os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-fPIC', '-shared', f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}',
           f'-DTCQ_TORCH_VERSION="{torch.__version__}"',
           *(f'-I{p}' for p in cpp_extension.include_paths()), f'-I{cuda / "include"}', f'-I{sysconfig.get_paths()["include"]}',
           f'-I{ROOT / "include"}', str(src), '-o', str(BIND), *(f'-L{p}' for p in libs), *(f'-Wl,-rpath,{p}' for p in libs),
           '-ltorch_python', '-ltorch', '-ltorch_cpu', '-lc10', '-lc10_cuda']
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or r.returncode:
        sys.stderr.write(' '.join(cmd) + '\n' + r.stdout + r.stderr)
    if r.returncode:
        raise RuntimeError('g++ failed on bind.cpp')
    stamp.write_text(made_for)
    return BIND


def build(force=False, verbose=False, extra=()):
    OBJ.mkdir(exist_ok=True)
    if force:
        for o in OBJ.glob('*.o'):
            o.unlink()
    srcs = sorted(CSRC.glob('*.cu'))
    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = [o for o, _ in ex.map(lambda s: _compile(s, verbose, extra), srcs)]
    if force or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        cmd = [NVCC, *ARCH, '-shared', '-o', str(LIB), *map(str, objs)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode:
            sys.stderr.write(' '.join(cmd) + '\n' + r.stdout + r.stderr)
            raise RuntimeError('link failed')
    build_bind(force, verbose)                       # last: without it all operators but the streaming memory's work
    return LIB


if __name__ == '__main__':
    ap = argparse.ArgumentParser()
    ap.add_argument('--force', action='store_true')
    ap.add_argument('--verbose', action='store_true')
    ap.add_argument('--ptxas', action='store_true', help='print register / shared-memory use (-Xptxas -v)')
    a = ap.parse_args()
    print(build(force=a.force or a.ptxas, verbose=a.verbose or a.ptxas))
