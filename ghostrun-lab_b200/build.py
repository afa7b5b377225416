"""Build librlenv_b200.so in-tree for sm_100a (nvcc, one object per board compiled in parallel), and policy_ops_b200.so, the
PyTorch binding of its policy operators (g++ against torch's headers; it calls the library, and is not linked with it).

    python ghostrun-lab_b200/build.py [--force]

The libraries land next to this file (ghostrun-lab_b200/librlenv_b200.so) so they travel with the repository
snapshot; each is rebuilt when one of its sources under csrc/ or a header under include/ is newer, the binding also when it
was built for another torch or Python. Without torch the library alone is built.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
from pathlib import Path
import subprocess
import sys

HERE = Path(__file__).resolve().parent
CSRC = HERE / 'csrc'
INCLUDE = HERE.parent / 'include'   # the C-ABI header the definitions are compiled against
OUT = HERE / 'librlenv_b200.so'
OPS = HERE / 'policy_ops_b200.so'   # imported as a module by policy_ops.py
OPS_SOURCE = 'policy_ops.cpp'
BUILD = HERE / '_build'
UNITS = ['rlenv_b200.cu', 'board_nrom.cu', 'board_uxrom.cu', 'board_mmc1.cu', 'board_mmc3.cu', 'board_cnrom.cu', 'board_mmc2.cu', 'stem.cu',
         'norm.cu', 'heads.cu', 'sample.cu']
NVCC = os.environ.get('NVCC', '/usr/local/cuda/bin/nvcc' if Path('/usr/local/cuda/bin/nvcc').exists() else 'nvcc')
FLAGS = ['-gencode', 'arch=compute_100a,code=sm_100a', '-O3', '-std=c++17', '-lineinfo', '-fmad=false',
         '--expt-relaxed-constexpr', '-Xcompiler', '-fPIC', '-Xcompiler', '-ffp-contract=off']


def built_for() -> str | None:
    """What the binding is compiled for, as it stands in its file: this torch and this Python. None: there is no torch."""
    try:
        import torch
    except ImportError:
        return None
    return f'policy_ops_b200 for torch {torch.__version__}, {sys.implementation.cache_tag};'


def older(product: Path, sources) -> bool:
    return not product.exists() or any(p.stat().st_mtime > product.stat().st_mtime for p in sources)


def lib_stale() -> bool:
    return older(OUT, [*(p for p in CSRC.iterdir() if p.name != OPS_SOURCE), *INCLUDE.glob('*.h')])


def ops_stale() -> bool:
    """Also where the binding was built for another torch or Python. Without a torch there is none to build."""
    want = built_for()
    return want is not None and (older(OPS, [CSRC / OPS_SOURCE, *INCLUDE.glob('*.h')]) or want.encode() not in OPS.read_bytes())


def stale() -> bool:
    return lib_stale() or ops_stale()


def build_ops() -> Path:
    """The PyTorch binding, compiled for this interpreter and this torch."""
    import sysconfig
    import torch
    root = Path(torch.__file__).parent
    cuda = Path(NVCC).parents[1] / 'include' if '/' in NVCC else Path('/usr/local/cuda/include')
    headers = [root / 'include', root / 'include/torch/csrc/api/include', cuda, sysconfig.get_paths()['include']]
    tmp = OPS.with_suffix('.so.tmp')
    cmd = ['g++', '-O2', '-std=c++17', '-fPIC', '-shared', '-Wall', '-DTORCH_API_INCLUDE_EXTENSION_H',
           f'-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}', f'-DBUILT_FOR="{built_for()}"',
           *[a for h in headers for a in ('-isystem', str(h))], str(CSRC / OPS_SOURCE), '-o', str(tmp), '-L', str(root / 'lib'), '-lc10', '-ltorch', '-ltorch_cpu', '-ltorch_python',
           '-lc10_cuda']
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f'g++ failed on policy_ops.cpp:\n{r.stderr[-4000:]}')
    return tmp


def build(force: bool = False, verbose: bool = False) -> Path:
    """The library, with the binding beside it where there is a torch; each is built again only where it is out of date."""
    need_lib, need_ops = force or lib_stale(), built_for() is not None and (force or ops_stale())
    with cf.ThreadPoolExecutor(len(UNITS) + 1) as ex:
        ops = ex.submit(build_ops) if need_ops else None
        if need_lib:
            build_lib(ex, verbose)
    if ops is not None:
        os.replace(ops.result(), OPS)
    return OUT


def build_lib(ex: cf.Executor, verbose: bool) -> None:
    BUILD.mkdir(exist_ok=True)
    extra = ['-Xptxas', '-v'] if verbose else []

    def compile_unit(u):
        obj = BUILD / (Path(u).stem + '.o')
        cmd = [NVCC, *FLAGS, *extra, '-c', str(CSRC / u), '-o', str(obj)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f'nvcc failed on {u}:\n{r.stderr[-4000:]}')
        return obj, r.stderr

    results = list(ex.map(compile_unit, UNITS))
    if verbose:
        for _, err in results:
            sys.stderr.write(err)
    objs = [str(o) for o, _ in results]
    tmp = OUT.with_suffix('.so.tmp')
    subprocess.run([NVCC, '-gencode', 'arch=compute_100a,code=sm_100a', '-shared', '-cudart', 'static', *objs,
                    '-o', str(tmp)], check=True)
    os.replace(tmp, OUT)


if __name__ == '__main__':
    print(build(force='--force' in sys.argv, verbose='-v' in sys.argv))
