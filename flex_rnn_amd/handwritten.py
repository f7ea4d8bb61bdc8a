"""Hand-written kernels (flex_rnn_amd/csrc/*.hip) and the operators over them (csrc/frnn_ops.cpp).

The operators are C++: they allocate, pack argument blocks and launch through the C ABI of include/frnn_rt.h.  When one needs
a kernel for the first time on a device it asks `_load` here by number; the kernel is then compiled with its constants into the
same on-disk cache as the generated ones (or found there) and loaded.

Operators and kernels share argument blocks, so they have to come from the same sources: these are read once, at import, the
library's file name holds their hash (and PyTorch's version, whose C++ interface it uses), and another library is not looked at.
"""
from __future__ import annotations

import contextlib
import ctypes
import glob
import hashlib
import os
import subprocess
import threading
from concurrent.futures import ThreadPoolExecutor
from typing import Dict, Tuple

import torch as th

from . import runtime

_HERE = os.path.dirname(os.path.abspath(__file__))
_CSRC = os.path.join(_HERE, 'csrc')
DTYPES = {th.bfloat16: 0, th.float16: 1, th.float32: 2}      # the kernels' type codes

_lock = threading.Lock()
_modules: list = []             # loaded code objects stay as long as the process
_lib = None


def require(ok, message: str):
    """Argument checks raise what the compiled operators' own checks raise (and also do so under `python -O`)."""
    if not ok:
        raise AssertionError(message)


def sources() -> Dict[str, str]:
    """File name -> text of everything that operators and kernels are made of."""
    out = {}
    for path in sorted([os.path.join(_CSRC, 'frnn_ops.cpp'), os.path.join(os.path.dirname(_HERE), 'include', 'frnn_rt.h'), os.path.abspath(__file__),
                        *(os.path.join(_CSRC, f'{n}.hip') for n in ('layer_norm', 'linear_attention', 'slice_sum'))]):
        if os.path.isfile(path):
            with open(path) as f:
                out[os.path.basename(path)] = f.read()
    return out


def library_name(texts: Dict[str, str], torch_version: str) -> str:
    h = hashlib.sha256(torch_version.encode())
    for name in sorted(texts):
        h.update(f'\0{name}\0'.encode() + texts[name].encode())
    return f'libfrnn_ops.{h.hexdigest()[:16]}.so'


_sources = sources()
OPS_PATH = os.path.join(_HERE, library_name(_sources, th.__version__))


# ------------------------------------------------------------------ kernels by number
Kernel = Tuple[str, str, Tuple[Tuple[str, int], ...]]        # source, kernel, constants


def _block(dtype: int, width: int, out: int, dots: int, fast: int, wide: int) -> Kernel:
    """The walk of linear attention; see csrc/linear_attention.hip.  Two tiles in LDS where two workgroups per compute unit
    still fit (bfloat16 up to 128 columns)."""
    w = (64, 128, 256)[width]
    return ('linear_attention.hip', 'la_block', (('KERNEL_BLOCK', 1), ('IN', dtype), ('W', w), ('OUT', out), ('DOTS', dots), ('FAST', fast), ('WIDE', wide),
                                                 ('NBUF', 2 if dtype == 0 and w <= 128 else 1), ('OCC', 2)))


def _norm(name: str, backward: int):
    def kernel(dtype, pieces, lanes_log, wide) -> Kernel:
        return ('layer_norm.hip', name, (('IN', dtype), ('K', pieces), ('TH', max(256, 1 << lanes_log)), ('GL', 1 << lanes_log), ('WIDE', wide),
                                         ('BACKWARD', backward)))
    return kernel


# kind (as in frnn_ops.cpp) -> number of 6-bit fields, and the kernel they stand for
_KINDS = {
    1: (6, _block),
    2: (0, lambda: ('linear_attention.hip', 'la_gate', (('KERNEL_GATE', 1), ('IN', 0)))),
    3: (1, lambda dtype: ('linear_attention.hip', 'la_step', (('KERNEL_STEP', 1), ('IN', dtype)))),
    4: (0, lambda: ('slice_sum.hip', 'slice_sum', ())),
    5: (4, _norm('ln_fw', 0)),
    6: (4, _norm('ln_bw', 1)),
}


def decode(key: int) -> Kernel:
    for kind, (n, kernel) in _KINDS.items():
        if key >> (6 * n) == kind:
            return kernel(*[key >> (6 * (n - 1 - i)) & 63 for i in range(n)])
    raise KeyError(key)


def builds():
    """Every code object that an operator can ask for."""
    out = [_KINDS[2][1](), _KINDS[4][1]()]
    for dt in DTYPES.values():
        out.append(_KINDS[3][1](dt))
        for w in range(3):
            out += [_block(dt, w, o, d, fast, 0) for o, d in ((1, 0), (1, 1), (0, 0)) for fast in (0, 1)]
            out += [_block(dt, w, 1, d, 1, 1) for d in (0, 1) if dt != 2]
        shapes = [(k, lanes, 0) for k in (1, 2, 4) for lanes in range(7) if k == 1 or lanes == 6] + [(4 if dt == 2 else 2, lanes, 1) for lanes in (8, 9, 10)]
        out += [_KINDS[kind][1](dt, *s) for kind in (5, 6) for s in shapes]
    return out


def build(source: str, name: str, defines=(), force: bool = False) -> str:
    """Path of the code object of kernel `name` from csrc/`source`, compiled with `defines` on a cache miss."""
    opts = ' '.join([runtime.EMITTER_OPTS] + [f'-D{k}={v}' for k, v in defines])
    return runtime.compile_kernel(name, _sources[source], opts=opts, force=force)


def build_all(force: bool = False, workers: int = 6) -> int:
    """Compiles every kernel, side by side; returns their number."""
    cases = builds()
    with ThreadPoolExecutor(max_workers=workers) as pool:
        list(pool.map(lambda c: build(*c, force=force), cases))
    return len(cases)


def _load(device: int, key: int, message: int, capacity: int) -> int:
    try:
        source, name, defines = decode(key)
        with th.cuda.device(device):
            if th.cuda.is_current_stream_capturing():
                raise runtime.RuntimeError_(f'kernel {name} is not loaded yet and cannot be while a graph is captured: '
                                            'make one call with these types and sizes before the capture')
            module = runtime.Module(build(source, name, defines))
            _modules.append(module)
            return module.kernel(name).handle.value
    except BaseException as e:  # noqa: B902  (nothing may leave through the C++ caller)
        text = f'{type(e).__name__}: {e}'.encode()[:capacity - 1] + b'\0'
        ctypes.memmove(message, text, len(text))
        return 0


_LOADER = ctypes.CFUNCTYPE(ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64)
_loader = _LOADER(_load)


# ------------------------------------------------------------------ the operators' library
def build_library(verbose: bool = False) -> str:
    """Compiles csrc/frnn_ops.cpp -> flex_rnn_amd/libfrnn_ops.<hash>.so (host code only, against PyTorch's headers) and removes
    those of other sources."""
    root = os.path.dirname(th.__file__)
    tmp = OPS_PATH + f'.tmp{os.getpid()}'
    rocm = os.environ.get('ROCM_PATH', '/opt/rocm')
    cmd = ['g++', '-std=c++17', '-O2', '-Wall', '-Wno-unused', '-fPIC', '-shared', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1',
           f'-D_GLIBCXX_USE_CXX11_ABI={int(th.compiled_with_cxx11_abi())}', '-I', os.path.join(os.path.dirname(_HERE), 'include'),
           '-isystem', os.path.join(root, 'include'), '-isystem', os.path.join(root, 'include', 'torch', 'csrc', 'api', 'include'),
           '-isystem', os.path.join(rocm, 'include'), os.path.join(_CSRC, 'frnn_ops.cpp'), '-o', tmp, '-L', os.path.join(root, 'lib'),
           '-lc10', '-ltorch_cpu', '-ltorch', '-lc10_hip', '-L', _HERE, '-lfrnn_rt', '-Wl,-rpath,$ORIGIN']
    if verbose:
        print(' '.join(cmd))
    subprocess.run(cmd, check=True)
    os.replace(tmp, OPS_PATH)
    for old in glob.glob(os.path.join(_HERE, 'libfrnn_ops*.so')):
        if old != OPS_PATH:
            with contextlib.suppress(FileNotFoundError):         # (another process builds, too)
                os.remove(old)
    return OPS_PATH


def load() -> ctypes.CDLL:
    """Registers the operators with PyTorch (once)."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                how = 'Run `python -c "import __graft_entry__ as g; g.build()"`.'
                if not os.path.isfile(OPS_PATH):
                    raise runtime.RuntimeError_(f'{OPS_PATH} is missing: the operators have not been built from these sources. {how}')
                try:
                    runtime.lib()                   # (the kernels' runtime, which the operators link against)
                    th.ops.load_library(OPS_PATH)
                    lib = ctypes.CDLL(OPS_PATH)
                    lib.frnn_ops_set_loader.argtypes = [_LOADER]
                    lib.frnn_ops_set_loader.restype = None
                    lib.frnn_ops_set_loader(_loader)
                except (OSError, AttributeError) as e:
                    raise runtime.RuntimeError_(f'{OPS_PATH} cannot be loaded ({e}). {how}') from e
                _lib = lib
    return _lib


def load_if_built():
    """At import: traced and compiled code finds the operators registered.  Without the library, or with one that cannot be loaded,
    the rest of the package works, and the first call says what to do."""
    if os.path.isfile(OPS_PATH) and os.path.isfile(runtime.LIB_PATH):
        try:
            load()
        except runtime.RuntimeError_:
            pass


def op(name: str):
    load()
    return getattr(th.ops.flex_rnn, name).default


# ------------------------------------------------------------------ host-side rules, as the operators apply them
def segments(groups: int, blocks: int) -> Tuple[int, int]:
    """(segments, blocks per segment) of a walk over `blocks` blocks by `groups` workgroups."""
    out = (ctypes.c_int64 * 2)()
    load().frnn_ops_segments(ctypes.c_int64(groups), ctypes.c_int64(blocks), out)
    return out[0], out[1]


def blocks_between_borders(B: int, T: int, H: int, M: int, N: int, shared: bool) -> int:
    f = load().frnn_ops_every
    f.restype = ctypes.c_int64
    return 1 << f(*(ctypes.c_int64(x) for x in (B, T, H, M, N, shared)))


def norm_shape(rows: int, heads: int, C: int, size: int) -> Dict[str, int]:
    out = (ctypes.c_int64 * 5)()
    load().frnn_ops_norm_shape(ctypes.c_int64(rows), ctypes.c_int64(heads), ctypes.c_int64(C), ctypes.c_int64(size), out)
    return dict(zip(('wide', 'threads', 'pieces', 'lanes', 'teams'), out))
