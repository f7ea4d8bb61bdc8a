"""Hand-written kernels (flex_rnn_amd/csrc/*.hip): compiled per set of preprocessor constants into the same on-disk cache as
the generated ones, loaded once per device, launched through the same C-ABI runtime on the current stream.

`kernel()` finds or builds one; `launch()` packs the argument block and launches; `slice_sum()` is the reduction over
leading slices that the backward passes of `linear.py` and `norm.py` share.
"""
from __future__ import annotations

import contextlib
import os
import struct
import threading
from concurrent.futures import ThreadPoolExecutor
from typing import Dict, Iterable, Tuple

import torch as th

from . import runtime

_CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), 'csrc')
DTYPES = {th.bfloat16: 0, th.float16: 1, th.float32: 2}      # the kernels' type codes

_lock = threading.Lock()
_sources: Dict[str, str] = {}
_kernels: Dict[tuple, runtime.Kernel] = {}


def require(ok, message: str):
    """Argument checks raise what the compiled operators' own checks raise (and also do so under `python -O`)."""
    if not ok:
        raise AssertionError(message)


def build(source: str, name: str, defines: Tuple[Tuple[str, int], ...] = (), force: bool = False) -> str:
    """Path of the code object of kernel `name` from csrc/`source`, compiled with `defines` on a cache miss."""
    with _lock:
        if source not in _sources:
            with open(os.path.join(_CSRC, source)) as f:
                _sources[source] = f.read()
    opts = ' '.join([runtime.EMITTER_OPTS] + [f'-D{k}={v}' for k, v in defines])
    return runtime.compile_kernel(name, _sources[source], opts=opts, force=force)


def build_all(cases: Iterable[tuple], force: bool = False, workers: int = 6) -> int:
    """Compiles `cases` = (source, name, defines), side by side; returns their number."""
    cases = list(cases)
    with ThreadPoolExecutor(max_workers=workers) as pool:
        list(pool.map(lambda c: build(*c, force=force), cases))
    return len(cases)


def kernel(device: th.device, source: str, name: str, defines: Tuple[Tuple[str, int], ...] = ()) -> runtime.Kernel:
    key = (device.index, source, name, defines)
    k = _kernels.get(key)
    if k is None:
        with th.cuda.device(device):
            if th.cuda.is_current_stream_capturing():
                raise runtime.RuntimeError_(f'kernel {name} is not loaded yet and cannot be while a graph is captured: '
                                            'make one call with these types and head sizes before the capture')
            k = runtime.Module(build(source, name, defines)).kernel(name)
        k = _kernels.setdefault(key, k)
    return k


_packers: Dict[str, struct.Struct] = {}


def launch(k: runtime.Kernel, device: th.device, grid: int, threads: int, layout: str, *args):
    """Launches `k` on the current stream of `device`; `layout` names the argument block's 8-byte fields (struct)."""
    p = _packers.get(layout)
    if p is None:
        p = _packers[layout] = struct.Struct('<' + layout)
    launch_bytes(k, device, grid, 1, threads, p.pack(*args))


def launch_bytes(k: runtime.Kernel, device: th.device, grid: int, grid_y: int, threads: int, block: bytes):
    """The same with a packed argument block."""
    if grid <= 0:
        return
    require(grid * threads < 2 ** 32, f'{k.name}: a launch of {grid} workgroups is more than the hardware takes; split the batch')
    with (th.cuda.device(device) if th.cuda.current_device() != device.index else contextlib.nullcontext()):
        k.launch((grid, grid_y, 1), (threads, 1, 1), block, stream=th.cuda.current_stream(device).cuda_stream)


def slice_sum(x: th.Tensor, slices: int, out: th.Tensor):
    """out[...] = the sum of `slices` leading fp32 slices of `x`, in `out`'s type."""
    X = out.numel()
    if X == 0:
        return
    k = kernel(x.device, 'slice_sum.hip', 'slice_sum')
    # columns side by side while there are enough of them to fill a row of threads; else the threads share the slices
    cw = 1
    while cw < 64 and cw < X:
        cw *= 2
    groups = -(-X // cw)
    # many slices over few columns: parts of at least 64 trips per thread row, joined by a second launch
    parts = max(1, min(512 // groups, slices // (64 * (256 // cw))))
    if parts > 1:
        part = th.empty((parts, X), dtype=th.float32, device=x.device)
        launch(k, x.device, groups * parts, 256, '7q', x.data_ptr(), part.data_ptr(), slices, X, 2, cw, parts)
        x, slices = part, parts
    launch(k, x.device, groups, 256, '7q', x.data_ptr(), out.data_ptr(), slices, X, DTYPES[out.dtype], cw, 1)
