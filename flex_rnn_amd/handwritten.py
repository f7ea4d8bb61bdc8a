"""Hand-written kernels (flex_rnn_amd/csrc/*.hip): compiled per set of preprocessor constants into the same on-disk cache as
the generated ones, loaded once per device, launched through the same C-ABI runtime on the current stream.

`kernel()` finds or builds one; `launch()` packs the argument block and launches; `slice_sums()` is the reduction over
leading slices that the backward passes of `linear.py` and `norm.py` share.
"""
from __future__ import annotations

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


class Once(th.autograd.Function):
    """Calls `op(*args)`, the gradient of an operator; a gradient of that is refused (it would silently miss terms)."""

    @staticmethod
    def forward(ctx, op, *args):
        return op(*args)

    @staticmethod
    def backward(ctx, *grads):
        raise AssertionError('linear_attention and layer_norm can be differentiated once')


def once(op, *args):
    return Once.apply(op, *args) if th.is_grad_enabled() else op(*args)


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
    if grid * threads >= 2 ** 32:
        require(False, f'{k.name}: a launch of {grid} workgroups is more than the hardware takes; split the batch')
    index = device.index
    if th.cuda.current_device() != index:
        with th.cuda.device(device):
            k.launch((grid, grid_y, 1), (threads, 1, 1), block, stream=_raw_stream(index))
    else:
        k.launch((grid, grid_y, 1), (threads, 1, 1), block, stream=_raw_stream(index))


def _raw_stream(index: int) -> int:
    return th._C._cuda_getCurrentRawStream(index)


def slice_sums(pairs, slices: int):
    """For one or two `(x, out)` of one size and type: out[...] = the sum of `slices` leading fp32 slices of `x`."""
    out = pairs[0][1] if pairs else None
    if not pairs or out.numel() == 0:
        return
    X, dev = out.numel(), out.device
    k = kernel(dev, 'slice_sum.hip', 'slice_sum')
    # as many columns side by side as leave 256 workgroups (up to a 256-byte row of them); the other threads share the slices
    cw = 1
    while cw < 64 and cw < X and X // (2 * cw) * len(pairs) >= 256:
        cw *= 2
    groups = -(-X // cw)
    # many slices over few columns: parts of at least 16 trips per thread, joined by a second launch
    parts = max(1, min(512 // (groups * len(pairs)), slices // (16 * (256 // cw))))
    ins, outs = [x for x, _ in pairs], [o for _, o in pairs]

    def run(ins, outs, slices, type_, parts):
        ptrs = [t.data_ptr() for t in (ins[0], outs[0], ins[-1], outs[-1])]
        launch_bytes(k, dev, groups * parts, len(pairs), 256, _SUM.pack(*ptrs, slices, X, type_, cw, parts))

    if parts > 1:
        part = th.empty((len(pairs), parts, X), dtype=th.float32, device=dev)
        run(ins, list(part), slices, 2, parts)
        ins, slices = list(part), parts
    run(ins, outs, slices, DTYPES[out.dtype], 1)


_SUM = struct.Struct('<9q')
