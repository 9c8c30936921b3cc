"""Host side of the norm over a list of gradients: what of each tensor is one run of memory, then one call into the C-ABI
(csrc/m355_gradnorm.hip)."""

from __future__ import annotations

import ctypes
from array import array

import numpy as np

from . import _lib
from ._dispatch import _torch as _check_torch
from ._lib import BF16, F16, F32, F64, Tensor
from ._logits import _on, _span, _stream

_vp, _i32, _i64, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
_L = _torch_module = _codes = None
assert ctypes.sizeof(Tensor) == 32  # ptr, out, n, (dtype, reserved): four 64-bit words an entry, see _table


def _bind():
    """(torch, library), the argument types declared; raises without a GPU or the library."""
    global _L, _torch_module, _codes
    if _L is None:
        torch = _check_torch()
        L = _lib.lib()
        L.m355_global_norm_workspace_bytes.restype = _sz
        L.m355_global_norm_workspace_bytes.argtypes = [_i64]
        L.m355_global_norm.restype = _i32
        L.m355_global_norm.argtypes = [_i64, _vp, _vp, _vp, _i32, _vp, _sz, _vp]
        L.m355_clip_global_norm.restype = _i32
        L.m355_clip_global_norm.argtypes = [_i64, _vp, ctypes.c_double, _vp, _vp, _i32, _vp, _sz, _vp]
        _codes = {torch.float64: F64, torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
        _torch_module, _L = torch, L
    return _torch_module, _L


def dense(t) -> bool:
    """Whether a tensor's elements are one run of memory without gaps or repeats, in some order."""
    if t.is_contiguous():
        return True
    want = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if s != want:
            return False
        want *= n
    return True


class _List:
    """The tensors of a list, None entries left out, as runs of memory (copies of those that have gaps or repeats)."""

    def __init__(self, grads, torch):
        if isinstance(grads, (torch.Tensor, np.ndarray)):
            raise TypeError("a list of gradients is expected, got one array")
        self.grads = grads = list(grads)
        self.places = range(len(grads))
        plain = {type(g) for g in grads} <= {torch.Tensor}  # tensors only: nothing to sort out
        tensors = grads
        if not plain:
            self.places = [i for i, g in enumerate(grads) if g is not None]
            tensors = [grads[i] for i in self.places]
        devices = {g.device for g in tensors if plain or isinstance(g, torch.Tensor)}
        self.want_torch = bool(devices)
        if len(devices) > 1:
            raise ValueError("gradients on several devices")
        self.device = devices.pop() if devices else torch.device("cuda", torch.cuda.current_device())
        if self.device.type != "cuda":
            raise ValueError("gradients are CUDA tensors (or NumPy arrays)")
        if not plain:
            tensors = [g if isinstance(g, torch.Tensor) else
                       torch.from_numpy(np.array(np.asarray(g), order="C", copy=True)).to(self.device) for g in tensors]
        self.tensors = tensors
        self.dtypes = [g.dtype for g in self.tensors]
        kinds = set(self.dtypes)
        for dt in kinds:
            if dt not in _codes:
                raise TypeError(f"gradients are float64, float32, float16 or bfloat16, got {dt}")
        # float32 only if every array is at most 32 bits wide and there is one: the rule of the elementwise functions
        self.norm_dtype = torch.float32 if kinds and torch.float64 not in kinds else torch.float64
        self.runs = [t if t.is_contiguous() or dense(t) else t.contiguous() for t in self.tensors]

    def table(self, outs=None):
        """The m355_tensor array as words; its address is the caller's to keep alive."""
        words = []
        if outs is None:
            for t, dt in zip(self.runs, self.dtypes):
                words += (t.data_ptr(), 0, t.numel(), _codes[dt])
        else:
            for t, dt, o in zip(self.runs, self.dtypes, outs):
                words += (t.data_ptr(), o.data_ptr(), t.numel(), _codes[dt])
        return array("Q", words)


def global_norm(grads, sumsq_only=False):
    """The norm as a 0-d tensor (NumPy inputs: a float), or with sumsq_only the float64 sum of squares as a tensor."""
    torch, L = _bind()
    ls = _List(grads, torch)
    n = len(ls.runs)
    with _on(torch, ls.device):
        res = torch.empty((), dtype=torch.float64 if sumsq_only else ls.norm_dtype, device=ls.device)
        need = L.m355_global_norm_workspace_bytes(n)
        ws = torch.empty(need, dtype=torch.uint8, device=ls.device)
        table = ls.table()
        _lib.check(L.m355_global_norm(n, table.buffer_info()[0] if n else None, res.data_ptr() if sumsq_only else None,
                                      None if sumsq_only else res.data_ptr(), F32 if res.dtype is torch.float32 else F64,
                                      ws.data_ptr(), need, _stream(torch, ls.device)))
    return res if ls.want_torch or sumsq_only else float(res.item())


def _outputs(ls, out, torch):
    """(the caller's outputs, where the kernel writes: they, or a copy where the elements lie in another order or with gaps)."""
    if len(out) != len(ls.grads):
        raise ValueError(f"out has {len(out)} entries, the list of gradients {len(ls.grads)}")
    given = [out[i] for i in ls.places]
    if not all(isinstance(o, torch.Tensor) for o in given) or {o.device for o in given} - {ls.device}:
        raise ValueError("out: tensors on the gradients' device")
    outs = []
    for t, r, o, dt in zip(ls.tensors, ls.runs, given, ls.dtypes):
        if o is not r:
            if o.dtype is not dt or o.shape != t.shape:
                raise ValueError("out: tensors of the gradients' shapes and dtypes")
            if not (o.is_contiguous() and r.is_contiguous()) and not (o.stride() == r.stride() and dense(o)):
                if any(s == 0 and m > 1 for s, m in zip(o.stride(), o.shape)):
                    raise ValueError("out: elements that share memory")
                o = torch.empty_like(r)
        outs.append(o)
    for i, (o, r) in enumerate(zip(given, outs)):
        if o is not r and o.numel():  # what the library does not see: it checks the runs it is given
            lo, hi = _span(o)
            for j, t in enumerate(ls.tensors):
                for other in (given[j], t):
                    if j != i and other.numel():
                        a, b = _span(other)
                        if a < hi and lo < b:
                            raise ValueError("an output with gaps overlaps or interleaves with another tensor of the list")
    return given, outs


def clip_global_norm(grads, max_norm, out=None, sumsq=None):
    torch, L = _bind()
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    ls = _List(grads, torch)
    n = len(ls.runs)
    with _on(torch, ls.device):
        if out is None:
            given = outs = [torch.empty_like(t) for t in ls.runs]
        else:
            given, outs = _outputs(ls, out, torch)
        norm = torch.empty((), dtype=ls.norm_dtype, device=ls.device)
        need = L.m355_global_norm_workspace_bytes(n)
        ws = torch.empty(need, dtype=torch.uint8, device=ls.device)
        table = ls.table(outs)
        _lib.check(L.m355_clip_global_norm(n, table.buffer_info()[0] if n else None, max_norm,
                                           None if sumsq is None else sumsq.data_ptr(), norm.data_ptr(),
                                           F32 if norm.dtype is torch.float32 else F64, ws.data_ptr(), need,
                                           _stream(torch, ls.device)))
        for o, r in zip(given, outs):
            if o is not r:
                o.detach().copy_(r)
        if out is not None:
            torch.autograd.graph.increment_version(given)  # autograd sees a write to what it may have saved
    res = list(given) if len(given) == len(ls.grads) else [None] * len(ls.grads)
    for i, o in zip(ls.places, given):
        res[i] = o if out is not None or isinstance(ls.grads[i], torch.Tensor) else o.cpu().numpy()
    return norm if ls.want_torch else float(norm.item()), res
