"""Host side of the norm over a list of gradients: what of each tensor is one run of memory, then one call into the C-ABI
(csrc/m355_gradnorm.hip)."""

from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from ._dispatch import _is_torch, _torch
from ._lib import BF16, F16, F32, F64, Tensor
from ._logits import _on

_vp, _i32, _i64, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
_codes = None
_bound = False


def _bind():
    global _bound, _codes
    L = _lib.lib()
    if not _bound:
        import torch

        tp = ctypes.POINTER(Tensor)
        L.m355_global_norm_workspace_bytes.restype = _sz
        L.m355_global_norm_workspace_bytes.argtypes = [_i64]
        L.m355_global_norm.restype = _i32
        L.m355_global_norm.argtypes = [_i64, tp, _vp, _vp, _i32, _vp, _sz, _vp]
        L.m355_clip_global_norm.restype = _i32
        L.m355_clip_global_norm.argtypes = [_i64, tp, ctypes.c_double, _vp, _vp, _i32, _vp, _sz, _vp]
        _codes = {torch.float64: F64, torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
        _bound = True
    return L


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
    """The tensors of a list (None entries left out) and the table the library reads."""

    def __init__(self, grads, torch):
        if _is_torch(grads) or isinstance(grads, np.ndarray):
            raise TypeError("a list of gradients is expected, got one array")
        self.grads = list(grads)
        self.want_torch = False
        device, tensors, places, small = None, [], [], True
        for i, g in enumerate(self.grads):
            if g is None:
                continue
            if _is_torch(g):
                self.want_torch = True
                if not g.is_cuda:
                    raise ValueError("gradients are CUDA tensors (or NumPy arrays)")
                if device is None:
                    device = g.device
                elif g.device != device:
                    raise ValueError("gradients on several devices")
            tensors.append(g)
            places.append(i)
        self.device = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        for j, g in enumerate(tensors):
            if not _is_torch(g):
                g = tensors[j] = torch.from_numpy(np.array(np.asarray(g), order="C", copy=True)).to(self.device)
            dt = g.dtype
            if dt not in _codes:
                raise TypeError(f"gradients are float64, float32, float16 or bfloat16, got {dt}")
            if dt is torch.float64:
                small = False
        self.tensors, self.places = tensors, places
        # float32 only if every array is at most 32 bits wide and there is one: the rule of the elementwise functions
        self.norm_dtype = torch.float32 if small and tensors else torch.float64

    def runs(self):
        """The tensors as runs of memory (copies of those that have gaps or repeats)."""
        return [t if dense(t) else t.contiguous() for t in self.tensors]


def _table(runs, outs=None):
    table = (Tensor * max(len(runs), 1))()
    for i, t in enumerate(runs):
        e = table[i]
        e.ptr, e.n, e.dtype = t.data_ptr(), t.numel(), _codes[t.dtype]
        if outs is not None:
            e.out = outs[i].data_ptr()
    return table


def _workspace(L, n, torch, device):
    need = L.m355_global_norm_workspace_bytes(n)
    return torch.empty(need, dtype=torch.uint8, device=device), need


def global_norm(grads, sumsq_only=False):
    """The norm as a 0-d tensor (NumPy inputs: a float), or with sumsq_only the float64 sum of squares as a tensor."""
    torch = _torch()
    L = _bind()
    ls = _List(grads, torch)
    with _on(torch, ls.device):
        runs = ls.runs()
        res = torch.empty((), dtype=torch.float64 if sumsq_only else ls.norm_dtype, device=ls.device)
        ws, need = _workspace(L, len(runs), torch, ls.device)
        _lib.check(L.m355_global_norm(len(runs), _table(runs), res.data_ptr() if sumsq_only else None,
                                      None if sumsq_only else res.data_ptr(), F32 if res.dtype == torch.float32 else F64,
                                      ws.data_ptr(), need, torch.cuda.current_stream(ls.device).cuda_stream))
    return res if ls.want_torch or sumsq_only else float(res.item())


def clip_global_norm(grads, max_norm, out=None, sumsq=None):
    torch = _torch()
    L = _bind()
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    ls = _List(grads, torch)
    n = len(ls.tensors)
    with _on(torch, ls.device):
        runs = ls.runs()
        if out is None:
            given = outs = [torch.empty_like(t) for t in runs]
        else:
            given = [out[i] for i in ls.places] if len(out) == len(ls.grads) else []
            if len(given) != n:
                raise ValueError(f"out has {len(out)} entries, the list of gradients {len(ls.grads)}")
            outs = []
            for t, r, o in zip(ls.tensors, runs, given):
                if not _is_torch(o) or o.dtype != t.dtype or o.device != t.device or o.shape != t.shape:
                    raise ValueError("out: tensors of the gradients' shapes and dtypes on their device")
                if o.stride() == r.stride() or (o.is_contiguous() and r.is_contiguous()):
                    outs.append(o)
                else:  # another order of elements in memory, or gaps: through a copy
                    if any(s == 0 and m > 1 for s, m in zip(o.stride(), o.shape)):
                        raise ValueError("out: elements that share memory")
                    outs.append(torch.empty_like(r))
        norm = torch.empty((), dtype=ls.norm_dtype, device=ls.device)
        ws, need = _workspace(L, n, torch, ls.device)
        _lib.check(L.m355_clip_global_norm(n, _table(runs, outs), max_norm, None if sumsq is None else sumsq.data_ptr(),
                                           norm.data_ptr(), F32 if norm.dtype == torch.float32 else F64, ws.data_ptr(),
                                           need, torch.cuda.current_stream(ls.device).cuda_stream))
        for o, r in zip(given, outs):
            if o is not r:
                o.detach().copy_(r)
    res = [None] * len(ls.grads)
    for i, o in zip(ls.places, given):
        res[i] = o if _is_torch(ls.grads[i]) or out is not None else o.cpu().numpy()
    return norm if ls.want_torch else float(norm.item()), res
