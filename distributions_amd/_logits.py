"""Host side of the categorical given by logits: shapes, dtypes and strides of the arguments, then one call into the C-ABI
(csrc/m355_logits.hip)."""

from __future__ import annotations

import ctypes
from math import prod

import numpy as np

from . import _lib
from ._dispatch import _device_of, _is_torch, _shape_of, _torch
from ._lib import BF16, F16, F32, F64, I32, I64, LogitAdjust, Operand

_codes = None  # torch dtype -> code of the types logits may have
_bound = False
_vp, _i32, _i64, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
MASK_NONE, MASK_BYTES, MASK_BITS = 0, 1, 2


def _bind():
    global _bound, _codes
    L = _lib.lib()
    if not _bound:
        import torch

        ap, op = ctypes.POINTER(LogitAdjust), ctypes.POINTER(Operand)
        L.m355_logits_adjust.restype = _i32
        L.m355_logits_adjust.argtypes = [_i64, _i64, _i32, _vp, _i64, ap, _vp, _i64, _vp]
        L.m355_logits_adjust_grad_workspace_bytes.restype = _sz
        L.m355_logits_adjust_grad_workspace_bytes.argtypes = [_i64, _i64, _i32]
        L.m355_logits_adjust_grad.restype = _i32
        L.m355_logits_adjust_grad.argtypes = [_i64, _i64, _i32, _vp, _i64, _vp, _i64, ap, _vp, _vp, _vp, _sz, _vp]
        L.m355_logits_workspace_bytes.restype = _sz
        L.m355_logits_workspace_bytes.argtypes = [_i64, _i64, _i32]
        L.m355_logits_logpdf.restype = _i32
        L.m355_logits_logpdf.argtypes = [_i64, _i64, _i32, _vp, _i64, _vp, _i32, _vp, _vp, _sz, _vp]
        L.m355_logits_sum_logpdf_grad.restype = _i32
        L.m355_logits_sum_logpdf_grad.argtypes = [_i64, _i64, _i32, _vp, _i64, _vp, _i32, op, _vp, _vp, _i64, _vp, _sz, _vp]
        _codes = {torch.float64: F64, torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
        _bound = True
    return L


def _tensor(a, torch, device):
    """A CUDA tensor of `a`'s own dtype (Python numbers and lists: what NumPy makes of them)."""
    if _is_torch(a):
        return a if a.device == device else a.to(device)
    return torch.from_numpy(np.array(np.asarray(a), order="C", copy=True)).to(device)


def _logits(a, torch, device, what="logits"):
    """Logits as a CUDA tensor of a type the kernels take; integers become float64."""
    t = _tensor(a, torch, device)
    if t.dtype not in _codes:
        if t.is_floating_point() or t.is_complex():
            raise TypeError(f"{what}: float64, float32, float16 or bfloat16, got {t.dtype}")
        t = t.to(torch.float64)
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{what}: shape (..., k) with k >= 1, got {tuple(t.shape)}")
    return t


def _rows(t):
    """(tensor, row stride) of a tensor (..., k) as rows of k contiguous elements; copied only where no view does."""
    if t.dim() == 1:
        t = t.unsqueeze(0)
    elif t.dim() > 2:
        t = t.flatten(0, -2)
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _is_number(a):
    return isinstance(a, (float, int, np.floating, np.integer)) and not isinstance(a, bool)


def _row_operand(o, a, batch, torch, device, keep, what, positive=False):
    """Fill Operand `o` with a per-row argument: a number, or an array that broadcasts to the rows' shape."""
    o.div = o.mod = 1
    o.reserved = 0
    if _is_number(a):
        if positive and not a > 0:
            raise ValueError(f"{what} must be positive, got {a}")
        o.ptr, o.scalar, o.dtype = None, float(a), F64
        return
    t = _tensor(a, torch, device)
    if t.dtype not in (torch.float64, torch.float32):
        t = t.to(torch.float64)
    if t.shape != batch:
        try:
            whole = np.broadcast_shapes(tuple(t.shape), tuple(batch)) == tuple(batch)
        except ValueError:
            whole = False
        if not whole:
            raise ValueError(f"{what} of shape {tuple(t.shape)} does not broadcast to the rows' shape {tuple(batch)}")
        if t.numel() != 1:
            t = t.expand(batch)
    t = t.contiguous()
    keep.append(t)
    o.ptr, o.scalar, o.dtype, o.mod = t.data_ptr(), 0.0, F64 if t.dtype == torch.float64 else F32, max(t.numel(), 1)


def _row_ints(a, batch, torch, device, keep, what):
    """Pointer to int64 values, one per row, or None."""
    if a is None:
        return None
    t = _tensor(a, torch, device)
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise TypeError(f"{what}: integers, got {t.dtype}")
    if t.dtype != torch.int64:
        t = t.to(torch.int64)
    if t.shape != batch:
        try:
            t = t.expand(batch)
        except RuntimeError:
            raise ValueError(f"{what} of shape {tuple(t.shape)} does not broadcast to the rows' shape {tuple(batch)}") from None
    t = t.contiguous()
    keep.append(t)
    return t.data_ptr()


def _wide_rows(t, batch, width, keep, what):
    """(pointer, row stride) of an array (width,), (..., width) that broadcasts to the rows' shape; stride 0 where all rows
    share it."""
    if t.dim() < 1 or t.shape[-1] != width:
        raise ValueError(f"{what}: the last axis must have {width} entries, got shape {tuple(t.shape)}")
    if prod(t.shape[:-1]) == 1:
        t = t.reshape(width).contiguous()
        keep.append(t)
        return t, 0
    if t.shape[:-1] != batch:
        try:
            t = t.expand(tuple(batch) + (width,))
        except RuntimeError:
            raise ValueError(f"{what} of shape {tuple(t.shape)} does not broadcast to the rows' shape {tuple(batch)}") from None
    t, stride = _rows(t)
    keep.append(t)
    return t, stride


def _adjustment(batch, k, dtype, torch, device, history, lengths, prompt_lengths, repetition, presence, frequency, bias,
                temperature, mask):
    """The C struct of an adjustment, the tensors it points to, and the bias as given (tensor or None)."""
    keep = []
    d = LogitAdjust()
    _row_operand(d.repetition, repetition, batch, torch, device, keep, "repetition", positive=True)
    _row_operand(d.presence, presence, batch, torch, device, keep, "presence")
    _row_operand(d.frequency, frequency, batch, torch, device, keep, "frequency")
    _row_operand(d.temperature, temperature, batch, torch, device, keep, "temperature", positive=True)
    if history is None:
        if lengths is not None or prompt_lengths is not None:
            raise ValueError("lengths and prompt_lengths belong to a history")
        for what, a, neutral in (("repetition", repetition, 1), ("presence", presence, 0), ("frequency", frequency, 0)):
            if not (_is_number(a) and a == neutral):
                raise ValueError(f"{what} needs a history")
    else:
        h = _tensor(history, torch, device)
        if h.dtype not in (torch.int64, torch.int32):
            if h.is_floating_point() or h.is_complex() or h.dtype == torch.bool:
                raise TypeError(f"history: integer ids, got {h.dtype}")
            h = h.to(torch.int64)
        if h.dim() < 1:
            raise ValueError("history: shape (..., n)")
        if h.shape[-1] >= 1 << 31:
            raise ValueError("history: fewer than 2**31 ids per row")
        h, d.history_stride = _wide_rows(h, batch, h.shape[-1], keep, "history")
        d.history, d.history_len = h.data_ptr(), h.shape[-1]
        d.history_dtype = I64 if h.dtype == torch.int64 else I32
        d.lengths = _row_ints(lengths, batch, torch, device, keep, "lengths")
        d.prompt_lengths = _row_ints(prompt_lengths, batch, torch, device, keep, "prompt_lengths")
    given = None
    if bias is not None:
        given = b = _tensor(bias, torch, device)
        if b.dtype != dtype and not (b.dtype == torch.float32 and dtype != torch.float64):
            given = b = b.to(torch.float64 if dtype == torch.float64 else torch.float32)
        b, d.bias_stride = _wide_rows(b, batch, k, keep, "bias")
        d.bias, d.bias_dtype = b.data_ptr(), _codes[b.dtype]
    if mask is not None:
        m = _tensor(mask, torch, device)
        if m.dtype == torch.bool:
            d.mask_kind, width = MASK_BYTES, k
        elif m.dtype == torch.int32:
            d.mask_kind, width = MASK_BITS, (k + 31) // 32
        else:
            raise TypeError(f"mask: bool (one per category) or int32 (32 categories a word), got {m.dtype}")
        m, d.mask_stride = _wide_rows(m, batch, width, keep, "mask")
        d.mask = m.data_ptr()
    return d, keep, given


def _span(t):
    """First and past-the-last byte of a tensor's memory."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _out_rows(out, z, inputs, torch):
    """Checks a caller's output for logits `z` (2-d rows, their stride): returns its rows and stride."""
    if not _is_torch(out) or out.dtype != z.dtype or out.device != z.device:
        raise ValueError("out: a tensor of the logits' dtype on their device")
    if tuple(out.shape) != tuple(inputs[0].shape):
        raise ValueError(f"out has shape {tuple(out.shape)}, the logits {tuple(inputs[0].shape)}")
    if not out.numel():
        return out.reshape(z.shape), 0
    o = out.unsqueeze(0) if out.dim() == 1 else out
    if o.dim() > 2:
        try:
            o = o.view(-1, o.shape[-1])
        except RuntimeError:
            raise ValueError("out: rows a constant stride apart") from None
    if (o.shape[1] > 1 and o.stride(1) != 1) or (o.shape[0] > 1 and o.stride(0) < o.shape[1]):
        raise ValueError("out: rows of contiguous elements that do not overlap")
    lo, hi = _span(o)
    same = o.data_ptr() == z.data_ptr() and (o.shape[0] == 1 or o.stride(0) == z.stride(0))
    for t in ([] if same else [z]) + list(inputs[1:]):
        if t.numel():
            a, b = _span(t)
            if a < hi and lo < b:
                raise ValueError("out overlaps an input (out may be the logits themselves, in place)")
    return o, o.stride(0)


class _on:
    """The device as HIP's current one for the launch; no switch where it is already."""

    def __init__(self, torch, device):
        self.ctx = None if torch.cuda.current_device() == device.index else torch.cuda.device(device)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *a):
        if self.ctx is not None:
            self.ctx.__exit__(*a)


def adjust(logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias, temperature, mask, out):
    torch = _torch()
    L = _bind()
    args = (logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias, temperature, mask)
    device = _device_of(args, torch)
    want_torch = out is not None or any(_is_torch(a) for a in args)
    with _on(torch, device):
        t = _logits(logits, torch, device)
        batch, k = t.shape[:-1], t.shape[-1]
        z, stride = _rows(t)
        d, keep, _ = _adjustment(batch, k, z.dtype, torch, device, history, lengths, prompt_lengths, repetition, presence,
                                 frequency, bias, temperature, mask)
        if out is None:
            res = torch.empty(t.shape, dtype=z.dtype, device=device)
            o, ostride = res, k
        else:
            res = out
            o, ostride = _out_rows(out, z, [t] + keep, torch)
        if z.shape[0]:
            _lib.check(L.m355_logits_adjust(z.shape[0], k, _codes[z.dtype], z.data_ptr(), stride, ctypes.byref(d),
                                            o.data_ptr(), ostride, torch.cuda.current_stream(device).cuda_stream))
        del keep
    return res if want_torch else res.cpu().numpy()


def adjust_grad(g, logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias, temperature, mask):
    torch = _torch()
    L = _bind()
    args = (g, logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias, temperature, mask)
    device = _device_of(args, torch)
    want_torch = any(_is_torch(a) for a in args)
    with _on(torch, device):
        t = _logits(logits, torch, device)
        batch, k = t.shape[:-1], t.shape[-1]
        z, stride = _rows(t)
        gt = _tensor(g, torch, device)
        if gt.shape != t.shape:
            raise ValueError(f"g has shape {tuple(gt.shape)}, the logits {tuple(t.shape)}")
        gz, gstride = _rows(gt.to(z.dtype))
        d, keep, b = _adjustment(batch, k, z.dtype, torch, device, history, lengths, prompt_lengths, repetition, presence,
                                 frequency, bias, temperature, mask)
        rows, code = z.shape[0], _codes[z.dtype]
        dz = torch.empty(t.shape, dtype=z.dtype, device=device)
        db, ws, need = None, None, 0
        if b is not None:
            shared = d.bias_stride == 0
            db = torch.empty(k if shared else t.shape, dtype=b.dtype, device=device)
            if shared:
                need = L.m355_logits_adjust_grad_workspace_bytes(rows, k, code)
                ws = torch.empty(need, dtype=torch.uint8, device=device)
                if not rows:
                    db.zero_()
        if rows:
            _lib.check(L.m355_logits_adjust_grad(rows, k, code, gz.data_ptr(), gstride, z.data_ptr(), stride,
                                                 ctypes.byref(d), dz.data_ptr(), None if db is None else db.data_ptr(),
                                                 None if ws is None else ws.data_ptr(), need,
                                                 torch.cuda.current_stream(device).cuda_stream))
        if b is not None:
            db = db.reshape(b.shape) if d.bias_stride == 0 else _sum_to(db, b.shape)
        del keep
    if want_torch:
        return dz, db
    return dz.cpu().numpy(), None if db is None else db.cpu().numpy()


def _sum_to(t, shape):
    """The gradient of an operand that was broadcast along some of the rows' axes only."""
    if tuple(t.shape) == tuple(shape):
        return t
    lead = t.dim() - len(shape)
    axes = tuple(range(lead)) + tuple(lead + i for i, n in enumerate(shape) if n == 1 and t.shape[lead + i] != 1)
    acc = t.dtype if t.element_size() >= 4 else None
    s = t.sum(dim=axes, keepdim=True) if acc is not None else t.float().sum(dim=axes, keepdim=True).to(t.dtype)
    return s.reshape(shape)


def _observations(x, batch, torch, device):
    t = _tensor(x, torch, device)
    if t.dtype not in (torch.int64, torch.int32, torch.float64, torch.float32):
        if t.is_complex():
            raise TypeError("observations are integers or floats")
        t = t.to(torch.float32 if t.is_floating_point() else torch.int64)
    if t.shape != batch:
        try:
            t = t.expand(batch)
        except RuntimeError:
            raise ValueError(f"x of shape {tuple(t.shape)} does not broadcast to the rows' shape {tuple(batch)}") from None
    code = {torch.int64: I64, torch.int32: I32, torch.float64: F64, torch.float32: F32}[t.dtype]
    return t.contiguous(), code


def _value_dtype(z, torch):
    return torch.float64 if z.dtype == torch.float64 else torch.float32


def logpdf(x, logits):
    torch = _torch()
    L = _bind()
    device = _device_of((x, logits), torch)
    want_torch = _is_torch(x) or _is_torch(logits)
    with _on(torch, device):
        t = _logits(logits, torch, device)
        batch, k = t.shape[:-1], t.shape[-1]
        z, stride = _rows(t)
        xt, xcode = _observations(x, batch, torch, device)
        out = torch.empty(batch, dtype=_value_dtype(z, torch), device=device)
        rows, code = z.shape[0], _codes[z.dtype]
        if rows:
            need = L.m355_logits_workspace_bytes(rows, k, code)
            ws = torch.empty(need, dtype=torch.uint8, device=device)
            _lib.check(L.m355_logits_logpdf(rows, k, code, z.data_ptr(), stride, xt.data_ptr(), xcode, out.data_ptr(),
                                            ws.data_ptr(), need, torch.cuda.current_stream(device).cuda_stream))
    return out if want_torch else out.cpu().numpy()


def sum_logpdf(x, logits, weights, grad, out=None):
    """(total, gradient or None) of sum(weights * logpdf(x, logits))."""
    torch = _torch()
    L = _bind()
    args = (x, logits, weights)
    device = _device_of(args, torch)
    want_torch = out is not None or any(_is_torch(a) for a in args)
    with _on(torch, device):
        t = _logits(logits, torch, device)
        batch, k = t.shape[:-1], t.shape[-1]
        z, stride = _rows(t)
        xt, xcode = _observations(x, batch, torch, device)
        keep = []
        w = Operand()
        _row_operand(w, 1.0 if weights is None else weights, batch, torch, device, keep, "weights")
        total = torch.empty((), dtype=_value_dtype(z, torch), device=device)
        rows, code = z.shape[0], _codes[z.dtype]
        dz, o, ostride = None, None, 0
        if grad and out is None:
            dz = torch.empty(t.shape, dtype=z.dtype, device=device)
            o, ostride = dz, k
        elif grad:
            dz = out
            o, ostride = _out_rows(out, z, [t, xt] + keep, torch)
        need = L.m355_logits_workspace_bytes(rows, k, code)
        ws = torch.empty(max(need, 8), dtype=torch.uint8, device=device)
        _lib.check(L.m355_logits_sum_logpdf_grad(rows, k, code, z.data_ptr(), stride, xt.data_ptr(), xcode,
                                                 ctypes.byref(w), total.data_ptr(),
                                                 o.data_ptr() if grad and rows else None, ostride, ws.data_ptr(),
                                                 max(need, 8), torch.cuda.current_stream(device).cuda_stream))
        del keep
    if want_torch:
        return total, dz
    return float(total.item()), None if dz is None else dz.cpu().numpy()
