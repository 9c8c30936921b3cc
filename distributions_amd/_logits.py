"""Host side of the categorical given by logits: shapes, dtypes and strides of the arguments, then one call into the C-ABI
(csrc/m355_logits.hip)."""

from __future__ import annotations

import ctypes
import struct
from math import prod

import numpy as np

from . import _lib
from ._dispatch import _device_of
from ._dispatch import _torch as _check_torch
from ._lib import BF16, F16, F32, F64, I32, I64, LogitAdjust, Operand

_L = _torch_module = None
_codes = None  # torch dtype -> code of the types logits may have
_x_codes = None  # ... observations may have
_row_codes = None  # ... arguments per row may have
_vp, _i32, _i64, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
MASK_NONE, MASK_BYTES, MASK_BITS = 0, 1, 2
_ONE, _ZERO = (0, 1.0, 1, 1, F64, 0), (0, 0.0, 1, 1, F64, 0)  # scalar operands
# Calls of a few microseconds on the GPU come one after the other here, so the C structs are packed in one go: filling them
# field by field took longer than the kernels.
_OPERAND = "Qdqqii"
_pack_operand = struct.Struct("=" + _OPERAND).pack
_pack_adjust = struct.Struct("=QqqQQQqQqiiii" + 4 * _OPERAND).pack
assert struct.calcsize("=" + _OPERAND) == ctypes.sizeof(Operand)
assert struct.calcsize("=QqqQQQqQqiiii" + 4 * _OPERAND) == ctypes.sizeof(LogitAdjust)


def _bind():
    """(torch, library), the argument types declared; raises without a GPU or the library."""
    global _L, _torch_module, _codes, _x_codes, _row_codes
    if _L is None:
        torch = _check_torch()
        L = _lib.lib()
        bp = ctypes.c_char_p  # a packed struct
        L.m355_logits_adjust.restype = _i32
        L.m355_logits_adjust.argtypes = [_i64, _i64, _i32, _vp, _i64, bp, _vp, _i64, _vp]
        L.m355_logits_adjust_grad_workspace_bytes.restype = _sz
        L.m355_logits_adjust_grad_workspace_bytes.argtypes = [_i64, _i64, _i32]
        L.m355_logits_adjust_grad.restype = _i32
        L.m355_logits_adjust_grad.argtypes = [_i64, _i64, _i32, _vp, _i64, _vp, _i64, bp, _vp, _vp, _vp, _sz, _vp]
        L.m355_logits_workspace_bytes.restype = _sz
        L.m355_logits_workspace_bytes.argtypes = [_i64, _i64, _i32]
        L.m355_logits_logpdf.restype = _i32
        L.m355_logits_logpdf.argtypes = [_i64, _i64, _i32, _vp, _i64, _vp, _i32, _vp, _vp]
        L.m355_logits_sum_logpdf_grad.restype = _i32
        L.m355_logits_sum_logpdf_grad.argtypes = [_i64, _i64, _i32, _vp, _i64, _vp, _i32, bp, _vp, _vp, _i64, _vp, _sz, _vp]
        _codes = {torch.float64: F64, torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
        _row_codes = {torch.float64: F64, torch.float32: F32}
        _x_codes = {torch.int64: I64, torch.int32: I32, torch.float64: F64, torch.float32: F32}
        _torch_module, _L = torch, L
    return _torch_module, _L


def _stream(torch, device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _device(logits, args, torch):
    """The logits' device if they are on a GPU, else that of the first argument that is."""
    return logits.device if isinstance(logits, torch.Tensor) and logits.is_cuda else _device_of(args, torch)


def _tensor(a, torch, device):
    """A CUDA tensor of `a`'s own dtype (Python numbers and lists: what NumPy makes of them)."""
    if isinstance(a, torch.Tensor):
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


def _any_tensor(torch, first, *more):
    return isinstance(first, torch.Tensor) or any(isinstance(a, torch.Tensor) for a in more)


def _is_number(a):
    return type(a) is float or type(a) is int or (isinstance(a, (float, int, np.floating, np.integer)) and not isinstance(a, bool))


def _row_operand(a, batch, torch, device, keep, what, positive=False):
    """The fields of an Operand from a per-row argument: a number, or an array that broadcasts to the rows' shape."""
    if isinstance(a, torch.Tensor):
        code = _row_codes.get(a.dtype)
        if code is not None and a.shape == batch and a.is_contiguous() and a.device == device:  # nothing to convert
            keep.append(a)
            return a.data_ptr(), 0.0, 1, a.numel() or 1, code, 0
    elif _is_number(a):
        if positive and not a > 0:
            raise ValueError(f"{what} must be positive, got {a}")
        return 0, float(a), 1, 1, F64, 0
    t = _tensor(a, torch, device)
    if t.dtype not in _row_codes:
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
    return t.data_ptr(), 0.0, 1, t.numel() or 1, _row_codes[t.dtype], 0


def _row_ints(a, batch, torch, device, keep, what):
    """Pointer to int64 values, one per row, or 0."""
    if a is None:
        return 0
    t = _tensor(a, torch, device)
    if t.dtype is torch.int64 and t.shape == batch and t.is_contiguous():
        keep.append(t)
        return t.data_ptr()
    if t.dtype is not torch.int64:
        if t.is_floating_point() or t.is_complex() or t.dtype is torch.bool:
            raise TypeError(f"{what}: integers, got {t.dtype}")
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
    lead = t.shape[:-1]
    if prod(lead) == 1:
        t = t.reshape(width).contiguous()
        keep.append(t)
        return t, 0
    if lead != batch:
        try:
            t = t.expand(tuple(batch) + (width,))
        except RuntimeError:
            raise ValueError(f"{what} of shape {tuple(t.shape)} does not broadcast to the rows' shape {tuple(batch)}") from None
    t, stride = _rows(t)
    keep.append(t)
    return t, stride


def _partly(bias, shared, batch):
    """Whether a bias is shared along some of the rows' axes: its gradient comes per element and is summed by _sum_to."""
    return not shared and bias.shape[:-1] != batch


def _adjustment(batch, k, dtype, torch, device, history, lengths, prompt_lengths, repetition, presence, frequency, bias,
                temperature, mask, grad=False):
    """The C struct of an adjustment (packed; grad: of its gradient), the tensors it points to, the bias as given (tensor or
    None) and whether all rows share it."""
    keep, shared = [], False
    temp = _row_operand(temperature, batch, torch, device, keep, "temperature", positive=True)
    hist = hist_len = hist_stride = hist_code = lens = prompts = 0
    if history is None:
        if lengths is not None or prompt_lengths is not None:
            raise ValueError("lengths and prompt_lengths belong to a history")
        for what, a, neutral in (("repetition", repetition, 1.0), ("presence", presence, 0.0), ("frequency", frequency, 0.0)):
            if a is not neutral and not (_is_number(a) and a == neutral):
                raise ValueError(f"{what} needs a history")
        rep, pres, freq = _ONE, _ZERO, _ZERO
    else:
        rep = _row_operand(repetition, batch, torch, device, keep, "repetition", positive=True)
        pres = _row_operand(presence, batch, torch, device, keep, "presence")
        freq = _row_operand(frequency, batch, torch, device, keep, "frequency")
        h = _tensor(history, torch, device)
        if h.dtype is not torch.int64 and h.dtype is not torch.int32:
            if h.is_floating_point() or h.is_complex() or h.dtype is torch.bool:
                raise TypeError(f"history: integer ids, got {h.dtype}")
            h = h.to(torch.int64)
        if h.dim() < 1:
            raise ValueError("history: shape (..., n)")
        hist_len = h.shape[-1]
        if hist_len >= 1 << 31:
            raise ValueError("history: fewer than 2**31 ids per row")
        h, hist_stride = _wide_rows(h, batch, hist_len, keep, "history")
        hist, hist_code = h.data_ptr(), I64 if h.dtype is torch.int64 else I32
        lens = _row_ints(lengths, batch, torch, device, keep, "lengths")
        prompts = _row_ints(prompt_lengths, batch, torch, device, keep, "prompt_lengths")
    given = None
    bias_ptr = bias_stride = bias_code = 0
    if bias is not None:
        given = b = _tensor(bias, torch, device)
        if b.dtype is not dtype and not (b.dtype is torch.float32 and dtype is not torch.float64):
            given = b = b.to(torch.float64 if dtype is torch.float64 else torch.float32)
        b, bias_stride = _wide_rows(b, batch, k, keep, "bias")
        shared = prod(given.shape[:-1]) == 1
        if grad and not shared:  # an expanded view has stride 0 too, but a gradient per row; the values are not read there
            bias_stride = k
        bias_ptr, bias_code = b.data_ptr(), _codes[b.dtype]
        if grad and _partly(given, shared, batch):  # what is summed afterwards is not rounded to 16 bits before
            bias_code = _codes[_value_dtype(dtype, torch)]
    mask_ptr = mask_stride = mask_kind = 0
    if mask is not None:
        m = _tensor(mask, torch, device)
        if m.dtype is torch.bool:
            mask_kind, width = MASK_BYTES, k
        elif m.dtype is torch.int32:
            mask_kind, width = MASK_BITS, (k + 31) // 32
        else:
            raise TypeError(f"mask: bool (one per category) or int32 (32 categories a word), got {m.dtype}")
        m, mask_stride = _wide_rows(m, batch, width, keep, "mask")
        mask_ptr = m.data_ptr()
    packed = _pack_adjust(hist, hist_len, hist_stride, lens, prompts, bias_ptr, bias_stride, mask_ptr, mask_stride, hist_code,
                          bias_code, mask_kind, 0, *rep, *pres, *freq, *temp)
    return packed, keep, given, shared


def _span(t):
    """First and past-the-last byte of a tensor's memory."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _out_rows(out, z, inputs, torch):
    """Checks a caller's output for logits `z` (2-d rows, their stride): returns its rows and stride."""
    if not isinstance(out, torch.Tensor) or out.dtype != z.dtype or out.device != z.device:
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


class _Here:
    """No switch of devices: a context that does nothing."""

    def __enter__(self):
        pass

    def __exit__(self, *a):
        pass


_here = _Here()


def _on(torch, device):
    """The device as HIP's current one for the launch; no switch where it is already."""
    return _here if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def adjust(logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias, temperature, mask, out):
    torch, L = _bind()
    args = (logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias, temperature, mask)
    device = _device(logits, args, torch)
    with _on(torch, device):
        t = _logits(logits, torch, device)
        shape = t.shape
        k = shape[-1]
        z, stride = _rows(t)
        d, keep, _, _ = _adjustment(shape[:-1], k, z.dtype, torch, device, history, lengths, prompt_lengths, repetition, presence,
                                    frequency, bias, temperature, mask)
        if out is None:
            res = torch.empty(shape, dtype=z.dtype, device=device)
            o, ostride = res, k
        else:
            res = out
            o, ostride = _out_rows(out, z, [t] + keep, torch)
        if z.shape[0]:
            _lib.check(L.m355_logits_adjust(z.shape[0], k, _codes[z.dtype], z.data_ptr(), stride, d, o.data_ptr(), ostride,
                                            _stream(torch, device)))
        if out is not None:
            torch.autograd.graph.increment_version(out)  # autograd sees a write to what it may have saved
        del keep
    return res if out is not None or _any_tensor(torch, *args) else res.cpu().numpy()


def adjust_grad(g, logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias, temperature, mask):
    torch, L = _bind()
    args = (g, logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias, temperature, mask)
    device = _device(logits, args, torch)
    with _on(torch, device):
        t = _logits(logits, torch, device)
        shape = t.shape
        k = shape[-1]
        z, stride = _rows(t)
        gt = _tensor(g, torch, device)
        if gt.shape != shape:
            raise ValueError(f"g has shape {tuple(gt.shape)}, the logits {tuple(shape)}")
        gz, gstride = _rows(gt.to(z.dtype))
        d, keep, b, shared = _adjustment(shape[:-1], k, z.dtype, torch, device, history, lengths, prompt_lengths, repetition,
                                         presence, frequency, bias, temperature, mask, grad=True)
        rows, code = z.shape[0], _codes[z.dtype]
        dz = torch.empty(shape, dtype=z.dtype, device=device)
        db, ws, need = None, None, 0
        if b is not None:
            partly = _partly(b, shared, shape[:-1])
            db = torch.empty(k if shared else shape, dtype=_value_dtype(z.dtype, torch) if partly else b.dtype, device=device)
            if shared:
                need = L.m355_logits_adjust_grad_workspace_bytes(rows, k, code)
                ws = torch.empty(need, dtype=torch.uint8, device=device)
                if not rows:
                    db.zero_()
        if rows:
            _lib.check(L.m355_logits_adjust_grad(rows, k, code, gz.data_ptr(), gstride, z.data_ptr(), stride, d, dz.data_ptr(),
                                                 None if db is None else db.data_ptr(), None if ws is None else ws.data_ptr(),
                                                 need, _stream(torch, device)))
        if b is not None:
            back = b.dtype
            if b is not bias and getattr(bias, "dtype", None) is not None:  # it was converted: back to its own type
                back = _float_type(bias, back, torch)
            db = _sum_to(db, b.shape).to(back) if partly else db.reshape(b.shape).to(back)
        del keep
    if _any_tensor(torch, logits, *args):
        return dz, db
    return dz.cpu().numpy(), None if db is None else db.cpu().numpy()


def _float_type(a, otherwise, torch):
    """The torch dtype of an array that holds floats of a type the kernels know, else `otherwise`."""
    dt = a.dtype if isinstance(a, torch.Tensor) else {"float64": torch.float64, "float32": torch.float32,
                                                      "float16": torch.float16}.get(str(a.dtype))
    return dt if dt in _codes else otherwise


def _sum_to(t, shape):
    """The gradient of an operand that was broadcast along some of the rows' axes only: summed along those by halves, in
    float64 and a fixed order.  (Additions of slices: a library sum over many blocks clears memory in a way that a captured
    graph does not repeat.)"""
    lead = t.dim() - len(shape)
    axes = tuple(range(lead)) + tuple(lead + i for i, n in enumerate(shape) if n == 1 and t.shape[lead + i] != 1)
    for axis in axes:
        if t.shape[axis] == 0:
            t = t.new_zeros([1 if i == axis else n for i, n in enumerate(t.shape)])
        while t.shape[axis] > 1:
            n = t.shape[axis]
            half = (n + 1) // 2
            low, high = t.narrow(axis, 0, half), t.narrow(axis, half, n - half)
            t = low.to(_torch_module.float64, copy=True)
            t.narrow(axis, 0, n - half).add_(high)
    return t.reshape(shape)


def _observations(x, batch, torch, device):
    t = _tensor(x, torch, device)
    code = _x_codes.get(t.dtype)
    if code is not None and t.shape == batch and t.is_contiguous():
        return t, code
    if t.dtype not in _x_codes:
        if t.is_complex():
            raise TypeError("observations are integers or floats")
        t = t.to(torch.float32 if t.is_floating_point() else torch.int64)
    if t.shape != batch:
        try:
            t = t.expand(batch)
        except RuntimeError:
            raise ValueError(f"x of shape {tuple(t.shape)} does not broadcast to the rows' shape {tuple(batch)}") from None
    return t.contiguous(), _x_codes[t.dtype]


def _value_dtype(dtype, torch):
    return torch.float64 if dtype is torch.float64 else torch.float32


def logpdf(x, logits):
    torch, L = _bind()
    device = _device(logits, (x, logits), torch)
    with _on(torch, device):
        t = _logits(logits, torch, device)
        batch, k = t.shape[:-1], t.shape[-1]
        z, stride = _rows(t)
        xt, xcode = _observations(x, batch, torch, device)
        out = torch.empty(batch, dtype=_value_dtype(z.dtype, torch), device=device)
        if z.shape[0]:
            _lib.check(L.m355_logits_logpdf(z.shape[0], k, _codes[z.dtype], z.data_ptr(), stride, xt.data_ptr(), xcode,
                                            out.data_ptr(), _stream(torch, device)))
    return out if isinstance(logits, torch.Tensor) or isinstance(x, torch.Tensor) else out.cpu().numpy()


def sum_logpdf(x, logits, weights, grad, out=None):
    """(total, gradient or None) of sum(weights * logpdf(x, logits))."""
    torch, L = _bind()
    args = (x, logits, weights)
    device = _device(logits, args, torch)
    with _on(torch, device):
        t = _logits(logits, torch, device)
        shape = t.shape
        batch, k = shape[:-1], shape[-1]
        z, stride = _rows(t)
        xt, xcode = _observations(x, batch, torch, device)
        keep = []
        w = _pack_operand(*_row_operand(1.0 if weights is None else weights, batch, torch, device, keep, "weights"))
        total = torch.empty((), dtype=_value_dtype(z.dtype, torch), device=device)
        rows, code = z.shape[0], _codes[z.dtype]
        dz, o, ostride = None, None, 0
        if grad and out is None:
            dz = torch.empty(shape, dtype=z.dtype, device=device)
            o, ostride = dz, k
        elif grad:
            dz = out
            o, ostride = _out_rows(out, z, [t, xt] + keep, torch)
        need = L.m355_logits_workspace_bytes(rows, k, code)
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        _lib.check(L.m355_logits_sum_logpdf_grad(rows, k, code, z.data_ptr(), stride, xt.data_ptr(), xcode, w, total.data_ptr(),
                                                 o.data_ptr() if grad and rows else None, ostride, ws.data_ptr(), need,
                                                 _stream(torch, device)))
        if grad and out is not None:
            torch.autograd.graph.increment_version(out)
        del keep
    if out is not None or _any_tensor(torch, logits, *args):
        return total, dz
    return float(total.item()), None if dz is None else dz.cpu().numpy()
