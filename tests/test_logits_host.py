"""CPU tests of the operators on logits and gradient lists: what the C-ABI refuses (before any HIP call), and the host
layer's handling of shapes and strides on CPU tensors."""

import ctypes
import math

import pytest
import torch

import distributions_amd
from distributions_amd import _gradnorm, _logits
from distributions_amd._lib import BF16, F16, F32, F64, I32, I64, LogitAdjust, Operand, Tensor

INVALID, WORKSPACE = -1, -4
P = 4096  # a pointer that is never read: every call here is refused or empty


@pytest.fixture(scope="module")
def L():
    """The library with the argument types the host layer declares; torch stands in for a GPU (nothing is launched here)."""
    patch = pytest.MonkeyPatch()
    for m in (_logits, _gradnorm):
        patch.setattr(m, "_check_torch", lambda: torch)
        for n in ("_L", "_torch_module", "_codes"):
            patch.setattr(m, n, None)
        lib = m._bind()[1]
    yield lib
    patch.undo()


def adjustment(**kw):
    d = LogitAdjust()
    for o, v in ((d.repetition, 1.0), (d.presence, 0.0), (d.frequency, 0.0), (d.temperature, 1.0)):
        o.scalar, o.div, o.mod = v, 1, 1
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def test_adjust_refusals(L):
    def call(rows=4, k=10, dtype=F32, z=P, zs=10, d=None, o=P, os=10):
        return L.m355_logits_adjust(rows, k, dtype, z, zs, bytes(d if d is not None else adjustment()), o, os, None)

    assert call(rows=0) == 0
    for kw in (dict(rows=-1), dict(k=0), dict(k=1 << 31), dict(dtype=I64), dict(dtype=9), dict(z=None), dict(o=None), dict(zs=-1),
               dict(os=9), dict(d=adjustment(history=P, history_len=-1, history_dtype=I64)),
               dict(d=adjustment(history=P, history_len=1 << 31, history_dtype=I64)),
               dict(d=adjustment(history=P, history_len=4, history_dtype=F32)), dict(d=adjustment(bias=P, bias_dtype=F64)),
               dict(d=adjustment(bias=P, bias_dtype=F32), dtype=F64), dict(d=adjustment(bias=P, bias_dtype=BF16), dtype=F16),
               dict(d=adjustment(bias=P, bias_dtype=F32, bias_stride=-1)), dict(d=adjustment(mask_kind=1)), dict(d=adjustment(mask_kind=3, mask=P)),
               dict(d=adjustment(temperature=Operand(P, 0.0, 1, 4, I64, 0))), dict(d=adjustment(temperature=Operand(P, 0.0, 0, 4, F64, 0)))):
        assert call(**kw) == INVALID, kw
        assert L.m355_last_error()
    assert L.m355_logits_adjust(4, 10, F32, P, 10, None, P, 10, None) == INVALID


def test_adjust_grad_refusals(L):
    def call(rows=4, k=10, dtype=F32, g=P, z=P, d=None, dz=P, db=None, ws=P, wsb=1 << 20):
        return L.m355_logits_adjust_grad(rows, k, dtype, g, 10, z, 10, bytes(d if d is not None else adjustment()), dz, db, ws, wsb, None)

    shared = adjustment(bias=P, bias_dtype=F32)
    need = L.m355_logits_adjust_grad_workspace_bytes(4, 10, F32)
    assert need >= 80
    assert call(rows=0) == 0
    assert call(db=P) == INVALID  # no bias
    assert call(g=None) == INVALID
    assert call(z=None, d=adjustment(history=P, history_len=2, history_dtype=I32)) == INVALID
    assert call(d=shared, db=P, wsb=need - 1) == WORKSPACE and call(d=shared, db=P, ws=None) == WORKSPACE


def test_density_refusals(L):
    one = Operand(None, 1.0, 1, 1, F64, 0)

    def value(rows=4, k=10, dtype=F32, z=P, x=P, xd=I64, o=P, zs=10):
        return L.m355_logits_logpdf(rows, k, dtype, z, zs, x, xd, o, None)

    assert value(rows=0) == 0
    for kw in (dict(rows=-1), dict(k=0), dict(k=1 << 31), dict(dtype=I32), dict(z=None), dict(x=None), dict(xd=BF16), dict(o=None), dict(zs=-1)):
        assert value(**kw) == INVALID, kw
    need = L.m355_logits_workspace_bytes(4, 10, F32)

    def grad(rows=4, w=one, t=P, dz=P, ds=10, ws=P, wsb=1 << 20):
        return L.m355_logits_sum_logpdf_grad(rows, 10, F32, P, 10, P, I64, None if w is None else bytes(w), t, dz, ds, ws, wsb, None)

    for kw in (dict(w=None), dict(t=None), dict(ds=9), dict(ws=None), dict(w=Operand(P, 0.0, 1, 4, I64, 0))):
        assert grad(**kw) == INVALID, kw
    assert grad(wsb=need - 1) == WORKSPACE


def table(*rows):
    t = (Tensor * max(len(rows), 1))()
    for e, (ptr, out, n, dt) in zip(t, rows):
        e.ptr, e.out, e.n, e.dtype = ptr, out, n, dt
    return t


def test_norm_and_clip_refusals(L):
    ws = 1 << 20

    def clip(rows, max_norm=1.0, wsp=P, wsb=ws, dt=F32, count=None):
        return L.m355_clip_global_norm(len(rows) if count is None else count, table(*rows), max_norm, None, P, dt, wsp, wsb, None)

    a = 1 << 20
    assert L.m355_global_norm(-1, table(), None, P, F32, P, ws, None) == INVALID
    for rows in ([(a, a, 10, I64)], [(a, a, -1, F32)], [(None, a, 10, F32)], [(a, None, 10, F32)]):
        assert clip(rows) == INVALID, rows
    # outputs that overlap: the same tensor twice, shifted by one element, an input of another, one inside another
    for rows in ([(a, a, 10, F32), (a, a, 10, F32)], [(a, a + 4, 10, F32)], [(a, 2 * a, 10, F32), (3 * a, a + 36, 10, F32)],
                 [(a, 2 * a, 100, F64), (3 * a, 2 * a + 8, 2, BF16)], [(a, 2 * a, 10, F32), (2 * a, 3 * a, 10, F32)]):
        assert clip(rows) == INVALID and b"overlap" in L.m355_last_error(), rows
    good = [(a, a, 10, F32)]
    for kw in (dict(max_norm=-1.0), dict(max_norm=math.nan), dict(dt=BF16), dict(wsp=None)):
        assert clip(good, **kw) == INVALID, kw
    need = L.m355_global_norm_workspace_bytes(1)
    assert clip(good, wsb=need - 1) == WORKSPACE
    assert L.m355_global_norm(1, table(*good), None, P, F32, P, need - 1, None) == WORKSPACE
    assert L.m355_global_norm_workspace_bytes(1000) > L.m355_global_norm_workspace_bytes(1)


def test_rows_and_layouts():
    t = torch.zeros(3, 4, 10)
    r, s = _logits._rows(t[:, -1])
    assert r.shape == (3, 10) and s == 40 and r.data_ptr() == t[:, -1].data_ptr()
    r, s = _logits._rows(t)
    assert r.shape == (12, 10) and s == 10
    r, s = _logits._rows(t.transpose(1, 2))
    assert r.shape == (30, 4) and s == 4
    r, s = _logits._rows(t[0, 0])
    assert r.shape == (1, 10)
    r, s = _logits._rows(torch.zeros(10).expand(5, 10))
    assert s == 0
    assert _gradnorm.dense(torch.zeros(3, 4).t()) and _gradnorm.dense(torch.zeros(2, 3, 4).permute(2, 0, 1))
    assert not _gradnorm.dense(torch.zeros(3, 4)[:, :3]) and not _gradnorm.dense(torch.zeros(3, 1).expand(3, 4))
    assert _gradnorm.dense(torch.zeros(0, 4)) and _gradnorm.dense(torch.zeros(()))


def test_expanded_bias_is_not_shared(L):
    """Whether rows share a bias is a matter of its shape: an expanded view has row stride 0 and a gradient per row."""
    codes = dict(zip((torch.float64, torch.float32, torch.float16, torch.bfloat16), (F64, F32, F16, BF16)))
    one = torch.zeros(10)
    for batch, bias, shared in (((4,), one.expand(4, 10), False), ((2, 7), one.expand(2, 1, 10), False), ((2, 7), one.expand(7, 10), False),
                                ((2, 7), one.expand(2, 7, 10), False), ((4,), one, True), ((4,), one[None], True),
                                ((2, 7), one[None, None], True), ((1,), one.expand(1, 10), True)):
        assert _logits._codes == codes
        for grad in (False, True):
            packed, keep, given, got = _logits._adjustment(batch, 10, torch.float32, torch, torch.device("cpu"), None, None, None, 1.0, 0.0,
                                                           0.0, bias, 1.0, None, grad=grad)
            stride = LogitAdjust.from_buffer_copy(packed).bias_stride
            assert given is bias and got is shared and (stride != 0) == (grad and not shared), (batch, bias.shape, grad)


def test_sharded_clip_adds_the_ranks(monkeypatch):
    """The sum of squares of this rank is what is all-reduced, and the reduced one is what scales."""
    from distributions_amd import sharded

    seen = {}
    monkeypatch.setattr(_gradnorm, "global_norm", lambda g, sumsq_only=False: torch.tensor(9.0, dtype=torch.float64))
    monkeypatch.setattr(sharded, "allreduce_sum_", lambda t, group=None: t.add_(16.0))
    monkeypatch.setattr(_gradnorm, "clip_global_norm", lambda g, m, out, sumsq: seen.update(m=m, sumsq=float(sumsq)) or (5.0, g))
    assert sharded.clip_global_norm(["g"], 2.0) == (5.0, ["g"]) and seen == {"m": 2.0, "sumsq": 25.0}
