"""Categorical given by logits on the GPU: adjustment and its gradient, log-density, weighted sum and its gradient, against
plain float64 implementations.  Tolerances are worst-case bounds counted from the roundings of the formulas: u is half a
step of the arithmetic (2^-24, float64: 2^-53), ut half a step of the storage type."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = math.inf


def steps(dtype):
    """(u, ut, half the smallest subnormal) of a storage type."""
    u = 2.0**-53 if dtype == torch.float64 else 2.0**-24
    info = torch.finfo(dtype)
    return u, info.eps / 2, info.tiny * info.eps / 2


def within(got, ref, bound):
    """|got - ref| <= bound where ref is finite; the same infinities and NaN elsewhere."""
    got, ref = got.detach().cpu().double(), ref.double()
    assert got.shape == ref.shape
    fin = ref.isfinite()
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got[~fin & ~ref.isnan()], ref[~fin & ~ref.isnan()])
    d = (got[fin] - ref[fin]).abs()
    b = bound.expand(ref.shape)[fin] if isinstance(bound, torch.Tensor) else torch.full_like(d, bound)
    assert bool((d <= b).all()), f"worst {float((d / b.clamp(min=1e-300)).max()):.3g} times the bound"


# ------------------------------------------------------------------------------------------------ plain forms
def allowed_of(mask, k, rows):
    if mask is None:
        return torch.ones(rows, k, dtype=torch.bool)
    m = mask.cpu()
    if m.dtype == torch.int32:
        v = torch.arange(k)
        m = (m.long()[..., v // 32] >> (v % 32)) & 1 == 1
    return m.reshape(-1, k).expand(rows, k)


def per_row(a, rows):
    return torch.as_tensor(a, dtype=torch.float64).cpu().reshape(-1).expand(rows)


def counts_of(history, lengths, prompts, rows, k):
    call = torch.zeros(rows, k, dtype=torch.float64)
    cgen = torch.zeros(rows, k, dtype=torch.float64)
    if history is None:
        return call, cgen
    h = history.cpu().long().reshape(-1, history.shape[-1]).expand(rows, -1)
    n = h.shape[1]
    for r in range(rows):
        last = n if lengths is None else max(0, min(n, int(lengths.reshape(-1)[r])))
        first = 0 if prompts is None else int(prompts.reshape(-1)[r])
        for to, ids in ((call, h[r, :last]), (cgen, h[r, max(first, 0) : last])):
            for v in ids.tolist():
                if 0 <= v < k:
                    to[r, v] += 1
    return call, cgen


def plain_adjust(z, history=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None,
                 temperature=1.0, mask=None):
    """(result, bound on the error) in float64."""
    dtype = z.dtype
    u, ut, tiny = steps(dtype)
    k = z.shape[-1]
    x = z.cpu().double().reshape(-1, k)
    rows = x.shape[0]
    call, cgen = counts_of(history, lengths, prompt_lengths, rows, k)
    rep, pres, freq, t = (per_row(a, rows)[:, None] for a in (repetition, presence, frequency, temperature))
    s = torch.where(call > 0, torch.where(x > 0, x / rep, x * rep), x)
    size = s.abs() + freq.abs() * cgen + pres.abs() * (cgen > 0)
    s = s - (freq * cgen + pres * (cgen > 0))
    if bias is not None:
        b = bias.cpu().double().reshape(-1, k).expand(rows, k)
        s = s + b
        size = size + b.abs()
    ok = allowed_of(mask, k, rows)
    ref = torch.where(ok, s / t, -INF)
    # roundings before the last, each at most u times `size` / T: rep, 1 / rep, its product, freq, freq * c, pres, their sum,
    # the difference, the sum with the bias, T, 1 / T, its product: 12
    bound = ut * ref.abs() + 12 * u * size / t.abs() + tiny
    return ref.reshape(z.shape), torch.nan_to_num(bound, nan=0.0, posinf=0.0).reshape(z.shape)


def plain_adjust_grad(g, z, history=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0,
                      bias=None, temperature=1.0, mask=None):
    k = z.shape[-1]
    x, gg = z.cpu().double().reshape(-1, k), g.cpu().double().reshape(-1, k)
    rows = x.shape[0]
    call, _ = counts_of(history, lengths, prompt_lengths, rows, k)
    rep, t = (per_row(a, rows)[:, None] for a in (repetition, temperature))
    ok = allowed_of(mask, k, rows)
    db = torch.where(ok, gg / t, 0.0)
    dz = torch.where(ok & (call > 0), torch.where(x > 0, db / rep, db * rep), db)
    return dz.reshape(z.shape), db


def plain_logpdf(x, z, weights=None):
    """log-densities, total and gradient in float64 with their bounds."""
    dtype = z.dtype
    u, ut, tiny = steps(dtype)
    k = z.shape[-1]
    zz = z.cpu().double().reshape(-1, k)
    rows = zz.shape[0]
    xx = torch.as_tensor(x).cpu().double().reshape(-1).expand(rows)
    w = torch.ones(rows, dtype=torch.float64) if weights is None else torch.as_tensor(weights).cpu().double().reshape(-1).expand(rows)
    m = zz.max(dim=1, keepdim=True).values
    mm = torch.where(m == -INF, 0.0, m)
    e = (zz - mm).exp()
    s = e.sum(dim=1, keepdim=True)
    inside = (xx >= 0) & (xx < k) & (xx == xx.floor())
    xi = torch.where(inside, xx, 0.0).long()[:, None]
    zx = zz.gather(1, xi)
    empty = (s == 0)[:, 0]
    lp = torch.where(inside & ~empty, (zx - mm - s.log())[:, 0], -INF)
    # sum of k terms, one after the other at worst over a 64th of the row, then joined: k / 64 + 24 roundings; 2^t itself off
    # by 2 u (float64 exp: less), and the roundings of z - m, of log2 e and of their product, which move the exponent by less
    # than 3 u |z - m|: weighted by p, 3 u sum(p |z - m|); log: 2 u |log s|; the two differences: u each
    p = torch.where(s > 0, e / s, 0.0)
    spread = torch.nan_to_num((p * (zz - mm).abs()).sum(1), nan=0.0, posinf=0.0)
    off_s = (k / 64 + 24) * u + 4 * u + 4 * u * spread
    finite = lambda t: torch.nan_to_num(t, nan=0.0, posinf=0.0, neginf=0.0).abs()  # noqa: E731
    b_lp = 1.01 * off_s + 2 * u * finite(s.log()[:, 0]) + u * finite((zx - mm)[:, 0]) + 2 * u * finite(lp)
    grad = torch.zeros(rows, k, dtype=torch.float64)
    live = (w != 0) & inside & ~empty
    hot = torch.zeros(rows, k, dtype=torch.float64).scatter_(1, xi, 1.0)
    grad = torch.where(live[:, None], w[:, None] * (hot - p), 0.0)
    d = torch.nan_to_num((zz - mm).abs(), nan=0.0, posinf=0.0)
    rel_p = 4 * u + 4 * u * d + (1.01 * off_s + 4 * u)[:, None]
    floor = 2.0**-125 if dtype != torch.float64 else 2.0**-1000  # where exp is flushed
    b_g = ut * finite(grad) + finite(w)[:, None] * (finite(p) * rel_p + 2 * u * hot + floor) + tiny
    terms = torch.where(w == 0, 0.0, w * lp)
    total = terms.sum()
    b_total = float((finite(w) * b_lp).sum() + 2 * u * finite(terms).sum())
    shape = z.shape[:-1]
    return lp.reshape(shape), b_lp.reshape(shape), total, b_total, grad.reshape(z.shape), b_g.reshape(z.shape)


def make(shape, dtype, seed, device, scale=3.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(device)


# ----------------------------------------------------------------------------------------------------- adjust
SIZES = [(1, 1), (1, 2), (3, 7), (2, 33), (5, 64), (3, 1023), (2, 4097), (2, 8192), (3, 20011)]


def adjust_args(rows, k, seed, device, history=37, mask="bool", bias="shared", wide=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    r = lambda lo, hi: (lo + (hi - lo) * torch.rand(rows, generator=gen, dtype=torch.float64)).to(wide).to(device)  # noqa: E731
    a = dict(temperature=r(0.5, 2.0))
    if history:
        h = torch.randint(-2, max(2, min(k + 2, 50)), (rows, history), generator=gen)
        h[:, ::5] = torch.randint(0, k, h[:, ::5].shape, generator=gen)
        a.update(history=h.to(device), lengths=torch.randint(-1, history + 3, (rows,), generator=gen).to(device),
                 prompt_lengths=torch.randint(0, history + 1, (rows,), generator=gen).to(device) // 2,
                 repetition=r(0.8, 1.5), presence=r(-0.5, 1.0), frequency=r(-0.2, 0.5))
    if bias:
        shape = (k,) if bias == "shared" else (rows, k)
        a["bias"] = torch.randn(*shape, generator=gen, dtype=torch.float64).to(wide).to(device)
    if mask:
        ok = torch.rand(rows, k, generator=gen) < 0.6
        ok[-1] = False  # a row that allows nothing
        if mask == "bits":
            words = (k + 31) // 32
            bits = torch.zeros(rows, words * 32, dtype=torch.int64)
            bits[:, :k] = ok
            w = (bits.reshape(rows, words, 32) << torch.arange(32)).sum(2)
            ok = torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)
        a["mask"] = ok.to(device)
    return a


@pytest.mark.parametrize("rows, k", SIZES)
@pytest.mark.parametrize("dt", DT)
def test_adjust_and_its_gradient(gpu, dt, rows, k):
    from distributions_amd import categorical_logits as cl

    dtype = DT[dt]
    wide = torch.float64 if dt == "f64" else torch.float32
    u, ut, tiny = steps(dtype)
    z, g = make((rows, k), dtype, 1, gpu), make((rows, k), dtype, 2, gpu)
    for i, (mask, bias, history) in enumerate([("bool", "shared", 37), ("bits", "rows", 300), (None, None, 5), ("bits", "shared", 0),
                                               ("bool", None, 0), (None, "rows", 0)]):
        a = adjust_args(rows, k, 10 + i, gpu, history, mask, bias, wide)
        ref, bound = plain_adjust(z, **a)
        out = cl.adjust(z, **a)
        assert out.dtype == dtype
        within(out, ref, bound)
        dz, db = cl.adjust_grad(g, z, **a)
        rz, rb = plain_adjust_grad(g, z, **a)
        # T, 1 / T, its product, rep, 1 / rep, its product: 6 roundings
        within(dz, rz, ut * rz.abs() + 6 * u * rz.abs() + tiny)
        if bias is None:
            assert db is None
        elif bias == "rows":
            within(db, rb, 3 * u * rb.abs() + 2.0**-149)
        else:  # added in float64; the result rounded to float32 (u) again
            within(db, rb.sum(0), 4 * u * rb.abs().sum(0) + 2.0**-149)
    same = [cl.adjust(z, **a) for _ in range(2)] + [cl.adjust_grad(g, z, **a)[1] for _ in range(2)]
    assert torch.equal(same[0], same[1]) and torch.equal(same[2], same[3])


def test_adjust_infinities_nan_and_lowest_values(gpu):
    from distributions_amd import categorical_logits as cl

    for dtype in DT.values():
        low = torch.finfo(dtype).min
        z = torch.tensor([[0.0, -0.0, INF, -INF, math.nan, low, -low, 1.0, -1.0]] * 2, dtype=dtype, device=gpu)
        ok = torch.tensor([[True] * 9, [True, True, False, True, False, True, False, False, True]], device=gpu)
        h = torch.tensor([[0, 1, 2, 3, 5, 8, 8, 9, -1]] * 2, device=gpu)
        a = dict(history=h, repetition=2.0, mask=ok)
        ref, bound = plain_adjust(z, **a)
        ref = ref.to(dtype).double()  # lowest * 2 leaves the type
        out = cl.adjust(z, **a)
        within(out, ref, bound)
        # NaN and infinities of g where nothing is allowed stay out of the gradient
        g = torch.where(ok, torch.ones_like(z), torch.full_like(z, math.nan))
        dz, db = cl.adjust_grad(g, z, bias=torch.zeros(9, dtype=dtype, device=gpu), **a)
        assert bool(dz.isfinite().all()) and bool(db.isfinite().all())
        assert bool((dz[1][~ok[1]] == 0).all())
        # x <= 0 takes the branch of the product: at 0 the slope is `repetition`
        assert float(dz[0, 0]) == 2.0 and float(dz[0, 2]) == 0.5 and float(dz[0, 8]) == 2.0 and float(dz[0, 7]) == 1.0
        lowest = torch.full((9,), low, dtype=dtype, device=gpu)  # a mask spelled as the type's lowest value
        within(cl.adjust(torch.ones(1, 9, dtype=dtype, device=gpu), bias=lowest), torch.full((1, 9), low, dtype=torch.float64), abs(low) * 2.0**-7)


def ends_of_the_range(dt):
    """Positive arguments whose reciprocal, or which themselves, are no normal numbers of the arithmetic, and some that are."""
    if dt == "f64":
        return [1.0, 5e-324, 1e-309, 2.0**-1022 * 0.75, 2.0**-1022, 2.0**1022, 2.0**1022 * 1.5, 1.7e308, 0.7]
    return [1.0, 1e-300, 1e-60, 1.4e-45, 1e-39, 2.0**-126 * 0.75, 2.0**-126, 2.0**126, 2.0**126 * 1.5, 3e38, 1e39, 1e60, 0.7]


def values_for(args, rows, k, dtype, seed):
    """Values of all sizes, zeros and infinities, whose quotients by and products with `args` (one per row) stay off the border
    where the type, or float32 before it, overflows."""
    gen = torch.Generator().manual_seed(seed)
    top, low = math.log2(torch.finfo(dtype).max), math.log2(torch.finfo(dtype).tiny)
    x = torch.exp2(low + (top - 1 - low) * torch.rand(rows, k, generator=gen, dtype=torch.float64))
    x *= torch.sign(torch.randn(rows, k, generator=gen, dtype=torch.float64))
    x = x.to(dtype).double()
    small = torch.rand(rows, k, generator=gen) < 0.5
    x = torch.where(small, torch.randn(rows, k, generator=gen).to(dtype).double(), x)
    for q in (x / args, x * args):
        for edge in (top, 128 if dtype != torch.float64 else top):
            x = torch.where((torch.log2(q.abs()) - edge).abs() < 0.1, 0.0, x)
    x[:, 0], x[:, 1 % k] = 0.0, -0.0
    if k > 4:
        x[:, 2], x[:, 3] = INF, -INF
    return x.to(dtype)


def in_range(ref, dtype):
    """What rounds past the type's largest value (from half a step above it) is infinite."""
    return torch.where(ref.to(dtype).isinf(), torch.sign(ref) * INF, ref)


@pytest.mark.parametrize("k", [3, 101, 5003])
@pytest.mark.parametrize("dt", DT)
def test_arguments_at_the_ends_of_the_range(gpu, dt, k):
    """Temperatures and repetition penalties without a normal reciprocal: 0 / T is 0 and x / T what it is, whatever T > 0."""
    from distributions_amd import categorical_logits as cl

    dtype = DT[dt]
    u, ut, tiny = steps(dtype)
    least = 2.0**-1074 if dt == "f64" else 2.0**-149
    ends = torch.tensor(ends_of_the_range(dt), dtype=torch.float64)
    args = ends.repeat(6)[:, None]
    rows = len(args)
    z, g = values_for(args, rows, k, dtype, 1), values_for(args, rows, k, dtype, 2)
    h = torch.arange(0, k, 2).expand(rows, -1).contiguous()
    seen = torch.zeros(rows, k, dtype=torch.bool)
    seen[:, ::2] = True
    zd, gd = z.double(), g.double()
    # the argument, its reciprocal, the product; a result or, before the reciprocal's factor of at most 2, a power of two taken
    # from the value may be subnormal: half a step times 2 and another half
    bound = lambda ref: (ut + 3 * u) * torch.nan_to_num(ref, posinf=0.0, neginf=0.0).abs() + tiny + 1.5 * least  # noqa: E731
    z, g, t = z.to(gpu), g.to(gpu), args[:, 0].to(gpu)
    by_t = in_range(zd / args, dtype)
    for history in (None, h.to(gpu)):
        within(cl.adjust(z, history=history, temperature=t), by_t, bound(by_t))
        ref = in_range(gd / args, dtype)
        dz, db = cl.adjust_grad(g, z, history=history, temperature=t, bias=torch.zeros_like(z))
        within(dz, ref, bound(ref))
        within(db, ref, bound(ref))
    by_rep = in_range(torch.where(seen, torch.where(zd > 0, zd / args, zd * args), zd), dtype)
    within(cl.adjust(z, history=h.to(gpu), repetition=t), by_rep, bound(by_rep))
    by_rep = in_range(torch.where(seen, torch.where(zd > 0, gd / args, gd * args), gd), dtype)
    within(cl.adjust_grad(g, z, history=h.to(gpu), repetition=t)[0], by_rep, bound(by_rep))
    # one argument for all rows, as a Python number (and as float32 where that holds it)
    for v in ends.tolist():
        ref = in_range(zd / v, dtype)
        ok = ((torch.log2(ref.abs()) - math.log2(torch.finfo(dtype).max)).abs() > 0.1) & ((torch.log2(ref.abs()) - 128).abs() > 0.1) | (ref == INF)
        ref = torch.where(ok | ~ref.isfinite(), ref, 0.0)
        zz = torch.where(ok | ~ref.isfinite(), z.cpu(), torch.zeros_like(z.cpu())).to(gpu)
        within(cl.adjust(zz, temperature=v), ref, bound(ref))


@pytest.mark.parametrize("k", [3, 101, 5003])
@pytest.mark.parametrize("dt", DT)
def test_shared_bias_with_temperatures_at_the_ends_of_the_range(gpu, dt, k):
    """The column sums of the same: few rows of such temperatures among others, with and without a history."""
    from distributions_amd import categorical_logits as cl

    dtype = DT[dt]
    u, ut, tiny = steps(dtype)
    least = 2.0**-1074 if dt == "f64" else 2.0**-149
    ends = torch.tensor(ends_of_the_range(dt), dtype=torch.float64)
    rows = 150
    args = torch.full((rows, 1), 0.7, dtype=torch.float64)
    args[7 : 7 + 11 * len(ends) : 11, 0] = ends
    g = values_for(args, rows, k, dtype, 3)
    g[:, 2:] = g[:, 2:].abs()  # infinities of one sign
    g[:, 2:] = torch.where((g.double() / args).abs() < 1e30, g, torch.ones_like(g))[:, 2:] if dt != "f64" else g[:, 2:]
    if dt == "f64":
        g = torch.where((g.abs() / args < 1e300) | (g == 0), g, torch.zeros_like(g))
    small = args[:, 0] < 1e-20
    g[small] = 0.0  # 0 / T is 0, and not NaN
    ref = g.double() / args
    assert bool(ref.isfinite().all())
    size = ref.abs().sum(0)
    zero = torch.zeros(rows, k, dtype=dtype, device=gpu)
    wide = torch.float64 if dt == "f64" else torch.float32
    for history in (None, torch.zeros(rows, 3, dtype=torch.int64, device=gpu)):
        dz, db = cl.adjust_grad(g.to(gpu), zero, history=history, temperature=args[:, 0].to(gpu), bias=torch.zeros(k, dtype=wide, device=gpu))
        rd = in_range(ref, dtype)
        within(dz, rd, (ut + 3 * u) * torch.nan_to_num(rd, posinf=0.0, neginf=0.0).abs() + tiny + 1.5 * least)
        # terms as above, float64 additions, float32 result
        total = in_range(ref.sum(0), wide)
        within(db, total, 4 * u * size + rows * 2.0**-53 * size + rows * 2 * least)


def test_adjust_long_and_degenerate_histories(gpu):
    from distributions_amd import categorical_logits as cl

    k = 300
    z = make((3, k), torch.float32, 3, gpu)
    one = torch.zeros(3, 5000, dtype=torch.int32, device=gpu)  # one token, 5000 times
    lengths = torch.tensor([5000, 1, 0], device=gpu)
    a = dict(history=one, lengths=lengths, frequency=0.01, presence=0.5, repetition=1.3)
    ref, bound = plain_adjust(z, **a)
    within(cl.adjust(z, **a), ref, bound)
    shared = torch.arange(k, device=gpu)[None, :].expand(3, k)  # a history all rows share, without a copy
    a = dict(history=shared, repetition=1.7)
    ref, bound = plain_adjust(z, **a)
    within(cl.adjust(z, **a), ref, bound)
    far = torch.tensor([[2**40, -(2**40), 2**32, k, -k, 0]], device=gpu)  # ids that are no categories, also modulo 2^32
    a = dict(history=far, presence=1.0)
    ref, bound = plain_adjust(z, **a)
    within(cl.adjust(z, **a), ref, bound)
    a = dict(history=torch.zeros(3, 0, dtype=torch.int64, device=gpu), presence=1.0, repetition=2.0)
    assert torch.equal(cl.adjust(z, **a), z)
    assert cl.adjust(z[:0], temperature=2.0).shape == (0, k)


def test_adjust_counters_past_16_bits(gpu):
    """A history longer than 32767 ids takes wider counters: one token 40000 times, some of them in the prompt."""
    from distributions_amd import categorical_logits as cl

    k, n = 5000, 40001
    z = make((2, k), torch.float32, 3, gpu)
    h = torch.full((2, n), 4097, dtype=torch.int32, device=gpu)
    h[1, ::3] = 4096
    a = dict(history=h, prompt_lengths=torch.tensor([1, 30000], device=gpu), frequency=0.25, presence=0.5, repetition=1.3)
    ref, bound = plain_adjust(z, **a)
    assert float(ref[0, 4097]) < -9999
    within(cl.adjust(z, **a), ref, bound)
    dz, _ = cl.adjust_grad(z, z, **a)
    rz, _ = plain_adjust_grad(z, z, **a)
    within(dz, rz, 8 * 2.0**-24 * rz.abs())


@pytest.mark.parametrize("dt, mask, bias", [("f32", "bits", "shared"), ("bf16", "bool", "rows"), ("f16", "bits", None), ("f64", None, "rows")])
def test_adjust_many_rows_of_several_chunks(gpu, dt, mask, bias):
    """Rows dealt to the XCDs (their number no multiple of eight), several chunks a row, histories of several rounds."""
    from distributions_amd import categorical_logits as cl

    rows, k = 131, 20011
    dtype, wide = DT[dt], torch.float64 if dt == "f64" else torch.float32
    u, ut, tiny = steps(dtype)
    z, g = make((rows, k), dtype, 1, gpu), make((rows, k), dtype, 2, gpu)
    a = adjust_args(rows, k, 5, gpu, 1500, mask, bias, wide)
    ref, bound = plain_adjust(z, **a)
    within(cl.adjust(z, **a), ref, bound)
    dz, db = cl.adjust_grad(g, z, **a)
    rz, rb = plain_adjust_grad(g, z, **a)
    within(dz, rz, ut * rz.abs() + 6 * u * rz.abs() + tiny)
    if bias == "rows":
        within(db, rb, 3 * u * rb.abs() + 2.0**-149)
    elif bias:
        within(db, rb.sum(0), 4 * u * rb.abs().sum(0) + 2.0**-149)


def strided(z):
    """The same values in other layouts: odd offset, row gap, transposed, last of three axes, expanded."""
    rows, k = z.shape
    big = torch.full((rows, k + 5), 7.0, dtype=z.dtype, device=z.device)
    big[:, 3 : 3 + k] = z
    yield big[:, 3 : 3 + k]
    yield z.t().contiguous().t()
    cube = torch.full((rows, 3, k), 7.0, dtype=z.dtype, device=z.device)
    cube[:, 2] = z
    yield cube[:, 2, :]
    flat = torch.full((rows * k + 1,), 7.0, dtype=z.dtype, device=z.device)
    flat[1:] = z.reshape(-1)
    yield flat[1:].reshape(rows, k)


@pytest.mark.parametrize("dt", DT)
def test_layouts(gpu, dt):
    from distributions_amd import categorical_logits as cl

    rows, k = 4, 1021
    z = make((rows, k), DT[dt], 5, gpu)
    x = torch.tensor([0, 1020, -1, 77], device=gpu)
    w = torch.tensor([1.0, 0.5, 2.0, -1.0], device=gpu)
    a = adjust_args(rows, k, 6, gpu, wide=torch.float64 if dt == "f64" else torch.float32)
    want, lp = cl.adjust(z, **a), cl.logpdf(x, z)
    total, (_, grad) = cl.sum_logpdf_grad(x, z, w)
    dz, db = cl.adjust_grad(z, z, **a)
    for y in strided(z):
        assert torch.equal(cl.adjust(y, **a), want)
        assert torch.equal(cl.logpdf(x, y), lp)
        t2, (_, g2) = cl.sum_logpdf_grad(x, y, w)
        assert torch.equal(t2, total) and torch.equal(g2, grad)
        got = cl.adjust_grad(y, y, **a)
        assert torch.equal(got[0], dz) and torch.equal(got[1], db)
    # leading axes; arguments that broadcast along some of them
    y = z.reshape(2, 2, k)
    assert torch.equal(cl.logpdf(x.reshape(2, 2), y), lp.reshape(2, 2))
    t = torch.tensor([[0.5], [2.0]], device=gpu)
    assert torch.equal(cl.adjust(y, temperature=t)[1], cl.adjust(y[1], temperature=2.0))
    bias = make((2, 1, k), torch.float32, 8, gpu) if dt != "f64" else make((2, 1, k), torch.float64, 8, gpu)
    _, db = cl.adjust_grad(y, y, bias=bias, temperature=t)
    ref = (y.cpu().double() / t.cpu().double()[:, :, None]).sum(1, keepdim=True)
    size = (y.cpu().double().abs() / t.cpu().double()[:, :, None]).sum(1, keepdim=True)
    u = steps(bias.dtype)[0]
    within(db, ref, 6 * u * size)
    one = cl.logpdf(77, z[3])
    assert one.shape == () and torch.equal(one, lp[3])
    assert torch.equal(cl.logpdf(77, z[3:4].expand(5, k)), lp[3].expand(5))


def test_out_in_place(gpu):
    from distributions_amd import categorical_logits as cl

    for dtype in (torch.bfloat16, torch.float32, torch.float64):
        z = make((6, 5003), dtype, 9, gpu)
        a = adjust_args(6, 5003, 11, gpu, wide=torch.float64 if dtype == torch.float64 else torch.float32)
        want = cl.adjust(z, **a)
        y = z.clone()
        assert cl.adjust(y, out=y, **a) is y and torch.equal(y, want)
        pad = torch.full((6, 5010), 7.0, dtype=dtype, device=gpu)
        cl.adjust(z, out=pad[:, 2:5005], **a)
        assert torch.equal(pad[:, 2:5005], want) and bool((pad[:, :2] == 7).all()) and bool((pad[:, 5005:] == 7).all())
        x = torch.tensor([0, 5002, 3, -1, 7, 2500], device=gpu)
        total, (_, grad) = cl.sum_logpdf_grad(x, z)
        y = z.clone()
        t2, (_, g2) = cl.sum_logpdf_grad(x, y, out=y)
        assert g2 is y and torch.equal(y, grad) and torch.equal(t2, total)


def test_outputs_count_as_writes(gpu):
    """What autograd has saved and an output overwrites is an error in the backward pass, as with any operation in place."""
    from distributions_amd import categorical_logits as cl
    from distributions_amd import gradients

    x = torch.tensor([1, 2, 3], device=gpu)
    for write in (lambda y: cl.adjust(y, temperature=2.0, out=y), lambda y: cl.sum_logpdf_grad(x, y, out=y),
                  lambda y: gradients.clip_global_norm([y], 0.1, out=[y]), lambda y: cl.adjust(y[1:], temperature=2.0, out=y[1:]),
                  lambda y: gradients.clip_global_norm([y[:, 1:]], 0.1, out=[y[:, 1:]])):
        leaf = torch.randn(3, 50, device=gpu, requires_grad=True)
        y = leaf.exp()  # saves its result
        before = y._version
        write(y.detach())
        assert y._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    z = torch.randn(3, 50, device=gpu)  # and nothing else does
    cl.adjust(z, temperature=2.0), cl.sum_logpdf_grad(x, z), gradients.clip_global_norm([z], 0.1)
    assert z._version == 0
    with torch.inference_mode():
        z = torch.randn(3, 50, device=gpu)
        cl.adjust(z, temperature=2.0, out=z), gradients.clip_global_norm([z], 0.1, out=[z])


# ------------------------------------------------------------------------------------------------- log-density
@pytest.mark.parametrize("rows, k", SIZES + [(2, 50021), (1, 131072), (1, 262147), (300, 515), (700, 64), (5, 32), (9, 129), (4, 512), (3, 513)])
@pytest.mark.parametrize("dt", DT)
def test_logpdf_total_and_gradient(gpu, dt, rows, k):
    from distributions_amd import categorical_logits as cl

    dtype = DT[dt]
    z = make((rows, k), dtype, k + rows, gpu)
    gen = torch.Generator().manual_seed(k)
    x = torch.randint(0, k, (rows,), generator=gen)
    w = torch.randn(rows, generator=gen, dtype=torch.float64 if dt == "f64" else torch.float32)
    if rows > 2:
        x[1], w[2] = -1, 0.0
    lp, b_lp, total, b_total, grad, b_g = plain_logpdf(x, z, w)
    got = cl.logpdf(x.to(gpu), z)
    assert got.dtype == (torch.float64 if dt == "f64" else torch.float32)
    within(got, lp, b_lp)
    w0 = torch.where(x < 0, 0.0, w)  # -inf would swallow the total
    _, _, total, b_total, _, _ = plain_logpdf(x, z, w0)
    within(cl.sum_logpdf(x.to(gpu), z, w0.to(gpu)), total, b_total)
    t, (none, g) = cl.sum_logpdf_grad(x.to(gpu), z, w.to(gpu))
    assert none is None and g.dtype == dtype
    within(g, grad, b_g)
    t, _ = cl.sum_logpdf_grad(x.to(gpu), z, w0.to(gpu))
    within(t, total, b_total)
    again = cl.sum_logpdf_grad(x.to(gpu), z, w.to(gpu))
    assert torch.equal(again[1][1], g)


@pytest.mark.parametrize("k", [3, 700, 70001])
@pytest.mark.parametrize("dt", DT)
def test_rows_without_a_finite_answer(gpu, dt, k):
    from distributions_amd import categorical_logits as cl

    dtype = DT[dt]
    z = make((8, k), dtype, 4, gpu)
    z[0] = -INF  # nothing left
    z[1, 1:] = -INF  # one category left
    z[2, 2] = math.nan
    z[3, 0] = INF
    z[4] = torch.finfo(dtype).min  # a mask spelled as the lowest value: uniform
    z[5, 0] = -torch.finfo(dtype).min  # the largest value next to small ones
    z[6] = math.nan  # padding
    z[7, 2] = -INF  # the observation is not allowed, others are
    x = torch.tensor([1, 0, 0, 0, 2, 0, 1, 2], device=gpu)
    w = torch.tensor([1.0, 1, 1, 1, 1, 1, 0, 1], device=gpu)
    lp = cl.logpdf(x, z).cpu().double()
    assert lp[0] == -INF and lp[1] == 0 and lp[2].isnan() and lp[3].isnan() and lp[6].isnan() and lp[7] == -INF
    assert abs(float(lp[4]) + math.log(k)) <= 1e-4 * math.log(k) and lp[5] == 0
    total, (_, g) = cl.sum_logpdf_grad(x, z, w)
    g = g.cpu().double()
    assert total.isnan()
    assert bool((g[0] == 0).all()) and bool((g[1] == 0).all()) and bool(g[2].isnan().all()) and bool(g[3].isnan().all())
    assert bool((g[6] == 0).all())
    *_, ref, b = plain_logpdf(x[4:], z[4:], w[4:])
    within(g[4:], ref, b)
    keep = torch.tensor([0.0, 1, 0, 0, 1, 1, 0, 0], device=gpu)
    assert bool(cl.sum_logpdf(x, z, keep).isfinite())
    # labels that are no category, in every type they may have
    for bad in ([-1, k, k + 5, -(2**40)], [-1.0, float(k), 0.5, math.nan]):
        xb = torch.tensor(bad * 2, device=gpu)
        assert bool((cl.logpdf(xb, z[5:6].expand(8, k)) == -INF).all())
        t, (_, g) = cl.sum_logpdf_grad(xb, z[5:6].expand(8, k))
        assert t == -INF and bool((g == 0).all())
    for good in (torch.int32, torch.int64, torch.float32, torch.float64, torch.int16):
        assert torch.equal(cl.logpdf(torch.tensor([2], device=gpu).to(good), z[5:6]), cl.logpdf(2, z[5:6]))


def test_gradients_against_differences(gpu):
    """The whole chain adjust -> sum_logpdf in float64 against central differences, leaf by leaf."""
    from distributions_amd import categorical_logits as cl

    rows, k = 3, 11
    z = make((rows, k), torch.float64, 20, gpu, 1.0)
    a = adjust_args(rows, k, 21, gpu, 9, None, "shared", torch.float64)
    x = torch.tensor([1, 5, 10], device=gpu)
    w = torch.tensor([1.0, 0.3, 2.0], dtype=torch.float64, device=gpu)

    def f(zz, bias):
        return float(cl.sum_logpdf(x, cl.adjust(zz, **{**a, "bias": bias}), w))

    _, (_, g) = cl.sum_logpdf_grad(x, cl.adjust(z, **a), w)
    dz, db = cl.adjust_grad(g, z, **a)
    h = 1e-5  # error h^2 / 6 times a third derivative below 10, and 2^-52 |f| / h
    for i in range(rows):
        for j in range(k):
            if abs(float(z[i, j])) < 2 * h:
                continue  # the kink of the repetition penalty
            e = torch.zeros_like(z)
            e[i, j] = h
            assert abs((f(z + e, a["bias"]) - f(z - e, a["bias"])) / (2 * h) - float(dz[i, j])) < 1e-8
    for j in range(k):
        e = torch.zeros_like(a["bias"])
        e[j] = h
        assert abs((f(z, a["bias"] + e) - f(z, a["bias"] - e)) / (2 * h) - float(db[j])) < 1e-8


def test_offsets_past_32_bits(gpu):
    """Rows 2^31 elements apart: the third starts 2^32 elements behind the first."""
    from distributions_amd import categorical_logits as cl

    k = 1000
    flat = torch.empty(2**32 + k, dtype=torch.bfloat16, device=gpu)
    z = flat.as_strided((3, k), (2**31, 1))
    z.copy_(make((3, k), torch.bfloat16, 30, gpu))
    small = z.contiguous()
    x = torch.tensor([0, 999, 500], device=gpu)
    a = adjust_args(3, k, 31, gpu)
    assert torch.equal(cl.logpdf(x, z), cl.logpdf(x, small))
    assert torch.equal(cl.adjust(z, **a), cl.adjust(small, **a))
    total, (_, g) = cl.sum_logpdf_grad(x, small)
    t2, _ = cl.sum_logpdf_grad(x, z, out=z)
    assert torch.equal(total, t2) and torch.equal(z, g)


def test_many_short_rows(gpu):
    """More rows than the launch has workgroups for one each, k from 1 to the borders of the short kernels."""
    from distributions_amd import categorical_logits as cl

    for k, dtype in ((1, torch.float32), (10, torch.bfloat16), (32, torch.float64), (33, torch.float32), (300, torch.float16)):
        rows = 5000
        z = make((rows, k), dtype, k, gpu)
        x = torch.arange(rows, device=gpu) % (k + 1) - 1  # one in k + 1 is no category
        lp, b_lp, _, _, grad, b_g = plain_logpdf(x, z)
        within(cl.logpdf(x, z), lp, b_lp)
        _, (_, g) = cl.sum_logpdf_grad(x, z)
        within(g, grad, b_g)
        wide = torch.float64 if dtype == torch.float64 else torch.float32
        a = adjust_args(rows, k, 3, gpu, 0, "bits", "rows", wide)
        ref, bound = plain_adjust(z, **a)
        within(cl.adjust(z, **a), ref, bound)
        dz, db = cl.adjust_grad(z, z, **a)
        rz, rb = plain_adjust_grad(z, z, **a)
        u, ut, tiny = steps(dtype)
        within(dz, rz, ut * rz.abs() + 6 * u * rz.abs() + tiny)
        within(db, rb, 3 * u * rb.abs() + 2.0**-149)


# the borders between launch variants of the density and its gradient: row lengths in pieces of 16 bytes are 2^8 ... 2^14 for
# one type or another, one piece more, and a tail behind it
BORDERS = [512, 520, 1024, 1037, 2048, 2057, 4096, 4107, 8192 + 8, 10007, 16384, 16395, 32768, 32779, 65536, 65541, 131080]


@pytest.mark.parametrize("k", BORDERS)
@pytest.mark.parametrize("dt", DT)
def test_density_at_the_borders_of_its_variants(gpu, dt, k):
    from distributions_amd import categorical_logits as cl

    z = make((4, k), DT[dt], k, gpu)
    x = torch.tensor([k - 1, 0, k // 2, k - 9])
    w = torch.tensor([1.0, -0.5, 2.0, 0.25], dtype=torch.float64 if dt == "f64" else torch.float32)
    lp, b_lp, total, b_total, grad, b_g = plain_logpdf(x, z, w)
    within(cl.logpdf(x.to(gpu), z), lp, b_lp)
    t, (_, g) = cl.sum_logpdf_grad(x.to(gpu), z, w.to(gpu))
    within(t, total, b_total)
    within(g, grad, b_g)
    t2, (_, g2) = cl.sum_logpdf_grad(x.to(gpu), z, w.to(gpu), out=z)
    assert g2 is z and torch.equal(g2, g) and torch.equal(t2, t)


@pytest.mark.parametrize("dt", DT)
def test_many_long_rows(gpu, dt):
    """From 1024 rows on, longer than the value's kernel of 256 threads holds at once."""
    from distributions_amd import categorical_logits as cl

    rows, k = 1030, 9001
    z = make((rows, k), DT[dt], 3, gpu)
    x = torch.arange(rows) * 8 % k
    lp, b_lp, *_ = plain_logpdf(x, z)
    within(cl.logpdf(x.to(gpu), z), lp, b_lp)


@pytest.mark.parametrize("rows, k", [(8192, 3), (8193, 3), (20000, 40), (12289, 600)])
@pytest.mark.parametrize("dt", DT)
def test_total_over_many_rows(gpu, dt, rows, k):
    """From 8193 rows on several workgroups add the rows, and a last one what they have added."""
    from distributions_amd import categorical_logits as cl

    z = make((rows, k), DT[dt], 1, gpu)
    gen = torch.Generator().manual_seed(2)
    x = torch.randint(0, k, (rows,), generator=gen)
    w = torch.randn(rows, generator=gen, dtype=torch.float64 if dt == "f64" else torch.float32)
    w[::7] = 0
    x[::7] = -1  # padding
    _, _, total, b_total, grad, b_g = plain_logpdf(x, z, w)
    within(cl.sum_logpdf(x.to(gpu), z, w.to(gpu)), total, b_total)
    t, (_, g) = cl.sum_logpdf_grad(x.to(gpu), z, w.to(gpu))
    within(t, total, b_total)
    within(g, grad, b_g)
    again, _ = cl.sum_logpdf_grad(x.to(gpu), z, w.to(gpu))
    assert torch.equal(again, t)


@pytest.mark.parametrize("history", [0, 3])
@pytest.mark.parametrize("rows, k", [(5003, 1), (5003, 10), (5003, 100), (700, 257), (5003, 2051)])
@pytest.mark.parametrize("dt", DT)
def test_shared_bias_gradient_over_many_rows(gpu, dt, rows, k, history):
    """Column sums of few columns over several blocks of rows."""
    from distributions_amd import categorical_logits as cl

    dtype, wide = DT[dt], torch.float64 if dt == "f64" else torch.float32
    u, ut, tiny = steps(dtype)
    z, g = make((rows, k), dtype, 1, gpu), make((rows, k), dtype, 2, gpu)
    a = adjust_args(rows, k, 5, gpu, history, "bool" if k != 100 else "bits", "shared", wide)
    dz, db = cl.adjust_grad(g, z, **a)
    rz, rb = plain_adjust_grad(g, z, **a)
    within(dz, rz, ut * rz.abs() + 6 * u * rz.abs() + tiny)
    # terms: T, 1 / T, the product; float64 additions, one after the other at worst; the result's own rounding
    within(db, rb.sum(0), (4 * u + rows * 2.0**-53) * rb.abs().sum(0) + 2.0**-149)
    assert torch.equal(db, cl.adjust_grad(g, z, **a)[1])


def repeated(base, rows):
    return base.repeat((rows // len(base) + 1,) + (1,) * (base.dim() - 1))[:rows]


def same_as_repeated(got, base):
    """Whether `got` is `base` again and again, compared without another copy of it."""
    n = len(got) // len(base) * len(base)
    return bool((got[:n].view(-1, *base.shape) == base).all()) and torch.equal(got[n:], base[: len(got) - n])


@pytest.mark.parametrize("rows, k", [(2**21 + 3001, 520), (2**23 + 777, 129), (2**27 + 777, 2)])
def test_density_of_more_rows_than_workgroups(gpu, rows, k):
    """Workgroups that walk on to further rows (there are 2^21 at most): every row as in a launch that has one for each."""
    from distributions_amd import categorical_logits as cl

    n = 1021
    z = make((n, k), torch.bfloat16, 1, gpu)
    gen = torch.Generator().manual_seed(2)
    x = torch.randint(0, k, (n,), generator=gen, dtype=torch.int32)
    w = torch.randn(n, generator=gen)
    w[::7], x[3::11] = 0.0, -1
    lp, b_lp, _, _, grad, b_g = plain_logpdf(x, z, w)
    lp0 = cl.logpdf(x.to(gpu), z)
    within(lp0, lp, b_lp)
    _, (_, g0) = cl.sum_logpdf_grad(x.to(gpu), z, w.to(gpu))
    within(g0, grad, b_g)
    big_z, big_x = repeated(z, rows), repeated(x.to(gpu), rows)
    w[3::11] = 0.0  # a finite total
    big_w = repeated(w.to(gpu), rows)
    assert same_as_repeated(cl.logpdf(big_x, big_z), lp0)
    total, (_, g) = cl.sum_logpdf_grad(big_x, big_z, big_w)
    assert same_as_repeated(g, torch.where(w.to(gpu)[:, None] == 0, torch.zeros_like(g0), g0))
    times = torch.full((n,), rows // n, dtype=torch.float64)
    times[: rows % n] += 1
    keep = w != 0
    terms, off = (times * w.double() * lp)[keep], (times * w.double().abs() * b_lp)[keep]
    # the rows' own bounds; float64 additions; the total's rounding
    within(total, terms.sum(), float(off.sum() + (2 * 2.0**-24 + rows * 2.0**-53) * terms.abs().sum()))


def test_adjust_of_more_rows_than_workgroups(gpu):
    """The same for the adjustment: with a history (the counters in LDS are cleared between the rows), without one, and with
    more pieces than 32 bits count."""
    from distributions_amd import categorical_logits as cl

    n, k, rows = 1021, 11, 2**21 + 3001
    z = make((n, k), torch.bfloat16, 1, gpu)
    a = adjust_args(n, k, 5, gpu, 6, "bool", "rows")
    ref, bound = plain_adjust(z, **a)
    small = cl.adjust(z, **a)
    within(small, ref, bound)
    dz0, db0 = cl.adjust_grad(z, z, **a)
    big = {name: repeated(v, rows) for name, v in a.items()}
    big_z = repeated(z, rows)
    assert same_as_repeated(cl.adjust(big_z, **big), small)
    dz, db = cl.adjust_grad(big_z, big_z, **big)
    assert same_as_repeated(dz, dz0) and same_as_repeated(db, db0)
    del dz, db, big, big_z
    for rows, k in ((2**28 + 777, 3), (2**32 + 777, 1)):
        z = make((n, k), torch.bfloat16, 1, gpu)
        bias = make((k,), torch.bfloat16, 2, gpu)
        small = cl.adjust(z, bias=bias, temperature=0.7)
        ref, bound = plain_adjust(z, bias=bias, temperature=0.7)
        within(small, ref, bound)
        big = repeated(z, rows)
        assert same_as_repeated(cl.adjust(big, bias=bias, temperature=0.7, out=big), small)
        del big


@pytest.mark.parametrize("k", [20, 3000])
def test_weights_below_the_arithmetic(gpu, k):
    """A float64 weight that float32 rounds to 0 is no padding: its row counts in the total."""
    from distributions_amd import categorical_logits as cl

    z = make((4, k), torch.float32, 2, gpu)
    x = torch.tensor([0, 1, 2, 3], device=gpu)
    w = torch.tensor([1.0, 1e-60, 0.0, 2.0], dtype=torch.float64, device=gpu)
    total, (_, g) = cl.sum_logpdf_grad(x, z, w)
    lp, b_lp, ref, b_total, grad, b_g = plain_logpdf(x, z, w)
    within(total, ref, b_total)
    within(g, grad, b_g)


@pytest.mark.parametrize("dt", DT)
def test_shared_bias_gradient_of_no_rows(gpu, dt):
    """Through the C-ABI, with the workspace it asks for (none): the sums over no rows are 0, and nothing else is written."""
    from distributions_amd import _lib, _logits
    from distributions_amd import categorical_logits as cl

    dtype, k = DT[dt], 1003
    torch_, L = _logits._bind()
    for history in (None, torch.zeros(0, 5, dtype=torch.int64, device=gpu)):
        buf = torch.full((k + 40,), 7.0, dtype=dtype, device=gpu)
        bias = torch.zeros(k, dtype=dtype, device=gpu)
        d, keep, *_ = _logits._adjustment((0,), k, dtype, torch_, bias.device, history, None, None, 1.0, 0.0, 0.0, bias, 1.0, None)
        code = _logits._codes[dtype]
        assert L.m355_logits_adjust_grad_workspace_bytes(0, k, code) == 0
        _lib.check(L.m355_logits_adjust_grad(0, k, code, None, k, None, k, d, None, buf[20:].data_ptr(), None, 0,
                                             _logits._stream(torch_, bias.device)))
        assert bool((buf[20 : 20 + k] == 0).all()) and bool((buf[:20] == 7).all()) and bool((buf[20 + k :] == 7).all())
        empty = torch.empty(0, k, dtype=dtype, device=gpu)
        dz, db = cl.adjust_grad(empty, empty, history=history, bias=bias)
        assert dz.shape == (0, k) and db.shape == (k,) and bool((db == 0).all())


@pytest.mark.parametrize("dt", DT)
def test_expanded_bias(gpu, dt):
    """A bias that is an expanded view gets a gradient per row, as a contiguous one of the same shape does."""
    from distributions_amd import categorical_logits as cl

    k, wide = 1003, torch.float64 if dt == "f64" else torch.float32
    for batch, bshape in (((4,), (4, k)), ((2, 7), (2, 7, k)), ((2, 7), (2, 1, k)), ((2, 7), (7, k)), ((1,), (1, k)), ((3, 5), (1, 5, k))):
        z, g = make((*batch, k), DT[dt], 1, gpu), make((*batch, k), DT[dt], 2, gpu)
        for bdt in {DT[dt], wide}:
            base = make((k,), bdt, 3, gpu)
            bias = base.expand(bshape)
            full = bias.contiguous()
            assert torch.equal(cl.adjust(z, bias=bias), cl.adjust(z, bias=full))
            dz, db = cl.adjust_grad(g, z, bias=bias, temperature=0.7)
            dz2, db2 = cl.adjust_grad(g, z, bias=full, temperature=0.7)
            assert torch.equal(dz, dz2) and db.shape == bshape and db.dtype == bdt and torch.equal(db, db2)
            if len(batch) == 1 or bshape == (*batch, k):
                u, ut, tiny = steps(bdt)
                ref = g.cpu().double() / 0.7
                # T, 1 / T, its product in the arithmetic of the logits, then the bias' own type
                within(db, ref.reshape(bshape), (ut + 3 * steps(DT[dt])[0]) * ref.abs() + tiny)


def test_bias_of_another_type(gpu):
    from distributions_amd import categorical_logits as cl

    z = make((5, 700), torch.float32, 2, gpu)
    for dtype in (torch.float64, torch.bfloat16, torch.float16):
        b = make((700,), dtype, 3, gpu)
        assert torch.equal(cl.adjust(z, bias=b), cl.adjust(z, bias=b.float()))
        dz, db = cl.adjust_grad(z, z, bias=b)
        assert db.dtype == dtype and torch.equal(db, cl.adjust_grad(z, z, bias=b.float())[1].to(dtype))
    dz, db = cl.adjust_grad(z.cpu().numpy(), z.cpu().numpy(), bias=np.zeros(700))
    assert db.dtype == np.float64


def test_numpy_and_types(gpu):
    from distributions_amd import categorical_logits as cl

    z = np.random.default_rng(0).normal(size=(4, 9))
    lp = cl.logpdf([0, 1, 2, 9], z)
    assert isinstance(lp, np.ndarray) and lp.dtype == np.float64 and np.isneginf(lp[3])
    ref = z - np.log(np.exp(z).sum(1, keepdims=True))
    assert np.allclose(lp[:3], ref[[0, 1, 2], [0, 1, 2]], rtol=1e-13)
    total, (none, g) = cl.sum_logpdf_grad([0, 1, 2, 3], z)
    assert isinstance(total, float) and none is None and g.shape == z.shape
    assert np.allclose(g, np.eye(9)[:4] - np.exp(ref), atol=1e-14)
    out = cl.adjust(z.astype(np.float32), history=[[1, 1]] * 4, frequency=0.5, mask=np.arange(9) < 5)
    assert out.dtype == np.float32 and np.isneginf(out[:, 5:]).all()
    assert np.allclose(out[:, 1], z[:, 1].astype(np.float32) - 1.0, atol=1e-6)
    assert cl.logpdf(1, [0, 0, 0]).dtype == np.float64  # integers become float64


def test_refusals(gpu):
    from distributions_amd import categorical_logits as cl

    z = make((4, 10), torch.float32, 1, gpu)
    h = torch.zeros(4, 3, dtype=torch.int64, device=gpu)
    bad = [
        (ValueError, dict(repetition=0.0, history=h)), (ValueError, dict(temperature=-1.0)), (ValueError, dict(repetition=1.2)),
        (ValueError, dict(presence=0.1)), (ValueError, dict(lengths=h[:, 0])), (TypeError, dict(history=h.float())),
        (ValueError, dict(history=h[:3])), (ValueError, dict(history=h, lengths=h[:3, 0])), (TypeError, dict(history=h, lengths=z[:, 0])),
        (ValueError, dict(bias=z[:, :9])), (ValueError, dict(bias=z[:3])), (TypeError, dict(mask=z)), (ValueError, dict(mask=z[:, :9] > 0)),
        (ValueError, dict(mask=h[:, :2].int())), (ValueError, dict(temperature=z[:3, 0])), (ValueError, dict(out=z[:3])),
        (ValueError, dict(out=z.double())), (ValueError, dict(out=z.t().contiguous().t())), (ValueError, dict(out=z[:1].expand(4, 10))),
        (ValueError, dict(out=torch.empty(8, 10, device=gpu)[::2], bias=None, mask=None, temperature=z.new_ones(3))),
    ]
    for err, kw in bad:
        with pytest.raises(err):
            cl.adjust(z, **kw)
    buf = torch.zeros(5, 10, device=gpu)
    with pytest.raises(ValueError, match="overlaps"):
        cl.adjust(buf[:4], out=buf[1:])
    with pytest.raises(ValueError, match="overlaps"):
        cl.adjust(z, bias=buf[:4], out=buf[:4])
    with pytest.raises(ValueError):
        cl.adjust_grad(z[:, :9], z)
    with pytest.raises(ValueError):
        cl.logpdf(torch.zeros(3, device=gpu), z)
    with pytest.raises(ValueError):
        cl.logpdf(0, torch.zeros(3, 0, device=gpu))
    with pytest.raises(TypeError):
        cl.logpdf(0, z.to(torch.complex64))
    with pytest.raises(ValueError):
        cl.sum_logpdf(0, z, torch.ones(3, device=gpu))


# --------------------------------------------------------------------------- runs of them together, streams, graphs
def step(z, x, w, a, max_norm):
    """A training step of a constrained categorical: adjust, log-density, its gradient, back through adjust, clip."""
    from distributions_amd import categorical_logits as cl
    from distributions_amd import gradients

    s = cl.adjust(z, **a)
    total, (_, g) = cl.sum_logpdf_grad(x, s, w)
    dz, db = cl.adjust_grad(g, z, **a)
    norm, (dz, db) = gradients.clip_global_norm([dz, db], max_norm)
    return total, norm, dz, db


@pytest.mark.parametrize("dt", ["f64", "f32", "bf16"])
def test_step_against_autograd(gpu, dt):
    rows, k = 40, 2003
    dtype = DT[dt]
    wide = torch.float64 if dt == "f64" else torch.float32
    u, ut, _ = steps(dtype)
    z = make((rows, k), dtype, 40, gpu, 1.5)
    a = adjust_args(rows, k, 41, gpu, 25, "bool", "shared", wide)
    a["mask"][:] = True
    a["mask"][:, ::7] = False
    x = torch.arange(rows, device=gpu) * 7 + 1
    w = torch.ones(rows, dtype=wide, device=gpu)
    w[::6] = 0
    total, norm, dz, db = step(z, x, w, a, 0.5)
    zr = z.cpu().double().requires_grad_()
    br = a["bias"].cpu().double().requires_grad_()
    call, cgen = counts_of(a["history"], a["lengths"], a["prompt_lengths"], rows, k)
    p = {n: a[n].cpu().double()[:, None] for n in ("repetition", "presence", "frequency", "temperature")}
    s = torch.where(call > 0, torch.where(zr > 0, zr / p["repetition"], zr * p["repetition"]), zr)
    s = (s - p["frequency"] * cgen - p["presence"] * (cgen > 0) + br) / p["temperature"]
    s = s.masked_fill(~a["mask"].cpu(), -INF)
    ref = (w.cpu().double() * (s.gather(1, x.cpu()[:, None])[:, 0] - torch.logsumexp(s, 1))).sum()
    ref.backward()
    n = torch.sqrt(zr.grad.square().sum() + br.grad.square().sum())
    # logits between -20 and 20 are rounded once on the way (20 ut each), gradients twice: relative to the whole
    tol = 40 * ut + 4000 * u
    assert abs(float(total) - float(ref.detach())) <= tol * rows
    assert abs(float(norm) - float(n)) <= tol * float(n)
    f = 0.5 / float(n)
    assert float((dz.cpu().double() - zr.grad * f).norm()) <= tol * 0.5
    assert float((db.cpu().double() - br.grad * f).norm()) <= tol * 0.5


def test_bias_shared_by_some_axes(gpu):
    """A bias that is broadcast along some of the rows' axes: its gradient, eager and captured."""
    from distributions_amd import categorical_logits as cl

    for shape, bshape in (((3, 7, 50), (3, 1, 50)), ((3, 7, 50), (7, 50)), ((2, 5, 3, 9), (2, 1, 3, 9)), ((2, 5, 3, 9), (5, 1, 9))):
        g = make(shape, torch.float32, 1, gpu)
        z = make(shape, torch.float32, 2, gpu)
        bias = make(bshape, torch.float32, 3, gpu)
        full = (1,) * (len(shape) - len(bshape)) + bshape
        axes = [i for i, (m, n) in enumerate(zip(full, shape)) if m != n]
        ref = g.cpu().double().sum(axes, keepdim=True).reshape(bshape)
        size = g.cpu().double().abs().sum(axes, keepdim=True).reshape(bshape)
        _, db = cl.adjust_grad(g, z, bias=bias)
        within(db, ref, 8 * 2.0**-24 * size)  # T and its quotient 1; at most 4 + 2 additions by halves
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            cl.adjust_grad(g, z, bias=bias)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _, captured = cl.adjust_grad(g, z, bias=bias)
        for i in range(3):
            g.copy_(make(shape, torch.float32, 10 + i, gpu))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(captured, cl.adjust_grad(g, z, bias=bias)[1])


@pytest.mark.parametrize("bdt", DT)
@pytest.mark.parametrize("dt", DT)
def test_bias_shared_along_a_long_axis(gpu, dt, bdt):
    """The sum over the rows that share a bias is rounded to the bias' type once, whatever that is and whichever axes it has."""
    from distributions_amd import categorical_logits as cl

    dtype, b_dtype, k = DT[dt], DT[bdt], 37
    u, ut, tiny = steps(dtype)[0], *steps(b_dtype)[1:]
    if dt != "f64":
        u = 2.0**-24
    for shape, bshape in (((2, 1500, k), (2, 1, k)), ((1500, 2, k), (2, k)), ((40, 3, 40, k), (1, 3, 1, k)), ((3000, k), (k,))):
        g, z = make(shape, dtype, 1, gpu), make(shape, dtype, 2, gpu)
        bias = make(bshape, b_dtype, 3, gpu)
        t = (0.5 + torch.rand(shape[:-1], generator=torch.Generator().manual_seed(4))).to(gpu)
        _, db = cl.adjust_grad(g, z, bias=bias, temperature=t)
        assert db.dtype == b_dtype and db.shape == bshape
        terms = g.cpu().double() / t.cpu().double()[..., None]
        full = (1,) * (len(shape) - len(bshape)) + bshape
        axes = [i for i, (m, n) in enumerate(zip(full, shape)) if m != n]
        ref, size = terms.sum(axes).reshape(bshape), terms.abs().sum(axes).reshape(bshape)
        # each term: 1 / T and its product, 2 u; float64 additions: 3000 * 2^-53; then the rounding to the bias' type, for 16
        # bits by way of float32 (u), and from float32 where the kernel's output is that
        within(db, ref, ut * ref.abs() + 2 * 2.0**-24 * ref.abs() * (bdt != "f64" or dt != "f64") + (2 * u + 3000 * 2.0**-53) * size + tiny)


def test_two_streams_at_once(gpu):
    """Steps of two problems that are under way together on two streams give what each gives alone."""
    work, want = [], []
    for i, (rows, k) in enumerate(((300, 4001), (17, 60000))):
        z = make((rows, k), torch.bfloat16, 70 + i, gpu)
        a = adjust_args(rows, k, 72 + i, gpu, 300, "bool", "shared")
        a["mask"][-1] = True
        x = torch.arange(rows, device=gpu)
        a["mask"][torch.arange(rows, device=gpu), x] = True
        work.append((z, x, torch.ones(rows, device=gpu), a, 0.3))
        want.append(step(*work[-1]))
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*work[i]))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(p, q) for r in runs for p, q in zip(w, r))


def test_streams_and_captured_graphs(gpu):
    """A step on another stream, and two captured graphs of it replayed in turn with eager work in between."""
    rows, k = 33, 5003
    z = make((rows, k), torch.bfloat16, 50, gpu)
    a = adjust_args(rows, k, 51, gpu, 40, "bits", "shared")
    a["mask"][-1] = -1
    x = torch.arange(rows, device=gpu)
    w = torch.ones(rows, device=gpu)
    want = step(z, x, w, a, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(z, x, w, a, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graphs = []
    for max_norm in (0.1, 1e9):
        with torch.cuda.stream(side):
            step(z, x, w, a, max_norm)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(z, x, w, a, max_norm)
        graphs.append((graph, res, max_norm))
    for i in range(4):
        z.copy_(make((rows, k), torch.bfloat16, 60 + i, gpu))
        for graph, res, max_norm in graphs:
            for r in res:
                r.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            eager = step(z, x, w, a, max_norm)
            assert all(torch.equal(p, q) for p, q in zip(res, eager)), (i, max_norm)
