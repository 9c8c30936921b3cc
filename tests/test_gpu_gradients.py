"""Norm over a list of gradients and clipping by it, on the GPU, against float64."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = (torch.float64, torch.float32, torch.float16, torch.bfloat16)
INF = math.inf


def plain_norm(grads):
    return math.sqrt(math.fsum(float(g.cpu().double().square().sum()) for g in grads if g is not None and g.numel()))


def check(norm, clipped, grads, before, max_norm):
    """norm and clipped values of `before` (float64 copies of the gradients)."""
    ref = math.sqrt(math.fsum(float(b.square().sum()) for b in before))
    n = sum(b.numel() for b in before)
    # float64 sum of n squares: n roundings of 2^-53 at worst, halved by the root; then the norm's own rounding
    tol = n * 2.0**-53 + (2.0**-24 if norm.dtype == torch.float32 else 2.0**-52)
    assert abs(float(norm) - ref) <= tol * ref
    f = max_norm / ref if ref > max_norm else 1.0
    for g, c, b in zip(grads, clipped, before):
        assert c.dtype == g.dtype and c.shape == g.shape
        info = torch.finfo(c.dtype)
        want = b * f
        # the factor (n 2^-53 + a few), the product, and for 16-bit types the float32 on the way: 2^-24
        rel = info.eps / 2 + n * 2.0**-53 + 2.0**-51 + (2.0**-24 if c.element_size() == 2 else 0.0)
        d = (c.cpu().double() - want).abs()
        assert bool((d <= rel * want.abs() + info.tiny * info.eps / 2).all())


def make(sizes, dtype, device, seed=0, scale=0.1):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * scale).to(dtype).to(device) for s in sizes]


SIZES = [[1], [2, 3, 5], [255, 256, 257, 0, 1], [4096, 16384, 16385, 40000, 7], [2**20 + 3, 11, 300000], [17] * 300 + [100003] * 3]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_and_clip(gpu, dtype, sizes):
    from distributions_amd import gradients as G

    grads = make(sizes, dtype, gpu)
    before = [g.cpu().double() for g in grads]
    ref = plain_norm(grads)
    norm = G.global_norm(grads)
    assert norm.shape == () and norm.dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
    for max_norm in (0.3 * ref, 10 * ref, 0.0):
        n, clipped = G.clip_global_norm(grads, max_norm)
        assert torch.equal(n, norm)
        check(n, clipped, grads, before, max_norm)
        assert all(torch.equal(g.cpu().double(), b) for g, b in zip(grads, before))  # the gradients are left as they are
        out = [torch.full_like(g, 7) for g in grads]
        n, given = G.clip_global_norm(grads, max_norm, out=out)
        assert all(a is b for a, b in zip(given, out)) and all(torch.equal(a, b) for a, b in zip(out, clipped))
        inplace = [g.clone() for g in grads]
        n, given = G.clip_global_norm(inplace, max_norm, out=inplace)
        assert all(torch.equal(a, b) for a, b in zip(inplace, clipped))


def test_mixed_types_strides_and_none(gpu):
    from distributions_amd import gradients as G

    a = torch.randn(37, 53, device=gpu)
    buf = torch.randn(1001, device=gpu).to(torch.bfloat16)
    grads = [a.t(), None, buf[1:1000], a[:, 3:9].contiguous().to(torch.float16), torch.randn(5, 6, 7, device=gpu)[:, ::2, 1:4],
             torch.tensor(3.0, device=gpu), torch.randn(4, 1, device=gpu).expand(4, 6), torch.randn(2, 3, 4, 5, device=gpu).permute(0, 2, 3, 1)]
    real = [g for g in grads if g is not None]
    before = [g.cpu().double() for g in real]
    n, clipped = G.clip_global_norm(grads, 1.0)
    assert clipped[1] is None and n.dtype == torch.float32
    check(n, [c for c in clipped if c is not None], real, before, 1.0)
    assert G.global_norm([torch.ones(4, device=gpu), torch.ones(5, dtype=torch.float64, device=gpu)]).dtype == torch.float64
    # outputs of another layout, and outputs with gaps: what lies in the gaps stays
    gap = torch.full((37, 60), 7.0, device=gpu)
    for out in ([torch.empty(53, 37, device=gpu)], [torch.empty(37, 53, device=gpu).t()], [gap[:, :53].t()]):
        n, (c,) = G.clip_global_norm([a.t()], 1.0, out=out)
        assert c is out[0]
        check(n, [c], [a.t()], [a.t().cpu().double()], 1.0)
    assert bool((gap[:, 53:] == 7).all())
    n, _ = G.clip_global_norm([gap[:, :53]], 0.5, out=[gap[:, :53]])  # in place through gaps
    assert bool((gap[:, 53:] == 7).all()) and abs(plain_norm([gap[:, :53]]) - 0.5) < 1e-6


def test_guards_around_the_outputs(gpu):
    from distributions_amd import gradients as G

    for dtype in DTYPES:
        for n in (1, 7, 8, 9, 4095, 16391):
            buf = torch.full((n + 32,), 7.0, dtype=dtype, device=gpu)
            g = make([n], dtype, gpu)[0]
            G.clip_global_norm([g], 0.01, out=[buf[13 : 13 + n]])
            assert bool((buf[:13] == 7).all()) and bool((buf[13 + n :] == 7).all())
            assert torch.equal(buf[13 : 13 + n], G.clip_global_norm([g], 0.01)[1][0])


def test_large_small_and_not_finite_values(gpu):
    from distributions_amd import gradients as G

    big = torch.full((1000,), 1e30, device=gpu)  # float32 squares of these overflow
    assert abs(float(G.global_norm([big])) / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    n, (c,) = G.clip_global_norm([big], 1.0)
    assert abs(float(c[0]) - 1 / math.sqrt(1000)) < 1e-8
    tiny = torch.full((1000,), 1e-30, device=gpu)
    assert abs(float(G.global_norm([tiny])) / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    for bad in (INF, -INF, math.nan):
        g = [torch.randn(300, device=gpu), torch.tensor([1.0, bad], device=gpu)]
        n, c = G.clip_global_norm(g, 0.1)
        assert not math.isfinite(float(n))
        assert all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(g, c))
    zero = [torch.zeros(10, device=gpu)]
    n, c = G.clip_global_norm(zero, 0.0)
    assert float(n) == 0 and bool((c[0] == 0).all())
    n, c = G.clip_global_norm([torch.randn(10, device=gpu)], INF)
    assert math.isfinite(float(n))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [8, 300000])  # one workgroup, and the general launches
def test_norm_that_float32_does_not_hold(gpu, dtype, n):
    """Finite gradients whose norm is returned as infinite are left as they are: what is returned and what is done agree."""
    from distributions_amd import gradients as G
    from distributions_amd import sharded

    for value, finite in ((3e38, False), (1e38 / math.sqrt(n), True)):
        grads = [torch.full((n,), value, dtype=dtype, device=gpu), torch.zeros(5, dtype=dtype, device=gpu)]
        before = [g.clone() for g in grads]
        for clip in (G.clip_global_norm, sharded.clip_global_norm):
            norm, clipped = clip(grads, 1.0)
            assert norm.dtype == torch.float32 and bool(norm.isfinite()) == finite
            assert torch.equal(clipped[0], before[0]) != finite and torch.equal(norm, G.global_norm(grads))
            if finite:
                check(norm, clipped, grads, [b.cpu().double() for b in before], 1.0)
            inplace = [g.clone() for g in grads]
            clip(inplace, 1.0, out=inplace)
            assert all(torch.equal(a, b) for a, b in zip(inplace, clipped))
    # a float64 tensor in the list: the norm is float64 and finite, and everything is scaled
    grads = [torch.full((n,), 3e38, dtype=dtype, device=gpu), torch.ones(3, dtype=torch.float64, device=gpu)]
    norm, clipped = G.clip_global_norm(grads, 1.0)
    check(norm, clipped, grads, [g.cpu().double() for g in grads], 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tensor_of_more_than_2_to_the_31_elements(gpu, dtype):
    """Offsets past 32 bits, of elements and of bytes, and the tensors behind such a one."""
    from distributions_amd import gradients as G

    big = torch.zeros(2**31 + 4099, dtype=dtype, device=gpu)
    at = torch.tensor([0, 2**30 + 1, 2**31 - 1, 2**31 + 7, 2**31 + 4098], device=gpu)
    big[at] = torch.tensor([2.0, 4.0, 2.0, 4.0, 2.0], dtype=dtype, device=gpu)  # squares: 44
    grads = [torch.tensor([1.0], dtype=dtype, device=gpu), big, torch.tensor([2.0, 0.0], dtype=dtype, device=gpu)]
    assert float(G.global_norm(grads)) == 7.0
    norm, clipped = G.clip_global_norm(grads, 3.5, out=grads)
    assert float(norm) == 7.0 and clipped[1] is big
    assert big[at].tolist() == [1.0, 2.0, 1.0, 2.0, 1.0] and int(torch.count_nonzero(big)) == 5
    assert grads[0].tolist() == [0.5] and grads[2].tolist() == [1.0, 0.0]


def test_empty_lists_twice_listed_and_numpy(gpu):
    from distributions_amd import gradients as G
    from distributions_amd import normal

    assert float(G.global_norm([])) == 0.0 and float(G.global_norm([None])) == 0.0
    n, c = G.clip_global_norm([None, torch.zeros(0, device=gpu)], 1.0)
    assert float(n) == 0 and c[0] is None and c[1].shape == (0,)
    g = torch.randn(100, device=gpu)
    assert abs(float(G.global_norm([g, g])) - math.sqrt(2) * plain_norm([g])) < 1e-5
    rng = np.random.default_rng(0)
    x = rng.normal(size=1000)
    _, grads = normal.sum_logpdf_grad(x, 0.3, 1.2)  # NumPy, scalars as 0-d arrays
    n, c = G.clip_global_norm(grads, 1.0)
    ref = math.sqrt(sum(float((np.asarray(q) ** 2).sum()) for q in grads))
    assert isinstance(n, float) and abs(n - ref) < 1e-12 * ref and isinstance(c[0], np.ndarray)
    assert np.allclose(c[0], grads[0] / ref, rtol=1e-13) and np.asarray(c[1]).shape == ()
    _, grads = normal.sum_logpdf_grad(torch.from_numpy(x).to(gpu), 0.3, 1.2, x_grad=False)
    n, c = G.clip_global_norm(grads, 1.0)
    assert c[0] is None and abs(math.sqrt(float(c[1]) ** 2 + float(c[2]) ** 2) - min(1.0, float(n))) < 1e-12


def test_refusals(gpu):
    from distributions_amd import M355Error
    from distributions_amd import gradients as G

    g = torch.randn(100, device=gpu)
    with pytest.raises(TypeError):
        G.global_norm(g)
    with pytest.raises(TypeError):
        G.global_norm([torch.ones(3, dtype=torch.int64, device=gpu)])
    with pytest.raises(ValueError):
        G.global_norm([g.cpu()])
    for m in (-1.0, math.nan):
        with pytest.raises(ValueError):
            G.clip_global_norm([g], m)
    for out in ([], [g[:50]], [g.double()], [torch.zeros(1, device=gpu).expand(100)]):
        with pytest.raises(ValueError):
            G.clip_global_norm([g], 1.0, out=out)
    for grads, out in (([g, g], [g, g]), ([g[:60]], [g[1:61]]), ([g[:50], g[50:]], [g[:50], g[:50]])):
        with pytest.raises(M355Error, match="overlaps"):
            G.clip_global_norm(grads, 1.0, out=out)
    m = torch.randn(10, 10, device=gpu)
    with pytest.raises(ValueError, match="gaps"):  # column blocks: their spans interleave
        G.clip_global_norm([m[:, :6], m[:, 5:]], 1.0, out=[m[:, :6], m[:, 5:]])
    n, _ = G.clip_global_norm([g[:50], g[50:]], 1.0, out=[g[:50], g[50:]])  # neighbours are no overlap
    assert abs(plain_norm([g]) - 1.0) < 1e-6


def test_sharded_one_rank(gpu):
    from distributions_amd import gradients as G
    from distributions_amd import sharded

    grads = make([1000, 33], torch.float32, gpu)
    n, c = G.clip_global_norm(grads, 0.5)
    n2, c2 = sharded.clip_global_norm(grads, 0.5)
    assert torch.equal(n, n2) and all(torch.equal(a, b) for a, b in zip(c, c2))
