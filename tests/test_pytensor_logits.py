"""The PyTensor Op of the categorical given by logits, against tests/pytensor_standin.py (or PyTensor where it is installed
and the stand-in steps aside)."""

import numpy as np
import pytest

from tests.test_pytensor_ops import HAVE

pytestmark = pytest.mark.skipif(HAVE, reason="the stand-in replaces PyTensor here")


def test_make_node():
    from tests.pytensor_standin import installed

    with installed() as (ops, pytensor):
        pt = pytensor.tensor
        out = ops.symbolic("categorical_logits").logpdf(pt.lvector("x"), pt.dmatrix("z"))
        assert out.dtype == "float64" and out.type.shape == (None,)
        assert ops.M355LogitsLogpdf()(pt.lvector(), pt.fmatrix()).dtype == "float32"
        assert ops.M355LogitsLogpdf()(1, pt.dvector()).type.shape == ()
        with pytest.raises(ValueError, match="logits"):
            ops.M355LogitsLogpdf()(pt.lvector(), pt.dvector())


@pytest.mark.gpu
def test_value_and_gradient(gpu):
    from tests.pytensor_standin import installed

    rng = np.random.default_rng(0)
    z = rng.normal(size=(6, 13))
    x = np.array([0, 12, 5, -1, 7, 3])
    x[3] = 4
    ref = z - np.log(np.exp(z).sum(1, keepdims=True))
    with installed() as (ops, pytensor):
        pt = pytensor.tensor
        zv, xv = pt.dmatrix("z"), pt.lvector("x")
        zv.type.shape, xv.type.shape = (6, 13), (6,)
        lp = ops.symbolic("categorical_logits").logpdf(xv, zv)
        lp.type.shape = (6,)
        assert np.allclose(lp.eval({xv: x, zv: z}), ref[np.arange(6), x], rtol=1e-13)
        w = np.array([1.0, 2.0, 0.0, -1.0, 0.5, 3.0])
        gx, gz = pytensor.grad((lp * pt.constant(w)).sum(), [xv, zv])
        ex, ez = pytensor.function([xv, zv], [gx, gz])(x, z)
        assert np.all(ex == 0) and ex.shape == (6,)
        assert np.allclose(ez, w[:, None] * (np.eye(13)[x] - np.exp(ref)), atol=1e-14)
