"""A training step of the dense operators in every kernel that the rule of tiles chooses, against 64 bits with the
tolerances derived in test_gpu_dense.py."""
import pytest
import torch

from dense_variants import F32, FEW_ROWS, GLU, LINEAR, SHORT, VARIANTS
from test_gpu_dense import DT, dev, glu64, glu_grads64, grads64, linear64, rand, within  # noqa: F401

pytestmark = pytest.mark.gpu


def cases(gated):
    return [(dt, *s) for key, names in ((F32, ("f32",)), (SHORT, ("bf16", "f16"))) for s in VARIANTS[gated, key] + FEW_ROWS
            for dt in names]


@pytest.mark.parametrize("dt,n,k,m", cases(LINEAR))
def test_linear(dev, dt, n, k, m):  # noqa: F811
    from bcfft import dense
    x, w = rand(dev, n, k, dt=DT[dt], seed=201), rand(dev, m, k, dt=DT[dt], seed=202, scale=k ** -0.5)
    b, dy = rand(dev, m, dt=DT[dt], seed=203), rand(dev, n, m, dt=DT[dt], seed=204)
    ins = [t.clone().requires_grad_() for t in (x, w, b)]
    y = dense.linear(*ins, activation="gelu")
    want, slack, z, zs, slope = linear64(x, w, b, None, "gelu")
    within(y.detach(), want, slack)
    y.backward(dy)
    for t, (grad, gslack) in zip(ins, grads64(x, w, dy, slope, zs, "gelu", DT[dt])):
        within(t.grad, grad, gslack)


@pytest.mark.parametrize("dt,n,k,m", cases(GLU))
def test_glu(dev, dt, n, k, m):  # noqa: F811
    from bcfft import dense
    x, dh = rand(dev, n, k, dt=DT[dt], seed=211), rand(dev, n, m, dt=DT[dt], seed=212)
    wg, wu = (rand(dev, m, k, dt=DT[dt], seed=s, scale=k ** -0.5) for s in (213, 214))
    ins = [t.clone().requires_grad_() for t in (x, wg, wu)]
    h = dense.glu(*ins)
    want, slack, parts = glu64(x, wg, wu, "silu")
    within(h.detach(), want, slack)
    h.backward(dh)
    for t, (grad, gslack) in zip(ins, glu_grads64(x, wg, wu, dh, parts, DT[dt])):
        within(t.grad, grad, gslack)
