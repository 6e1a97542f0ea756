"""Top-logit distillation on the CPU: refusals of the C entry points and of the Python functions (before
any launch), and the registered operators' shapes."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

OK, SHAPE, DTYPE, ALIGN, ARG = 0, 1, 3, 4, 6
P = ctypes.c_void_p(64)                      # never dereferenced: every call below ends before a launch


def topk(lib, logits=P, dt=2, n=4, v=100, stride=100, k=8, t=1.0, values=P, indices=P, rest=P):
    return lib.bcfft_topk_logits(logits, dt, n, v, stride, k, t, values, indices, rest, None)


@pytest.mark.parametrize("bad,status", [
    (dict(dt=7), DTYPE), (dict(n=-1), SHAPE), (dict(v=0), SHAPE), (dict(stride=99), SHAPE), (dict(k=0), SHAPE),
    (dict(k=101), SHAPE), (dict(k=1025, v=4000, stride=4000), SHAPE), (dict(t=0.0), ARG), (dict(t=-1.0), ARG),
    (dict(t=float("nan")), ARG), (dict(t=float("inf")), ARG), (dict(logits=None), ARG), (dict(values=None), ARG),
    (dict(indices=None), ARG), (dict(rest=None), ARG), (dict(logits=ctypes.c_void_p(65)), ALIGN),
    (dict(dt=0, logits=ctypes.c_void_p(66)), ALIGN), (dict(indices=ctypes.c_void_p(66)), ALIGN),
    (dict(n=1 << 31), SHAPE), (dict(v=1 << 31, stride=1 << 31), SHAPE)])
def test_topk_refusals(built_lib, bad, status):
    from bcfft import _lib
    assert topk(_lib.load(), **bad) == status


def test_empty_is_no_op(built_lib):
    from bcfft import _lib
    lib = _lib.load()
    assert topk(lib, logits=None, n=0, values=None, indices=None, rest=None) == OK
    assert lib.bcfft_distill_topk(None, 2, 0, 100, 100, None, 2, None, 4, 8, None, None, 1.0, None, None, None,
                                  None) == OK


@pytest.mark.parametrize("bad,status", [
    (dict(dt=5), DTYPE), (dict(vdt=-1), DTYPE), (dict(v=(1 << 18) + 1, stride=1 << 20), SHAPE), (dict(k=0), SHAPE),
    (dict(k=1025), SHAPE), (dict(ib=2), ARG), (dict(t=0.0), ARG), (dict(logits=None), ARG), (dict(values=None), ARG),
    (dict(indices=None), ARG), (dict(loss=None), ARG), (dict(stats=ctypes.c_void_p(72)), ALIGN),
    (dict(grad=ctypes.c_void_p(65)), ALIGN), (dict(ib=8, indices=ctypes.c_void_p(68)), ALIGN),
    (dict(stride=50), SHAPE)])
def test_distill_refusals(built_lib, bad, status):
    from bcfft import _lib
    a = dict(logits=P, dt=2, n=4, v=100, stride=100, values=P, vdt=2, indices=P, ib=4, k=8, rest=None, weight=None,
             t=1.0, loss=P, stats=None, grad=None)
    a.update(bad)
    assert _lib.load().bcfft_distill_topk(a["logits"], a["dt"], a["n"], a["v"], a["stride"], a["values"], a["vdt"],
                                          a["indices"], a["ib"], a["k"], a["rest"], a["weight"], a["t"], a["loss"],
                                          a["stats"], a["grad"], None) == status


@pytest.mark.parametrize("bad,status", [
    (dict(stats=None), ARG), (dict(up=None), ARG), (dict(grad=None), ARG), (dict(stats=ctypes.c_void_p(72)), ALIGN),
    (dict(up=ctypes.c_void_p(66)), ALIGN), (dict(k=2000), SHAPE)])
def test_distill_backward_refusals(built_lib, bad, status):
    from bcfft import _lib
    a = dict(k=8, stats=P, up=P, grad=P)
    a.update(bad)
    assert _lib.load().bcfft_distill_topk_backward(P, 2, 4, 100, 100, P, 2, P, 4, a["k"], None, None, 1.0, a["stats"],
                                                   a["up"], a["grad"], None) == status


def test_host_tensors_are_refused(built_lib):
    import bc_eval
    from bcfft import distill
    z = torch.randn(3, 50)
    with pytest.raises(RuntimeError, match="ROCm device"):
        distill.topk_logits(z, 4)
    with pytest.raises(RuntimeError, match="ROCm device"):
        distill.topk_kl(z, z[:, :4], torch.zeros(3, 4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="ROCm device"):
        distill.topk_kl(z.clone().requires_grad_(), z[:, :4], torch.zeros(3, 4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="ROCm device"):
        distill.topk_kl_grad(z, z[:, :4], torch.zeros(3, 4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="ROCm device"):
        bc_eval.teacher_cache(z, 4)


def test_fake_shapes():
    import bcfft.torch_ops  # noqa: F401
    with FakeTensorMode():
        z = torch.empty(2, 5, 1000, dtype=torch.bfloat16)
        values, indices, rest = torch.ops.bcfft.topk_logits(z, 16, 2.0)
        assert values.shape == (2, 5, 16) and values.dtype == torch.bfloat16
        assert indices.shape == (2, 5, 16) and indices.dtype == torch.int32
        assert rest.shape == (2, 5) and rest.dtype == torch.float32
        loss = torch.ops.bcfft.topk_kl(z, values, indices, rest, None, 2.0)
        assert loss.shape == (2, 5) and loss.dtype == torch.float32
        loss, grad = torch.ops.bcfft.topk_kl_grad(z, values, indices, None, None, 1.0)
        assert grad.shape == z.shape and grad.dtype == z.dtype
        with pytest.raises(ValueError):
            torch.ops.bcfft.topk_logits(z, 1001, 1.0)
