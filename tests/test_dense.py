"""Dense projections on the CPU: refusals of the C entry points (before any launch) and of the Python
functions, workspace sizes."""
import ctypes

import pytest
import torch

OK, SHAPE, DTYPE, ALIGN, ARG = 0, 1, 3, 4, 6
P = ctypes.c_void_p(64)                      # never dereferenced: every call below ends before a launch
ODD = ctypes.c_void_p(65)


def linear(lib, x=P, dt=2, n=4, xs=64, k=64, m=32, w=P, b=None, r=None, rs=0, act=0, y=P, z=None, ws=None, wb=0):
    return lib.bcfft_dense_linear(x, dt, n, xs, k, m, w, b, r, rs, act, y, z, ws, wb, None)


@pytest.mark.parametrize("bad,status", [
    (dict(dt=9), DTYPE), (dict(n=-1), SHAPE), (dict(n=(1 << 23) + 1), SHAPE), (dict(k=0, xs=1), SHAPE),
    (dict(m=0), SHAPE), (dict(k=(1 << 20) + 1, xs=1 << 21), SHAPE), (dict(m=(1 << 20) + 1), SHAPE), (dict(xs=63), SHAPE),
    (dict(r=P, rs=31), SHAPE), (dict(act=4), ARG), (dict(act=-1), ARG), (dict(x=None), ARG), (dict(w=None), ARG),
    (dict(y=None), ARG), (dict(x=ODD), ALIGN), (dict(w=ODD), ALIGN), (dict(b=ODD), ALIGN), (dict(r=ODD, rs=32), ALIGN),
    (dict(y=ODD), ALIGN), (dict(z=ctypes.c_void_p(66)), ALIGN), (dict(ws=ctypes.c_void_p(72)), ALIGN),
    (dict(dt=0, x=ctypes.c_void_p(66)), ALIGN)])
def test_linear_refusals(built_lib, bad, status):
    from bcfft import _lib
    assert linear(_lib.load(), **bad) == status


@pytest.mark.parametrize("bad,status", [
    (dict(dt=9), DTYPE), (dict(xs=63), SHAPE), (dict(act=4), ARG), (dict(wg=None), ARG), (dict(wu=None), ARG),
    (dict(h=None), ARG), (dict(wu=ODD), ALIGN), (dict(gu=ctypes.c_void_p(66)), ALIGN)])
def test_glu_refusals(built_lib, bad, status):
    from bcfft import _lib
    a = dict(x=P, dt=2, n=4, xs=64, k=64, m=32, wg=P, wu=P, act=2, h=P, gu=None)
    a.update(bad)
    assert _lib.load().bcfft_dense_glu(a["x"], a["dt"], a["n"], a["xs"], a["k"], a["m"], a["wg"], a["wu"], a["act"],
                                       a["h"], a["gu"], None, 0, None) == status


@pytest.mark.parametrize("bad,status", [
    (dict(n=0), ARG), (dict(act=3, z=None), ARG), (dict(w=None), ARG), (dict(x=None), ARG), (dict(dy=None), ARG),
    (dict(ds=31), SHAPE), (dict(dx=ODD), ALIGN), (dict(ws=None), ARG), (dict(wb=16), ARG)])
def test_linear_backward_refusals(built_lib, bad, status):
    from bcfft import _lib
    a = dict(x=P, dt=2, n=4, xs=64, k=64, m=32, w=P, dy=P, ds=32, z=P, act=2, dx=P, dw=P, db=P, ws=P, wb=1 << 30)
    a.update(bad)
    assert _lib.load().bcfft_dense_linear_backward(
        a["x"], a["dt"], a["n"], a["xs"], a["k"], a["m"], a["w"], a["dy"], a["ds"], a["z"], a["act"], a["dx"], a["dw"],
        a["db"], a["ws"], a["wb"], None) == status


@pytest.mark.parametrize("bad,status", [
    (dict(n=0), ARG), (dict(gu=None), ARG), (dict(wg=None), ARG), (dict(x=None), ARG), (dict(dh=None), ARG),
    (dict(m=(1 << 19) + 1, ds=1 << 20), SHAPE), (dict(ws=None), ARG), (dict(wb=16), ARG), (dict(dw=ODD), ALIGN)])
def test_glu_backward_refusals(built_lib, bad, status):
    from bcfft import _lib
    a = dict(x=P, dt=2, n=4, xs=64, k=64, m=32, wg=P, wu=P, dh=P, ds=32, gu=P, act=2, dx=P, dw=P, ws=P, wb=1 << 30)
    a.update(bad)
    assert _lib.load().bcfft_dense_glu_backward(
        a["x"], a["dt"], a["n"], a["xs"], a["k"], a["m"], a["wg"], a["wu"], a["dh"], a["ds"], a["gu"], a["act"],
        a["dx"], a["dw"], a["ws"], a["wb"], None) == status


def test_no_rows_and_workspace_sizes(built_lib):
    from bcfft import _lib
    lib = _lib.load()
    assert linear(lib, n=0, x=None, w=None, y=None) == OK
    for op in range(4):
        assert lib.bcfft_dense_workspace_bytes(op, 0, 64, 64, 2, 0) == 0
        assert lib.bcfft_dense_workspace_bytes(op, 100, 64, 64, 2, 2) >= 0
        assert lib.bcfft_dense_workspace_bytes(op, 100, 0, 64, 2, 0) == -1
        assert lib.bcfft_dense_workspace_bytes(op, 100, 64, 64, 5, 0) == -1
    assert lib.bcfft_dense_workspace_bytes(4, 100, 64, 64, 2, 0) == -1
    # the backward of an activation holds dz; of the gated form dg and du
    assert lib.bcfft_dense_workspace_bytes(2, 100, 64, 64, 2, 2) >= 100 * 64 * 2
    assert lib.bcfft_dense_workspace_bytes(3, 100, 64, 64, 2, 2) >= 100 * 64 * 4


def test_host_tensors_are_refused(built_lib):
    from bcfft import dense
    x, w = torch.randn(3, 8), torch.randn(4, 8)
    for grad in (False, True):
        with pytest.raises(RuntimeError, match="ROCm device"):
            dense.linear(x.clone().requires_grad_(grad), w)
        with pytest.raises(RuntimeError, match="ROCm device"):
            dense.glu(x.clone().requires_grad_(grad), w, w)


def test_fake_shapes(built_lib):
    """FakeTensors: the registered operators give shapes and dtypes without a device or a launch."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from bcfft import _lib, dense, torch_ops  # noqa: F401
    with FakeTensorMode():
        for dt in (torch.float32, torch.bfloat16):
            x, w = torch.empty(2, 5, 64, device="cuda", dtype=dt), torch.empty(48, 64, device="cuda", dtype=dt)
            y = torch.ops.bcfft.dense_linear(x, w, None, None, "gelu")
            h = torch.ops.bcfft.dense_glu(x, w, w, "silu")
            for t in (y, h):
                assert t.shape == (2, 5, 48) and t.dtype == dt and t.device.type == "cuda"
            if _lib.native_op():
                assert dense.linear(x, w).shape == dense.glu(x, w, w).shape == (2, 5, 48)
        with pytest.raises(ValueError, match="in_features"):
            torch.ops.bcfft.dense_linear(x, w.t(), None, None, "none")
        with pytest.raises(ValueError, match="in_features"):
            torch.ops.bcfft.dense_glu(x, w, w[:3], "silu")


def test_traced_gradients_are_refused(built_lib):
    """A C++ autograd node would read memory that a FakeTensor does not have."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from bcfft import _lib, dense, distill
    if not _lib.native_op():
        pytest.skip("the C++ operators are not built")
    with FakeTensorMode():
        x = torch.empty(4, 64, device="cuda", requires_grad=True)
        w = torch.empty(48, 64, device="cuda")
        for call in (lambda: dense.linear(x, w), lambda: dense.glu(x, w, w),
                     lambda: distill.topk_kl(x, w[:4, :3], torch.empty(4, 3, device="cuda", dtype=torch.int32))):
            with pytest.raises(RuntimeError, match="traced"):
                call()
