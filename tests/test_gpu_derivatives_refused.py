"""Second derivatives of the dense projections and the distillation loss are refused on the GPU too where the
gradient that comes in needs none itself (a gradient penalty)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "ctypes"])
def path(request, monkeypatch):
    from bcfft import _lib
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    if request.param == "ctypes":
        monkeypatch.setattr(_lib, "_native", False)
    else:
        assert _lib.native_op(), "libbcfft_torch.so not loaded"


@pytest.mark.parametrize("rows", [4, 0])
@pytest.mark.parametrize("name", ["linear", "glu", "topk_kl"])
def test_gradient_penalty(path, name, rows):
    """loss + penalty on its gradient: without the refusal the penalty's own gradient is missing from the sum."""
    from bcfft import dense, distill
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(rows, 64, generator=g, device="cuda", requires_grad=True)
    w = torch.randn(48, 64, generator=g, device="cuda", requires_grad=True)
    indices = torch.arange(3, device="cuda", dtype=torch.int32).expand(rows, 3)
    calls = {"linear": lambda: dense.linear(x, w, activation="gelu"), "glu": lambda: dense.glu(x, w, w),
             "topk_kl": lambda: distill.topk_kl(x, x.detach()[:, :3], indices)}
    loss = calls[name]().sum()
    (dx,) = torch.autograd.grad(loss, x, create_graph=True)
    assert dx.shape == x.shape and dx.requires_grad
    with pytest.raises(RuntimeError, match="differentiate twice"):
        (loss + dx.square().sum()).backward()
    # without create_graph nothing changes
    (dx,) = torch.autograd.grad(calls[name]().sum(), x)
    assert not dx.requires_grad


def test_the_residuals_gradient_is_the_incoming_one(path):
    """dr = dy: right to any order, recorded or not."""
    from bcfft import dense
    x, r, dy = (torch.randn(4, 64, device="cuda", requires_grad=True) for _ in range(3))
    w = torch.randn(64, 64, device="cuda")
    (dr,) = torch.autograd.grad(dense.linear(x, w, residual=r), r, dy, create_graph=True)
    (second,) = torch.autograd.grad(dr.square().sum(), dy)
    assert torch.equal(second, 2 * dy)
