"""Rewired dense MLPs (patch_llama_fft.fuse_dense_mlp) on the GPU where they leave the dense kernels: against the
same modules in fp64, a few 2^-24 of sums of 64 and 96 products apart, with room for a factor of 50."""
import types

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
HIDDEN, INNER = 64, 96


class MLP(nn.Module):
    def __init__(self, device):
        super().__init__()
        self.gate_proj, self.up_proj = (nn.Linear(HIDDEN, INNER, bias=False, device=device) for _ in range(2))
        self.down_proj = nn.Linear(INNER, HIDDEN, bias=False, device=device)
        self.act_fn = nn.SiLU()

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


@pytest.fixture
def mlp():
    import patch_llama_fft as P
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    torch.manual_seed(0)
    m = MLP(torch.device("cuda:0"))
    assert P.fuse_dense_mlp(types.SimpleNamespace(model=types.SimpleNamespace(layers=[types.SimpleNamespace(mlp=m)]))) == 1
    return m


def plain(m, x):
    w = [p.detach().double().requires_grad_() for p in (m.gate_proj.weight, m.up_proj.weight, m.down_proj.weight)]
    return (m.act_fn(x.double() @ w[0].t()) * (x.double() @ w[1].t())) @ w[2].t(), w


def close(got, want):
    assert float((got.double() - want).norm() / want.norm()) < 1e-5


def test_replaced_activation(mlp):
    x = torch.randn(5, HIDDEN, device="cuda:0")
    with torch.no_grad():
        close(mlp(x), plain(mlp, x)[0])
        mlp.act_fn = nn.GELU()
        close(mlp(x), plain(mlp, x)[0])


def test_compiled_forward_and_training_step(mlp):
    """torch.compile: the operators are in the trace without a gradient, the modules with one."""
    compiled = torch.compile(mlp, backend="aot_eager", fullgraph=True)
    x = torch.randn(5, HIDDEN, device="cuda:0")
    with torch.no_grad():
        assert torch.equal(compiled(x), mlp(x))
    y = compiled(x)
    want, weights = plain(mlp, x)
    close(y.detach(), want.detach())
    dy = torch.randn_like(y)
    y.backward(dy)
    want.backward(dy.double())
    for p, w in zip((mlp.gate_proj.weight, mlp.up_proj.weight, mlp.down_proj.weight), weights):
        close(p.grad, w.grad)


def test_transforms_and_forward_mode(mlp):
    """torch.func.grad, jvp and vmap over a rewired MLP: derivatives of the fp64 formula."""
    x, t = torch.randn(5, HIDDEN, device="cuda:0"), torch.randn(5, HIDDEN, device="cuda:0")
    x64 = x.double().requires_grad_()
    want = plain(mlp, x64)[0]
    (dx,) = torch.autograd.grad(want.sum(), x64, retain_graph=True)
    close(torch.func.grad(lambda v: mlp(v).sum())(x), dx)
    close(torch.func.vmap(mlp)(x), want.detach())
    for p in mlp.parameters():
        p.requires_grad_(False)
    y, jvp = torch.func.jvp(mlp, (x,), (t,))
    _, want_jvp = torch.autograd.functional.jvp(lambda v: plain(mlp, v)[0], x.double(), t.double())
    close(y, want.detach())
    close(jvp, want_jvp)
