"""The dense projections and the distillation loss under autograd's own machinery: checkpoints, saved tensors kept on
the host, a graph walked twice, an input overwritten between forward and backward, a backward on another stream. The
same kernels on the same values: equal bits."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "ctypes"])
def path(request, monkeypatch):
    from bcfft import _lib
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    if request.param == "ctypes":
        monkeypatch.setattr(_lib, "_native", False)
    else:
        assert _lib.native_op(), "libbcfft_torch.so not loaded"


def operands():
    g = torch.Generator(device="cuda").manual_seed(3)

    def t(*shape, scale=0.3):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)
    x, wg, wu, wd, bias, wo = t(70, 96), t(130, 96), t(130, 96), t(96, 130), t(96), t(500, 96)
    values, indices = t(70, 6, scale=2.0), torch.randint(0, 500, (70, 6), generator=g, device="cuda")
    return [x, wg, wu, wd, bias, wo], values, indices


def step(ins, values, indices):
    from bcfft import dense, distill
    x, wg, wu, wd, bias, wo = ins
    y = dense.linear(dense.glu(x, wg, wu), wd, bias, activation="gelu", residual=x)
    return distill.topk_kl(dense.linear(y, wo), values, indices, temperature=1.5)


def fresh(ins):
    return [t.detach().clone().requires_grad_() for t in ins]


def grads_of(run, ins):
    ins = fresh(ins)
    loss = run(ins)
    loss.sum().backward()
    return [loss.detach()] + [t.grad for t in ins]


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


def test_checkpoints_and_saved_tensors_on_the_host(path):
    ins, values, indices = operands()
    want = grads_of(lambda i: step(i, values, indices), ins)
    for reentrant in (True, False):
        got = grads_of(lambda i: checkpoint(lambda *a: step(a, values, indices), *i, use_reentrant=reentrant), ins)
        assert same(got, want)

    def offloaded(i):
        with torch.autograd.graph.save_on_cpu():
            return step(i, values, indices)
    assert same(grads_of(offloaded, ins), want)


def test_a_graph_walked_twice(path):
    ins, values, indices = operands()
    leaves = fresh(ins)
    loss = step(leaves, values, indices).sum()
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    second = torch.autograd.grad(loss, leaves)
    assert same(first, second)
    with pytest.raises(RuntimeError, match="second time|already been freed"):
        torch.autograd.grad(loss, leaves)


def test_overwritten_operands_are_noticed(path):
    """x, a weight, the teacher's values: what the backward reads again must be what the forward read."""
    for which in (0, 2, 5, 6):
        ins, values, indices = operands()
        leaves = fresh(ins)
        loss = step(leaves, values, indices).sum()
        with torch.no_grad():
            (values if which == 6 else leaves[which]).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_backward_under_another_stream(path):
    """The backward runs on the forward's stream whichever is current where it is called."""
    ins, values, indices = operands()
    want = grads_of(lambda i: step(i, values, indices), ins)
    side = torch.cuda.Stream()
    leaves = fresh(ins)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = step(leaves, values, indices)
        total = loss.sum()
    torch.cuda.current_stream().wait_stream(side)
    total.backward()
    torch.cuda.synchronize()
    assert same([loss.detach()] + [t.grad for t in leaves], want)
