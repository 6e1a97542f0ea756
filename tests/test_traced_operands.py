"""Gradients of traced calls are refused whichever operand or mode traces, on the CPU: an autograd node that
launches kernels would leave nothing in the trace."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from bcfft import _lib, dense, distill

INDICES = torch.zeros(4, 3, dtype=torch.int32)
CALLS = {
    "linear": lambda x, o: dense.linear(x, o["weight"], o["bias"], activation="gelu", residual=o["residual"]),
    "glu": lambda x, o: dense.glu(x, o["weight"], o["w_up"]),
    "topk_kl": lambda x, o: distill.topk_kl(x, o["values"], INDICES, rest=o["rest"], weight=o["w"]),
}


@pytest.fixture
def operands(built_lib):
    if not _lib.native_op():
        pytest.skip("the C++ operators are not built")
    return dict(weight=torch.randn(48, 64), w_up=torch.randn(48, 64), bias=torch.randn(48), residual=torch.randn(4, 48),
                values=torch.randn(4, 3), rest=torch.randn(4), w=torch.randn(4))


@pytest.mark.parametrize("name,which", [("linear", "weight"), ("linear", "bias"), ("linear", "residual"),
                                        ("glu", "weight"), ("glu", "w_up"), ("topk_kl", "values"), ("topk_kl", "rest"),
                                        ("topk_kl", "w")])
def test_any_traced_operand(operands, name, which):
    with FakeTensorMode():
        operands[which] = torch.empty(tuple(operands[which].shape))
    x = torch.randn(4, 64, requires_grad=True)
    with pytest.raises(RuntimeError, match="traced"):
        CALLS[name](x, operands)


@pytest.mark.parametrize("name", list(CALLS))
def test_traced_by_a_mode(operands, name):
    """make_fx over memory that is there, and a FakeTensorMode around it: no operand says that it is traced."""
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda x: CALLS[name](x, operands))(torch.randn(4, 64, requires_grad=True))
    x = torch.randn(4, 64, requires_grad=True)
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(RuntimeError, match="traced"):
        CALLS[name](x, operands)
