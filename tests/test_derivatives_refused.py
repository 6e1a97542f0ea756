"""Derivatives that the dense projections and the distillation loss do not compute are refused by name instead of
coming out as zero, on the CPU (the refusals stand before the device check): forward mode."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from bcfft import _lib, dense, distill

INDICES = torch.zeros(4, 3, dtype=torch.int32)


def operands(device):
    def t(*shape):
        return torch.randn(*shape).to(device)
    return dict(x=t(4, 64), weight=t(48, 64), w_up=t(48, 64), bias=t(48), residual=t(4, 48), logits=t(4, 50), values=t(4, 3),
                rest=t(4), w=t(4), indices=INDICES.to(device))


CALLS = {
    "linear": (lambda o: dense.linear(o["x"], o["weight"], o["bias"], activation="gelu", residual=o["residual"]),
               ("x", "weight", "bias", "residual")),
    "glu": (lambda o: dense.glu(o["x"], o["weight"], o["w_up"]), ("x", "weight", "w_up")),
    "topk_kl": (lambda o: distill.topk_kl(o["logits"], o["values"], o["indices"], rest=o["rest"], weight=o["w"]),
                ("logits", "values", "rest", "w")),
    "topk_kl_grad": (lambda o: distill.topk_kl_grad(o["logits"], o["values"], o["indices"], rest=o["rest"], weight=o["w"]),
                     ("logits", "values", "rest", "w")),
    "topk_logits": (lambda o: distill.topk_logits(o["logits"], 3), ("logits",)),
}


@pytest.fixture(params=["native", "ctypes"])
def path(request, built_lib, monkeypatch):
    """The C++ operators (on the meta device too, which has kernels there) and the ctypes fallback."""
    if request.param == "ctypes":
        monkeypatch.setattr(_lib, "_native", False)
        return ["cpu"]
    if not _lib.native_op():
        pytest.skip("the C++ operators are not built")
    return ["cpu", "meta"]


@pytest.mark.parametrize("name", list(CALLS))
def test_forward_mode_is_refused(path, name):
    call, duals = CALLS[name]
    for device in path:
        for which in duals:
            for no_grad in (False, True):              # torch.no_grad() leaves forward mode on
                with fwAD.dual_level():
                    o = operands(device)
                    o[which] = fwAD.make_dual(o[which], torch.ones_like(o[which]))
                    with torch.set_grad_enabled(not no_grad), pytest.raises(RuntimeError, match="forward-mode"):
                        call(o)


@pytest.mark.parametrize("name", list(CALLS))
def test_operands_without_a_tangent_are_not(path, name):
    """A dual level alone, or the primal of a dual tensor, changes nothing."""
    call, duals = CALLS[name]
    with fwAD.dual_level():
        o = operands(path[-1])
        dual = fwAD.make_dual(o[duals[0]], torch.ones_like(o[duals[0]]))
        with fwAD._set_fwd_grad_enabled(False):
            o[duals[0]] = fwAD.unpack_dual(dual).primal
        if path[-1] == "meta":
            call(o)
        else:
            with pytest.raises(RuntimeError, match="ROCm device"):
                call(o)


@pytest.mark.parametrize("name", ["linear", "glu", "topk_kl"])
def test_functional_jvp_is_refused(path, name):
    call, duals = CALLS[name]
    o = operands(path[-1])

    def f(t):
        return call({**o, duals[0]: t})
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(f, (o[duals[0]],), (torch.ones_like(o[duals[0]]),))


@pytest.mark.parametrize("name", list(CALLS))
def test_registered_operators_refuse_forward_mode(built_lib, name):
    """torch.ops.bcfft.* (forward only) drop into the operators below autograd: they look at their operands too."""
    import bcfft.torch_ops  # noqa: F401
    ops = torch.ops.bcfft
    calls = {
        "linear": lambda o: ops.dense_linear(o["x"], o["weight"], o["bias"], o["residual"], "gelu"),
        "glu": lambda o: ops.dense_glu(o["x"], o["weight"], o["w_up"], "silu"),
        "topk_kl": lambda o: ops.topk_kl(o["logits"], o["values"], o["indices"], o["rest"], o["w"], 1.0),
        "topk_kl_grad": lambda o: ops.topk_kl_grad(o["logits"], o["values"], o["indices"], o["rest"], o["w"], 1.0),
        "topk_logits": lambda o: ops.topk_logits(o["logits"], 3, 1.0),
    }
    for device in ("cpu", "meta"):
        for which in CALLS[name][1]:
            with fwAD.dual_level():
                o = operands(device)
                o[which] = fwAD.make_dual(o[which], torch.ones_like(o[which]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    calls[name](o)
