"""Which path a rewired dense MLP takes (patch_llama_fft.fuse_dense_mlp), on the CPU: FakeTensors on a ROCm
device, so no launch, and the two operators replaced by recorders."""
import types

import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode

import patch_llama_fft as P

HIDDEN, INNER = 32, 48


class MLP(nn.Module):
    def __init__(self, act=None, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        kw = dict(bias=False, device=device, dtype=dtype)
        self.gate_proj, self.up_proj = nn.Linear(HIDDEN, INNER, **kw), nn.Linear(HIDDEN, INNER, **kw)
        self.down_proj = nn.Linear(INNER, HIDDEN, **kw)
        self.act_fn = nn.SiLU() if act is None else act

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


def model_of(*mlps):
    return types.SimpleNamespace(model=types.SimpleNamespace(layers=[types.SimpleNamespace(mlp=m) for m in mlps]))


@pytest.fixture
def fused_calls(monkeypatch):
    """The calls of the dense operators, which stand in by their shapes."""
    from bcfft import _lib, dense
    monkeypatch.setattr(_lib, "_native", True)
    calls = []

    def glu(x, w_gate, w_up, *, activation="silu"):
        calls.append("glu")
        return x.new_empty((*x.shape[:-1], w_gate.shape[0]))

    def linear(x, weight, bias=None, *, activation=None, residual=None):
        calls.append("linear")
        return x.new_empty((*x.shape[:-1], weight.shape[0]))

    monkeypatch.setattr(P, "_dense", types.SimpleNamespace(
        glu=glu, linear=linear, MAX_FEATURES=dense.MAX_FEATURES, MAX_TOKENS=dense.MAX_TOKENS))
    return calls


@pytest.fixture
def fake():
    with FakeTensorMode() as mode, torch.no_grad():
        yield mode


def rewired():
    mlp = MLP()
    assert P.fuse_dense_mlp(model_of(mlp)) == 1
    return mlp, torch.empty(2, 3, HIDDEN, device="cuda", dtype=torch.bfloat16)


def test_plain_modules_run_fused(fake, fused_calls):
    mlp, x = rewired()
    assert mlp(x).shape == x.shape and fused_calls == ["glu", "linear"]


def test_replaced_activation_runs_the_modules(fake, fused_calls):
    """An activation replaced after the call is the one that is computed."""
    mlp, x = rewired()
    seen = []

    class Watched(nn.GELU):
        def forward(self, z):
            seen.append(tuple(z.shape))
            return super().forward(z)

    class Scaled(nn.SiLU):
        def forward(self, z):
            seen.append(tuple(z.shape))
            return 2 * super().forward(z)

    for act in (Watched(), Scaled()):
        mlp.act_fn = act
        assert mlp(x).shape == x.shape
        assert fused_calls == [] and seen.pop() == (2, 3, INNER)
    mlp.act_fn = nn.SiLU()
    mlp(x)
    assert fused_calls == ["glu", "linear"]
    assert P.fuse_dense_mlp(model_of(MLP(act=Scaled()))) == 0


def test_hooked_activation_is_called(fake, fused_calls):
    mlp, x = rewired()
    seen = []
    for register in (mlp.act_fn.register_forward_hook, mlp.act_fn.register_forward_pre_hook):
        handle = register(lambda *a: seen.append(len(a)))
        mlp(x)
        assert len(seen) == 1 and fused_calls == []
        handle.remove()
        seen.clear()
    mlp(x)
    assert fused_calls == ["glu", "linear"]


@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "down_proj", "act_fn"])
def test_replaced_instance_forward_is_called(fake, fused_calls, name):
    """m.forward = ..., as offloading wrappers set it: the module's class stays what it was."""
    mlp, x = rewired()
    m = getattr(mlp, name)
    own, seen = m.forward, []

    def wrapper(z):
        seen.append(name)
        return own(z)

    m.forward = wrapper
    assert mlp(x).shape == x.shape
    assert seen == [name] and fused_calls == []
    del m.forward
    mlp(x)
    assert fused_calls == ["glu", "linear"]


@pytest.mark.parametrize("register", [
    torch.nn.modules.module.register_module_forward_hook,
    torch.nn.modules.module.register_module_forward_pre_hook,
    torch.nn.modules.module.register_module_full_backward_hook,
    torch.nn.modules.module.register_module_full_backward_pre_hook])
def test_hooks_on_every_module_run_the_modules(fake, fused_calls, register):
    """torch's global module hooks fire for the projections too."""
    mlp, x = rewired()
    handle = register(lambda m, *a: None)
    try:
        mlp(x)
        assert fused_calls == []
    finally:
        handle.remove()
    mlp(x)
    assert fused_calls == ["glu", "linear"]


class Sharded(torch.Tensor):
    """A tensor of a kind of its own, as sharded and quantised weights are: it says that it is on the GPU, holds
    no memory there, and computes its products itself (here by a fake twin)."""
    @staticmethod
    def __new__(cls, twin):
        t = torch.Tensor._make_wrapper_subclass(cls, twin.shape, dtype=twin.dtype, device=twin.device)
        t.twin = twin
        return t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        if func is torch.ops.aten.detach.default:
            return cls(args[0].twin)
        flat, spec = torch.utils._pytree.tree_flatten((args, kwargs or {}))
        args, kwargs = torch.utils._pytree.tree_unflatten([t.twin if isinstance(t, Sharded) else t for t in flat], spec)
        cls.seen.append(func)
        return func(*args, **kwargs)

    __torch_function__ = torch._C._disabled_torch_function_impl


@pytest.mark.parametrize("where", ["gate_proj", "up_proj", "down_proj", "bias", "x"])
def test_tensor_subclasses_run_the_modules(fused_calls, where):
    with torch.no_grad(), FakeTensorMode():
        mlp, x = rewired()
    Sharded.seen = []
    if where == "bias":
        with x.fake_mode:
            twin = torch.empty(HIDDEN, device="cuda", dtype=torch.bfloat16)
        mlp.down_proj.bias = nn.Parameter(Sharded(twin), requires_grad=False)
    elif where == "x":
        x = Sharded(x)
    else:
        m = getattr(mlp, where)
        m.weight = nn.Parameter(Sharded(m.weight.detach()), requires_grad=False)
    with torch.no_grad():
        assert mlp(x).shape == x.shape
    assert fused_calls == [] and len(Sharded.seen) >= 1


def test_traced_gradients_run_the_modules(fused_calls, monkeypatch):
    """The operators record no gradient of a traced call (torch.compile, FakeTensors, make_fx, a mode that
    watches every operation): the modules do. Without a gradient the operators themselves are traced."""
    with FakeTensorMode() as mode:
        mlp, x = rewired()
        mlp(x)
        assert fused_calls == []
        with torch.no_grad():
            mlp(x)
        assert fused_calls == ["glu", "linear"]
        for p in mlp.parameters():
            p.requires_grad_(False)
        mlp(x)
        assert fused_calls == ["glu", "linear"] * 2
        mlp(x.requires_grad_())
        assert fused_calls == ["glu", "linear"] * 2

    # the same decision for memory that is there, by the state of the tracer alone
    real = torch.empty(2, requires_grad=True)
    assert not P._untraceable(real)
    with monkeypatch.context() as mp:
        mp.setattr(torch.compiler, "is_compiling", lambda: True)
        assert P._untraceable(real) and not P._untraceable(real.detach())
    with mode:
        assert P._untraceable(real)
        with torch.no_grad():
            assert not P._untraceable(real)


def test_sizes_past_the_operators_run_the_modules(fake, fused_calls):
    from bcfft import dense
    mlp, _ = rewired()
    for rows, calls in ((dense.MAX_TOKENS, 2), (dense.MAX_TOKENS + 1, 0), (0, 2)):
        x = torch.empty(rows, HIDDEN, device="cuda", dtype=torch.bfloat16)
        assert mlp(x).shape == x.shape and len(fused_calls) == calls
        fused_calls.clear()
    for hidden, inner, calls in ((dense.MAX_FEATURES, INNER, 2), (dense.MAX_FEATURES + 1, INNER, 0),
                                 (HIDDEN, dense.MAX_FEATURES // 2, 2), (HIDDEN, dense.MAX_FEATURES // 2 + 1, 0),
                                 (0, INNER, 0), (HIDDEN, 0, 0)):
        mlp = MLP()
        for name, shape in (("gate_proj", (inner, hidden)), ("up_proj", (inner, hidden)), ("down_proj", (hidden, inner))):
            getattr(mlp, name).weight = nn.Parameter(torch.empty(shape, device="cuda", dtype=torch.bfloat16))
        assert P.fuse_dense_mlp(model_of(mlp)) == 1
        x = torch.empty(3, hidden, device="cuda", dtype=torch.bfloat16)
        assert mlp(x).shape == x.shape and len(fused_calls) == calls
        fused_calls.clear()


def test_residuals_that_the_epilogue_does_not_add(fake, fused_calls):
    """Of another dtype, a shape that broadcasts, a subclass, or with a traced gradient: added after the modules."""
    mlp, x = rewired()
    assert mlp(x, residual=torch.empty_like(x)).dtype == x.dtype and fused_calls == ["glu", "linear"]
    fused_calls.clear()
    y = mlp(x, residual=torch.empty(2, 3, HIDDEN, device="cuda"))
    assert y.dtype == torch.float32 and y.shape == x.shape
    assert mlp(x, residual=torch.empty(HIDDEN, device="cuda", dtype=x.dtype)).shape == x.shape
    assert mlp(x, residual=torch.empty(4, 2, 3, HIDDEN, device="cuda", dtype=x.dtype)).shape == (4, 2, 3, HIDDEN)
    Sharded.seen = []
    mlp(x, residual=Sharded(x))
    assert fused_calls == [] and len(Sharded.seen) == 1
    for p in mlp.parameters():
        p.requires_grad_(False)
    with torch.enable_grad():
        mlp(x, residual=torch.empty_like(x).requires_grad_())
    assert fused_calls == []


def test_an_mlp_with_a_forward_of_its_own_is_left_alone(fake, fused_calls):
    """An offloading wrapper around the whole MLP stays; the rewiring itself can be repeated."""
    mlp = MLP()
    own, seen = mlp.forward, []

    def wrapper(x):
        seen.append(1)
        return own(x)

    mlp.forward = wrapper
    assert P.fuse_dense_mlp(model_of(mlp, MLP())) == 1
    x = torch.empty(2, 3, HIDDEN, device="cuda", dtype=torch.bfloat16)
    mlp(x)
    assert seen == [1] and fused_calls == []
    again, _ = rewired()
    assert P.fuse_dense_mlp(model_of(again)) == 1


def test_transforms_run_the_modules(fake, fused_calls):
    """Forward-mode derivatives and torch.func transforms pass through the modules, which have rules for them."""
    import torch.autograd.forward_ad as fwAD
    mlp, x = rewired()
    with fwAD.dual_level():
        mlp(x)
        assert fused_calls == ["glu", "linear"]        # a level alone changes nothing
        y = mlp(fwAD.make_dual(x, torch.ones_like(x)))
        assert fwAD.unpack_dual(y).tangent.shape == x.shape
        mlp(x, residual=fwAD.make_dual(x, torch.ones_like(x)))
    y, t = torch.func.jvp(mlp, (x,), (torch.ones_like(x),))
    assert t.shape == x.shape
    assert torch.func.vmap(mlp)(x).shape == x.shape
    assert fused_calls == ["glu", "linear"]


def test_copies_and_saved_models_are_their_own():
    """A copied or saved-and-loaded MLP runs its own weights, rewired as the original."""
    import copy
    import io
    mlp = MLP(device="cpu", dtype=torch.float32)
    x = torch.randn(2, HIDDEN)
    want = mlp(x).detach()
    assert P.fuse_dense_mlp(model_of(mlp)) == 1
    file = io.BytesIO()
    torch.save(mlp, file)
    file.seek(0)
    for other in (copy.deepcopy(mlp), torch.load(file, weights_only=False)):
        assert torch.equal(other(x), want) and torch.equal(mlp(x), want)
        with torch.no_grad():
            other.down_proj.weight.zero_()
        assert not bool(other(x).any()) and torch.equal(mlp(x), want)
        assert "forward" in other.__dict__ and P.fuse_dense_mlp(model_of(other)) == 1


def test_compiled_before_any_call(built_lib, monkeypatch):
    """The first call may be a traced one: until another has loaded the C++ operators, the modules are traced."""
    from bcfft import _lib
    if not _lib.native_op():
        pytest.skip("the C++ operators are not built")
    graphs = []

    def backend(gm, inputs):
        graphs.append([str(n.target) for n in gm.graph.nodes if n.op == "call_function"])
        return gm

    with FakeTensorMode(), torch.no_grad():
        for loaded in (None, True, False):              # False: not built, or another engine library
            monkeypatch.setattr(_lib, "_native", loaded)
            torch._dynamo.reset()
            graphs.clear()
            mlp, x = rewired()
            assert torch.compile(mlp, backend=backend, fullgraph=True)(x).shape == x.shape
            ours = [g.split(".")[1] for g in graphs[0] if g.startswith("bcfft_native")]
            assert len(graphs) == 1 and ours == (["dense_glu", "dense_linear"] if loaded else []), graphs
            assert mlp(x).shape == x.shape             # FakeTensors without a compiler
