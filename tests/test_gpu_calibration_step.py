"""The dense kernels and the top-logit distillation as they are used together: a calibration step of a partly
patched LLaMA (calibrate_bc.py:253-299) whose unpatched MLPs run through fuse_dense_mlp and whose loss comes
from a teacher_cache, against the same model and loss in plain torch.

Both runs share the block-circulant kernels; what differs is the dense products (fp32 sums of 256 and 512
terms in another order, a few 1e-6 relative) and the loss (1e-6). Two layers and their backward multiply
that by far less than 50: 1e-4 in the norm of each gradient."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    import bcfft
    bcfft.load()
    return torch.device("cuda:0")


def build(dev, dtype=torch.float32, layers=3):
    transformers = pytest.importorskip("transformers")
    import patch_llama_fft as P
    torch.manual_seed(0)
    cfg = transformers.LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=layers,
                                   num_attention_heads=4, num_key_value_heads=4, vocab_size=1000,
                                   max_position_embeddings=64, tie_word_embeddings=False)
    teacher = transformers.LlamaForCausalLM(cfg).eval()
    with torch.no_grad():
        for p in teacher.parameters():
            if p.dim() > 1:
                p.mul_(4.0)                            # logits that tell tokens apart
    student = copy.deepcopy(teacher)
    P.patch_mlp_with_block_circulant(student, num_layers_to_patch=1, block_size=64)
    return teacher.to(dev).to(dtype), student.to(dev).to(dtype)


def plain_kl(student, teacher, k, t):
    top = torch.topk(teacher.double(), k, dim=-1).indices
    rest = torch.ones_like(teacher).scatter_(-1, top, 0.0).bool()

    def entries(z):
        logp = torch.log_softmax(z.double() / t, -1)
        return torch.cat([logp.gather(-1, top), torch.logsumexp(logp.masked_fill(~rest, float("-inf")), -1, keepdim=True)], -1)
    p, q = entries(teacher), entries(student)
    return (p.exp() * (p - q)).sum(-1)


def test_calibration_step(dev):
    import bc_eval as E
    import patch_llama_fft as P
    teacher, student = build(dev)
    fused = copy.deepcopy(student)
    assert P.fuse_dense_mlp(fused) == 2                # layer 0 is block-circulant
    assert set(fused.state_dict()) == set(student.state_dict())
    ids = torch.randint(1, 1000, (4, 17), generator=torch.Generator().manual_seed(1)).to(dev)
    mask = torch.ones_like(ids)
    mask[1, 9:] = 0                                    # a ragged batch: padded positions weigh nothing
    with torch.no_grad():
        tl = teacher(input_ids=ids, attention_mask=mask).logits
    cache = E.teacher_cache(tl, k=20, temperature=2.0)
    got = E.distill_kl(fused(input_ids=ids, attention_mask=mask).logits, cache, weight=mask.float())
    want = plain_kl(student(input_ids=ids, attention_mask=mask).logits, tl, 20, 2.0) * mask
    assert float((got.double() - want).norm() / want.norm()) < 1e-4
    assert not bool(got[mask == 0].any())
    (got.sum() / mask.sum()).backward()
    (want.sum() / mask.sum()).backward()
    checked = 0
    for (name, a), (_, b) in zip(fused.named_parameters(), student.named_parameters()):
        assert (a.grad is None) == (b.grad is None), name
        if a.grad is not None and float(b.grad.norm()) > 0:
            assert float((a.grad - b.grad).norm() / b.grad.norm()) < 1e-4, name
            checked += 1
    assert checked >= 20


def test_fused_dense_mlp_forward(dev):
    """bf16, no gradient: prefill and single tokens, with and without the residual, against the modules in fp64.
    h is rounded once to bf16 (2^-8 at most, half a step) and y once: below 2 * 2^-8 in the norm, the inner
    sums' 2^-20 included."""
    import patch_llama_fft as P
    _, student = build(dev, torch.bfloat16)
    P.fuse_dense_mlp(student)
    mlp = student.model.layers[2].mlp
    wide = copy.deepcopy(mlp).double()
    wide.__dict__.pop("forward", None)
    for n in (1, 5, 200):
        x = torch.randn(2, n, 256, device=dev).to(torch.bfloat16)
        with torch.no_grad():
            want = wide.down_proj(torch.nn.functional.silu(wide.gate_proj(x.double())) * wide.up_proj(x.double()))
            y = mlp(x)
            assert y.shape == x.shape and y.dtype == x.dtype
            assert float((y.double() - want).norm() / want.norm()) < 2 * 2.0 ** -8
            z = mlp(x, residual=x)
            want = want + x.double()
            assert float((z.double() - want).norm() / want.norm()) < 2 * 2.0 ** -8


def test_fused_dense_mlp_other_inputs(dev):
    """Host tensors and other dtypes run the modules' own forward; layers that do not fit are left alone."""
    import patch_llama_fft as P
    teacher, _ = build(dev)
    host = copy.deepcopy(teacher).cpu()
    assert P.fuse_dense_mlp(host) == 3
    x = torch.randn(2, 3, 256)
    want = host.model.layers[0].mlp.down_proj(torch.nn.functional.silu(host.model.layers[0].mlp.gate_proj(x)) *
                                              host.model.layers[0].mlp.up_proj(x))
    assert torch.equal(host.model.layers[0].mlp(x), want)
    assert torch.equal(host.model.layers[0].mlp(x, residual=x), want + x)
    biased = copy.deepcopy(teacher)
    biased.model.layers[1].mlp.gate_proj = torch.nn.Linear(256, 512, bias=True).to(dev)
    biased.model.layers[2].mlp.act_fn = torch.nn.GELU()
    assert P.fuse_dense_mlp(biased) == 1
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        assert P.fuse_dense_mlp(teacher) == 3
        y = teacher.model.layers[0].mlp(torch.randn(2, 3, 256, device=dev))
    assert y.dtype == torch.bfloat16                   # autocast's own products


def test_fused_dense_mlp_hooks_and_replaced_modules(dev):
    """A projection with a hook, or replaced after the call, is called as the module it is."""
    import patch_llama_fft as P
    teacher, _ = build(dev)
    assert P.fuse_dense_mlp(teacher) == 3
    mlp = teacher.model.layers[0].mlp
    x = torch.randn(2, 3, 256, device=dev)
    with torch.no_grad():
        want = mlp(x)
    seen = []
    hook = mlp.up_proj.register_forward_hook(lambda m, i, o: seen.append(o.shape))
    y = mlp(x).detach()
    assert seen == [(2, 3, 512)]
    assert float((y - want).norm() / want.norm()) < 1e-4
    hook.remove()
    assert torch.equal(mlp(x).detach(), want) and len(seen) == 1
    mlp.down_proj = torch.nn.Sequential(mlp.down_proj, torch.nn.Tanh())
    assert float((mlp(x).detach() - want.tanh()).abs().max()) < 1e-4
    mlp.gate_proj = torch.nn.Linear(256, 512, bias=True).to(dev)
    assert mlp(x).shape == x.shape
