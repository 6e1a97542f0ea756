"""What is measured of the operators that a partly patched model runs beside its block-circulant layers.

Four operators, each with its plain form in elementary torch operations:
  teacher  a teacher's k largest logits per row, their indices and the log of the mass left over
  distill  KL divergence from those logits to a student's softmax, with the gradient of the student's logits
  linear   act(x W^T + b) + residual, forward, or forward and backward
  glu      act(x Wg^T) * (x Wu^T), forward, or forward and backward
The feature sizes are those of LLaMA-2-7B as in this repository's benchmark (hidden 4096, intermediate 11008,
vocabulary 32000); token counts are one decoded token, a 20-prompt batch, a 1700-token prefill, and 8192 tokens.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one calibration batch of 20 prompts: the teacher's last-token logits, as a model in fp32 gives them
        dict(name="teacher_20_prompts", op="teacher", n=20, v=32000, k=64, dtype="f32", temperature=2.0),
        # the teacher's cache over the tokens of a prefill batch
        dict(name="teacher_1700_tokens", op="teacher", n=1700, v=32000, k=100, dtype="bf16", temperature=1.0),
        # the last-token calibration step, one value per prompt
        dict(name="distill_20_prompts", op="distill", n=20, v=32000, k=64, dtype="f32", rest=True, weight=False,
             temperature=2.0, form="grad"),
        # every token of a ragged batch, padded rows of weight 0, through autograd
        dict(name="distill_1700_autograd", op="distill", n=1700, v=32000, k=33, dtype="f16", rest=False, weight=True,
             temperature=1.0, form="autograd"),
        # every token of a training batch, loss and gradient in one call
        dict(name="distill_8192_tokens", op="distill", n=8192, v=32000, k=100, dtype="bf16", rest=True, weight=True,
             temperature=1.0, form="grad"),
        # attention's output projection of one decoded token, added to the residual stream
        dict(name="linear_1_token", op="linear", n=1, k=4096, m=4096, dtype="bf16", bias=False, act="none",
             residual=True, train=False),
        # a 20-prompt decode step of a model in fp32
        dict(name="linear_20_f32", op="linear", n=20, k=4096, m=4096, dtype="f32", bias=True, act="none",
             residual=False, train=False),
        # the down projection of a prefill batch, added to the residual stream
        dict(name="linear_1700_down", op="linear", n=1700, k=11008, m=4096, dtype="bf16", bias=False, act="none",
             residual=True, train=False),
        # a training step of a projection with bias and activation
        dict(name="linear_2048_train", op="linear", n=2048, k=4096, m=4096, dtype="f16", bias=True, act="gelu",
             residual=True, train=True),
        # the MLP's gate and up projections: one decoded token, a long prefill, a training step of ragged length
        dict(name="glu_1_token", op="glu", n=1, k=4096, m=11008, dtype="bf16", act="silu", train=False),
        dict(name="glu_8192_tokens", op="glu", n=8192, k=4096, m=11008, dtype="bf16", act="silu", train=False),
        dict(name="glu_1700_train", op="glu", n=1700, k=4096, m=11008, dtype="bf16", act="silu", train=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _features(rng, lo, hi):
    """Mostly multiples of 32, as layers have them; any number now and then."""
    f = _log(rng, lo, hi)
    return f if rng.random() < 0.25 else max(32, f // 32 * 32)


def draw(rng):
    op = rng.choice(["teacher", "distill", "linear", "linear", "glu", "glu"])
    if op == "teacher":
        v = _log(rng, 500, 131072)
        n = _log(rng, 1, max(1, min(4096, 1700 * 32000 // v)))
        return dict(op=op, n=n, v=v, k=_log(rng, 1, 256), dtype=rng.choice(["f32", "f16", "bf16"]),
                    temperature=rng.choice([1.0, 2.0, 0.7]))
    if op == "distill":
        v = _log(rng, 500, 131072)
        n = _log(rng, 1, max(1, min(8192, 4096 * 32000 // v)))
        return dict(op=op, n=n, v=v, k=_log(rng, 1, 256), dtype=rng.choice(["f32", "f16", "bf16"]),
                    rest=rng.random() < 0.5, weight=rng.random() < 0.5, temperature=rng.choice([1.0, 2.0, 0.7]),
                    form=rng.choice(["grad", "autograd"]))
    k, m = _features(rng, 64, 11008), _features(rng, 64, 11008)
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    train = rng.random() < 0.5
    most = 8192 * 4096 * 11008 // (k * m) // (3 if train else 1) // (8 if dtype == "f32" else 1)
    n = _log(rng, 1, max(1, min(8192, most)))
    if op == "linear":
        return dict(op=op, n=n, k=k, m=m, dtype=dtype, bias=rng.random() < 0.5,
                    act=rng.choice(["none", "relu", "silu", "gelu"]), residual=rng.random() < 0.5, train=train)
    return dict(op=op, n=n, k=k, m=m, dtype=dtype, act=rng.choice(["silu", "gelu"]), train=train)


def work(case):
    e, n = _BYTES[case["dtype"]], case["n"]
    if case["op"] == "teacher":
        v, k = case["v"], case["k"]
        return {"bytes": n * v * e + n * k * (e + 4) + 4 * n, "flops": 4 * n * v}
    if case["op"] == "distill":
        v, k = case["v"], case["k"]
        rows = 4 * n * (1 + case["rest"] + case["weight"] + (case["form"] == "autograd"))
        return {"bytes": 2 * n * v * e + n * k * (e + 4) + rows, "flops": 8 * n * v}
    k, m = case["k"], case["m"]
    if case["op"] == "linear":
        outer = m * case["bias"] + n * m * (1 + case["residual"])
        b, f = n * k + m * k + outer, 2 * n * k * m
        if case["train"]:  # and dy read; dx, dw, db written
            b, f = b + n * m + n * k + m * k + m * case["bias"], 3 * f
        return {"bytes": b * e, "flops": f}
    b, f = n * k + 2 * m * k + n * m, 4 * n * k * m
    if case["train"]:
        b, f = b + n * m + n * k + 2 * m * k, 3 * f
    return {"bytes": b * e, "flops": f}


# ------------------------------------------------------------------------------------------- inputs
def _logits(g, n, v, dtype):
    """Logits as a language model gives them: a broad bell, a few tokens that stand out, and the last few
    entries, which only pad the vocabulary, masked out."""
    z = torch.randn(n, v, generator=g, device="cuda") * 2.0
    at = torch.randint(0, v, (n, 24), generator=g, device="cuda")
    z.scatter_add_(1, at, torch.randn(n, 24, generator=g, device="cuda").abs() * 5.0)
    z[:, v - v // 100:] = -math.inf
    return z.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, n = _DTYPES[case["dtype"]], case["n"]
    s = dict(case=dict(case))

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    if case["op"] == "teacher":
        s["logits"] = _logits(g, n, case["v"], dt)
        return s
    if case["op"] == "distill":
        v, k, t = case["v"], case["k"], case["temperature"]
        s["logits"] = _logits(g, n, v, dt)
        teacher = torch.where(torch.isinf(s["logits"]), s["logits"].float(),
                              0.8 * s["logits"].float() + torch.randn(n, v, generator=g, device="cuda"))
        top = torch.topk(teacher, k, dim=-1)
        s["values"], s["indices"] = top.values.to(dt), top.indices.to(torch.int32)
        s["rest"] = None
        if case["rest"]:
            s["rest"] = torch.logsumexp(teacher.scatter(1, top.indices, -math.inf) / t, dim=-1)
        s["weight"] = None
        if case["weight"]:  # every seventh row is padding
            s["weight"] = (torch.arange(n, device="cuda") % 7 != 3).float()
        if case["form"] == "autograd":
            s["upstream"] = torch.rand(n, generator=g, device="cuda") + 0.5
            s["logits"].requires_grad_(True)
        return s
    k, m = case["k"], case["m"]
    s["x"] = rand(n, k)
    s["x"][:, :: 97] *= 8  # the few loud channels of a trained model's activations
    if case["op"] == "linear":
        s["w"] = rand(m, k, scale=1.0 / math.sqrt(k))
        s["b"] = rand(m, scale=0.5) if case["bias"] else None
        s["r"] = rand(n, m) if case["residual"] else None
    else:
        s["wg"], s["wu"] = rand(m, k, scale=1.0 / math.sqrt(k)), rand(m, k, scale=1.0 / math.sqrt(k))
    if case["train"]:
        s["dy"] = rand(n, m)
        for name in ("x", "w", "b", "r", "wg", "wu"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------- the framework's calls
_package = None


def _ours():
    global _package
    if _package is None:
        path = os.path.join(_ROOT, "llama-fft_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import bcfft.dense
        import bcfft.distill
        _package = bcfft
    return _package


def _run_own(s):
    c, ours = s["case"], _ours()
    if c["op"] == "teacher":
        values, indices, rest = ours.distill.topk_logits(s["logits"], c["k"], temperature=c["temperature"])
        return {"values": values, "indices": indices, "rest": rest}
    if c["op"] == "distill":
        if c["form"] == "grad":
            loss, grad = ours.distill.topk_kl_grad(s["logits"], s["values"], s["indices"], rest=s["rest"],
                                                   weight=s["weight"], temperature=c["temperature"])
            return {"loss": loss, "dlogits": grad}
        loss = ours.distill.topk_kl(s["logits"], s["values"], s["indices"], rest=s["rest"], weight=s["weight"],
                                    temperature=c["temperature"])
        (grad,) = torch.autograd.grad(loss, s["logits"], s["upstream"])
        return {"loss": loss.detach(), "dlogits": grad}
    if c["op"] == "linear":
        act = None if c["act"] == "none" else c["act"]
        if not c["train"]:
            return {"y": ours.dense.linear(s["x"], s["w"], s["b"], activation=act, residual=s["r"])}
        y = ours.dense.linear(s["x"], s["w"], s["b"], activation=act, residual=s["r"])
        names = [q for q in ("x", "w", "b", "r") if s[q] is not None]
        grads = torch.autograd.grad(y, [s[q] for q in names], s["dy"])
        return {"y": y.detach(), **{"d" + q: d for q, d in zip(names, grads)}}
    h = ours.dense.glu(s["x"], s["wg"], s["wu"], activation=c["act"])
    if not c["train"]:
        return {"h": h}
    dx, dwg, dwu = torch.autograd.grad(h, [s["x"], s["wg"], s["wu"]], s["dy"])
    return {"h": h.detach(), "dx": dx, "dwg": dwg, "dwu": dwu}


# ------------------------------------------------------------------------------------------- the plain forms
def _act(z, act):
    """act(z) and act'(z)."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_teacher(s):
    c, z = s["case"], s["logits"].float()
    k, t = c["k"], c["temperature"]
    ordered, index = torch.sort(z, dim=-1, descending=True, stable=True)
    left = ordered[:, k:]
    top = ordered[:, :1]
    rest = (torch.log(torch.exp((left - top) / t).sum(-1)) + top[:, 0] / t)
    return {"values": ordered[:, :k].to(s["logits"].dtype), "indices": index[:, :k].to(torch.int32), "rest": rest}


def _plain_distill(s):
    """The loss is a small difference of logarithms: each row's few sums and logarithms are kept in 64 bits."""
    c, t = s["case"], s["case"]["temperature"]
    logits, index = s["logits"].detach().float(), s["indices"].long()
    teacher = s["values"].double() / t
    if s["rest"] is not None:
        teacher = torch.cat([teacher, s["rest"][:, None].double()], 1)
    teacher = teacher - teacher.amax(-1, keepdim=True)
    p = torch.exp(teacher)
    total = p.sum(-1, keepdim=True)
    p, logp = p / total, teacher - torch.log(total)
    top = logits.amax(-1, keepdim=True)
    e = torch.exp((logits - top) / t)
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    logq = (logits.gather(1, index).double() - top) / t - torch.log(total)
    grad, k = e / total.float(), index.shape[1]
    if s["rest"] is not None:
        outside = e.scatter(1, index, 0.0)
        left = outside.sum(-1, keepdim=True, dtype=torch.float64)
        logq = torch.cat([logq, torch.log(left) - torch.log(total)], 1)
        grad = grad - outside * (p[:, k:] / left).float()
    grad = grad.scatter_add(1, index, -p[:, :k].float())
    loss = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p)).sum(-1).float()
    scale = torch.full_like(loss, 1.0)
    if s["weight"] is not None:
        loss, scale = loss * s["weight"], scale * s["weight"]
    if c["form"] == "autograd":
        scale = scale * s["upstream"]
    return {"loss": loss, "dlogits": (grad * (scale / t)[:, None]).to(s["logits"].dtype)}


def _plain_linear(s):
    c, dt = s["case"], s["x"].dtype
    x, w = s["x"].detach().float(), s["w"].detach().float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    y, slope = _act(z, c["act"]) if c["act"] != "none" or c["train"] else (z, None)
    if s["r"] is not None:
        y = y + s["r"].detach().float()
    out = {"y": y.to(dt)}
    if c["train"]:
        dz = s["dy"].float() * slope
        out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
        if s["b"] is not None:
            out["db"] = dz.sum(0).to(dt)
        if s["r"] is not None:
            out["dr"] = s["dy"]
    return out


def _plain_glu(s):
    c, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].detach().float(), s["wg"].detach().float(), s["wu"].detach().float()
    g, u = x @ wg.t(), x @ wu.t()
    a, slope = _act(g, c["act"])
    out = {"h": (a * u).to(dt)}
    if c["train"]:
        dh = s["dy"].float()
        dg, du = dh * u * slope, dh * a
        out["dx"] = (dg @ wg + du @ wu).to(dt)
        out["dwg"], out["dwu"] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt)
    return out


def run(state):
    if own:
        return _run_own(state)
    plain = {"teacher": _plain_teacher, "distill": _plain_distill, "linear": _plain_linear, "glu": _plain_glu}
    return plain[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The operators' definitions in 64 bits: logarithms of sums by logsumexp, gradients by the derivative of each
    formula written out."""
    s = prepare(case, seed)
    s = {q: v.detach() if isinstance(v, torch.Tensor) else v for q, v in s.items()}
    if case["op"] == "teacher":
        z = s["logits"].double() / case["temperature"]
        index = torch.argsort(z, dim=-1, descending=True, stable=True)[:, : case["k"]]
        return {"values": s["logits"].gather(1, index).double(), "indices": index.to(torch.int32),
                "rest": torch.logsumexp(z.scatter(1, index, -math.inf), -1)}
    if case["op"] == "distill":
        return _exact_distill(case, s)
    if case["op"] == "linear":
        z = s["x"].double() @ s["w"].double().t()
        z = z if s["b"] is None else z + s["b"].double()
        a, slope = _exact_act(z, case["act"])
        y = a if s["r"] is None else a + s["r"].double()
        if not case["train"]:
            return {"y": y}
        dz = s["dy"].double() * slope
        return {"y": y, "dx": dz @ s["w"].double(), "dw": dz.t() @ s["x"].double(),
                **({} if s["b"] is None else {"db": dz.sum(0)}), **({} if s["r"] is None else {"dr": s["dy"].double()})}
    x, wg, wu = s["x"].double(), s["wg"].double(), s["wu"].double()
    u = x @ wu.t()
    a, slope = _exact_act(x @ wg.t(), case["act"])
    if not case["train"]:
        return {"h": a * u}
    dg, du = s["dy"].double() * u * slope, s["dy"].double() * a
    return {"h": a * u, "dx": dg @ wg + du @ wu, "dwg": dg.t() @ x, "dwu": du.t() @ x}


def _exact_act(z, act):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    phi = torch.special.ndtr(z)
    return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def _exact_distill(case, s):
    t, index, k = case["temperature"], s["indices"].long(), case["k"]
    logq = torch.log_softmax(s["logits"].double() / t, -1)
    entries = s["values"].double() / t
    if s["rest"] is not None:
        entries = torch.cat([entries, s["rest"].double()[:, None]], 1)
    logp = torch.log_softmax(entries, -1)
    outside = logq.scatter(1, index, -math.inf)
    terms = logq.gather(1, index)
    grad = torch.exp(logq)
    if s["rest"] is not None:
        left = torch.logsumexp(outside, -1, keepdim=True)
        terms = torch.cat([terms, left], 1)
        grad = grad - torch.exp(logp[:, k:] + outside - left)
    grad = grad.scatter_add(1, index, -torch.exp(logp[:, :k]))
    loss = (torch.exp(logp) * (logp - terms)).masked_fill(logp == -math.inf, 0.0).sum(-1)
    scale = torch.ones_like(loss) if s["weight"] is None else s["weight"].double()
    up = s["upstream"].double() if case["form"] == "autograd" else 1.0
    return {"loss": loss * scale, "dlogits": grad * (scale * up / t)[:, None]}
