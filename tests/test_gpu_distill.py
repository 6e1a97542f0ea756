"""Top-logit distillation on the GPU against a plain implementation in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, half an fp32 step):
  a term exp(x / T) = exp2(y): the argument is rounded once (|y| u), the hardware exponential is good to
  2 u. Weighted by the terms' shares, the mean of |y| is at most log2(V) <= 18. A thread adds at most 128
  terms in fp32 (128 u), the rest is fp64. log of the sum: (18 ln 2 + 2 + 128) u < 9e-6 absolute.
  rest = that + its own rounding.   loss: two such logarithms.
  gradient: q and P_rest q / q_rest each carry at most (126 ln 2 + 2 + 128 + 8) u = 1.4e-5 relative (|y| <= 126
  before an exponential is flushed), then the output's rounding, eps / 2, or half the smallest subnormal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LOG_TOL = 9e-6
NEG = -math.inf


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    import bcfft
    bcfft.load()
    return torch.device("cuda:0")


def logits_of(n, v, dt, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(n, v, generator=g) * scale
    if v >= 20:
        z[:, :: max(1, v // 10)] += 4.0
    return z.to(dt)


def teacher_oracle(z, k, t):
    z = z.double().cpu()
    order = torch.sort(z, dim=-1, descending=True, stable=True).indices
    top, left = order[..., :k], order[..., k:]
    return top, torch.logsumexp(z.gather(-1, left) / t, -1) if left.shape[-1] else torch.full(z.shape[:-1], NEG).double()


def kl_oracle(s, values, indices, rest, weight, t):
    """loss, gradient of its sum and the gradient's magnitude (sum of the absolute terms), in fp64 on the
    host, row by row, entries one by one."""
    s, values = s.double().cpu(), values.double().cpu()
    n, v = s.shape
    loss, grad, size = torch.zeros(n).double(), torch.zeros(n, v).double(), torch.zeros(n, v).double()
    for i in range(n):
        w = 1.0 if weight is None else float(weight[i])
        entries = [(float(values[i, j]) / t, int(indices[i, j])) for j in range(values.shape[1])
                   if 0 <= int(indices[i, j]) < v]
        r = NEG if rest is None else float(rest[i])
        a = torch.tensor([e for e, _ in entries] + [r]).double()
        if w == 0.0 or bool((a == NEG).all()):
            continue
        p = torch.softmax(a, 0)
        logp = torch.log_softmax(a, 0)
        at = sorted({e for _, e in entries})
        logq = torch.log_softmax(s[i] / t, 0)
        others = torch.ones(v, dtype=torch.bool)
        others[at] = False
        log_rest = torch.logsumexp(logq[others], 0) if bool(others.any()) else torch.tensor(NEG).double()
        q = torch.exp(logq)
        g, m = q.clone(), q.clone()
        total = 0.0
        for (_, e), pj, lj in zip(entries, p, logp):
            g[e] -= pj
            m[e] += pj
            if pj > 0:
                total += float(pj * (lj - logq[e]))
        if p[-1] > 0:
            total += float(p[-1] * (logp[-1] - log_rest))
            if log_rest > NEG:
                # exp(logq - log_rest); both may be near -3e38, where a double no longer holds log(count)
                share = p[-1] * torch.softmax(s[i][others] / t, 0)
                g[others] -= share
                m[others] += share
        loss[i], grad[i], size[i] = total * w, g * (w / t), m * abs(w / t)
    return loss, grad, size


def check_loss(got, want, weight=None):
    w = 1.0 if weight is None else weight.double().cpu().abs()
    got = got.double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    fine = torch.isfinite(want)
    tol = 2 * LOG_TOL * w + 2.0 ** -23 * want.abs()
    assert bool(((got - want).abs() <= tol)[fine].all()), float(((got - want).abs() - tol)[fine].max())


def check_grad(got, want, size, scale=1.0):
    eps = torch.finfo(got.dtype).eps
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-37
    got = got.double().cpu()
    tol = eps / 2 * want.abs() * scale + 1.5e-5 * size * scale + tiny
    off = (got - want * scale).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


# ------------------------------------------------------------------ the teacher's top logits
SIZES = [(1, 1, 1), (2, 7, 7), (3, 8, 3), (3, 9, 1), (5, 100, 100), (4, 1000, 64), (3, 4099, 256), (2, 5000, 1024),
         (7, 32000, 64), (2, 50257, 300), (2, 66001, 33), (1, 140000, 128)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n,v,k", SIZES)
def test_topk_logits(dev, dt, n, v, k):
    from bcfft import distill
    z = logits_of(n, v, DT[dt], seed=v + k)
    values, indices, rest = distill.topk_logits(z.to(dev), k, temperature=1.5)
    top, want = teacher_oracle(z, k, 1.5)
    assert values.dtype == z.dtype and indices.dtype == torch.int32 and rest.dtype == torch.float32
    assert torch.equal(indices.cpu().long(), top)
    assert torch.equal(values.cpu(), z.gather(-1, top))
    rest = rest.double().cpu()
    assert torch.equal(rest == NEG, want == NEG)
    fine = want > NEG
    assert bool(((rest - want).abs() <= LOG_TOL + 2.0 ** -23 * want.abs())[fine].all())


@pytest.mark.parametrize("dt", list(DT))
def test_topk_ties_and_special_values(dev, dt):
    """Rows of equal logits (more than the LDS list of candidates), two values, signed zeros, NaN, infinities."""
    from bcfft import distill
    v = 6000
    z = torch.zeros(9, v)
    z[0] = 1.25
    z[1] = torch.where(torch.arange(v) % 3 == 0, 2.0, -1.0)
    z[2, ::2] = -0.0
    z[3] = torch.linspace(-3, 3, v)
    z[3, [17, 4000]] = math.nan
    z[4] = NEG
    z[5] = NEG
    z[5, [5, 77]] = 0.5
    z[6] = -100.0
    z[6, 3000] = 300.0
    z[7, 11] = math.inf
    z[7, 12] = NEG
    z[8] = torch.where(torch.arange(v) % 5 == 0, 1.0, 1.0078125)
    z = z.to(DT[dt])
    for k in (1, 2, 40, 1000):
        values, indices, rest = distill.topk_logits(z.to(dev), k)
        top, want = teacher_oracle(z, k, 1.0)
        assert torch.equal(indices.cpu().long(), top), k
        assert torch.equal(torch.nan_to_num(values.cpu(), nan=7.0), torch.nan_to_num(z.gather(-1, top), nan=7.0))
        rest = rest.double().cpu()
        ok = ~torch.isnan(want)
        assert torch.equal(torch.isnan(rest), ~ok)
        fine = ok & torch.isfinite(want)
        assert torch.equal(rest[ok & ~fine], want[ok & ~fine])
        assert bool(((rest - want).abs() <= LOG_TOL + 2.0 ** -23 * want.abs())[fine].all())


def test_topk_strides_offsets_and_shapes(dev):
    from bcfft import distill
    base = logits_of(12, 1003, torch.bfloat16, seed=3).to(dev)
    views = [base[:, 1:], base[:, 5:900], base[::2], base.t().contiguous().t(), base.view(3, 4, 1003),
             base[:, ::3], base[:1].expand(4, 1003), base[0]]
    for z in views:
        values, indices, rest = distill.topk_logits(z, 9)
        top, want = teacher_oracle(z.cpu(), 9, 1.0)
        assert values.shape == z.shape[:-1] + (9,) and rest.shape == z.shape[:-1]
        assert torch.equal(indices.cpu().long(), top)
        assert bool(((rest.double().cpu() - want).abs() <= LOG_TOL + 2.0 ** -23 * want.abs()).all())
    values, indices, rest = distill.topk_logits(base[:0], 9)
    assert values.shape == (0, 9) and rest.shape == (0,)


# ------------------------------------------------------------------ loss and gradient
def entries_of(s, k, dt, seed):
    g = torch.Generator().manual_seed(seed)
    t = s.float() * 0.8 + torch.randn(s.shape, generator=g)
    top = torch.topk(t, k, dim=-1).indices
    return t, top, t.gather(-1, top).to(dt)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (2, 7, 7), (3, 9, 2), (4, 1000, 64), (3, 4099, 33), (3, 5000, 1024),
                                   (3, 32000, 100), (2, 66001, 20), (1, 140000, 5)])
def test_kl_and_gradient(dev, dt, with_rest, n, v, k):
    from bcfft import distill
    t = 2.0
    s = logits_of(n, v, DT[dt], seed=k)
    teacher, top, values = entries_of(s, k, DT[dt], seed=v)
    rest = torch.logsumexp(teacher.scatter(1, top, NEG).double() / t, -1).float() if with_rest else None
    weight = torch.rand(n, generator=torch.Generator().manual_seed(1)) + 0.25
    want, dwant, size = kl_oracle(s, values, top, rest, weight, t)
    args = dict(rest=None if rest is None else rest.to(dev), weight=weight.to(dev), temperature=t)
    loss, grad = distill.topk_kl_grad(s.to(dev), values.to(dev), top.to(dev), **args)
    check_loss(loss, want, weight)
    check_grad(grad, dwant, size)
    # int32 indices, loss alone, and the two-launch form through autograd
    x = s.to(dev).requires_grad_()
    assert torch.equal(distill.topk_kl(s.to(dev), values.to(dev), top.to(dev).int(), **args), loss)
    l2 = distill.topk_kl(x, values.to(dev), top.to(dev).int(), **args)
    assert torch.equal(l2.detach(), loss)
    up = torch.rand(n, generator=torch.Generator().manual_seed(2)) + 0.5
    l2.backward(up.to(dev))
    check_grad(x.grad, dwant * up[:, None].double(), size * up[:, None].double())


@pytest.mark.parametrize("dt", list(DT))
def test_kl_masks_duplicates_and_empty_rows(dev, dt):
    from bcfft import distill
    n, v, k, t = 10, 333, 6, 1.3
    s = logits_of(n, v, DT[dt], seed=9)
    _, top, values = entries_of(s, k, DT[dt], seed=10)
    top = top.clone()
    values = values.clone()
    rest = torch.randn(n)
    weight = torch.ones(n)
    s[0, 200:] = NEG                                  # padded vocabulary outside the entries
    top[0] = torch.arange(6)
    top[1, 3:] = -1                                   # padding entries
    top[2] = torch.tensor([5, 9, 5, 5, 9, 300])       # the same index several times
    top[3] = -1                                       # rest alone
    top[4], rest[4] = 4000, NEG                       # nothing at all: loss 0
    weight[5] = 0.0                                   # weight 0: logits may hold anything
    s[5] = math.nan
    values[6, 2:] = NEG                               # entries without mass
    rest[6] = NEG
    s[7, :] = -50.0                                   # the teacher's token far below / above the others
    s[7, int(top[7, 0])] = 60.0
    s[8, int(top[8, 1])] = NEG                        # mass on a masked token: loss inf
    s[9, :] = NEG                                     # only the entries are visible
    s[9, top[9]] = 1.0
    rest[9] = NEG
    top = top.to(torch.int64)
    top[1, 4] = (1 << 32) + 2                         # out of range, also where 32 bits would wrap
    want, dwant, size = kl_oracle(s, values, top, rest, weight, t)
    assert float(want[8]) == math.inf
    loss, grad = distill.topk_kl_grad(s.to(dev), values.to(dev), top.to(dev), rest=rest.to(dev),
                                      weight=weight.to(dev), temperature=t)
    check_loss(loss, want)
    check_grad(grad, dwant, size)
    assert float(loss[4]) == 0.0 and not bool(grad[4].any())
    assert float(loss[5]) == 0.0 and not bool(grad[5].any())
    x = s.to(dev).requires_grad_()
    l2 = distill.topk_kl(x, values.to(dev), top.to(dev), rest=rest.to(dev), weight=weight.to(dev), temperature=t)
    assert torch.equal(l2.detach(), loss)
    l2.sum().backward()
    check_grad(x.grad, dwant, size)


def test_rest_without_mass_left_in_the_student(dev):
    """The teacher leaves mass to other tokens, the student none: loss inf, gradient q - P at the entries."""
    from bcfft import distill
    s = torch.full((1, 40), NEG)
    s[0, :3] = torch.tensor([0.5, 0.25, -1.0])
    top = torch.tensor([[0, 1, 2]])
    values = torch.tensor([[1.0, 0.0, 0.0]])
    loss, grad = distill.topk_kl_grad(s.to(dev), values.to(dev), top.to(dev), rest=torch.zeros(1, device=dev))
    assert float(loss[0]) == math.inf
    p = torch.softmax(torch.tensor([1.0, 0.0, 0.0, 0.0]).double(), 0)[:3]
    want = torch.zeros(1, 40).double()
    want[0, :3] = torch.softmax(s[0, :3].double(), 0) - p
    check_grad(grad, want, want.abs() + 1.0)


def test_kl_nan_propagates(dev):
    from bcfft import distill
    s = logits_of(2, 500, torch.float32).to(dev)
    s[1, 3] = math.nan
    _, top, values = entries_of(torch.nan_to_num(s.cpu()), 8, torch.float32, 1)
    loss, grad = distill.topk_kl_grad(s, values.to(dev), top.to(dev))
    assert bool(torch.isfinite(loss[0])) and bool(torch.isfinite(grad[0]).all())
    assert bool(torch.isnan(loss[1])) and bool(torch.isnan(grad[1]).any())


def test_kl_equals_full_softmax_kl(dev):
    """With every token an entry, in any order, it is bc_eval.softmax_kl; through teacher_cache / distill_kl."""
    import bc_eval
    s = logits_of(5, 300, torch.float32, seed=1).to(dev)
    t = logits_of(5, 300, torch.float32, seed=2).to(dev)
    cache = bc_eval.teacher_cache(t, k=300, temperature=2.0)
    got = bc_eval.distill_kl(s, cache).double()
    want = bc_eval.softmax_kl(s.double(), t.double(), 2.0)
    assert bool(((got - want).abs() <= 2 * LOG_TOL + 2.0 ** -23 * want.abs()).all())


def test_gradient_against_differences(dev):
    """Central differences of the loss along random directions d, |d| <= 1. Loss error 2 LOG_TOL per side
    over 2 h; the third derivative of a log-sum-exp along d is at most 8 / T^3, and the loss holds two of
    them: h^2 / 6 * 16."""
    from bcfft import distill
    n, v, k, h = 4, 2000, 30, 0.05
    s = logits_of(n, v, torch.float32, seed=5)
    teacher, top, values = entries_of(s, k, torch.float32, 6)
    rest = torch.logsumexp(teacher.scatter(1, top, NEG), -1)
    a = (values.to(dev), top.to(dev))
    g = torch.Generator().manual_seed(7)
    _, grad = distill.topk_kl_grad(s.to(dev), *a, rest=rest.to(dev))
    for _ in range(5):
        d = torch.rand(n, v, generator=g) * 2 - 1
        up = distill.topk_kl((s + h * d).to(dev), *a, rest=rest.to(dev)).double()
        down = distill.topk_kl((s - h * d).to(dev), *a, rest=rest.to(dev)).double()
        slope = (grad.double() * d.to(dev).double()).sum(-1)
        # s +- h d is rounded to fp32: at most 2^-24 |s| per logit, times a gradient of at most 1 per row
        tol = 4 * LOG_TOL / (2 * h) + h * h / 6 * 16 + 2.0 ** -24 * 16 / h
        assert bool(((up - down) / (2 * h) - slope).abs().max() <= tol)


def test_noncontiguous_logits_and_upstream(dev):
    from bcfft import distill
    base = logits_of(8, 1001, torch.float16, seed=11).to(dev)
    s = base[1::2, 3:900]
    _, top, values = entries_of(s.cpu(), 7, torch.float16, 12)
    want, dwant, size = kl_oracle(s.cpu(), values, top, None, None, 1.0)
    x = base.clone().requires_grad_()
    loss = distill.topk_kl(x[1::2, 3:900], values.to(dev), top.to(dev))
    check_loss(loss, want)
    loss.sum().backward()                             # upstream: an expanded scalar
    check_grad(x.grad[1::2, 3:900], dwant, size)
    assert not bool(x.grad[::2].any()) and not bool(x.grad[:, :3].any()) and not bool(x.grad[:, 900:].any())


def test_repeatable_on_streams_and_in_graphs(dev):
    from bcfft import distill
    s = logits_of(64, 32000, torch.bfloat16, seed=21).to(dev)
    values, indices, rest = distill.topk_logits(s.flip(0), 64)
    loss, grad = distill.topk_kl_grad(s, values, indices, rest=rest)
    for _ in range(3):
        again = distill.topk_logits(s.flip(0), 64)
        assert all(torch.equal(a, b) for a, b in zip(again, (values, indices, rest)))
        l2, g2 = distill.topk_kl_grad(s, values, indices, rest=rest)
        assert torch.equal(loss, l2) and torch.equal(grad, g2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        l3, g3 = distill.topk_kl_grad(s, values, indices, rest=rest)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(loss, l3) and torch.equal(grad, g3)
    static = s.clone()
    with torch.cuda.stream(side):
        distill.topk_kl_grad(static, values, indices, rest=rest)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cv, ci, cr = distill.topk_logits(static, 64)
        gl, gg = distill.topk_kl_grad(static, values, indices, rest=rest)
    for shift in (0.0, 0.5, -0.25):
        fresh = (s.float() * (1.0 + shift)).to(s.dtype)
        static.copy_(fresh)
        graph.replay()
        el, eg = distill.topk_kl_grad(fresh, values, indices, rest=rest)
        ev, ei, er = distill.topk_logits(fresh, 64)
        torch.cuda.synchronize()
        assert torch.equal(gl, el) and torch.equal(gg, eg)
        assert torch.equal(cv, ev) and torch.equal(ci, ei) and torch.equal(cr, er)


def test_refusals(dev):
    from bcfft import distill
    s = logits_of(3, 100, torch.float32).to(dev)
    values, indices = s[:, :4].contiguous(), torch.zeros(3, 4, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="k = 0"):
        distill.topk_logits(s, 0)
    with pytest.raises(ValueError, match="k = 101"):
        distill.topk_logits(s, 101)
    with pytest.raises(ValueError, match="temperature"):
        distill.topk_logits(s, 4, temperature=0.0)
    with pytest.raises(TypeError, match="unsupported dtype"):
        distill.topk_logits(s.double(), 4)
    with pytest.raises(ValueError, match="temperature"):
        distill.topk_kl(s, values, indices, temperature=math.inf)
    with pytest.raises(ValueError, match="indices"):
        distill.topk_kl(s, values, indices[:, :3])
    with pytest.raises(TypeError, match="int32 or int64"):
        distill.topk_kl(s, values, indices.short())
    with pytest.raises(ValueError, match="rest"):
        distill.topk_kl(s, values, indices, rest=s[:2, 0])
    with pytest.raises(ValueError, match="weight is on cpu"):
        distill.topk_kl(s, values, indices, weight=torch.ones(3))
    with pytest.raises(ValueError, match="requires grad"):
        distill.topk_kl(s, values.requires_grad_(), indices)
    with pytest.raises(ValueError, match="vocabulary"):
        distill.topk_kl(torch.zeros(1, (1 << 18) + 1, device=dev), values[:1].detach(), indices[:1])


def test_ctypes_path_is_identical(dev, monkeypatch):
    """The Python / ctypes path and the C++ operators run the same kernels: equal bits."""
    from bcfft import _lib, distill
    assert _lib.native_op(), "libbcfft_torch.so not loaded"
    for shape, k, idx in (((3, 4, 501), 7, torch.int64), ((6, 32000), 64, torch.int32), ((0, 90), 5, torch.int32)):
        s = logits_of(max(1, int(torch.tensor(shape[:-1]).prod())), shape[-1], torch.float16, seed=31)
        s = s[:int(torch.tensor(shape[:-1]).prod())].reshape(shape).to(dev)
        w = torch.rand(shape[:-1], device=dev)

        def all_of():
            values, indices, rest = distill.topk_logits(s.flip(-1), k, 1.5)
            x = s.clone().requires_grad_()
            loss = distill.topk_kl(x, values, indices.to(idx), rest=rest, weight=w, temperature=1.5)
            (g,) = torch.autograd.grad(loss, x, torch.ones_like(loss) * 0.5)
            return [values, indices, rest, loss.detach(), g,
                    *distill.topk_kl_grad(s, values, indices.to(idx), rest=rest, weight=w.double(), temperature=1.5)]
        native = all_of()
        with monkeypatch.context() as mp:
            mp.setattr(_lib, "_native", False)
            other = all_of()
        assert all(p.shape == q.shape and p.dtype == q.dtype and torch.equal(p, q) for p, q in zip(native, other))


@pytest.mark.parametrize("dt", list(DT))
def test_rows_masked_by_the_lowest_value(dev, dt):
    """Masks of the type's lowest value instead of -inf: alone, beside real logits, and with -inf under them."""
    from bcfft import distill
    low = torch.finfo(DT[dt]).min
    v = 3000
    z = torch.full((5, v), low)
    z[1, :10] = torch.arange(10.0)
    z[2, 5] = 3.0
    z[2, 100:] = NEG
    z[3, 7:] = NEG
    z[4] = -z[4]                                      # and the largest value
    z[4, 9:] = 0.0
    z = z.to(DT[dt])
    for k in (1, 4, 12, 200):
        values, indices, rest = distill.topk_logits(z.to(dev), k)
        top, want = teacher_oracle(z, k, 1.0)
        assert torch.equal(indices.cpu().long(), top) and torch.equal(values.cpu(), z.gather(-1, top))
        rest = rest.double().cpu()
        fine = want.abs() < 3e38                      # (lowest + log(v) itself may not be a finite fp32)
        assert bool(((rest - want).abs() <= LOG_TOL + 2.0 ** -23 * want.abs())[fine & torch.isfinite(want)].all())
        assert torch.equal(rest == NEG, want < -3.4028235e38)
    top = torch.tensor([[0, 1, 5], [0, 1, 50], [5, 6, 7], [0, 1, 2], [20, 21, 2]])
    vals = torch.tensor([[1.0, 0.5, 0.25]]).expand(5, 3).contiguous()
    for rest in (None, torch.zeros(5)):
        want, dwant, size = kl_oracle(z, vals, top, rest, None, 1.0)
        loss, grad = distill.topk_kl_grad(z.to(dev), vals.to(dev), top.to(dev), rest=None if rest is None else rest.to(dev))
        fine = want < 1e37
        assert torch.equal(torch.isfinite(loss.cpu()) & (loss.cpu() < 1e37), fine)
        check_loss(loss[fine.to(dev)], want[fine])
        check_grad(grad, dwant, size)


def test_extreme_temperatures(dev):
    from bcfft import distill
    s = logits_of(4, 700, torch.float32, seed=41, scale=5.0)
    _, top, values = entries_of(s, 9, torch.float32, 42)
    for t in (1e-6, 1e-3, 30.0, 1e6):
        want, dwant, size = kl_oracle(s, values, top, None, None, t)
        loss, grad = distill.topk_kl_grad(s.to(dev), values.to(dev), top.to(dev), temperature=t)
        # a logit over T is rounded to fp32 before the exponential: 2^-24 of |s| / T where it counts
        extra = 4 * 2.0 ** -24 * want.abs()
        assert bool(((loss.double().cpu() - want).abs() <= 2 * LOG_TOL + 2.0 ** -23 * want.abs() + extra).all())
        check_grad(grad, dwant, size)
        v2, i2, rest = distill.topk_logits(s.to(dev), 9, t)
        at, r = teacher_oracle(s, 9, t)
        assert torch.equal(i2.cpu().long(), at)
        assert bool(((rest.double().cpu() - r).abs() <= LOG_TOL + 2.0 ** -22 * r.abs()).all())


def test_offsets_past_32_bits(dev):
    """Logits and gradients of 9000 x 262144 (2.4e9 elements): what the last rows hold."""
    from bcfft import distill
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of device memory")
    n, v, k = 9000, 1 << 18, 7
    z = torch.randn(n, v, generator=torch.Generator(device=dev).manual_seed(51), device=dev, dtype=torch.float16)
    values, indices, rest = distill.topk_logits(z, k, 2.0)
    rows = [0, n - 2, n - 1]
    top, want = teacher_oracle(z[rows], k, 2.0)
    assert torch.equal(indices[rows].cpu().long(), top)
    assert bool(((rest[rows].double().cpu() - want).abs() <= LOG_TOL + 2.0 ** -23 * want.abs()).all())
    shifted = indices.roll(1, 0)                          # another row's entries: q and P differ
    loss, grad = distill.topk_kl_grad(z, values, shifted, rest=rest, temperature=2.0)
    lk, dk, size = kl_oracle(z[rows], values[rows], shifted[rows], rest[rows], None, 2.0)
    check_loss(loss[rows], lk)
    check_grad(grad[rows], dk, size)
    zg = z.requires_grad_()
    distill.topk_kl(zg, values, shifted, rest=rest, temperature=2.0).sum().backward()
    check_grad(zg.grad[rows], dk, size)


def test_more_rows_than_one_launch(dev):
    """2^21 + 5 rows: rows behind the first launch's find their own operands."""
    from bcfft import distill
    n, v, k, t = (1 << 21) + 5, 9, 3, 1.5
    g = torch.Generator(device=dev).manual_seed(52)
    z = torch.randn(n, v, generator=g, device=dev).to(torch.float16)
    weight = torch.rand(n, generator=g, device=dev)
    values, indices, rest = distill.topk_logits(z, k, t)
    z64 = z.double()
    keys = z64 * 64 - torch.arange(v, device=dev) * 2.0 ** -20      # equal logits: lower index first
    top = keys.topk(k, dim=-1).indices
    assert torch.equal(indices.long(), top) and torch.equal(values, z.gather(-1, top))
    left = torch.ones_like(z64).scatter_(-1, top, 0.0).bool()
    r64 = torch.logsumexp((z64 / t).masked_fill(~left, NEG), -1)
    assert bool(((rest.double() - r64).abs() <= LOG_TOL + 2.0 ** -23 * r64.abs()).all())
    s = torch.randn(n, v, generator=g, device=dev)
    logq = torch.log_softmax(s.double() / t, -1)
    logp = torch.log_softmax(torch.cat([values.double() / t, rest.double()[:, None]], -1), -1)
    log_rest = torch.logsumexp(logq.masked_fill(~left, NEG), -1)
    p, q = logp.exp(), logq.exp()
    want = ((p[:, :k] * (logp[:, :k] - logq.gather(-1, top))).sum(-1) + p[:, k] * (logp[:, k] - log_rest)) * weight.double()
    share = torch.where(left, p[:, k:] * torch.exp(logq - log_rest[:, None]), 0.0).scatter_(-1, top, p[:, :k])
    f = weight.double()[:, None] / t
    dwant, size = ((q - share) * f).cpu(), ((q + share) * f).cpu()
    loss, grad = distill.topk_kl_grad(s, values, indices, rest=rest, weight=weight, temperature=t)
    check_loss(loss, want.cpu(), weight)
    check_grad(grad, dwant, size)
    sg = s.clone().requires_grad_()
    loss = distill.topk_kl(sg, values, indices.long(), rest=rest, weight=weight, temperature=t)
    loss.backward(torch.full_like(loss, 3.0))
    check_grad(sg.grad, dwant, size, 3.0)


@pytest.mark.parametrize("dt", list(DT))
def test_many_equal_terms(dev, dt):
    """Rows that are read again: each thread adds thousands of equal exponentials (of 2.5 under the bound, and of
    2.5 under the others' own maximum where the bound lies far above), whose roundings all have one sign."""
    from bcfft import distill
    v, k = (1 << 22) + 3, 8
    z = torch.full((2, v), -1.5)
    z[0, :: v // 40] = 1.0
    z[1] = -72.5
    z[1, 5] = -70.0
    z[1, 1:: v // 40] = 1.0
    z = z.to(DT[dt])
    values, indices, rest = distill.topk_logits(z.to(dev), k)
    top, want = teacher_oracle(z, k, 1.0)
    assert torch.equal(indices.cpu().long(), top) and torch.equal(values.cpu(), z.gather(-1, top))
    assert bool(((rest.double().cpu() - want).abs() <= LOG_TOL + 2.0 ** -23 * want.abs()).all())
    v = 1 << 18
    s = torch.full((2, v), -2.3)
    s[0, :: v // 40] = 0.0
    s[1] = -102.3
    s[1, 100:110] = -100.0
    s[1, :4] = 0.0
    s = s.to(DT[dt])
    top = torch.tensor([[0, 1, 7], [0, 1, 2]])
    vals, rest = torch.tensor([[1.0, 0.5, 0.25]]).expand(2, 3).contiguous(), torch.tensor([2.0, 1.0])
    want, dwant, size = kl_oracle(s, vals, top, rest, None, 1.0)
    loss, grad = distill.topk_kl_grad(s.to(dev), vals.to(dev), top.to(dev), rest=rest.to(dev))
    check_loss(loss, want)
    check_grad(grad, dwant, size)
