"""Dense projections on the GPU against a plain implementation in 64 bits.

Tolerances, from the arithmetic, u = 2^-24 (half an fp32 step), h = eps / 2 of the dtype:
  a product summed over K terms in fp32, in any order: rounding errors of random sign add up to at most
  8 sqrt(K) u times the sum of the terms' magnitudes (eight standard deviations of K steps of u each);
  the output is rounded once: h |y|, or half a step of the smallest subnormal.
  activations: 16 u of their value and slope; an error d of their input gives at most 1.2 d (|act'|,
  |act''| <= 1.2).
  dz is rounded once to dtype where there is an activation: h |dz| per element, independent, so 8 h times
  the root of the sum of (dz w)^2 in dx."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    import bcfft
    bcfft.load()
    return torch.device("cuda:0")


def act64(z, act):
    """act(z), act'(z) in fp64."""
    if act is None:
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    phi = torch.special.ndtr(z)
    return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def rand(dev, *shape, dt, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)


def within(got, want, slack, extra=0.0):
    h = torch.finfo(got.dtype).eps / 2
    tol = h * (want.abs() + slack) + slack + TINY[got.dtype] + extra
    off = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((off <= tol).all()), f"off by {float((off - tol).max())} more than {float(tol.max())}"


def sum_slack(a, b):
    """a @ b's accumulation error: 8 sqrt(K) u times the magnitudes."""
    return 8 * math.sqrt(a.shape[-1]) * U * (a.abs() @ b.abs())


def linear64(x, w, b, r, act):
    """y and its slack; z, its slack, and the slope."""
    x, w = x.double(), w.double()
    z = x @ w.t()
    zs = sum_slack(x, w.t())
    if b is not None:
        z = z + b.double()
        zs = zs + U * z.abs()
    v, slope = act64(z, act)
    ys = 1.2 * zs + 16 * U * v.abs()
    y = v if r is None else v + r.double()
    return y, ys + U * y.abs(), z, zs, slope


def grads64(x, w, dy, slope, zs, act, dt):
    """dx, dw, db and their slacks."""
    x, w, dy = x.double(), w.double(), dy.double()
    dz = dy * slope
    err = dy.abs() * (1.2 * zs + 16 * U) if act else torch.zeros_like(dz)
    h = torch.finfo(dt).eps / 2 if act else 0.0
    tiny = TINY[dt] if act else 0.0
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    dxs = sum_slack(dz, w) + err @ w.abs() + 8 * h * torch.sqrt((dz * dz) @ (w * w)) + tiny * w.abs().sum(0)
    dws = (sum_slack(dz.t(), x) + err.t() @ x.abs() + 8 * h * torch.sqrt((dz * dz).t() @ (x * x)) +
           tiny * x.abs().sum(0))
    dbs = (8 * math.sqrt(dz.shape[0]) * U * dz.abs() + err).sum(0)
    return (dx, dxs), (dw, dws), (db, dbs)


SIZES = [(1, 1, 1), (1, 64, 16), (2, 7, 5), (3, 72, 24), (16, 264, 130), (17, 100, 40), (32, 129, 33), (33, 64, 128),
         (65, 200, 136), (130, 1000, 72), (257, 136, 264), (300, 65, 517)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n,k,m", SIZES)
def test_linear_forward(dev, dt, n, k, m):
    from bcfft import dense
    x, w = rand(dev, n, k, dt=DT[dt], seed=1), rand(dev, m, k, dt=DT[dt], seed=2, scale=k ** -0.5)
    b, r = rand(dev, m, dt=DT[dt], seed=3), rand(dev, n, m, dt=DT[dt], seed=4)
    for act, bias, res in ((None, None, None), ("silu", b, None), ("gelu", b, r), ("relu", None, r)):
        y = dense.linear(x, w, bias, activation=act, residual=res)
        want, slack, *_ = linear64(x, w, bias, res, act)
        within(y, want, slack)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n,k,m", SIZES)
def test_linear_backward(dev, dt, n, k, m):
    from bcfft import dense
    x, w = rand(dev, n, k, dt=DT[dt], seed=5), rand(dev, m, k, dt=DT[dt], seed=6, scale=k ** -0.5)
    b, r, dy = (rand(dev, *s, dt=DT[dt], seed=7 + i) for i, s in enumerate(((m,), (n, m), (n, m))))
    for act, bias, res in ((None, None, None), (None, b, r), ("gelu", b, r), ("silu", None, None), ("relu", b, None)):
        ins = [t.clone().requires_grad_() if t is not None else None for t in (x, w, bias, res)]
        y = dense.linear(ins[0], ins[1], ins[2], activation=act, residual=ins[3])
        want, slack, z, zs, slope = linear64(x, w, bias, res, act)
        within(y.detach(), want, slack)
        y.backward(dy)
        # at a kink the slope is either side's: leave out z that rounding may move across it
        if act == "relu":
            near = (z.abs() <= zs)
            assert float(near.double().mean()) < 0.01
            if bool(near.any()):
                continue
        (dx, dxs), (dw, dws), (db, dbs) = grads64(x, w, dy, slope, zs, act, DT[dt])
        within(ins[0].grad, dx, dxs)
        within(ins[1].grad, dw, dws)
        if bias is not None:
            within(ins[2].grad, db, dbs)
        if res is not None:
            assert torch.equal(ins[3].grad, dy)


def glu64(x, wg, wu, act):
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    gs, us = sum_slack(x, wg.t()), sum_slack(x, wu.t())
    v, slope = act64(g, act)
    vs = 1.2 * gs + 16 * U * v.abs()
    h = v * u
    return h, vs * u.abs() + us * v.abs() + vs * us + U * h.abs(), (g, gs, u, us, v, vs, slope)


def glu_grads64(x, wg, wu, dh, parts, dt):
    x, wg, wu, dh = x.double(), wg.double(), wu.double(), dh.double()
    g, gs, u, us, v, vs, slope = parts
    dg, du = dh * u * slope, dh * v
    eg = dh.abs() * (us * 1.2 + u.abs() * (1.2 * gs + 16 * U)) + 4 * U * dg.abs()
    eu = dh.abs() * vs + 2 * U * du.abs()
    h = torch.finfo(dt).eps / 2
    out = []
    both, weights, err = torch.cat([dg, du], 1), torch.cat([wg, wu], 0), torch.cat([eg, eu], 1) + TINY[dt]
    out.append((both @ weights, sum_slack(both, weights) + err @ weights.abs() +
                8 * h * torch.sqrt((both * both) @ (weights * weights))))
    for d, e in ((dg, eg), (du, eu)):
        out.append((d.t() @ x, sum_slack(d.t(), x) + (e + TINY[dt]).t() @ x.abs() +
                    8 * h * torch.sqrt((d * d).t() @ (x * x))))
    return out


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n,k,m", SIZES)
def test_glu(dev, dt, n, k, m):
    from bcfft import dense
    x, dh = rand(dev, n, k, dt=DT[dt], seed=11), rand(dev, n, m, dt=DT[dt], seed=12)
    wg, wu = (rand(dev, m, k, dt=DT[dt], seed=s, scale=k ** -0.5) for s in (13, 14))
    for act in ("silu", "gelu", None):
        h = dense.glu(x, wg, wu, activation=act)
        want, slack, parts = glu64(x, wg, wu, act)
        within(h, want, slack)
        ins = [t.clone().requires_grad_() for t in (x, wg, wu)]
        h2 = dense.glu(*ins, activation=act)
        assert torch.equal(h2.detach(), h)
        h2.backward(dh)
        for t, (grad, gslack) in zip(ins, glu_grads64(x, wg, wu, dh, parts, DT[dt])):
            within(t.grad, grad, gslack)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,k,m", [(4096, 136, 4096), (1700, 320, 4096), (2048, 264, 1000), (100, 4096, 4096)])
def test_large_tiles(dev, dt, n, k, m):
    """Sizes that run the larger tiles and the splits of k, forward and backward."""
    from bcfft import dense
    x, w = rand(dev, n, k, dt=DT[dt], seed=21), rand(dev, m, k, dt=DT[dt], seed=22, scale=k ** -0.5)
    wu, dy = rand(dev, m, k, dt=DT[dt], seed=23, scale=k ** -0.5), rand(dev, n, m, dt=DT[dt], seed=24)
    b = rand(dev, m, dt=DT[dt], seed=25)
    ins = [t.clone().requires_grad_() for t in (x, w, b)]
    y = dense.linear(*ins, activation="silu")
    want, slack, z, zs, slope = linear64(x, w, b, None, "silu")
    within(y.detach(), want, slack)
    y.backward(dy)
    for t, (grad, gslack) in zip(ins, grads64(x, w, dy, slope, zs, "silu", DT[dt])):
        within(t.grad, grad, gslack)
    ins = [t.clone().requires_grad_() for t in (x, w, wu)]
    h = dense.glu(*ins)
    want, slack, parts = glu64(x, w, wu, "silu")
    within(h.detach(), want, slack)
    h.backward(dy)
    for t, (grad, gslack) in zip(ins, glu_grads64(x, w, wu, dy, parts, DT[dt])):
        within(t.grad, grad, gslack)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_strides_offsets_and_shapes(dev, dt):
    """Operands at any element-aligned address, rows of a stride, leading dimensions, an expanded gradient."""
    from bcfft import dense
    base = rand(dev, 40, 301, dt=DT[dt], seed=31)
    store = rand(dev, 50 * 96 + 3, dt=DT[dt], seed=32)
    w = store[3:3 + 50 * 96].view(50, 96)                      # misaligned weight
    for x in (base[:, 5:101], base[::2, :96], base[:, :288:3], base[:, :96].view(4, 10, 96), base[:1, :96].expand(7, 96),
              base[0, :96], base[:36, :96].view(2, 18, 96).transpose(0, 1)):
        xin, win = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
        y = dense.linear(x, w, activation="silu")
        want, slack, z, zs, slope = linear64(x.reshape(-1, 96), w, None, None, "silu")
        assert y.shape == x.shape[:-1] + (50,)
        within(y.reshape(-1, 50), want, slack)
        dense.linear(xin, win, activation="silu").sum().backward()
        (dx, dxs), (dw, dws), _ = grads64(x.reshape(-1, 96), w, torch.ones_like(want), slope, zs, "silu", DT[dt])
        within(xin.grad.reshape(-1, 96), dx, dxs)
        within(win.grad, dw, dws)
        h = dense.glu(x, w, w)
        want, slack, _ = glu64(x.reshape(-1, 96), w, w, "silu")
        within(h.reshape(-1, 50), want, slack)
    r = base[:20, 10:60]                                       # a residual with a row stride
    y = dense.linear(base[:20, :96], w, residual=r)
    want, slack, *_ = linear64(base[:20, :96], w, None, r, None)
    within(y, want, slack)


@pytest.mark.parametrize("dt", list(DT))
def test_nan_and_inf_stay_in_their_rows(dev, dt):
    """Rows past an operand's end are read as repeats of the last one and the end of k as zero: nothing
    that lies there reaches another output."""
    from bcfft import dense
    for n, k, m in ((20, 100, 40), (140, 72, 150)):
        x, w = rand(dev, n, k, dt=DT[dt], seed=41), rand(dev, m, k, dt=DT[dt], seed=42)
        clean = dense.linear(x, w)
        x[n - 1, k - 1] = math.nan
        w[m - 1, 0] = math.inf
        y = dense.linear(x, w)
        assert bool(torch.isnan(y[n - 1]).all())
        assert torch.equal(y[:n - 1, :m - 1], clean[:n - 1, :m - 1])
        assert not bool(torch.isfinite(y[:, m - 1]).any())


def test_no_rows(dev):
    from bcfft import dense
    x = torch.empty(0, 64, device=dev, requires_grad=True)
    w, wu, b = (torch.randn(*s, device=dev, requires_grad=True) for s in ((32, 64), (32, 64), (32,)))
    y = dense.linear(x, w, b, activation="gelu")
    assert y.shape == (0, 32)
    y.sum().backward()
    assert x.grad.shape == (0, 64) and not bool(w.grad.any()) and not bool(b.grad.any())
    w.grad = None
    dense.glu(x, w, wu).sum().backward()
    assert not bool(w.grad.any()) and not bool(wu.grad.any())


def test_partial_gradients_and_no_grad(dev):
    from bcfft import dense
    x, w, b = rand(dev, 40, 64, dt=torch.bfloat16, seed=1), rand(dev, 48, 64, dt=torch.bfloat16, seed=2), rand(dev, 48, dt=torch.bfloat16, seed=3)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    dense.linear(*full, activation="silu").sum().backward()
    for i in range(3):
        part = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        dense.linear(*part, activation="silu").sum().backward()
        assert torch.equal(part[i].grad, full[i].grad)
        assert all(part[j].grad is None for j in range(3) if j != i)
    r = rand(dev, 40, 48, dt=torch.bfloat16, seed=4).requires_grad_()
    dense.linear(x, w, b, activation="silu", residual=r).sum().backward()
    assert torch.equal(r.grad, torch.ones_like(r))
    with torch.no_grad():
        y = dense.linear(*full)
    assert not y.requires_grad
    g = [t.clone().requires_grad_() for t in (x, w, w)]
    dense.glu(*g).sum().backward()
    for i in range(3):
        part = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, w))]
        dense.glu(*part).sum().backward()
        assert torch.equal(part[i].grad, g[i].grad)
    with pytest.raises(RuntimeError):                     # no second derivatives
        (dx,) = torch.autograd.grad(dense.linear(full[0], full[1]).sum(), full[0], create_graph=True)
        dx.sum().backward()


def test_gradient_against_differences(dev):
    """Central differences of <dy, y(x + h d)> in fp32: y's error (its slack, per element, both sides) over
    2 h, and h^2 / 6 times the third derivative along d (|act'''| <= 2, per element |dy| |d W|^3)."""
    from bcfft import dense
    n, k, m, h = 24, 40, 36, 0.02
    x, w, wu = (rand(dev, *s, dt=torch.float32, seed=51 + i, scale=0.3) for i, s in enumerate(((n, k), (m, k), (m, k))))
    dy = rand(dev, n, m, dt=torch.float32, seed=55)
    for fn in ("linear", "glu"):
        def run(v):
            return dense.linear(v, w, activation="gelu") if fn == "linear" else dense.glu(v, w, wu)
        xin = x.clone().requires_grad_()
        (dx,) = torch.autograd.grad(run(xin), xin, dy)
        d = rand(dev, n, k, dt=torch.float32, seed=56)
        d = d / d.norm()
        slope = float((dx.double() * d.double()).sum())
        up, down = (float((run(x + s * h * d).double() * dy.double()).sum()) for s in (1, -1))
        _, slack, *_ = linear64(x, w, None, None, "gelu") if fn == "linear" else glu64(x, w, wu, "silu")
        noise = 2 * float((dy.double().abs() * (slack + 2.0 ** -24)).sum()) / (2 * h)
        rounding = 2.0 ** -24 * float((x.abs().double() * dx.abs().double()).sum()) / h
        along = [(d.double() @ q.double().t()).abs() for q in (w, wu)]
        u = (x.double() @ wu.double().t()).abs() + 1
        third = (2 * along[0] ** 3) if fn == "linear" else (2 * along[0] ** 3 * u + 3 * 1.2 * along[0] ** 2 * along[1])
        bend = h * h / 6 * float((dy.double().abs() * third).sum()) * 2
        assert abs((up - down) / (2 * h) - slope) <= noise + rounding + bend


def test_repeatable_streams_and_graphs(dev):
    from bcfft import dense
    x, w, wu = (rand(dev, *s, dt=torch.bfloat16, seed=61 + i, scale=0.1) for i, s in enumerate(((200, 1024), (512, 1024), (512, 1024))))
    dh = rand(dev, 200, 512, dt=torch.bfloat16, seed=65)

    def step(v):
        ins = [t.detach().clone().requires_grad_() for t in (v, w, wu)]
        h = dense.glu(*ins)
        return (h.detach(),) + torch.autograd.grad(h, ins, dh)

    first = step(x)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step(x)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    static = x.clone()
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                    # two graphs: each its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(static)
            y = dense.linear(static, w, activation="gelu")
        graphs.append((g, out, y))
    for scale in (1.0, 0.5, -2.0):
        static.copy_(x * scale)
        for g, _, _ in graphs:
            g.replay()
        want, yw = step(x * scale), dense.linear(x * scale, w, activation="gelu")
        torch.cuda.synchronize()
        for _, out, y in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(y, yw)


def test_refusals(dev):
    from bcfft import dense
    x, w = torch.randn(3, 64, device=dev), torch.randn(32, 64, device=dev)
    with pytest.raises(ValueError, match="weight"):
        dense.linear(x, w[:, :32])
    with pytest.raises(ValueError, match="w_up"):
        dense.glu(x, w, w[:16])
    with pytest.raises(ValueError, match="bias"):
        dense.linear(x, w, torch.zeros(31, device=dev))
    with pytest.raises(ValueError, match="residual"):
        dense.linear(x, w, residual=torch.zeros(1, 32, device=dev))
    with pytest.raises(TypeError, match="one dtype"):
        dense.linear(x, w.half())
    with pytest.raises(TypeError, match="unsupported dtype"):
        dense.linear(x.double(), w.double())
    with pytest.raises(ValueError, match="activation"):
        dense.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="weight is on cpu"):
        dense.linear(x, w.cpu())
    with pytest.raises(ValueError, match="scalar"):
        dense.linear(torch.tensor(1.0, device=dev), w)


def test_ctypes_path_is_identical(dev, monkeypatch):
    """The Python / ctypes path and the C++ operators run the same kernels: equal bits, forward and backward."""
    from bcfft import _lib, dense
    assert _lib.native_op(), "libbcfft_torch.so not loaded"
    for n, k, m, dt in ((5, 72, 24, torch.float16), (200, 1000, 130, torch.bfloat16), (0, 64, 32, torch.float32), (40, 129, 33, torch.float32)):
        x, w, wu = (rand(dev, *s, dt=dt, seed=71 + i, scale=0.1) for i, s in enumerate(((n, k), (m, k), (m, k))))
        b, r, dy = (rand(dev, *s, dt=dt, seed=75 + i) for i, s in enumerate(((m,), (n, m), (n, m))))

        def both():
            out = []
            ins = [t.clone().requires_grad_() for t in (x, w, b, r)]
            y = dense.linear(ins[0], ins[1], ins[2], activation="gelu", residual=ins[3])
            out += [y.detach(), *torch.autograd.grad(y, ins, dy)]
            ins = [t.clone().requires_grad_() for t in (x, w, wu)]
            h = dense.glu(*ins)
            return out + [h.detach(), *torch.autograd.grad(h, ins, dy), dense.linear(x, w), dense.glu(x, w, wu)]
        native = both()
        with monkeypatch.context() as mp:
            mp.setattr(_lib, "_native", False)
            other = both()
        assert all(torch.equal(p, q) for p, q in zip(native, other))


def test_second_derivative_is_refused(dev):
    from bcfft import dense
    x, w, wu = (rand(dev, *s, dt=torch.float32, seed=81).requires_grad_() for s in ((4, 16), (8, 16), (8, 16)))
    for y in (dense.linear(x, w, activation="gelu"), dense.glu(x, w, wu)):
        up = torch.ones_like(y).requires_grad_()
        (dx,) = torch.autograd.grad(y, x, up, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            dx.sum().backward()


def test_offsets_past_32_bits(dev):
    """Rows of x that lie 2^20 elements apart (2.2e9 in all), and outputs, saved inputs and gradients of
    70000 x 32000 (2.2e9): what the last ones hold."""
    from bcfft import dense
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GB of device memory")
    dt = torch.bfloat16
    wide = torch.empty(2100, 1 << 20, dtype=dt, device=dev)
    wide[:, :64] = rand(dev, 2100, 64, dt=dt, seed=91)
    x, w = wide[:, :64], rand(dev, 40, 64, dt=dt, seed=92, scale=0.125)
    assert torch.equal(dense.linear(x, w), dense.linear(x.contiguous(), w))
    dy = rand(dev, 2100, 40, dt=dt, seed=93)
    xg, wg = x.detach().requires_grad_(), w.clone().requires_grad_()
    dense.linear(xg, wg, activation="silu").backward(dy)
    xc, wc = x.detach().contiguous().requires_grad_(), w.clone().requires_grad_()
    dense.linear(xc, wc, activation="silu").backward(dy)
    assert torch.equal(wg.grad, wc.grad) and torch.equal(xg.grad, xc.grad)
    del wide, x, xg

    n, k, m = 70000, 32, 32000
    x, w, wu = (rand(dev, *s, dt=dt, seed=94 + i, scale=0.2) for i, s in enumerate(((n, k), (m, k), (m, k))))
    b, r = rand(dev, m, dt=dt, seed=97), rand(dev, n, m, dt=dt, seed=98)
    y = dense.linear(x, w, b, activation="gelu", residual=r)
    rows = slice(n - 300, n)
    want, slack, *_ = linear64(x[rows], w, b, r[rows], "gelu")
    within(y[rows], want, slack)
    del y, want, slack
    ins = [t.clone().requires_grad_() for t in (x, w, wu)]
    h = dense.glu(*ins)
    g64, u64 = x[rows].double() @ w.double().t(), x[rows].double() @ wu.double().t()
    v, slope = act64(g64, "silu")
    gs, us = sum_slack(x[rows].double(), w.double().t()), sum_slack(x[rows].double(), wu.double().t())
    within(h[rows], v * u64, (1.2 * gs + 16 * U * v.abs()) * u64.abs() + v.abs() * us + U * (v * u64).abs())
    h.backward(r)                                         # r in dh's place
    d = r[rows].double()
    eps = torch.finfo(dt).eps / 2
    w64, wu64 = w.double(), wu.double()
    dg, du = d * u64 * slope, d * v
    dx = dg @ w64 + du @ wu64
    mag = sum_slack(torch.cat([dg, du], 1), torch.cat([w64, wu64], 0))
    rounding = 8 * eps * torch.sqrt((dg * dg) @ (w64 * w64) + (du * du) @ (wu64 * wu64))
    inner = (d.abs() * (us * slope.abs() + u64.abs() * (1.2 * gs + 16 * U))) @ w64.abs() + \
            (d.abs() * (1.2 * gs + 16 * U * v.abs())) @ wu64.abs()
    within(ins[0].grad[rows], dx, mag + rounding + inner)
    del dg, du, d, g64, u64, v, slope, gs, us, mag, rounding, inner
    cols = slice(m - 40, m)                               # the last output features' weight gradients
    x64, d = x.double(), r[:, cols].double()
    g64, u64 = x64 @ w64[cols].t(), x64 @ wu64[cols].t()
    v, slope = act64(g64, "silu")
    gs, us = sum_slack(x64, w64[cols].t()), sum_slack(x64, wu64[cols].t())
    dg, du = d * u64 * slope, d * v
    for got, dz, err in ((ins[1].grad, dg, d.abs() * (us * slope.abs() + u64.abs() * (1.2 * gs + 16 * U))),
                         (ins[2].grad, du, d.abs() * (1.2 * gs + 16 * U * v.abs()))):
        want = dz.t() @ x64
        slack = sum_slack(dz.t(), x64) + err.t() @ x64.abs() + 8 * eps * torch.sqrt((dz * dz).t() @ (x64 * x64))
        within(got[cols], want, slack)


def test_two_streams_at_once(dev):
    """Calls that overlap on two streams share nothing: each has its own workspace (split k, dz, packed rows)."""
    from bcfft import dense
    args = [[rand(dev, *s, dt=torch.float16, seed=101 + 7 * i + j, scale=0.1)
             for j, s in enumerate(((70, 2001), (130, 2001), (130, 2001), (70, 130)))] for i in range(2)]

    def step(x, w, wu, dh):
        ins = [t.detach().clone().requires_grad_() for t in (x, w, wu)]
        h = dense.glu(*ins, activation="gelu") + dense.linear(ins[0], ins[1], activation="silu")
        return (h.detach(),) + torch.autograd.grad(h, ins, dh)

    want = [step(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n,k,m", [(33, 129, 40), (40, 2049, 130), (48, 96, 17), (49, 1003, 64), (64, 777, 33),
                                   (64, 4096, 24), (61, 130, 9000), (65, 777, 33)])
def test_33_to_64_rows(dev, dt, n, k, m):
    """Both sides of the rule between the few-rows kernel and tiles, with rows that need packing and without."""
    from bcfft import dense
    x, w, wu = (rand(dev, *s, dt=DT[dt], seed=111 + i, scale=c) for i, (s, c) in
                enumerate((((n, k), 1.0), ((m, k), k ** -0.5), ((m, k), k ** -0.5))))
    b, r = rand(dev, m, dt=DT[dt], seed=115), rand(dev, n, m, dt=DT[dt], seed=116)
    want, slack, *_ = linear64(x, w, b, r, "gelu")
    within(dense.linear(x, w, b, activation="gelu", residual=r), want, slack)
    x64, w64, u64 = x.double(), w.double(), wu.double()
    g, u = x64 @ w64.t(), x64 @ u64.t()
    v, _ = act64(g, "silu")
    gs, us = sum_slack(x64, w64.t()), sum_slack(x64, u64.t())
    within(dense.glu(x, w, wu), v * u, (1.2 * gs + 16 * U * v.abs()) * u.abs() + v.abs() * us + U * (v * u).abs())


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n,k,m", [(1, 260, 300), (5, 4099, 16500), (31, 515, 70), (32, 4096, 513), (33, 130, 70)])
def test_few_tokens_weight_gradient(dev, dt, n, k, m):
    """Up to 32 tokens: whole and ragged blocks of 256 columns, 64 and 256 rows per workgroup."""
    from bcfft import dense
    x, w = rand(dev, n, k, dt=DT[dt], seed=121), rand(dev, m, k, dt=DT[dt], seed=122, scale=k ** -0.5).requires_grad_()
    dy = rand(dev, n, m, dt=DT[dt], seed=123)
    dense.linear(x, w).backward(dy)
    d64, x64 = dy.double(), x.double()
    within(w.grad, d64.t() @ x64, sum_slack(d64.t(), x64))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n,k,m", [(65, 64, 1040), (129, 520, 50), (300, 2008, 1100), (700, 136, 2000), (193, 4104, 4100),
                                   (1025, 72, 100)])
def test_more_than_64_rows(dev, dt, n, k, m):
    """Blocks of 64 rows of the few-rows kernel, and tiles, with ends inside them."""
    from bcfft import dense
    x, w, wu = (rand(dev, *s, dt=DT[dt], seed=131 + i, scale=c) for i, (s, c) in
                enumerate((((n, k), 1.0), ((m, k), k ** -0.5), ((m, k), k ** -0.5))))
    b, r = rand(dev, m, dt=DT[dt], seed=135), rand(dev, n, m, dt=DT[dt], seed=136)
    want, slack, *_ = linear64(x, w, b, r, "silu")
    within(dense.linear(x, w, b, activation="silu", residual=r), want, slack)
    x64, w64, u64 = x.double(), w.double(), wu.double()
    g, u = x64 @ w64.t(), x64 @ u64.t()
    v, _ = act64(g, "gelu")
    gs, us = sum_slack(x64, w64.t()), sum_slack(x64, u64.t())
    within(dense.glu(x, w, wu, activation="gelu"), v * u, (1.2 * gs + 16 * U * v.abs()) * u.abs() + v.abs() * us + U * (v * u).abs())


@pytest.mark.parametrize("n", [64 * 65535, 64 * 65535 + 1, 1 << 23])
def test_millions_of_rows(dev, n):
    """Blocks of 64 rows up to what one grid dimension holds, and past it."""
    from bcfft import dense
    x, w = rand(dev, n, 7, dt=torch.float16, seed=141), rand(dev, 5, 7, dt=torch.float16, seed=142)
    want = x.double() @ w.double().t()
    within(dense.linear(x, w), want, sum_slack(x.double(), w.double().t()))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n,k,m", SIZES)
def test_relu_gradients(dev, dt, n, k, m):
    """relu in every size: where rounding may move z across the kink, no gradient comes in (either slope times 0)."""
    from bcfft import dense
    x, w, wu = (rand(dev, *s, dt=DT[dt], seed=151 + i, scale=c) for i, (s, c) in
                enumerate((((n, k), 1.0), ((m, k), k ** -0.5), ((m, k), k ** -0.5))))
    b, dy = rand(dev, m, dt=DT[dt], seed=155), rand(dev, n, m, dt=DT[dt], seed=156)
    want, slack, z, zs, slope = linear64(x, w, b, None, "relu")
    dy0 = torch.where(z.abs() <= zs, torch.zeros_like(dy), dy)
    assert int((dy0 != dy).sum()) <= max(4, z.numel() // 100)
    ins = [t.clone().requires_grad_() for t in (x, w, b)]
    y = dense.linear(*ins, activation="relu")
    within(y.detach(), want, slack)
    y.backward(dy0)
    for t, (grad, gslack) in zip(ins, grads64(x, w, dy0, slope, zs, "relu", DT[dt])):
        within(t.grad, grad, gslack)
    want, slack, parts = glu64(x, w, wu, "relu")
    dy0 = torch.where(parts[0].abs() <= parts[1], torch.zeros_like(dy), dy)
    assert int((dy0 != dy).sum()) <= max(4, z.numel() // 100)
    ins = [t.clone().requires_grad_() for t in (x, w, wu)]
    h = dense.glu(*ins, activation="relu")
    within(h.detach(), want, slack)
    h.backward(dy0)
    for t, (grad, gslack) in zip(ins, glu_grads64(x, w, wu, dy0, parts, DT[dt])):
        within(t.grad, grad, gslack)
