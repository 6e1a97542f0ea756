"""The dense projections of a partly patched model on the matrix cores (C ABI: bcfft_dense_*).

The reference's patcher replaces the projections of the first or last k layers
(patch_llama_fft.py:343-394; one of 32 MLPs by default); the others stay nn.Linear. These are their
operators, differentiable in every operand:

    y = linear(x, weight, bias, activation="gelu", residual=r)     act(x W^T + b) + r, one kernel
    h = glu(x, w_gate, w_up, activation="silu")                    act(x Wg^T) * (x Wu^T), one kernel

patch_llama_fft.fuse_dense_mlp routes the dense MLPs of a model through them. Every function enqueues on the
current stream of x's device and does not synchronise. There is no CPU path: a host tensor raises
RuntimeError. To capture a training step into a graph, capture forward and backward together, with no eager
graph of the same parameters alive. A call that records a gradient runs eagerly (under torch.compile, in a
torch.compiler.disable region); torch.ops.bcfft.dense_linear / dense_glu carry the forward through a trace.
Dual tensors (forward-mode differentiation) are refused.
"""
from __future__ import annotations

import torch

from . import _lib

MAX_FEATURES = 1 << 20
MAX_TOKENS = 1 << 23
_LINEAR, _GLU, _LINEAR_BACKWARD, _GLU_BACKWARD = range(4)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """(..., K) -> (N, K) as the library takes it: adjacent elements, a 16-byte aligned start, and rows that
    start on 16 bytes too if K fills whole 16-byte pieces. Rows of such a stride stay where they are."""
    x = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    n, k = x.shape
    e = x.element_size()
    if (n > 1 and (not k <= x.stride(0) <= MAX_FEATURES or x.stride(0) * e % 16 and k * e % 16 == 0) or
            k > 1 and x.stride(1) != 1):
        x = x.contiguous()
    return _aligned(x)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % 16 else t


def _weight(w: torch.Tensor) -> torch.Tensor:
    return _aligned(w.detach().contiguous())


def _stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _check(what: str, x: torch.Tensor, weights, vectors, activation) -> int:
    """Shapes, dtypes and devices of a call; the activation's code."""
    _lib.require_device(x, what)
    _lib.dtype_code(x.dtype)
    if x.dim() < 1:
        raise ValueError(f"{what}: x must be (..., in_features), got a scalar")
    k = x.shape[-1]
    first = weights[0][1]
    for name, w in weights:
        if w.dim() != 2 or w.shape[1] != k or w.shape != first.shape:
            raise ValueError(f"{what}: {name} {tuple(w.shape)} must be (out_features, in_features = {k})")
    m = first.shape[0]
    if not (1 <= k <= MAX_FEATURES and 1 <= m <= MAX_FEATURES):
        raise ValueError(f"{what}: features ({k}, {m}) must lie in [1, {MAX_FEATURES}]")
    if x.numel() // k > MAX_TOKENS:
        raise ValueError(f"{what}: {x.numel() // k} rows, at most {MAX_TOKENS}")
    for name, t, shape in vectors:
        if t is not None and t.shape != shape:
            raise ValueError(f"{what}: {name} {tuple(t.shape)} must be {tuple(shape)}")
    for name, t in list(weights) + [v[:2] for v in vectors]:
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{what}: {name} is {t.dtype} but x is {x.dtype}; all operands share one dtype")
        if t is not None and t.device != x.device:
            raise ValueError(f"{what}: {name} is on {t.device} but x is on {x.device}; move it to x's device")
    return _activation(what, activation)


def _activation(what: str, activation) -> int:
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"{what}: activation {activation!r}, expected one of {list(_lib.ACTIVATIONS)}")
    return _lib.ACTIVATIONS[activation]


def _workspace(op: int, n: int, k: int, m: int, x: torch.Tensor, act: int):
    need = _lib.load().bcfft_dense_workspace_bytes(op, n, k, m, _lib.dtype_code(x.dtype), act)
    if need < 0:
        raise ValueError(f"bcfft.dense: sizes ({n}, {k}, {m}) are not served")
    return (torch.empty(need, dtype=torch.uint8, device=x.device) if need else None), need


def _linear_forward(x2d, weight, bias, residual2d, act, keep):
    n, k = x2d.shape
    m = weight.shape[0]
    y = torch.empty((n, m), dtype=x2d.dtype, device=x2d.device)
    z = torch.empty((n, m), dtype=torch.float32, device=x2d.device) if keep else None
    if n == 0:
        return y, z
    with _lib.device_guard(x2d.device):
        ws, need = _workspace(_LINEAR, n, k, m, x2d, act)
        _lib.check(_lib.load().bcfft_dense_linear(
            x2d.data_ptr(), _lib.dtype_code(x2d.dtype), n, _stride(x2d), k, m, weight.data_ptr(), _ptr(bias),
            _ptr(residual2d), 0 if residual2d is None else _stride(residual2d), act, y.data_ptr(), _ptr(z), _ptr(ws),
            need, _lib.stream_handle(x2d.device)), "bcfft_dense_linear")
    return y, z


class _Linear(torch.autograd.Function):
    """Keeps x, the weight and, where there is an activation, its input in fp32: rounded to 16 bits it
    would add its own error to dx and dw on top of dz's and theirs."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        x2d, w = _rows(x.detach()), _weight(weight)
        b = None if bias is None else bias.detach().contiguous()
        r = None if residual is None else _rows(residual.detach())
        keep = act != 0 and any(ctx.needs_input_grad[:3])
        y, z = _linear_forward(x2d, w, b, r, act, keep)
        ctx.save_for_backward(x, weight, z)
        ctx.act = act
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    @_lib.first_order
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        x2d, w, d2d = _rows(x.detach()), _weight(weight), _rows(dy)
        n, k = x2d.shape
        m = w.shape[0]
        dx = torch.empty((n, k), dtype=x.dtype, device=x.device) if need_x else None
        dw = torch.empty((m, k), dtype=x.dtype, device=x.device) if need_w else None
        db = torch.empty((m,), dtype=x.dtype, device=x.device) if need_b else None
        if n == 0:
            dw, db = (None if t is None else t.zero_() for t in (dw, db))
        elif need_x or need_w or need_b:
            with _lib.device_guard(x.device):
                ws, need = _workspace(_LINEAR_BACKWARD, n, k, m, x2d, ctx.act)
                _lib.check(_lib.load().bcfft_dense_linear_backward(
                    x2d.data_ptr(), _lib.dtype_code(x.dtype), n, _stride(x2d), k, m, w.data_ptr(), d2d.data_ptr(),
                    _stride(d2d), _ptr(z), ctx.act, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), need,
                    _lib.stream_handle(x.device)), "bcfft_dense_linear_backward")
        return None if dx is None else dx.view(x.shape), dw, db, dy if need_r else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """y = act(x weight^T + bias) + residual in one kernel, differentiable in every operand.

    x (..., in_features), weight (out_features, in_features), bias (out_features), residual (...,
    out_features), all float32, float16 or bfloat16 alike, any sizes up to 2^20 features. activation: None,
    "relu", "silu" or "gelu" (exact). fp32 accumulation, one rounding. Up to 32 rows (64 where
    it pays) run the weight-streaming kernel. The gradient of an activation's input is rounded once to the
    dtype before the two products that read it; bias gradients sum the unrounded values."""
    if _lib.native_op():                         # the same call as one C++ op (csrc/bcfft_torch_ops.cpp)
        return _lib.NATIVE_OPS["dense_linear"](x, weight, bias, residual, _activation("bcfft.dense.linear", activation))
    _lib.refuse_forward_mode("bcfft.dense.linear", x, weight, bias, residual)
    lead = x.shape[:-1]
    act = _check("bcfft.dense.linear", x, [("weight", weight)],
                 [("bias", bias, weight.shape[:1]), ("residual", residual, lead + weight.shape[:1])], activation)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act)
    b = None if bias is None else bias.detach().contiguous()
    y, _ = _linear_forward(_rows(x.detach()), _weight(weight), b,
                           None if residual is None else _rows(residual.detach()), act, False)
    return y.view(*lead, weight.shape[0])


def _glu_forward(x2d, w_gate, w_up, act, keep):
    n, k = x2d.shape
    m = w_gate.shape[0]
    h = torch.empty((n, m), dtype=x2d.dtype, device=x2d.device)
    gu = torch.empty((2, n, m), dtype=torch.float32, device=x2d.device) if keep else None
    if n == 0:
        return h, gu
    with _lib.device_guard(x2d.device):
        ws, need = _workspace(_GLU, n, k, m, x2d, act)
        _lib.check(_lib.load().bcfft_dense_glu(
            x2d.data_ptr(), _lib.dtype_code(x2d.dtype), n, _stride(x2d), k, m, w_gate.data_ptr(), w_up.data_ptr(), act,
            h.data_ptr(), _ptr(gu), _ptr(ws), need, _lib.stream_handle(x2d.device)), "bcfft_dense_glu")
    return h, gu


class _Glu(torch.autograd.Function):
    """Keeps x, both weights and g, u in fp32 (8 bytes per element of h)."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        x2d, wg, wu = _rows(x.detach()), _weight(w_gate), _weight(w_up)
        h, gu = _glu_forward(x2d, wg, wu, act, True)
        ctx.save_for_backward(x, w_gate, w_up, gu)
        ctx.act = act
        return h.view(*x.shape[:-1], wg.shape[0])

    @staticmethod
    @_lib.first_order
    def backward(ctx, dh):
        x, w_gate, w_up, gu = ctx.saved_tensors
        need_x, need_g, need_u = ctx.needs_input_grad[:3]
        x2d, wg, wu, d2d = _rows(x.detach()), _weight(w_gate), _weight(w_up), _rows(dh)
        n, k = x2d.shape
        m = wg.shape[0]
        dx = torch.empty((n, k), dtype=x.dtype, device=x.device) if need_x else None
        dw = torch.empty((2, m, k), dtype=x.dtype, device=x.device) if need_g or need_u else None
        if n == 0:
            dw = None if dw is None else dw.zero_()
        else:
            with _lib.device_guard(x.device):
                ws, need = _workspace(_GLU_BACKWARD, n, k, m, x2d, ctx.act)
                _lib.check(_lib.load().bcfft_dense_glu_backward(
                    x2d.data_ptr(), _lib.dtype_code(x.dtype), n, _stride(x2d), k, m, wg.data_ptr(), wu.data_ptr(),
                    d2d.data_ptr(), _stride(d2d), gu.data_ptr(), ctx.act, _ptr(dx), _ptr(dw), _ptr(ws), need,
                    _lib.stream_handle(x.device)), "bcfft_dense_glu_backward")
        return (None if dx is None else dx.view(x.shape), dw[0] if need_g else None, dw[1] if need_u else None, None)


def glu(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *, activation: str | None = "silu") -> torch.Tensor:
    """h = act(x w_gate^T) * (x w_up^T): both projections, the activation and the product in one kernel,
    differentiable in every operand.

    x (..., in_features), w_gate and w_up (out_features, in_features), all float32, float16 or bfloat16
    alike. activation: "silu" (LLaMA), "gelu" (exact), "relu" or None. fp32 up to h's one rounding; the
    backward rounds dg and du once to the dtype before the products that read them."""
    if _lib.native_op():
        return _lib.NATIVE_OPS["dense_glu"](x, w_gate, w_up, _activation("bcfft.dense.glu", activation))
    _lib.refuse_forward_mode("bcfft.dense.glu", x, w_gate, w_up)
    act = _check("bcfft.dense.glu", x, [("w_gate", w_gate), ("w_up", w_up)], [], activation)
    if 2 * w_gate.shape[0] > MAX_FEATURES:
        raise ValueError(f"bcfft.dense.glu: out_features = {w_gate.shape[0]}, at most {MAX_FEATURES // 2}")
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        return _Glu.apply(x, w_gate, w_up, act)
    h, _ = _glu_forward(_rows(x.detach()), _weight(w_gate), _weight(w_up), act, False)
    return h.view(*x.shape[:-1], w_gate.shape[0])
