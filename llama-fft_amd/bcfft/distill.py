"""Distillation from a teacher's top logits (C ABI: bcfft_topk_logits, bcfft_distill_topk*).

The reference calibrates a patched model by KL(teacher || student) against a cache of whole rows of
teacher logits (calibrate_bc.py:192-212, 281-294; the loss: bench_all_in_one.py:112-120). Here the cache
holds the teacher's k largest logits per row with their indices and, as `rest`, the log of the mass
outside them, and the loss and its gradient are one HIP kernel each over the student's logits:

    values, indices, rest = topk_logits(teacher_logits, k, temperature=T)
    loss = topk_kl(student_logits, values, indices, rest=rest, temperature=T)       # differentiable
    loss, dlogits = topk_kl_grad(student_logits, values, indices, rest=rest, temperature=T)

Every function enqueues on the current stream of the logits' device and does not synchronise. There is no
CPU path: a host tensor raises RuntimeError. Dual tensors (forward-mode differentiation) are refused.
"""
from __future__ import annotations

import math

import torch

from . import _lib

MAX_ENTRIES = 1024          # teacher entries per row
MAX_VOCAB = 1 << 18         # student logits per row


def _rows(logits: torch.Tensor, what: str) -> torch.Tensor:
    """(..., V) -> (N, V) with adjacent elements; rows of any stride stay where they are."""
    if logits.dim() < 1:
        raise ValueError(f"{what}: logits must be (..., vocabulary), got a scalar")
    _lib.dtype_code(logits.dtype)
    v = logits.shape[-1]
    if v == 0:
        raise ValueError(f"{what}: empty vocabulary")
    x = logits if logits.dim() == 2 else logits.reshape(-1, v)
    if x.stride(1) != 1 and v > 1 or x.shape[0] > 1 and x.stride(0) < v:
        x = x.contiguous()
    return x


def _stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _check_temperature(temperature: float, what: str) -> float:
    t = float(temperature)
    if not (math.isfinite(t) and 1e-6 <= t <= 1e6):
        raise ValueError(f"{what}: temperature must lie in [1e-6, 1e6], got {temperature}")
    return t


def topk_logits(logits: torch.Tensor, k: int, temperature: float = 1.0):
    """The k largest logits of each row: (values, indices, rest).

    logits (..., V) float32 / float16 / bfloat16. values (..., k) in logits' dtype, descending; equal
    logits come lowest index first, NaN before everything. indices (..., k) int32. rest (...) float32 =
    log(sum of exp(logit / temperature) over the logits not taken), -inf where none is left.
    1 <= k <= min(V, 1024). Not differentiable (the teacher is a constant)."""
    if _lib.native_op():                         # the same call as one C++ op (csrc/bcfft_torch_ops.cpp)
        return _lib.NATIVE_OPS["topk_logits"](logits, k, temperature)
    what = "bcfft.distill.topk_logits"
    _lib.refuse_forward_mode(what, logits)
    _lib.require_device(logits, what)
    x = _rows(logits.detach(), what)
    n, v = x.shape
    if not 1 <= k <= min(v, MAX_ENTRIES):
        raise ValueError(f"{what}: k = {k} must lie in [1, min(vocabulary = {v}, {MAX_ENTRIES})]")
    t = _check_temperature(temperature, what)
    values = torch.empty((n, k), dtype=x.dtype, device=x.device)
    indices = torch.empty((n, k), dtype=torch.int32, device=x.device)
    rest = torch.empty((n,), dtype=torch.float32, device=x.device)
    with _lib.device_guard(x.device):
        _lib.check(_lib.load().bcfft_topk_logits(x.data_ptr(), _lib.dtype_code(x.dtype), n, v, _stride(x), k, t,
                                                 values.data_ptr(), indices.data_ptr(), rest.data_ptr(),
                                                 _lib.stream_handle(x.device)), "bcfft_topk_logits")
    lead = logits.shape[:-1]
    return values.view(*lead, k), indices.view(*lead, k), rest.view(lead)


class _Operands:
    """The checked, flattened operands of one loss call, and its two launches."""

    def __init__(self, logits, values, indices, rest, weight, temperature, what):
        _lib.refuse_forward_mode(what, logits, values, rest, weight)
        _lib.require_device(logits, what)
        self.x = _rows(logits.detach(), what)
        self.n, self.v = self.x.shape
        self.t = _check_temperature(temperature, what)
        lead = logits.shape[:-1]
        if self.v > MAX_VOCAB:
            raise ValueError(f"{what}: vocabulary of {self.v}, at most {MAX_VOCAB}")
        if values.shape != indices.shape or values.dim() < 1 or values.shape[:-1] != lead:
            raise ValueError(f"{what}: values {tuple(values.shape)} and indices {tuple(indices.shape)} must both be "
                             f"{tuple(lead)} + (k,)")
        self.k = values.shape[-1]
        if not 1 <= self.k <= MAX_ENTRIES:
            raise ValueError(f"{what}: k = {self.k} entries per row, must lie in [1, {MAX_ENTRIES}]")
        _lib.dtype_code(values.dtype)
        if indices.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{what}: indices must be int32 or int64, got {indices.dtype}")
        for name, t in (("rest", rest), ("weight", weight)):
            if t is not None and (t.shape != lead or not t.is_floating_point()):
                raise ValueError(f"{what}: {name} must be floating point of shape {tuple(lead)}, got {t.dtype} "
                                 f"{tuple(t.shape)}")
        for name, t in (("values", values), ("indices", indices), ("rest", rest), ("weight", weight)):
            if t is not None and t.device != logits.device:
                raise ValueError(f"{what}: {name} is on {t.device} but logits is on {logits.device}")
            if t is not None and t.requires_grad:
                raise ValueError(f"{what}: {name} requires grad, but the teacher's side and the weights are "
                                 "constants here: detach it")
        self.values = values.reshape(self.n, self.k).contiguous()
        self.indices = indices.reshape(self.n, self.k).contiguous()
        self.rest = None if rest is None else rest.reshape(self.n).to(torch.float32).contiguous()
        self.weight = None if weight is None else weight.reshape(self.n).to(torch.float32).contiguous()

    def _head(self):
        x = self.x
        return (x.data_ptr(), _lib.dtype_code(x.dtype), self.n, self.v, _stride(x), self.values.data_ptr(),
                _lib.dtype_code(self.values.dtype), self.indices.data_ptr(), self.indices.element_size(), self.k,
                0 if self.rest is None else self.rest.data_ptr(),
                0 if self.weight is None else self.weight.data_ptr(), self.t)

    def forward(self, stats: bool, grad: bool):
        x = self.x
        loss = torch.empty((self.n,), dtype=torch.float32, device=x.device)
        st = torch.empty((self.n, 4), dtype=torch.float32, device=x.device) if stats else None
        g = torch.empty((self.n, self.v), dtype=x.dtype, device=x.device) if grad else None
        with _lib.device_guard(x.device):
            _lib.check(_lib.load().bcfft_distill_topk(*self._head(), loss.data_ptr(),
                                                      0 if st is None else st.data_ptr(),
                                                      0 if g is None else g.data_ptr(),
                                                      _lib.stream_handle(x.device)), "bcfft_distill_topk")
        return loss, st, g

    def backward(self, stats, upstream):
        x = self.x
        g = torch.empty((self.n, self.v), dtype=x.dtype, device=x.device)
        up = upstream.reshape(self.n).to(torch.float32).contiguous()
        with _lib.device_guard(x.device):
            _lib.check(_lib.load().bcfft_distill_topk_backward(*self._head(), stats.data_ptr(), up.data_ptr(),
                                                               g.data_ptr(), _lib.stream_handle(x.device)),
                       "bcfft_distill_topk_backward")
        return g


class _TopKKL(torch.autograd.Function):
    """Forward: the losses and each row's sums (16 bytes a row). Backward: one pass that reads the logits
    again and writes their gradient."""

    @staticmethod
    def forward(ctx, logits, values, indices, rest, weight, temperature):
        op = _Operands(logits, values, indices, rest, weight, temperature, "bcfft.distill.topk_kl")
        loss, stats, _ = op.forward(stats=True, grad=False)
        ctx.save_for_backward(logits, values, indices, rest, weight, stats)
        ctx.temperature = temperature
        return loss.view(logits.shape[:-1])

    @staticmethod
    @_lib.first_order
    def backward(ctx, dloss):
        logits, values, indices, rest, weight, stats = ctx.saved_tensors
        op = _Operands(logits, values, indices, rest, weight, ctx.temperature, "bcfft.distill.topk_kl")
        return op.backward(stats, dloss).view(logits.shape), None, None, None, None, None


def topk_kl(logits: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, *, rest: torch.Tensor | None = None,
            weight: torch.Tensor | None = None, temperature: float = 1.0) -> torch.Tensor:
    """KL(teacher || student) per row from the teacher's top logits, differentiable in logits.

    logits (..., V), V <= 262144; values / indices (..., k), k <= 1024: the teacher's logits (any of the
    three dtypes) and int32 / int64 token indices. An index outside [0, V) marks no entry (padding); the
    same index twice adds up. rest (...): topk_logits' log of the mass outside the entries at the same
    temperature, one more outcome "any other token"; without it the teacher is renormalised over its
    entries. weight (...): factor per row; a row of weight 0, or without any teacher mass, has loss 0 and
    gradient 0 whatever its logits hold. Returns float32 losses (...), without a factor temperature^2.

    The gradient comes in logits' dtype; teacher side and weights are constants. To capture a training
    step into a graph, capture forward and backward together."""
    if _lib.native_op():
        return _lib.NATIVE_OPS["topk_kl"](logits, values, indices, rest, weight, temperature)
    if torch.is_grad_enabled() and logits.requires_grad:
        _lib.refuse_forward_mode("bcfft.distill.topk_kl", logits, values, rest, weight)
        _lib.require_device(logits, "bcfft.distill.topk_kl")
        return _TopKKL.apply(logits, values, indices, rest, weight, temperature)
    op = _Operands(logits, values, indices, rest, weight, temperature, "bcfft.distill.topk_kl")
    return op.forward(stats=False, grad=False)[0].view(logits.shape[:-1])


def topk_kl_grad(logits: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, *,
                 rest: torch.Tensor | None = None, weight: torch.Tensor | None = None, temperature: float = 1.0):
    """(loss, dlogits) in one launch that reads the logits once: topk_kl's losses and the gradient of
    their SUM with respect to the logits, in logits' dtype, contiguous. For a mean give weight = 1 / rows.
    `logits.backward(dlogits)` carries it into the model. Same operands as topk_kl; not recorded by autograd."""
    if _lib.native_op():
        return _lib.NATIVE_OPS["topk_kl_grad"](logits, values, indices, rest, weight, temperature)
    op = _Operands(logits, values, indices, rest, weight, temperature, "bcfft.distill.topk_kl_grad")
    loss, _, g = op.forward(stats=False, grad=True)
    return loss.view(logits.shape[:-1]), g.view(logits.shape)
