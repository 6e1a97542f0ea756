"""torch.library registration of the BC forward and spectra (`torch.ops.bcfft.*`).

The HIP kernels behind bcfft.ops are opaque to PyTorch's tracers; registering them as custom
ops with fake (meta) kernels lets FakeTensor / torch.export / torch.compile trace a model that
calls them, with output shapes and dtypes computed on the host from the C ABI's own sizing
(bcfft_spectra_bytes). The real kernels are bcfft.ops' (C ABI, include/bcfft.h): no CPU path,
a host tensor fails loudly as in bcfft.ops.

    torch.ops.bcfft.forward(x2d, spec, bias, block_size, out_features, algo) -> y
    torch.ops.bcfft.spectra(c, transpose_conj) -> spec
    torch.ops.bcfft.forward_glu(x2d, spec_gu, block_size, gate_features, algo) -> h
    torch.ops.bcfft.forward_mlp(x2d, spec_gu, spec_down, block_size, inter_features, mode) -> y
    torch.ops.bcfft.dense_linear(x, weight, bias, residual, activation) -> y (forward only)
    torch.ops.bcfft.dense_glu(x, w_gate, w_up, activation) -> h (forward only)
    torch.ops.bcfft.topk_logits(logits, k, temperature) -> values, indices, rest
    torch.ops.bcfft.topk_kl(logits, values, indices, rest, weight, temperature) -> loss (forward only)
    torch.ops.bcfft.topk_kl_grad(...) -> loss, dlogits
"""
from __future__ import annotations

import torch

from . import _lib, dense, distill, ops


@torch.library.custom_op("bcfft::forward", mutates_args=())
def forward(x2d: torch.Tensor, spec: torch.Tensor, bias: torch.Tensor | None, block_size: int,
            out_features: int, algo: str = "auto") -> torch.Tensor:
    """y = BC(x2d) (+ bias): bcfft.ops.forward (patch_llama_fft.py:246-271's forward)."""
    return ops.forward(x2d, spec, bias, block_size, out_features, algo=algo)


@forward.register_fake
def _forward_fake(x2d, spec, bias, block_size, out_features, algo="auto"):
    if x2d.dim() != 2:
        raise ValueError("bcfft::forward: x2d must be (N, in_features)")
    if block_size <= 0 or x2d.shape[1] % block_size or out_features % block_size:
        raise ValueError(f"bcfft::forward: features ({x2d.shape[1]}, {out_features}) not multiples of {block_size}")
    out_dtype = x2d.dtype if bias is None else torch.promote_types(x2d.dtype, bias.dtype)
    return x2d.new_empty((x2d.shape[0], out_features), dtype=out_dtype)


@torch.library.custom_op("bcfft::spectra", mutates_args=())
def spectra(c: torch.Tensor, transpose_conj: bool = False) -> torch.Tensor:
    """Packed weight spectra of c (nO, nI, b): bcfft.ops.spectra (rfft of c, :256-257)."""
    return ops.spectra(c, transpose_conj)


@spectra.register_fake
def _spectra_fake(c, transpose_conj=False):
    if c.dim() != 3:
        raise ValueError("bcfft::spectra: c must be (out_blocks, in_blocks, block_size)")
    n_out, n_in, b = c.shape
    if transpose_conj:
        n_out, n_in = n_in, n_out
    return c.new_empty((ops.spectra_numel(n_out, n_in, b),), dtype=torch.float32)


@torch.library.custom_op("bcfft::forward_glu", mutates_args=())
def forward_glu(x2d: torch.Tensor, spec_gu: torch.Tensor, block_size: int, gate_features: int,
                algo: str = "auto") -> torch.Tensor:
    """h = silu(BC_gate(x2d)) * BC_up(x2d): bcfft.ops.forward_glu (the patched LLaMA MLP's inner
    product, patch_llama_fft.py:343-394)."""
    return ops.forward_glu(x2d, spec_gu, block_size, gate_features, algo=algo)


@forward_glu.register_fake
def _forward_glu_fake(x2d, spec_gu, block_size, gate_features, algo="auto"):
    if x2d.dim() != 2 or block_size <= 0 or x2d.shape[1] % block_size or gate_features % block_size:
        raise ValueError("bcfft::forward_glu: x2d must be (N, in_features), features multiples of block_size")
    return x2d.new_empty((x2d.shape[0], gate_features))


@torch.library.custom_op("bcfft::forward_mlp", mutates_args=())
def forward_mlp(x2d: torch.Tensor, spec_gu: torch.Tensor, spec_down: torch.Tensor, block_size: int,
                inter_features: int, mode: str = "auto") -> torch.Tensor:
    """y = BC_down(silu(BC_gate(x2d)) * BC_up(x2d)): bcfft.ops.forward_mlp (SURVEY.md §8 f4;
    microbench_dense_vs_bc.py:183-188)."""
    return ops.forward_mlp(x2d, spec_gu, spec_down, block_size, inter_features, mode=mode)


@forward_mlp.register_fake
def _forward_mlp_fake(x2d, spec_gu, spec_down, block_size, inter_features, mode="auto"):
    if x2d.dim() != 2 or block_size <= 0 or x2d.shape[1] % block_size or inter_features % block_size:
        raise ValueError("bcfft::forward_mlp: x2d must be (N, hidden), features multiples of block_size")
    return x2d.new_empty(x2d.shape)


@torch.library.custom_op("bcfft::dense_linear", mutates_args=())
def dense_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None, activation: str = "none") -> torch.Tensor:
    """act(x W^T + bias) + residual: bcfft.dense.linear's forward (the projections that
    patch_llama_fft.py:343-394 leaves dense)."""
    _lib.refuse_forward_mode("bcfft::dense_linear", x, weight, bias, residual)
    with torch.no_grad():
        return dense.linear(x, weight, bias, activation=None if activation == "none" else activation, residual=residual)


@dense_linear.register_fake
def _dense_linear_fake(x, weight, bias=None, residual=None, activation="none"):
    _lib.refuse_forward_mode("bcfft::dense_linear", x, weight, bias, residual)
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError("bcfft::dense_linear: weight must be (out_features, in_features)")
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.custom_op("bcfft::dense_glu", mutates_args=())
def dense_glu(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """act(x Wg^T) * (x Wu^T): bcfft.dense.glu's forward (the dense MLP's inner product)."""
    _lib.refuse_forward_mode("bcfft::dense_glu", x, w_gate, w_up)
    with torch.no_grad():
        return dense.glu(x, w_gate, w_up, activation=None if activation == "none" else activation)


@dense_glu.register_fake
def _dense_glu_fake(x, w_gate, w_up, activation="silu"):
    _lib.refuse_forward_mode("bcfft::dense_glu", x, w_gate, w_up)
    if x.dim() < 1 or w_gate.dim() != 2 or w_gate.shape[1] != x.shape[-1] or w_up.shape != w_gate.shape:
        raise ValueError("bcfft::dense_glu: w_gate and w_up must be (out_features, in_features)")
    return x.new_empty((*x.shape[:-1], w_gate.shape[0]))


@torch.library.custom_op("bcfft::topk_logits", mutates_args=())
def topk_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A teacher's k largest logits, indices and rest: bcfft.distill.topk_logits (calibrate_bc.py:192-212)."""
    _lib.refuse_forward_mode("bcfft::topk_logits", logits)
    return distill.topk_logits(logits, k, temperature)


@topk_logits.register_fake
def _topk_logits_fake(logits, k, temperature=1.0):
    _lib.refuse_forward_mode("bcfft::topk_logits", logits)
    if logits.dim() < 1 or not 1 <= k <= logits.shape[-1]:
        raise ValueError("bcfft::topk_logits: logits must be (..., V) with 1 <= k <= V")
    lead = logits.shape[:-1]
    return (logits.new_empty((*lead, k)), logits.new_empty((*lead, k), dtype=torch.int32),
            logits.new_empty(lead, dtype=torch.float32))


@torch.library.custom_op("bcfft::topk_kl", mutates_args=())
def topk_kl(logits: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, rest: torch.Tensor | None = None,
            weight: torch.Tensor | None = None, temperature: float = 1.0) -> torch.Tensor:
    """KL per row from the teacher's top logits: bcfft.distill.topk_kl's forward (calibrate_bc.py:281-294)."""
    _lib.refuse_forward_mode("bcfft::topk_kl", logits, values, rest, weight)
    return distill.topk_kl(logits.detach(), values, indices, rest=rest, weight=weight, temperature=temperature)


@topk_kl.register_fake
def _topk_kl_fake(logits, values, indices, rest=None, weight=None, temperature=1.0):
    _lib.refuse_forward_mode("bcfft::topk_kl", logits, values, rest, weight)
    if values.shape != indices.shape or values.shape[:-1] != logits.shape[:-1]:
        raise ValueError("bcfft::topk_kl: values and indices must both be logits' leading shape + (k,)")
    return logits.new_empty(logits.shape[:-1], dtype=torch.float32)


@torch.library.custom_op("bcfft::topk_kl_grad", mutates_args=())
def topk_kl_grad(logits: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, rest: torch.Tensor | None = None,
                 weight: torch.Tensor | None = None, temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Losses and the gradient of their sum in one launch: bcfft.distill.topk_kl_grad."""
    _lib.refuse_forward_mode("bcfft::topk_kl_grad", logits, values, rest, weight)
    return distill.topk_kl_grad(logits.detach(), values, indices, rest=rest, weight=weight, temperature=temperature)


@topk_kl_grad.register_fake
def _topk_kl_grad_fake(logits, values, indices, rest=None, weight=None, temperature=1.0):
    _lib.refuse_forward_mode("bcfft::topk_kl_grad", logits, values, rest, weight)
    return (_topk_kl_fake(logits, values, indices, rest, weight, temperature),
            torch.empty(logits.shape, dtype=logits.dtype, device=logits.device))


def registered() -> bool:
    """True once the ops are visible under torch.ops.bcfft (importing this module registers them)."""
    return all(hasattr(torch.ops.bcfft, n) for n in ("forward", "spectra", "forward_glu", "forward_mlp",
                                                          "topk_logits", "topk_kl", "topk_kl_grad", "dense_linear",
                                                          "dense_glu"))


__all__ = ["forward", "spectra", "forward_glu", "forward_mlp", "topk_logits", "topk_kl", "topk_kl_grad",
           "dense_linear", "dense_glu", "registered", "_lib"]
