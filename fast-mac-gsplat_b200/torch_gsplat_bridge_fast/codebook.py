"""Attributes shared through a codebook, differentiable.

Not part of the reference API, which keeps every attribute per Gaussian. A
compressed scene keeps a codebook of C attribute rows (spherical-harmonic
coefficients, say) and a code per Gaussian, or a few weighted codes. The codes
are learned from assignment logits [G, C]:

    p = code_log_probs(logits, top_k=4)                       # best codes and their log probabilities
    w = torch.softmax(p.top_log_probs, -1)
    colors = spherical_harmonics_colors(codebook, means3d, c2w, codes=p.top_codes, code_weights=w)
    image = rasterize_pinhole_gaussians(means3d, scales, quats, opacities, colors, ...)
    loss = ... + 1e-3 * p.entropy.mean() + 1e-2 * code_balance_loss(logits, p.top_codes).loss

Codebooks and logits are float32, bfloat16 or float16; sums are float32 and
rounded once, and every result is the same from call to call. Codes are int32 or
int64. A negative code is an empty slot; a code of C or more is taken as empty
and raises RuntimeError from the next call of this module or from
check_device_errors(). All calls run on the current stream of the tensors'
device, synchronise nothing and can be captured into a CUDA graph. Gradients of
gradients are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _native as N
from .rasterize import _ops

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_INTS = (torch.int32, torch.int64)


class CodeLogProbs(NamedTuple):
    log_probs: Optional[Tensor]  # [...], None without codes
    entropy: Tensor  # [...]
    top_log_probs: Tensor  # [..., top_k], largest first
    top_codes: Tensor  # [..., top_k] int32


class CodeBalance(NamedTuple):
    loss: Tensor  # []
    counts: Tensor  # [C] int32


class _Lookup(torch.autograd.Function):
    """gsplat_b200::codebook_fwd / codebook_bwd."""

    @staticmethod
    def forward(ctx, codebook, codes, weights, scale, out_dtype):
        ctx.save_for_backward(codebook, codes, weights)
        ctx.scale = scale
        return _ops().codebook_fwd(codebook, codes, weights, scale, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_out):
        codebook, codes, weights = ctx.saved_tensors
        need = ctx.needs_input_grad
        g_codebook, g_weights = _ops().codebook_bwd(g_out, codebook, codes, weights, ctx.scale, bool(need[0]),
                                                    bool(need[2]))
        return g_codebook, None, g_weights, None, None


class _LogProbs(torch.autograd.Function):
    """gsplat_b200::code_log_probs_fwd / code_log_probs_bwd."""

    @staticmethod
    def forward(ctx, logits, codes, top_k):
        log_probs, entropy, top_log_probs, top_codes, stats = _ops().code_log_probs_fwd(logits, codes, top_k, True)
        ctx.save_for_backward(logits, codes, top_codes, stats)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_codes)
        return (log_probs if codes is not None else None), entropy, top_log_probs, top_codes

    @staticmethod
    @once_differentiable
    def backward(ctx, g_log_probs, g_entropy, g_top, _g_codes):
        if g_log_probs is None and g_entropy is None and g_top is None:
            return None, None, None
        logits, codes, top_codes, stats = ctx.saved_tensors
        return _ops().code_log_probs_bwd(g_log_probs, g_entropy, g_top, logits, codes, top_codes, stats), None, None


class _Balance(torch.autograd.Function):
    """gsplat_b200::code_balance_fwd / code_balance_bwd."""

    @staticmethod
    def forward(ctx, logits, codes):
        loss, counts, stats, state = _ops().code_balance_fwd(logits, codes, True)
        ctx.save_for_backward(logits, stats, state)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, g_loss, _g_counts):
        if g_loss is None:
            return None, None
        return _ops().code_balance_bwd(g_loss, *ctx.saved_tensors), None


def _check(name: str, t: Tensor, codes: Optional[Tensor]) -> None:
    if t.dtype not in _FLOATS:
        raise ValueError(f"{name} must be float32, bfloat16 or float16")
    if codes is not None and codes.dtype not in _INTS:
        raise ValueError("codes must be int32 or int64")
    if not t.is_cuda or (codes is not None and codes.device != t.device):
        raise ValueError(f"{name} and codes must be on the same CUDA device")


def codebook_lookup(codebook: Tensor, codes: Tensor, weights: Optional[Tensor] = None, *, scale: float = 1.0,
                    out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """scale * codebook[codes]: codebook [C, ...], codes of any shape -> [*codes.shape, ...].
    With float32 weights of the shape [..., J] of the codes, the J rows of the last
    axis are added up with them -> [...] + codebook.shape[1:]. Empty slots add
    nothing; a result without any is zero. `out_dtype` is the codebook's or float32.

    Differentiable in codebook and weights. The codebook's rows may be strided
    (`sh[:, :9]`); its gradient sums the uses of a row in a fixed order."""
    if codebook.ndim < 1 or codebook.numel() == 0:
        raise ValueError("codebook must have shape [C, ...] with at least one row and value")
    if weights is not None:
        if codes.ndim < 1 or weights.shape != codes.shape or codes.shape[-1] < 1:
            raise ValueError("weights must have the shape [..., J] of codes")
        if weights.dtype != torch.float32:
            raise ValueError("weights must be float32")
        if weights.device != codebook.device:
            raise ValueError("weights and codebook must be on the same CUDA device")
    if out_dtype is None:
        out_dtype = codebook.dtype
    elif out_dtype != codebook.dtype and out_dtype != torch.float32:
        raise ValueError("out_dtype must be the codebook's or float32")
    _check("codebook", codebook, codes)
    if torch.is_grad_enabled() and (codebook.requires_grad or (weights is not None and weights.requires_grad)):
        return _Lookup.apply(codebook, codes, weights, float(scale), out_dtype)
    return _ops().codebook_fwd(codebook, codes, weights, float(scale), out_dtype)


def code_log_probs(logits: Tensor, codes: Optional[Tensor] = None, *, top_k: int = 0) -> CodeLogProbs:
    """Per row of logits [..., C]: the log probability of codes [...] (0 for an
    empty one), the entropy of softmax(logits), and the top_k most probable codes
    with their log probabilities (ties to the lower code). All float32.

    A logit of -inf is a code out of use. A row with no other has log
    probabilities -inf, entropy 0 and gradient 0. A row with NaN or +inf has NaN.
    Differentiable in logits through the three float outputs."""
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must have shape [..., C] with at least one code")
    if codes is not None and codes.shape != logits.shape[:-1]:
        raise ValueError("codes must have the shape [...] of logits [..., C]")
    top_k = int(top_k)
    if not 0 <= top_k <= min(N.GSB_CODE_MAX_TOP, logits.shape[-1]):
        raise ValueError(f"top_k must be between 0 and min({N.GSB_CODE_MAX_TOP}, C); got {top_k}")
    _check("logits", logits, codes)
    if torch.is_grad_enabled() and logits.requires_grad:
        return CodeLogProbs(*_LogProbs.apply(logits, codes, top_k))
    log_probs, entropy, top_log_probs, top_codes, _ = _ops().code_log_probs_fwd(logits, codes, top_k, False)
    return CodeLogProbs(log_probs if codes is not None else None, entropy, top_log_probs, top_codes)


def code_balance_loss(logits: Tensor, codes: Tensor) -> CodeBalance:
    """How unevenly codes [...] or [..., J] use the codebook, as a loss on the
    logits [..., C] they were chosen from: C * sum_c f_c P_c, with f_c the share of
    code c among the codes and P_c the mean of softmax(logits)_c over the rows that
    have a code. 1 for even use, 0 without any code. `counts` [C] is how often each
    code occurs. Differentiable in logits through P; the counts are constants."""
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must have shape [..., C] with at least one code")
    lead = logits.shape[:-1]
    if codes.shape != lead and (codes.ndim != logits.ndim or codes.shape[:-1] != lead or codes.shape[-1] < 1):
        raise ValueError("codes must have the shape [...] or [..., J] of logits [..., C]")
    _check("logits", logits, codes)
    if torch.is_grad_enabled() and logits.requires_grad:
        return CodeBalance(*_Balance.apply(logits, codes))
    loss, counts, _, _ = _ops().code_balance_fwd(logits, codes, False)
    return CodeBalance(loss, counts)
