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
device, synchronise nothing and can be captured into a CUDA graph (a captured
.backward() needs leaves that no live eager graph holds, as in torch everywhere).
Gradients of gradients are refused. The checks of arguments and the autograd nodes
are in the native host module; torch.ops.gsplat_b200.codebook_fwd,
code_log_probs_fwd and so on are the same operators without autograd.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor

from .rasterize import _host


class CodeLogProbs(NamedTuple):
    log_probs: Optional[Tensor]  # [...], None without codes
    entropy: Tensor  # [...]
    top_log_probs: Tensor  # [..., top_k], largest first
    top_codes: Tensor  # [..., top_k] int32


class CodeBalance(NamedTuple):
    loss: Tensor  # []
    counts: Tensor  # [C] int32


def codebook_lookup(codebook: Tensor, codes: Tensor, weights: Optional[Tensor] = None, *, scale: float = 1.0,
                    out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """scale * codebook[codes]: codebook [C, ...], codes of any shape -> [*codes.shape, ...].
    With float32 weights of the shape [..., J] of the codes, the J rows of the last
    axis are added up with them -> [...] + codebook.shape[1:]. Empty slots add
    nothing; a result without any is zero. `out_dtype` is the codebook's or float32.

    Differentiable in codebook and weights. The codebook's rows may be strided
    (`sh[:, :9]`); its gradient sums the uses of a row in a fixed order."""
    return _host().codebook_lookup(codebook, codes, weights, scale, out_dtype)


def code_log_probs(logits: Tensor, codes: Optional[Tensor] = None, *, top_k: int = 0) -> CodeLogProbs:
    """Per row of logits [..., C]: the log probability of codes [...] (0 for an
    empty one), the entropy of softmax(logits), and the top_k most probable codes
    with their log probabilities (ties to the lower code). All float32.

    A logit of -inf is a code out of use. A row with no other has log
    probabilities -inf, entropy 0 and gradient 0. A row with NaN or +inf has NaN.
    Differentiable in logits through the three float outputs."""
    return CodeLogProbs(*_host().code_log_probs(logits, codes, top_k))


def code_balance_loss(logits: Tensor, codes: Tensor) -> CodeBalance:
    """How unevenly codes [...] or [..., J] use the codebook, as a loss on the
    logits [..., C] they were chosen from: C * sum_c f_c P_c, with f_c the share of
    code c among the codes and P_c the mean of softmax(logits)_c over the rows that
    have a code. 1 for even use, 0 without any code. `counts` [C] is how often each
    code occurs. Differentiable in logits through P; the counts are constants. A row
    without a code takes no part and gets no gradient, whatever its logits hold."""
    return CodeBalance(*_host().code_balance_loss(logits, codes))
