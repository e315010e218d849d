"""Operators for programs that score or generate with hidden states and logits of their own (no model handle):

* ``token_logprobs`` - the log probability of given tokens with the entropy and the top alternatives of every row, with its
  gradient to the logits; ``ByteNetLMTime.score_tokens`` runs it behind the model's own forward;
* ``quantize_fp8`` / ``quantize_fp8_weight`` / ``linear_fp8`` - 8-bit floating point with a power-of-two scale for each block
  of 128, and the product on it.

They run on PyTorch's current stream of the tensors' device, through ``torch.ops.evodiff_amd`` (csrc/torch_ops.cpp) over the
C ABI (``ed_token_logprobs``, ``ed_fp8_*`` in include/evodiff_hip.h).  There is no CPU path.  Outputs and workspaces come from
PyTorch's allocator, so the calls can be captured into a HIP graph.  A backward pass is captured together with its forward and
asks for its gradients with ``torch.autograd.grad``: ``.backward()`` accumulates into leaves on the stream that first used
them.  While an eager graph of the same leaf logits, or of the leaf that they are a view of, is alive, a forward with gradients
refuses to be captured.  None of them has a forward-mode derivative: dual tensors are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from . import torch_ops
from ._lib import EvoDiffHipError


class _Fp8Pair(NamedTuple):
    q: torch.Tensor
    scale: torch.Tensor


class _Fp8Values(_Fp8Pair):
    k: Optional[int] = None

    def __new__(cls, q, scale, k=None):
        pair = tuple.__new__(cls, (q, scale))
        pair.k = k
        return pair

    def _replace(self, **fields):
        return type(self)(*super()._replace(**fields), self.k)


class Fp8Rows(_Fp8Values):
    """Rows in 8 bits: a pair of ``q`` (rows, Kb * 128) float8_e4m3fn and ``scale`` (rows, Kb) float8_e8m0fnu, Kb = ceil(K / 128),
    that remembers its width ``k`` = K (None for a pair made of two tensors alone: not known, and not checked)."""


class Fp8Weight(_Fp8Values):
    """A weight in 8 bits: a pair of ``q`` (N, Kb * 128) float8_e4m3fn and ``scale`` (ceil(N / 128), Kb) float8_e8m0fnu, with its
    width ``k`` as in ``Fp8Rows``."""


class TokenLogprobs(NamedTuple):
    """Per row of the logits: ``logprob`` of the given token (None without targets), ``entropy`` in nats, and the ``top_k``
    likeliest tokens ``top_token`` (int64) with their ``top_logprob``.  fp32, shaped like the logits without classes."""
    logprob: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprob: torch.Tensor
    top_token: torch.Tensor


def _on_gpu(t):
    if not t.is_cuda:
        raise EvoDiffHipError("evodiff_amd has no CPU path: move the inputs to the GPU")


def _no_gradient(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise EvoDiffHipError(name + " has no gradient: call it under torch.no_grad() or on detached tensors")


def quantize_fp8(x: torch.Tensor) -> Fp8Rows:
    """``x`` (..., K) fp32 / bf16 / fp16 -> rows in 8 bits, a scale for 128 channels of a row (leading dimensions are
    flattened).  Rounded to nearest even; infinities and NaN become NaN.  It has no gradient, and refuses an
    ``x`` that asks for one."""
    _on_gpu(x)
    _no_gradient("quantize_fp8", x)
    return Fp8Rows(*torch_ops.load().quantize_fp8(x), x.shape[-1])


def quantize_fp8_weight(w: torch.Tensor) -> Fp8Weight:
    """``w`` (N, K) fp32 / bf16 / fp16 -> a weight in 8 bits, one scale for 128 x 128 values.  Like ``quantize_fp8`` it has no gradient
    and refuses a ``w`` that asks for one: a parameter is quantised under ``torch.no_grad()``."""
    _on_gpu(w)
    _no_gradient("quantize_fp8_weight", w)
    return Fp8Weight(*torch_ops.load().quantize_fp8_weight(w), w.shape[-1])


def linear_fp8(x: Union[torch.Tensor, Fp8Rows], weight: Fp8Weight, bias: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None, fast_sums: bool = False) -> torch.Tensor:
    """``x @ weight.T + bias`` with both operands in 8 bits and fp32 sums, rounded once.  ``x``: (..., K) fp32 / bf16 / fp16,
    quantised inside as ``quantize_fp8`` does (the results are equal bit for bit), or ``Fp8Rows`` for rows that several products
    share.  ``weight``: from ``quantize_fp8_weight``, of as many channels as ``x``.  ``bias``: fp32 (N,).  ``out_dtype``: that of ``x``
    by default (bf16 for ``Fp8Rows``).  ``fast_sums`` (16-bit outputs): sums as the 8-bit matrix instruction takes them, up to three
    times as fast on large products - of eight neighbouring products the bits under 2^-13 of the largest are dropped (4e-5 to 6e-5 in
    2-norm on ordinary data, up to 7 * 2^-13 of the terms' magnitudes, which is more than the rounding where large terms cancel).
    An operator of inference: it has no gradient, and refuses an ``x`` or ``bias`` that asks for one."""
    rows, scale, k = (x.q, x.scale, x.k) if isinstance(x, Fp8Rows) else (x, None, x.shape[-1] if x.dim() else 0)
    _on_gpu(rows)
    if k is not None and weight.k is not None and k != weight.k:
        raise EvoDiffHipError("linear_fp8: x has %d channels, the weight has %d" % (k, weight.k))
    _no_gradient("linear_fp8", rows, bias)
    return torch_ops.load().linear_fp8(rows, scale, weight.q, weight.scale, bias, out_dtype, bool(fast_sums))


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor], top_k: int = 0,
                   select: Optional[torch.Tensor] = None, n_classes: Optional[int] = None) -> TokenLogprobs:
    """The log probability of ``targets`` under ``logits`` (..., V) fp32 / bf16 / fp16, with the entropy and the ``top_k``
    alternatives (at most 32, equal values by lowest index) of every row, in one pass over the logits and fp32 sums.

    ``targets``: int64, shaped like the logits without classes, or None.  ``select``: bool or uint8 of that shape; rows where it is
    false are not read: results 0, tokens -1, gradient 0.  ``n_classes``: only the first ``n_classes`` classes count.
    -inf forbids a class; a row without any other has logprob -inf, entropy 0, alternatives at -inf and no gradient.  A row with
    NaN or +inf yields NaN, and so does a target outside [0, n_classes) for its logprob, and for the row's gradient if that logprob
    has a part in the loss.  Logits may be a view with up to two
    strided leading dimensions (``logits[:, :-1]``); others are copied first.

    Differentiable once in ``logprob``, ``entropy`` and ``top_logprob``."""
    _on_gpu(logits)
    n_classes = (logits.shape[-1] if logits.dim() else 0) if n_classes is None else int(n_classes)
    out = torch_ops.load().token_logprobs(logits, targets, select, top_k, n_classes)
    return TokenLogprobs(out[0] if targets is not None else None, *out[1:])
