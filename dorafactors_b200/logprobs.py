"""Log probabilities of given tokens from a language model's logits, native.

One pass over the logits gives, for each row, the log probability of its target
token, the logsumexp, and on request the distribution's entropy and the most
likely alternatives; one more pass gives the logits' gradient.  Neither forms
the softmax in memory.  It serves a cross-entropy loss (``-logprobs``), policy
losses with an entropy term, and scoring with top alternatives.

Values are fp32 whatever the logits' type (fp32, fp16 or bf16); the gradient is
in the logits' type, rounded once.  There is no CPU path.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native

MAX_TOP_K = 64


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns, each in the targets' shape (the top ones with a last dimension of ``top_k``)."""

    logprobs: torch.Tensor
    logsumexp: torch.Tensor
    entropy: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]


def _check(logits, targets, temperature, what: str):
    if logits.ndim < 1 or logits.shape[:-1] != targets.shape:
        raise ValueError(f"{what}: targets {tuple(targets.shape)} do not match logits {tuple(logits.shape)}")
    if logits.shape[-1] == 0:
        raise ValueError(f"{what}: the vocabulary is empty")
    if targets.dtype is not torch.int64:
        raise ValueError(f"{what}: targets must be int64, got {targets.dtype}")
    _native.require_cuda(logits, targets, what=what)
    _native.dtype_code(logits)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"{what}: temperature must be positive and finite, got {temperature}")


def _overlap(a, lda, b, ldb, rows, vocab) -> bool:
    """Whether the memory spans of two row-strided tensors of one type meet."""
    e = a.element_size()
    a0, b0 = a.data_ptr(), b.data_ptr()
    return rows > 0 and a0 < b0 + ((rows - 1) * ldb + vocab) * e and b0 < a0 + ((rows - 1) * lda + vocab) * e


def _forward(logits, targets, temperature, entropy, top_k, ignore_index):
    _check(logits, targets, temperature, "token_logprobs")
    if not 0 <= top_k <= min(MAX_TOP_K, logits.shape[-1]):
        raise ValueError(f"token_logprobs: top_k must be in 0 .. {min(MAX_TOP_K, logits.shape[-1])}, got {top_k}")
    data, rows, vocab, ld = _native.rows_of(logits)
    dev, shape = logits.device, targets.shape
    lp = torch.empty(shape, dtype=torch.float32, device=dev)
    lse = torch.empty_like(lp)
    ent = torch.empty_like(lp) if entropy else None
    top = idx = None
    if top_k:
        top = torch.empty((*shape, top_k), dtype=torch.float32, device=dev)
        idx = torch.empty((*shape, top_k), dtype=torch.int64, device=dev)
    if rows:
        _native.token_logprobs_fwd(data, ld, targets.contiguous(), ignore_index, temperature, lp, lse, ent, top_k, top,
                                   idx, rows, vocab)
    return lp, lse, ent, top, idx


def token_logprobs_backward(g_logprobs, g_entropy, g_logsumexp, logits, targets, logsumexp, entropy=None, *,
                            temperature: float = 1.0, ignore_index: int = -100, out=None) -> torch.Tensor:
    """Gradient of the logits, from the forward's ``logsumexp`` and ``entropy`` (needed
    with ``g_entropy``) and the gradients of logprobs, entropy and logsumexp (None: zero).
    ``out`` may be ``logits`` itself, which saves a tensor of their size."""
    what = "token_logprobs_backward"
    _check(logits, targets, temperature, what)
    if g_entropy is not None and entropy is None:
        raise ValueError(f"{what}: g_entropy needs the forward's entropy")
    _native.require_cuda(logits, g_logprobs, g_entropy, g_logsumexp, logsumexp, entropy, out, what=what)
    vectors = []
    for v, name in ((g_logprobs, "g_logprobs"), (g_entropy, "g_entropy"), (g_logsumexp, "g_logsumexp"),
                    (logsumexp, "logsumexp"), (entropy if g_entropy is not None else None, "entropy")):
        if v is not None:
            if v.shape != targets.shape:
                raise ValueError(f"{what}: {name} {tuple(v.shape)} does not match targets {tuple(targets.shape)}")
            v = v.float().contiguous()
        vectors.append(v)
    g_lp, g_ent, g_lse, lse, ent = vectors
    data, rows, vocab, ld = _native.rows_of(logits)
    if out is None:
        d, ldd = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device), vocab
        res = d
    else:
        if out.shape != logits.shape or out.dtype is not logits.dtype:
            raise ValueError(f"{what}: out must have the logits' shape and type")
        d, _, _, ldd = _native.rows_of(out)
        if d.data_ptr() != out.data_ptr():
            raise ValueError(f"{what}: out must hold its rows at one stride")
        if not (d.data_ptr() == data.data_ptr() and ldd == ld) and _overlap(d, ldd, data, ld, rows, vocab):
            raise ValueError(f"{what}: out overlaps the logits without being them")
        res = out
    if rows:
        _native.token_logprobs_bwd(data, ld, targets.contiguous(), ignore_index, temperature, lse, ent, g_lp, g_ent,
                                   g_lse, d, ldd, rows, vocab)
    return res


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, temperature, entropy, top_k, ignore_index):
        lp, lse, ent, top, idx = _forward(logits, targets, temperature, entropy, top_k, ignore_index)
        ctx.save_for_backward(logits, targets, lse, ent)
        ctx.temperature, ctx.ignore_index = temperature, ignore_index
        ctx.set_materialize_grads(False)
        if top_k:
            ctx.mark_non_differentiable(top, idx)
        return lp, lse, ent, top, idx

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_lse, g_ent, _top, _idx):
        logits, targets, lse, ent = ctx.saved_tensors
        if g_lp is None and g_lse is None and g_ent is None:
            return None, None, None, None, None, None
        d = token_logprobs_backward(g_lp, g_ent, g_lse, logits, targets, lse, ent, temperature=ctx.temperature,
                                    ignore_index=ctx.ignore_index)
        return d, None, None, None, None, None


def token_logprobs(logits, targets, *, temperature: float = 1.0, entropy: bool = False, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of ``targets`` [...] under ``logits`` [..., vocab] / ``temperature``.

    ``logprobs``, ``logsumexp`` and ``entropy`` are differentiable in the logits, the
    ``top_k`` (0 to 64) alternatives are not.  Alternatives are in descending order, ties
    to the lower index.  Rows whose target is ``ignore_index`` are not read: they give
    zeros (alternatives -1) and a zero gradient.  A row of -inf alone gives -inf with
    entropy and gradient 0; a row with a NaN or +inf gives NaN.  A target outside the
    vocabulary gives a NaN log probability and sets the device error word
    (``_native.device_error``).
    """
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, float(temperature), entropy, int(top_k), ignore_index))
    return TokenLogprobs(*_forward(logits, targets, float(temperature), entropy, int(top_k), ignore_index))
