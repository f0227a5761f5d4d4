"""Log probabilities of given tokens, with the entropy of every position and its most likely alternatives.

What scoring, served log probabilities and policy gradients need from logits, without the ``[T, V]`` log softmax: one
pass over the logits forward, one pass backward, both hand-written kernels for bf16, fp16 and fp32 (the reference has
no counterpart; its losses go through ``F.log_softmax``, lm_engine/model_wrapper/distillation.py:132-139).
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib

MAX_TOP_K = 128
KERNEL_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


class TokenLogprobs(NamedTuple):
    """``logprobs`` is ``None`` without tokens, ``top_logprobs`` and ``top_ids`` with ``top_k = 0``."""

    logprobs: torch.Tensor | None
    entropy: torch.Tensor
    top_logprobs: torch.Tensor | None
    top_ids: torch.Tensor | None


def token_logprobs_reference(logits: torch.Tensor, tokens: torch.Tensor | None = None, top_k: int = 0, temperature=1.0,
                             ignore_index: int = -100) -> TokenLogprobs:
    x = logits if logits.dtype == torch.float64 else logits.float()
    logp = torch.log_softmax(x / temperature, -1)
    picked = top = ids = None
    if tokens is not None:
        tokens = tokens.long()          # a narrow type would take the vocabulary and ignore_index modulo its range
        inside = (tokens >= 0) & (tokens < x.size(-1))
        at = torch.where(inside, tokens, 0)
        picked = torch.where(inside, logp.gather(-1, at[..., None])[..., 0], float("nan"))
        picked = torch.where(tokens == ignore_index, 0.0, picked)
    p = logp.exp()
    entropy = -(p * logp.masked_fill(p == 0, 0.0)).sum(-1)
    if top_k:
        ids = x.detach().sort(dim=-1, descending=True, stable=True).indices[..., :top_k].contiguous()
        top = logp.gather(-1, ids)
    return TokenLogprobs(picked, entropy, top, ids)


def logit_rows(x: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """``(x, inner, ld_inner, ld_outer)``: row ``r`` of ``x`` read as ``[rows, V]`` starts at
    ``(r // inner) * ld_outer + (r % inner) * ld_inner`` elements.  Copied only where no two strides say where its rows
    are, or the vocabulary is not dense."""
    V = x.shape[-1]
    if x.is_contiguous():
        return x, x.numel() // V or 1, V, 0
    levels: list[tuple[int, int]] = []          # (size, stride) from the inside, dimensions of size 1 left out
    for d in range(x.dim() - 2, -1, -1):
        size, stride = x.size(d), x.stride(d)
        if size == 1:
            continue
        if levels and stride == levels[-1][0] * levels[-1][1]:
            levels[-1] = (levels[-1][0] * size, levels[-1][1])
        else:
            levels.append((size, stride))
    if len(levels) > 2 or (V > 1 and x.stride(-1) != 1):
        x = x.contiguous()
        return x, max(x.numel() // V, 1), V, 0
    (inner, ld_inner), (_, ld_outer) = (levels + [(1, 0), (1, 0)])[:2]
    return x, inner, ld_inner, ld_outer


def kernel_usable(logits: torch.Tensor, temperature, *others: torch.Tensor | None) -> bool:
    """A temperature that is a tensor may want a gradient: it is left to the PyTorch operations."""
    if logits.dtype not in KERNEL_TYPES or isinstance(temperature, torch.Tensor) or logits.shape[-1] > 1 << 30:
        return False
    return _lib.eager(logits, *others)


def check_logits(logits: torch.Tensor, temperature) -> None:
    if not logits.shape or not logits.shape[-1] or (logits.dtype not in KERNEL_TYPES and not logits.is_floating_point()):
        raise ValueError(f"logits need a floating type and a vocabulary, got {logits.dtype} of {tuple(logits.shape)}")
    if not isinstance(temperature, torch.Tensor) and not 0 < temperature < math.inf:
        raise ValueError(f"temperature has to be positive, got {temperature}")


def integers(t: torch.Tensor) -> bool:
    return t.dtype == torch.int64 or not (t.is_floating_point() or t.is_complex() or t.dtype == torch.bool)


def as_int64(t: torch.Tensor) -> torch.Tensor:
    return t.contiguous() if t.dtype == torch.int64 else t.to(torch.int64).contiguous()


def check_tokens(name: str, tokens: torch.Tensor, logits: torch.Tensor) -> None:
    if tokens.shape != logits.shape[:-1] or not integers(tokens):
        raise ValueError(f"{name} have to be integers of shape {tuple(logits.shape[:-1])}, got {tokens.dtype} of "
                         f"{tuple(tokens.shape)}")


def statement_gradient(logits, statement, upstream):
    """Gradient of the logits by the PyTorch operations: where a graph of it is asked for, or where the upstream values have no
    address (in a vmap over the backward pass, so with ``autograd.grad(is_grads_batched=True)``)."""
    graph = torch.is_grad_enabled()
    with torch.enable_grad():
        x = logits.view_as(logits)
        outs, grads = zip(*((o, g) for o, g in zip(statement(x), upstream) if g is not None))
        return torch.autograd.grad(outs, [x], grads, create_graph=graph)[0]


def _forward(logits, tokens, top_k, temperature, ignore_index, with_stats):
    x, inner, ld_inner, ld_outer = logit_rows(logits)
    shape = x.shape
    V = shape[-1]
    rows = x.numel() // V
    logprobs = top = ids = stats = None
    if tokens is not None:              # (empty_like costs half of what a shape and a device do)
        logprobs = torch.empty_like(tokens, dtype=torch.float32)
        entropy = torch.empty_like(logprobs)
    else:
        entropy = torch.empty(tuple(shape[:-1]), dtype=torch.float32, device=x.device)
    if top_k:
        top = torch.empty((*shape[:-1], top_k), dtype=torch.float32, device=x.device)
        ids = torch.empty_like(top, dtype=torch.int64)
    if with_stats:
        stats = torch.empty(4 * rows, dtype=torch.float32, device=x.device)
    rc = _lib.cuda_lib().lme_token_logprobs_fwd(
        x.data_ptr(), KERNEL_TYPES[x.dtype], rows, inner, ld_inner, ld_outer, V,
        None if tokens is None else tokens.data_ptr(), ignore_index, temperature, top_k,
        None if tokens is None else logprobs.data_ptr(), entropy.data_ptr(), top.data_ptr() if top_k else None,
        ids.data_ptr() if top_k else None, stats.data_ptr() if with_stats else None, _lib.stream_ptr())
    if rc:
        _lib.check(rc, "lme_token_logprobs_fwd")
    _lib.count_launch()
    return logprobs, entropy, top, ids, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature, ignore_index):
        logprobs, entropy, top, ids, ctx.stats = _forward(logits, tokens, top_k, temperature, ignore_index, True)
        ctx.save_for_backward(logits, tokens, ids)
        ctx.meta = (top_k, temperature, ignore_index)
        ctx.set_materialize_grads(False)
        if top_k:
            ctx.mark_non_differentiable(ids)
        return logprobs, entropy, top, ids

    @staticmethod
    def backward(ctx, d_logprobs, d_entropy, d_top, _):
        logits, tokens, ids = ctx.saved_tensors
        top_k, temperature, ignore_index = ctx.meta
        if d_logprobs is None and d_entropy is None and d_top is None:
            return None, None, None, None, None
        small = [None if t is None else t.contiguous() for t in (tokens, ids, d_logprobs, d_entropy, d_top)]
        try:
            at = None if torch.is_grad_enabled() else [_lib.ptr(t) for t in small]
        except RuntimeError:                # (checks beforehand would cost 4 us of the 100 us that a small call takes)
            at = None
        if at is None:
            grad = statement_gradient(
                logits, lambda x: token_logprobs_reference(x, tokens, top_k, temperature, ignore_index)[:3],
                (d_logprobs, d_entropy, d_top))
            return grad, None, None, None, None
        x, inner, ld_inner, ld_outer = logit_rows(logits)
        V = x.size(-1)
        grad = torch.empty_like(x, memory_format=torch.contiguous_format)
        rc = _lib.cuda_lib().lme_token_logprobs_bwd(
            x.data_ptr(), KERNEL_TYPES[x.dtype], x.numel() // V, inner, ld_inner, ld_outer, V, at[0],
            ignore_index, temperature, top_k, ctx.stats.data_ptr(), *at[1:], grad.data_ptr(), _lib.stream_ptr())
        if rc:
            _lib.check(rc, "lme_token_logprobs_bwd")
        _lib.count_launch()
        return grad, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, top_k: int = 0, temperature: float = 1.0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Of ``softmax(logits / temperature)`` over the last dimension, all in fp32 (fp64 for fp64 logits):

    * the log probability of each position's token; 0 at positions whose token is ``ignore_index``, NaN (and no gradient) where
      a token is outside of the vocabulary,
    * the entropy of every position, those with ``ignore_index`` too,
    * with ``top_k`` (at most 128 and the vocabulary) the log probabilities and ids of the tokens with the largest logits,
      in order, the lowest id first among equal ones.

    Logits may be slices of larger ones and of minus infinity for forbidden tokens, which add nothing; a row of nothing else, or
    with a NaN, has NaN results.  Differentiable in the logits; they must hold the whole vocabulary."""
    check_logits(logits, temperature)
    if tokens is not None:
        check_tokens("tokens", tokens, logits)
    if top_k and not 0 < top_k <= min(MAX_TOP_K, logits.size(-1)):
        raise ValueError(f"top_k has to be in 0..{min(MAX_TOP_K, logits.size(-1))}, got {top_k}")
    if not kernel_usable(logits, temperature, tokens):
        return token_logprobs_reference(logits, tokens, top_k, temperature, ignore_index)
    if tokens is not None:
        tokens = as_int64(tokens)
    top_k, temperature, ignore_index = int(top_k), float(temperature), int(ignore_index)
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, top_k, temperature, ignore_index))
    logprobs, entropy, top, ids, _ = _forward(logits, tokens, top_k, temperature, ignore_index, False)
    return TokenLogprobs(logprobs, entropy, top, ids)
