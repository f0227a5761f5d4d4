"""Log probabilities of given tokens, with the entropy of every position and its most likely alternatives.

What scoring, served log probabilities and policy gradients need from logits, without the ``[T, V]`` log softmax: one
pass over the logits forward, one pass backward, both hand-written kernels for bf16, fp16 and fp32 (the reference has
no counterpart; its losses go through ``F.log_softmax``, lm_engine/model_wrapper/distillation.py:132-139).
"""

from __future__ import annotations

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
        inside = (tokens >= 0) & (tokens < x.size(-1))
        at = torch.where(inside, tokens, 0).long()
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
    V = x.size(-1)
    if x.is_contiguous():
        return x, max(x.numel() // V, 1), V, 0
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
    return (logits.dtype in KERNEL_TYPES and not isinstance(temperature, torch.Tensor)
            and logits.size(-1) <= 1 << 30 and _lib.eager(logits, *(t for t in others if t is not None)))


def check_logits(logits: torch.Tensor, temperature) -> None:
    if logits.dim() == 0 or logits.size(-1) == 0 or not logits.is_floating_point():
        raise ValueError(f"logits need a floating type and a vocabulary, got {logits.dtype} of {tuple(logits.shape)}")
    if not isinstance(temperature, torch.Tensor) and not 0 < temperature < float("inf"):
        raise ValueError(f"temperature has to be positive, got {temperature}")


def check_tokens(name: str, tokens: torch.Tensor, logits: torch.Tensor) -> None:
    if tokens.shape != logits.shape[:-1] or tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool:
        raise ValueError(f"{name} have to be integers of shape {tuple(logits.shape[:-1])}, got {tokens.dtype} of "
                         f"{tuple(tokens.shape)}")


def _forward(logits, tokens, top_k, temperature, ignore_index, with_stats):
    x, inner, ld_inner, ld_outer = logit_rows(logits)
    shape, dev = logits.shape[:-1], logits.device
    entropy = torch.empty(shape, dtype=torch.float32, device=dev)
    logprobs = torch.empty(shape, dtype=torch.float32, device=dev) if tokens is not None else None
    top = torch.empty((*shape, top_k), dtype=torch.float32, device=dev) if top_k else None
    ids = torch.empty((*shape, top_k), dtype=torch.int64, device=dev) if top_k else None
    stats = torch.empty((*shape, 4), dtype=torch.float32, device=dev) if with_stats else None
    _lib.check(_lib.cuda_lib().lme_token_logprobs_fwd(
        x.data_ptr(), KERNEL_TYPES[x.dtype], entropy.numel(), inner, ld_inner, ld_outer, x.size(-1), _lib.ptr(tokens),
        ignore_index, temperature, top_k, _lib.ptr(logprobs), entropy.data_ptr(), _lib.ptr(top), _lib.ptr(ids),
        _lib.ptr(stats), _lib.stream_ptr()), "lme_token_logprobs_fwd")
    _lib.count_launch()
    return logprobs, entropy, top, ids, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature, ignore_index):
        logprobs, entropy, top, ids, stats = _forward(logits, tokens, top_k, temperature, ignore_index, True)
        ctx.save_for_backward(logits, tokens, ids, stats)
        ctx.meta = (top_k, temperature, ignore_index)
        ctx.set_materialize_grads(False)
        if ids is not None:
            ctx.mark_non_differentiable(ids)
        return logprobs, entropy, top, ids

    @staticmethod
    def backward(ctx, d_logprobs, d_entropy, d_top, _):
        logits, tokens, ids, stats = ctx.saved_tensors
        top_k, temperature, ignore_index = ctx.meta
        grads = (d_logprobs, d_entropy, d_top)
        if all(g is None for g in grads):
            return None, None, None, None, None
        if torch.is_grad_enabled():         # a graph of the gradients is asked for
            x = logits.view_as(logits)
            outs = token_logprobs_reference(x, tokens, top_k, temperature, ignore_index)[:3]
            outs, grads = zip(*((o, g) for o, g in zip(outs, grads) if g is not None))
            return *torch.autograd.grad(outs, [x], grads, create_graph=True), None, None, None, None
        d_logprobs, d_entropy, d_top = (None if g is None else g.float().contiguous() for g in grads)
        x, inner, ld_inner, ld_outer = logit_rows(logits)
        tokens, ids, stats = (None if t is None else _lib.aligned(t) for t in (tokens, ids, stats))
        grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        _lib.check(_lib.cuda_lib().lme_token_logprobs_bwd(
            x.data_ptr(), KERNEL_TYPES[x.dtype], x.numel() // x.size(-1), inner, ld_inner, ld_outer, x.size(-1),
            _lib.ptr(tokens), ignore_index, temperature, top_k, stats.data_ptr(), _lib.ptr(ids), _lib.ptr(d_logprobs),
            _lib.ptr(d_entropy), _lib.ptr(d_top), grad.data_ptr(), _lib.stream_ptr()), "lme_token_logprobs_bwd")
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
    if not 0 <= top_k <= min(MAX_TOP_K, logits.size(-1)):
        raise ValueError(f"top_k has to be in 0..{min(MAX_TOP_K, logits.size(-1))}, got {top_k}")
    if not kernel_usable(logits, temperature, tokens):
        return token_logprobs_reference(logits, tokens, top_k, temperature, ignore_index)
    if tokens is not None:
        tokens = tokens.to(torch.int64).contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, int(top_k), float(temperature), int(ignore_index)))
    return TokenLogprobs(*_forward(logits, tokens, int(top_k), float(temperature), int(ignore_index), False)[:4])
