"""Distillation from a teacher that is known by its most likely tokens, and the labels' cross entropy in the same passes.

The full distributions of both models (lm_engine/model_wrapper/distillation.py:113-146) are ``[T, V]`` each; a teacher's best
tokens (:func:`lm_engine_b200.ops.token_logprobs` with ``top_k``) can be kept or stored instead.  One kernel forward (a pass over the
student's logits) and one backward (a pass that writes their gradient), for bf16, fp16 and fp32.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn.functional as F

from ..enums import KLDivergenceMethod
from . import _lib
from .logprobs import (KERNEL_TYPES, MAX_TOP_K, as_int64, check_logits, check_tokens, integers, kernel_usable, logit_rows,
                       statement_gradient)

#: The teacher's mass outside of its listed tokens is one minus their sum, which the rounding of fp32 log probabilities moves by
#: about this much: a smaller rest counts as none, and as this much where its logarithm is asked for.
NO_TAIL = 2.0 ** -20
#: The kernel keeps a bit per logit in shared memory; beyond this the PyTorch operations serve.
MAX_KERNEL_VOCAB = 3_000_000


class TopkDistillation(NamedTuple):
    """Per position; ``nll`` is ``None`` without labels."""

    kl_divergence: torch.Tensor
    nll: torch.Tensor | None


def topk_distillation_reference(logits: torch.Tensor, top_ids: torch.Tensor, top_logprobs: torch.Tensor,
                                labels: torch.Tensor | None = None,
                                kl_divergence_method: KLDivergenceMethod = KLDivergenceMethod.backward, tail: bool = True,
                                temperature=1.0, ignore_index: int = -100) -> TopkDistillation:
    V = logits.size(-1)
    top_ids, labels = top_ids.long(), None if labels is None else labels.long()    # (narrow types would compare modulo their range)
    teacher = top_logprobs.detach().double()
    there = (top_ids >= 0) & (top_ids < V) & (teacher != -torch.inf)
    same = (top_ids[..., :, None] == top_ids[..., None, :]) & there[..., None, :]
    there = there & ~same.tril(-1).any(-1)                      # an id's first entry counts
    asked = there.any(-1)
    ids = torch.where(there, top_ids, 0)
    x = logits if logits.dtype == torch.float64 else logits.float()
    if labels is None:
        read = asked
    else:
        read = asked | (labels != ignore_index)
    x = torch.where(read[..., None], x, 0.0)                    # other rows are not looked at
    logp = torch.log_softmax(x / temperature, -1)
    listed = torch.zeros(logits.shape, dtype=torch.int32, device=logits.device).scatter_add(-1, ids, there.int()) > 0
    others = logp.double().masked_fill(listed, -torch.inf)      # in the logarithm: they may be less likely than a number can say
    none = (others == -torch.inf).all(-1)
    log_rest = torch.where(none, -torch.inf, others.masked_fill(none[..., None], 0.0).logsumexp(-1))
    student = torch.where(there, logp.gather(-1, ids).double(), 0.0)
    teacher = torch.where(there, teacher, -torch.inf)
    if not tail:
        teacher = teacher - torch.where(asked, teacher.logsumexp(-1), 0.0)[..., None]
    q = teacher.exp()
    q_rest = torch.zeros_like(log_rest)
    if tail:
        q_rest = 1 - q.sum(-1)
        q_rest = torch.where(q_rest < NO_TAIL, 0.0, q_rest)
    if kl_divergence_method == KLDivergenceMethod.backward:
        kl = torch.where(q > 0, q * (teacher - student), 0.0).sum(-1)
        rest = q_rest * (q_rest.clamp(min=NO_TAIL).log() - log_rest)
        kl = kl + torch.where(q_rest > 0, rest, 0.0)
    else:
        finite = there & (student != -torch.inf)
        away = torch.where(finite, student, 0.0) - torch.where(finite, teacher, 0.0)
        kl = torch.where(finite, student.exp() * away, 0.0).sum(-1)
        log_rest = torch.where(none, 0.0, log_rest)
        kl = kl + torch.where(none, 0.0, log_rest.exp() * (log_rest - q_rest.clamp(min=NO_TAIL).log()))
    kl = torch.where(asked, kl, 0.0).to(x.dtype)
    if labels is None:
        return TopkDistillation(kl, None)
    inside = (labels >= 0) & (labels < V)
    nll = F.cross_entropy(x.reshape(-1, V), torch.where(inside, labels, 0).reshape(-1),
                          reduction="none").view(labels.shape)
    nll = torch.where(labels == ignore_index, 0.0, torch.where(inside, nll, float("nan")))
    return TopkDistillation(kl, nll)


class _TopkDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_ids, top_logprobs, labels, method, tail, temperature, ignore_index):
        x, inner, ld_inner, ld_outer = logit_rows(logits)
        K, V = top_ids.size(-1), x.size(-1)
        rows = x.numel() // V
        if labels is None:
            kl, nll = torch.empty(tuple(x.shape[:-1]), dtype=torch.float32, device=x.device), None
        else:                               # (empty_like costs half of what a shape and a device do)
            kl = torch.empty_like(labels, dtype=torch.float32)
            nll = torch.empty_like(kl)
        ctx.entries = torch.empty_like(top_ids, dtype=torch.int32)
        ctx.stats = torch.empty(12 * rows, dtype=torch.float32, device=x.device)
        rc = _lib.cuda_lib().lme_topk_distillation_fwd(
            x.data_ptr(), KERNEL_TYPES[x.dtype], rows, inner, ld_inner, ld_outer, V, top_ids.data_ptr(),
            top_logprobs.data_ptr(), K, _lib.ptr(labels), ignore_index, temperature,
            method is KLDivergenceMethod.forward, tail, kl.data_ptr(), _lib.ptr(nll), ctx.entries.data_ptr(),
            ctx.stats.data_ptr(), _lib.stream_ptr())
        if rc:
            _lib.check(rc, "lme_topk_distillation_fwd")
        _lib.count_launch()
        ctx.save_for_backward(logits, top_ids, top_logprobs, labels)
        ctx.meta = (method, tail, temperature, ignore_index)
        ctx.set_materialize_grads(False)
        return kl, nll

    @staticmethod
    def backward(ctx, d_kl, d_nll):
        logits, top_ids, top_logprobs, labels = ctx.saved_tensors
        method, tail, temperature, ignore_index = ctx.meta
        nothing = (None,) * 7
        if d_kl is None and d_nll is None:
            return None, *nothing
        small = [None if t is None else t.contiguous() for t in (top_logprobs, labels, d_kl, d_nll)]
        try:
            at = None if torch.is_grad_enabled() else [_lib.ptr(t) for t in small]
        except RuntimeError:                # upstream values without an address
            at = None
        if at is None:
            return statement_gradient(
                logits, lambda x: topk_distillation_reference(x, top_ids, top_logprobs, labels, method, tail, temperature,
                                                              ignore_index), (d_kl, d_nll)), *nothing
        x, inner, ld_inner, ld_outer = logit_rows(logits)
        V = x.size(-1)
        grad = torch.empty_like(x, memory_format=torch.contiguous_format)
        rc = _lib.cuda_lib().lme_topk_distillation_bwd(
            x.data_ptr(), KERNEL_TYPES[x.dtype], x.numel() // V, inner, ld_inner, ld_outer, V, ctx.entries.data_ptr(),
            at[0], top_ids.size(-1), at[1], ignore_index, temperature, method is KLDivergenceMethod.forward,
            ctx.stats.data_ptr(), at[2], at[3], grad.data_ptr(), _lib.stream_ptr())
        if rc:
            _lib.check(rc, "lme_topk_distillation_bwd")
        _lib.count_launch()
        return grad, *nothing


def topk_distillation(logits: torch.Tensor, top_ids: torch.Tensor, top_logprobs: torch.Tensor,
                      labels: torch.Tensor | None = None,
                      kl_divergence_method: KLDivergenceMethod | str = KLDivergenceMethod.backward, tail: bool = True,
                      temperature: float = 1.0, ignore_index: int = -100) -> TopkDistillation:
    """Divergence of every position between the student ``p = softmax(logits / temperature)`` over the whole vocabulary and a
    teacher ``q`` given by ``k <= 128`` tokens per position (``top_ids``, ``top_logprobs`` ``[..., k]``, in any order).

    ``kl_divergence_method``: ``backward`` = ``sum q ln(q / p)``, ``forward`` = ``sum p ln(p / q)``.  With ``tail`` the sums have one
    more bucket, all tokens that are not listed; ``top_logprobs`` are then log probabilities at the same temperature, and the
    teacher's rest is one minus their sum (none below 2^-20, which is also the least that ``forward`` divides by).  Without it
    (``backward`` only) they may be logits as well, divided by the temperature, and are renormalised over the list.

    An entry with an id outside of the vocabulary or a value of minus infinity is absent, an id given twice counts with its first
    entry.  A position without entries has divergence 0 and takes no part; so padding is ids of -1.

    ``labels``: the negative log likelihood of the labels at temperature one, from the same passes; 0 where a label is
    ``ignore_index``, NaN (and no gradient) outside of the vocabulary.  Both results are fp32 (fp64 for fp64 logits) and differentiable in
    the logits, which must hold the whole vocabulary; the teacher gets no gradient."""
    check_logits(logits, temperature)
    method = KLDivergenceMethod(kl_divergence_method)
    if method == KLDivergenceMethod.forward and not tail:
        raise ValueError("kl_divergence_method forward needs the tail: without it tokens outside of the list have no probability")
    K = top_ids.size(-1) if top_ids.dim() else 0
    if not 1 <= K <= MAX_TOP_K:
        raise ValueError(f"a teacher's list has 1..{MAX_TOP_K} tokens, got top_ids of {tuple(top_ids.shape)}")
    if top_ids.shape[:-1] != logits.shape[:-1] or not integers(top_ids):
        raise ValueError(f"top_ids have to be integers of shape {tuple(logits.shape[:-1])} and the list, got "
                         f"{top_ids.dtype} of {tuple(top_ids.shape)}")
    if top_logprobs.shape != top_ids.shape or not top_logprobs.is_floating_point():
        raise ValueError(f"top_logprobs need a floating type and shape {tuple(top_ids.shape)}, got {top_logprobs.dtype} of "
                         f"{tuple(top_logprobs.shape)}")
    if labels is not None:
        check_tokens("labels", labels, logits)
    if logits.size(-1) > MAX_KERNEL_VOCAB or not kernel_usable(logits, temperature, top_ids, top_logprobs, labels):
        return topk_distillation_reference(logits, top_ids, top_logprobs, labels, method, tail, temperature, ignore_index)
    if labels is not None:
        labels = as_int64(labels)
    return TopkDistillation(*_TopkDistillation.apply(
        logits, as_int64(top_ids), top_logprobs.detach().float().contiguous(), labels, method, bool(tail),
        float(temperature), int(ignore_index)))
