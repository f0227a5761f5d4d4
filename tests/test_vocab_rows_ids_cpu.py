"""Ids of every integer type, on the PyTorch operations: compared with the vocabulary and the ignored index as numbers, not
in their own type.  And transforms, which take the PyTorch operations too."""

import math

import pytest
import torch

from lm_engine_b200.ops import (token_logprobs, token_logprobs_reference, topk_distillation,
                                topk_distillation_reference)

TYPES = [torch.uint8, torch.int8, torch.int16, torch.int32, torch.uint16, torch.uint32, torch.uint64]


def _logits(V=1000):
    return torch.randn(4, V, generator=torch.Generator().manual_seed(1), dtype=torch.float64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", [token_logprobs, token_logprobs_reference])
def test_tokens_of_every_integer_type(dtype, score):
    x, tok = _logits(), torch.tensor([5, 100, 127, 0])      # (1000 is no number of eight bits)
    want = torch.log_softmax(x, -1).gather(-1, tok[:, None])[:, 0]
    assert torch.allclose(score(x, tok.to(dtype)).logprobs, want, rtol=1e-12, atol=0)


def test_tokens_that_are_the_ignored_index_in_eight_bits():
    x = _logits()
    tok = torch.tensor([156, 5, 255, 7], dtype=torch.uint8)     # 156 = -100 and 255 = -1 modulo 256
    want = torch.log_softmax(x, -1).gather(-1, tok.long()[:, None])[:, 0]
    for ignore in (-100, -1, 261):                              # 261 = 5 modulo 256
        assert torch.allclose(token_logprobs(x, tok, ignore_index=ignore).logprobs, want, rtol=1e-12, atol=0)
    assert token_logprobs(x, tok, ignore_index=7).logprobs[3] == 0
    signed = torch.tensor([3, -100, -1, 7], dtype=torch.int8)
    out = token_logprobs(x, signed).logprobs
    assert out[1] == 0 and math.isnan(out[2]) and out[[0, 3]].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("distil", [topk_distillation, topk_distillation_reference])
def test_lists_and_labels_of_every_integer_type(dtype, distil):
    x = _logits().requires_grad_(True)
    ids, labels = torch.tensor([[1, 2], [100, 7], [120, 3], [0, 127]]), torch.tensor([5, 100, 127, 0])
    lq = torch.log(torch.rand(4, 2, generator=torch.Generator().manual_seed(2)) / 2)
    want, got = distil(x, ids, lq, labels), distil(x, ids.to(dtype), lq, labels.to(dtype))
    assert torch.equal(got.kl_divergence, want.kl_divergence) and torch.equal(got.nll, want.nll)
    assert float(got.kl_divergence.detach().min()) > 0
    nll = torch.nn.functional.cross_entropy(x, labels, reduction="none")
    assert torch.allclose(got.nll, nll, rtol=1e-12, atol=0)
    a, b = (torch.autograd.grad(o.kl_divergence.sum() + o.nll.sum(), x)[0] for o in (want, got))
    assert torch.equal(a, b)


def test_labels_and_lists_beside_the_ignored_index():
    x = _logits()
    ids = torch.tensor([[1, 2], [-1, -1], [3, -100], [0, 127]], dtype=torch.int8)
    labels = torch.tensor([156, 5, 255, 7], dtype=torch.uint8)
    lq = torch.full((4, 2), -1.0)
    out = topk_distillation(x, ids, lq, labels)
    want = topk_distillation(x, ids.long(), lq, labels.long())
    assert torch.equal(out.kl_divergence, want.kl_divergence) and torch.equal(out.nll, want.nll)
    assert out.kl_divergence[1] == 0 and float(out.nll[0]) > 0


@pytest.mark.parametrize("method,tail", [("backward", True), ("backward", False), ("forward", True)])
def test_transforms_over_positions(method, tail):
    """vmap over positions, gradients position by position, and a derivative along a direction."""
    x = _logits(40)
    ids, labels = torch.tensor([[1, 2], [9, 7], [12, -1], [0, 27]]), torch.tensor([5, 10, -100, 0])
    lq = torch.log(torch.rand(4, 2, generator=torch.Generator().manual_seed(2)) / 2)
    want = topk_distillation(x, ids, lq, labels, method, tail)
    one = lambda v, i, q, t: topk_distillation(v, i, q, t, method, tail)        # noqa: E731
    got = torch.func.vmap(one)(x, ids, lq, labels)
    assert torch.allclose(got.kl_divergence, want.kl_divergence) and torch.allclose(got.nll, want.nll)
    per = torch.func.vmap(torch.func.grad(lambda *a: sum(one(*a))))(x, ids, lq, labels)
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(sum(o.sum() for o in one(leaf, ids, lq, labels)), leaf)
    assert torch.allclose(per, g)
    along = torch.randn(x.shape, generator=torch.Generator().manual_seed(3), dtype=x.dtype)
    _, d = torch.func.jvp(lambda v: sum(o.sum() for o in one(v, ids, lq, labels)), (x,), (along,))
    assert torch.allclose(d, (g * along).sum())
