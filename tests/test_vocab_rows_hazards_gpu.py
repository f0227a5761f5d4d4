"""Token log probabilities and distillation where parts of the kernels meet: stages of the ring that are filled again while
rows take the careful steps, repeated entries of a teacher's list, upstream gradients that are not plain tensors."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _logits(rows, V, dtype, seed):
    return (2 * torch.randn(1, rows, V, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")).to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,V", [(300, 50257), (1500, 12001)])
def test_rows_with_forbidden_tokens_repeat_to_the_bit(rows, V, dtype):
    """Minus infinity ends the tried steps: no branch then hangs on what a step adds before its stage is requested again.  A
    stage that is overwritten under its reads changes sums from call to call, and against 64 bits."""
    from lm_engine_b200.ops import token_logprobs, topk_distillation

    x = _logits(rows, V, dtype, 5)
    x[..., ::3] = -math.inf
    lq, ids = torch.log_softmax(x.float(), -1).topk(9, -1)
    lq = lq - 0.5
    first = None
    for _ in range(100):
        s = token_logprobs(x, ids[..., 3], top_k=9, temperature=0.8)
        d = topk_distillation(x, ids, lq, ids[..., 1], temperature=1.3)
        got = [*s, *d]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))
    best = x.sort(dim=-1, descending=True, stable=True).indices[..., :9]       # (topk orders equal ones as it likes)
    assert torch.equal(first[3], best)
    logp = torch.log_softmax(x.double() / 0.8, -1)
    # a thread's sum of V / 128 exponentials, each off by 2^-22 and its exponent's rounding (24 nats: 2^-19), added in 32 bits
    off = (V / 128 + 100) * 2.0 ** -24 + 2.0 ** -19
    assert float((first[0] - logp.gather(-1, ids[..., 3:4])[..., 0]).abs().max()) < off
    entropy = -(logp.exp() * logp.masked_fill(logp == -math.inf, 0.0)).sum(-1)
    assert float((first[1] - entropy).abs().max()) < off * (2 + math.log2(V))


@pytest.mark.parametrize("rows", [2, 250, 900])
@pytest.mark.parametrize("method,tail", [("backward", False), ("backward", True), ("forward", True)])
@pytest.mark.parametrize("value", [900.0, -900.0, math.nan, math.inf])
def test_values_of_repeated_entries_are_not_looked_at(rows, method, tail, value):
    """One CTA or several per row (the entries of a token lie in one of them, the values' largest is of all)."""
    from lm_engine_b200.ops import topk_distillation

    V, K = 20000, 24
    x = _logits(rows, V, F32, 3).requires_grad_(True)
    lq, ids = (x.detach() + _logits(rows, V, F32, 4)).topk(K, -1)
    if tail:
        lq = torch.log_softmax(lq, -1) - 0.5
    ids[..., 9], ids[..., 20] = ids[..., 2], ids[..., 17]
    fewer = ids.clone()
    fewer[..., 9] = fewer[..., 20] = -1
    lq[..., 9] = lq[..., 20] = value
    d = torch.rand(1, rows, device="cuda") + 0.5

    def run(which):
        kl = topk_distillation(x, which, lq, None, method, tail).kl_divergence
        return kl, *torch.autograd.grad(kl, x, d)

    (kl, g), (kl_fewer, g_fewer) = run(ids), run(fewer)
    assert kl.isfinite().all()
    # the same entries count: the same sums, whatever stands at the others
    assert torch.equal(kl, kl_fewer) and torch.equal(g, g_fewer)


@pytest.mark.parametrize("create_graph", [False, True])
def test_batched_upstream_gradients(create_graph):
    """Upstream values of a vmap over the backward pass have no memory of their own: the PyTorch operations take them."""
    from torch.utils.flop_counter import FlopCounterMode

    from lm_engine_b200.ops import _lib, token_logprobs, topk_distillation

    rows, V = 6, 300
    x = _logits(rows, V, F32, 7).requires_grad_(True)
    lq, ids = torch.log_softmax(x.detach(), -1).topk(5, -1)
    lq = lq - 0.5
    s, d = token_logprobs(x, ids[..., 2], top_k=3, temperature=0.7), topk_distillation(x, ids, lq, ids[..., 1], temperature=1.5)
    for out in (s.logprobs, s.entropy, s.top_logprobs, d.kl_divergence, d.nll):
        up = torch.eye(out.numel(), device="cuda").view(-1, *out.shape)
        (all_at_once,) = torch.autograd.grad([out], [x], [up], is_grads_batched=True, retain_graph=True, create_graph=create_graph)
        assert all_at_once.requires_grad == create_graph
        before = _lib.launch_count
        one_by_one = torch.stack([torch.autograd.grad([out], [x], [u], retain_graph=True)[0] for u in up])
        assert _lib.launch_count == before + len(up)
        # both fp32, of sums of 300 exponentials: (300 / 128 + 100) 2^-24 relatively, on terms that add up to at most 2 / 0.7
        # times 1 + |log p| <= 16; entropies' twice
        assert float((all_at_once.detach() - one_by_one).abs().max()) < 104 * 2.0 ** -24 * 2 * 3 * 16
    j = torch.autograd.functional.jacobian(lambda v: token_logprobs(v, ids[..., 2]).logprobs, x.detach(), vectorize=True)
    assert j.shape == (1, rows, 1, rows, V) and j.isfinite().all()
    with FlopCounterMode(display=False):
        (g,) = torch.autograd.grad([d.kl_divergence.sum()], [x], retain_graph=True)
    (h,) = torch.autograd.grad([d.kl_divergence.sum()], [x])
    assert float((g - h).abs().max()) < 104 * 2.0 ** -24 * 3 * 16


def _time(run):
    run()
    best = math.inf
    for _ in range(5):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(3):
            run()
        end.record()
        end.synchronize()
        best = min(best, start.elapsed_time(end))
    return best


def test_the_most_alternatives_of_ordinary_rows_are_selected_from_few():
    """Nearly as many alternatives as a CTA has threads: rows whose candidates do not fit are read some thirty times more,
    which one row in twenty is enough to show."""
    from lm_engine_b200.ops import token_logprobs

    x = _logits(2048, 128256, BF, 13)
    want = x[0, :8].sort(dim=-1, descending=True, stable=True).indices
    few = _time(lambda: token_logprobs(x, top_k=64))
    for k in (65, 100, 127, 128):
        assert torch.equal(token_logprobs(x, top_k=k).top_ids[0, :8], want[:, :k])
        assert _time(lambda: token_logprobs(x, top_k=k)) < 3 * few          # (measured: 1.1 to 1.6; 16 with such rows)


@pytest.mark.parametrize("rows", [1, 500])
@pytest.mark.parametrize("V", [130, 1500, 4096, 8200, 8300, 33000])
@pytest.mark.parametrize("k", [64, 65, 128])
def test_alternatives_of_few_and_odd_segments(rows, V, k):
    from lm_engine_b200.ops import token_logprobs

    for dtype in (BF, F32):
        x = _logits(rows, V, dtype, V)
        for variant in range(4):
            y = x.clone()
            if variant == 1:
                y[..., V // 3:] = -math.inf
            elif variant == 2:
                y[..., ::2] = math.nan
            elif variant == 3:
                y[..., : V - k] -= 100.0                # the best lie at the row's end, in the last segment
            want = y.sort(dim=-1, descending=True, stable=True).indices[..., :k]
            assert torch.equal(token_logprobs(y, top_k=k).top_ids, want)
