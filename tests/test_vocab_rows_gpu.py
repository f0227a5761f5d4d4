"""Token log probabilities and distillation from a teacher's best tokens: the kernels against the statements in 64 bits.

Tolerances.  A thread adds at most L = ceil(V / 256) + 32 exponentials in fp32, and an exponential is off by its exponent's
rounding, two steps of 2^-24 relative to t <= 150 of which only the sum's own |log p| counts, and 2^-22 of the approximate
exponential: the sum is off by SUM = (L + 3 * 24 + 8) 2^-24 at most, relatively.  A log probability carries that and its
rounding; an entropy carries it twice, once times log2 V; gradients carry it relative to the terms they are added from, and half a
step of their type.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _sum_error(V):
    return (math.ceil(V / 256) + 32 + 72 + 8) * 2.0 ** -24


def _rows(B, S, V, dtype, seed, layout="dense"):
    """Logits of the wanted layout; what lies around them is NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 2 * torch.randn(B, S, V, generator=g, device="cuda")
    x[..., :: max(V // 9, 1)] += 6
    x = x.to(dtype)
    if layout == "dense":
        return x
    wide = torch.full((B, S + 1, V + 11), math.nan, device="cuda").to(dtype)
    at = {"odd start": wide.view(-1)[3:3 + x.numel()].view(B, S, V) if V > 1 else wide[:, :-1, 5:5 + V],
          "shift": wide[:, :-1, :V], "pitch": wide[:, 1:, 5:5 + V]}[layout]
    return at.copy_(x)


def _check(got, want, tol, what):
    got, want = got.double(), want.double()
    finite = want.isfinite()
    assert torch.equal(got.isfinite(), finite), what
    assert torch.equal(got.isnan(), want.isnan()), what
    off = (got - want).abs()[finite] - (tol.expand_as(want)[finite] if isinstance(tol, torch.Tensor) else tol)
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()))


def _score(x, tok, k, temperature, seed=0, grads=True):
    from lm_engine_b200.ops import token_logprobs, token_logprobs_reference

    x = x.detach().requires_grad_(grads)
    V = x.size(-1)
    out = token_logprobs(x, tok, top_k=k, temperature=temperature)
    x64 = x.detach().double().requires_grad_(True)
    want = token_logprobs_reference(x64, tok, k, temperature)
    e = _sum_error(V)
    assert out.entropy.dtype == F32
    if tok is not None:
        _check(out.logprobs, want.logprobs, e + want.logprobs.detach().nan_to_num(0).abs() * 2.0 ** -23, "logprobs")
    _check(out.entropy, want.entropy, e * (2 + math.log2(V + 1)) + want.entropy.detach().nan_to_num(0) * 2.0 ** -23, "entropy")
    if k:
        assert torch.equal(out.top_ids, want.top_ids)
        _check(out.top_logprobs, want.top_logprobs,
               e + want.top_logprobs.detach().nan_to_num(0, 0, 0).abs() * 2.0 ** -23, "top")
    if not grads:
        return out
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    pairs = [(a, b, torch.randn(a.shape, generator=g, device="cuda")) for a, b in
             ((out.logprobs, want.logprobs), (out.entropy, want.entropy), (out.top_logprobs, want.top_logprobs)) if a is not None]
    (got,) = torch.autograd.grad([p[0] for p in pairs], [x], [p[2] for p in pairs])
    (ref,) = torch.autograd.grad([p[1] for p in pairs], [x64], [p[2].double() for p in pairs])
    assert got.dtype == x.dtype and got.shape == x.shape
    logp = torch.log_softmax(x64.detach() / temperature, -1)
    p = logp.exp()
    size = sum((d.abs().sum(-1) if d.dim() > p.dim() - 1 else d.abs())[..., None] for _, _, d in pairs)
    size = (size * (2 + logp.clamp(min=-300).abs() + math.log2(V + 1)) / temperature).nan_to_num(0)     # terms that add up to
    eps = torch.finfo(x.dtype).eps / 2                                                                # a gradient, over p
    patch = torch.zeros_like(p)                     # upstream values of single tokens, scaled and added in fp32
    if tok is not None:
        here = (tok >= 0) & (tok < V)
        patch.scatter_add_(-1, torch.where(here, tok, 0).long()[..., None], torch.where(here, pairs[0][2].abs(), 0.0).double()[..., None])
    if k:
        patch.scatter_add_(-1, out.top_ids, pairs[-1][2].abs().double())
    size_p = (p * size).nan_to_num(0) * (4 * e) + patch / temperature * 2.0 ** -22
    # an exponential below 2^-126 counts as none: off by that times the same factors, over a sum of 2^-1/2 at least (a thread's
    # base is its sum's logarithm rounded to a power of two)
    tiny = size * 2.0 ** -125.5 + (2.0 ** -25 if x.dtype == HF else 2.0 ** -126)
    _check(got, ref, ref.abs().nan_to_num(0) * (eps + 2.0 ** -22) + size_p + tiny, "gradient")
    return out


SIZES = [(1, 1, 1, 1), (1, 1, 2, 2), (2, 3, 7, 3), (1, 5, 8, 8), (1, 2, 9, 0), (3, 1, 100, 100), (1, 4, 1000, 128), (2, 3, 2047, 20),
         (1, 1, 8200, 64), (1, 24, 50257, 5), (1, 1, 128256, 20), (1, 333, 5003, 1), (1, 700, 1031, 128), (2, 160, 32000, 50),
         (1, 3, 200001, 128)]


@pytest.mark.parametrize("B,S,V,k", SIZES)
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_scores(B, S, V, k, dtype):
    x = _rows(B, S, V, dtype, V)
    tok = torch.randint(V, (B, S), generator=torch.Generator(device="cuda").manual_seed(V), device="cuda")
    if tok.numel() > 1:
        tok[0, 0] = -100
    _score(x, tok, k, 1.0)


@pytest.mark.parametrize("layout", ["odd start", "shift", "pitch"])
@pytest.mark.parametrize("V", [1, 13, 1001, 4104, 20011])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_scores_of_slices(layout, V, dtype):
    x = _rows(2, 3, V, dtype, V, layout)
    tok = torch.randint(V, (2, 3), device="cuda")
    _score(x, tok, min(V, 17), 0.6)
    _score(x, None, min(V, 3), 1.9)
    _score(x, tok.int(), 0, 1.0)


@pytest.mark.parametrize("rows", [1, 700])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("k", [1, 20, 128])
def test_alternatives_of_rows_with_many_equal_values(rows, dtype, k):
    V = 9001
    x = torch.zeros(1, rows, V, device="cuda", dtype=dtype)
    _score(x, None, k, 1.0)                                            # constant: the first ids
    x = torch.arange(V, device="cuda").float().mul_(2.0 ** -9).to(dtype).expand(1, rows, V)
    _score(x, None, k, 1.0)                                            # ascending, many equal in bf16, rows of stride 0
    _score(x.flip(-1), None, k, 1.0)
    x = torch.zeros(1, rows, V, device="cuda", dtype=dtype)
    x[..., 5::7] = 1.0
    x[..., 4::31] = -0.0
    _score(x, None, k, 1.0)
    x[..., :] = -math.inf
    x[..., V - 1] = 3.0
    x[..., 17] = 2.0
    _score(x, torch.full((1, rows), 17, device="cuda"), k, 1.0, grads=False)    # fewer finite values than k
    x = torch.zeros(1, rows, V, device="cuda", dtype=dtype)
    x[..., ::256] = 5.0                                                # all in one thread's vectors
    x[..., 1::256] = 5.0
    _score(x, None, k, 1.0)


@pytest.mark.parametrize("rows", [2, 400])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_infinities_and_nan(rows, dtype):
    from lm_engine_b200.ops import token_logprobs

    V = 5000
    x = _rows(1, rows, V, dtype, 7)
    tok = torch.zeros(1, rows, dtype=torch.long, device="cuda") + 1
    banned = x.clone()
    banned[..., ::3] = -math.inf
    _score(banned, tok, 20, 0.7)
    lowest = x.clone()
    lowest[..., ::3] = torch.finfo(dtype).min
    _score(lowest, tok, 20, 1.0)
    for value in (math.nan, math.inf):
        bad = x.clone()
        bad[0, 1, 4003] = value
        out = _score(bad, tok, 5, 1.0, grads=False)
        assert out.entropy[0, 1].isnan() and out.logprobs[0, 1].isnan() and int(out.top_ids[0, 1, 0]) == 4003
        assert out.entropy[0, 0].isfinite()
        leaf = bad.requires_grad_(True)
        out = token_logprobs(leaf, tok, top_k=5)
        (g,) = torch.autograd.grad([out.logprobs.sum() + out.entropy.sum()], [leaf])
        assert g[0, 1].isnan().all() and g[0, 0].isfinite().all()
    nothing = x.clone()
    nothing[0, 0] = -math.inf
    out = _score(nothing, tok, 5, 1.0, grads=False)
    assert out.entropy[0, 0].isnan() and out.top_ids[0, 0].tolist() == [0, 1, 2, 3, 4]


def test_scores_outside_of_the_vocabulary_and_empty():
    from lm_engine_b200.ops import token_logprobs

    x = _rows(1, 5, 777, BF, 3).requires_grad_(True)
    tok = torch.tensor([[0, 777, -1, -100, 776]], device="cuda")
    out = token_logprobs(x, tok)
    assert out.logprobs[0].isnan().tolist() == [False, True, True, False, False] and float(out.logprobs[0, 3].detach()) == 0
    (g,) = torch.autograd.grad([out.logprobs], [x], [torch.ones(1, 5, device="cuda")])
    assert float(g[0, 1:4].abs().max()) == 0 and float(g[0, 0].abs().max()) > 0
    none = token_logprobs(x[:, :0], tok[:, :0], top_k=3)
    assert none.top_ids.shape == (1, 0, 3) and none.logprobs.shape == (1, 0)
    (g,) = torch.autograd.grad([none.entropy.sum()], [x])
    assert float(g.abs().max()) == 0


@pytest.mark.parametrize("temperature", [1e-3, 1e4])
def test_scores_at_extreme_temperatures(temperature):
    _score(_rows(1, 40, 3001, F32, 5), torch.arange(40, device="cuda")[None], 9, temperature)


# ------------------------------------------------------------------------------------------------ distillation
def _lists(x, K, seed, tail=True, temperature=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    V = x.size(-1)
    teacher = x.float().nan_to_num(0, 0, -30) + torch.randn(x.shape, generator=g, device="cuda")
    lq, ids = (teacher / temperature).topk(min(K, V), -1)
    if tail:
        lq = lq - (teacher / temperature).logsumexp(-1, keepdim=True)
    order = torch.randperm(min(K, V), generator=g, device="cuda")
    lq, ids = lq[..., order], ids[..., order]
    if K > V:
        ids = torch.cat([ids, ids[..., :1].expand(*ids.shape[:-1], K - V)], -1)
        lq = torch.cat([lq, lq[..., :1].expand(*lq.shape[:-1], K - V)], -1)
    return ids, lq


def _distill(x, ids, lq, labels, method, tail, temperature, seed=0, slack=1.0):
    from lm_engine_b200.ops import topk_distillation, topk_distillation_reference

    x = x.detach().requires_grad_(True)
    V = x.size(-1)
    out = topk_distillation(x, ids, lq, labels, method, tail, temperature)
    x64 = x.detach().double().requires_grad_(True)
    want = topk_distillation_reference(x64, ids, lq, labels, method, tail, temperature)
    e = _sum_error(V)
    kl = want.kl_divergence.detach()
    # weights of the logarithms add up to one on each side; forward multiplies the sum's error by its logarithms too
    size = 2 if method == "backward" else 2 + 4 * math.log2(V + 2) + kl.nan_to_num(0, 0, 0).abs()
    _check(out.kl_divergence, kl, e * size + kl.nan_to_num(0, 0, 0).abs() * 2.0 ** -23, "divergence")
    if labels is not None:
        _check(out.nll, want.nll, e + want.nll.detach().nan_to_num(0, 0, 0).abs() * 2.0 ** -23, "nll")
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    d = [torch.randn(o.shape, generator=g, device="cuda") for o in out if o is not None]
    (got,) = torch.autograd.grad([o for o in out if o is not None], [x], d)
    (ref,) = torch.autograd.grad([o for o in want if o is not None], [x64], [v.double() for v in d])
    assert got.dtype == x.dtype and got.shape == x.shape
    p = torch.softmax(x64.detach() / temperature, -1)
    inside = (ids >= 0) & (ids < V)
    q = torch.zeros_like(p).scatter_add_(-1, torch.where(inside, ids, 0), torch.where(inside, lq.double(), -math.inf).exp())
    if not tail:
        q = q / q.sum(-1, keepdim=True).clamp(min=1e-30)
    # the teacher's rest is spread over what is not listed as the student has it
    rest = (1 - q.sum(-1, keepdim=True)).clamp(min=0) if tail else torch.zeros_like(kl)[..., None]
    share = torch.softmax((x64.detach() / temperature).masked_fill(q > 0, -math.inf), -1).nan_to_num(0)
    if method == "backward":
        terms = p + q + rest * share
    else:
        terms = p * (4 + p.clamp(min=1e-30).log().abs() + q.clamp(min=2.0 ** -20).log().abs() + math.log2(V + 2)
                     + kl.abs()[..., None] + torch.where(q > 0, lq.double().abs().clamp(max=1e4).amax(-1, keepdim=True), 0.0))
    terms = terms * d[0].abs()[..., None] / temperature
    if labels is not None:
        terms = terms + torch.softmax(x64.detach(), -1) * d[1].abs()[..., None]
    eps = torch.finfo(x.dtype).eps / 2
    # an exponential below 2^-126 counts as none: off by that times what terms has beside p
    flushed = 2.0 if method == "backward" else 4 + 300 + kl.abs()[..., None] + lq.double().abs().clamp(max=1e4).amax(-1, keepdim=True)
    tiny = 2.0 ** -126 * (flushed * d[0].abs()[..., None] / temperature + 1).nan_to_num(0, 0, 0)
    tiny = tiny + (2.0 ** -25 if x.dtype == HF else 2.0 ** -126)
    _check(got, ref, ref.abs().nan_to_num(0) * (eps + 2.0 ** -22) + terms.nan_to_num(0) * (4 * e * slack) + tiny, "gradient")
    return out, got


METHODS = [("backward", True), ("backward", False), ("forward", True)]


@pytest.mark.parametrize("B,S,V,K", [(1, 1, 1, 1), (1, 1, 2, 1), (2, 3, 7, 3), (1, 5, 8, 8), (1, 4, 9, 16), (3, 1, 100, 99),
                                     (1, 4, 1000, 128), (2, 3, 2047, 20), (1, 1, 8200, 64), (1, 24, 50257, 5), (1, 2, 128256, 100),
                                     (1, 333, 5003, 1), (1, 700, 1031, 128), (2, 160, 32000, 50), (1, 3, 200001, 128)])
@pytest.mark.parametrize("method,tail", METHODS)
def test_distillation(B, S, V, K, method, tail):
    for dtype, temperature, labelled in ((BF, 1.0, True), (F32, 2.0, True), (HF, 0.8, False)):
        x = _rows(B, S, V, dtype, V)
        ids, lq = _lists(x, K, V, tail, temperature)
        labels = torch.randint(V, (B, S), generator=torch.Generator(device="cuda").manual_seed(V), device="cuda")
        if labels.numel() > 2:
            labels[0, 0], labels[-1, -1] = -100, ids[-1, -1, 0]
        _distill(x, ids, lq, labels if labelled else None, method, tail, temperature)


@pytest.mark.parametrize("layout", ["odd start", "shift", "pitch"])
@pytest.mark.parametrize("V", [13, 1001, 4104, 20011])
def test_distillation_of_slices(layout, V):
    for dtype in (BF, F32):
        x = _rows(2, 3, V, dtype, V, layout)
        ids, lq = _lists(x, 9, V)
        _distill(x, ids, lq, ids[..., 2], "backward", True, 1.0)
        _distill(x, ids, lq, torch.randint(V, (2, 3), device="cuda"), "forward", True, 1.5)


@pytest.mark.parametrize("rows", [6, 400])
@pytest.mark.parametrize("method,tail", METHODS)
def test_lists_with_absent_and_repeated_entries(rows, method, tail):
    from lm_engine_b200.ops import topk_distillation

    V, K = 3001, 12
    x = _rows(1, rows, V, BF, 1)
    ids, lq = _lists(x, K, 2, tail)
    ids[0, 0] = -1                                  # no entry
    ids[0, 1, 3], ids[0, 1, 7] = V, -5              # outside
    lq[0, 2, ::2] = -math.inf                       # without a value
    ids[0, 3, 5], ids[0, 3, 9] = ids[0, 3, 1], ids[0, 3, 1]     # again, with other values
    ids[0, 4, 1], lq[0, 4, 1] = ids[0, 4, 0], -math.inf         # again, absent
    lq[0, 4, 0], ids[0, 4, 2] = -math.inf, ids[0, 4, 0]         # the first is absent, the second counts
    labels = torch.full((1, rows), 5, device="cuda")
    labels[0, 0], labels[0, 1], labels[0, 5] = -100, V, ids[0, 5, 0]
    with torch.no_grad():
        x[0, 0, 17] = math.nan                      # not looked at: no entry, no label
    from lm_engine_b200.ops import topk_distillation_reference

    leaf = x.detach().requires_grad_(True)
    x64 = leaf.detach().double().requires_grad_(True)
    out = topk_distillation(leaf, ids, lq, labels, method, tail)
    want = topk_distillation_reference(x64, ids, lq, labels, method, tail)
    e = _sum_error(V) * 60
    _check(out.kl_divergence, want.kl_divergence, e, "divergence")
    _check(out.nll, want.nll, e, "nll")
    (got,) = torch.autograd.grad([out.kl_divergence, out.nll], [leaf], [torch.ones(1, rows, device="cuda")] * 2)
    (ref,) = torch.autograd.grad([want.kl_divergence, want.nll], [x64], [torch.ones(1, rows, device="cuda").double()] * 2)
    assert float(got[0, 0].abs().max()) == 0
    _check(got, ref, ref.abs() * (2.0 ** -8) + 2.0 ** -14, "gradient")


@pytest.mark.parametrize("rows", [3, 400])
@pytest.mark.parametrize("method,tail", METHODS)
def test_distillation_with_forbidden_tokens(rows, method, tail):
    V, K = 4000, 10
    x = _rows(1, rows, V, BF, 1)
    x[..., ::3] = -math.inf
    x[0, 0, 20:] = -math.inf                        # the list holds all that is allowed
    ids, lq = _lists(x.masked_fill(x == -math.inf, -300.0), K, 2, tail)
    ids[0, 0] = torch.tensor([j for j in range(20) if j % 3][:K], device="cuda")
    _distill(x, ids, lq, ids[..., 0], method, tail, 1.0)
    x[0, 1, ids[0, 1, 1]] = -math.inf               # a listed token that the student forbids
    from lm_engine_b200.ops import topk_distillation

    leaf = x.requires_grad_(True)
    out = topk_distillation(leaf, ids, lq, None, method, tail)
    (g,) = torch.autograd.grad(out.kl_divergence.sum(), leaf)
    assert (float(out.kl_divergence[0, 1].detach()) == math.inf) == (method == "backward")
    assert g.isfinite().all() and out.kl_divergence[0, 2].isfinite()


def test_nothing_left_for_the_other_tokens():
    x = _rows(1, 300, 2000, F32, 1)
    ids, lq = _lists(x, 20, 3)
    lq = lq - lq.logsumexp(-1, keepdim=True)
    _distill(x, ids, lq, None, "backward", True, 1.0)
    _distill(x, ids, lq, None, "forward", True, 1.0)


def test_teacher_logits_of_any_size_are_renormalised():
    x = _rows(1, 300, 2000, F32, 1)
    ids, lq = _lists(x, 20, 3, tail=False)
    a, ga = _distill(x, ids, lq, None, "backward", False, 1.0)
    for shift in (900.0, -900.0):
        from lm_engine_b200.ops import topk_distillation

        b = topk_distillation(x, ids, lq.double() + shift, None, "backward", False)     # taken as fp32: 2^-15 of rounding
        assert float((a.kl_divergence - b.kl_divergence).detach().abs().max()) < 2.0 ** -14 * 20


# ------------------------------------------------------------------------------------------------ as they are used
def _both(x, tok, ids, lq):
    from lm_engine_b200.ops import token_logprobs, topk_distillation

    s = token_logprobs(x, tok, top_k=7, temperature=0.9)
    d = topk_distillation(x, ids, lq, tok, "backward", True, 1.1)
    return s.logprobs, s.entropy, s.top_logprobs, d.kl_divergence, d.nll


@pytest.mark.parametrize("rows", [1, 500])
def test_repeats_to_the_bit(rows):
    x = _rows(1, rows, 40000, BF, 2).requires_grad_(True)
    ids, lq = _lists(x.detach(), 30, 4)
    tok = ids[..., 0]
    d = torch.randn(1, rows, device="cuda")
    runs = []
    for _ in range(3):
        outs = _both(x, tok, ids, lq)
        runs.append([*outs, *torch.autograd.grad([outs[0], outs[1], outs[3], outs[4]], [x], [d] * 4)])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_captured_with_a_backward_pass_and_replayed():
    x = _rows(1, 60, 9000, BF, 2).requires_grad_(True)
    ids, lq = _lists(x.detach(), 30, 4)
    tok, d = ids[..., 0].clone(), torch.randn(1, 60, device="cuda")

    def step():
        outs = _both(x, tok, ids, lq)
        return [*outs, *torch.autograd.grad([outs[0], outs[1], outs[3], outs[4]], [x], [d] * 4)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        other = _rows(1, 60, 9000, BF, 9)
        x.copy_(other)
        tok.copy_(torch.randint(9000, (1, 60), device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    xs = [_rows(1, 200, 30000, BF, s).requires_grad_(True) for s in (1, 2)]
    lists = [_lists(x.detach(), 30, 4) for x in xs]
    want = [_both(x, ids[..., 0], ids, lq) for x, (ids, lq) in zip(xs, lists)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [None, None]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _both(xs[i], lists[i][0][..., 0], *lists[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_gradients_of_gradients_and_tensor_temperatures():
    from lm_engine_b200.ops import token_logprobs, topk_distillation

    x = _rows(1, 4, 50, F32, 2).requires_grad_(True)
    ids, lq = _lists(x.detach(), 5, 4)

    def twice(v, ids, lq):
        out, kl = token_logprobs(v, ids[..., 0], top_k=2), topk_distillation(v, ids, lq, ids[..., 1])
        total = out.logprobs.sum() + out.entropy.sum() + out.top_logprobs.sum() + kl.kl_divergence.sum() + kl.nll.sum()
        (g,) = torch.autograd.grad(total, v, create_graph=True)
        (h,) = torch.autograd.grad(g.square().sum(), v)
        return g, h

    x64 = x.detach().double().requires_grad_(True)
    for a, b in zip(twice(x, ids, lq), twice(x64, ids, lq)):
        assert float((a.double() - b).norm() / b.norm()) < 2.0 ** -16       # (a chain of some tens of fp32 operations)
    t = torch.tensor(1.5, device="cuda", requires_grad=True)
    out = token_logprobs(x, ids[..., 0], temperature=t)
    assert torch.autograd.grad(out.entropy.sum(), t)[0].isfinite()


def test_a_second_backward_pass_and_saved_tensors_elsewhere():
    x = _rows(2, 30, 1003, BF, 2, "pitch").requires_grad_(True)
    ids, lq = _lists(x.detach(), 5, 4)
    d = [torch.randn(2, 30, device="cuda")] * 4

    def run():
        outs = _both(x, ids[..., 0], ids, lq)
        return [outs[0], outs[1], outs[3], outs[4]]

    outs = run()
    (a,) = torch.autograd.grad(outs, [x], d, retain_graph=True)
    (b,) = torch.autograd.grad(outs, [x], d)
    with torch.autograd.graph.save_on_cpu():
        outs = run()
    (c,) = torch.autograd.grad(outs, [x], d)
    assert torch.equal(a, b) and torch.equal(a, c)


def test_transforms_see_the_operations():
    from torch.fx.experimental.proxy_tensor import make_fx

    from lm_engine_b200.ops import token_logprobs

    x, tok = _rows(1, 4, 100, BF, 2)[0], torch.arange(4, device="cuda")
    f = lambda v: token_logprobs(v, tok, top_k=3)[:3]       # noqa: E731
    traced = make_fx(f)(x)
    other = _rows(1, 4, 100, BF, 5)[0]
    for a, b in zip(traced(other), f(other)):
        assert float((a - b).abs().max()) < 2.0 ** -16


def test_a_long_batch_passes_32_bits():
    """Rows whose offsets pass 2^32 elements."""
    from lm_engine_b200.ops import token_logprobs

    V, rows = 131072, 33000
    x = torch.zeros(rows, V, dtype=BF, device="cuda")
    tok = torch.arange(rows, device="cuda")
    x[tok, tok] = 9.0
    out = token_logprobs(x, tok, top_k=2)
    want = 9 - math.log(math.exp(9) + V - 1)
    assert float((out.logprobs - want).abs().max()) < _sum_error(V) + 2.0 ** -22
    assert torch.equal(out.top_ids[:, 0], tok) and torch.equal(out.top_ids[1:, 1], torch.zeros_like(tok[1:]))


@pytest.mark.parametrize("rows", [1, 500])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_rows_whose_logits_leave_the_range_of_their_first_ones(rows, dtype):
    """A thread's sums run over (values hundreds above its first ones), meet minus infinity or the type's lowest late in the
    row, or begin with them."""
    V = 30011
    x = _rows(1, rows, V, dtype, 11)
    tok = torch.full((1, rows), V - 3, device="cuda")
    ids, lq = _lists(x, 12, 2)
    low = torch.finfo(dtype).min
    cases = []
    for first in (-400.0, -90.0):
        y = x.clone()
        y[..., : 2 * V // 3] += first
        cases.append(y)
    y = x.clone()
    y[..., V // 2:] += 300.0
    y[..., ::7] = -math.inf
    cases.append(y)
    for value in (-math.inf, low):
        y = x.clone()
        y[..., 17000:] = value
        cases.append(y)
        y = x.clone()
        y[..., :17000] = value
        cases.append(y)
    y = torch.full_like(x, low)                     # all forbidden by the lowest value: as likely as each other
    cases.append(y)
    y = y.clone()
    y[..., 5::2] = -math.inf
    cases.append(y)
    if dtype != HF:
        cases.append(x + 4000)
    for y in cases:
        y = y.clone()
        y[..., V - 3] = y[..., :].amax(-1)
        _score(y, tok, 20, 1.0)
        _score(y, tok, 0, 0.7)
    for y in cases[:6]:
        y = y.clone()
        keep = y.gather(-1, ids)
        y.scatter_(-1, ids, torch.where(keep > -80, keep, 0.0).to(dtype))       # (listed ones stay likely: finite losses)
        _distill(y, ids, lq, ids[..., 0], "backward", False, 2.0)
        _distill(y, ids, lq, ids[..., 0], "backward", False, 1.3)
        _distill(y, ids, lq, None, "forward", True, 1.0)


@pytest.mark.parametrize("rows,V", [(700, 9001), (2000, 12001)])
def test_many_calls_give_the_same_bits(rows, V):
    """Stages of the ring are requested again while their last values are in use nearby."""
    from lm_engine_b200.ops import token_logprobs, topk_distillation

    x = _rows(1, rows, V, F32, 3)
    ids, lq = _lists(x, 16, 4)
    first = None
    for _ in range(300):
        a = [*token_logprobs(x, ids[..., 0], top_k=1), *topk_distillation(x, ids, lq, ids[..., 1])]
        first = first or a
        assert all(torch.equal(u, v) for u, v in zip(first, a))


def test_kernels_are_what_runs():
    from lm_engine_b200.ops import _lib, token_logprobs, topk_distillation

    for dtype in (BF, HF, F32):
        x = _rows(1, 3, 515, dtype, 1, "odd start").requires_grad_(True)
        ids, lq = _lists(x.detach(), 4, 1)
        before = _lib.launch_count
        token_logprobs(x, ids[..., 0], top_k=2).entropy.sum().backward()
        topk_distillation(x, ids, lq, ids[..., 0]).nll.sum().backward()
        assert _lib.launch_count == before + 4
    assert _lib.read_status()[0] == 0


def test_teacher_to_student():
    """The two together as a distillation step uses them: the teacher's best tokens, the loss, the student's gradient."""
    from lm_engine_b200.ops import token_logprobs, token_logprobs_reference, topk_distillation, topk_distillation_reference

    teacher, student = _rows(2, 100, 32000, BF, 1), _rows(2, 100, 32000, BF, 2).requires_grad_(True)
    labels = torch.randint(32000, (2, 100), device="cuda")
    labels[0, :40] = -100
    best = token_logprobs(teacher, top_k=64)
    out = topk_distillation(student, best.top_ids, best.top_logprobs, labels)
    (got,) = torch.autograd.grad(out.kl_divergence.mean() + out.nll.sum() / 160, student)
    x64 = student.detach().double().requires_grad_(True)
    t64 = token_logprobs_reference(teacher.double(), top_k=64)
    want = topk_distillation_reference(x64, t64.top_ids, t64.top_logprobs, labels)
    (ref,) = torch.autograd.grad(want.kl_divergence.mean() + want.nll.sum() / 160, x64)
    e = _sum_error(32000)
    assert torch.equal(best.top_ids, t64.top_ids)
    # the list's error reaches the divergence through its weights, times its logarithms (at most 2 log2 V)
    assert float((out.kl_divergence - want.kl_divergence).abs().max()) < 30 * e
    assert float((out.nll - want.nll).abs().max()) < e + 20 * 2.0 ** -23
    assert float((got.double() - ref).norm() / ref.norm()) < 2.0 ** -8      # half a step of bf16, and 30 e


@pytest.mark.parametrize("method", ["forward", "backward"])
def test_distillation_wrapper(method):
    from lm_engine_b200.model_wrapper.distillation import ModelWrapperForDistillation
    from lm_engine_b200.models import dense_config
    from lm_engine_b200.ops import _lib, token_logprobs_reference, topk_distillation_reference
    from lm_engine_b200.parallel.manager import ProcessGroupManager

    ProcessGroupManager.destroy_process_groups()
    ProcessGroupManager(zero_stage=0)
    torch.manual_seed(3)

    def cfg(hidden):
        return dense_config(vocab_size=512, hidden_size=hidden, num_layers=2, num_attention_heads=4, num_key_value_heads=2,
                            intermediate_size=256, head_dim=64, max_position_embeddings=64).to_dict()

    w = ModelWrapperForDistillation(
        pretrained_config=cfg(128), micro_batch_size=2, sequence_length=64, teacher_pretrained_config=cfg(256),
        teacher_model_dtype="bf16", kl_divergence_method=method, kl_divergence_weight=0.5, kl_divergence_top_k=32,
        dtype="bf16").cuda()
    w.place_teacher(torch.device("cuda"))
    tokens = torch.randint(0, 512, (2, 65), device="cuda")
    out = w(tokens, lm_loss_multiplier=1 / 128)
    out["loss"].backward()
    s, t = (m(input_ids=tokens[:, :-1]).logits.double() for m in (w.model, w.teacher_model))
    best = token_logprobs_reference(t, top_k=32)
    want = topk_distillation_reference(s, best.top_ids, best.top_logprobs, tokens[:, 1:], method)
    e = _sum_error(512) * 60
    assert abs(float(out["kl_divergence"]) - float(want.kl_divergence.mean())) < e
    assert abs(float(out["lm_loss"]) - float(want.nll.mean())) < e
    assert all(p.grad is not None and torch.isfinite(p.grad.float()).all() for p in w.model.parameters())
    assert all(p.grad is None for p in w.teacher_model.parameters()) and _lib.read_status()[0] == 0


@pytest.mark.parametrize("rows", [1, 450])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("V", [3001, 40001])
def test_alternatives_beside_outliers_and_masks(rows, dtype, V):
    """Values that stretch the range of a row's largest ones: masks by the type's lowest, outliers, both infinities."""
    x = _rows(1, rows, V, dtype, 21)
    low = torch.finfo(dtype).min
    for k in (1, 20, 128):
        y = x.clone()
        y[..., V // 3:] = low
        _score(y, None, k, 1.0, grads=False)
        y = x.clone()
        y[..., : V - 200] = low
        _score(y, None, k, 1.0, grads=False)
        y = x.clone()
        y[..., V // 2] = 30000.0
        y[..., V // 5] = -30000.0
        _score(y, None, k, 1.0, grads=False)
        y = torch.where(torch.arange(V, device="cuda") % 17 == 3, x, torch.tensor(low, device="cuda").to(dtype))
        _score(y, None, k, 1.0, grads=False)
        y = x * 0 - 5
        y[..., 7::50] = -4.0
        y[..., 8::50] = 3.0
        _score(y, None, k, 1.0, grads=False)
        y = x.clone()
        y[..., V // 7] = math.inf
        y[..., V // 3] = math.nan
        y[..., 2 * V // 3] = -math.inf
        _score(y, None, k, 1.0, grads=False)


def test_distillation_of_no_rows_and_of_long_rows():
    from lm_engine_b200.ops import topk_distillation

    x = _rows(1, 4, 300, BF, 1).requires_grad_(True)
    ids, lq = _lists(x.detach(), 4, 1)
    out = topk_distillation(x[:, :0], ids[:, :0], lq[:, :0], ids[:, :0, 0])
    assert out.kl_divergence.shape == out.nll.shape == (1, 0)
    (g,) = torch.autograd.grad(out.kl_divergence.sum() + out.nll.sum(), x)
    assert float(g.abs().max()) == 0
    x = _rows(1, 2, 1_200_003, BF, 1)
    ids, lq = _lists(x, 100, 1)
    _distill(x, ids, lq, ids[..., 7], "backward", True, 1.0)
    _score(x, ids[..., 3], 100, 1.0)


@pytest.mark.parametrize("offset", [0.0, 100.0])
def test_fp32_gradients_of_the_forward_divergence_are_fp32(offset):
    """Logits whose largest come late in a row, far above a thread's first: the gradient subtracts logarithms."""
    from lm_engine_b200.ops import topk_distillation, topk_distillation_reference

    x = _rows(1, 300, 20000, F32, 8) * 0.5
    x[..., 15000:] += 30.0
    x = (x + offset).requires_grad_(True)
    ids, lq = _lists(x.detach(), 20, 4)
    x64 = x.detach().double().requires_grad_(True)
    for temperature in (1.0, 2.0, 0.7):
        (got,) = torch.autograd.grad(topk_distillation(x, ids, lq, ids[..., 0], "forward", True, temperature)
                                     .kl_divergence.sum(), x)
        (ref,) = torch.autograd.grad(topk_distillation_reference(x64, ids, lq, ids[..., 0], "forward", True, temperature)
                                     .kl_divergence.sum(), x64)
        # p (log p - log q - KL): logarithms of at most 2^5, a few roundings of 2^-24 each, of terms that partly cancel
        assert float((got.double() - ref).norm() / ref.norm()) < 2.0 ** -24 * 2 ** 5 * 4


@pytest.mark.parametrize("temperature", [0.5, 0.6, 3.0, 50.0])
def test_labels_beside_other_temperatures(temperature):
    for dtype in (BF, F32):
        x = _rows(1, 40, 20003, dtype, 6)
        x[..., 9000:] += 4.0
        for method, tail in METHODS:
            ids, lq = _lists(x, 16, 2, tail, temperature)
            _distill(x, ids, lq, ids[..., 3], method, tail, temperature)


def test_upstream_gradients_of_rows_without_a_part_are_not_used():
    from lm_engine_b200.ops import token_logprobs, topk_distillation

    x = _rows(1, 4, 700, BF, 1).requires_grad_(True)
    ids, lq = _lists(x.detach(), 6, 2)
    ids[0, 0] = ids[0, 1] = -1
    labels = torch.tensor([[3, -100, -100, 5]], device="cuda")
    out = topk_distillation(x, ids, lq, labels)
    nan = math.nan
    d_kl, d_nll = torch.tensor([[nan, nan, 1.0, 1.0]], device="cuda"), torch.tensor([[1.0, nan, nan, 1.0]], device="cuda")
    (g,) = torch.autograd.grad([out.kl_divergence, out.nll], [x], [d_kl, d_nll])
    assert g.isfinite().all() and float(g[0, 1].abs().max()) == 0 and float(g[0, 0].abs().max()) > 0
    (g,) = torch.autograd.grad([token_logprobs(x, labels).logprobs], [x], [d_nll])
    assert g.isfinite().all() and float(g[0, 1:3].abs().max()) == 0


@pytest.mark.parametrize("gap", [60.0, 100.0, 300.0, 2000.0])
@pytest.mark.parametrize("method,tail", METHODS)
def test_lists_that_hold_all_but_nothing(gap, method, tail):
    """What is not listed is less likely than fp32 or fp64 can say; its gradient is the teacher's rest all the same."""
    V = 5003
    for dtype, temperature in ((F32, 1.0), (BF, 2.0), (F32, 0.7)):
        x = _rows(1, 12, V, dtype, 4) - gap
        ids, lq = _lists(x, 10, 3, tail, temperature)
        x = x.scatter(-1, ids, x.gather(-1, ids) + gap)
        lq = lq - 0.05 if tail else lq
        _distill(x, ids, lq, ids[..., 1], method, tail, temperature)
    x = _rows(1, 3, V, F32, 4)
    x[0, 1] = -math.inf
    from lm_engine_b200.ops import topk_distillation

    leaf = x.requires_grad_(True)
    out = topk_distillation(leaf, ids[:, :3], lq[:, :3], None, method, tail)
    (g,) = torch.autograd.grad(out.kl_divergence.sum(), leaf)
    assert out.kl_divergence[0, 1].isnan() and g[0, 1].isnan().all() and g[0, 0].isfinite().all()


@pytest.mark.parametrize("V,k,layout", [(15, 15, "odd start"), (32, 5, "pitch"), (64, 5, "dense"), (1187, 87, "odd start")])
def test_alternatives_of_many_short_rows(V, k, layout):
    """More rows than CTAs at once, their ends read element by element."""
    from lm_engine_b200.ops import token_logprobs, token_logprobs_reference

    x = _rows(1, 2500, V, BF, 3, layout)
    want = token_logprobs_reference(x.double(), None, k).top_ids
    for _ in range(50):
        assert torch.equal(token_logprobs(x, None, top_k=k).top_ids, want)
