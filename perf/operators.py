"""Scoring tokens from logits and distilling from a teacher's top alternatives: what is measured of the two operators.

Kinds of a case:

``score``    log probabilities of given tokens, the entropy of every position and its ``k`` best alternatives
``policy``   the same with the gradient of the logits from given gradients of the log probabilities and entropies
``distill``  Kullback-Leibler divergence between a student and the ``k`` best tokens of a teacher (with or without a
             bucket for the rest of the vocabulary), the cross entropy of the labels, and the gradient of the logits

A case's ``tokens`` are all positions (``batch`` sequences together), ``vocab`` the vocabulary, ``type`` the logits' type.
``shift`` means that the logits are those of every position but the last of each sequence, read in place.  ``banned`` is the
share of the vocabulary that a grammar or a padded vocabulary forbids (logits of minus infinity).
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = 8192 * 128256


def listed() -> list[dict]:
    return [
        # a served request: the token just sampled, with twenty alternatives for the client
        dict(name="score-1x128256-top20", kind="score", batch=1, tokens=1, vocab=128256, type="bf16", k=20,
             temperature=0.7, shift=False, banned=0.0),
        # a batch of served sequences whose sampler works in fp32 on a vocabulary of odd size; a grammar bans a tenth of it
        dict(name="score-24x50257-top5-fp32", kind="score", batch=24, tokens=24, vocab=50257, type="fp32", k=5,
             temperature=1.0, shift=False, banned=0.1),
        # the likelihood of one short document, read in place from the logits of all of its positions
        dict(name="score-333x32000", kind="score", batch=1, tokens=333, vocab=32000, type="bf16", k=0, temperature=1.0,
             shift=True, banned=0.0),
        # evaluation of two sequences of a 128k-vocabulary model
        dict(name="score-4094x128256", kind="score", batch=2, tokens=4094, vocab=128256, type="bf16", k=0,
             temperature=1.0, shift=True, banned=0.0),
        # a teacher's pass: the best 64 tokens of every position are all that is kept of it
        dict(name="score-4096x128256-top64", kind="score", batch=1, tokens=4096, vocab=128256, type="bf16", k=64,
             temperature=1.0, shift=False, banned=0.0),
        # policy gradient on a short rollout, vocabulary of odd size, fp16
        dict(name="policy-777x50257-fp16", kind="policy", batch=1, tokens=777, vocab=50257, type="fp16", k=0,
             temperature=1.0, shift=False, banned=0.0),
        # policy gradient at a training batch, sampling temperature below one
        dict(name="policy-4096x128256", kind="policy", batch=2, tokens=4096, vocab=128256, type="bf16", k=0,
             temperature=0.8, shift=False, banned=0.0),
        # distillation of one short document in fp32
        dict(name="distill-250x32000-top32-fp32", kind="distill", batch=1, tokens=250, vocab=32000, type="fp32", k=32,
             method="backward", tail=True, labels=True, temperature=1.0, shift=False, banned=0.0),
        # distillation towards the student's own modes, vocabulary of odd size
        dict(name="distill-2047x50257-top20", kind="distill", batch=1, tokens=2047, vocab=50257, type="bf16", k=20,
             method="forward", tail=True, labels=True, temperature=1.0, shift=False, banned=0.0),
        # stored teacher logits without the rest of the vocabulary, softened student, labels at temperature one
        dict(name="distill-4096x128256-top100", kind="distill", batch=1, tokens=4096, vocab=128256, type="bf16", k=100,
             method="backward", tail=False, labels=True, temperature=2.0, shift=False, banned=0.0),
        # the distillation loss of a training batch of a 128k-vocabulary model
        dict(name="distill-8192x128256-top64", kind="distill", batch=2, tokens=8192, vocab=128256, type="bf16", k=64,
             method="backward", tail=True, labels=True, temperature=1.0, shift=False, banned=0.0),
    ]


def _spread(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["score", "score", "policy", "distill", "distill"])
    vocab = rng.choice([32000, 50257, 50304, 128256, _spread(rng, 1000, 200000)])
    type_ = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    tokens = _spread(rng, 1, min(8192, LARGEST // vocab // (2 if type_ == "fp32" else 1)))
    case = dict(kind=kind, batch=2 if tokens % 2 == 0 and tokens > 2 and rng.random() < 0.5 else 1, tokens=tokens,
                vocab=vocab, type=type_, k=rng.choice([0, 1, 5, 20, _spread(rng, 2, 100)]) if kind == "score" else 0,
                temperature=rng.choice([1.0, 1.0, 0.7, 1.5]), shift=rng.random() < 0.3,
                banned=rng.choice([0.0, 0.0, 0.2]))
    if kind == "distill":
        method = rng.choice(["forward", "backward"])
        case.update(k=_spread(rng, 1, 100), method=method, tail=method == "forward" or rng.random() < 0.6,
                    labels=rng.random() < 0.7)
    return case


# ------------------------------------------------------------------------------------------------------ inputs
def _model_logits(g, shape, banned):
    """Logits as a trained model has them: a broad background, and some tokens per position that stand out."""
    x = torch.randn(shape, generator=g, device=DEV).mul_(2.0)
    peaks = torch.randint(shape[-1], (*shape[:-1], min(24, shape[-1])), generator=g, device=DEV)
    height = 6 + 9 * torch.rand(peaks.shape, generator=g, device=DEV).square_()
    x.scatter_reduce_(-1, peaks, height, "amax")
    if banned is not None:
        x.masked_fill_(banned, -math.inf)
    return x


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, S, V, dt = case["batch"], case["tokens"] // case["batch"], case["vocab"], TYPES[case["type"]]
    banned = torch.rand(V, generator=g, device=DEV) < case["banned"] if case["banned"] else None
    shape = (B, S + 1, V) if case["shift"] else (B, S, V)
    if case["kind"] == "distill":
        teacher = _model_logits(g, shape, banned)
        logits = teacher.clone().add_(torch.randn(shape, generator=g, device=DEV)).to(dt)
        teacher = teacher[:, :-1] if case["shift"] else teacher
        best, ids = teacher.topk(case["k"], dim=-1)
        if case["tail"]:                        # log probabilities over the whole vocabulary, at the loss's temperature
            best = best / case["temperature"] - (teacher / case["temperature"]).logsumexp(-1, keepdim=True)
        del teacher
    else:
        logits = _model_logits(g, shape, banned).to(dt)
    logits = logits[:, :-1] if case["shift"] else logits
    state = dict(case=case)
    allowed = torch.arange(V, device=DEV) if banned is None else (~banned).nonzero()[:, 0]
    tokens = allowed[torch.randint(len(allowed), (B, S), generator=g, device=DEV)]
    likely = torch.rand(B, S, generator=g, device=DEV) < 0.7
    tokens = torch.where(likely, logits.argmax(-1), tokens)
    tokens[torch.rand(B, S, generator=g, device=DEV) < 0.06] = IGNORE       # prompts and padding
    if case["kind"] == "distill":
        ids[tokens == IGNORE] = -1              # nothing is distilled there either
        state.update(top_ids=ids, top_logprobs=best, labels=tokens if case["labels"] else None,
                     d_kl=torch.rand(B, S, generator=g, device=DEV) + 0.5,
                     d_nll=torch.rand(B, S, generator=g, device=DEV) + 0.5)
    else:
        state["tokens"] = tokens
        if case["kind"] == "policy":
            state.update(d_logprobs=torch.randn(B, S, generator=g, device=DEV),
                         d_entropy=0.1 * torch.rand(B, S, generator=g, device=DEV))
    state["logits"] = logits.detach().requires_grad_(case["kind"] != "score")
    return state


# ------------------------------------------------------------------------------------------------------ one pass
def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s: dict):
    from lm_engine_b200 import ops

    c, x = s["case"], s["logits"]
    if c["kind"] == "distill":
        out = ops.topk_distillation(x, s["top_ids"], s["top_logprobs"], s["labels"], kl_divergence_method=c["method"],
                                    tail=c["tail"], temperature=c["temperature"], ignore_index=IGNORE)
        if s["labels"] is None:
            (grad,) = torch.autograd.grad([out.kl_divergence], [x], [s["d_kl"]])
            return dict(kl_divergence=out.kl_divergence, grad=grad)
        (grad,) = torch.autograd.grad([out.kl_divergence, out.nll], [x], [s["d_kl"], s["d_nll"]])
        return dict(kl_divergence=out.kl_divergence, nll=out.nll, grad=grad)
    out = ops.token_logprobs(x, s["tokens"], top_k=c["k"], temperature=c["temperature"], ignore_index=IGNORE)
    got = dict(logprobs=out.logprobs, entropy=out.entropy)
    if c["kind"] == "policy":
        (got["grad"],) = torch.autograd.grad([out.logprobs, out.entropy], [x], [s["d_logprobs"], s["d_entropy"]])
    if c["k"]:
        got.update(top_logprobs=out.top_logprobs, top_ids=out.top_ids)
    return got


def _log_softmax(x):
    """Logarithms of the softmax along the last dimension, the largest first taken away."""
    d = x - x.amax(-1, keepdim=True)
    return d - d.exp().sum(-1, keepdim=True).log()


def _best(x, k):
    """Places of the ``k`` largest values in order, the lowest place first among equal ones: the value's bits as an ordered
    integer in the upper half of a key, the place counted down in the lower."""
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    place = torch.arange(x.size(-1), device=x.device)
    return 0xFFFFFFFF - ((bits << 32) + (0xFFFFFFFF - place)).topk(k, dim=-1).values.bitwise_and_(0xFFFFFFFF)


@torch.no_grad()
def _run_plain(s: dict):
    c = s["case"]
    return _plain_distill(s, c) if c["kind"] == "distill" else _plain_score(s, c)


def _plain_score(s, c):
    x = s["logits"].float()
    logp = _log_softmax(x / c["temperature"])
    valid = s["tokens"] != IGNORE
    at = torch.where(valid, s["tokens"], 0)[..., None]
    p = logp.exp()
    p_logp = torch.where(p > 0, p * logp, 0.0)
    got = dict(logprobs=torch.where(valid, logp.gather(-1, at)[..., 0], 0.0), entropy=-p_logp.sum(-1))
    if c["k"]:
        ids = _best(x, c["k"])
        got.update(top_logprobs=logp.gather(-1, ids), top_ids=ids)
    if c["kind"] == "policy":
        g_tok = torch.where(valid, s["d_logprobs"], 0.0)[..., None]
        g_ent = s["d_entropy"][..., None]
        grad = -(g_tok + g_ent * got["entropy"][..., None]) * p - g_ent * p_logp
        grad.scatter_add_(-1, at, g_tok)
        got["grad"] = (grad / c["temperature"]).to(s["logits"].dtype)
    return got


#: A teacher's mass outside of its listed tokens is 1 - their sum; below this it is the rounding of that sum.
NO_TAIL = 2.0 ** -20


def _plain_distill(s, c):
    x = s["logits"].float()
    logp = _log_softmax(x / c["temperature"])
    there = s["top_ids"] >= 0
    at = torch.where(there, s["top_ids"], 0)
    some = there.any(-1)
    # the listed tokens: a handful per row, in 64 bits
    s_top = torch.where(there, logp.gather(-1, at), -math.inf).double()
    t_top = torch.where(there, s["top_logprobs"].double(), -math.inf)
    listed = torch.zeros_like(logp, dtype=torch.bool).scatter_(-1, at, there)
    p = logp.exp()
    p_rest = torch.where(listed, 0.0, p).sum(-1).double()
    if not c["tail"]:
        t_top = t_top - torch.where(some, t_top.logsumexp(-1), 0.0)[..., None]
    q = t_top.exp()
    q_rest = torch.where(1 - q.sum(-1) < NO_TAIL, 0.0, 1 - q.sum(-1)) if c["tail"] else torch.zeros_like(p_rest)
    if c["method"] == "backward":
        kl = torch.where(q > 0, q * (t_top - s_top), 0.0).sum(-1)
        kl = kl + torch.where(q_rest > 0, q_rest * (q_rest.log() - p_rest.log()), 0.0)
        rest = torch.where(p_rest > 0, q_rest / p_rest, 0.0)
        grad_rest = (q.sum(-1) + q_rest - rest).float()[..., None] * p
        grad_top = (s_top.exp() * (q.sum(-1) + q_rest)[..., None] - q).float()
    else:
        away = torch.where(there & (s_top > -math.inf), s_top - t_top, 0.0)
        rest = p_rest.log() - q_rest.clamp(min=NO_TAIL).log()
        kl = (s_top.exp() * away).sum(-1) + torch.where(p_rest > 0, p_rest * rest, 0.0)
        rest = torch.where(p_rest > 0, rest, 0.0)
        grad_rest = (rest - kl).float()[..., None] * p
        grad_top = (s_top.exp() * (away - kl[..., None])).float()
    kl = torch.where(some, kl, 0.0).float()
    grad = torch.where(listed, 0.0, grad_rest).scatter_add_(-1, at, torch.where(there, grad_top, 0.0))
    del p, grad_rest, listed
    grad.mul_(torch.where(some, s["d_kl"], 0.0)[..., None] / c["temperature"])
    got = dict(kl_divergence=kl)
    if s["labels"] is not None:
        valid = s["labels"] != IGNORE
        at = torch.where(valid, s["labels"], 0)[..., None]
        logp = _log_softmax(x) if c["temperature"] != 1 else logp
        g = torch.where(valid, s["d_nll"], 0.0)[..., None]
        got["nll"] = torch.where(valid, -logp.gather(-1, at)[..., 0], 0.0)
        grad.add_(g * logp.exp()).scatter_add_(-1, at, -g)
    got["grad"] = grad.to(s["logits"].dtype)
    return got


# ------------------------------------------------------------------------------------------------------ floors
def work(case: dict) -> dict:
    """Logits read once, their gradient written once, and the small operands.  Per logit: the difference to the largest,
    the exponential, two sums, and for a gradient the exponential again with its factors."""
    n, size = case["tokens"] * case["vocab"], 4 if case["type"] == "fp32" else 2
    moved, flops = n * size + case["tokens"] * 16, 5 * n
    if case["kind"] == "score":
        moved += case["tokens"] * case["k"] * 12
    else:
        moved, flops = moved + n * size + case["tokens"] * 8, 10 * n
    if case["kind"] == "distill":
        moved += case["tokens"] * case["k"] * 12
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------------------------------ 64 bits
def exact(case: dict, seed: int):
    """The definitions in 64 bits, gradients by differentiation; a block of rows at a time."""
    s = prepare(case, seed)
    rows = max(1, (1 << 26) // case["vocab"])
    flat = {k: v.reshape(case["tokens"], *v.shape[2:]) if isinstance(v, torch.Tensor) and k != "logits" else v
            for k, v in s.items()}
    x = s["logits"].detach().reshape(case["tokens"], case["vocab"])
    parts = []
    for a in range(0, case["tokens"], rows):
        part = {k: v[a:a + rows] if isinstance(v, torch.Tensor) and k != "logits" else v for k, v in flat.items()}
        parts.append((_exact_distill if case["kind"] == "distill" else _exact_score)(
            case, x[a:a + rows].double().requires_grad_(True), part))
    B = case["batch"]
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    out = {k: v.reshape(B, case["tokens"] // B, *v.shape[1:]) for k, v in out.items()}
    if case["kind"] != "distill" and case["k"]:
        out["top_ids"] = None
    return out


def _exact_score(case, x, s):
    logp = torch.log_softmax(x / case["temperature"], -1)
    kept = s["tokens"] != IGNORE
    picked = torch.zeros_like(logp[:, 0])
    picked[kept] = logp[kept, s["tokens"][kept]]
    entropy = -(logp.exp() * logp.clamp(min=-1e9)).sum(-1)
    out = dict(logprobs=picked.detach(), entropy=entropy.detach())
    if case["kind"] == "policy":
        ((picked * s["d_logprobs"].double()).sum() + (entropy * s["d_entropy"].double()).sum()).backward()
        out["grad"] = x.grad
    if case["k"]:
        out["top_logprobs"] = logp.detach().sort(-1, descending=True).values[:, :case["k"]].clone()
    return out


def _exact_distill(case, x, s):
    T, V = x.shape
    logp = torch.log_softmax(x / case["temperature"], -1)
    kept = s["top_ids"][:, 0] >= 0
    ids = s["top_ids"][kept]
    teacher, student = s["top_logprobs"][kept].double(), logp[kept].gather(1, ids)
    others = torch.ones(len(ids), V, dtype=torch.bool, device=x.device)
    others[torch.arange(len(ids), device=x.device)[:, None], ids] = False
    rest = torch.where(others, logp[kept].exp(), 0.0).sum(1)
    if case["tail"]:
        left = 1 - teacher.exp().sum(1)
        none = left < NO_TAIL
    else:
        teacher = torch.log_softmax(teacher, 1)
    if case["method"] == "backward":
        kl = torch.nn.functional.kl_div(student.clamp(min=-1e300), teacher, reduction="none", log_target=True).sum(1)
        if case["tail"]:
            kl = kl + torch.where(none, 0.0, left * (left.clamp(min=NO_TAIL).log() - rest.clamp(min=1e-300).log()))
    else:
        left = torch.where(none, NO_TAIL, left)
        kl = (student.exp() * (student.clamp(min=-1e300) - teacher.clamp(min=-1e300))).sum(1)
        kl = kl + rest * (rest.clamp(min=1e-300).log() - left.log())
    all_kl = torch.zeros(T, dtype=x.dtype, device=x.device)
    all_kl[kept] = kl
    total = (all_kl * s["d_kl"].double()).sum()
    out = dict(kl_divergence=all_kl.detach())
    if s["labels"] is not None:
        nll = torch.nn.functional.cross_entropy(x, s["labels"], ignore_index=IGNORE, reduction="none")
        total = total + (nll * s["d_nll"].double()).sum()
        out["nll"] = nll.detach()
    if total.requires_grad:
        total.backward()
    out["grad"] = x.grad if x.grad is not None else torch.zeros_like(x)
    return out
