"""Token log probabilities and distillation from a teacher's best tokens: the PyTorch statements against formulas written
apart and against differences, and what the entry points refuse."""

import math

import pytest
import torch

from lm_engine_b200.enums import KLDivergenceMethod
from lm_engine_b200.ops import token_logprobs, topk_distillation
from lm_engine_b200.ops.logprobs import logit_rows

F64 = torch.float64


def _logits(*shape, seed=0):
    return 2 * torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=F64)


def test_scores_by_the_definition():
    x, tok = _logits(2, 3, 11), torch.tensor([[0, 10, -100], [4, 11, 7]])
    x[0, 1, 3] = -math.inf
    out = token_logprobs(x, tok, top_k=4, temperature=0.5)
    for b in range(2):
        for s in range(3):
            w = [math.exp(float(v) / 0.5) for v in x[b, s]]
            p = [v / sum(w) for v in w]
            order = sorted(range(11), key=lambda j: (-float(x[b, s, j]), j))[:4]
            assert out.top_ids[b, s].tolist() == order
            assert out.top_logprobs[b, s].tolist() == pytest.approx([math.log(p[j]) for j in order], rel=1e-12)
            assert float(out.entropy[b, s]) == pytest.approx(-sum(v * math.log(v) for v in p if v > 0), rel=1e-12)
            t = int(tok[b, s])
            got = float(out.logprobs[b, s])
            if t == -100:
                assert got == 0
            elif t == 11:
                assert math.isnan(got)
            else:
                assert got == pytest.approx(math.log(p[t]), rel=1e-12)


def test_equal_logits_go_by_their_ids():
    x = torch.zeros(2, 9)
    x[0, 5] = -0.0
    x[1, 2] = x[1, 7] = 1.0
    out = token_logprobs(x, top_k=4)
    assert out.logprobs is None
    assert out.top_ids.tolist() == [[0, 1, 2, 3], [2, 7, 0, 1]]
    x[1, 4] = math.nan
    assert token_logprobs(x, top_k=2).top_ids[1].tolist() == [4, 2]


@pytest.mark.parametrize("banned", [False, True])
def test_score_gradients_against_differences(banned):
    x, tok = _logits(3, 7, seed=1), torch.tensor([2, -100, 6])
    fixed = torch.zeros(3, 7, dtype=torch.bool)
    if banned:
        fixed[:, 1] = True

    def f(y):
        out = token_logprobs(y.masked_fill(fixed, -math.inf), tok, top_k=2, temperature=1.3)
        return out.logprobs, out.entropy, out.top_logprobs

    assert torch.autograd.gradcheck(f, x.requires_grad_(True))


def _divergence(x, ids, lq, method, tail, temperature):
    """One position, by the definition, in plain floats."""
    w = [math.exp(float(v) / temperature) for v in x]
    p = [v / sum(w) for v in w]
    entries = {}
    for i, v in zip(ids.tolist(), lq.tolist()):
        if 0 <= i < len(p) and v > -math.inf and i not in entries:
            entries[i] = v
    if not entries:
        return 0.0
    if not tail:
        total = sum(math.exp(v) for v in entries.values())
        entries = {i: v - math.log(total) for i, v in entries.items()}
    q = {i: math.exp(v) for i, v in entries.items()}
    p_rest = sum(v for j, v in enumerate(p) if j not in q)
    q_rest = 1 - sum(q.values()) if tail else 0.0
    q_rest = 0.0 if q_rest < 2 ** -20 else q_rest
    if method == "backward":
        kl = sum(q[i] * (entries[i] - math.log(p[i])) for i in q)
        return kl + (q_rest * math.log(q_rest / p_rest) if q_rest else 0.0)
    kl = sum(p[i] * (math.log(p[i]) - entries[i]) for i in q)
    return kl + (p_rest * math.log(p_rest / max(q_rest, 2 ** -20)) if p_rest else 0.0)


CASES = [("backward", True), ("backward", False), ("forward", True)]


def _lists(V):
    g = torch.Generator().manual_seed(3)
    teacher = torch.log_softmax(2 * torch.randn(6, V, generator=g, dtype=F64), -1)
    lq, ids = teacher.topk(4, -1)
    ids[1] = -1                                        # nothing
    ids[2, 1] = V                                      # outside
    lq[2, 3] = -math.inf                               # no value
    ids[3, 2], ids[3, 3] = ids[3, 0], ids[3, 0]        # given again
    lq[4] = lq[4] - lq[4].logsumexp(-1)                # nothing left for the others
    return ids, lq


@pytest.mark.parametrize("method,tail", CASES)
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_divergence_by_the_definition(method, tail, temperature):
    V = 9
    x, (ids, lq) = _logits(6, V, seed=2), _lists(V)
    labels = torch.tensor([0, 3, -100, 8, 9, 1])
    out = topk_distillation(x, ids, lq, labels, method, tail, temperature)
    want = [_divergence(x[i], ids[i], lq[i], method, tail, temperature) for i in range(6)]
    assert out.kl_divergence.tolist() == pytest.approx(want, rel=1e-9, abs=1e-12)
    nll = torch.nn.functional.cross_entropy(x[[0, 1, 3, 5]], labels[[0, 1, 3, 5]], reduction="none")
    assert torch.equal(out.nll[[0, 1, 3, 5]], nll) and float(out.nll[2]) == 0 and out.nll[4].isnan()
    assert topk_distillation(x, ids, lq, None, method, tail, temperature).nll is None


@pytest.mark.parametrize("method,tail", CASES)
def test_divergence_gradients_against_differences(method, tail):
    V = 9
    x, (ids, lq) = _logits(6, V, seed=4).requires_grad_(True), _lists(V)
    labels = torch.tensor([0, -100, -100, 8, 2, 1])
    assert torch.autograd.gradcheck(lambda y: tuple(topk_distillation(y, ids, lq, labels, method, tail, 1.7)), x)


def test_divergence_of_a_model_from_itself_is_zero():
    x = _logits(5, 40, seed=5)
    best = token_logprobs(x, top_k=40)
    for k in (1, 7, 40):
        for method, tail in CASES:
            if not tail and k < 40:
                continue
            out = topk_distillation(x, best.top_ids[:, :k], best.top_logprobs[:, :k], None, method, tail)
            assert float(out.kl_divergence.abs().max()) < 1e-12


def test_rows_without_loss_are_not_looked_at():
    x = _logits(2, 5)
    x[1] = math.nan
    x.requires_grad_(True)
    ids, lq = torch.tensor([[0], [-1]]), torch.tensor([[-1.0], [-1.0]])
    out = topk_distillation(x, ids, lq, torch.tensor([1, -100]))
    (g,) = torch.autograd.grad(out.kl_divergence.sum() + out.nll.sum(), x)
    assert float(out.kl_divergence[1].detach()) == float(out.nll[1].detach()) == 0 and torch.equal(g[1], torch.zeros(5, dtype=F64))


def test_places_of_rows():
    big = torch.arange(4 * 6 * 10.0).view(4, 6, 10)
    for t in (big, big[:, :-1], big[1], big[:, 2], big[..., 1:8], big[2:3, :, :9], big[None, :, 1:], big[:, :1],
              big[:1, :1, 3:5], big.permute(1, 0, 2), big.transpose(1, 2), big[..., 0, :1], torch.zeros(3)):
        x, inner, a, b = logit_rows(t)
        flat = x.as_strided((x.untyped_storage().size() // 4,), (1,), 0)
        V = t.size(-1)
        for r, want in enumerate(t.reshape(-1, V)):
            at = x.storage_offset() + (r // inner) * b + (r % inner) * a
            assert torch.equal(flat[at:at + V], want)
    assert logit_rows(big[:, :-1])[0].data_ptr() == big.data_ptr()          # read in place


def test_refusals():
    x, tok = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.long)
    ids, lq = torch.zeros(2, 3, 4, dtype=torch.long), torch.zeros(2, 3, 4)
    for bad in (lambda: token_logprobs(torch.zeros(2, 0)), lambda: token_logprobs(x.long(), tok),
                lambda: token_logprobs(x, tok[:1]), lambda: token_logprobs(x, tok.float()),
                lambda: token_logprobs(x, tok > 0), lambda: token_logprobs(x, tok, top_k=9),
                lambda: token_logprobs(torch.zeros(2, 500), top_k=129), lambda: token_logprobs(x, tok, top_k=-1),
                lambda: token_logprobs(x, tok, temperature=0.0), lambda: token_logprobs(x, tok, temperature=-1.0),
                lambda: token_logprobs(x, tok, temperature=math.nan), lambda: token_logprobs(x, tok, temperature=math.inf),
                lambda: topk_distillation(x, ids[:, :2], lq), lambda: topk_distillation(x, ids.float(), lq),
                lambda: topk_distillation(x, ids, lq[..., :3]), lambda: topk_distillation(x, ids, lq.long()),
                lambda: topk_distillation(x, ids[..., :0], lq[..., :0]),
                lambda: topk_distillation(x, ids[..., :1].expand(2, 3, 129), lq[..., :1].expand(2, 3, 129)),
                lambda: topk_distillation(x, ids, lq, tok[..., None]), lambda: topk_distillation(x, ids, lq, tok.double()),
                lambda: topk_distillation(x, ids, lq, kl_divergence_method="sideways"),
                lambda: topk_distillation(x, ids, lq, kl_divergence_method=KLDivergenceMethod.forward, tail=False),
                lambda: topk_distillation(x, ids, lq, temperature=0.0), lambda: topk_distillation(x[0, 0, 0], ids, lq)):
        with pytest.raises(ValueError):
            bad()


def test_entry_points_refuse_on_the_host():
    """Sizes that no kernel may see come back as errors before anything is launched."""
    from lm_engine_b200.ops import _lib

    if torch.cuda.is_available():
        pytest.skip("the CPU's run shows it")
    lib = _lib.cuda_lib()
    for bad in (dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(inner=0), dict(V=0), dict(k=129), dict(k=9), dict(k=-1),
                dict(temperature=0.0), dict(temperature=math.nan)):
        a = {**dict(dtype=0, rows=1, inner=1, V=8, k=2, temperature=1.0), **bad}
        assert lib.lme_token_logprobs_fwd(None, a["dtype"], a["rows"], a["inner"], 8, 8, a["V"], None, -100,
                                          a["temperature"], a["k"], None, None, None, None, None, None) == -1
    for bad in (dict(k=0), dict(k=129), dict(V=0), dict(dtype=5), dict(forward=1, tail=0), dict(temperature=-1.0)):
        a = {**dict(dtype=0, V=8, k=2, temperature=1.0, forward=0, tail=1), **bad}
        assert lib.lme_topk_distillation_fwd(None, a["dtype"], 1, 1, 8, 8, a["V"], None, None, a["k"], None, -100,
                                             a["temperature"], a["forward"], a["tail"], None, None, None, None, None) == -1
    assert lib.lme_token_logprobs_fwd(None, 0, 1, 1, 8, 8, (1 << 30) + 1, None, -100, 1.0, 0, None, None, None, None, None,
                                      None) == -6
    assert lib.lme_token_logprobs_fwd(None, 0, 1 << 31, 1, 8, 8, 8, None, -100, 1.0, 0, None, None, None, None, None,
                                      None) == -6
    # nothing to write to, and statistics that are not on 16 bytes
    assert lib.lme_token_logprobs_fwd(None, 0, 1, 1, 8, 8, 8, None, -100, 1.0, 0, None, None, None, None, None, None) == -1
    assert lib.lme_token_logprobs_fwd(16, 0, 1, 1, 8, 8, 8, None, -100, 1.0, 2, None, 16, None, 16, None, None) == -1
    assert lib.lme_token_logprobs_fwd(16, 0, 1, 1, 8, 8, 8, None, -100, 1.0, 0, None, 16, None, None, 8, None) == -2
    assert lib.lme_token_logprobs_bwd(16, 0, 1, 1, 8, 8, 8, None, -100, 1.0, 0, None, None, None, None, None, 16, None) == -1
    assert lib.lme_topk_distillation_bwd(16, 0, 1, 1, 8, 8, 8, None, 16, 2, None, -100, 1.0, 0, 16, None, None, 16, None) == -1
    assert lib.lme_token_logprobs_fwd(None, 0, 0, 1, 8, 8, 8, None, -100, 1.0, 0, None, None, None, None, None, None) == 0


def _wrapper(top_k, method, tail=True):
    from lm_engine_b200.model_wrapper.distillation import ModelWrapperForDistillation
    from lm_engine_b200.models import dense_config
    from lm_engine_b200.parallel.manager import ProcessGroupManager

    ProcessGroupManager.destroy_process_groups()
    ProcessGroupManager(zero_stage=0)
    torch.manual_seed(2)

    def cfg(hidden):
        return dense_config(vocab_size=96, hidden_size=hidden, num_layers=2, num_attention_heads=4, num_key_value_heads=2,
                            intermediate_size=64, max_position_embeddings=16).to_dict()

    return ModelWrapperForDistillation(
        pretrained_config=cfg(32), micro_batch_size=2, sequence_length=16, teacher_pretrained_config=cfg(48),
        teacher_model_dtype="fp32", kl_divergence_method=method, kl_divergence_weight=0.5, kl_divergence_top_k=top_k,
        kl_divergence_tail=tail)


@pytest.mark.parametrize("method", ["forward", "backward"])
def test_distillation_training_from_best_tokens(method):
    """A list of the whole vocabulary is the full divergence; a shorter one is a lower bound of it (data processing)."""
    tokens = torch.randint(0, 96, (2, 17), generator=torch.Generator().manual_seed(0))
    results = {}
    for top_k in (None, 96, 8):
        w = _wrapper(top_k, method)
        out = w(tokens, lm_loss_multiplier=1 / 32)
        out["loss"].backward()
        grads = [p.grad for p in w.parameters() if p.grad is not None]
        assert all(p.grad is None for p in w.teacher_model.parameters()) and grads
        results[top_k] = (out, grads)
    full, full_grads = results[None]
    listed, listed_grads = results[96]
    for name in full:
        torch.testing.assert_close(listed[name], full[name], rtol=1e-5, atol=1e-6)
    for a, b in zip(listed_grads, full_grads):
        torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-6)
    short = results[8][0]
    assert 0 < float(short["kl_divergence"].detach()) < float(full["kl_divergence"].detach())
    torch.testing.assert_close(short["lm_loss"], full["lm_loss"], rtol=1e-5, atol=1e-6)


def test_teacher_arguments():
    from lm_engine_b200.arguments import TeacherArgs

    assert TeacherArgs(model_name="t", kl_divergence_method="forward").kl_divergence_top_k is None
    assert TeacherArgs(model_name="t", kl_divergence_method="backward", kl_divergence_top_k=64,
                       kl_divergence_tail=False).kl_divergence_top_k == 64
    for bad in (dict(kl_divergence_top_k=0), dict(kl_divergence_top_k=129),
                dict(kl_divergence_top_k=8, kl_divergence_tail=False)):
        with pytest.raises(Exception):
            TeacherArgs(model_name="t", kl_divergence_method="forward", **bad)
