"""Operators on token probabilities on the CPU: the plain forms against 64 bits and against differences, refusals, what losses and the
engine make of them."""
import itertools

import pytest
import torch

import flextrain_b200 as ft
from conftest import build_tiny
from flextrain_b200 import ops
from flextrain_b200.bench.naive import clone_params, naive_forward
from flextrain_b200.nn.loss import DistillationLoss, PolicyLoss, TokenScorer
from token_loss_oracle import (check_distill, check_not_finite, check_policy, check_scores, check_scores_grad, distill, on_rows, policy, scores, some_teacher,
                               wide)

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("T,V,dtype,K,tau,cap", [(6, 1, F32, 1, 1.0, 0.0), (6, 7, F32, 7, 0.7, 0.0), (9, 257, BF16, 5, 1.0, 30.0), (7, 300, F16, 20, 2.0, 0.0),
                                                 (1, 64, F32, 0, 1.0, 0.0)])
def test_scores(T, V, dtype, K, tau, cap):
    check_scores(T, V, dtype, "cpu", K, tau, cap, gap=2, shift=1, masked=T > 6)
    check_scores(T, V, dtype, "cpu", K, tau, cap, given=False)


@pytest.mark.parametrize("T,V,dtype,K,tau,cap,apart", [(6, 7, F32, 0, 1.0, 0.0, True), (9, 257, BF16, 5, 0.5, 30.0, False), (7, 300, F16, 20, 2.0, 0.0, True)])
def test_scores_gradient(T, V, dtype, K, tau, cap, apart):
    check_scores_grad(T, V, dtype, "cpu", K, tau, cap, gap=2, shift=1, apart=apart)
    for which in ("l", "h", "t", ""):
        check_scores_grad(T, V, dtype, "cpu", K, tau, cap, which=which)
    if K:
        check_scores_grad(T, V, dtype, "cpu", K, tau, cap, twice=True)


@pytest.mark.parametrize("old,kept,adv,bonus,masked", list(itertools.product((False, True), (False, True), (False, True), (0.0, 0.01), (False, True))))
def test_policy(old, kept, adv, bonus, masked):
    check_policy(12, 61, F32, "cpu", old=old, kept=kept, adv=adv, bonus=bonus, masked=masked)


@pytest.mark.parametrize("dtype,tau,cap,apart", [(BF16, 1.0, 30.0, False), (F16, 0.7, 0.0, True), (F32, 2.0, 10.0, False)])
def test_policy_types(dtype, tau, cap, apart):
    check_policy(12, 61, dtype, "cpu", tau, cap, gap=1, shift=1, apart=apart)


def teacher_changes():
    def padded(z, ids, t):
        ids[:, 2:] = -1
        return ids, t

    def none_left(z, ids, t):
        ids[1:3] = -1
        ids[4:6] = z.shape[1]
        return ids, t

    def twice(z, ids, t):
        ids[:, 1] = ids[:, 0]
        t[:, :2] -= 1.0
        return ids, t

    def no_mass(z, ids, t):
        t[:, 0] = float("-inf")
        t[3] = float("-inf")
        return ids, t

    def above_one(z, ids, t):
        return ids, t + 0.7

    return dict(none=None, padded=padded, none_left=none_left, twice=twice, no_mass=no_mass, above_one=above_one)


CHANGES = list(teacher_changes())


@pytest.mark.parametrize("rest,ce,change", list(itertools.product(("drop", "bucket"), (0.0, 0.3, 1.0), CHANGES)))
def test_distill(rest, ce, change):
    check_distill(9, 61, F32, "cpu", 5, 2.0 if ce else 1.0, rest=rest, ce=ce, change=teacher_changes()[change])


@pytest.mark.parametrize("dtype,tau,cap,rest,K,V,given,masked", [(BF16, 2.0, 30.0, "bucket", 7, 7, True, False), (F16, 0.7, 0.0, "drop", 1, 40, False, True),
                                                                (F32, 1.0, 10.0, "bucket", 6, 7, False, False), (BF16, 1.0, 0.0, "drop", 1, 1, True, False)])
def test_distill_sizes(dtype, tau, cap, rest, K, V, given, masked):
    check_distill(9, V, dtype, "cpu", K, tau, cap, rest, gap=1, shift=1, apart=masked, given=given, masked=masked)


def test_gradients_against_differences():
    """The 64-bit definitions themselves, by central differences of their losses: step 1e-5, whose square times a third derivative of
    order one is 1e-10, and 2e-16 / 1e-5 of rounding."""
    T, V = 5, 11
    _, z = wide(T, V, F32, "cpu")
    z = z.double()
    t = torch.tensor([0, 10, 3, -100, 5])
    on = on_rows(T, V, t, None)
    lp = scores(z, t, torch.ones(T, dtype=torch.bool) & on, 1.3, 20.0, 0)[2].detach()
    old = torch.zeros(T, dtype=torch.float64)
    old[on] = lp - torch.tensor([0.05, -0.1, 0.8, -0.9], dtype=torch.float64)
    a = torch.tensor([1.0, -2.0, 0.5, 1.0, -1.0], dtype=torch.float64)
    ids, teacher = some_teacher(z, 3, 1.3, 20.0)
    forms = [lambda z: policy(z, t, on, 1.3, 20.0, a, old, old + 0.3, 0.2, 0.2, 0.1, 0.02, 1.0)[:2]]
    forms += [lambda z, r=r, ce=ce: distill(z, ids, teacher, t, on, r, ce, 1.3, 20.0, 1.0)[:2] for r in ("drop", "bucket") for ce in (0.0, 0.4)]
    for form in forms:
        value = lambda z: (form(z)[0][0] if isinstance(form(z)[0], list) else form(z)[0]).sum()                     # noqa: E731
        want, h = form(z)[1], 1e-5
        for i, j in itertools.product(range(T), range(V)):
            up, down = z.clone(), z.clone()
            up[i, j] += h
            down[i, j] -= h
            assert abs(float((value(up) - value(down)) / (2 * h) - want[i, j])) < 1e-7


def test_masked_vocabulary_and_rows_without_a_distribution():
    check_not_finite("cpu")


def test_ties_go_to_the_lowest_id():
    z = torch.tensor([[0.0, -0.0, 1.0, 1.0, -0.0, 0.0], [2.0] * 6, [-0.0, 0.0, -0.0, 0.0, -0.0, 0.0]])
    assert ops.token_logprobs(z, top_k=5).top_ids.tolist() == [[2, 3, 0, 1, 4], [0, 1, 2, 3, 4], [0, 1, 2, 3, 4]]


def test_no_rows():
    z, t = torch.empty(0, 9), torch.empty(0, dtype=torch.int64)
    s = ops.token_logprobs(z, t, top_k=3)
    assert s.logprobs.shape == (0,) and s.top_ids.shape == (0, 3)
    assert ops.token_logprobs_bwd_(z, t, s, dlogprobs=torch.empty(0)).shape == (0, 9)
    assert ops.policy_loss_(z, t).loss.shape == (0,) and ops.distill_loss_(z, torch.empty(0, 2, dtype=torch.int64), torch.empty(0, 2)).shape == (0,)


def refusals(device):
    z = torch.randn(4, 10, device=device)
    t = torch.zeros(4, dtype=torch.int64, device=device)
    s = ops.token_logprobs(z, t, top_k=2)
    ids, q = torch.zeros(4, 3, dtype=torch.int64, device=device), torch.zeros(4, 3, device=device)
    one = torch.ones(4, device=device)
    wide_z = torch.randn(4, 30, device=device)
    yield lambda: ops.token_logprobs(z[0])
    yield lambda: ops.token_logprobs(z.double())
    yield lambda: ops.token_logprobs(z.long())
    yield lambda: ops.token_logprobs(z[:, :0])
    yield lambda: ops.token_logprobs(z, t[:3])
    yield lambda: ops.token_logprobs(z, t.float())
    yield lambda: ops.token_logprobs(z, t, loss_mask=one[:2])
    yield lambda: ops.token_logprobs(z, t.view(4, 1))
    yield lambda: ops.token_logprobs(z, t, top_k=-1)
    yield lambda: ops.token_logprobs(z, t, top_k=11)
    yield lambda: ops.token_logprobs(torch.randn(4, 200, device=device), t, top_k=129)
    for tau in (0.0, -1.0, float("nan"), float("inf")):
        yield lambda tau=tau: ops.token_logprobs(z, t, temperature=tau)
    yield lambda: ops.token_logprobs(z, t, softcap=-1.0)
    yield lambda: ops.token_logprobs(z, t, softcap=float("nan"))
    yield lambda: ops.token_logprobs_bwd_(z, None, s, dlogprobs=one)
    yield lambda: ops.token_logprobs_bwd_(z, t, s._replace(lse=None), dlogprobs=one)
    yield lambda: ops.token_logprobs_bwd_(z, t, s._replace(entropy=None), dentropy=one)
    yield lambda: ops.token_logprobs_bwd_(z, t, s._replace(top_ids=None), dtop_logprobs=q)
    yield lambda: ops.token_logprobs_bwd_(z, t, s, dtop_logprobs=q)
    yield lambda: ops.token_logprobs_bwd_(z, t, s, dlogprobs=one[:1])
    yield lambda: ops.token_logprobs_bwd_(z, t, s, dlogprobs=one, out=z[:3])
    yield lambda: ops.token_logprobs_bwd_(z, t, s, dlogprobs=one, out=z.bfloat16())
    yield lambda: ops.token_logprobs_bwd_(wide_z[:, :10], t, s, dlogprobs=one, out=wide_z[:, 5:15])
    yield lambda: ops.token_logprobs_bwd_(z, t, s, dlogprobs=one, out=torch.empty(10, 4, device=device).t())
    yield lambda: ops.token_logprobs_bwd_(z[:1].expand(4, 10), t, s, dlogprobs=one)
    yield lambda: ops.policy_loss_(z[:1].expand(4, 10), t)
    yield lambda: ops.policy_loss_(z.t().contiguous().t(), t)
    yield lambda: ops.policy_loss_(wide_z[:1, :10].expand(4, 10), t, out=wide_z[:, :10])            # (the expanded row lies in it)
    yield lambda: ops.policy_loss_(z, None)
    yield lambda: ops.policy_loss_(z, t, one[:2])
    yield lambda: ops.policy_loss_(z, t, one, old_logprobs=one[:, None])
    yield lambda: ops.policy_loss_(z, t, one, clip_low=1.5)
    yield lambda: ops.policy_loss_(z, t, one, clip_low=-0.1)
    yield lambda: ops.policy_loss_(z, t, one, clip_high=-0.1)
    yield lambda: ops.policy_loss_(z, t, one, ref_logprobs=one.to(torch.complex64))
    yield lambda: ops.distill_loss_(z, ids, q, rest="keep")
    yield lambda: ops.distill_loss_(z, ids[:, :0], q[:, :0])
    yield lambda: ops.distill_loss_(z, ids, q[:, :2])
    yield lambda: ops.distill_loss_(z, ids, None)
    yield lambda: ops.distill_loss_(z, ids[0], q[0])
    yield lambda: ops.distill_loss_(z, ids.float(), q)
    yield lambda: ops.distill_loss_(z, ids.expand(4, 3).repeat(1, 50), q.repeat(1, 50))
    yield lambda: ops.distill_loss_(z, ids, q, ce_weight=0.5)
    yield lambda: ops.distill_loss_(z, ids, q, targets=t, ce_weight=1.5)
    yield lambda: ops.distill_loss_(z, ids, q, targets=t[:1])
    yield lambda: ops.distill_loss_(z.half(), ids, q, out=z)


def test_refusals():
    for n, call in enumerate(refusals("cpu")):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"refusal {n} was taken")


# ------------------------------------------------------------------------------------- losses and the engine
DIMS = dict(vocab_size=256, n_layers=2, d_model=64, n_heads=4, n_kv_heads=2, head_dim=16, expert_dim=128, ffn_dim=128, num_routed_experts=0,
            num_shared_experts=0, top_k=0, is_causal=True)


def _sequences(lengths=(40, 24, 61)):
    """Prompts without a target, a mask, one sequence of more than one chunk."""
    g = torch.Generator().manual_seed(0)
    out = []
    for i, n in enumerate(lengths):
        t = torch.randint(0, 256, (n,), generator=g)
        tgt = torch.roll(t, -1)
        tgt[-1] = -100
        tgt[:3] = -100
        out.append(ft.Sequence(t, targets=tgt, seq_id=i, advantages=torch.randn(n, generator=g),
                               loss_mask=(torch.arange(n) % 7 != 5).float() if i == 1 else None))
    return out


def _model(cap=0.0, seed=None):
    am = build_tiny(dims=DIMS, max_seq_len=64, batch_tokens=96)
    am.head.final_softcap = cap
    if seed is not None:
        g = torch.Generator().manual_seed(seed)
        w = am.buffers.head_params()["w_head_proj"]
        w.copy_(torch.randn(w.shape, generator=g) * 0.2)
    return am


def _rows(am, P, s, cap, tau):
    am.head.final_softcap = 0.0
    z = naive_forward(am, P, s.tokens)
    am.head.final_softcap = cap
    u = cap * torch.tanh(z / cap) if cap else z
    on = (s.targets != -100) & (s.loss_mask > 0 if s.loss_mask is not None else True)
    lp = torch.log_softmax(u / tau, -1)
    return z, lp, lp.gather(1, s.targets.clamp(min=0)[:, None])[:, 0], -(lp.exp() * lp).sum(-1), on


def _gradients_agree(am, P, loss):
    loss.backward()
    bm, n = am.buffers, 0
    for (scope, l, name), p in P.items():
        g = {"embed": bm.embed_grads(), "head": bm.head_grads()}.get(scope) or bm.grads(l)
        gname = "g_" + name[2:] if name.startswith("w_") else "g_" + name
        if gname in g and p.grad is not None:
            # both sides sum fp32 products of two layers in their own orders: some 16 roundings, 2^-24 each, of the tensor's largest
            # (68 of the embedding: 6.5e-5)
            torch.testing.assert_close(g[gname].float(), p.grad, rtol=3e-4, atol=3e-6 + 16 * 2.0 ** -24 * float(p.grad.abs().max()),
                                       msg=lambda m: f"{scope}/{l}/{name}: {m}")
            n += 1
    assert n > 5


@pytest.mark.parametrize("cap,tau,K", [(0.0, 1.0, 0), (5.0, 0.7, 6)])
def test_score(cap, tau, K):
    """Scores of every sequence against the model written out, also where a sequence takes several chunks and a chunk several pieces of
    the head; nothing of a step changes."""
    am, seqs = _model(cap, seed=1), _sequences()
    am.head.head_chunk_size = 17
    got = am.score(seqs, top_k=K, temperature=tau)
    P = clone_params(am)
    for s, g in zip(seqs, got):
        assert s.scores is g
        _, lp, given, ent, on = _rows(am, P, s, cap, tau)
        torch.testing.assert_close(g.logprobs, (given * on).detach(), rtol=1e-4, atol=1e-5)
        torch.testing.assert_close(g.entropy, (ent * on).detach(), rtol=1e-4, atol=1e-5)
        torch.testing.assert_close(s.per_token_loss, -g.logprobs)
        if K:
            want = lp.detach().topk(K)
            torch.testing.assert_close(g.top_logprobs[on], want.values[on], rtol=1e-4, atol=1e-5)
            assert bool((g.top_ids[~on] == -1).all())
        else:
            assert g.top_ids is None
    assert am.step_num == 0 and am.fwd_bwd_serial == 0
    for bad in (dict(top_k=129), dict(top_k=-1), dict(temperature=0.0)):
        with pytest.raises(ValueError):
            am.score(seqs, **bad)
    with pytest.raises(RuntimeError):
        am.fwd_bwd(seqs, loss_fn=TokenScorer())


@pytest.mark.parametrize("cap,tau,ref", [(0.0, 1.0, True), (5.0, 0.7, False)])
def test_policy_loss_through_the_engine(cap, tau, ref):
    """Rollouts scored under the old weights, then a step's loss and gradients under others."""
    seqs = _sequences()
    am = _model(cap, seed=1)
    for s, g in zip(seqs, am.score(seqs, temperature=tau)):
        # (at the same weights all ratios are one)
        s.old_logprobs = g.logprobs + 0.3 * torch.sin(torch.arange(len(s)).float())
        if ref:
            s.ref_logprobs = g.logprobs + 0.2 * torch.cos(torch.arange(len(s)).float())
    if not ref:
        seqs[0].advantages = seqs[1].advantages = seqs[2].advantages = None
    P = clone_params(am)
    total = 0.0
    for s in seqs:
        _, lp, given, ent, on = _rows(am, P, s, cap, tau)
        a = s.advantages if s.advantages is not None else torch.ones(len(s))
        r = torch.exp(given - s.old_logprobs)
        l = -torch.minimum(r * a, r.clamp(0.8, 1.25) * a) - 0.01 * ent
        if ref:
            d = s.ref_logprobs - given
            l = l + 0.1 * (d.exp() - d - 1)
        total = total + (l * on).sum()
    loss = PolicyLoss(0.2, 0.25, kl_coef=0.1, entropy_coef=0.01, temperature=tau)
    held_out = am.evaluate(seqs, loss_fn=loss)
    st = am.fwd_bwd(seqs, loss_scale_factor=1.0, loss_fn=loss)
    assert abs(st.loss_sum - total.item()) < 1e-3 * max(1.0, abs(total.item())) and held_out.loss_sum == st.loss_sum
    _gradients_agree(am, P, total)


def test_a_reference_without_advantages_counts():
    seqs = _sequences((40,))
    seqs[0].advantages = None
    seqs[0].ref_logprobs = torch.full((40,), -3.0)
    am = _model(seed=1)
    with_it = am.evaluate(seqs, loss_fn=PolicyLoss(kl_coef=0.5)).loss_sum
    assert with_it > am.evaluate(seqs, loss_fn=PolicyLoss()).loss_sum


@pytest.mark.parametrize("cap,tau,rest,ce", [(0.0, 2.0, "drop", 0.3), (5.0, 1.0, "bucket", 0.0)])
def test_distillation_through_the_engine(cap, tau, rest, ce):
    """A teacher's alternatives as score() gives them; one sequence without a teacher, one with fewer of its tokens."""
    seqs = _sequences()
    K = 8
    for s, g in zip(seqs, _model(cap, seed=2).score(seqs, top_k=K, temperature=tau)):
        s.teacher_ids, s.teacher_logprobs = g.top_ids, g.top_logprobs
    seqs[0].teacher_ids, seqs[0].teacher_logprobs = seqs[0].teacher_ids[:, :5], seqs[0].teacher_logprobs[:, :5]
    seqs[1].teacher_ids = seqs[1].teacher_logprobs = None
    am = _model(cap, seed=1)
    P = clone_params(am)
    total = 0.0
    for s in seqs:
        z, lp, _, _, on = _rows(am, P, s, cap, tau)
        l = torch.zeros(len(s))
        if s.teacher_ids is not None:
            ids, t = s.teacher_ids[on], s.teacher_logprobs[on]
            q = torch.softmax(t, -1) if rest == "drop" else t.exp()
            kl = (q * (q.log() - lp[on].gather(1, ids))).sum(-1)
            if rest == "bucket":
                others = torch.logsumexp(lp[on].scatter(1, ids, float("-inf")), -1)
                kl = kl + (1 - q.sum(-1)) * ((1 - q.sum(-1)).log() - others)
            l = torch.zeros(len(s)).index_put((on.nonzero()[:, 0],), (1 - ce) * tau * tau * kl)
        # (without a teacher's token all tokens are the rest, which has probability one for both)
        hard = torch.nn.functional.cross_entropy(cap * torch.tanh(z / cap) if cap else z, s.targets, reduction="none")
        total = total + ((l + ce * hard) * on).sum()
    loss = DistillationLoss(rest=rest, ce_weight=ce, temperature=tau)
    held_out = am.evaluate(seqs, loss_fn=loss)
    st = am.fwd_bwd(seqs, loss_scale_factor=1.0, loss_fn=loss)
    assert abs(st.loss_sum - total.item()) < 1e-3 * max(1.0, abs(total.item())) and held_out.loss_sum == st.loss_sum
    _gradients_agree(am, P, total)


def test_what_sequences_carry_is_checked():
    am = _model()
    ids, lps = torch.zeros(40, 3, dtype=torch.int64), torch.zeros(40, 3)
    for kw in (dict(teacher_ids=ids), dict(teacher_ids=ids, teacher_logprobs=lps[:, :2]), dict(teacher_ids=ids[:30], teacher_logprobs=lps[:30]),
               dict(teacher_ids=lps, teacher_logprobs=lps), dict(teacher_ids=ids[:, 0], teacher_logprobs=lps[:, 0]), dict(old_logprobs=lps[:3, 0]),
               dict(teacher_ids=ids.repeat(1, 50), teacher_logprobs=lps.repeat(1, 50))):
        s = _sequences((40,))
        for k, v in kw.items():
            setattr(s[0], k, v)
        with pytest.raises(ValueError):
            am.fwd_bwd(s)
    s = _sequences((40, 24))
    s[0].old_logprobs = torch.zeros(40)
    with pytest.raises(ValueError):
        am.fwd_bwd(s, loss_fn=PolicyLoss())
    with pytest.raises(ValueError):
        am.fwd_bwd(_sequences(), loss_fn=DistillationLoss())

    class Bare:                                               # a sequence of one's own class
        tokens, targets = s[1].tokens, s[1].targets
        old_logprobs, teacher_ids, teacher_logprobs = torch.zeros(24), ids[:24].tolist(), lps[:24]

    got = am.score([Bare()], top_k=2)[0]
    assert got.logprobs.shape == (24,) and got.top_ids.shape == (24, 2)
    assert am.evaluate([Bare()], loss_fn=DistillationLoss()).loss_sum > 0
