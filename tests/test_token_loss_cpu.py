"""Operators on token probabilities on the CPU: the plain forms against 64 bits and against differences, refusals, what losses and the
engine make of them."""
import itertools

import pytest
import torch

from flextrain_b200 import ops
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
