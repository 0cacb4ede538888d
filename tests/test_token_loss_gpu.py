"""Operators on token probabilities on a GPU: every operator against its definition in 64 bits over types, sizes, strides and options."""
import itertools

import pytest
import torch

from flextrain_b200 import ops
from test_token_loss_cpu import CHANGES, refusals, teacher_changes
from token_loss_oracle import check_distill, check_not_finite, check_policy, check_scores, check_scores_grad, some_targets, value_error, wide

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = (BF16, F16, F32)
# around a vector, a warp's and a block's worth of them, odd ones; rows of a cluster's shared memory; long ones
VOCABS = (1, 2, 7, 8, 9, 33, 250, 1000, 2047, 2048, 2049, 4099, 8200, 32000, 50257, 131073)


def test_refusals():
    for n, call in enumerate(refusals("cuda")):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"refusal {n} was taken")
    z = torch.randn(4, 9, device="cuda")
    for call in (lambda: ops.token_logprobs(z, torch.zeros(4, dtype=torch.int64)), lambda: ops.policy_loss_(z, torch.zeros(4, dtype=torch.int64, device="cuda"), torch.ones(4)),
                 lambda: ops.policy_loss_(z, torch.zeros(4, dtype=torch.int64, device="cuda"), out=torch.empty(4, 9))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scores(V, dtype):
    check_scores(6, V, dtype, "cuda")
    check_scores(7, V, dtype, "cuda", K=min(V, 5), tau=0.7, gap=1, shift=1, masked=True)


@pytest.mark.parametrize("V,K", [(9, 9), (128, 128), (129, 128), (1000, 1), (1000, 128), (4099, 20), (50257, 64), (131073, 128), (300000, 100)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_alternatives(V, K, dtype):
    check_scores(5, V, dtype, "cuda", K=K, given=False)
    check_scores(6, V, dtype, "cuda", K=K, tau=2.0, cap=20.0, gap=5, shift=3)


def _tied(kind, T, V, dtype):
    z = torch.zeros(T, V, device="cuda", dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    if kind == "signs":
        z[:, ::2] = -0.0
    if kind == "few":                                         # a handful of values, thousands of times each
        z.copy_(torch.randint(-2, 3, (T, V), device="cuda", generator=g))
    if kind == "rising":
        z.copy_(torch.arange(V, device="cuda") * (20.0 / V))
    if kind == "front":                                       # the likely ones side by side
        z.copy_(torch.randn(T, V, device="cuda", generator=g) - 6.0 * (torch.arange(V, device="cuda") > 500))
    if kind == "allowed":                                     # fewer tokens allowed than asked for
        z.fill_(float("-inf"))
        z[:, V // 2:V // 2 + 3] = torch.randn(T, 3, device="cuda", generator=g).to(dtype)
    if kind == "same":
        z.fill_(-3.0)
    return z


@pytest.mark.parametrize("kind", ["signs", "few", "rising", "front", "allowed", "same"])
@pytest.mark.parametrize("V,K", [(40, 20), (5000, 128), (60000, 20), (131073, 128)])
def test_alternatives_of_equal_logits(kind, V, K):
    for dtype in TYPES:
        check_scores(4, V, dtype, "cuda", K=K, given=False, z=_tied(kind, 4, V, dtype))


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scores_gradient(V, dtype):
    check_scores_grad(6, V, dtype, "cuda")
    check_scores_grad(7, V, dtype, "cuda", K=min(V, 9), tau=0.7, cap=20.0, gap=1, shift=1, apart=False)


@pytest.mark.parametrize("which", ["", "l", "h", "t", "lt", "ht"])
def test_scores_gradient_of_some_outputs(which):
    for K in (4, 128):
        check_scores_grad(6, 4099, BF16, "cuda", K=K, which=which, twice=True)
        check_scores_grad(6, 4096, F32, "cuda", K=K, which=which, twice=True, apart=False)


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_policy(V, dtype):
    check_policy(12, V, dtype, "cuda")
    check_policy(13, V, dtype, "cuda", tau=0.7, cap=20.0, gap=1, shift=1, apart=False, masked=True)


@pytest.mark.parametrize("old,kept,adv,bonus", list(itertools.product((False, True), (False, True), (False, True), (0.0, 0.01))))
def test_policy_options(old, kept, adv, bonus):
    check_policy(20, 3001, BF16, "cuda", old=old, kept=kept, adv=adv, bonus=bonus)


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_distill(V, dtype):
    K = min(V, 6)
    check_distill(7, V, dtype, "cuda", K, rest="bucket")
    check_distill(7, V, dtype, "cuda", K, tau=2.0, cap=20.0, rest="drop", ce=0.3, gap=1, shift=1, apart=False)
    check_distill(7, V, dtype, "cuda", K, tau=0.7, rest="bucket", ce=0.5, gap=2, shift=2, masked=True)


@pytest.mark.parametrize("rest,ce,change", list(itertools.product(("drop", "bucket"), (0.0, 0.3, 1.0), CHANGES)))
def test_distill_teachers(rest, ce, change):
    check_distill(9, 2049, F32, "cuda", 5, 2.0 if ce else 1.0, rest=rest, ce=ce, change=teacher_changes()[change])
    check_distill(9, 50264, BF16, "cuda", 128, 2.0 if ce else 1.0, rest=rest, ce=ce, change=teacher_changes()[change], apart=False)


def test_not_finite():
    check_not_finite("cuda")


def test_long_rows():
    """Rows that shared memory does not hold, also off the 16-byte grid."""
    check_scores(3, 900001, BF16, "cuda", K=9, gap=2, shift=1)
    check_scores(3, 450000, F32, "cuda", K=3, cap=20.0)
    check_policy(5, 450000, F32, "cuda")
    check_policy(5, 900001, F16, "cuda", tau=0.7, gap=1, apart=False)
    check_distill(4, 450001, F32, "cuda", 7, rest="bucket", ce=0.2, tau=2.0)
    check_distill(4, 1600000, BF16, "cuda", 7, cap=20.0, apart=False)
    check_scores_grad(4, 900001, BF16, "cuda", K=5)
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.empty(1, 1600001, device="cuda", dtype=BF16))


def test_rows_beyond_31_bits():
    """A row that begins beyond 2^31 elements."""
    big = torch.empty((1 << 31) + 300000, device="cuda", dtype=BF16)
    z = big.as_strided((2, 4099), (1 << 31, 1))
    z.copy_(wide(2, 4099, BF16, "cuda")[1])
    near = wide(2, 4099, BF16, "cuda")[1]
    t = torch.tensor([5, 4098], device="cuda")
    a, b = ops.token_logprobs(z, t, top_k=7), ops.token_logprobs(near, t, top_k=7)
    # the second rows begin at different places in a piece of 16 bytes, so their tokens are summed in other groups: sums of the same
    # positive terms, each within value_error of the exact one, differ by twice that; gradients by that and by a rounding on either side
    tol = 2 * value_error(4099)
    same = lambda x, y, half=0.0: bool(((x.double() - y.double()).abs() <= (tol + 2.02 * half) * (y.double().abs() + (half == 0))).all())
    assert all(same(a[i], b[i]) for i in (0, 1, 2, 4)) and torch.equal(a.top_ids, b.top_ids)
    assert same(ops.policy_loss(z, t).loss, ops.policy_loss(near, t).loss)
    out = torch.empty_like(near)
    ops.token_logprobs_bwd_(near, t, b, dlogprobs=torch.ones(2, device="cuda"), out=out)
    ops.token_logprobs_bwd_(z, t, b, dlogprobs=torch.ones(2, device="cuda"))
    assert torch.equal(z, out)                                # (nothing is summed)
    z.copy_(near)
    ops.policy_loss_(near, t, out=out)
    ops.policy_loss_(z, t)
    assert same(z, out, 2.0 ** -8)


def test_many_rows_and_a_stream_of_ones_own():
    """More rows than fit on the GPU at once; work on another stream than the current one; an expanded row is read."""
    T, V = 5000, 513
    z = wide(T, V, BF16, "cuda")[1]
    t = some_targets(T, V, "cuda")
    want = ops.policy_loss_(z, t, out=(first := torch.empty_like(z)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.policy_loss_(z, t, out=(second := torch.empty_like(z)))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second) and torch.equal(got.loss, want.loss)
    one = z[:1].expand(9, V)
    s = ops.token_logprobs(one, torch.full((9,), 3, device="cuda"), top_k=4)
    assert bool((s.logprobs == s.logprobs[0]).all()) and bool((s.top_ids == s.top_ids[0]).all())


def test_captured_and_replayed():
    """All of them in one graph, replayed on new inputs; the same bits as eager calls."""
    T, V, K = 9, 8200, 6
    z, t = wide(T, V, BF16, "cuda")[1].clone(), some_targets(T, V, "cuda")
    outs = [torch.empty_like(z) for _ in range(3)]

    def all_of_them():
        s = ops.token_logprobs(z, t, top_k=K)
        ops.token_logprobs_bwd_(z, t, s, dlogprobs=s.logprobs, dentropy=s.entropy, out=outs[0])
        p = ops.policy_loss_(z, t, s.entropy, old_logprobs=s.logprobs, entropy_coef=0.1, out=outs[1])
        return [*s, *p, ops.distill_loss_(z, s.top_ids, s.top_logprobs, targets=t, rest="bucket", out=outs[2])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        all_of_them()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = all_of_them()
    for seed in (1, 2):
        z.copy_(wide(T, V, BF16, "cuda", seed=seed)[1])
        graph.replay()
        got = [x.clone() for x in held + outs]
        want = all_of_them()
        assert all(torch.equal(x, y) for x, y in zip(got, want + outs))


def test_teacher_to_student():
    """As they are used together: a teacher's alternatives, a student's loss and gradient from them; the same logits agree."""
    T, V, K, tau = 33, 50257, 64, 2.0
    z = wide(T, V, BF16, "cuda")[1]
    t = some_targets(T, V, "cuda")
    s = ops.token_logprobs(z, None, temperature=tau, top_k=K)
    loss = ops.distill_loss_(z, s.top_ids, s.top_logprobs, rest="bucket", temperature=tau, out=(out := torch.empty_like(z)))
    # KL of a distribution with itself: terms of up to 12 that cancel, errors as in the comparisons; gradients are what is left of p
    assert float(loss.abs().max()) < tau * tau * 13 * 2.0 ** -24 * (40 + 4 * (V / 256) ** 0.5)
    assert float(out.abs().max()) < 2e-5 * tau
    student = wide(T, V, BF16, "cuda", seed=4)[1]
    before = ops.distill_loss(student, s.top_ids, s.top_logprobs, targets=t, temperature=tau)
    grad = torch.empty_like(student)
    ops.distill_loss_(student, s.top_ids, s.top_logprobs, targets=t, temperature=tau, out=grad)
    after = ops.distill_loss(student - grad, s.top_ids, s.top_logprobs, targets=t, temperature=tau)
    assert float((after - before).sum()) < 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,V", [(2100, 300), (700, 20011), (500, 40008)])
def test_more_rows_than_begin_at_once(T, V, dtype):
    """Rows are taken over from blocks that have not begun; a third of them and more are left out, some side by side."""
    check_scores(T, V, dtype, "cuda", masked=True)
    check_scores(T, V, dtype, "cuda", K=12, masked=True, gap=1)
    check_policy(T, V, dtype, "cuda", masked=True, gap=3, apart=False)
    check_policy(T, V, dtype, "cuda", cap=20.0)
    check_distill(T, V, dtype, "cuda", 9, tau=2.0, rest="bucket", ce=0.3, masked=True, shift=1)


@pytest.mark.parametrize("live", [0, 1, 500])
def test_few_rows_count(live):
    """Long runs of rows that are left out."""
    T, V = 1500, 20000
    z = wide(T, V, BF16, "cuda")[1]
    t = torch.full((T,), -100, device="cuda")
    t[T - live:] = 5
    s = ops.token_logprobs(z, t, top_k=3)
    assert int((s.logprobs != 0).sum()) == live and int((s.top_ids[:, 0] >= 0).sum()) == live
    out = torch.full_like(z, 3.0)
    p = ops.policy_loss_(z, t, out=out)
    assert bool((out[: T - live] == 0).all()) and bool((out[T - live:].abs().sum(-1) > 0).all()) and int((p.loss != 0).sum()) == live
    out.fill_(3.0)
    ops.distill_loss_(z, t.clamp(min=0)[:, None], torch.zeros(T, 1, device="cuda"), targets=t, out=out)
    assert bool((out[: T - live] == 0).all()) and bool((out[T - live:].abs().sum(-1) > 0).all())


def test_grpo_loss_takes_the_kernel():
    """GRPOLoss: no mask but -100, the logits as they are; its values and gradient against the definition."""
    from flextrain_b200.nn.loss import GRPOLoss, TokenSlice
    from token_loss_oracle import near, near_grad, on_rows, policy
    T, V = 12, 3001
    z = wide(T, V, BF16, "cuda")[1].clone()
    t = some_targets(T, V - 1, "cuda")
    t[3] = -100
    adv, ref = torch.linspace(-2, 2, T, device="cuda"), torch.linspace(-9, -7, T, device="cuda")
    on = on_rows(T, V, t, None, device="cuda")
    (loss, _, _), want, size = policy(z, t, on, 1.0, 0.0, adv, None, ref, 0.2, 0.2, 0.1, 0.0, 0.5)
    logits = z.clone()
    got = GRPOLoss(kl_beta=0.1)(z, TokenSlice(t, torch.zeros(T, device="cuda"), adv, ref), 0.5, 30.0)
    # the penalty's e^d (d of up to 6 here: 400) multiplies the log probability's error
    near(got, loss, V, factor=400.0)
    near_grad(z, want, size, logits)


def test_score_and_losses_through_the_engine():
    """A bf16 model on the GPU: scores equal those of its own logits; distillation from itself is near nothing; a policy step runs."""
    import flextrain_b200 as ft
    from conftest import TINY_DIMS, build_tiny
    from flextrain_b200.nn.loss import DistillationLoss, PolicyLoss
    am = build_tiny(dims=TINY_DIMS, device="cuda", dtype=BF16)
    g = torch.Generator().manual_seed(0)
    seqs = []
    for n in (100, 37, 64):
        toks = torch.randint(0, 1024, (n,), generator=g)
        tgt = torch.roll(toks, -1)
        tgt[-1] = -100
        seqs.append(ft.Sequence(toks, targets=tgt, seq_id=n))
    scores = am.score(seqs, top_k=128)
    for s, x in zip(seqs, scores):
        assert x.logprobs.shape == (len(s),) and x.top_ids.shape == (len(s), 128) and x.logprobs[-1] == 0
        assert bool((x.logprobs[:-1] < 0).all()) and bool((x.entropy[:-1] <= 6.9315).all())
        s.old_logprobs, s.teacher_ids, s.teacher_logprobs, s.advantages = x.logprobs, x.top_ids, x.top_logprobs, torch.ones(len(s))
    # against itself: KL of equal distributions, terms of up to 13 that cancel (near(): 13 (40 + 8) 2^-24 = 4e-5 a position)
    assert abs(am.evaluate(seqs, loss_fn=DistillationLoss(rest="bucket")).loss_sum) < 4e-5 * 198
    st = am.fwd_bwd(seqs, loss_fn=PolicyLoss(kl_coef=0.1, entropy_coef=0.01))
    am.step()
    assert st.active_tokens == 198 and torch.isfinite(torch.tensor(st.loss_sum))
