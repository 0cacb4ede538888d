"""Operators on token probabilities on the CPU: scores behind a tensor-parallel gather, and what else a later look at them found."""
import json
import os
import socket
import subprocess
import sys
import types

import pytest
import torch

from conftest import build_tiny
from flextrain_b200 import ops
from flextrain_b200.engine.active_model import ActiveModel
from flextrain_b200.io.sequence import Sequence
from flextrain_b200.nn.loss import CrossEntropyLoss, DistillationLoss, GRPOLoss, PolicyLoss
from flextrain_b200.ops import TokenLogprobs
from token_loss_oracle import distill, near, near_grad, on_rows, policy, scores, scores_grad, some_targets, some_teacher, wide

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DIMS = dict(vocab_size=256, n_layers=2, d_model=64, n_heads=4, n_kv_heads=2, head_dim=16, expert_dim=128, ffn_dim=128, num_routed_experts=0,
            num_shared_experts=0, top_k=0, is_causal=True)


class StagedGather:
    """A tensor-parallel group of two equal halves whose results lie in one staging buffer for each size, as those over peer memory do:
    the next gather of the same size writes over the last."""

    def __init__(self):
        self.stage = {}

    def all_gather(self, t):
        raw = torch.cat([t, t]).contiguous()
        stage = self.stage.setdefault(raw.numel() * raw.element_size(), torch.empty(raw.numel() * raw.element_size(), dtype=torch.uint8))
        stage.copy_(raw.view(-1).view(torch.uint8))
        return stage.view(raw.dtype).view(raw.shape)


def test_scores_gathered_through_one_staging_buffer():
    """Every field of a score comes back as itself, also those of one size (with one alternative all four fp32 fields are)."""
    n = 8
    for K in (1, 3):
        half = TokenLogprobs(*(torch.arange(n // 2, dtype=F32) + 10 * i for i in (1, 2, 3)), torch.arange(n // 2 * K).view(-1, K),
                             torch.arange(n // 2 * K, dtype=F32).view(-1, K) + 40)
        s = Sequence(torch.zeros(n, dtype=torch.int64))
        meta = types.SimpleNamespace(extra={"pieces": [(0, 0, n)]})
        ActiveModel._write_back_scores(types.SimpleNamespace(tp=StagedGather()), [([s], meta, half)])
        for got, want in zip(s.scores, half):
            assert torch.equal(got, torch.cat([want, want]))


def test_scores_and_their_losses_under_tensor_parallelism(tmp_path):
    """Two ranks, staged gathers: scores of ragged sequences, and losses of what sequences carry for each position, as unsharded.  Both
    sides sum fp32 products of two layers in other orders; a swapped field, or a shard's values at another's positions, is off by units.
    (Alternatives of nearly equal logits may change places: a few of them in a thousand.)"""
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    out = str(tmp_path / "scores.json")
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1", "--master-port", str(port),
           os.path.join(os.path.dirname(os.path.abspath(__file__)), "tp_score_worker.py"), out]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    res = json.load(open(out))
    assert res["fields"] == 9 * (5 + 5 + 2) and res["worst"] < 1e-4 and res["ids"] <= res["ids_of"] // 200, res


def _sequences(n=3, length=20):
    g = torch.Generator().manual_seed(0)
    out = []
    for i in range(n):
        t = torch.randint(0, 256, (length,), generator=g)
        tgt = torch.roll(t, -1)
        tgt[-1] = -100
        out.append(Sequence(t, targets=tgt, seq_id=i))
    return out


def test_what_only_some_sequences_carry_is_refused_by_the_losses_that_read_it():
    """Old log probabilities of some sequences only are refused by PolicyLoss, and by nothing that does not read them."""
    am, seqs = build_tiny(dims=DIMS, max_seq_len=64, batch_tokens=96), _sequences()
    for s, x in zip(seqs[:2], am.score(seqs)):
        s.old_logprobs = x.logprobs
    with pytest.raises(ValueError, match="old_logprobs"):
        am.fwd_bwd(seqs, loss_fn=PolicyLoss())
    assert am.fwd_bwd_serial == 0
    assert am.score(seqs)[2].logprobs[0] < 0
    assert am.evaluate(seqs).loss_sum > 0 and am.evaluate(seqs, loss_fn=GRPOLoss()).loss_sum > 0
    am.fwd_bwd(seqs, loss_fn=CrossEntropyLoss())


def test_a_reference_of_some_sequences_only():
    """With a penalty a mixture is refused: zeros in its place would be a penalty of e^(-logp); without one nothing reads it."""
    am, seqs = build_tiny(dims=DIMS, max_seq_len=64, batch_tokens=96), _sequences()
    for s in seqs:
        s.advantages = torch.zeros(len(s))
    seqs[0].ref_logprobs = am.score(seqs)[0].logprobs
    for call in (am.evaluate, am.fwd_bwd):
        with pytest.raises(ValueError, match="ref_logprobs"):
            call(seqs, loss_fn=PolicyLoss(kl_coef=0.1))
    assert am.evaluate(seqs, loss_fn=PolicyLoss()).loss_sum == 0
    assert abs(am.evaluate(seqs[:1], loss_fn=PolicyLoss(kl_coef=0.1)).loss_sum) < 1e-6 and am.evaluate(seqs[1:], loss_fn=PolicyLoss(kl_coef=0.1)).loss_sum == 0


def test_scores_are_left_in_the_callers_own_objects():
    """Sequences of one's own class: ``scores`` and ``per_token_loss`` arrive as with a Sequence; a class that refuses them is no error."""
    am, seqs = build_tiny(dims=DIMS, max_seq_len=64, batch_tokens=96), _sequences()

    class Bare:
        def __init__(self, s):
            self.tokens, self.targets = s.tokens, s.targets

    class Closed:
        __slots__ = ("tokens", "targets")

        def __init__(self, s):
            self.tokens, self.targets = s.tokens, s.targets

    class Strict(Closed):
        __slots__ = ()

        def __setattr__(self, name, value):
            if name not in ("tokens", "targets"):
                raise ValueError(f"no field {name}")
            super().__setattr__(name, value)

    mine, closed = [Bare(s) for s in seqs[:2]], [Closed(seqs[2]), Strict(seqs[2])]
    got = am.score(mine + closed, top_k=2)
    for s, x, given in zip(seqs, am.score(seqs, top_k=2), got):
        assert torch.equal(x.logprobs, given.logprobs) and torch.equal(x.top_ids, given.top_ids)
    for s, x, given in zip(mine, got, seqs):
        assert s.scores is x and torch.equal(s.per_token_loss, given.per_token_loss)


def test_scores_leave_the_device_with_their_round(monkeypatch):
    """What is held on the device is a round's scores at most, not a call's."""
    am, seqs = build_tiny(dims=DIMS, max_seq_len=64, batch_tokens=48), _sequences(7)
    held, write = [], ActiveModel._write_back_scores
    monkeypatch.setattr(ActiveModel, "_write_back_scores", lambda self, pending: (held.append([len(r) for r, _, _ in pending]), write(self, pending)))
    got = am.score(seqs, top_k=3)
    held = [h for h in held if h]
    assert len(held) > 2 and sum(h[0] for h in held) == 7
    one_by_one = [am.score([s], top_k=3)[0] for s in seqs]
    for x, y in zip(got, one_by_one):
        torch.testing.assert_close(x.logprobs, y.logprobs, rtol=1e-5, atol=1e-5)


def test_per_token_values_of_any_kind():
    """Log probabilities as lists, arrays and doubles, also where the loss does not read them."""
    am, seqs = build_tiny(dims=DIMS, max_seq_len=64, batch_tokens=96), _sequences()
    plain = am.evaluate(seqs).loss_sum
    values = [-torch.rand(len(s), dtype=torch.float64) - 5 for s in seqs]
    want = None
    for kind in (lambda v: v, lambda v: v.tolist(), lambda v: v.numpy(), lambda v: v.float()):
        for s, v in zip(seqs, values):
            s.ref_logprobs = s.old_logprobs = kind(v)
        assert am.evaluate(seqs).loss_sum == plain
        got = am.evaluate(seqs, loss_fn=PolicyLoss(kl_coef=0.1)).loss_sum
        want = got if want is None else want
        assert got == want


def test_distillation_of_sequences_without_a_teacher(monkeypatch):
    """With cross entropy in the mixture they have its part; without, a process by itself refuses, and a rank among others takes part
    (others may hold the teacher's sequences, and would wait for it)."""
    am, seqs = build_tiny(dims=DIMS, max_seq_len=64, batch_tokens=96), _sequences()
    plain = am.evaluate(seqs).loss_sum
    assert abs(am.evaluate(seqs, loss_fn=DistillationLoss(ce_weight=0.25)).loss_sum - 0.25 * plain) < 1e-4 * plain
    with pytest.raises(ValueError, match="teacher_ids"):
        am.evaluate(seqs, loss_fn=DistillationLoss())
    monkeypatch.setattr(torch.distributed, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.distributed, "get_world_size", lambda *a: 2)
    assert am.evaluate(seqs, loss_fn=DistillationLoss()).loss_sum == 0


def check_rows_of_nan(device):
    """NaN wherever it lies in a row that counts reaches the loss and the whole gradient: a stretch as long as what one block of several
    reads, all that is not the teacher's, a teacher's token of no weight, a row without a teacher's tokens; so do rows of -inf alone."""
    V, K, nan, inf = 40000, 3, float("nan"), float("inf")
    for dtype in (BF16, F16, F32):
        z = torch.randn(8, V, generator=torch.Generator().manual_seed(8)).to(dtype).to(device)
        ids = torch.tensor([1, 17, 39999], device=device).repeat(8, 1)
        q = torch.tensor([-1.0, -2.0, -1.5], device=device).repeat(8, 1)
        z[1, 10000:30000] = nan
        z[2], z[2, [1, 17, 39999]] = nan, torch.randn(3).to(z)
        z[3, 39999], q[3, 2] = nan, -inf
        z[4, 20000:], ids[4] = nan, -1
        z[5], ids[5] = -inf, -1
        z[6, 5000:], z[6, :5000], ids[6] = nan, -inf, torch.tensor([2, 3, 4])
        t = torch.full((8,), 7, device=device)
        for rest in ("drop", "bucket"):
            for ce in (0.0, 0.3):
                for rows in (slice(0, 8), slice(3, 4)):
                    out = torch.zeros_like(z[rows])
                    kw = dict(targets=t[rows], rest=rest, ce_weight=ce)
                    loss = ops.distill_loss_(z[rows], ids[rows], q[rows], out=out, **kw)
                    clean = torch.tensor([r in (0, 7) for r in range(8)], device=device)[rows]
                    for value in (loss, ops.distill_loss(z[rows], ids[rows], q[rows], **kw)):
                        assert bool((value.isfinite() == clean).all()) and bool((value.isnan() == ~clean).all()), (dtype, rest, ce, value)
                    assert bool((out.isfinite().all(-1) == clean).all()) and bool((out.isnan().all(-1) == ~clean).all()), (dtype, rest, ce)


def test_rows_of_nan():
    check_rows_of_nan("cpu")


def check_cross_entropy_alone(device):
    """``ce_weight=1``: the cross entropy and its gradient, whatever the teacher says, also where the student has nothing at its token (a
    divergence of infinity) and where its log probabilities are NaN."""
    inf = float("inf")
    for dtype in (BF16, F16, F32):
        for V in (40, 20011):
            z = torch.randn(4, V, generator=torch.Generator().manual_seed(6)).to(dtype).to(device)
            z[0, 3] = z[2, 3] = -inf
            t = torch.tensor([5, 3, 39, -100], device=device)
            ids = torch.tensor([3, 5, -1], device=device).repeat(4, 1)
            q = torch.log(torch.tensor([0.5, 0.2, 0.1], device=device)).repeat(4, 1)
            q[2, 0] = float("nan")
            x = z.double().requires_grad_()
            want = torch.nn.functional.cross_entropy(x, t, reduction="none")
            d, = torch.autograd.grad(want.sum(), x)
            size = torch.softmax(z.double(), -1).scatter_add(1, t.clamp(min=0)[:, None], torch.ones(4, 1, dtype=torch.float64, device=device))
            for rest in ("drop", "bucket"):
                for tau in (1.0, 2.0):
                    kw = dict(targets=t, rest=rest, ce_weight=1.0, temperature=tau)
                    out = torch.empty_like(z)
                    for loss in (ops.distill_loss(z, ids, q, **kw), ops.distill_loss_(z, ids, q, out=out, **kw)):
                        near(loss, want.detach(), V)
                    near_grad(out, d, size, z)


def test_cross_entropy_alone():
    check_cross_entropy_alone("cpu")


def check_common_offset(device, offset, T=24):
    """Logits far from zero: a probability depends on their differences, so losses and gradients are held to what they are held to near
    zero (1e-5 of the gradient's terms and a rounding to its type)."""
    V, K, scale = 2000, 5, 1024.0                             # (gradients of fp16 that are not among its smallest numbers)
    for dtype in (F16, BF16, F32):
        z = (wide(T, V, F32, device)[1] + offset).to(dtype)
        t = some_targets(T, V, device)
        on = on_rows(T, V, t, None, device=device)
        a = torch.linspace(-2, 2, T, device=device)
        for bonus in (0.0, 0.01):
            (loss, lp, ent), want, size = policy(z, t, on, 1.0, 0.0, a, None, None, 0.2, 0.2, 0.0, bonus, scale)
            got = ops.policy_loss_(z, t, a, entropy_coef=bonus, grad_scale=scale, out=(out := torch.empty_like(z)))
            near(got.loss, loss, V, factor=2.0)
            near(got.logprobs, lp, V)
            near(got.entropy, ent, V, size=3.0)
            near_grad(out, want, size, z)
        for rest, ce, tau in (("drop", 0.0, 1.0), ("bucket", 0.3, 2.0), ("drop", 0.3, 0.7)):
            ids, teacher = some_teacher(z, K, tau, 0.0)
            loss, want, size = distill(z, ids, teacher, t, on, rest, ce, tau, 0.0, scale)
            got = ops.distill_loss_(z, ids, teacher, targets=t, rest=rest, ce_weight=ce, temperature=tau, grad_scale=scale, out=(out := torch.empty_like(z)))
            near(got, loss, V, factor=max(1.0, tau * tau), size=12.0)
            near_grad(out, want, size, z)


@pytest.mark.parametrize("offset", [0.0, 36.0, -300.0, 1000.0, 2500.0])
def test_common_offset(offset):
    check_common_offset("cpu", offset)


def check_infinite_ratio(device):
    """A token that the old policy had no probability of: nothing times an advantage of zero is nothing, the clip holds a positive one."""
    inf = float("inf")
    z = torch.randn(4, 50, generator=torch.Generator().manual_seed(2)).to(device)
    t, a = torch.tensor([1, 2, 3, 4], device=device), torch.tensor([0.0, -0.0, 2.0, -1.0], device=device)
    old = torch.tensor([-1000.0, -inf, -1000.0, -1000.0], device=device)
    out = torch.empty_like(z)
    for loss in (ops.policy_loss(z, t, a, old_logprobs=old).loss, ops.policy_loss_(z, t, a, old_logprobs=old, out=out).loss):
        assert loss[:2].tolist() == [0.0, 0.0] and abs(float(loss[2]) + 2.4) < 1e-6 and loss[3] == inf
    assert bool((out[:3] == 0).all())


def test_infinite_ratio():
    check_infinite_ratio("cpu")


def check_extreme_scales(device):
    """Temperatures and soft-caps whose reciprocals or squares fp32 does not have are refused; the ones beside them are not."""
    z = torch.randn(3, 9, generator=torch.Generator().manual_seed(2)).to(device)
    t = torch.tensor([1, 2, 3], device=device)
    for kw in (dict(temperature=1e-40), dict(temperature=1e30), dict(softcap=1e-40), dict(softcap=1e39), dict(softcap=5e-324), dict(softcap=float("inf"))):
        for call in (lambda kw: ops.token_logprobs(z, t, **kw), lambda kw: ops.policy_loss(z, t, **kw), lambda kw: ops.distill_loss(z, t[:, None], z[:, :1], **kw)):
            with pytest.raises(ValueError):
                call(kw)
    flat = torch.full((3,), -torch.log(torch.tensor(9.0)).item(), device=device)
    for kw in (dict(temperature=1e18), dict(softcap=1e-37)):
        torch.testing.assert_close(ops.token_logprobs(z, t, **kw).logprobs, flat, rtol=1e-6, atol=0)
    likeliest = ops.token_logprobs(z, z.argmax(-1), temperature=1e-6)
    assert likeliest.logprobs.tolist() == [0.0] * 3 and likeliest.entropy.tolist() == [0.0] * 3
    torch.testing.assert_close(ops.token_logprobs(z, t, softcap=1e30).logprobs, ops.token_logprobs(z, t).logprobs, rtol=1e-5, atol=1e-6)


def test_extreme_scales():
    check_extreme_scales("cpu")
    am = build_tiny(dims=DIMS, max_seq_len=64, batch_tokens=96)
    for tau in (1e-40, 1e30):
        with pytest.raises(ValueError, match="score"):
            am.score(_sequences(1), temperature=tau)


def check_infinity_under_a_cap(device):
    """A logit of +inf is at the cap, with no slope: scores, losses and gradients as the definition has them."""
    T, V, cap = 5, 2100, 15.0
    for dtype in (BF16, F16, F32):
        z = wide(T, V, dtype, device)[1].clone()
        z[:, 7] = float("inf")
        t = torch.tensor([7, 3, 2099, -100, 7], device=device)
        on = on_rows(T, V, t, None, device=device)
        _, _, lp, ent, lse, ids, top = scores(z, t, on, 1.0, cap, 4)
        s = ops.token_logprobs(z, t, softcap=cap, top_k=4)
        for got, want in zip((s.logprobs, s.entropy, s.lse), (lp, ent, lse)):
            near(got[on], want.detach(), V, cap, size=3.0)
        assert torch.equal(s.top_ids[on], ids)
        near(s.top_logprobs[on], top.detach(), V, cap)
        (loss, _, _), want, size = policy(z, t, on, 1.0, cap, None, None, None, 0.2, 0.2, 0.0, 0.01, 1.0)
        near(ops.policy_loss_(z, t, entropy_coef=0.01, softcap=cap, out=(out := torch.empty_like(z))).loss, loss, V, cap)
        near_grad(out, want, size, z, cap)
        assert bool((out[:, 7].float().abs() < 1e-25).all())  # (4 e^-2y of a y that the kernel stops at; in fp32, fp16 has no 1e-25)
        teacher_ids, q = some_teacher(z, 5, 1.0, cap)
        loss, want, size = distill(z, teacher_ids, q, t, on, "bucket", 0.3, 1.0, cap, 1.0)
        near(ops.distill_loss_(z, teacher_ids, q, targets=t, rest="bucket", ce_weight=0.3, softcap=cap, out=out), loss, V, cap, size=12.0)
        near_grad(out, want, size, z, cap)
        one = torch.ones(T, device=device)
        want, size = scores_grad(z, t, on, 1.0, cap, one, one, None, None, 1.0)
        ops.token_logprobs_bwd_(z, t, s, dlogprobs=one, dentropy=one, softcap=cap, out=out)
        near_grad(out, want, size, z, cap)


def test_infinity_under_a_cap():
    check_infinity_under_a_cap("cpu")


def check_given_token_under_a_mask(device):
    """A given token, an alternative and a teacher's token whose logits are the type's lowest value: their log probabilities are that less
    what the others sum to, finite numbers, so that the same policy's ratio is one and the cross entropy is finite."""
    for dtype in (BF16, F32, F16):
        for V in (6, 30000):
            low = torch.finfo(dtype).min
            z = torch.randn(3, V, generator=torch.Generator().manual_seed(11)).to(dtype).to(device)
            z[:, 2] = low
            if V == 6:
                z[2, 1:5] = low
            t = torch.tensor([2, 2, 1], device=device)
            s = ops.token_logprobs(z, t, top_k=min(V, 6))
            x = z.double()
            want = torch.log_softmax(x, -1)
            given = want.gather(1, t[:, None])[:, 0]
            # (a rounding of the difference and one of the sum's logarithm, the first of the value's size)
            at_most = lambda v: 2.0 ** -22 * (40 + 4 * (V / 256) ** 0.5) * (1 + v.abs())                                  # noqa: E731
            assert bool(s.logprobs.isfinite().all()) and bool(((s.logprobs - given).abs() <= at_most(given)).all())
            top = want.gather(1, s.top_ids)
            assert bool(s.top_logprobs.isfinite().all()) and bool(((s.top_logprobs - top).abs() <= at_most(top)).all())
            a = torch.tensor([1.0, -2.0, 0.5], device=device)
            out = torch.empty_like(z)
            for loss in (ops.policy_loss(z, t, a, old_logprobs=s.logprobs).loss, ops.policy_loss_(z, t, a, old_logprobs=s.logprobs, out=out).loss):
                assert torch.equal(loss, -a)
            # dL/dx = a (p - 1[t])
            grad = a.double()[:, None] * (torch.softmax(x, -1) - torch.nn.functional.one_hot(t, V))
            assert bool(((out - grad).abs() <= (torch.finfo(dtype).eps / 2 + 2e-5) * grad.abs() + torch.finfo(dtype).smallest_normal).all())
            ids, q = torch.tensor([0, 1], device=device).repeat(3, 1), torch.log(torch.tensor([0.5, 0.25], device=device)).repeat(3, 1)
            for rest in ("drop", "bucket"):
                loss = ops.distill_loss_(z, ids, q, targets=t, rest=rest, ce_weight=0.5, out=out)
                assert bool(loss.isfinite().all()) and bool(out.isfinite().all())
                alone = ops.distill_loss(z, ids, q, targets=t, rest=rest, ce_weight=1.0)
                assert bool(((alone + given).abs() <= at_most(given)).all())


def test_given_token_under_a_mask():
    check_given_token_under_a_mask("cpu")
