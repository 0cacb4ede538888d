"""Operators on token probabilities on a GPU: what a later look at them found."""
import pytest
import torch

from flextrain_b200.nn.loss import GRPOLoss, TokenSlice
from test_token_loss_more_cpu import (check_common_offset, check_cross_entropy_alone, check_extreme_scales, check_infinite_ratio,
                                      check_given_token_under_a_mask, check_infinity_under_a_cap, check_rows_of_nan)
from token_loss_oracle import near, some_targets, wide

pytestmark = pytest.mark.gpu


def test_rows_of_nan():
    check_rows_of_nan("cuda")


def test_cross_entropy_alone():
    check_cross_entropy_alone("cuda")


@pytest.mark.parametrize("offset", [0.0, 36.0, -300.0, 1000.0, 2500.0])
def test_common_offset(offset):
    check_common_offset("cuda", offset, T=600)                # (a row has a dozen gradients apart from each other, and fp16 shows one in a hundred)


def test_grpo_loss_of_every_kind_that_it_took():
    """What the plain form takes the kernel's does too: an advantage for all rows, columns as rows, targets of another type, negative
    targets but -100 (which count as token 0), a reference that no penalty reads."""
    T, V = 9, 301
    z = wide(T, V, torch.float32, "cpu")[1].clone()
    t = some_targets(T, V, "cpu").clamp(max=V - 1)
    t[5] = -1
    adv = torch.linspace(-1, 1, T)
    ref = torch.linspace(-7, -5, T)
    cases = [dict(advantages=torch.tensor(0.5)), dict(advantages=torch.tensor([0.5])), dict(advantages=adv.double()), dict(),
             dict(advantages=adv, ref_logprobs=torch.tensor(-6.0)), dict(advantages=adv, ref_logprobs=ref)]
    for kl, targets, more in [(0.1, t, c) for c in cases] + [(0.1, t.float(), cases[2]), (0.1, t.int(), {}), (0.0, t, dict(ref_logprobs=ref[:3])),
                                                             (-0.5, t, dict(ref_logprobs=ref))]:
        want_z = z.clone()
        want = GRPOLoss(kl_beta=kl)(want_z, TokenSlice(targets, **more), 0.5)
        for columns in (False, True):
            got_z = z.cuda().t().contiguous().t() if columns else z.cuda()
            got = GRPOLoss(kl_beta=kl)(got_z, TokenSlice(targets.cuda(), **{k: v.cuda() for k, v in more.items()}), 0.5)
            # both sides' errors: the penalty's e^d multiplies the log probability's, which is up to 16 times 2.6e-6 off (near()); a
            # gradient is off by the same share of itself, 8e-5 of both sides, and 1e-5 by its probability
            near(got.cpu(), want.double(), V, factor=2 * 55.0)
            assert bool(((got_z.cpu() - want_z).abs() <= 1e-4 * (want_z.abs() + 1e-3)).all()), (kl, targets.dtype, list(more), columns)


def test_infinite_ratio():
    check_infinite_ratio("cuda")


def test_extreme_scales():
    check_extreme_scales("cuda")


def test_infinity_under_a_cap():
    check_infinity_under_a_cap("cuda")


def test_given_token_under_a_mask():
    check_given_token_under_a_mask("cuda")
