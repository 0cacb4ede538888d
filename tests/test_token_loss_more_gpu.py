"""Operators on token probabilities on a GPU: what a later look at them found."""
import pytest

from test_token_loss_more_cpu import check_common_offset, check_cross_entropy_alone, check_rows_of_nan

pytestmark = pytest.mark.gpu


def test_rows_of_nan():
    check_rows_of_nan("cuda")


def test_cross_entropy_alone():
    check_cross_entropy_alone("cuda")


@pytest.mark.parametrize("offset", [0.0, -300.0, 1000.0, 2500.0])
def test_common_offset(offset):
    check_common_offset("cuda", offset, T=600)                # (a row has a dozen gradients apart from each other, and fp16 shows one in a hundred)
