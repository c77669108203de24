"""Refusals of the wattn_paged_* entry points at the edges of their ranges. (As
in test_paged_abi.py: made-up addresses, where no GPU is.)"""
import pytest
import torch

from tests.test_paged_abi import ATTEND, W, refused  # noqa: F401

pytestmark = pytest.mark.skipif(torch.cuda.is_available(),
                                reason="made-up device addresses are only passed where no GPU is")


@pytest.mark.parametrize("scale", [2.5e38, 3.0e38, -1.0, -float("inf")])
def test_scales_that_overflow_in_base_2_are_refused(W, scale):
    """Scores are taken times log2 e: a scale that is infinite then would make
    0 times it NaN."""
    refused(W, W.lib.wattn_paged_attend, ATTEND, 21, scale, -1, b"scale")
