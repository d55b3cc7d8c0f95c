"""Refusals of the paged serving operators at the ends of their ranges, on the
CPU (stand-in addresses, as in test_paged_refusals.py)."""
import os

import pytest

from myos import _lib
from test_paged_refusals import BASE, built, logits  # noqa: F401

TOP = 1 << 30


def listed(pen, width, nbias):
    return logits(dict(history=BASE, history_width=width, history_stride=width, bias_starts=BASE, bias_ids=BASE,
                       bias_vals=BASE, num_bias=nbias, **pen))


def test_a_row_lists_fewer_than_2_31_tokens_and_biases():
    """A block counts its row's tokens and biases in 31 bits."""
    assert listed(dict(presence=BASE), TOP, TOP) == _lib.ERR_SHAPE


@pytest.mark.skipif(os.path.exists("/dev/nvidiactl") or os.path.exists("/dev/nvidia0"), reason="no-GPU behaviour")
@pytest.mark.parametrize("pen,width,nbias", [
    (dict(repetition=BASE), TOP, TOP - 1), (dict(frequency=BASE), TOP - 1, TOP),
    ({}, TOP, TOP)])  # no penalties: the tokens are not listed
def test_one_fewer_passes_the_checks(pen, width, nbias):
    assert listed(pen, width, nbias) == _lib.ERR_CUDA
