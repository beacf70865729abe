"""The vocabulary loss on the GPU, row by row and column by column, where their sizes lie far apart: in either form every result is as good
as what it sums, whatever else its operands' rows hold."""
import numpy as np
import pytest

from tests import language_bounds as B
from tests import language_ref as R
from tests.test_gpu_language import K, Loss, form, lib  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu

SHAPES = [(40, 33, 170), (300, 96, 1000), (64, 256, 4000), (7, 512, 4099), (600, 128, 2048)]


def check(K, x, w, b, labels, grads="xwb"):
    ref = R.vocab_loss(x, w, b, labels)
    c = Loss(K, x, w, b, labels, grads=grads)
    c.run()
    wrong = B.beyond(c.get(), ref, B.bounds(x, w, ref))
    assert not wrong, "; ".join(wrong)


@pytest.mark.parametrize("what", ["w", "x", "both"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_loss_columns_of_unlike_sizes(K, form, shape, what):
    check(K, *B.columns_of_unlike_sizes(*shape, 5, what))


@pytest.mark.parametrize("what", ["w", "x"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_loss_rows_of_far_unlike_sizes(K, form, shape, what):
    check(K, *B.rows_of_unlike_sizes(*shape, 5, what))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_loss_scored_columns_of_unlike_sizes(K, form, shape):
    check(K, *B.columns_of_unlike_sizes(*shape, 6, "both"), grads="")
