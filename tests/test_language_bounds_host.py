"""The bounds that the vocabulary loss's gradients are held to entry by entry tell operands whose pieces keep what they should from ones that
do not: on the CPU, with the scheme in numpy."""
import numpy as np
import pytest

from tests import language_bounds as B
from tests import language_ref as R

SHAPES = [(40, 33, 170), (64, 256, 1000)]


def case(make, shape, what):
    x, w, b, labels = make(*shape, 5, what)
    return x, w, b, dict(R.vocab_loss(x, w, b, labels), labels=labels)


@pytest.mark.parametrize("what", ["w", "x", "both"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_columns_of_unlike_sizes(shape, what):
    x, w, b, ref = case(B.columns_of_unlike_sizes, shape, what)
    tol = B.bounds(x, w, ref)
    assert not B.beyond(B.loss_in_pieces(x, w, b, ref), ref, tol)
    assert B.beyond(B.loss_in_pieces(x, w, b, ref, low=0), ref, tol), "pieces that end at 2^-40 of a row's largest pass"


@pytest.mark.parametrize("what", ["w", "x"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rows_of_unlike_sizes(shape, what):
    x, w, b, ref = case(B.rows_of_unlike_sizes, shape, what)
    tol = B.bounds(x, w, ref)
    assert not B.beyond(B.loss_in_pieces(x, w, b, ref), ref, tol)
    assert B.beyond(B.loss_in_pieces(x, w, b, ref, by_row=False), ref, tol), "one power for the whole matrix passes"
    assert B.beyond(B.loss_in_pieces(x, w, b, ref, by_term=False), ref, tol), "powers of G's entries pass"
