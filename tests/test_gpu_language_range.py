"""The vocabulary loss on the GPU at the ends of a float's range, in either form: gradients whose sums pass it before they are scaled, and values
that are not finite."""
import numpy as np
import pytest

from tests import language_bounds as B
from tests import language_ref as R
from tests.test_gpu_language import HALF, K, Loss, form, lib, loss_inputs, rms  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


# N, D, V, the large operand, its size and the other's, words that are labels; the last one's gW is not cut
@pytest.mark.parametrize("acc", [False, True])
@pytest.mark.parametrize("case", [(300, 2, 5, "x", 1e37, 1e-37, 5), (300, 2, 5, "w", 2e38, 2e-38, 5), (400, 3, 300, "x", 1e37, 5e-38, 5),
                                  (400, 3, 300, "w", 2e38, 1.5e-38, 5), (600, 385, 16130, "x", 1e36, 2e-38, 1)], ids=str)
def test_gradients_whose_sums_overflow_unscaled(K, form, case, acc):
    """gW sums hundreds of rows of 1e36 and more, gx differences of words of 2e38: only the mean is a float."""
    N, D, V, big, far, near, words = case
    rng = np.random.default_rng(8)
    a, b = rng.uniform(0.8, 1.0, (N, D)), rng.uniform(0.8, 1.0, (V, D)) * rng.choice((-1, 1), (V, 1))
    x, w = ((a * far, b * near) if big == "x" else (a * near, b * far))
    x, w = x.astype(np.float32), w.astype(np.float32)
    labels = rng.integers(0, words, N).astype(np.int32)
    ref = R.vocab_loss(x, w, None, labels)
    assert np.abs(ref["gw" if big == "x" else "gx"]).max() * N > 3.45e38 > float(np.abs(x).max())
    old = {k: (ref[k] * rng.uniform(-1, 1, ref[k].shape)).astype(np.float32) for k in ("gx", "gw", "gb")} if acc else None
    c = Loss(K, x, w, None, labels, old=old)
    c.run()
    wrong = B.beyond(c.get(), ref, B.bounds(x, w, ref), old=old)
    assert not wrong, "; ".join(wrong)


@pytest.mark.parametrize("gout", [1e30, -1e-30])
@pytest.mark.parametrize("shape", [(40, 33, 170), (300, 96, 1000)], ids=str)
def test_gradients_of_large_and_small_losses(K, form, shape, gout):
    """The loss's own gradient far from 1, taken into the operands' sizes or not."""
    x, w, b, labels = loss_inputs(*shape, 61, True, 0.1)
    for size in (1.0, 2.0 ** -40, 2.0 ** 40):
        xs, ws = x * np.float32(size), w * np.float32(1 / size)
        ref = R.vocab_loss(xs, ws, b, labels, gout=np.float32(gout))
        c = Loss(K, xs, ws, b, labels, gout=gout)
        c.run()
        got = {k: v for k, v in c.get().items() if k == "loss" or np.abs(ref[k]).max() < 3e38}  # 2^40 times 1e30 is not a float
        assert len(got) >= 4
        wrong = B.beyond(got, ref, B.bounds(xs, ws, ref))
        assert not wrong, "; ".join(wrong)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("shape", [(40, 33, 170), (300, 96, 1000), (9, 512, 4099)], ids=str)
def test_a_row_that_is_not_finite(K, form, shape, value):
    """It has no loss and no gradient, gW and gb have none, and the other rows have theirs."""
    N, D, V = shape
    x, w, b, labels = loss_inputs(*shape, 62, True, 0.0)
    ref = R.vocab_loss(x, w, b, labels)
    tol = B.bounds(x, w, ref)
    x[7, 3] = value
    c = Loss(K, x, w, b, labels)
    c.run()
    got = c.get()
    assert not np.isfinite(got["loss"]) and not np.isfinite(got["rows"][7]) and np.isnan(got["gx"][7]).all()
    assert np.isnan(got["gw"]).all() and np.isnan(got["gb"]).all()
    others = np.arange(N) != 7
    assert (np.abs(got["rows"][others] - ref["rows"][others]) <= tol["rows"][others] + HALF * ref["rows"][others]).all()
    assert rms(got["gx"][others] - ref["gx"][others]) <= rms(tol["gx"][others]) + HALF * rms(ref["gx"])


@pytest.mark.parametrize("shape", [(40, 33, 170), (300, 96, 1000), (9, 512, 4099)], ids=str)
def test_words_that_are_not_finite(K, form, shape):
    """A word of NaN, or a bias of NaN or +inf, leaves no row a loss.  A word with an infinity leaves none in pieces; on fp32 products the rows
    that give it -inf keep theirs."""
    x, w, b, labels = loss_inputs(*shape, 63, True, 0.0)
    labels[labels == 5] = 4
    for where, value in ((b, np.nan), (b, np.inf), (w[:, 1], np.nan), (w[:, 1], np.inf), (w[:, 1], -np.inf)):
        keep = where[5]
        where[5] = value
        c = Loss(K, x, w, b, labels, grads="")
        c.run()
        rows = c.get()["rows"]
        if where is not b and np.isinf(value) and form == "fp32":
            out = x[:, 1] * value < 0
            where[5] = keep
            masked = b.copy()
            masked[5] = -np.inf
            ref = R.vocab_loss(x, w, masked, labels)
            assert out.any() and not out.all()
            assert (np.isfinite(rows) == out).all()
            assert (np.abs(rows - ref["rows"])[out] <= (B.bounds(x, w, ref)["rows"] + HALF * ref["rows"])[out]).all()
        else:
            assert np.isnan(rows).all()
        where[5] = keep
