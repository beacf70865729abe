"""The vocabulary loss on the GPU at the ends of a float's range, in either form: gradients whose sums pass it before they are scaled."""
import numpy as np
import pytest

from tests import language_bounds as B
from tests import language_ref as R
from tests.test_gpu_language import K, Loss, form, lib, loss_inputs  # noqa: F401  (fixtures)

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
    assert np.abs(ref["gw" if big == "x" else "gx"]).max() * N > 3.45e38 > np.abs(x).max()
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
