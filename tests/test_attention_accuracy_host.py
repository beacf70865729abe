"""The accuracy check itself, without a device: fp32 arithmetic passes it, one operand without its low piece does not."""
import numpy as np
import pytest

from tests import attention_accuracy as A

SHAPES = [(2, 33, 77, 4, 2, 64, (77, 12)), (1, 65, 40, 2, 2, 128, None), (2, 20, 150, 2, 1, 80, (150, 0)), (1, 9, 300, 2, 2, 32, None)]
CUTS = [("s", "q"), ("s", "k"), ("o", "p"), ("o", "v"), ("dp", "go"), ("dp", "v"), ("gq", "ds"), ("gq", "k"), ("gk", "ds"), ("gk", "q"),
        ("gv", "p"), ("gv", "go")]


def plain32(q, k, v, lens, scale, go):
    """attention in fp32, the formulas as they stand"""
    f = np.float32
    out = {"o": np.zeros_like(q), "gq": np.zeros_like(q), "gk": np.zeros_like(k), "gv": np.zeros_like(v)}
    G_ = q.shape[2] // k.shape[2]
    for b in range(q.shape[0]):
        n = k.shape[1] if lens is None else int(lens[b])
        for h in range(q.shape[2]) if n else ():
            Q, K, V, G = q[b, :, h], k[b, :n, h // G_], v[b, :n, h // G_], go[b, :, h]
            s = (Q @ K.T) * f(scale)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            o = p @ V
            ds = p * (G @ V.T - (G * o).sum(1, keepdims=True)) * f(scale)
            out["o"][b, :, h], out["gq"][b, :, h] = o, ds @ K
            out["gk"][b, :n, h // G_] += ds.T @ Q
            out["gv"][b, :n, h // G_] += p.T @ G
    return out


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_fp32_passes(shape):
    q, k, v, g, lens = A.random_inputs(shape, 1)
    scale = shape[5] ** -0.5
    A.check(plain32(q, k, v, lens, scale, g), A.forward_backward(q, k, v, lens, scale, g))


@pytest.mark.parametrize("cut", CUTS, ids="-".join)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_an_operand_without_its_low_piece_shows(shape, cut):
    q, k, v, g, lens = A.random_inputs(shape, 2)
    scale = shape[5] ** -0.5
    want, got = A.forward_backward(q, k, v, lens, scale, g), A.forward_backward(q, k, v, lens, scale, g, cut)
    with pytest.raises(AssertionError, match="off by"):
        A.check(got, want)


def test_rows_of_two_groups_do_not_see_each_other():
    """What one group holds leaves the other's results as they are, and fp32 keeps them."""
    shape = (1, 40, 70, 2, 2, 64, None)
    fq, fk = np.arange(40) % 7 == 3, np.arange(70) % 9 == 0
    q, k, v, g = A.two_groups(shape, 3, fq, fk)
    big = [t.copy() for t in (q, k, v, g)]
    big[2][:, fk] *= np.float32(2.0 ** 40)
    big[3][:, fq] *= np.float32(2.0 ** 40)
    one, two = A.forward_backward(q, k, v, None, 0.125, g), A.forward_backward(*big[:3], None, 0.125, big[3])
    pick = {"o": ~fq, "gq": ~fq, "gk": ~fk, "gv": ~fk}
    for name, at in pick.items():
        assert np.abs(one[name][:, at, :, 2:] - two[name][:, at, :, 2:]).max() < 1e-12, name
    A.check(plain32(*big[:3], None, 0.125, big[3]), two, pick=pick, skip=2)
