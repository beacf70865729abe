"""Attention's kernels on the GPU, each row on its own scale: random inputs, and values, gradients, keys and queries far larger than
the ones a row counts."""
import numpy as np
import pytest

from newch_amd import abi, hip
from tests import attention_accuracy as A

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    L = abi.load(abi.LIB_PATH)
    assert L.nc_device_count() > 0, "no HIP device visible: the GPU tests need an MI355X"
    return hip.Kernels(L)


# B, Lq, Lk, Hq, Hkv, D: every kernel and what it is built for -- rows of tokens; few keys (one pass back, two waves to 32 keys back,
# packed back); packed keys whole, in parts joined either way, with two groups of waves, of every padded width
SHAPES = [(2, 1, 700, 4, 4, 64), (1, 2, 600, 12, 3, 128), (1, 3, 300, 2, 1, 250), (2, 60, 77, 4, 2, 64), (1, 300, 40, 2, 2, 30),
          (1, 70, 128, 3, 3, 128), (1, 50, 120, 2, 2, 80), (1, 70, 200, 2, 1, 64), (1, 40, 170, 2, 2, 96), (1, 33, 300, 2, 2, 32),
          (2, 150, 333, 4, 2, 80), (1, 20, 3000, 2, 2, 128), (1, 3000, 700, 2, 2, 96), (1, 130, 600, 2, 1, 200), (33, 9, 161, 8, 8, 128),
          (40, 10, 300, 7, 7, 64), (1, 400, 520, 2, 2, 16)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_random_inputs(K, shape):
    print("random", shape, flush=True)
    q, k, v, g, _ = A.random_inputs((*shape, None), 51)
    # a few queries' errors do not average: rows alone
    A.check(A.run(K, q, k, v, g, None, shape[5] ** -0.5), A.forward_backward(q, k, v, None, shape[5] ** -0.5, g), str(shape), whole=shape[1] > 8)


def members(n, where):
    i = np.arange(n)
    return {"first": i < 1, "some": i % 7 == 3, "tile": (i // 32) % 2 == 0 if n > 32 else i < n // 2, "last": i == n - 1}[where]


@pytest.mark.parametrize("where", ["first", "some", "tile", "last"])
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[5] > 2 and s[1] > 1], ids=str)
def test_far_larger_values_that_a_row_does_not_count(K, shape, where):
    """Values, and output gradients, of one group from 2^7 to 2^50 times the other's, whose probabilities across are zero: the other
    group's outputs and gradients do not lose a bit to them, wherever they lie among the tiles."""
    B, Lq, Lk, Hq, Hkv, D = shape
    fq, fk = members(Lq, where), members(Lk, where)
    q, k, v, g = A.two_groups((*shape, None), 52, fq, fk)
    scale = D ** -0.5
    for e in (7, 11, 13, 16, 20, 30, 40, 50):
        print("values", shape, where, e, flush=True)
        big, far = v.copy(), g.copy()
        big[:, fk] *= np.float32(2.0 ** e)
        far[:, fq] *= np.float32(2.0 ** e)
        got, want = A.run(K, q, k, big, far, None, scale), A.forward_backward(q, k, big, None, scale, far)
        A.check(got, want, f"2^{e} near", pick={"o": ~fq, "gq": ~fq, "gk": ~fk, "gv": ~fk}, skip=2, whole=False)
        A.check(got, want, f"2^{e} far", pick={"o": fq, "gq": fq, "gk": fk, "gv": fk}, skip=2, whole=False)


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1] > 1], ids=str)
def test_values_of_every_magnitude_weighed_alike(K, shape):
    """A key's probability falls as its value grows: each adds as much to o, and o holds all of them."""
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v, g, _ = A.random_inputs((*shape, None), 53)
    scale, rng = D ** -0.5, np.random.default_rng(54)
    e = rng.integers(-20, 21, Lk).astype(np.float32)
    e[0] = 0
    a = np.float32(np.sqrt(np.log(2.0) / scale) * 2.0)
    q[..., 0], k[..., 0] = a, (-e / np.float32(4.0))[None, :, None] * a  # scores lower by e ln 2
    v *= np.exp2(e)[None, :, None, None].astype(np.float32)
    print("weighed", shape, flush=True)
    got, want = A.run(K, q, k, v, g, None, scale, backward=False), A.forward_backward(q, k, v, None, scale, g)
    # scores of up to 14 units more than the others': their roundings, of 14 / 2.3 times the size
    r = np.linalg.norm(got["o"] - want["o"], axis=-1) / np.linalg.norm(want["mag"]["o"], axis=-1)
    assert r.max() <= 7 * A.ROW, r.max()


@pytest.mark.parametrize("which", ["keys", "queries"])
@pytest.mark.parametrize("where", ["first", "some", "last"])
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1] > 1], ids=str)
def test_far_larger_keys_or_queries(K, shape, where, which):
    """Keys of 2^7 to 2^60 times the others that no query counts, or such queries without an output gradient: the others' scores,
    outputs and gradients keep their bits."""
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v, g, _ = A.random_inputs((*shape, None), 55)
    scale, fq, fk = D ** -0.5, np.zeros(Lq, bool), np.zeros(Lk, bool)
    # a column in which every query has 8 D^1/2 and the far keys -2 of their size: scores of -16 of their size, and 1.5 around it
    q[..., 0], k[..., 0] = 8 * np.sqrt(D), 0
    if which == "keys":
        fk = members(Lk, where)
        k[:, fk, :, 0] = -3
    else:
        fq = members(Lq, where)
        g[:, fq] = 0
    for e in (7, 11, 13, 16, 30, 60):
        print(which, shape, where, e, flush=True)
        q2, k2 = q.copy(), k.copy()
        q2[:, fq] *= np.float32(2.0 ** e)
        k2[:, fk] *= np.float32(2.0 ** e)
        got, want = A.run(K, q2, k2, v, g, None, scale), A.forward_backward(q2, k2, v, None, scale, g)
        A.check(got, want, f"{which} 2^{e}", pick={"o": ~fq, "gq": ~fq, "gk": ~fk, "gv": ~fk}, skip=1, whole=False)
        lse = np.abs(got["lse"] - want["lse"])[:, :, ~fq]
        assert lse.max() <= 2.0 ** -17 * max(1.0, np.abs(want["lse"][:, :, ~fq]).max()), lse.max()


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1] > 1], ids=str)
def test_rows_of_every_magnitude(K, shape):
    """Values, output gradients and keys from 2^-20 to 2^20 of each other row by row, stored and added: each row keeps its bits."""
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v, g, _ = A.random_inputs((*shape, None), 61)
    rng = np.random.default_rng(62)
    v *= np.exp2(rng.integers(-20, 21, v.shape[:3])).astype(np.float32)[..., None]
    g *= np.exp2(rng.integers(-20, 21, g.shape[:3])).astype(np.float32)[..., None]
    q *= np.exp2(rng.integers(-20, 1, q.shape[:3])).astype(np.float32)[..., None]
    k *= np.exp2(rng.integers(-20, 1, k.shape[:3])).astype(np.float32)[..., None]
    print("magnitudes", shape, flush=True)
    want = A.forward_backward(q, k, v, None, D ** -0.5, g)
    got = A.run(K, q, k, v, g, None, D ** -0.5)
    A.check(got, want, str(shape), whole=False)
    added = A.run(K, q, k, v, g, None, D ** -0.5, old=0.0)
    for i in ("gq", "gk", "gv"):
        assert (added[i] == got[i]).all(), i


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1] > 1], ids=str)
def test_keys_that_are_hardly_counted(K, shape):
    """Keys whose probabilities are 2^-20 to 2^-60 in every row: their gradients are small, not rough.  Their scores are 42 units below
    the others' at most, whose roundings are 42 / 2.3 times the size."""
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v, g, _ = A.random_inputs((*shape, None), 63)
    e = np.where(np.arange(Lk) % 3 == 1, np.linspace(20, 60, Lk), 0.0)
    a = np.float32(np.sqrt(np.log(2.0) * np.sqrt(D)))
    q[..., 0], k[..., 0] = a, (-e * a)[None, :, None]
    print("hardly", shape, flush=True)
    got, want = A.run(K, q, k, v, g, None, D ** -0.5), A.forward_backward(q, k, v, None, D ** -0.5, g)
    for i in ("gk", "gv"):
        err, top = (np.linalg.norm(t[..., 1:], axis=-1) for t in (got[i] - want[i], want["mag"][i]))
        assert (err <= 18 * A.ROW * top).all(), (i, (err / top).max())
