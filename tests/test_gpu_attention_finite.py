"""Operands that are not finite in every attention kernel, and the per-head norm's rows at its ends."""
import numpy as np
import pytest

from newch_amd import abi, hip
from newch_amd.hipmem import DeviceBuffer, synchronize
from tests import attention_accuracy as A

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    L = abi.load(abi.LIB_PATH)
    assert L.nc_device_count() > 0, "no HIP device visible: the GPU tests need an MI355X"
    return hip.Kernels(L)


# rows of tokens whole, in parts joined by rows; nine rows and more: few keys, packed, in parts joined either way
FINITE_SHAPES = [(1, 1, 40, 2, 2, 64), (1, 1, 3000, 1, 1, 64), (1, 8, 40, 2, 2, 64), (1, 2, 2000, 8, 2, 100), (1, 9, 40, 2, 2, 64),
                 (1, 20, 300, 2, 2, 64), (1, 20, 3000, 2, 2, 128), (1, 3000, 700, 2, 2, 96), (1, 40, 90, 2, 1, 200)]


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan], ids=str)
@pytest.mark.parametrize("operand", ["q", "k", "v"])
@pytest.mark.parametrize("shape", FINITE_SHAPES, ids=str)
def test_a_value_that_is_not_finite_gives_nan_where_it_counts(K, shape, operand, value):
    """In a query its row, in a key every row of the heads that share it, in a value that column of them; the same in every kernel, and
    the other sequences, heads and rows as they are."""
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v, g, _ = A.random_inputs((*shape, None), 56)
    want = A.forward_backward(q, k, v, None, D ** -0.5, g)
    rows, cols = np.zeros((1, Lq, Hq), bool), np.ones(D, bool)
    if operand == "q":
        q[0, Lq // 2, 0, 1] = value
        rows[0, Lq // 2, 0] = True
    else:
        (k if operand == "k" else v)[0, Lk // 3, 0, 1] = value
        rows[0, :, : Hq // Hkv] = True
        if operand == "v":
            cols[:] = False
            cols[1] = True
    print("not finite", shape, operand, value, flush=True)
    got = A.run(K, q, k, v, g, None, D ** -0.5, backward=False)
    nan = rows[..., None] & cols
    assert np.isnan(got["o"][nan]).all()
    if operand != "v":
        assert np.isnan(got["lse"].transpose(0, 2, 1)[rows]).all()
    assert np.isfinite(got["o"][~nan]).all()
    err = np.where(nan, 0.0, got["o"] - want["o"])
    assert (np.linalg.norm(err, axis=-1) <= A.ROW * np.linalg.norm(want["mag"]["o"], axis=-1)).all()


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan], ids=str)
@pytest.mark.parametrize("operand", ["q", "k", "v"])
@pytest.mark.parametrize("shape", FINITE_SHAPES, ids=str)
def test_gradients_that_meet_a_value_that_is_not_finite(K, shape, operand, value):
    """In a query: its own gradient and those of its head's keys and values.  In a key or a value: the gradients of all that share the
    head.  Other heads' are as they are."""
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v, g, _ = A.random_inputs((*shape, None), 60)
    want = A.forward_backward(q, k, v, None, D ** -0.5, g)
    rows = np.zeros((1, Lq, Hq), bool)
    if operand == "q":
        q[0, Lq // 2, 0, 1] = value
        rows[0, Lq // 2, 0] = True
    else:
        (k if operand == "k" else v)[0, Lk // 3, 0, 1] = value
        rows[0, :, : Hq // Hkv] = True
    print("gradients", shape, operand, value, flush=True)
    got = A.run(K, q, k, v, g, None, D ** -0.5)
    assert np.isnan(got["gq"][rows]).all()
    assert np.isnan(got["gk"][:, :, 0]).all()
    if operand != "v":
        assert np.isnan(got["gv"][:, :, 0]).all()
    for i, rest in (("gq", ~rows), ("gk", np.arange(Hkv) > 0), ("gv", np.arange(Hkv) > 0)):
        pick = rest if i == "gq" else np.broadcast_to(rest, (1, Lk, Hkv))
        err, top = (np.linalg.norm(t[pick], axis=-1) for t in (got[i] - want[i], want["mag"][i]))
        assert (err <= A.ROW * top).all(), i


@pytest.mark.parametrize("shape", FINITE_SHAPES, ids=str)
def test_scores_that_are_all_infinite_are_not_no_keys(K, shape):
    """A query of +inf in a column where every key is negative: every score is -inf, and the row is NaN, not the zeros of no keys."""
    q, k, v, g, _ = A.random_inputs((*shape, None), 57)
    k[..., 0] = -1 - np.abs(k[..., 0])
    q[0, 0, 0, 0] = np.inf
    print("all -inf", shape, flush=True)
    got = A.run(K, q, k, v, g, None, shape[5] ** -0.5, backward=False)
    assert np.isnan(got["o"][0, 0, 0]).all() and np.isnan(got["lse"][0, 0, 0])


@pytest.mark.parametrize("shape", [(1, 1, 40, 2, 2, 64), (1, 1, 3000, 1, 1, 64)], ids=str)
def test_scores_past_a_float_in_tokens(K, shape):
    """Finite keys whose scores are below a float's range count nothing while another key counts; all of them below it leave a softmax
    of nothing but -inf, which is NaN."""
    B, Lq, Lk, Hq, Hkv, D = shape
    q, k, v, g, _ = A.random_inputs((*shape, None), 58)
    q[..., 0], k[..., 0] = 1e30, -1e30
    print("past a float", shape, flush=True)
    got = A.run(K, q, k, v, g, None, 1.0, backward=False)
    assert np.isnan(got["o"]).all() and np.isnan(got["lse"]).all()
    k[:, 7, :, 0] = 0
    got = A.run(K, q, k, v, g, None, 1.0, backward=False)
    assert (got["o"] == v[:, 7][:, None]).all()


# ---- the per-head norm's rows at its ends ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 40, 3])
def test_norm_rows_of_zeros_nan_and_infinities(K, D):
    """Zeros: zeros, and NaN where eps is 0, as the formula has it.  NaN makes its row NaN; an infinity zeros and, in its own place,
    NaN.  Other rows do not see them."""
    x = np.random.default_rng(59).standard_normal((1, 5, 2, D)).astype(np.float32)
    x[0, 1, 0] = 0
    x[0, 2, 1, 0] = np.nan
    x[0, 3, 0, 1] = -np.inf
    for eps in (1e-6, 0.0):
        X, y = A.up(x), DeviceBuffer.from_numpy(np.zeros_like(x))
        K.qk_norm_rope_fwd(1, 5, 2, D, 1, X.ptr, (10 * D, 2 * D, D), None, None, eps, None, 0, (), 1.0, 0, y.ptr)
        synchronize()
        got = y.to_numpy(np.float32, x.shape)
        assert (got[0, 1, 0] == 0).all() if eps else np.isnan(got[0, 1, 0]).all()
        assert np.isnan(got[0, 2, 1]).all()
        assert np.isnan(got[0, 3, 0, 1]) and (np.delete(got[0, 3, 0], 1) == 0).all()
        rest = np.ones((5, 2), bool)
        rest[1, 0] = rest[2, 1] = rest[3, 0] = False
        w = x[0][rest].astype(np.float64)
        w /= np.sqrt((w * w).mean(-1, keepdims=True) + eps)
        assert (np.abs(got[0][rest] - w) <= 16 * 2.0 ** -24 * np.abs(w)).all()  # the sum of squares 8 + 5 additions, halved by the root; 5 more
