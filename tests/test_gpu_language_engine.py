"""A language model's two ends through the engine at their edges: nothing to work on, single tokens and rows, views of every input, one tensor
in several places, calls after a refused one, persistent results and gradients switched off."""
import ctypes
from ctypes import c_double, c_float, c_int32, c_uint64

import numpy as np
import pytest

from newch_amd import abi
from tests import language_ref as R
from tests.ncdrive import NcError
from tests.test_gpu_language import HALF, agree, eng, lib, loss_inputs, rms  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def embedding(L, w, t, scale=1.0, padding=-1):
    return L.nc_embedding(w, t, c_float(scale), c_int32(padding))


def loss_of(L, x, w, b, labels, ignore=-100, total=0):
    return L.nc_linear_cross_entropy(x, w, b, labels, c_int32(ignore), total)


def drop(L, x, r, p, seed=5, offset=6):
    return L.nc_dropout_seeded(x, r, c_double(p), c_uint64(seed), c_uint64(offset))


@pytest.mark.parametrize("total", [0, 1])
@pytest.mark.parametrize("lead", [(0,), (2, 0)], ids=str)
def test_loss_of_no_rows(eng, lead, total):
    L, rng = eng.lib, np.random.default_rng(1)
    w, b = rng.standard_normal((9, 5)).astype(np.float32), rng.standard_normal(9).astype(np.float32)
    x, pw, pb = eng.param(np.zeros(lead + (5,), np.float32)), eng.param(w), eng.param(b)
    y = loss_of(L, x, pw, pb, eng.tensor(np.zeros(lead, np.int32)), total=total)
    got = eng.read(y)
    assert got.shape == () and (got == 0 if total else np.isnan(got))
    if total:
        assert L.nc_backward(y) == 0, L.nc_error(eng.ctx)
        assert (eng.grad(pw) == 0).all() and (eng.grad(pb) == 0).all()
    eng.step_end()


def test_loss_of_one_row_without_a_dim(eng):
    L = eng.lib
    x, w, b, labels = loss_inputs(1, 6, 9, 71, True, 0.0)
    px, pw = eng.param(x[0]), eng.param(w)
    y = loss_of(L, px, pw, eng.tensor(b), eng.tensor(np.array(labels[0], np.int32)))
    ref = R.vocab_loss(x, w, b, labels)
    assert L.nc_backward(y) == 0, L.nc_error(eng.ctx)
    agree({"gx": eng.grad(px)[None], "gw": eng.grad(pw), "loss": eng.read(y)}, ref, x, w)
    eng.step_end()


def test_loss_of_views(eng):
    """Rows apart, turned and strided inputs; gradients reach what the views are of."""
    L, rng = eng.lib, np.random.default_rng(72)
    base_x, base_w, base_b = (rng.standard_normal(s).astype(np.float32) for s in ((40, 12), (6, 30), (31, 2)))
    px, pw, pb = eng.param(base_x), eng.param(base_w), eng.param(base_b)
    labels = rng.integers(0, 30, (2, 10)).astype(np.int32)
    x = L.nc_slice(L.nc_slice(px, 0, 3, 20, 1), 1, 2, 6, 1)  # rows 12 apart
    w = L.nc_transpose(pw, 0, 1)
    b = L.nc_slice(L.nc_transpose(pb, 0, 1), 1, 1, 30, 1)
    nd, shp = abi.shape_arg((60,))
    b = L.nc_reshape(b, nd, shp)
    b = L.nc_slice(b, 0, 0, 30, 2)
    t = L.nc_transpose(eng.tensor(np.ascontiguousarray(labels.T)), 0, 1)
    nd, shp = abi.shape_arg((20,))
    y = loss_of(L, x, w, b, L.nc_reshape(t, nd, shp))
    eng.check()
    hx, hw, hb = base_x[3:23, 2:8], base_w.T, base_b.T[:, 1:].reshape(-1)[::2]
    ref = R.vocab_loss(hx, hw, hb, labels.reshape(-1))
    assert L.nc_backward(y) == 0, L.nc_error(eng.ctx)
    gx, gw = eng.grad(px), eng.grad(pw)
    agree({"gx": gx[3:23, 2:8], "gw": gw.T, "loss": eng.read(y)}, ref, hx, hw)
    gx[3:23, 2:8] = 0
    assert (gx == 0).all()
    eng.step_end()


def test_loss_of_one_tensor_as_rows_and_words(eng):
    L = eng.lib
    _, w, _, labels = loss_inputs(30, 20, 30, 73, False, 0.1)
    p = eng.param(w)
    y = loss_of(L, p, p, None, eng.tensor(labels))
    ref = R.vocab_loss(w, w, None, labels)
    assert L.nc_backward(y) == 0, L.nc_error(eng.ctx)
    tol = R.vocab_loss_tol(w, w, ref)
    want = ref["gx"] + ref["gw"]
    assert rms(eng.grad(p) - want) <= tol["gx"] + tol["gw"] + 4 * HALF * rms(want)
    eng.step_end()


def test_calls_after_a_refused_one(eng):
    """A bad label or token fails its call alone; the next one's answer is its own."""
    L = eng.lib
    x, w, b, labels = loss_inputs(50, 12, 40, 74, False, 0.0)
    ref = R.vocab_loss(x, w, None, labels)
    tx, tw = eng.tensor(x), eng.tensor(w)
    for bad in (40, -1, 2 ** 31 - 1):
        for at in (0, 49):
            wrong = labels.copy()
            wrong[at] = bad
            for call, text in ((lambda: loss_of(L, tx, tw, None, eng.tensor(wrong)), f"label {bad} at row {at} "),
                               (lambda: embedding(L, tw, eng.tensor(wrong)), f"token {bad} at position {at} ")):
                assert not call()
                with pytest.raises(NcError, match=text):
                    eng.check()
                got = eng.read(loss_of(L, tx, tw, None, eng.tensor(labels)))
                assert abs(got - ref["loss"]) <= R.vocab_loss_tol(x, w, ref)["loss"]
                assert (eng.read(embedding(L, tw, eng.tensor(labels))) == w[labels]).all()
    eng.step_end()


def test_loss_kept_and_without_gradients(eng):
    L = eng.lib
    x, w, b, labels = loss_inputs(50, 12, 40, 75, True, 0.2)
    ref = R.vocab_loss(x, w, b, labels)
    tol = R.vocab_loss_tol(x, w, ref)["loss"]
    px, pw, pb, lab = eng.param(x), eng.param(w), eng.param(b), eng.tensor(labels)
    L.nc_persistent_begin(eng.ctx)
    kept = loss_of(L, px, pw, pb, lab)
    rows = embedding(L, pw, lab)
    L.nc_persistent_end(eng.ctx)
    assert not rows  # an ignored label is no token
    with pytest.raises(NcError):
        eng.check()
    L.nc_set_grad_enabled(eng.ctx, 0)
    y = loss_of(L, px, pw, pb, lab)
    assert not L.nc_requires_grad(y)
    L.nc_set_grad_enabled(eng.ctx, 1)
    assert abs(eng.read(y) - ref["loss"]) <= tol
    eng.step_end()
    assert L.nc_is_persistent(kept) and abs(eng.read(kept) - ref["loss"]) <= tol
    L.nc_release(kept)


def test_embedding_of_single_tokens_and_empty_tables(eng):
    L, rng = eng.lib, np.random.default_rng(76)
    w = rng.standard_normal((9, 10)).astype(np.float32)
    p = eng.param(w)
    y = embedding(L, p, eng.tensor(np.array(4, np.int32)), 2.0)
    assert eng.read(y).shape == (10,) and (eng.read(y) == w[4] * np.float32(2)).all()
    G = rng.standard_normal(10).astype(np.float32)
    eng.backward_with(y, G)
    want = np.zeros_like(w)
    want[4] = G * np.float32(2)
    assert (eng.grad(p) == want).all()
    none = eng.tensor(np.zeros((0, 10), np.float32))
    assert eng.read(embedding(L, none, eng.tensor(np.zeros((3, 0), np.int32)))).shape == (3, 0, 10)
    assert not embedding(L, none, eng.tensor(np.zeros(2, np.int32)))
    with pytest.raises(NcError, match=r"token 0 at position 0 outside \[0, 0\)"):
        eng.check()
    e = embedding(L, p, eng.tensor(np.zeros((0,), np.int32)))
    L.nc_clear_grad(p)
    assert L.nc_backward(L.nc_sum(e, abi.ALL_AXES, 0)) == 0, L.nc_error(eng.ctx)
    assert (eng.grad(p) == 0).all()
    eng.step_end()


def test_embedding_gradient_reaches_a_view(eng):
    L, rng = eng.lib, np.random.default_rng(77)
    w = rng.standard_normal((9, 12)).astype(np.float32)
    tokens = rng.integers(0, 12, (5, 3)).astype(np.int32)
    p = eng.param(w)
    y = embedding(L, L.nc_transpose(p, 0, 1), eng.tensor(tokens))
    G = rng.standard_normal((5, 3, 9)).astype(np.float32)
    eng.backward_with(y, G)
    ref, size = R.embedding_grad(tokens, G, 12, 1.0)
    assert (np.abs(eng.grad(p).T - ref) <= R.embedding_grad_tol(size)).all()
    eng.step_end()


@pytest.mark.parametrize("p", [0.0, 1.0])
def test_dropout_of_all_and_nothing(eng, p):
    L, rng = eng.lib, np.random.default_rng(78)
    x, r, G = (rng.standard_normal((3, 5)).astype(np.float32) for _ in range(3))
    px, pr = eng.param(x), eng.param(r)
    y = drop(L, px, pr, p)
    assert (eng.read(y) == (r if p else x + r)).all()
    eng.backward_with(y, G)
    assert (eng.grad(px) == (0 if p else G)).all() and (eng.grad(pr) == G).all()
    e = drop(L, eng.tensor(np.zeros((0, 4), np.float32)), None, p)
    assert eng.read(e).shape == (0, 4)
    eng.step_end()


def test_backward_twice(eng):
    """A retained graph's second backward adds the same again, with the mask of the first."""
    L, rng = eng.lib, np.random.default_rng(79)
    w, tokens = rng.standard_normal((12, 8)).astype(np.float32), rng.integers(0, 12, 20).astype(np.int32)
    G = rng.standard_normal((20, 8)).astype(np.float32)
    p = eng.param(w)
    y = drop(L, embedding(L, p, eng.tensor(tokens), 1.5), None, 0.3)
    loss = L.nc_sum(L.nc_mul(y, eng.tensor(G)), abi.ALL_AXES, 0)
    for times in (1, 2):
        assert L.nc_backward_ex(loss, abi.BACKWARD_RETAIN, None, 0) == 0, L.nc_error(eng.ctx)
        ref, size = R.embedding_grad(tokens, R.dropout(G, 0.3, 5, 6), 12, 1.5)
        assert (np.abs(eng.grad(p) - times * ref) <= times * R.embedding_grad_tol(size, ref)).all()
    eng.step_end()
