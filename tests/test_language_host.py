"""A language model's two ends without a device: refusals through both interfaces, the generator's published values, and the 64-bit
references against differences."""
import ctypes
from ctypes import c_double, c_float, c_int32, c_uint64

import numpy as np
import pytest

from newch_amd import abi, hip
from tests import language_ref as R
from tests.ncdrive import Engine


@pytest.fixture(scope="module")
def lib():
    return abi.load(abi.LIB_PATH)


@pytest.fixture()
def eng(lib):
    if lib.nc_device_count() > 0:
        pytest.skip("a HIP device is visible: the no-device behaviour is not observable here")
    e = Engine(lib=lib)
    yield e
    e.close()


def f32(*shape):
    return np.zeros(shape, np.float32)


def i32(*shape):
    return np.zeros(shape, np.int32)


def refused(e, t, status, text):
    assert not t
    assert e.lib.nc_status_code(e.ctx) == status, e.lib.nc_error(e.ctx)
    assert text in e.lib.nc_error(e.ctx).decode(), e.lib.nc_error(e.ctx)
    e.lib.nc_clear_error(e.ctx)


def test_embedding_refusals(eng):
    L, t = eng.lib, eng.tensor
    w, tok = t(f32(5, 3)), t(i32(2, 4))
    call = lambda w=w, tok=tok, s=1.0: L.nc_embedding(w, tok, c_float(s), c_int32(-1))
    refused(eng, call(), abi.ERR_STATE, "no HIP device")
    refused(eng, call(w=t(i32(5, 3))), abi.ERR_DTYPE, "f32")
    refused(eng, call(tok=t(f32(2, 4))), abi.ERR_DTYPE, "tokens must be i32")
    refused(eng, call(w=t(f32(5))), abi.ERR_SHAPE, "expected weight")
    refused(eng, call(w=t(f32(5, 0))), abi.ERR_SHAPE, "expected weight")
    refused(eng, call(tok=t(i32(1, 1, 1, 1, 1, 1))), abi.ERR_SHAPE, "at most 5 dims")
    refused(eng, call(s=float("nan")), abi.ERR_ARG, "scale")


def test_dropout_refusals(eng):
    L, t = eng.lib, eng.tensor
    x = t(f32(2, 4))
    call = lambda x=x, r=None, p=0.5: L.nc_dropout_seeded(x, r, c_double(p), c_uint64(1), c_uint64(2))
    refused(eng, call(), abi.ERR_STATE, "no HIP device")
    refused(eng, call(x=t(i32(2))), abi.ERR_DTYPE, "f32")
    refused(eng, call(r=t(i32(2, 4))), abi.ERR_DTYPE, "f32")
    refused(eng, call(r=t(f32(4, 2))), abi.ERR_SHAPE, "differ")
    for p in (-0.1, 1.5, float("nan")):
        refused(eng, call(p=p), abi.ERR_ARG, "p must be in [0, 1]")


def test_linear_cross_entropy_refusals(eng):
    L, t = eng.lib, eng.tensor
    x, w, b, lab = t(f32(2, 3, 4)), t(f32(7, 4)), t(f32(7)), t(i32(2, 3))
    call = lambda x=x, w=w, b=b, lab=lab: L.nc_linear_cross_entropy(x, w, b, lab, c_int32(-100), 0)
    refused(eng, call(), abi.ERR_STATE, "no HIP device")
    refused(eng, call(b=None), abi.ERR_STATE, "no HIP device")
    refused(eng, call(x=t(i32(2, 3, 4))), abi.ERR_DTYPE, "f32")
    refused(eng, call(b=t(i32(7))), abi.ERR_DTYPE, "f32")
    refused(eng, call(lab=t(f32(2, 3))), abi.ERR_DTYPE, "labels must be i32")
    refused(eng, call(w=t(f32(7, 5))), abi.ERR_SHAPE, "expected x")
    refused(eng, call(w=t(f32(0, 4))), abi.ERR_SHAPE, "expected x")
    refused(eng, call(lab=t(i32(6))), abi.ERR_SHAPE, "a label for each row")
    refused(eng, call(lab=t(i32(3, 2))), abi.ERR_SHAPE, "a label for each row")
    refused(eng, call(b=t(f32(4))), abi.ERR_SHAPE, "the bias needs 7")


def test_kernel_layer_refusals(lib):
    """Every one returns before it touches a device."""
    K = hip.Kernels(ctypes.CDLL(str(abi.LIB_PATH)))
    P = 4096  # an address that nothing reads

    def bad(text, fn, *a, **k):
        with pytest.raises(hip.HipLayerError, match=text):
            fn(*a, **k)

    bad("bad size", K.embedding_fwd, -1, 5, 4, P, 4, P, 1.0, P)
    bad("bad size", K.embedding_fwd, 1, 5, 0, P, 4, P, 1.0, P)
    bad("bad size", K.embedding_fwd, 1, 1 << 31, 4, P, 4, P, 1.0, P)
    bad("bad size", K.embedding_fwd, (1 << 30) + 1, 5, 4, P, 4, P, 1.0, P)
    bad("NULL", K.embedding_fwd, 1, 5, 4, None, 4, P, 1.0, P)
    bad("NULL", K.embedding_fwd, 1, 5, 4, P, 4, None, 1.0, P)
    bad("NULL", K.embedding_fwd, 1, 5, 4, P, 4, P, 1.0, None)
    bad("8-byte", K.embedding_fwd, 1, 5, 4, P, 4, P, 1.0, P, bad=P + 4)
    bad("rows closer", K.embedding_fwd, 1, 5, 4, P, 3, P, 1.0, P)
    n = K.embedding_bwd_workspace(9000, 5, 4)
    assert n > 0 and K.embedding_bwd_workspace(0, 5, 4) == 0
    bad("workspace of", K.embedding_bwd, 9000, 5, 4, P, -1, 1.0, P, P, P, n - 1)
    bad("workspace of", K.embedding_bwd, 9000, 5, 4, P, -1, 1.0, P, P, None, n)
    bad("16-byte", K.embedding_bwd, 9000, 5, 4, P, -1, 1.0, P, P, P + 4, n)
    bad("NULL", K.embedding_bwd, 9000, 5, 4, P, -1, 1.0, None, P, P, n)
    bad("NULL", K.embedding_bwd, 9000, 5, 4, P, -1, 1.0, P, None, P, n)
    for p in (-0.01, 1.01, float("nan")):
        bad("p must be", K.dropout_fwd, 4, p, 1, 2, P, None, P)
        bad("p must be", K.dropout_bwd, 4, p, 1, 2, P, P)
    bad("bad size", K.dropout_fwd, -1, 0.5, 1, 2, P, None, P)
    bad("bad size", K.dropout_fwd, 1 << 61, 0.5, 1, 2, P, None, P)
    bad("NULL", K.dropout_fwd, 4, 0.5, 1, 2, None, None, P)
    bad("NULL", K.dropout_bwd, 4, 0.5, 1, 2, P, None)
    bad("8-byte", K.dropout_fwd, 4, 0.5, 1, 2, P, None, P, offset_ptr=P + 4)
    n = K.linear_cross_entropy_workspace(5, 4, 7, gx=True, gw=True, gb=True)
    call = lambda N=5, D=4, V=7, x=P, ldx=4, w=P, ldw=4, lab=P, loss=P, ws=P, ws_bytes=n, **k: K.linear_cross_entropy(
        N, D, V, x, ldx, w, ldw, None, lab, loss, ws, ws_bytes, gx=P, gw=P, gb=P, **k)
    bad("bad size", call, N=-1)
    bad("bad size", call, N=1 << 31)
    bad("bad size", call, D=0)
    bad("bad size", call, D=(1 << 20) + 1, ldx=1 << 21, ldw=1 << 21)
    bad("bad size", call, V=0)
    bad("bad size", call, V=(1 << 26) + 1)
    for name in ("x", "w", "lab", "loss"):
        bad("NULL", call, **{name: None})
    bad("rows closer", call, ldx=3)
    bad("rows closer", call, ldw=3)
    bad("8-byte", call, bad=P + 4)
    bad("workspace of", call, ws_bytes=n - 1)
    bad("workspace of", call, ws=None)
    bad("16-byte", call, ws=P + 8)
    assert K.linear_cross_entropy_workspace(-1, 4, 7) == 0


def test_generator_gives_the_published_words():
    """The known answers published with the generator: all zeros, all ones, the digits of pi."""
    ones = 0xFFFFFFFF
    for counter, key, want in [((0,) * 4, (0,) * 2, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                               ((ones,) * 4, (ones,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                               ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                                (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]:
        assert tuple(int(v) for v in R.philox(counter, key)) == want


@pytest.mark.parametrize("bias,total", [(False, False), (True, True)])
def test_vocab_loss_reference_against_differences(bias, total):
    rng = np.random.default_rng(3)
    N, D, V, h = 5, 3, 7, 1e-5
    x, w, b = rng.standard_normal((N, D)), rng.standard_normal((V, D)), rng.standard_normal(V) if bias else None
    labels = np.array([0, 6, -100, 3, 3])
    loss = lambda: R.vocab_loss(x, w, b, labels, sum=total)["loss"]
    ref = R.vocab_loss(x, w, b, labels, sum=total)
    for name, a in (("gx", x), ("gw", w)) + ((("gb", b),) if bias else ()):
        got = np.zeros_like(a)
        for i in np.ndindex(a.shape):
            old = a[i]
            a[i] = old + h
            up = loss()
            a[i] = old - h
            got[i] = (up - loss()) / (2 * h)
            a[i] = old
        # the central difference is off by h^2 / 6 of a third derivative of order 10, and by eps / h of the loss
        assert np.abs(got - ref[name]).max() < 1e-8, name


def test_embedding_reference_against_differences():
    rng = np.random.default_rng(4)
    V, D = 6, 3
    w, tok = rng.standard_normal((V, D)), np.array([[1, 1, 5], [0, 1, 2]])
    g = rng.standard_normal((2, 3, D))
    gw, _ = R.embedding_grad(tok, g, V, 2.5)
    for i in np.ndindex(w.shape):  # linear: the difference is exact but for rounding
        d = np.zeros_like(w)
        d[i] = 1.0
        assert abs((R.embedding(d, tok, 2.5) * g).sum() - gw[i]) < 1e-12
    assert (R.embedding_grad(tok, g, V, 2.5, padding=1)[0][1] == 0).all()
