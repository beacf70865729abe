"""The attention block without a device: refusals through both interfaces, and the 64-bit references against differences."""
import ctypes
from ctypes import c_float, c_int64

import numpy as np
import pytest

from newch_amd import abi, hip
from tests import attention_ref as R
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


def i64(*v):
    return (c_int64 * max(len(v), 1))(*v)


def f32(*shape):
    return np.zeros(shape, np.float32)


def refused(e, t, status, text):
    assert not t
    assert e.lib.nc_status_code(e.ctx) == status, e.lib.nc_error(e.ctx)
    assert text in e.lib.nc_error(e.ctx).decode(), e.lib.nc_error(e.ctx)
    e.lib.nc_clear_error(e.ctx)


def test_rope_refusals(eng):
    L, t = eng.lib, eng.tensor
    x, pos = t(f32(2, 3, 4, 8)), t(np.zeros((3, 2), np.int32))
    call = lambda x=x, pos=pos, n=2, dims=(4, 4), base=1e4: L.nc_rope(x, pos, n, i64(*dims), c_float(base), 0)
    refused(eng, call(), abi.ERR_STATE, "no HIP device")
    refused(eng, call(x=t(f32(2, 3, 8))), abi.ERR_SHAPE, "expected x")
    refused(eng, call(x=t(f32(2, 3, 1, 257))), abi.ERR_SHAPE, "1 to 256 columns")
    refused(eng, call(x=t(np.zeros((2, 3, 4, 8), np.int32))), abi.ERR_DTYPE, "must be f32")
    refused(eng, call(pos=t(f32(3, 2))), abi.ERR_DTYPE, "positions must be i32")
    refused(eng, call(pos=t(np.zeros((2, 2), np.int32))), abi.ERR_SHAPE, "expected positions")
    refused(eng, call(pos=t(np.zeros((3, 3, 2), np.int32))), abi.ERR_SHAPE, "expected positions")
    refused(eng, call(dims=(4, 3)), abi.ERR_SHAPE, "axis 1 has 3 columns")
    refused(eng, call(dims=(0, 4)), abi.ERR_SHAPE, "axis 0 has 0 columns")
    refused(eng, call(dims=(4, 6)), abi.ERR_SHAPE, "4 left in the head")
    refused(eng, call(base=0.0), abi.ERR_ARG, "base")
    refused(eng, call(base=float("nan")), abi.ERR_ARG, "base")
    refused(eng, call(n=0), abi.ERR_ARG, "1 to 4 axes")
    refused(eng, call(n=5, dims=(2,) * 5), abi.ERR_ARG, "1 to 4 axes")
    refused(eng, L.nc_rope(x, pos, 2, None, c_float(1e4), 0), abi.ERR_ARG, "axes")
    assert not L.nc_rope(None, pos, 2, i64(4, 4), c_float(1e4), 0)


def test_qk_norm_rope_refusals(eng):
    L, t = eng.lib, eng.tensor
    x, pos, w = t(f32(2, 3, 4, 8)), t(np.zeros((2, 3, 1), np.int32)), t(f32(8))

    def call(x=x, q_heads=2, wq=w, wk=w, eps=1e-6, pos=pos, dims=(8,)):
        return L.nc_qk_norm_rope(x, q_heads, wq, wk, c_float(eps), pos, len(dims), i64(*dims), c_float(1e4), 0)

    refused(eng, call(), abi.ERR_STATE, "no HIP device")
    refused(eng, call(pos=None, dims=()), abi.ERR_STATE, "no HIP device")
    refused(eng, call(pos=None), abi.ERR_ARG, "axes")
    refused(eng, call(dims=()), abi.ERR_ARG, "axes")
    refused(eng, call(q_heads=5), abi.ERR_ARG, "5 query heads of 4")
    refused(eng, call(q_heads=-1), abi.ERR_ARG, "query heads")
    refused(eng, call(wk=t(f32(7))), abi.ERR_SHAPE, "weights need 8")
    refused(eng, call(wq=t(f32(1, 8))), abi.ERR_SHAPE, "weights need 8")
    refused(eng, call(wq=t(np.zeros(8, np.int32))), abi.ERR_DTYPE, "must be f32")
    refused(eng, call(eps=-1.0), abi.ERR_ARG, "eps")
    refused(eng, call(eps=float("inf")), abi.ERR_ARG, "eps")


def test_cross_attention_refusals(eng):
    L, t = eng.lib, eng.tensor
    q, k = t(f32(2, 3, 4, 8)), t(f32(2, 5, 2, 8))
    call = lambda q=q, k=k, v=k, n=None, scale=0.5: L.nc_cross_attention(q, k, v, n, c_float(scale))
    refused(eng, call(), abi.ERR_STATE, "no HIP device")
    refused(eng, call(q=t(f32(2, 3, 8))), abi.ERR_SHAPE, "expected q")
    refused(eng, call(v=t(f32(2, 6, 2, 8))), abi.ERR_SHAPE, "expected q")
    refused(eng, call(v=t(f32(2, 5, 2, 4))), abi.ERR_SHAPE, "expected q")
    refused(eng, call(k=t(f32(3, 5, 2, 8)), v=t(f32(3, 5, 2, 8))), abi.ERR_SHAPE, "expected q")
    refused(eng, call(k=t(f32(2, 5, 3, 8)), v=t(f32(2, 5, 3, 8))), abi.ERR_SHAPE, "cannot share 3")
    refused(eng, call(k=t(f32(2, 5, 0, 8)), v=t(f32(2, 5, 0, 8))), abi.ERR_SHAPE, "expected q")
    wide = t(f32(1, 1, 1, 257))
    refused(eng, call(q=wide, k=wide, v=wide), abi.ERR_SHAPE, "1 to 256 columns")
    refused(eng, call(q=t(np.zeros((2, 3, 4, 8), np.int32))), abi.ERR_DTYPE, "f32")
    refused(eng, call(n=t(f32(2))), abi.ERR_DTYPE, "key lengths must be i32")
    refused(eng, call(n=t(np.zeros(3, np.int32))), abi.ERR_SHAPE, "key length for each of 2")
    refused(eng, call(scale=float("inf")), abi.ERR_ARG, "scale")
    assert not call(k=None)


def test_kernel_layer_refusals():
    """Bad sizes and missing arguments come back as errors before anything touches a device."""
    K = hip.Kernels(ctypes.CDLL(str(abi.LIB_PATH)))
    p, s = 256, (8, 8, 8)  # an address that is never read

    def no(text, fn, *a, **kw):
        with pytest.raises(hip.HipLayerError, match=text):
            fn(*a, **kw)

    rope = lambda D=8, H=1, dims=(8,), pos=p, base=1e4, x=p, y=p: K.rope_fwd(1, 1, H, D, x, s, pos, 0, dims, base, 0, y)
    no("bad size", rope, D=257)
    no("bad size", rope, D=0, dims=())
    no("bad size", rope, H=-1)
    no("too many", rope, H=1 << 31)
    no("axis 0 has 7", rope, dims=(7,))
    no("axis 1 has 4", rope, dims=(6, 4))
    no("position axes", rope, dims=(2,) * 5, D=16)
    no("position axes", rope, pos=None)
    no("base", rope, base=-1.0)
    no("an axis and", rope, dims=())
    no("an axis and", rope, x=None)
    no("an axis and", rope, y=None)
    no("an axis and", K.rope_bwd, 1, 1, 1, 8, None, p, 0, (8,), 1e4, 0, p)
    rope(H=0, x=None, y=None)  # nothing to do is no error
    no("query heads", K.qk_norm_rope_fwd, 1, 1, 2, 8, 3, p, s, p, p, 0.0, p, 0, (8,), 1e4, 0, p)
    no("eps", K.qk_norm_rope_fwd, 1, 1, 2, 8, 1, p, s, p, p, -1.0, p, 0, (8,), 1e4, 0, p)
    no("workspace", K.qk_norm_rope_bwd, 1, 1, 2, 8, 1, p, s, p, p, 0.0, p, 0, (8,), 1e4, 0, p, p, p, p)
    no("are needed", K.qk_norm_rope_bwd, 1, 1, 2, 8, 1, None, s, p, p, 0.0, p, 0, (8,), 1e4, 0, p, p, None, None)
    attn = lambda Lq=1, Lk=1, Hq=2, Hkv=1, D=8, scale=1.0, q=p, k=p: K.cross_attention_fwd(
        1, Lq, Lk, Hq, Hkv, D, scale, q, s, k, s, p, s, None, p, None)
    no("bad size", attn, D=257)
    no("bad size", attn, Hkv=0)
    no("bad size", attn, Lk=-1)
    no("cannot share", attn, Hq=3, Hkv=2)
    no("past 2\\^31", attn, Lk=1 << 31)
    no("scale", attn, scale=float("nan"))
    no("are needed", attn, q=None)
    no("are needed", attn, k=None)
    no("are needed", K.cross_attention_bwd, 1, 1, 1, 2, 1, 8, 1.0, p, s, p, s, p, s, None, p, None, p, p, p, p)
    attn(Lq=0, q=None)
    # a workspace that is too small, or not at a multiple of 16 bytes
    sizes = (1, 40, 600, 2, 2, 64)
    for name, need, args in (("fwd", K.cross_attention_fwd_workspace(*sizes), (None, p, None)),
                             ("bwd", K.cross_attention_bwd_workspace(*sizes), (None, p, p, p, p, p, p))):
        assert need > 0
        call = getattr(K, "cross_attention_" + name)
        for ws, n in ((p, need - 1), (p + 8, need), (None, need)):
            no("workspace of .* 16-byte", call, *sizes, 1.0, p, s, p, s, p, s, *args, ws, n)
    need = K.qk_norm_rope_bwd_workspace(1, 1, 2, 8)
    no("workspace of .* 16-byte", K.qk_norm_rope_bwd, 1, 1, 2, 8, 1, p, s, p, p, 0.0, p, 0, (8,), 1e4, 0, p, p, p, p, p + 8, need)


# ---- the references themselves -----------------------------------------------------------------------------------
def differences(f, x, g, h=1e-6):
    """sum(g * f(x)) by central differences over x"""
    out = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i] += h
        down[i] -= h
        out[i] = ((f(up) - f(down)) * g).sum() / (2 * h)
    return out


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_reference_against_differences(interleaved):
    rng = np.random.default_rng(3)
    x, g = rng.standard_normal((2, 2, 3, 7)), rng.standard_normal((2, 2, 3, 7))
    wq, wk, pos = rng.standard_normal(7), rng.standard_normal(7), rng.integers(-9, 9, (2, 2, 2))
    args = (1e-3, pos, (4, 2), 100.0, interleaved)
    want = R.qk_norm_rope_bwd64(x, 2, wq, wk, *args, g)
    y = lambda x=x, wq=wq, wk=wk: R.qk_norm_rope64(x, 2, wq, wk, *args)[0]
    for name, x0, f in (("gx", x, lambda t: y(x=t)), ("gwq", wq, lambda t: y(wq=t)), ("gwk", wk, lambda t: y(wk=t))):
        assert np.abs(differences(f, x0, g) - want[name][0]).max() < 1e-7, name  # h^2 and 2^-52 / h, both about 1e-10


def test_attention_reference_against_differences():
    rng = np.random.default_rng(4)
    q, k, v = rng.standard_normal((3, 3, 4, 3)), rng.standard_normal((3, 5, 2, 3)), rng.standard_normal((3, 5, 2, 3))
    g, lens = rng.standard_normal(q.shape), [5, 0, 2]
    want = R.attention64(q, k, v, lens, 0.7, g)
    o = lambda q=q, k=k, v=v: R.attention64(q, k, v, lens, 0.7)["o"][0]
    for name, x0, f in (("gq", q, lambda t: o(q=t)), ("gk", k, lambda t: o(k=t)), ("gv", v, lambda t: o(v=t))):
        assert np.abs(differences(f, x0, g) - want[name][0]).max() < 1e-7, name
