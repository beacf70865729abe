"""Backwards after something went between: a failure, a look at an output.

A backward that fails for memory between taking a gradient and writing it leaves nothing behind: after nc_clear_error the next one
stores where nothing was written, and gives what it gives without the failure."""
import ctypes
from ctypes import c_float, c_int64

import numpy as np
import pytest

from newch_amd import abi
from tests.ncdrive import Engine

pytestmark = pytest.mark.gpu


class SmallArena(Engine):
    """Every device request of 16 KiB and more is an allocation of its own."""

    def __init__(self):
        self.lib = abi.load(abi.LIB_PATH)
        cfg = abi.Config(1 << 16, 1234, 0, 0)
        self.ctx = self.lib.nc_init(ctypes.byref(cfg))
        assert self.ctx


def attention(e, same):
    rng = np.random.default_rng(1)
    x = [e.param(rng.standard_normal(s)) for s in ((1, 512, 2, 64), (1, 64, 2, 64), (1, 64, 2, 64))]
    if same:  # keys as values too: the second gradient goes through scratch
        x[2] = x[1]
    return e.lib.nc_cross_attention(*x, None, c_float(0.125)), x[:2] if same else x


def norm(e, shared):
    rng = np.random.default_rng(2)
    x, wq, wk = e.param(rng.standard_normal((1, 200, 4, 64))), e.param(rng.standard_normal(64)), e.param(rng.standard_normal(64))
    if shared:
        wk = wq
    pos = e.tensor(np.arange(200, dtype=np.int32)[:, None].copy())
    y = e.lib.nc_qk_norm_rope(x, 2, wq, wk, c_float(1e-6), pos, 1, (c_int64 * 1)(64), c_float(1e4), 0)
    return y, [x, wq] if shared else [x, wq, wk]


def rope(e, _):
    x = e.param(np.random.default_rng(3).standard_normal((1, 200, 4, 64)))
    pos = e.tensor(np.arange(200, dtype=np.int32)[:, None].copy())
    return e.lib.nc_rope(x, pos, 1, (c_int64 * 1)(64), c_float(1e4), 0), [x]


def layer_norm(e, _):
    rng = np.random.default_rng(4)
    x, w, b = e.param(rng.standard_normal((512, 256))), e.param(rng.standard_normal(256)), e.param(rng.standard_normal(256))
    return e.lib.nc_layer_norm(x, 1, w, b, c_float(1e-5)), [x, w, b]


@pytest.mark.parametrize("op,how", [(attention, False), (attention, True), (norm, False), (norm, True), (rope, None), (layer_norm, None)],
                         ids=lambda p: getattr(p, "__name__", str(p)))
def test_the_next_backward_stores_what_the_failed_one_did_not(monkeypatch, op, how):
    def begin(fail_at):
        monkeypatch.setenv("NC_FAIL_ALLOC_AT", str(fail_at))
        e = SmallArena()
        y, leaves = op(e, how)
        e.check()
        g = np.random.default_rng(5).standard_normal(e.shape(y)).astype(np.float32)
        loss = e.lib.nc_sum(e.lib.nc_mul(y, e.tensor(g)), abi.ALL_AXES, 0)
        e.check()
        return e, loss, leaves

    def backward(e, loss):
        return e.lib.nc_backward_ex(loss, abi.BACKWARD_RETAIN, None, 0)

    e, loss, leaves = begin(0)
    first = e.lib.nc_device_alloc_count(e.ctx)
    assert backward(e, loss) == 0, e.lib.nc_error(e.ctx)
    last = e.lib.nc_device_alloc_count(e.ctx)
    want = [e.grad(t) for t in leaves]
    e.close()
    failures = 0
    for at in range(first + 1, last + 1):
        print(f"{op.__name__}: request {at} of {first + 1} to {last} fails", flush=True)
        e, loss, leaves = begin(at)
        if backward(e, loss) != 0:
            assert e.lib.nc_status_code(e.ctx) == abi.ERR_OOM
            failures += 1
            e.lib.nc_clear_error(e.ctx)
            assert backward(e, loss) == 0, e.lib.nc_error(e.ctx)
        for t, w in zip(leaves, want):
            assert (e.grad(t).view(np.uint32) == w.view(np.uint32)).all()
        e.close()
    assert failures


@pytest.mark.parametrize("Lk", [40, 300])
@pytest.mark.parametrize("write", [False, True])
def test_an_output_that_the_host_looked_at(write, Lk):
    """nc_data_f32 on attention's output, or on a view of it, between the forward and the backward, to read it or to write: the
    backward is the one of the forward that ran."""
    with Engine(lib=abi.load(abi.LIB_PATH)) as e:
        L, rng = e.lib, np.random.default_rng(6)
        q, k, v = (e.param(rng.standard_normal((2, n, 2, 64))) for n in (50, Lk, Lk))
        g = rng.standard_normal((2, 50, 2, 64)).astype(np.float32)
        grads = []
        for look in (False, True):
            for t in (q, k, v):
                L.nc_zero_grad(t)
            o = L.nc_cross_attention(q, k, v, e.tensor(np.array([Lk, 7], np.int32)), c_float(0.125))
            e.check()
            if look:
                was = e.read(o)
                p = ctypes.cast(L.nc_data_f32(L.nc_slice(o, 1, 0, 50, 1) if Lk == 300 else o), ctypes.POINTER(c_float))
                assert p and p[5] == was.reshape(-1)[5]
                if write:
                    p[5] = 1e9
            e.backward_with(o, g)
            grads.append([e.grad(t) for t in (q, k, v)])
        for a, b in zip(*grads):
            assert (a.view(np.uint32) == b.view(np.uint32)).all()
        e.step_end()
