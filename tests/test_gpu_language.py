"""A language model's two ends on the GPU against the 64-bit references: embedding rows and their gradient, dropout from a counter,
the cross entropy of a product; through the kernel layer on device buffers (odd sizes, strides, alignments, labels and tokens that do
not count, places that hold NaN) and through the engine with autograd, alone and together."""
import ctypes
from ctypes import c_double, c_float, c_int32, c_uint64

import numpy as np
import pytest

from newch_amd import abi, hip
from newch_amd.hipmem import DeviceBuffer, Stream, check, runtime, synchronize
from tests import language_ref as R
from tests.ncdrive import Engine, NcError

pytestmark = pytest.mark.gpu
HALF = R.HALF


@pytest.fixture(scope="module")
def lib():
    L = abi.load(abi.LIB_PATH)
    assert L.nc_device_count() > 0, "no HIP device visible: the GPU tests need an MI355X"
    return L


@pytest.fixture(scope="module")
def K(lib):
    return hip.Kernels(lib)


@pytest.fixture()
def eng(lib):
    e = Engine(lib=lib)
    yield e
    e.close()


GUARD = 64  # floats of NaN on either side of every output


class Out:
    """An output of `shape` between guards: `shift` floats off alignment, filled with `fill`."""

    def __init__(self, shape, fill=np.nan, shift=0):
        self.shape, self.n, self.at = shape, int(np.prod(shape)), GUARD + shift
        self.host = np.full(self.n + 2 * GUARD + shift, np.nan, np.float32)
        self.host[self.at: self.at + self.n] = np.asarray(fill, np.float32).reshape(-1) if np.ndim(fill) else fill
        self.buf = DeviceBuffer.from_numpy(self.host)
        self.ptr = self.buf.ptr + 4 * self.at

    def get(self):
        got = self.buf.to_numpy(np.float32, self.host.shape)
        assert np.isnan(got[: self.at]).all() and np.isnan(got[self.at + self.n:]).all(), "written out of bounds"
        return got[self.at: self.at + self.n].reshape(self.shape)


class Matrix:
    """A float matrix on the device, rows `gap` floats apart and `shift` floats off alignment, NaN between."""

    def __init__(self, a, gap=0, shift=0):
        a = np.asarray(a, np.float32)
        host = np.full((a.shape[0], a.shape[1] + gap), np.nan, np.float32)
        host[:, : a.shape[1]] = a
        self.buf = DeviceBuffer.from_numpy(np.concatenate([np.full(shift, np.nan, np.float32), host.reshape(-1)]))
        self.ptr, self.ld = self.buf.ptr + 4 * shift, a.shape[1] + gap


def up(a, shift=0):
    """(address, its buffer) of an array `shift` elements off alignment"""
    a = np.asarray(a)
    buf = DeviceBuffer.from_numpy(np.concatenate([np.zeros(shift, a.dtype), a.reshape(-1)]))
    return buf.ptr + shift * a.itemsize, buf


def rms(a):
    return float(np.sqrt(np.mean(np.square(np.asarray(a, np.float64))))) if np.size(a) else 0.0


# ---- embedding -----------------------------------------------------------------------------------------------------
# N, V, D, how the tokens fall
EMBED = [(1, 1, 1, "even"), (1, 5, 4, "even"), (2, 3, 2, "even"), (7, 5, 3, "even"), (33, 7, 64, "even"), (31, 1000, 250, "even"),
         (64, 64, 1024, "one"), (65, 50, 1025, "even"), (1000, 1, 8, "even"), (1023, 333, 100, "rank"), (1024, 10007, 16, "rank"),
         (1500, 40, 260, "one"), (4097, 2000, 33, "rank"), (5000, 70000, 12, "rank"), (3, 100, 5001, "even"), (257, 31, 4, "outside"),
         (20001, 3000, 20, "rank"), (40000, 7, 9, "even"), (70000, 100003, 5, "rank"),
         (8192, 31, 3, "rank"), (8193, 1023, 4, "rank"), (8200, 1024, 6, "even"), (9000, 1 << 20, 1, "even"), (10000, 50, 7, "outside"),
         (300000, 5000, 3, "rank"), (1024, 1000, 40, "rank"), (1024, 3, 1030, "one"), (1023, 700, 5, "outside"), (1025, 100, 33, "one"), (300, 9, 2000, "even"), (6, 9001, 1001, "even"), (3, 1501, 2889, "outside"), (9000, 70000, 37, "rank"), (2560, 1009, 131, "rank"), (2560, 20, 409, "outside"), (2561, 300, 64, "even"), (2561, 300, 410, "one"), (263000, 2, 2, "one"), (33000, 1500, 300, "rank")]


def some_tokens(rng, N, V, how):
    if how == "one":
        t = np.full(N, V // 2)
        t[rng.random(N) < 0.1] = 0
    elif how == "rank":
        t = np.minimum(np.exp(rng.random(N) * np.log(V + 1.0)) - 1, V - 1).astype(int)
    elif how == "outside":
        t = rng.integers(-3, V + 3, N)
        t[:2] = (-2 ** 31, 2 ** 31 - 1)
    else:
        t = rng.integers(0, V, N)
    return t.astype(np.int32)


@pytest.mark.parametrize("shape", EMBED, ids=str)
def test_embedding_rows(K, shape):
    N, V, D, how = shape
    rng = np.random.default_rng(N * 7 + V)
    w, tokens = rng.standard_normal((V, D)).astype(np.float32), some_tokens(rng, N, V, how)
    tok, _t = up(tokens)
    bad = DeviceBuffer.from_numpy(np.zeros(1, np.uint64))
    outside = np.flatnonzero((tokens < 0) | (tokens >= V))
    want = ~np.uint64(0) if not outside.size else (np.uint64(outside[0]) << np.uint64(32)) | np.uint64(np.uint32(tokens[outside[0]]))
    for gap, shift in ((0, 0), (3, 1), (4, 0)):
        m, y = Matrix(w, gap, shift), Out((N, D), shift=shift)
        K.embedding_fwd(N, V, D, m.ptr, m.ld, tok, 1.7, y.ptr, bad=bad.ptr)
        synchronize()
        ok = (tokens >= 0) & (tokens < V)
        exp = np.where(ok[:, None], w[np.where(ok, tokens, 0)] * np.float32(1.7), 0)
        assert (y.get() == exp).all()
        assert bad.to_numpy(np.uint64, 1)[0] == want


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("shape", EMBED, ids=str)
def test_embedding_gradient(K, shape, accumulate):
    N, V, D, how = shape
    rng = np.random.default_rng(N * 5 + V)
    tokens, g = some_tokens(rng, N, V, how), rng.standard_normal((N, D)).astype(np.float32)
    n = K.embedding_bwd_workspace(N, V, D)
    ws = DeviceBuffer.from_numpy(np.full(n, 0xCD, np.uint8))
    scale = np.float32(-0.3)
    old = rng.standard_normal((V, D)).astype(np.float32) if accumulate else np.zeros((V, D), np.float32)
    runs = []
    for padding, shift in ((-1, 0), (int(tokens[0]), 1), (-1, 0)):
        dead = (tokens < 0) | (tokens >= V) | ((tokens == padding) if padding >= 0 else False)
        gg = np.where(dead[:, None], np.nan, g)  # not read there
        gp, _g = up(gg.astype(np.float32), shift)
        tok, _t = up(tokens, shift)
        gw = Out((V, D), fill=old if accumulate else np.nan, shift=shift)
        K.embedding_bwd(N, V, D, tok, padding, float(scale), gp, gw.ptr, ws.ptr, n, accumulate=accumulate)
        synchronize()
        got = gw.get()
        ref, size = R.embedding_grad(tokens, g, V, np.float64(scale), padding)
        assert (np.abs(got - (ref + old)) <= R.embedding_grad_tol(size, old)).all()
        untouched = size.sum(1) == 0
        assert (got[untouched] == old[untouched]).all()
        runs.append(got)
    assert (runs[0] == runs[2]).all(), "the same call twice"


@pytest.mark.parametrize("D", [1, 2, 3, 5, 66, 1023])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("N", [0, 3, 3001])
def test_embedding_gradient_clears(K, N, shift, D):
    """Rows of all tokens that do not occur, however the table lies and however few they are."""
    for V in (1, 2, 37, 40000 // D + 1, 200000 // D + 3):
        rng = np.random.default_rng(V)
        tokens = (rng.integers(0, V, N) // 7 * 7).astype(np.int32)
        gp, _g = up(np.ones((max(N, 1), D), np.float32))
        tok, _t = up(tokens if N else np.zeros(1, np.int32))
        n = K.embedding_bwd_workspace(N, V, D)
        ws = DeviceBuffer.from_numpy(np.zeros(max(n, 16), np.uint8))
        gw = Out((V, D), shift=shift)
        K.embedding_bwd(N, V, D, tok, -1, 1.0, gp, gw.ptr, ws.ptr, n, accumulate=False)
        synchronize()
        count = np.bincount(tokens, minlength=V).astype(np.float32)
        assert (gw.get() == count[:, None]).all()


def test_embedding_of_nothing(K):
    gw = Out((5, 3))
    K.embedding_fwd(0, 5, 3, None, 3, None, 1.0, None)
    K.embedding_bwd(0, 5, 3, None, -1, 1.0, None, gw.ptr, accumulate=True)
    synchronize()
    assert np.isnan(gw.get()).all()
    K.embedding_bwd(0, 5, 3, None, -1, 1.0, None, gw.ptr, accumulate=False)
    synchronize()
    assert (gw.get() == 0).all()


def test_embedding_past_2_31_floats(K):
    """Rows of the table, tokens' rows and gradients more than 2^31 floats from the first."""
    V, D, N = 70001, 32768, 40
    rng = np.random.default_rng(5)
    tokens = np.concatenate([np.array([V - 1, 0, V - 1, 65537]), rng.integers(V - 300, V, N - 4)]).astype(np.int32)
    g = rng.standard_normal((N, D)).astype(np.float32)
    tok, _t = up(tokens)
    gp, _g = up(g)
    gw, y = DeviceBuffer.empty(4 * V * D), Out((N, D))
    ws = DeviceBuffer.empty(K.embedding_bwd_workspace(N, V, D))
    K.embedding_bwd(N, V, D, tok, -1, 1.0, gp, gw.ptr, ws.ptr, ws.nbytes, accumulate=False)
    K.embedding_fwd(N, V, D, gw.ptr, D, tok, 2.0, y.ptr)
    synchronize()
    ref, size = R.embedding_grad(tokens - (V - 300), g, 300, 1.0)
    tol = R.embedding_grad_tol(size)
    got = gw.to_numpy(np.float32, (300, D), offset=4 * (V - 300) * D)
    assert (np.abs(got - ref) <= tol).all()
    for v, i in ((0, 1), (65537, 3)):
        assert (gw.to_numpy(np.float32, D, offset=4 * v * D) == g[i]).all()
    assert (gw.to_numpy(np.float32, 5 * D, offset=4 * 40000 * D) == 0).all()
    mine = tokens >= V - 300
    assert (y.get()[mine] == got[tokens[mine] - (V - 300)] * np.float32(2)).all()


# ---- dropout ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 63, 255, 257, 1023, 4096, 100003])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999, 1.0])
def test_dropout(K, n, p):
    rng = np.random.default_rng(n)
    x, r, old = (rng.standard_normal(n).astype(np.float32) for _ in range(3))
    dropped = ~R.kept(n, p, 0xFEDCBA9876543210, 2 ** 63 + 5)
    x[dropped & (rng.random(n) < 0.2)] = np.nan  # a value that is dropped counts as 0, whatever it holds
    x[dropped & (rng.random(n) < 0.2)] = np.inf
    for shift in (0, 1, 3):
        xp, _x = up(x, shift)
        rp, _r = up(r, shift)
        y, z, gx, ga = Out((n,), shift=shift), Out((n,)), Out((n,), shift=shift), Out((n,), fill=old)
        key = (0xFEDCBA9876543210, 2 ** 63 + 5)
        K.dropout_fwd(n, p, *key, xp, None, y.ptr)
        K.dropout_fwd(n, p, *key, xp, rp, z.ptr)
        K.dropout_bwd(n, p, *key, xp, gx.ptr, accumulate=False)
        K.dropout_bwd(n, p, *key, xp, ga.ptr, accumulate=True)
        K.dropout_fwd(n, p, *key, xp, None, xp)  # in place
        synchronize()
        want = R.dropout(x, p, *key)
        assert (y.get() == want).all() and (gx.get() == want).all()
        assert (_x.to_numpy(np.float32, n + shift)[shift:] == want).all()
        for got, base in ((z.get(), r), (ga.get(), old)):
            exp = R.dropout(x, p, *key, residual=base)
            # the reference rounds in 64 bits before it does in 32: next to a tie they may part by one step of 2 HALF
            assert (np.abs(got.astype(np.float64) - exp) <= 2 * HALF * np.abs(exp)).all() and (got != exp).mean() < 1e-3


def test_dropout_offset_on_the_device(K):
    n, x = 1000, np.ones(1000, np.float32)
    xp, _x = up(x)
    y, z = Out((n,)), Out((n,))
    at = DeviceBuffer.from_numpy(np.array([41], np.uint64))
    K.dropout_fwd(n, 0.5, 9, 2 ** 64 - 40, xp, None, y.ptr, offset_ptr=at.ptr)  # the sum wraps to 1
    K.dropout_bwd(n, 0.5, 9, 1, xp, z.ptr, accumulate=False)
    synchronize()
    assert (y.get() == z.get()).all() and (y.get() == R.dropout(x, 0.5, 9, 1)).all()


def test_dropout_past_2_34_bytes(K):
    """Values whose generator blocks, byte offsets and places pass 32 bits, against the generator at their places."""
    n = (1 << 32) + 5
    x, gx = DeviceBuffer.empty(4 * n), DeviceBuffer.empty(4 * n)
    K.fill(x.ptr, 4, int(np.float32(1.0).view(np.uint32)), n)
    K.dropout_bwd(n, 0.25, 77, 3, x.ptr, gx.ptr, accumulate=False)
    synchronize()
    for first in (0, (1 << 30) - 8, (1 << 31) - 8, (1 << 32) - 8):
        m = min(64, n - first)
        got = gx.to_numpy(np.float32, m, offset=4 * first)
        assert ((got != 0) == R.kept(m, 0.25, 77, 3, first=first)).all()


# ---- the cross entropy of a product ------------------------------------------------------------------------------------
@pytest.fixture(params=["fp32", "split"])
def form(request, monkeypatch):
    """either form of the kernels, whatever the sizes"""
    monkeypatch.setenv("NC_HIP_VOCAB_FORM", request.param)
    return request.param


# N, D, V
LOSS = [(1, 1, 1), (1, 7, 3), (40, 31, 9001), (3, 1030, 4097), (260, 33, 300), (2, 4, 1), (5, 33, 17), (64, 64, 64), (65, 130, 257), (300, 96, 1000), (257, 256, 513), (1000, 40, 50),
        (130, 512, 2050), (513, 100, 5003), (1030, 260, 1027),
        (1, 128, 20000), (5, 512, 4099), (31, 1028, 2050), (32, 260, 8191), (33, 132, 16000), (64, 1164, 2050)]


def loss_inputs(N, D, V, seed, bias, ignored, confident=True):
    rng = np.random.default_rng(seed)
    w = (rng.standard_normal((V, D)) * 2 / np.sqrt(D)).astype(np.float32)
    labels = rng.integers(0, V, N).astype(np.int32)
    x = rng.standard_normal((N, D)).astype(np.float32)
    if confident:
        x += w[labels] * (4 * rng.random((N, 1)) ** 2).astype(np.float32)
    labels[rng.random(N) < ignored] = -100
    return x, w, rng.standard_normal(V).astype(np.float32) * 0.5 if bias else None, labels


class Loss:
    """One call's buffers; `run` enqueues it."""

    def __init__(self, K, x, w, bias, labels, grads="xwb", gap=0, shift=0, sum=False, gout=None, old=None, ignore=-100):
        self.K, (self.N, self.D), self.V = K, x.shape, len(w)
        self.x, self.w = Matrix(x, gap, shift), Matrix(w, gap, shift)
        self.bias, self._b = up(bias, shift) if bias is not None else (None, None)
        self.labels, self._l = up(labels, shift)
        self.loss, self.rows = Out((1,)), Out((self.N,))
        fill = lambda k: np.nan if old is None else old[k]
        self.g = {k: Out(s, fill=fill(k), shift=shift) for k, s in (("gx", x.shape), ("gw", w.shape), ("gb", (self.V,))) if k[1] in grads}
        self.gout, self._o = up(np.array([gout], np.float32)) if gout is not None else (None, None)
        n = K.linear_cross_entropy_workspace(self.N, self.D, self.V, **{k: True for k in self.g})
        self.ws = DeviceBuffer.from_numpy(np.full(n, 0xCD, np.uint8))
        self.bad = DeviceBuffer.from_numpy(np.zeros(1, np.uint64))
        self.opt = dict(sum=sum, accumulate=old is not None, ignore=ignore)

    def run(self, stream=None):
        self.K.linear_cross_entropy(self.N, self.D, self.V, self.x.ptr, self.x.ld, self.w.ptr, self.w.ld, self.bias, self.labels,
                                    self.loss.ptr, self.ws.ptr, self.ws.nbytes, gout=self.gout, rows=self.rows.ptr, bad=self.bad.ptr,
                                    stream=stream, **{k: o.ptr for k, o in self.g.items()}, **self.opt)

    def get(self):
        synchronize()
        return dict({k: o.get() for k, o in self.g.items()}, loss=self.loss.get()[0], rows=self.rows.get())


def agree(got, ref, x, w, old=None, scale=1.0):
    tol = R.vocab_loss_tol(x, w, ref)
    for k in got:
        want = ref[k] + (old[k] if old is not None and k in old else 0.0)
        err = rms(got[k].astype(np.float64) - want)
        extra = 2 * HALF * rms(want)
        assert err <= tol[k] + extra + 1e-37, f"{k}: {err:.3g} off, {tol[k] + extra:.3g} allowed, {rms(want):.3g} large"


@pytest.mark.parametrize("bias,ignored", [(False, 0.0), (True, 0.3)])
@pytest.mark.parametrize("shape", LOSS, ids=str)
def test_loss_and_gradients(K, form, shape, bias, ignored):
    x, w, b, labels = loss_inputs(*shape, 11, bias, ignored)
    ref = R.vocab_loss(x, w, b, labels)
    x = np.where(ref["on"][:, None], x, np.nan)  # rows that do not count may hold anything
    for gap, shift in ((0, 0), (3, 1)):
        c = Loss(K, x, w, b, labels, gap=gap, shift=shift)
        c.run()
        got = c.get()
        if not ref["on"].any():
            assert np.isnan(got.pop("loss"))
        agree(got, ref, x, w)
        assert (got["rows"][~ref["on"]] == 0).all() and (got["gx"][~ref["on"]] == 0).all()
        assert c.bad.to_numpy(np.uint64, 1)[0] == ~np.uint64(0)
        c.run()
        again = c.get()
        assert all((again[k].view(np.uint32) == got[k].view(np.uint32)).all() for k in c.g), "the same call twice"


@pytest.mark.parametrize("shape", [(5, 33, 17), (300, 96, 1000), (513, 100, 5003), (257, 256, 513), (7, 512, 4099), (40, 516, 4099)], ids=str)
def test_loss_added_gradients_sum_and_its_own_gradient(K, form, shape):
    x, w, b, labels = loss_inputs(*shape, 12, True, 0.2)
    labels[0] = shape[2] - 1
    rng = np.random.default_rng(1)
    for total, gout in ((True, None), (False, -2.5), (True, 3.0)):
        ref = R.vocab_loss(x, w, b, labels, sum=total, gout=1.0 if gout is None else gout)
        s = max(rms(ref["gw"]), 1e-12)
        old = {k: (rng.standard_normal(ref[k].shape) * s).astype(np.float32) for k in ("gx", "gw", "gb")}
        c = Loss(K, x, w, b, labels, sum=total, gout=gout, old=old)
        c.run()
        agree(c.get(), ref, x, w, old=old)


@pytest.mark.parametrize("shape", [(5, 33, 17), (300, 96, 1000), (1030, 260, 1027), (7, 512, 4099), (40, 516, 4099)], ids=str)
@pytest.mark.parametrize("grads", ["", "x", "w", "b", "xw"])
def test_loss_some_gradients(K, form, shape, grads):
    x, w, b, labels = loss_inputs(*shape, 13, False, 0.1)
    ref = R.vocab_loss(x, w, None, labels)
    c = Loss(K, x, w, None, labels, grads=grads)
    c.run()
    got = c.get()
    assert set(got) == {"loss", "rows"} | {"g" + k for k in grads}
    agree(got, ref, x, w)


@pytest.mark.parametrize("shape", [(5, 33, 17), (300, 96, 1000), (600, 128, 2048), (7, 512, 4099), (40, 516, 4099)], ids=str)
def test_loss_labels_outside(K, form, shape):
    N, D, V = shape
    x, w, b, labels = loss_inputs(*shape, 14, True, 0.2)
    labels[3], labels[1] = V, -7
    x[1] = x[3] = np.nan
    c = Loss(K, x, w, b, labels)
    c.run()
    ref = R.vocab_loss(x, w, b, labels)
    agree(c.get(), ref, x, w)
    assert c.bad.to_numpy(np.uint64, 1)[0] == (np.uint64(1) << np.uint64(32)) | np.uint64(np.uint32(-7 % 2 ** 32))


@pytest.mark.parametrize("shape", [(3, 5, 9), (300, 96, 1000), (600, 128, 2048), (7, 512, 4099), (40, 516, 4099)], ids=str)
def test_loss_no_row_counts(K, form, shape):
    x, w, b, labels = loss_inputs(*shape, 15, True, 0.0)
    labels[:] = 5  # the ignored label may be a word
    c = Loss(K, x * np.nan, w, b, labels, ignore=5)
    c.run()
    got = c.get()
    assert np.isnan(got["loss"]) and all((got[k] == 0).all() for k in ("gx", "gw", "gb", "rows"))
    c = Loss(K, x * np.nan, w, b, labels, ignore=5, sum=True)
    c.run()
    assert c.get()["loss"] == 0


def test_loss_of_no_rows(K, form):
    x, w, b, labels = loss_inputs(0, 6, 9, 16, True, 0.0)
    c = Loss(K, x, w, b, labels)
    c.run()
    got = c.get()
    assert np.isnan(got["loss"]) and (got["gw"] == 0).all() and (got["gb"] == 0).all()


@pytest.mark.parametrize("shape", [(40, 33, 170), (300, 96, 1000), (600, 128, 2048), (7, 512, 4099), (40, 516, 4099)], ids=str)
def test_loss_masked_words(K, form, shape):
    """A bias of -inf, or of the type's lowest value, takes words out: no probability, no gradient."""
    N, D, V = shape
    x, w, b, labels = loss_inputs(*shape, 17, True, 0.1)
    out = np.arange(V) % 3 == 1
    labels[(labels >= 0) & (labels % 3 == 1)] -= 1
    for value in (-np.inf, np.finfo(np.float32).min):
        b[out] = value
        c = Loss(K, x, w, b, labels)
        c.run()
        got, ref = c.get(), R.vocab_loss(x, w, b, labels)
        z = ref["z"]
        ref["z"] = np.where(out, 0, z)
        agree(got, ref, x, w)
        assert (got["gw"][out] == 0).all() and (got["gb"][out] == 0).all()


@pytest.mark.parametrize("shape", [(40, 33, 170), (300, 96, 1000), (600, 128, 2048), (7, 512, 4099), (40, 516, 4099)], ids=str)
def test_loss_rows_and_words_of_unlike_sizes(K, form, shape):
    """Rows of x and of w whose sizes lie many powers of two apart: each result keeps the precision of what it sums."""
    N, D, V = shape
    x, w, b, labels = loss_inputs(*shape, 18, False, 0.0, confident=False)
    rng = np.random.default_rng(2)
    x *= np.exp2(rng.integers(-12, 2, (N, 1))).astype(np.float32)
    w *= np.exp2(rng.integers(-12, 2, (V, 1))).astype(np.float32)
    c = Loss(K, x, w, None, labels)
    c.run()
    got, ref = c.get(), R.vocab_loss(x, w, None, labels)
    agree(got, ref, x, w)


@pytest.mark.parametrize("shape", [(300, 96, 1000), (600, 128, 2048)], ids=str)
def test_loss_certain_rows(K, form, shape):
    """Rows that are all but certain of their word keep the bits of what little gradient they have."""
    N, D, V = shape
    x, w, b, labels = loss_inputs(*shape, 19, False, 0.0)
    t = np.linspace(2, 12, N, dtype=np.float32)[:, None]
    x = (0.3 * x + t * w[labels] / (w[labels] ** 2).sum(-1, keepdims=True) * 3).astype(np.float32)
    c = Loss(K, x, w, None, labels)
    c.run()
    got, ref = c.get(), R.vocab_loss(x, w, None, labels)
    agree(got, ref, x, w)
    # each row by itself: z is off by rel(D) of its terms, the gradient of a row by as much of itself (and the sum over words)
    size = np.sqrt(((x.astype(np.float64) ** 2) @ (w.astype(np.float64) ** 2).T).max(-1))
    dz = 4 * (HALF * (7 + np.sqrt(D)) * size + 3 * HALF * np.abs(ref["z"]).max(-1))
    err = np.sqrt(((got["gx"] - ref["gx"]) ** 2).sum(-1))
    spread = np.abs(ref["G"]) @ np.sqrt((w.astype(np.float64) ** 2).sum(-1))
    assert (err <= (2 * dz + HALF * (20 + np.sqrt(V))) * spread).all()


@pytest.mark.parametrize("shape", [(40, 33, 170), (300, 96, 1000), (600, 128, 2048), (9, 512, 4099), (40, 516, 4099)], ids=str)
def test_loss_values_that_are_not_finite(K, form, shape):
    """NaN in a row that counts makes that row's loss and gradient NaN and leaves the other rows' theirs."""
    N, D, V = shape
    x, w, b, labels = loss_inputs(*shape, 20, True, 0.0)
    ref = R.vocab_loss(x, w, b, labels)
    x[7, 3] = np.nan
    c = Loss(K, x, w, b, labels)
    c.run()
    got = c.get()
    assert np.isnan(got["loss"]) and np.isnan(got["rows"][7]) and np.isnan(got["gx"][7]).all()
    others = np.arange(N) != 7
    assert np.isfinite(got["rows"][others]).all() and np.isfinite(got["gx"][others]).all()
    tol = R.vocab_loss_tol(np.where(np.isnan(x), 0, x), w, ref)
    assert rms(got["gx"][others] - ref["gx"][others]) <= 1.1 * tol["gx"]


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("shape", [(700, 40, 600), (1030, 260, 1027), (9, 5, 5000), (40, 516, 4099)], ids=str)
def test_loss_in_pieces(K, form, shape, rows, monkeypatch):
    """Rows taken a few at a time, gradients added from piece to piece; rows that do not count leave the last pieces empty."""
    monkeypatch.setenv("NC_HIP_VOCAB_ROWS", str(rows))
    x, w, b, labels = loss_inputs(*shape, 23, True, 0.6)
    labels[0] = 1
    ref = R.vocab_loss(x, w, b, labels)
    old = {k: ref[k].astype(np.float32)[::-1].copy() for k in ("gx", "gw", "gb")}
    for o in (None, old):
        c = Loss(K, x, w, b, labels, old=o)
        c.run()
        agree(c.get(), ref, x, w, old=o)


@pytest.mark.parametrize("shape,grads", [((2100, 100, 5003), ""), ((4200, 100, 5003), "xwb"), ((1300, 520, 3001), "xwb")], ids=str)
def test_loss_of_the_chosen_form(K, shape, grads):
    """Sizes that run on pieces by the kernels' own choice."""
    x, w, b, labels = loss_inputs(*shape, 24, True, 0.1)
    ref = R.vocab_loss(x, w, b, labels)
    c = Loss(K, x, w, b, labels, grads=grads)
    c.run()
    agree(c.get(), ref, x, w)


# ---- together ----------------------------------------------------------------------------------------------------------
class Ends:
    """Tokens looked up, dropped out over a residual, and their loss against the table itself: its gradient comes from both ends."""

    def __init__(self, K, N, V, D, seed):
        rng = np.random.default_rng(seed)
        self.K, self.N, self.V, self.D = K, N, V, D
        self.host = {"w": (rng.standard_normal((V, D)) / np.sqrt(D)).astype(np.float32), "tokens": rng.integers(0, V, N).astype(np.int32),
                     "labels": np.where(rng.random(N) < 0.2, -100, rng.integers(0, V, N)).astype(np.int32),
                     "r": rng.standard_normal((N, D)).astype(np.float32), "at": np.array([seed], np.uint64)}
        self.dev = {k: DeviceBuffer.from_numpy(v) for k, v in self.host.items()}
        f = lambda *s: DeviceBuffer.from_numpy(np.full(s, np.nan, np.float32))
        self.res = {"e": f(N, D), "y": f(N, D), "loss": f(1), "gy": f(N, D), "ge": f(N, D), "gw": f(V, D)}
        self.n1, self.n2 = K.embedding_bwd_workspace(N, V, D), K.linear_cross_entropy_workspace(N, D, V, gx=True, gw=True)
        self.ws = DeviceBuffer.empty(max(self.n1, self.n2))

    def run(self, stream=None):
        K, N, V, D, d, r = self.K, self.N, self.V, self.D, self.dev, self.res
        n = N * D
        K.embedding_fwd(N, V, D, d["w"].ptr, D, d["tokens"].ptr, 2.0, r["e"].ptr, stream=stream)
        K.dropout_fwd(n, 0.3, 5, 100, r["e"].ptr, d["r"].ptr, r["y"].ptr, offset_ptr=d["at"].ptr, stream=stream)
        K.linear_cross_entropy(N, D, V, r["y"].ptr, D, d["w"].ptr, D, None, d["labels"].ptr, r["loss"].ptr, self.ws.ptr, self.n2,
                               gx=r["gy"].ptr, gw=r["gw"].ptr, accumulate=False, stream=stream)
        K.dropout_bwd(n, 0.3, 5, 100, r["gy"].ptr, r["ge"].ptr, offset_ptr=d["at"].ptr, accumulate=False, stream=stream)
        K.embedding_bwd(N, V, D, d["tokens"].ptr, -1, 2.0, r["ge"].ptr, r["gw"].ptr, self.ws.ptr, self.n1, accumulate=True, stream=stream)

    def results(self):
        got = {k: b.to_numpy(np.float32, b.nbytes // 4) for k, b in self.res.items()}
        assert all(np.isfinite(v).all() for v in got.values())
        return got

    def expected(self):
        h = self.host
        y = h["r"].astype(np.float64) + R.dropout(h["w"][h["tokens"]] * np.float32(2), 0.3, 5, 100 + int(h["at"][0]))
        y = y.astype(np.float32)
        ref = R.vocab_loss(y, h["w"], None, h["labels"])
        keep = R.kept(y.size, 0.3, 5, 100 + int(h["at"][0])).reshape(y.shape)
        gw, _ = R.embedding_grad(h["tokens"], ref["gx"] * keep / 0.7, self.V, 2.0)
        return y, ref, ref["gw"] + gw


ENDS = [(37, 50, 24), (300, 1000, 96), (700, 2048, 128)]


@pytest.mark.parametrize("shape", ENDS, ids=str)
def test_ends_together(K, form, shape):
    a = Ends(K, *shape, 3)
    a.run()
    synchronize()
    got, (y, ref, gw) = a.results(), a.expected()
    tol = R.vocab_loss_tol(y, a.host["w"], ref)
    assert abs(got["loss"][0] - ref["loss"]) <= tol["loss"] + 2 * HALF * abs(ref["loss"])
    # what reaches the table through the lookup is gx's error twice over (scale 2 / 0.7), summed over a token's few positions
    most = np.bincount(a.host["tokens"]).max()
    assert rms(got["gw"].reshape(gw.shape) - gw) <= tol["gw"] + 3 * most * tol["gx"] + 4 * HALF * rms(gw)


@pytest.mark.parametrize("shape", ENDS, ids=str)
def test_ends_captured_and_replayed(K, form, shape):
    """The run as a graph: every replay, with other inputs, another offset and eager calls in between, gives the eager run's bits."""
    rt = runtime()
    a, other = Ends(K, *shape, 29), Ends(K, *shape, 30)
    a.run()
    other.run()
    synchronize()
    want, new = a.results(), other.results()
    s, graph, run = Stream(), ctypes.c_void_p(), ctypes.c_void_p()
    check(rt.hipStreamBeginCapture(ctypes.c_void_p(s.handle), ctypes.c_int(2)), "begin")  # relaxed: other streams as they are
    try:
        a.run(s.handle)
    finally:
        check(rt.hipStreamEndCapture(ctypes.c_void_p(s.handle), ctypes.byref(graph)), "end")
    check(rt.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)), "instantiate")
    for i in range(4):
        for k, b in a.dev.items():
            b.upload((other if i % 2 else a).host[k])
        for b in a.res.values():
            b.upload(np.full(b.nbytes // 4, np.nan, np.float32))
        synchronize()
        check(rt.hipGraphLaunch(run, ctypes.c_void_p(s.handle)), "launch")
        s.synchronize()
        other.run()
        synchronize()
        for k, v in (new if i % 2 else want).items():
            assert (a.results()[k].view(np.uint32) == v.view(np.uint32)).all(), f"replay {i}: {k}"
            assert (other.results()[k].view(np.uint32) == new[k].view(np.uint32)).all(), f"eager after replay {i}: {k}"
    check(rt.hipGraphExecDestroy(run), "destroy")
    check(rt.hipGraphDestroy(graph), "destroy")


def test_ends_on_two_streams_at_once(K, form):
    runs = [Ends(K, 300, 1000, 96, 41), Ends(K, 700, 2048, 128, 42)]
    streams = [Stream(), Stream()]
    for r in runs:
        r.run()
    synchronize()
    want = [r.results() for r in runs]
    for _ in range(5):
        for r, s in zip(runs, streams):
            r.run(s.handle)
    for s in streams:
        s.synchronize()
    for r, w in zip(runs, want):
        got = r.results()
        assert all((got[k].view(np.uint32) == w[k].view(np.uint32)).all() for k in w)


# ---- through the engine ----------------------------------------------------------------------------------------------
def test_engine_embedding(eng):
    rng = np.random.default_rng(6)
    L, V, D = eng.lib, 11, 6
    w = rng.standard_normal((V, D)).astype(np.float32)
    tokens = rng.integers(0, V, (3, 4, 2)).astype(np.int32)
    p, G = eng.param(w), rng.standard_normal((4, 3, 2, D)).astype(np.float32)
    t = L.nc_transpose(eng.tensor(tokens), 0, 1)  # a view of tokens
    y = L.nc_embedding(p, t, c_float(1.5), c_int32(3))
    tk = tokens.transpose(1, 0, 2)
    assert (eng.read(y) == w[tk] * np.float32(1.5)).all()
    eng.backward_with(y, G)
    ref, size = R.embedding_grad(tk, G, V, 1.5, 3)
    assert (np.abs(eng.grad(p) - ref) <= R.embedding_grad_tol(size)).all()
    y = L.nc_embedding(p, t, c_float(1.5), c_int32(-1))
    eng.backward_with(y, G)  # added to the first one
    ref2, size2 = R.embedding_grad(tk, G, V, 1.5)
    assert (np.abs(eng.grad(p) - ref - ref2) <= R.embedding_grad_tol(size + size2, size)).all()
    eng.step_end()


def test_engine_embedding_of_a_view_and_bad_tokens(eng):
    rng = np.random.default_rng(7)
    L = eng.lib
    w = rng.standard_normal((9, 10)).astype(np.float32)
    for v, host in ((L.nc_slice(eng.tensor(w), 1, 2, 5, 1), w[:, 2:7]), (L.nc_transpose(eng.tensor(w), 0, 1), w.T),
                    (L.nc_slice(eng.tensor(w), 0, 1, 3, 2), w[1:6:2])):
        y = L.nc_embedding(v, eng.tensor(np.array([0, 2, 1], np.int32)), c_float(1), c_int32(-1))
        assert (eng.read(y) == host[[0, 2, 1]]).all()
    for t, text in ((9, "token 9 at position 1 outside [0, 9)"), (-1, "token -1 at position 1")):
        y = L.nc_embedding(eng.tensor(w), eng.tensor(np.array([[3, t], [t, 0]], np.int32)), c_float(1), c_int32(-1))
        assert not y and L.nc_status_code(eng.ctx) == abi.ERR_ARG
        with pytest.raises(NcError, match=text.replace("[", r"\[").replace("(", r"\(").replace(")", r"\)")):
            eng.check()
    y = L.nc_embedding(eng.tensor(w), eng.tensor(np.zeros((0, 2), np.int32)), c_float(1), c_int32(-1))
    assert eng.read(y).shape == (0, 2, 10)
    eng.step_end()


def test_engine_dropout(eng):
    rng = np.random.default_rng(8)
    L, shape = eng.lib, (5, 7, 3)
    x, r, G = (rng.standard_normal(shape).astype(np.float32) for _ in range(3))
    px, pr = eng.param(x), eng.param(r)
    y = L.nc_dropout_seeded(px, pr, c_double(0.4), c_uint64(2 ** 64 - 1), c_uint64(17))
    exp = R.dropout(x, 0.4, 2 ** 64 - 1, 17, residual=r)
    assert np.allclose(eng.read(y), exp, rtol=2 * HALF, atol=0)
    eng.backward_with(y, G)
    assert (eng.grad(px) == R.dropout(G, 0.4, 2 ** 64 - 1, 17)).all() and (eng.grad(pr) == G).all()
    # x as its own residual, and a view
    y = L.nc_dropout_seeded(px, px, c_double(0.4), c_uint64(3), c_uint64(4))
    L.nc_clear_grad(px)
    eng.backward_with(y, G)
    exp = R.dropout(G, 0.4, 3, 4).astype(np.float64) + G
    assert (np.abs(eng.grad(px) - exp) <= 2 * HALF * np.abs(exp)).all()
    v = L.nc_transpose(px, 0, 2)
    assert (eng.read(L.nc_dropout_seeded(v, None, c_double(0.5), c_uint64(1), c_uint64(0)))
            == R.dropout(np.ascontiguousarray(x.transpose(2, 1, 0)), 0.5, 1, 0)).all()
    eng.step_end()


@pytest.mark.parametrize("flags", [0, abi.BACKWARD_RETAIN, abi.BACKWARD_FREE_GRAPH])
@pytest.mark.parametrize("bias", [False, True])
def test_engine_loss(eng, flags, bias):
    L = eng.lib
    x, w, b, labels = loss_inputs(60, 24, 90, 21, bias, 0.2)
    ref = R.vocab_loss(x, w, b, labels)
    px, pw, pb = eng.param(x.reshape(3, 20, 24)), eng.param(w), eng.param(b) if bias else None
    y = L.nc_linear_cross_entropy(px, pw, pb, eng.tensor(labels.reshape(3, 20)), c_int32(-100), 0)
    assert abs(eng.read(y) - ref["loss"]) <= R.vocab_loss_tol(x, w, ref)["loss"]
    loss = L.nc_scale(y, c_float(3.0))
    # the inputs may be written between the two
    L.nc_copy_from(px, np.zeros_like(x).ctypes.data_as(ctypes.c_void_p), x.nbytes)
    for times in range(2 if flags == abi.BACKWARD_RETAIN else 1):
        assert L.nc_backward_ex(loss, flags, None, 0) == 0, L.nc_error(eng.ctx)
    got = {"gx": eng.grad(px).reshape(x.shape), "gw": eng.grad(pw)}
    if bias:
        got["gb"] = eng.grad(pb)
    f = 3.0 * (2 if flags == abi.BACKWARD_RETAIN else 1)
    agree({k: v / np.float32(f) for k, v in got.items()}, ref, x, w)
    eng.step_end()


def test_engine_loss_refusals(eng):
    L = eng.lib
    x, w, b, labels = loss_inputs(6, 5, 9, 22, True, 0.0)
    labels[4] = 9
    y = L.nc_linear_cross_entropy(eng.param(x), eng.param(w), None, eng.tensor(labels), c_int32(-100), 0)
    assert not y and L.nc_status_code(eng.ctx) == abi.ERR_ARG
    with pytest.raises(NcError, match=r"label 9 at row 4 outside \[0, 9\)"):
        eng.check()
    labels[4] = 0
    t, pw = eng.tensor(x), eng.param(w)
    y = L.nc_linear_cross_entropy(t, pw, None, eng.tensor(labels), c_int32(-100), 0)
    L.nc_set_requires_grad(t, 1)
    assert L.nc_backward(y) != 0
    with pytest.raises(NcError, match="came to need a gradient"):
        eng.check()
    eng.step_end()


def test_engine_trains_tied_ends(eng):
    """A step of a model with one table at both ends: the gradient against differences of the 64-bit loss."""
    L = eng.lib
    rng = np.random.default_rng(9)
    N, V, D = 12, 30, 8
    w = (rng.standard_normal((V, D)) * 0.4).astype(np.float32)
    tokens, labels = rng.integers(0, V, N).astype(np.int32), rng.integers(0, V, N).astype(np.int32)
    labels[5] = -1
    keep = R.kept(N * D, 0.25, 6, 7).reshape(N, D) / 0.75

    def loss64(w):
        return R.vocab_loss(w[tokens] * 1.5 * keep, w, None, labels, ignore=-1)["loss"]

    p = eng.param(w)
    e = L.nc_dropout_seeded(L.nc_embedding(p, eng.tensor(tokens), c_float(1.5), c_int32(-1)), None, c_double(0.25), c_uint64(6), c_uint64(7))
    y = L.nc_linear_cross_entropy(e, p, None, eng.tensor(labels), c_int32(-1), 0)
    assert abs(eng.read(y) - loss64(w.astype(np.float64))) < 1e-5  # some 20 roundings of values below 10
    assert L.nc_backward(y) == 0, L.nc_error(eng.ctx)
    got, w64, h = eng.grad(p), w.astype(np.float64), 1e-5
    for i in [(0, 0), (int(tokens[0]), 3), (int(labels[2]), 5), (V - 1, D - 1), (int(tokens[5]), 1)]:
        d = np.zeros_like(w64)
        d[i] = h
        diff = (loss64(w64 + d) - loss64(w64 - d)) / (2 * h)
        assert abs(got[i] - diff) < 1e-6  # the difference 1e-9, the gradient some 100 roundings of terms below 0.1
    eng.step_end()
