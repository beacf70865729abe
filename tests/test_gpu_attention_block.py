"""The attention block on the GPU against the 64-bit references: rotary positions, the per-head norm with the rotation, cross
attention; through the kernel layer on device buffers (odd sizes, strides, alignments, lengths, masked places that hold
infinities and NaN) and through the engine with autograd, alone and together."""
import ctypes
from ctypes import c_float, c_int64

import numpy as np
import pytest

from newch_amd import abi, hip
from newch_amd.hipmem import DeviceBuffer, Stream, check, runtime, synchronize
from tests import attention_ref as R
from tests.ncdrive import Engine, NcError

pytestmark = pytest.mark.gpu


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


def i64(*v):
    return (c_int64 * max(len(v), 1))(*v)


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


def place(a, order="blhd", shift=0, gap=0):
    """(buffer, pointer, strides) of a [B, L, H, D] array laid out in another order of its first three axes, rows `gap` floats apart;
    what is not the array is NaN."""
    a = np.asarray(a, np.float32)
    sizes = dict(zip("blhd", a.shape))
    perm = ["blhd".index(c) for c in order]
    row = sizes["d"] + gap
    host = np.full([sizes[c] for c in order[:3]] + [row], np.nan, np.float32)
    host[..., : sizes["d"]] = a.transpose(perm)
    st, n = {}, row
    for c in reversed(order[:3]):
        st[c] = n
        n *= sizes[c]
    buf = DeviceBuffer.from_numpy(np.concatenate([np.full(shift, np.nan, np.float32), host.reshape(-1)]))
    return buf, buf.ptr + 4 * shift, [st["b"], st["l"], st["h"]]


def up(a):
    return None if a is None else DeviceBuffer.from_numpy(np.asarray(a))


def ptr(b):
    return None if b is None else b.ptr


# ---- rotary positions, with and without the norm ---------------------------------------------------------------------
# B, L, H, D, the axes' columns
ROPE_SHAPES = [(1, 1, 1, 2, (2,)), (1, 1, 1, 1, ()), (2, 3, 5, 64, (32, 32)), (1, 1, 40, 128, (128,)), (3, 7, 3, 80, (20, 30, 30)),
               (2, 65, 2, 128, (32, 48, 48)), (1, 9, 1, 256, (256,)), (2, 5, 3, 255, (128, 2)), (1, 33, 4, 65, (64,)),
               (2, 1030, 1, 8, (8,)), (1, 40, 17, 36, (8, 8)), (1, 1, 300, 40, (40,)), (1, 2100, 2, 96, (16, 8, 8, 24)),
               (2, 17, 33, 32, (16,)), (5, 3, 2, 6, (2, 2, 2)), (1, 2, 3, 250, (2, 244, 2))]


def rope_inputs(shape, seed, far=False):
    B, L, H, D, dims = shape
    rng = np.random.default_rng(seed)
    x, g = (rng.standard_normal((B, L, H, D)).astype(np.float32) for _ in range(2))
    hi = 2 ** 31 - 1 if far else 5000
    pos = rng.integers(-hi - far, hi, (B, L, max(len(dims), 1))).astype(np.int32)[..., : len(dims)]
    return x, g, pos, rng.standard_normal(D).astype(np.float32), rng.standard_normal(D).astype(np.float32)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", [s for s in ROPE_SHAPES if s[4]], ids=str)
def test_rope_kernel(K, shape, interleaved):
    B, L, H, D, dims = shape
    x, g, pos, _, _ = rope_inputs(shape, 1, far=H == 2)
    for batched, order, shift, gap in ((1, "blhd", 0, 0), (0, "hbld", 1, 3)):
        print(f"rope {shape} {batched} {order}", flush=True)
        p = np.ascontiguousarray(pos if batched else pos[0])
        X, xp, sx = place(x, order, shift, gap)
        P, G = up(p), up(g)
        y, gx = Out(x.shape, shift=shift), Out(x.shape, shift=shift)
        old = np.random.default_rng(2).standard_normal(x.shape).astype(np.float32)
        gx2 = Out(x.shape, fill=old)
        K.rope_fwd(B, L, H, D, xp, sx, P.ptr, batched, dims, 1e4, interleaved, y.ptr)
        K.rope_bwd(B, L, H, D, G.ptr, P.ptr, batched, dims, 1e4, interleaved, gx.ptr, accumulate=False)
        K.rope_bwd(B, L, H, D, G.ptr, P.ptr, batched, dims, 1e4, interleaved, gx2.ptr)
        synchronize()
        want, mag = R.rope64(x, p, dims, 1e4, interleaved)
        R.within(y.get(), want, R.ROPE_TOL * mag, "y")
        want, mag = R.rope64(g, p, dims, 1e4, interleaved, -1.0)
        R.within(gx.get(), want, R.ROPE_TOL * mag, "gx")
        R.within(gx2.get(), want + old, (R.ROPE_TOL + R.U) * mag + R.U * np.abs(old), "gx added")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", ROPE_SHAPES, ids=str)
def test_qk_norm_rope_kernel(K, shape, interleaved):
    B, L, H, D, dims = shape
    x, g, pos, wq, wk = rope_inputs(shape, 5)
    for qh, use_q, use_k, order, shift in ((H // 2, 1, 1, "blhd", 0), (H, 1, 0, "bhld", 1), (0, 0, 1, "lbhd", 2)):
        print(f"qk_norm_rope {shape} {qh} {order}", flush=True)
        X, xp, sx = place(x, order, shift, shift)
        P, G, Q, W = up(pos), up(g), up(wq) if use_q else None, up(wk) if use_k else None
        args = (xp, sx, ptr(Q), ptr(W), 1e-6, P.ptr if dims else None, 1, dims, 1e4, interleaved)
        y, gx = Out(x.shape, shift=shift), Out(x.shape)
        old = np.random.default_rng(6).standard_normal(D).astype(np.float32)
        gwq, gwk = Out((D,)), Out((D,), fill=old)
        n = K.qk_norm_rope_bwd_workspace(B, L, H, D)
        ws = DeviceBuffer.from_numpy(np.full(n, 0xCD, np.uint8))
        K.qk_norm_rope_fwd(B, L, H, D, qh, *args, y.ptr)
        K.qk_norm_rope_bwd(B, L, H, D, qh, *args, G.ptr, gx.ptr, gwq.ptr, gwk.ptr, ws.ptr, n, accumulate=(0, 0, 1))
        synchronize()
        ref = (x, qh, wq if use_q else None, wk if use_k else None, 1e-6, pos, dims, 1e4, interleaved)
        R.within(y.get(), *R.qk_norm_rope64(*ref), "y")
        want = R.qk_norm_rope_bwd64(*ref, g)
        R.within(gx.get(), *want["gx"], "gx")
        R.within(gwq.get(), *want["gwq"], "gwq")
        v, b = want["gwk"]
        R.within(gwk.get(), v + old, b + R.U * (np.abs(v) + np.abs(old)), "gwk added")


def test_rope_many_rows_of_one_batch_wrap(K):
    """Groups of tokens that run over the end of a sequence, positions shared by all sequences; x is one row repeated (strides 0)."""
    B, L, H, D = 700, 7, 1, 64
    rng = np.random.default_rng(7)
    x, pos = rng.standard_normal(D).astype(np.float32), rng.integers(0, 99, (L, 1)).astype(np.int32)
    X, P, y = up(x), up(pos), Out((B, L, H, D))
    K.rope_fwd(B, L, H, D, X.ptr, (0, 0, 0), P.ptr, 0, (64,), 1e4, 0, y.ptr)
    synchronize()
    want, mag = R.rope64(np.broadcast_to(x, (B, L, H, D)), pos, (64,), 1e4, 0)
    R.within(y.get(), want, R.ROPE_TOL * mag, "y")


def test_norm_of_zero_and_huge_rows(K):
    """A row of zeros stays zeros (eps 0 gives NaN, as the formula does); rows of NaN or infinities do not reach their neighbours."""
    x = np.ones((1, 4, 1, 64), np.float32)
    x[0, 0] = 0
    x[0, 1, 0, 3] = np.inf
    x[0, 2] = 1e15
    X, y = up(x), Out(x.shape)
    K.qk_norm_rope_fwd(1, 4, 1, 64, 1, X.ptr, (256, 64, 64), None, None, 1e-6, None, 0, (), 1.0, 0, y.ptr)
    synchronize()
    got = y.buf.to_numpy(np.float32, y.host.shape)[GUARD: GUARD + 256].reshape(4, 64)
    assert (got[0] == 0).all() and np.isnan(got[1]).any() and np.abs(got[2:] - 1).max() < 1e-6


# ---- cross attention ------------------------------------------------------------------------------------------------------
# B, Lq, Lk, Hq, Hkv, D, lengths
ATTN_SHAPES = [(1, 1, 1, 1, 1, 1, None), (2, 1, 5, 4, 2, 8, (5, 0)), (3, 1, 1500, 3, 3, 64, (1500, 1, 33)),
               (2, 1, 700, 16, 2, 128, (0, 700)), (2, 197, 197, 2, 2, 64, None), (3, 33, 77, 4, 1, 80, (77, 0, 12)),
               (1, 129, 65, 2, 1, 128, (64,)), (2, 64, 32, 3, 3, 32, (-4, 99)), (1, 300, 3, 2, 2, 40, None),
               (1, 5, 300, 6, 3, 96, (299,)), (1, 31, 130, 2, 2, 256, None), (2, 7, 40, 2, 1, 255, (40, 17)),
               (1, 2, 2, 1, 1, 3, None), (4, 16, 64, 8, 8, 64, (64, 63, 33, 32)), (1, 1, 4097, 8, 1, 64, None),
               (1, 260, 515, 4, 2, 100, (514,)), (1, 3, 0, 2, 1, 16, None)]


def attn_inputs(shape, seed, std=1.5):
    B, Lq, Lk, Hq, Hkv, D, lens = shape
    rng = np.random.default_rng(seed)
    q, g = (rng.standard_normal((B, Lq, Hq, D)).astype(np.float32) for _ in range(2))
    k, v = (rng.standard_normal((B, Lk, Hkv, D)).astype(np.float32) for _ in range(2))
    return q * np.float32(std), k * np.float32(std), v, g, None if lens is None else np.array(lens, np.int32)


def run_attention(K, shape, q, k, v, g, lens, order="blhd", shift=0, gap=0, old=None, scale=None, stream=None, want="qkv",
                  poison=0xFF):
    """Forward and backward on buffers between guards; k and v past the lengths are NaN and infinities."""
    B, Lq, Lk, Hq, Hkv, D, _ = shape
    k, v = k.copy(), v.copy()
    if lens is not None:
        for b, n in enumerate(np.clip(lens, 0, Lk)):
            k[b, n:], v[b, n:] = np.nan, np.inf
    scale = D ** -0.5 if scale is None else scale
    bufs = [place(t, order, shift, gap) for t in (q, k, v)]
    src = sum(((p, s) for _, p, s in bufs), ())
    N, G = up(lens), up(g)
    o, lse = Out(q.shape, shift=shift), Out((B, Hq, Lq))
    sizes = (B, Lq, Lk, Hq, Hkv, D)
    n1, n2 = K.cross_attention_fwd_workspace(*sizes), K.cross_attention_bwd_workspace(*sizes)
    ws = DeviceBuffer.from_numpy(np.full(max(n1, n2) + 256, poison, np.uint8))
    K.cross_attention_fwd(*sizes, scale, *src, ptr(N), o.ptr, lse.ptr, ws.ptr, n1, stream=stream)
    outs = {}
    for c, like in (("q", q), ("k", k), ("v", v)):
        outs["g" + c] = Out(like.shape, fill=np.nan if old is None else np.broadcast_to(old, like.shape), shift=shift) if c in want else None
    K.cross_attention_bwd(*sizes, scale, *src, ptr(N), o.ptr, lse.ptr, G.ptr, *(ptr(outs["g" + c]) for c in "qkv"), ws.ptr, n2,
                          accumulate=old is not None, stream=stream)
    synchronize()
    tail = ws.to_numpy(np.uint8, 256, offset=max(n1, n2))
    assert (tail == poison).all(), "written past the workspace"
    return {"o": o.get(), "lse": lse.get(), **{k: t.get() for k, t in outs.items() if t is not None}}


def check_attention(got, ref, old=0.0, what=""):
    for name, v in got.items():
        want, bound = ref[name]
        if name.startswith("g") and np.any(old):
            want, bound = want + old, bound + R.U * (np.abs(want) + np.abs(old))
        R.within(v, want, bound, f"{what} {name}")


@pytest.mark.parametrize("shape", ATTN_SHAPES, ids=str)
def test_attention_kernel(K, shape):
    q, k, v, g, lens = attn_inputs(shape, 11)
    D = shape[5]
    ref = R.attention64(q, k, v, lens, D ** -0.5, g)
    for order, shift, gap, old in (("blhd", 0, 0, None), ("bhld", 1, 5, 0.25), ("lhbd", 3, 0, None)):
        print(f"attention {shape} {order}", flush=True)
        old_v = None if old is None else np.float32(old)
        check_attention(run_attention(K, shape, q, k, v, g, lens, order, shift, gap, old_v), ref, old or 0.0, order)


# what the sizes above do not reach: rows of few keys cut among workgroups with heads that do not divide a tile; few keys of two
# to eight tiles; three to eight rows of odd widths; many parts of keys, or of queries; wide heads over several tiles
PATH_SHAPES = [(1, 900, 40, 6, 2, 64, (33,)), (2, 130, 200, 4, 2, 64, (200, 131)), (1, 70, 500, 2, 1, 32, (481,)),
               (1, 700, 150, 2, 2, 96, None), (2, 3, 400, 2, 2, 30, (400, 129)), (1, 2, 300, 8, 2, 250, (299,)),
               (2, 1, 600, 5, 1, 101, (0, 600)), (1, 1, 900, 3, 3, 255, None), (1, 2000, 50, 1, 1, 128, (45,)),
               (1, 40, 3000, 1, 1, 64, (2990,)), (1, 300, 290, 2, 1, 200, (285,)), (1, 9, 2100, 3, 3, 48, None),
               (1, 33, 260, 5, 5, 64, None), (300, 5, 9, 4, 2, 16, None), (1, 4, 4, 64, 1, 64, None),
               (1, 900, 70, 6, 2, 128, (65,)), (2, 100, 128, 2, 2, 90, (128, 31)), (1, 2000, 140, 1, 1, 128, (135,)),
               (1, 12, 0, 2, 1, 128, None), (2, 30, 0, 2, 2, 200, None), (2, 4, 0, 2, 2, 64, None),
               # more than a workgroup a CU
               (40, 10, 300, 7, 7, 64, tuple(range(290, 250, -1))), (33, 9, 161, 8, 8, 128, tuple(range(0, 165, 5))),
               (260, 9, 520, 1, 1, 30, None), (130, 9, 200, 2, 2, 90, None)]


@pytest.mark.parametrize("shape", PATH_SHAPES, ids=lambda s: str(s[:6]))
def test_attention_paths(K, shape):
    q, k, v, g, lens = attn_inputs(shape, 28)
    ref = R.attention64(q, k, v, lens, shape[5] ** -0.5, g)
    check_attention(run_attention(K, shape, q, k, v, g, lens, "bhld", 2, 3), ref)


@pytest.mark.parametrize("shape", [(2, 70, 45, 4, 2, 64, (45, 3)), (1, 300, 100, 2, 2, 128, (70,)), (1, 90, 400, 2, 1, 96, None)], ids=str)
@pytest.mark.parametrize("want", ["q", "k", "v", "qv", ""])
def test_attention_some_gradients(K, want, shape):
    q, k, v, g, lens = attn_inputs(shape, 12)
    check_attention(run_attention(K, shape, q, k, v, g, lens, want=want), R.attention64(q, k, v, lens, shape[5] ** -0.5, g))


@pytest.mark.parametrize("value", [np.inf, np.nan])
@pytest.mark.parametrize("shape", [(1, 70, 45, 2, 2, 64, None), (1, 70, 45, 2, 2, 128, None), (1, 70, 300, 2, 2, 64, None)], ids=str)
def test_attention_infinite_gradient_stays_in_its_row(K, shape, value):
    """An output gradient that is not finite leaves the other rows' gradients of the queries, and other heads', as they are."""
    q, k, v, g, lens = attn_inputs(shape, 33)
    g[0, 5, 0] = 0
    ref = R.attention64(q, k, v, lens, shape[5] ** -0.5, g)
    g[0, 5, 0] = value
    B, Lq, Lk, Hq, Hkv, D, _ = shape
    Q, K_, V, G = (up(t) for t in (q, k, v, g))
    src = (Q.ptr, (Lq * Hq * D, Hq * D, D), K_.ptr, (Lk * Hkv * D, Hkv * D, D), V.ptr, (Lk * Hkv * D, Hkv * D, D), None)
    o, lse, outs = Out(q.shape), Out((B, Hq, Lq)), [Out(t.shape) for t in (q, k, v)]
    n1, n2 = K.cross_attention_fwd_workspace(*shape[:6]), K.cross_attention_bwd_workspace(*shape[:6])
    ws = DeviceBuffer.empty(max(n1, n2, 1))
    K.cross_attention_fwd(*shape[:6], D ** -0.5, *src, o.ptr, lse.ptr, ws.ptr, n1)
    K.cross_attention_bwd(*shape[:6], D ** -0.5, *src, o.ptr, lse.ptr, G.ptr, *(t.ptr for t in outs), ws.ptr, n2, accumulate=False)
    synchronize()
    gq, gk, gv = (t.get() for t in outs)
    rest = np.ones(gq.shape[:3], bool)
    rest[0, 5, 0] = False
    assert not np.isfinite(gq[0, 5, 0]).any()
    R.within(gq[rest], ref["gq"][0][rest], ref["gq"][1][rest], "gq")
    for name, t in (("gk", gk), ("gv", gv)):
        R.within(t[:, :, 1], ref[name][0][:, :, 1], ref[name][1][:, :, 1], name)
        assert not np.isfinite(t[0, :, 0]).any()


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_attention_scales_and_sharp_rows(K, scale):
    """Rows all alike, a negative scale, and rows where one key takes nearly all (scores in the hundreds)."""
    shape = (1, 40, 90, 2, 2, 64, None)
    q, k, v, g, lens = attn_inputs(shape, 13)
    check_attention(run_attention(K, shape, q, k, v, g, lens, scale=scale), R.attention64(q, k, v, lens, scale, g))


@pytest.mark.parametrize("shape", [(1, 40, 90, 2, 2, 64, None), (1, 40, 300, 2, 2, 64, None), (1, 2, 90, 1, 1, 64, None)], ids=str)
@pytest.mark.parametrize("scale", [300.0, 1e6, 1e30])
def test_attention_large_scale_and_rows_of_zeros(K, shape, scale):
    """A query of zeros weighs its keys alike whatever the scale; the others hold what the scale takes."""
    q, k, v, g, lens = attn_inputs(shape, 34)
    q *= np.float32(0.125 / scale)
    q[0, 1] = 0
    check_attention(run_attention(K, shape, q, k, v, g, lens, scale=scale), R.attention64(q, k, v, lens, scale, g))


@pytest.mark.parametrize("shape", [(1, 40, 1, 2, 2, 64, None), (1, 40, 90, 2, 2, 128, None), (1, 40, 300, 2, 2, 64, None)], ids=str)
def test_attention_huge_queries_without_gradient(K, shape):
    """Scores without gradients (one key: but for roundings; or none of the output) against queries of 1e25: no NaN."""
    q, k, v, g, lens = attn_inputs(shape, 35)
    q *= np.float32(1e25)
    k *= np.float32(1e-25)
    if shape[2] > 1:
        g[:] = 0
    got = run_attention(K, shape, q, k, v, g, lens, scale=0.125)
    if shape[2] > 1:
        assert all((got[i] == 0).all() for i in ("gq", "gk", "gv"))
    else:
        check_attention(got, R.attention64(q, k, v, lens, 0.125, g))


@pytest.mark.parametrize("mag", [1e-12, 1e12])
def test_attention_magnitudes(K, mag):
    """Values and gradients of any magnitude, keys and queries whose magnitudes cancel: the pieces' scales follow them."""
    shape = (2, 40, 90, 2, 1, 64, (90, 50))
    q, k, v, g, lens = attn_inputs(shape, 14)
    m = np.float32(mag)
    q, k, v, g = q * m, k / m, v * m, g / m
    check_attention(run_attention(K, shape, q, k, v, g, lens), R.attention64(q, k, v, lens, 0.125, g))


def test_attention_rows_of_unlike_magnitudes(K):
    """Sequences, heads and tokens from 2^-20 to 2^20 of each other beside one another."""
    shape = (2, 70, 90, 4, 2, 64, None)
    q, k, v, g, lens = attn_inputs(shape, 15)
    rng = np.random.default_rng(16)
    v *= np.exp2(rng.integers(-10, 11, v.shape[:3])).astype(np.float32)[..., None]
    g *= np.exp2(rng.integers(-10, 11, g.shape[:3])).astype(np.float32)[..., None]
    v[0] *= np.float32(2.0 ** -20)
    q[:, :, 1] *= np.float32(2.0 ** -18)
    check_attention(run_attention(K, shape, q, k, v, g, lens), R.attention64(q, k, v, lens, 0.125, g))


def test_attention_nan_stays_in_its_sequence(K):
    """A NaN in a key that counts reaches its sequence's head, and nothing else."""
    shape = (2, 40, 70, 2, 2, 64, (70, 60))
    q, k, v, g, lens = attn_inputs(shape, 17)
    ref = R.attention64(q, k, v, lens, 0.125, g)
    k[0, 3, 1, 5] = np.nan
    N = up(lens)
    bufs = [place(t) for t in (q, k, v)]
    src = sum(((p, s) for _, p, s in bufs), ())
    o = DeviceBuffer.from_numpy(np.zeros_like(q))
    n = K.cross_attention_fwd_workspace(*shape[:6])
    ws = DeviceBuffer.empty(n)
    K.cross_attention_fwd(*shape[:6], 0.125, *src, N.ptr, o.ptr, None, ws.ptr, n)
    synchronize()
    got = o.to_numpy(np.float32, q.shape)
    assert np.isnan(got[0, :, 1]).all()
    clean = [(0, slice(None), 0), (1, slice(None), slice(None))]
    for at in clean:
        R.within(got[at], ref["o"][0][at], ref["o"][1][at], str(at))


# rows of a pair against keys: eight rows read in parts, parts joined by rows, and parts joined by pieces
@pytest.mark.parametrize("shape", [(1, 1, 3000, 1, 1, 64, None), (1, 20, 3000, 2, 2, 128, None), (1, 3000, 700, 2, 2, 96, None),
                                   (1, 300, 90, 2, 2, 64, None)], ids=str)
def test_attention_nan_query_stays_in_its_row(K, shape):
    """A row of queries that holds a NaN gives NaN, whichever way its keys' parts are joined, and its neighbours their values."""
    q, k, v, g, lens = attn_inputs(shape, 20)
    Lq, Hq = shape[1], shape[3]
    ref = R.attention64(q, k, v, lens, 0.125, None)
    q[0, Lq // 2, 0, 1] = np.nan
    o, lse, n = Out(q.shape), Out((1, Hq, Lq)), K.cross_attention_fwd_workspace(*shape[:6])
    bufs = [place(t) for t in (q, k, v)]
    src = sum(((p, s) for _, p, s in bufs), ())
    ws = DeviceBuffer.empty(max(n, 1))
    K.cross_attention_fwd(*shape[:6], 0.125, *src, None, o.ptr, lse.ptr, ws.ptr, n)
    synchronize()
    got, l = o.get(), lse.get()
    assert np.isnan(got[0, Lq // 2, 0]).all() and np.isnan(l[0, 0, Lq // 2])
    rest = np.ones((1, Lq, Hq), bool)
    rest[0, Lq // 2, 0] = False
    R.within(got[rest], ref["o"][0][rest], ref["o"][1][rest], "o")
    R.within(l.transpose(0, 2, 1)[rest], *(t.transpose(0, 2, 1)[rest] for t in ref["lse"]), "lse")


def test_attention_is_deterministic_and_takes_streams(K):
    """The same bits on another stream, twice, from workspaces that held other bytes."""
    shape = (2, 150, 333, 4, 2, 64, (333, 100))
    q, k, v, g, lens = attn_inputs(shape, 18)
    first = run_attention(K, shape, q, k, v, g, lens)
    s = Stream()
    for poison in (0xFF, 0x00, 0x7F):
        again = run_attention(K, shape, q, k, v, g, lens, stream=s.handle, poison=poison)
        for name, a in first.items():
            assert (a.view(np.uint32) == again[name].view(np.uint32)).all(), name


@pytest.mark.parametrize("shape", [(2, 0, 5, 2, 1, 64), (1, 0, 300, 2, 1, 64), (1, 0, 5, 2, 2, 128), (1, 0, 40, 2, 2, 200)], ids=str)
def test_attention_without_queries(K, shape):
    """No queries: nothing forward, gradients of the keys and values that are zero, or stay where they are added to."""
    B, Lq, Lk, Hq, Hkv, D = shape
    k, v = up(np.ones((B, Lk, Hkv, D), np.float32)), up(np.ones((B, Lk, Hkv, D), np.float32))
    s = (Lk * Hkv * D, Hkv * D, D)
    src = (None, (0, Hq * D, D), k.ptr, s, v.ptr, s, None)
    n = K.cross_attention_bwd_workspace(*shape)
    ws = DeviceBuffer.empty(max(n, 1))
    K.cross_attention_fwd(*shape, 0.1, *src, None, None)
    for old in (None, 0.5):
        gk, gv = (Out((B, Lk, Hkv, D), fill=np.nan if old is None else np.float32(old)) for _ in "kv")
        K.cross_attention_bwd(*shape, 0.1, *src, None, None, None, None, gk.ptr, gv.ptr, ws.ptr, n, accumulate=old is not None)
        synchronize()
        assert (gk.get() == (old or 0)).all() and (gv.get() == (old or 0)).all()


class Block:
    """Norm and rotation of the queries, attention to rotated keys, and its backward, on buffers of its own."""

    def __init__(self, K, shape, seed):
        B, Lq, Lk, Hq, Hkv, D, _ = self.shape = shape
        self.K, self.sizes = K, shape[:6]
        self.host = attn_inputs(shape, seed)
        self.q, self.k, self.v, self.g, self.n = (up(t) for t in self.host)
        self.wq = up(np.linspace(0.5, 1.5, D, dtype=np.float32))
        self.pos = up(np.arange(max(Lq, Lk), dtype=np.int32)[:, None])
        new = lambda *s: DeviceBuffer.from_numpy(np.full(s, np.nan, np.float32))
        self.x, self.y, self.o, self.lse = new(B, Lq, Hq, D), new(B, Lk, Hkv, D), new(B, Lq, Hq, D), new(B, Hq, Lq)
        self.gx, self.gk, self.gv, self.gq = new(B, Lq, Hq, D), new(B, Lk, Hkv, D), new(B, Lk, Hkv, D), new(B, Lq, Hq, D)
        self.gw = new(D)
        self.n1, self.n2 = K.cross_attention_fwd_workspace(*self.sizes), K.cross_attention_bwd_workspace(*self.sizes)
        self.n3 = K.qk_norm_rope_bwd_workspace(B, Lq, Hq, D)
        self.ws = DeviceBuffer.empty(max(self.n1, self.n2, self.n3, 1))

    def run(self, stream):
        B, Lq, Lk, Hq, Hkv, D = self.sizes
        sq, sk = (Lq * Hq * D, Hq * D, D), (Lk * Hkv * D, Hkv * D, D)
        K, rot = self.K, (0, (D // 2 * 2,), 100.0, 0)
        K.qk_norm_rope_fwd(B, Lq, Hq, D, Hq, self.q.ptr, sq, self.wq.ptr, None, 1e-6, self.pos.ptr, *rot, self.x.ptr, stream=stream)
        K.rope_fwd(B, Lk, Hkv, D, self.k.ptr, sk, self.pos.ptr, *rot, self.y.ptr, stream=stream)
        src = (self.x.ptr, sq, self.y.ptr, sk, self.v.ptr, sk, ptr(self.n))
        K.cross_attention_fwd(*self.sizes, 0.2, *src, self.o.ptr, self.lse.ptr, self.ws.ptr, self.n1, stream=stream)
        K.cross_attention_bwd(*self.sizes, 0.2, *src, self.o.ptr, self.lse.ptr, self.g.ptr, self.gx.ptr, self.gk.ptr, self.gv.ptr,
                              self.ws.ptr, self.n2, accumulate=False, stream=stream)
        K.qk_norm_rope_bwd(B, Lq, Hq, D, Hq, self.q.ptr, sq, self.wq.ptr, None, 1e-6, self.pos.ptr, *rot, self.gx.ptr, self.gq.ptr,
                           self.gw.ptr, None, self.ws.ptr, self.n3, accumulate=False, stream=stream)

    def results(self):
        got = [b.to_numpy(np.float32, b.nbytes // 4) for b in (self.x, self.y, self.o, self.lse, self.gx, self.gk, self.gv, self.gq, self.gw)]
        assert all(np.isfinite(t).all() for t in got)
        return [t.view(np.uint32) for t in got]


BLOCK_SHAPES = [(2, 70, 45, 4, 2, 64, (45, 3)), (1, 1, 700, 4, 4, 64, (650,)), (1, 300, 600, 2, 2, 80, (590,)), (1, 150, 270, 2, 1, 200, None)]


@pytest.mark.parametrize("shape", BLOCK_SHAPES, ids=str)
def test_block_captured_and_replayed(K, shape):
    """The block as a graph: every replay, with other inputs and eager calls in between, gives the eager run's bits."""
    rt = runtime()
    a, other = Block(K, shape, 29), Block(K, shape, 30)
    a.run(None)
    other.run(None)
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
        for b, h in zip((a.q, a.k, a.v, a.g), (other if i % 2 else a).host):
            b.upload(h)
        for b in (a.x, a.y, a.o, a.lse, a.gx, a.gk, a.gv, a.gq, a.gw):
            b.upload(np.full(b.nbytes // 4, np.nan, np.float32))
        synchronize()
        check(rt.hipGraphLaunch(run, ctypes.c_void_p(s.handle)), "launch")
        s.synchronize()
        other.run(None)
        synchronize()
        for x, y in zip(a.results(), new if i % 2 else want):
            assert (x == y).all(), f"replay {i}"
        for x, y in zip(other.results(), new):
            assert (x == y).all(), f"eager after replay {i}"
    check(rt.hipGraphExecDestroy(run), "destroy")
    check(rt.hipGraphDestroy(graph), "destroy")


def test_blocks_on_two_streams_at_once(K):
    """Two blocks with workspaces of their own, their calls in flight together, several times over."""
    blocks = [Block(K, BLOCK_SHAPES[0], 31), Block(K, BLOCK_SHAPES[2], 32)]
    for b in blocks:
        b.run(None)
    synchronize()
    want, streams = [b.results() for b in blocks], [Stream(), Stream()]
    for _ in range(5):
        for b, s in zip(blocks, streams):
            b.run(s.handle)
    synchronize()
    for b, w in zip(blocks, want):
        for x, y in zip(b.results(), w):
            assert (x == y).all()


# read by rows, split by each workgroup, packed
@pytest.mark.parametrize("Lq,Lk,D,step", [(2, 5, 32, (1 << 29) + 12), (20, 5, 32, (1 << 29) + 12), (20, 300, 128, (1 << 23) + 4)])
def test_attention_long_strides(K, Lq, Lk, D, step):
    """Keys whose rows lie over 2^31 floats apart from first to last, forward and backward."""
    sizes = (1, Lq, Lk, 1, 1, D)
    q, k, v, g, _ = attn_inputs((*sizes, None), 19)
    big = DeviceBuffer.empty(4 * (step * (Lk - 1) + D))
    for j in range(Lk):
        big.upload(np.ascontiguousarray(k[0, j, 0]), 4 * j * step)
    Q, V, G, o, lse, outs = up(q), up(v), up(g), Out(q.shape), Out((1, 1, Lq)), [Out(t.shape) for t in (q, k, v)]
    src = (Q.ptr, (Lq * D, D, D), big.ptr, (0, step, 0), V.ptr, (Lk * D, D, D), None)
    n1, n2 = K.cross_attention_fwd_workspace(*sizes), K.cross_attention_bwd_workspace(*sizes)
    ws = DeviceBuffer.empty(max(n1, n2, 1))
    K.cross_attention_fwd(*sizes, 0.2, *src, o.ptr, lse.ptr, ws.ptr, n1)
    K.cross_attention_bwd(*sizes, 0.2, *src, o.ptr, lse.ptr, G.ptr, *(t.ptr for t in outs), ws.ptr, n2, accumulate=False)
    synchronize()
    got = {"o": o.get(), "lse": lse.get(), **{"g" + c: t.get() for c, t in zip("qkv", outs)}}
    check_attention(got, R.attention64(q, k, v, None, 0.2, g))


# ---- through the engine ----------------------------------------------------------------------------------------------------
def test_engine_rope_and_norm(eng):
    """Slices of a fused projection (strided views), positions of a batch, gradients through the slices; a weight shared by
    queries and keys; leaves that are used twice add up."""
    L = eng.lib
    rng = np.random.default_rng(21)
    B, T, Hq, Hk, D = 2, 11, 4, 2, 40
    qkv = rng.standard_normal((B, T, (Hq + 2 * Hk) * D)).astype(np.float32)
    w = rng.standard_normal(D).astype(np.float32)
    pos = rng.integers(0, 50, (B, T, 2)).astype(np.int32)
    g = rng.standard_normal((B, T, Hq + Hk, D)).astype(np.float32)
    X, W, P = eng.param(qkv), eng.param(w), eng.tensor(pos)
    nd, shp = abi.shape_arg((B, T, Hq + 2 * Hk, D))
    x = L.nc_slice(L.nc_reshape(X, nd, shp), 2, 0, Hq + Hk, 1)
    dims, args = (16, 24), (1e-5, pos, (16, 24), 100.0, False)
    y = L.nc_qk_norm_rope(x, Hq, W, W, c_float(1e-5), P, 2, i64(*dims), c_float(100.0), 0)
    xs = qkv.reshape(B, T, Hq + 2 * Hk, D)[:, :, : Hq + Hk]
    R.within(eng.read(y), *R.qk_norm_rope64(xs, Hq, w, w, *args), "y")
    for times in (1, 2):
        eng.backward_with(y, g)
        want = R.qk_norm_rope_bwd64(xs, Hq, w, w, *args, g)
        gx = np.zeros((B, T, Hq + 2 * Hk, D)), np.zeros((B, T, Hq + 2 * Hk, D))
        for k in range(2):
            gx[k][:, :, : Hq + Hk] = want["gx"][k]
        R.within(eng.grad(X).reshape(gx[0].shape), times * gx[0], times * 2 * gx[1], "gx")
        R.within(eng.grad(W), times * (want["gwq"][0] + want["gwk"][0]), times * 2 * (want["gwq"][1] + want["gwk"][1]) + 1e-4 * R.U, "gw")
    r = L.nc_rope(x, P, 2, i64(*dims), c_float(100.0), 1)
    want, mag = R.rope64(xs, pos, dims, 100.0, True)
    R.within(eng.read(r), want, R.ROPE_TOL * mag, "rope")


def test_engine_norm_without_gradient_of_x(eng):
    """Only the weights want gradients; then no weight is given at all."""
    L = eng.lib
    rng = np.random.default_rng(22)
    x, w, g = rng.standard_normal((1, 5, 3, 24)).astype(np.float32), rng.standard_normal(24).astype(np.float32), rng.standard_normal((1, 5, 3, 24)).astype(np.float32)
    X, W = eng.tensor(x), eng.param(w)
    y = L.nc_qk_norm_rope(X, 3, W, None, c_float(1e-6), None, 0, None, c_float(0.0), 0)
    eng.check()
    eng.backward_with(y, g)
    R.within(eng.grad(W), *R.qk_norm_rope_bwd64(x, 3, w, None, 1e-6, np.zeros((5, 0)), (), 1.0, False, g)["gwq"], "gw")
    Y = eng.param(x)
    y = L.nc_qk_norm_rope(Y, 1, None, None, c_float(1e-6), None, 0, None, c_float(0.0), 0)
    eng.backward_with(y, g)
    R.within(eng.grad(Y), *R.qk_norm_rope_bwd64(x, 1, None, None, 1e-6, np.zeros((5, 0)), (), 1.0, False, g)["gx"], "gx")


@pytest.mark.parametrize("same", ["", "kv", "qkv"])
def test_engine_attention(eng, same):
    """Autograd through views: head-major keys transposed back; one tensor as keys and values, or as all three."""
    L = eng.lib
    B, Lq, Lk, H, D = 2, 19, 19 if same == "qkv" else 37, 3, 48
    q, k, v, g, _ = attn_inputs((B, Lq, Lk, H, H, D, None), 23)
    lens = np.array([Lk, 6], np.int32)
    if same:
        v = k
    if same == "qkv":
        q = k
    kt = np.ascontiguousarray(k.transpose(0, 2, 1, 3))
    KT = eng.param(kt)
    kk = L.nc_transpose(KT, 1, 2)
    V = kk if same else eng.param(v)
    Q = kk if same == "qkv" else eng.param(q)
    n = eng.tensor(lens)
    o = L.nc_cross_attention(Q, kk, V, n, c_float(D ** -0.5))
    ref = R.attention64(q, k, v, lens, D ** -0.5, g)
    R.within(eng.read(o), *ref["o"], "o")
    eng.backward_with(o, g)
    parts = ["gk"] + (["gv"] if same else []) + (["gq"] if same == "qkv" else [])
    want, bound = (sum(ref[i][j] for i in parts) for j in (0, 1))
    R.within(eng.grad(KT), want.transpose(0, 2, 1, 3), (bound + 4 * R.U * np.abs(want)).transpose(0, 2, 1, 3), "gk")
    if not same:
        R.within(eng.grad(V), *ref["gv"], "gv")
    if same != "qkv":
        R.within(eng.grad(Q), *ref["gq"], "gq")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("same", ["qk", "qv", "qkv"])
def test_engine_one_tensor_twice(eng, same, D):
    """One tensor as queries and keys, queries and values, or all: its gradient is the sum, in both backward kernels."""
    L = eng.lib
    B, T, H = 2, 90, 2
    q, k, v, g, _ = attn_inputs((B, T, T, H, H, D, None), 27)
    k, v = (q if "k" in same else k), (q if "v" in same else v)
    ref = R.attention64(q, k, v, None, D ** -0.5, g)
    Q = eng.param(q)
    K_, V = Q if "k" in same else eng.param(k), Q if "v" in same else eng.param(v)
    want, bound = (sum(ref["g" + c][j] for c in same) for j in (0, 1))
    for times in (1, 2):
        eng.backward_with(L.nc_cross_attention(Q, K_, V, None, c_float(D ** -0.5)), g)
        R.within(eng.grad(Q), times * want, times * (bound + 4 * R.U * np.abs(want)), "g of " + same)
    for c, t in (("k", K_), ("v", V)):
        if c not in same:
            R.within(eng.grad(t), 2 * ref["g" + c][0], 3 * ref["g" + c][1], "g" + c)


def test_engine_refuses_an_output_written_since(eng):
    L = eng.lib
    q, k, v, g, _ = attn_inputs((1, 4, 6, 2, 2, 16, None), 24)
    Q, K_, V = eng.param(q), eng.param(k), eng.param(v)
    o = L.nc_cross_attention(Q, K_, V, None, c_float(0.25))
    loss = L.nc_sum(o, abi.ALL_AXES, 0)
    L.nc_copy_from(o, q.ctypes.data_as(ctypes.c_void_p), q.nbytes)
    assert L.nc_backward(loss) == abi.ERR_STATE and b"written after the forward" in L.nc_error(eng.ctx)
    L.nc_clear_error(eng.ctx)
    eng.step_end()


def test_engine_refuses_inputs_written_since(eng):
    L = eng.lib
    q, k, v, g, _ = attn_inputs((1, 4, 6, 2, 2, 16, None), 24)
    Q, K_, V = eng.param(q), eng.param(k), eng.param(v)
    loss = L.nc_sum(L.nc_cross_attention(Q, K_, V, None, c_float(0.25)), abi.ALL_AXES, 0)
    L.nc_copy_from(K_, k.ctypes.data_as(ctypes.c_void_p), k.nbytes)
    assert L.nc_backward(loss) == abi.ERR_STATE and b"written after the forward" in L.nc_error(eng.ctx)
    L.nc_clear_error(eng.ctx)
    eng.step_end()


def test_engine_gradcheck_of_the_block(lib):
    """A fused projection, the norm with positions, attention with shared heads and lengths, and a linear, against differences by
    the engine's own checker (eps 1e-2: differences of fp32 losses; the reference engine's bound of 2e-2)."""
    rng = np.random.default_rng(25)
    B, T, Hq, Hk, D, C = 2, 3, 2, 1, 4, 5
    e = Engine(lib=lib)
    L = e.lib
    x = e.param(rng.standard_normal((B, T, C)))
    wp = e.param(0.5 * rng.standard_normal(((Hq + 2 * Hk) * D, C)))
    wq, wk = e.param(1 + 0.2 * rng.standard_normal(D)), e.param(1 + 0.2 * rng.standard_normal(D))
    fixed = {"pos": np.arange(T, dtype=np.int32)[:, None].copy(), "n": np.array([T, 2], np.int32),
             "c": rng.standard_normal((B, T, Hq, D)).astype(np.float32)}
    fn_t = ctypes.CFUNCTYPE(ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p)

    def block(ctx, ins, user):
        nd, shp = abi.shape_arg((B, T, Hq + 2 * Hk, D))
        qkv = L.nc_reshape(L.nc_linear_fn(ins[0], ins[1], None), nd, shp)
        qk = L.nc_qk_norm_rope(L.nc_slice(qkv, 2, 0, Hq + Hk, 1), Hq, ins[2], ins[3], c_float(1e-2), e.tensor(fixed["pos"]), 1,
                               i64(D), c_float(10.0), 0)
        o = L.nc_cross_attention(L.nc_slice(qk, 2, 0, Hq, 1), L.nc_slice(qk, 2, Hq, Hk, 1), L.nc_slice(qkv, 2, Hq + Hk, Hk, 1),
                                 e.tensor(fixed["n"]), c_float(D ** -0.5))
        return L.nc_sum(L.nc_mul(o, e.tensor(fixed["c"])), abi.ALL_AXES, 0)

    ins = (ctypes.c_void_p * 4)(x, wp, wq, wk)
    cb = fn_t(block)
    worst = L.nc_gradcheck(e.ctx, ctypes.cast(cb, ctypes.c_void_p), ins, 4, None, c_float(1e-2))
    e.check()
    assert worst < 2e-2, worst
    e.close()


@pytest.mark.parametrize("flags", [0, abi.BACKWARD_RETAIN, abi.BACKWARD_FREE_GRAPH])
def test_engine_block_trains_without_new_memory(eng, flags):
    """Steps of the whole block after the first allocate nothing on the device and repeat its bits."""
    L = eng.lib
    rng = np.random.default_rng(26)
    B, T, S, H, D = 2, 40, 23, 2, 64
    x, s = rng.standard_normal((B, T, H * D)).astype(np.float32), rng.standard_normal((B, S, H * D)).astype(np.float32)
    wq, wk = eng.param(rng.standard_normal(D)), eng.param(rng.standard_normal(D))
    X, Sx = eng.param(x), eng.param(s)
    leaves, first, allocs = [X, Sx, wq, wk], None, None
    for step in range(3):
        for p in leaves:
            L.nc_zero_grad(p)
        shape = lambda n: abi.shape_arg((B, n, H, D))
        pos = eng.tensor(np.arange(T, dtype=np.int32)[:, None].copy())
        q = L.nc_qk_norm_rope(L.nc_reshape(X, *shape(T)), H, wq, None, c_float(1e-6), pos, 1, i64(D), c_float(1e4), 0)
        kv = L.nc_reshape(Sx, *shape(S))
        k = L.nc_qk_norm_rope(kv, 0, None, wk, c_float(1e-6), None, 0, None, c_float(0.0), 0)
        o = L.nc_cross_attention(q, k, kv, eng.tensor(np.array([S, 9], np.int32)), c_float(D ** -0.5))
        loss = L.nc_mean(L.nc_mul(o, o), abi.ALL_AXES, 0)
        eng.check()
        assert L.nc_backward_ex(loss, flags, None, 0) == 0, L.nc_error(eng.ctx)
        got = [eng.grad(p) for p in leaves]
        if step == 0:
            first = got
        elif step == 1:
            allocs = L.nc_device_alloc_count(eng.ctx)
        for a, b in zip(first, got):
            assert (a.view(np.uint32) == b.view(np.uint32)).all()
        eng.step_end()
    assert L.nc_device_alloc_count(eng.ctx) == allocs
