"""The vocabulary loss in pieces at sizes whose products are not cut (gW of 256 tiles and more), run on tiles of 256 columns (z, gW and
scoring) or have rows too long for the registers of the pack; stored and added, with pieces of the rows that are empty."""
import numpy as np
import pytest

from tests import language_ref as R
from tests.test_gpu_language import HALF, K, Loss, agree, lib, loss_inputs, rms  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def pieces(monkeypatch):
    monkeypatch.setenv("NC_HIP_VOCAB_FORM", "split")


def run(K, x, w, b, labels, ref, old=None, grads="xwb"):
    c = Loss(K, np.where(ref["on"][:, None], x, np.nan).astype(np.float32), w, b, labels, old=old, grads=grads)
    c.run()
    got = c.get()
    agree(got, ref, x, w, old=old)
    off = ~ref["on"]
    assert (got["rows"][off] == 0).all()
    if grads:
        assert (got["gx"][off] == (0 if old is None else old["gx"][off])).all()
    return got


# 329 tiles of gW, 256 columns wide; 256, 128 wide, with z's 256 wide; 282 where no row is whole 16 bytes; z 256 wide by 20 tiles
SHAPES = [(300, 770, 12001), (700, 386, 16130), (65, 701, 12004), (5100, 40, 5003)]


@pytest.mark.parametrize("ignored", [0.0, 0.3])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients_of_many_tiles(K, shape, ignored):
    x, w, b, labels = loss_inputs(*shape, 51, True, ignored)
    ref = R.vocab_loss(x, w, b, labels)
    old = {k: ref[k].astype(np.float32)[::-1].copy() for k in ("gx", "gw", "gb")}
    first = run(K, x, w, b, labels, ref)
    run(K, x, w, b, labels, ref, old=old)
    again = run(K, x, w, b, labels, ref)
    assert all((first[k].view(np.uint32) == again[k].view(np.uint32)).all() for k in ("gx", "gw", "gb")), "the same call twice"


# rows that count: 300 in pieces of 256 and 44; some 210 of them, which leave the second piece empty; 700 and 490 in three and two of three
@pytest.mark.parametrize("ignored", [0.0, 0.3])
@pytest.mark.parametrize("shape", [(300, 770, 12001), (700, 386, 16130)], ids=str)
def test_gradients_of_many_tiles_in_pieces(K, shape, ignored, monkeypatch):
    monkeypatch.setenv("NC_HIP_VOCAB_ROWS", "256")
    x, w, b, labels = loss_inputs(*shape, 52, True, ignored)
    ref = R.vocab_loss(x, w, b, labels)
    assert ignored == 0 or (ref["on"].sum() - 1) // 256 < (shape[0] - 1) // 256
    old = {k: ref[k].astype(np.float32)[::-1].copy() for k in ("gx", "gw", "gb")}
    for o in (None, old):
        run(K, x, w, b, labels, ref, old=o)


def test_many_tiles_and_no_row_counts(K):
    x, w, b, labels = loss_inputs(300, 770, 12001, 53, True, 0.0)
    labels[:] = -100
    old = {k: np.full(s, 0.75, np.float32) for k, s in (("gx", x.shape), ("gw", w.shape), ("gb", b.shape))}
    for o in (None, old):
        c = Loss(K, x * np.nan, w, b, labels, old=o)
        c.run()
        got = c.get()
        assert np.isnan(got["loss"]) and all((got[k] == (0 if o is None else 0.75)).all() for k in ("gx", "gw", "gb"))


@pytest.mark.parametrize("shape", [(40, 2331, 1027), (300, 2053, 513), (33, 4096, 300)], ids=str)
def test_rows_too_long_for_registers(K, shape):
    x, w, b, labels = loss_inputs(*shape, 54, True, 0.2)
    ref = R.vocab_loss(x, w, b, labels)
    run(K, x, w, b, labels, ref)


@pytest.mark.parametrize("shape", [(1000, 130, 12001), (5100, 40, 5003), (40, 2331, 1027)], ids=str)
def test_scored_on_wide_tiles(K, shape):
    x, w, b, labels = loss_inputs(*shape, 55, True, 0.2)
    run(K, x, w, b, labels, R.vocab_loss(x, w, b, labels), grads="")
