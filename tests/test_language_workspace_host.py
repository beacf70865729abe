"""What workspace the vocabulary loss asks for: x and W packed, and beyond them no more than its limits say, at sizes far past what a
test can run."""
import ctypes

import pytest

from newch_amd import abi, hip

GiB = 1 << 30


@pytest.fixture()
def K():
    return hip.Kernels(ctypes.CDLL(str(abi.LIB_PATH)))


def up(n, m):
    return (n + m - 1) // m * m


SIZES = [(65536, 4096, 4000), (262144, 4096, 1000), (1 << 20, 4096, 300), (1 << 24, 64, 100), (524288, 256, 128000), (1 << 20, 2048, 128000),
         (8192, 2048, 128000), (8192, 16384, 128000), (300, 1 << 17, 513), (4096, 33, 1 << 21), (1, 1, 1)]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_workspace_in_pieces(K, size, monkeypatch):
    monkeypatch.setenv("NC_HIP_VOCAB_FORM", "split")
    N, D, V = size
    n, v, dk = up(N, 256), up(V, 256), up(D, 32)
    # packed operands; of every row its place, label, loss and power (20 bytes), of every word two powers
    fixed = 4 * dk * (n + v) + 20 * n + 8 * v
    score = K.linear_cross_entropy_workspace(N, D, V)
    # the statistics of 128 words each, and 36 bytes a row of a piece
    assert fixed <= score + 4 * v <= fixed + GiB // 2 + (64 << 20)
    full = K.linear_cross_entropy_workspace(N, D, V, gx=True, gw=True, gb=True)
    # z and its turned pieces; the parts of gx and of gW; statistics and sums of columns
    assert fixed <= full <= fixed + 4 * GiB + 2 * (GiB // 2) + (256 << 20)
    # gx's parts are the difference that gx makes
    parts = full - K.linear_cross_entropy_workspace(N, D, V, gw=True, gb=True)
    assert parts <= max(GiB // 2, 256 * up(D, 256) * 4)


@pytest.mark.parametrize("size", [(65536, 4096, 400), (1, 1, 1), (1 << 24, 64, 100), (64, 2048, 1 << 20), (300, 1 << 17, 513)], ids=str)
def test_workspace_of_fp32_products(K, size, monkeypatch):
    monkeypatch.setenv("NC_HIP_VOCAB_FORM", "fp32")
    N, D, V = size
    full = K.linear_cross_entropy_workspace(N, D, V, gx=True, gw=True, gb=True)
    assert full <= 4 * N * D + 8 * N + GiB + (192 << 20)  # x without the rows that do not count; losses; z; parts and statistics
