"""The embedding's gradient on the GPU to the roundings that its sums owe, term by term: few tokens eight at a time and then in fp64, sorted
ones in blocks of 8 or 32 that are added in fp64.  Gradients of one sign, so that partial sums are as large as they get."""
import numpy as np
import pytest

from tests import language_ref as R
from tests.test_gpu_language import HALF, K, Out, lib, up  # noqa: F401  (fixtures)
from newch_amd.hipmem import DeviceBuffer, synchronize

pytestmark = pytest.mark.gpu

# N, V, D and how many roundings of a sum no larger than the terms' sizes together: three of eight terms by pairs, or 7 or 31 one after
# the other; one of the fp64 sum; one of the product with the scale, or of that added to what was there
CASES = [(2560, 3, 64, 5), (512, 1, 2000, 5), (1024, 7, 33, 5), (2561, 300, 64, 9), (8193, 5, 4, 9), (20000, 7, 16, 33), (70000, 3, 5, 33),
         (40000, 1, 1, 33)]


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_embedding_gradient_roundings(K, case, accumulate):
    N, V, D, roundings = case
    rng = np.random.default_rng(N + D)
    tokens, g = rng.integers(0, V, N).astype(np.int32), rng.random((N, D), np.float32) + np.float32(0.5)
    old = rng.standard_normal((V, D)).astype(np.float32) * 100 if accumulate else np.zeros((V, D), np.float32)
    n = K.embedding_bwd_workspace(N, V, D)
    ws = DeviceBuffer.from_numpy(np.zeros(max(n, 16), np.uint8))
    gp, _g = up(g)
    tok, _t = up(tokens)
    gw = Out((V, D), fill=old if accumulate else np.nan)
    scale = np.float32(1.7)
    K.embedding_bwd(N, V, D, tok, -1, float(scale), gp, gw.ptr, ws.ptr, n, accumulate=accumulate)
    synchronize()
    ref, size = R.embedding_grad(tokens, g, V, np.float64(scale))
    # each rounding is off by HALF of what it rounds, which is off by those before it: below 33 HALF, so 1.00001 covers them
    assert (np.abs(gw.get() - (ref + old)) <= HALF * (roundings * 1.00001 * size + np.abs(ref + old))).all()
