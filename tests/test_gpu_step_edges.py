"""The serving-step operators at the edges of what a call may hold: runs of
different shape behind one another in a CTA, values that are not finite where a
row does not look, queries of any f32 magnitude, calls without rows."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_step import (BF16, F16, F32, P, call_attention, close, i32, make_attention,  # noqa: E402
                           ref_attention)

from woolly_b200 import ops  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_single_query_tiles_before_pairs(qt, hd):
    """More groups than SMs, so that a CTA has several: single query tiles over
    two key tiles and more, whose streams are merged through shared memory, and
    pairs, whose queries then take that place.  The calls repeat bit for bit."""
    counts = np.array([70, 1, 40, 130, 65, 3, 90, 64] * 4)  # 4 rows a token: pairs, singles and both
    lengths = np.random.default_rng(hd).integers(150, 420, counts.size)
    a = make_attention(31, lengths, counts, 32, 8, hd, qt)
    first = call_attention(a)
    close(first, *ref_attention(a))
    for _ in range(40):
        assert torch.equal(call_attention(a), first)
