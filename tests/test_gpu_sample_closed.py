"""wl_sample on rows in which a mask closed tokens: the same picks as the host's
rules, and never a closed token."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_sample_closed import NEAR, Draw, closed_rows  # noqa: E402

from woolly_b200 import ops  # noqa: E402
from woolly_b200.engine import GenerationConfig, sample_next_token  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("V,share", [(50, 0.1), (32000, 0.5), (32000, 0.0005), (51200, 0.9), (1000, 0.003)])
@pytest.mark.parametrize("kw", [dict(temperature=1.0), dict(temperature=0.7, top_p=0.9999999),
                                dict(temperature=0.0, top_p=0.9999999), dict(temperature=1.0, top_k=5, top_p=0.999),
                                dict(temperature=0.0)])
def test_a_closed_token_is_never_picked(V, share, kw):
    rows = 400
    x, shut = closed_rows(V, rows, V, share)
    rng = np.random.default_rng(1)
    u = rng.random(rows, dtype=np.float32)
    u[::4], u[1::4] = NEAR, 0.0
    got = ops.sample(torch.from_numpy(x).cuda(), kw["temperature"], kw.get("top_k", 0), kw.get("top_p", 1.0), u)
    got = got.cpu().numpy()
    assert not shut[np.arange(rows), got].any()
    if kw == dict(temperature=0.0):
        assert got.tolist() == x.argmax(1).tolist()


@pytest.mark.parametrize("V", [7, 32000])
def test_rows_that_leave_nothing(V):
    """Fallbacks are the host's: the last index without closed tokens, the last
    open one with them, whatever NaN and infinities do."""
    x = np.zeros((6, V), np.float32)
    x[1, V // 2:] = -np.inf
    x[2, 3] = np.nan
    x[3, 2] = np.inf
    x[3, -1] = -np.inf
    x[4] = -np.inf
    x[5, 1] = np.nan
    x[5, V - 3:] = -np.inf
    last = [V - 1, V // 2 - 1, V - 1, V - 2, V - 1, V - 4]
    for kw in (dict(temperature=0.0, top_p=0.99999994), dict(temperature=1.0, top_p=0.99999994)):
        got = ops.sample(torch.from_numpy(x).cuda(), kw["temperature"], 0, kw["top_p"], NEAR).tolist()
        with np.errstate(invalid="ignore"):
            host = [sample_next_token(r, GenerationConfig(**kw), Draw(NEAR)) for r in x]
        assert got[2:] == host[2:] == last[2:]
        for r in (0, 1):  # by the sums' rounding, some index that is open, or the last of them
            assert got[r] <= last[r] and host[r] <= last[r]
