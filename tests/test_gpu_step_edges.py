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


@pytest.mark.parametrize("hd,keys,step", [(64, 128, 3.5), (128, 128, 3.5), (256, 64, 7.0)])
@pytest.mark.parametrize("counts", [[1], [20, 5], [70]])
def test_the_maximum_rises_where_o_leaves_tmem(hd, keys, step, counts):
    """Scores that rise by 2^7 from one key tile of a stream to its next (`step`
    doublings every `keys` keys), past the lag of 2^6: O is rescaled at every
    tile, those at which it has just left TMEM among them.  What O held before
    then weighs 2^-7, and V lies around 1, so an O that counts twice shows as
    0.8% of the result; the bound is below 0.3%."""
    a = make_attention(32, [1024] * len(counts), counts, 4, 1, hd, F32)
    a["q"] *= 0.25
    a["q"][..., 0] = math.sqrt(hd)                       # so that k[0] adds to the score as it is
    a["cv"] += 1
    for i in range(len(counts)):
        for p in range(1024 // P):
            a["ck"][a["tables"][i, p], :, :, 0] = p * P // keys * step * math.log(2.0)
    want, tol = ref_attention(a)
    assert float((tol / want.abs()).median()) < 3e-3
    close(call_attention(a), want, tol)


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("size", [1e-30, 1e-4, 0.01, 1e5, 1e30])
def test_f32_queries_of_any_size(hd, size):
    """q times `size` over a scale divided by it: the scores are what they were,
    and q keeps its 22 bits, far outside of f16's range too."""
    a = make_attention(33, [300, 40, 700], [3, 70, 1], 8, 2, hd, F32)
    a["q"] *= size
    close(call_attention(a, scale=hd ** -0.5 / size), *ref_attention(a, scale=hd ** -0.5 / size))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_f32_queries_of_many_sizes_in_a_call(hd):
    """Heads of large queries over small keys and the reverse, rows of zeros,
    and one element far above the others of its row; several runs in a CTA."""
    counts = [70, 1, 40, 130] * 5
    a = make_attention(34, [200] * 20, counts, 32, 8, hd, F32)
    for h in range(8):
        a["q"][:, 4 * h:4 * h + 4] *= 2.0 ** (3 * h - 9)
        a["ck"][:, h] *= 2.0 ** (9 - 3 * h)
    a["q"][::7] = 0
    a["q"][3::5, ::3, 11] = 3e5
    a["ck"][:, :, :, 11] = 0
    want, tol = ref_attention(a)
    # The row is scaled so that its largest value lies in [2^14, 2^15).  There the
    # first f16 word leaves at most 2^-11 of an element; the second holds that to
    # 2^-11 of it (22 bits, which ref_attention counts) or, where it falls among f16's
    # subnormals, to half of their step, 2^-25, which is at most 2^-39 of the largest.
    # A score is off by that times the sum of |k|, twice that moves the normaliser too.
    k = a["ck"].double().abs().sum(-1).amax(dim=(0, 2)).repeat_interleave(4)  # per head
    big = a["q"].double().abs().amax(-1)
    tol += (2 * 2.0 ** -39 * hd ** -0.5 * big * k * a["cv"].double().abs().max())[..., None]
    close(call_attention(a), want, tol)


def token(a, cache, i, t):
    """All heads of token t of request i in a cache."""
    return a[cache][a["tables"][i, t // P], :, t % P]


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 129])
def test_nothing_below_the_window_is_felt(qt, hd, window):
    """inf and NaN in K and V right below every row's window, and values of the
    largest size further below, leave the result as it is."""
    a = make_attention(35, [300, 515, 40], [3, 70, 1], 4, 2, hd, qt)
    want, tol = ref_attention(a, window)
    big = torch.finfo(a["ck"].dtype).max
    for i, n in enumerate(a["lengths"]):
        for t in range(n - window + 1):
            for c in ("ck", "cv"):
                token(a, c, i, t)[:] = (math.nan, math.inf, -math.inf, big, -big)[t % 5] if n - window - t < 40 else big
    close(call_attention(a, window), want, tol)
    close(call_attention(a, window, masked=False), *ref_attention(
        dict(a, ck=a["ck"].nan_to_num(0, 0, 0), cv=a["cv"].nan_to_num(0, 0, 0)), window, masked=False))


def spoil(a, window, masked, where):
    """Puts inf, -inf and NaN into single columns of V at the tokens `where`
    [(request, node)] and gives, from the definition, the outputs that are not
    finite then: a column of a row is the sum of what its row attends."""
    rows, heads, hd = a["q"].shape
    out = torch.zeros(rows, heads, hd, dtype=torch.float64, device="cuda")
    G = heads // a["cv"].shape[1]
    for n, (i, c) in enumerate(where):
        L, r0 = int(a["lengths"][i]), int(a["start"][i])
        d = (5 * n + 3) % hd
        bad = (math.inf, -math.inf, math.nan, math.inf)[n % 4]
        token(a, "cv", i, L + c)[:, d] = bad
        for j in range(int(a["start"][i + 1]) - r0):
            r = r0 + j
            if c < 0:
                see, at = True, L + c
            else:
                see = bool(a["mask"][r, c // 32] >> np.uint32(c % 32) & 1) if masked else c <= j
                at = a["pos"][r0 + c]
            if see and (window == 0 or at > a["pos"][r] - window):
                out[r, :, d] += bad
    return out


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("shape", ["trees", "chains", "window", "many", "long"])
def test_what_is_not_finite_stays_with_the_rows_that_attend_it(qt, hd, shape):
    """inf and NaN in V of drafted tokens, later tokens of a prompt and tokens that
    only some rows have in their window reach the rows that attend them, as the
    sum says, and no others: runs of one CTA, parts of several, pairs of query
    tiles and merged streams."""
    window, masked, where = 0, True, None
    if shape == "trees":
        a = make_attention(36, [40, 300, 0], [20, 70, 5], 8, 2, hd, qt)
        where = [(0, 3), (0, 17), (1, 2), (1, 40), (1, 69), (2, 4)]
    elif shape == "chains":
        a, masked = make_attention(37, [0, 130], [150, 90], 4, 1, hd, qt, tree="chain"), False
        where = [(0, 60), (0, 140), (1, 1), (1, 89)]
    elif shape == "window":
        a, window = make_attention(38, [200, 333], [40, 9], 4, 2, hd, qt, tree="chain"), 100
        where = [(0, -95), (0, -60), (1, -97), (1, -92), (0, 3)]
    elif shape == "many":  # more groups than SMs: whole ones, several to a CTA
        a = make_attention(39, [100 + 9 * i for i in range(40)], [1 + 7 * (i % 11) for i in range(40)], 16, 4, hd, qt)
        where = [(i, (3 * i) % (1 + 7 * (i % 11))) for i in range(0, 40, 3)]
    else:
        a = make_attention(40, [5000], [6], 8, 1, hd, qt)
        where = [(0, 2), (0, 5)]
    want, tol = ref_attention(a, window, masked)
    plus = spoil(a, window, masked, where)
    got = call_attention(a, window, masked)
    odd = ~plus.isfinite()
    assert 0 < int(odd.sum()) < odd.numel() // 4
    assert torch.equal(got[odd].double().nan_to_num(nan=7.0), plus[odd].nan_to_num(nan=7.0))
    close(got.masked_fill(odd, 0), want.masked_fill(odd, 0), tol)
    assert torch.equal(got.nan_to_num(nan=7.0), call_attention(a, window, masked).nan_to_num(nan=7.0))


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_scores_that_are_not_finite_show(qt, hd):
    """NaN in a query or in an attended key, and a score of inf, give NaN as the
    softmax does, and no zeros; -inf scores weigh nothing, a masked key's NaN too."""
    a = make_attention(41, [0, 70, 300], [4, 30, 1], 4, 2, hd, qt)
    a["q"][2, 1, 5] = math.nan                     # one row of one head
    token(a, "ck", 1, 70 + 4)[0, 7] = math.nan     # node 4 of request 1, KV head 0
    token(a, "ck", 2, 11)[1, 0] = math.inf         # all of request 2's rows, KV head 1: heads 2 and 3
    r = int(a["start"][2])
    a["q"][r, :, 0] = a["q"][r, :, 0].abs() + 1
    a["q"][r, 3, 0] *= -1                          # head 3: the score is -inf
    nan = torch.zeros(a["rows"], 4, dtype=torch.bool, device="cuda")
    nan[2, 1] = True
    for j in range(30):
        if a["mask"][4 + j, 0] >> np.uint32(4) & 1:
            nan[4 + j, :2] = True
    nan[r, 2] = True
    b = dict(a, q=a["q"].nan_to_num(0), ck=a["ck"].clone())
    token(b, "ck", 1, 74)[0, 7] = 0
    token(b, "ck", 2, 11)[1, 0] = torch.finfo(a["ck"].dtype).max  # head 3: a weight of 0 all the same
    want, tol = ref_attention(b)
    tol[r, 3] = tol[:r].amax()  # that score's size is none of the others'
    got = call_attention(a)
    assert torch.equal(got.isnan().all(-1), nan) and torch.equal(got.isnan().any(-1), nan)
    close(got.masked_fill(nan[..., None], 0), want.masked_fill(nan[..., None], 0), tol)


def test_engine_biases_that_close_on_the_gpu(tiny_models):
    """Biases of -inf, with and without a grammar, end or steer a request alike
    on the host and on the GPU."""
    from woolly_b200.engine import BatchEngine, GenerationConfig
    from woolly_b200.model import CudaTransformer
    shut = {t: -math.inf for t in range(0, 1000, 2)}
    cfgs = [GenerationConfig(max_tokens=8, eos_below=0, temperature=0.9, seed=3, logit_bias=shut),
            GenerationConfig(max_tokens=8, eos_below=0, logit_bias=shut, allowed=lambda t: range(len(t), 300)),
            GenerationConfig(max_tokens=8, eos_below=0, logit_bias=shut,
                             allowed=lambda t: [4, 6, 7] if len(t) < 3 else [4, 6]),
            GenerationConfig(max_tokens=8, eos_below=0)]
    runs = []
    for dev in (False, True):
        m = CudaTransformer(tiny_models["gqa_q4_0"], max_sessions=4, max_context=64, max_batch=4)
        eng = BatchEngine(m, device_sampling=dev)
        ids = [eng.submit([5, 6, 7 + i], c) for i, c in enumerate(cfgs)]
        eng.run()
        runs.append([(eng.finished[i].tokens, eng.finished[i].reason) for i in ids])
        eng.close()
        m.close()
    assert runs[0] == runs[1]
    assert all(t % 2 or t >= 1000 for toks, _ in runs[0][:3] for t in toks)
    assert runs[0][2] == ([7, 7, 7], "constraint") and len(runs[0][0][0]) == 8


@pytest.mark.parametrize("n", [1, 1024, 1025, 3000])
def test_block_tables_without_rows(n):
    """Nothing to place: the lengths stay, requests that wanted rows are told."""
    from woolly_b200 import STEP_NO_ROWS, STEP_OK
    counts = np.zeros(n, int)
    counts[-1] = 2
    t = torch.full((n, 3), -1, dtype=torch.int32, device="cuda")
    plan = ops.block_tables(t, i32(np.arange(n) % 40), i32(counts), i32([4, 5]), i32([2]), 0)
    assert plan.status.tolist() == [STEP_OK] * (n - 1) + [STEP_NO_ROWS]
    assert plan.lengths.tolist() == [i % 40 for i in range(n)] and plan.free_count.tolist() == [2]
    assert plan.row_start.tolist() == [0] * (n + 1) and (t == -1).all()
    assert plan.slots.numel() == plan.requests.numel() == plan.positions.numel() == 0


@pytest.mark.parametrize("qt", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_attention_in_place(qt, hd):
    """The output on the queries: whole groups, cut ones, several in a CTA."""
    for n, (lengths, counts, heads, kvh) in enumerate((([300, 20], [70, 3], 8, 2), ([4000], [5], 4, 1),
                                                       ([130] * 40, [9, 70] * 20, 16, 4))):
        a = make_attention(42 + n, lengths, counts, heads, kvh, hd, qt)
        want = call_attention(a)
        assert call_attention(a, out=a["q"]) is a["q"]
        assert torch.equal(a["q"], want)


def test_logits_beside_their_output():
    """Column ranges of one matrix, the output's on either side."""
    for ld, x0, y0 in ((20, 0, 10), (20, 10, 0), (33, 11, 23), (33, 20, 2)):
        m = torch.randn(6, ld, device="cuda")
        x, y = m[:, x0:x0 + 10], m[:, y0:y0 + 10]
        prm = ops.logit_params(6, 1.3, 0.5, 0.25)
        kw = dict(history=i32([1, 1, 2, 7]), history_start=i32([0, 4]), prompt_lens=i32([1]), requests=i32([0] * 6))
        want, rest = ops.process_logits(x.clone(), prm, **kw), m.clone()
        assert ops.process_logits(x, prm, out=y, **kw) is y
        rest[:, y0:y0 + 10] = want
        assert torch.equal(m, rest)


FIRST_CALLS = """
import sys, threading
sys.path.insert(0, "tests")
import torch
from test_gpu_step import BF16, F16, F32, call_attention, make_attention
from woolly_b200 import ops
N = 8
cases = [make_attention(50, [300, 20], [3, 40], 8, 2, hd, qt) for qt in (F32, F16, BF16) for hd in (64, 128, 256)]
logits = torch.randn(4, 51200, device="cuda")
torch.cuda.synchronize()
ready, got, errors = threading.Barrier(N), [None] * N, []

def caller(i):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            out = []
            for a in cases:
                ready.wait()
                out.append(call_attention(a))
            ready.wait()
            out.append(ops.sample(logits, 1.0, 0, 1.0, 0.5))
            torch.cuda.current_stream().synchronize()
        got[i] = out
    except BaseException as e:
        errors.append(e)
        ready.abort()

threads = [threading.Thread(target=caller, args=(i,)) for i in range(N)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not errors, errors
assert all(torch.equal(x, y) for g in got for x, y in zip(g, got[0]))
"""


def test_first_calls_of_many_threads():
    """Kernels that need their shared memory allowed first, from threads that
    come at the same time in a process that has not used them."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, timeout=300, capture_output=True, text=True,
                       env=dict(os.environ, PYTHONPATH=root))
    assert r.returncode == 0, r.stderr[-3000:]


@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 10 ** 12])
def test_windows_past_every_token(window):
    """A window beyond 32 bits is none, and not what is left of it."""
    a = make_attention(51, [300, 40], [3, 20], 4, 2, 64, F16)
    assert torch.equal(call_attention(a, window), call_attention(a))


@pytest.mark.parametrize("hd,repeats", [(64, 256), (128, 128), (256, 64)])
def test_f32_loses_what_32_products_lose(hd, repeats):
    """Tensor products cut sums off, towards zero: at the j-th of 32 that are added
    up in TMEM, up to 2^-23 of what is there, which is j/32 of O: 33/2 x 2^-23 of O
    together.  (Not half of that on average: each of a product's 16 terms is cut off
    at the sum's last place, not the sum alone.)  All other roundings are to nearest
    and cancel over 8,192 keys and hd columns; the last, 2^-24 at most, is counted
    all the same.  With V positive the mean of the relative error shows the loss; 64
    products lose twice as much."""
    a = make_attention(52, [8192], [1], 4, 1, hd, F32)
    a["q"] /= 4 * math.sqrt(hd / 64)
    a["cv"] = a["cv"].abs() + 0.5
    pages = a["tables"][0, :512]
    k, v = (c[torch.as_tensor(pages, device="cuda")][:, 0].reshape(-1, hd).double() for c in (a["ck"], a["cv"]))
    want = torch.softmax(a["q"][0].double() @ k.T / math.sqrt(hd), -1) @ v
    b = dict(a, tables=np.concatenate([np.tile(pages, repeats), [-1]])[None], lengths=np.array([8192 * repeats]),
             pos=np.array([8192 * repeats]), mask=np.zeros_like(a["mask"]))
    lost = ((want - call_attention(b)[0].double()) / want).mean().item()
    print(lost)
    assert -2.0 ** -24 <= lost <= 33 / 2 * 2.0 ** -23 + 2.0 ** -24
