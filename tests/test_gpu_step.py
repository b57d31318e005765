"""A serving step on a paged cache: block tables and slot maps, cache writes,
attention of drafted tokens and logit rules, against plain 64-bit restatements
of their definitions (include/woolly_cuda.h)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from woolly_b200 import (STEP_BAD_REQUEST, STEP_NO_PAGES, STEP_NO_ROWS, STEP_OK,  # noqa: E402
                         STEP_TABLE_FULL, WoollyError, ops)

P = ops.KV_PAGE
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def i32(a):
    return torch.from_numpy(np.asarray(a, dtype=np.int32).copy()).cuda()


def up(x):
    return -(-x // P)


# ------------------------------------------------------------------ block tables
def ref_plan(tables, lengths, counts, free, top, rows, parents=None, words=0):
    """The definition, request by request."""
    T = tables.copy()
    top = max(0, min(top, len(free)))
    at = want = 0
    start, page_start, taken = [], [], 0
    req, pos, slot = [np.full(rows, -1, np.int64) for _ in range(3)]
    mask = np.zeros((rows, max(words, 1)), np.uint32)
    out_len, status = [], []
    nf = top
    for i, (l, c) in enumerate(zip(map(int, lengths), map(int, counts))):
        first, at = at, at + max(c, 0)
        start.append(min(first, rows))
        page_start.append(taken)
        s = STEP_OK
        if l < 0 or c < 0 or (words and c > 32 * words):
            s = STEP_BAD_REQUEST
        elif l + c > T.shape[1] * P:
            s = STEP_TABLE_FULL
        elif at > rows:
            s = STEP_NO_ROWS
        else:
            need = up(l + c) - up(l)
            want += need
            if need and want > nf:
                s = STEP_NO_PAGES
            else:
                for k in range(up(l), up(l + c)):
                    top -= 1
                    taken += 1
                    T[i, k] = free[top]
        status.append(s)
        out_len.append(l + c if s == STEP_OK else l)
        paths = []
        for j in range(min(at, rows) - min(first, rows)):
            r = first + j
            req[r] = i
            if s != STEP_OK:
                continue
            path = [j]
            if parents is not None:
                u = int(parents[r])
                if u < -1 or u >= j or (u >= 0 and paths[u] is None):
                    path = None
                else:
                    path = (paths[u] if u >= 0 else []) + [j]
                paths.append(path)
                if path is None:
                    continue
                for b in path:
                    mask[r, b // 32] |= np.uint32(1 << (b % 32))
                pos[r] = l + len(path) - 1
            else:
                pos[r] = l + j
            page = T[i, (l + j) // P]
            if page >= 0:
                slot[r] = int(page) * P + (l + j) % P
    start.append(min(at, rows))
    page_start.append(taken)
    return dict(row_start=start, requests=req, positions=pos, slots=slot, lengths=out_len, status=status,
                free_count=[top], page_start=page_start, mask=mask.view(np.int32)), T


def make_step(rng, n, max_len, max_count, spare, pages=None):
    lengths = rng.integers(0, max_len + 1, n)
    counts = rng.integers(0, max_count + 1, n)
    pages = pages or up(max_len + max_count) + 1
    held = up(lengths)
    perm = rng.permutation(int(held.sum()) + spare)
    T = np.full((n, pages), -1, np.int32)
    o = 0
    for i in range(n):
        T[i, :held[i]] = perm[o:o + held[i]]
        o += held[i]
    return lengths, counts, T, perm[o:].astype(np.int32)


def check_plan(plan, want, words):
    for f in ("row_start", "requests", "positions", "slots", "lengths", "status", "free_count", "page_start"):
        assert np.array_equal(getattr(plan, f).cpu().numpy(), np.asarray(want[f])), f
    if words:
        assert np.array_equal(plan.mask.cpu().numpy(), want["mask"])


@pytest.mark.parametrize("n,max_len,max_count,spare,rows", [
    (1, 0, 1, 4, 1), (1, 40, 17, 5, 17), (5, 33, 3, 2, 15), (37, 100, 1, 40, 64), (64, 70, 40, 30, 700),
    (1000, 50, 9, 400, 8200), (1025, 64, 2, 5000, 1500), (2500, 40, 5, 900, 9000), (3, 20, 4000, 900, 9000),
])
def test_block_tables(n, max_len, max_count, spare, rows):
    rng = np.random.default_rng(n * 7 + rows)
    lengths, counts, T, free = make_step(rng, n, max_len, max_count, spare)
    want, wt = ref_plan(T, lengths, counts, free, len(free), rows)
    t, f = i32(T), i32(free)
    plan = ops.block_tables(t, i32(lengths), i32(counts), f, i32([len(free)]), rows)
    check_plan(plan, want, 0)
    assert np.array_equal(t.cpu().numpy(), wt)
    assert np.array_equal(f.cpu().numpy(), free)  # the stack itself is only read


@pytest.mark.parametrize("n,max_count,words,kind", [
    (1, 1, 1, "tree"), (3, 31, 1, "tree"), (4, 33, 2, "tree"), (20, 64, 2, "tree"), (2, 200, 7, "tree"),
    (2, 1024, 32, "chain"), (6, 40, 1, "tree"), (9, 30, 1, "bad"),
])
def test_block_tables_trees(n, max_count, words, kind):
    rng = np.random.default_rng(words * 100 + n)
    lengths, counts, T, free = make_step(rng, n, 60, max_count, n * up(max_count) + n)
    rows = int(counts.sum()) + 5
    parents = np.full(rows, -1)
    o = 0
    for c in counts:
        for j in range(c):
            parents[o + j] = j - 1 if kind == "chain" else rng.integers(-1, j) if j else -1
        o += c
    if kind == "bad":  # a node its own parent, later nodes, other negatives
        pick = rng.integers(0, o, 6)
        parents[pick] = [40, -2, 1 << 30, -(1 << 31), 31, 30]
    want, wt = ref_plan(T, lengths, counts, free, len(free), rows, parents, words)
    t = i32(T)
    plan = ops.block_tables(t, i32(lengths), i32(counts), i32(free), i32([len(free)]), rows,
                            parents=i32(parents), words=words)
    check_plan(plan, want, words)
    assert np.array_equal(t.cpu().numpy(), wt)


def test_block_tables_odd_requests():
    """Negative and oversized lengths and counts, a table without a page, a
    free count beyond the list and below zero."""
    lengths = [5, -1, 2147483647, 30, 16, 0, 47, 48, 3]
    counts = [3, 2, 1, -7, 2147483647, 0, 1, 1, 2]
    T = np.arange(27, dtype=np.int32).reshape(9, 3)
    T[8, 0] = -1
    free = np.array([100, 101, 102], np.int32)
    for top in (3, 9, 0, -4, 1):
        for rows in (0, 4, 9, 40):
            want, wt = ref_plan(T, lengths, counts, free, top, rows)
            t = i32(T)
            plan = ops.block_tables(t, i32(lengths), i32(counts), i32(free), i32([top]), rows)
            check_plan(plan, want, 0)
            assert np.array_equal(t.cpu().numpy(), wt)


def test_block_tables_no_requests_and_strided_table():
    e = i32([])
    plan = ops.block_tables(i32(np.zeros((0, 4))), e, e, i32([7]), i32([1]), 6)
    assert plan.row_start.tolist() == [0] and plan.free_count.tolist() == [1]
    assert plan.slots.tolist() == [-1] * 6 and plan.requests.tolist() == [-1] * 6
    big = torch.full((4, 9), -1, dtype=torch.int32, device="cuda")
    plan = ops.block_tables(big[:, :5], i32([0] * 4), i32([20] * 4), i32(range(8)), i32([8]), 80)
    assert plan.status.tolist() == [0] * 4
    assert big[:, :2].flatten().tolist() == [7, 6, 5, 4, 3, 2, 1, 0] and (big[:, 2:] == -1).all()


@pytest.mark.parametrize("n,max_len,max_count,spare", [(1, 0, 1, 1), (7, 40, 50, 30), (70, 300, 40, 150),
                                                       (1500, 60, 20, 3000)])
def test_release_takes_a_step_back(n, max_len, max_count, spare):
    rng = np.random.default_rng(n)
    lengths, counts, T, free = make_step(rng, n, max_len, max_count, spare)
    t, L, f, c = i32(T), i32(lengths), i32(free), i32([len(free)])
    rows = int(counts.sum())
    plan = ops.block_tables(t, L, i32(counts), f, c, rows)
    back = ops.release_pages(t, plan.lengths, L, f, plan.free_count)
    assert back.status.tolist() == [0] * n
    assert torch.equal(back.lengths, L) and back.free_count.item() == len(free)
    assert np.array_equal(t.cpu().numpy(), T) and np.array_equal(f.cpu().numpy(), free)


def test_release_parts_in_place():
    """Finished requests, kept prefixes, holes, a full stack, bad lengths; the
    outputs on the arguments themselves."""
    T = np.arange(40, dtype=np.int32).reshape(8, 5)
    T[3, 2] = -1
    lengths = np.array([80, 33, 17, 70, -3, 16, 81, 64])
    keep = np.array([0, 17, 90, 10, 0, -1, 5, 16])
    free = np.full(9, -7, np.int32)
    free[:1] = 99
    t, L, f, c = i32(T), i32(lengths), i32(free), i32([1])
    out = ops.Released(L, torch.empty_like(L), c, i32(np.zeros(9)))
    ops.release_pages(t, L, i32(keep), f, c, out=out)
    # request 0 gives 5 pages, 1 gives one; 7 would give 3 and only 2 slots are left
    assert out.status.tolist() == [0, 0, 0, STEP_TABLE_FULL, STEP_BAD_REQUEST, STEP_BAD_REQUEST,
                                   STEP_BAD_REQUEST, STEP_NO_PAGES]
    assert L.tolist() == [0, 17, 17, 70, -3, 16, 81, 64]
    assert c.item() == 7 and f.tolist() == [99, 7, 4, 3, 2, 1, 0, -7, -7]
    assert (t[0] == -1).all() and t[1].tolist() == [5, 6, -1, 8, 9] and t[7].tolist() == T[7].tolist()


@pytest.mark.parametrize("n,rows", [(40, 200), (40, 9000), (1300, 1500)])
def test_block_tables_in_place(n, rows):
    """The new lengths and the free count on the arguments themselves, step after step."""
    rng = np.random.default_rng(rows)
    _, _, T, free = make_step(rng, n, 0, 1, 60 * n, pages=40)
    t, f, L, c = i32(T), i32(free), i32(np.zeros(n)), i32([len(free)])
    lengths, top = np.zeros(n, np.int64), len(free)
    out = ops.step_plan(n, rows)._replace(lengths=L, free_count=c)
    for _ in range(4):
        counts = rng.integers(0, 30 if rows > 5000 else 4, n)
        want, T = ref_plan(T, lengths, counts, free, top, rows)
        ops.block_tables(t, L, i32(counts), f, c, rows, out=out)
        check_plan(out, want, 0)
        assert np.array_equal(t.cpu().numpy(), T)
        lengths, top = np.array(want["lengths"]), want["free_count"][0]


# ------------------------------------------------------------------ cache writes
@pytest.mark.parametrize("src,cache", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("rows,kvh,hd", [(1, 1, 8), (5, 3, 64), (70, 8, 128), (33, 2, 256), (300, 5, 40)])
def test_kv_append(src, cache, rows, kvh, hd):
    rng = np.random.default_rng(rows)
    g = torch.Generator("cuda").manual_seed(rows)
    pages = up(rows) + 3
    fused = torch.randn(rows, 3, kvh, hd, generator=g, device="cuda").to(src)
    k, v = fused[:, 1], fused[:, 2]  # strided rows of a fused projection
    slots = rng.permutation(pages * P)[:rows].astype(np.int64)
    if rows > 4:
        slots[[0, 2, 4]] = [-1, pages * P, -(1 << 31)]  # skipped
    ck = torch.randn(pages, kvh, P, hd, generator=g, device="cuda").to(cache)
    cv = torch.randn(pages, kvh, P, hd, generator=g, device="cuda").to(cache)
    wk, wv = ck.clone(), cv.clone()
    for r, s in enumerate(slots):
        if 0 <= s < pages * P:
            wk[s // P, :, s % P], wv[s // P, :, s % P] = k[r].to(cache), v[r].to(cache)
    ops.kv_append(k, v, i32(slots), ck, cv)
    assert torch.equal(ck, wk) and torch.equal(cv, wv)


@pytest.mark.parametrize("cache", [F16, BF16])
@pytest.mark.parametrize("kvh,hd", [(1, 8), (3, 64), (2, 128), (2, 256), (1, 1024)])
def test_kv_commit(cache, kvh, hd):
    rng = np.random.default_rng(hd)
    n, T = 6, 50
    lengths = np.array([0, 15, 16, 33, 7, 40])
    width = up(40 + T) + 1
    perm = rng.permutation(n * width)
    tables = perm.reshape(n, width)
    acc = [sorted(rng.choice(T, k, replace=False)) for k in (1, 0, 50, 20, 3, 9)]
    acc[4] = [0, 1, 49]
    start = np.concatenate([[0], np.cumsum([len(a) for a in acc])])
    ck = torch.randn(n * width, kvh, P, hd, device="cuda").to(cache)
    cv = torch.randn(n * width, kvh, P, hd, device="cuda").to(cache)
    wk, wv = ck.clone(), cv.clone()
    for i in range(n):
        for j, a in enumerate(acc[i]):
            f, t = lengths[i] + a, lengths[i] + j
            for w, c in ((wk, ck), (wv, cv)):
                w[tables[i, t // P], :, t % P] = c[tables[i, f // P], :, f % P]
    ops.kv_commit(i32(tables), i32(lengths), i32(np.concatenate([np.asarray(a, int) for a in acc])),
                  i32(start), ck, cv)
    assert torch.equal(ck, wk) and torch.equal(cv, wv)


def test_kv_commit_bad_tables():
    """Pages and nodes outside the cache are skipped."""
    ck, cv = (torch.randn(4, 2, P, 64, device="cuda").to(F16) for _ in range(2))
    wk = ck.clone()
    tables = i32([[0, -1], [9, 1], [2, 3]])
    acc = i32([3, 30, 1, 2, 1 << 30, 2])
    ops.kv_commit(tables, i32([0, 0, -5]), acc, i32([0, 2, 5, 99]), ck, cv)
    wk[0, :, 0] = ck[0, :, 3]  # request 0: node 3 of page 0; node 30 lies on no page
    assert torch.equal(ck, wk)


# ------------------------------------------------------------------ attention
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def make_attention(seed, lengths, counts, heads, kvh, hd, qt, tree="tree", extra=0):
    rng = np.random.default_rng(seed)
    g = torch.Generator("cuda").manual_seed(seed)
    lengths, counts = np.asarray(lengths), np.asarray(counts)
    n, rows = len(lengths), int(counts.sum())
    pages = up(lengths + counts)
    perm = rng.permutation(int(pages.sum()) + 2)
    tables = np.full((n, max(1, int(pages.max())) + 1), -1, np.int64)
    o = 0
    for i in range(n):
        tables[i, :pages[i]] = perm[o:o + pages[i]]
        o += pages[i]
    words = max(1, -(-int(counts.max()) // 32)) if n else 1
    mask = np.zeros((rows, words), np.uint32)
    pos = np.zeros(rows, np.int64)
    r = 0
    for i in range(n):
        for j in range(counts[i]):
            p = -1 if j == 0 else j - 1 if tree == "chain" else int(rng.integers(max(-1, j - 9), j))
            if p >= 0:
                mask[r + j] = mask[r + p]
            pos[r + j] = lengths[i] if p < 0 else pos[r + p] + 1
            mask[r + j, j // 32] |= np.uint32(1 << (j % 32))
        r += counts[i]
    ct = F16 if qt == F32 else qt
    shape = (len(perm), kvh, P, hd)
    return dict(q=(torch.randn(rows + extra, heads, hd, generator=g, device="cuda") * 2).to(qt),
                ck=torch.randn(shape, generator=g, device="cuda").to(ct),
                cv=torch.randn(shape, generator=g, device="cuda").to(ct), tables=tables, lengths=lengths,
                start=np.concatenate([[0], np.cumsum(counts)]), pos=pos, mask=mask, rows=rows)


def ref_attention(a, window=0, masked=True, scale=None):
    """Values in 64 bits and the bound of each output's error: half a step of
    the output's type; each probability rounded to the type it is multiplied
    in (two f16 words of f32 ones: 2^-22), and, as its exponent, the scores'
    error -- hd f32 additions of products whose sizes sum to S, f32 queries cut
    to 22 bits -- which also moves the normaliser; 2^-19 covers the exponential,
    the rescaling and the merging of parts."""
    q = a["q"].double()
    rows, heads, hd = q.shape
    kvh = a["ck"].shape[1]
    G = heads // kvh
    scale = hd ** -0.5 if scale is None else scale
    qt = a["q"].dtype
    hp = 2.0 ** -21 if qt == F32 else HALF[qt]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for i, L in enumerate(a["lengths"]):
        r0, r1 = a["start"][i], a["start"][i + 1]
        T = r1 - r0
        if T == 0:
            continue
        keys = int(L + T)
        page = a["tables"][i, np.arange(keys) // P]
        good = (page >= 0) & (page < a["ck"].shape[0])
        idx = torch.from_numpy(np.where(good, page, 0)).cuda()
        off = torch.arange(keys, device="cuda") % P
        K, V = a["ck"][idx, :, off].double(), a["cv"][idx, :, off].double()  # [keys, kvh, hd]
        V[~torch.from_numpy(good).cuda()] = 0
        see = np.zeros((T, keys), bool)
        for j in range(T):
            if a["pos"][r0 + j] < 0:
                continue
            see[j, :L] = True
            for c in range(T):
                bit = c <= j if not masked else (c // 32 < a["mask"].shape[1]
                                                 and a["mask"][r0 + j, c // 32] >> np.uint32(c % 32) & 1)
                see[j, L + c] = bool(bit)
            if window > 0:
                at = np.concatenate([np.arange(L), a["pos"][r0:r1]])
                see[j] &= at > a["pos"][r0 + j] - window
            see[j] &= good
        see = torch.from_numpy(see).cuda()
        for h in range(heads):
            k, v = K[:, h // G], V[:, h // G]
            x = q[r0:r1, h]
            s = (x @ k.T * scale).masked_fill(~see, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(m.isinf(), 0.0, m)), 0.0)
            l = p.sum(-1, keepdim=True)
            p = torch.where(l > 0, p / l, 0.0)
            o = p @ v
            S = (x.abs() @ k.abs().T * scale).masked_fill(~see, 0).amax(-1, keepdim=True)
            A = p @ v.abs()
            out[r0:r1, h] = o
            hq = 2.0 ** -21 if qt == F32 else 0.0
            tol[r0:r1, h] = (HALF[qt] * o.abs() + (hp + 2 * (hd * 2.0 ** -24 + hq) * S + 2.0 ** -19) * A) + 1e-30
    return out, tol


def call_attention(a, window=0, masked=True, out=None, **kw):
    return ops.tree_attention(a["q"], a["ck"], a["cv"], i32(a["tables"]), i32(a["lengths"]), i32(a["start"]),
                              i32(np.pad(a["pos"], (0, a["q"].shape[0] - a["rows"]))),
                              mask=i32(np.pad(a["mask"], ((0, a["q"].shape[0] - a["rows"]), (0, 0))).view(np.int32))
                              if masked else None, window=window, out=out, **kw)


def close(got, want, tol):
    assert not got.isnan().any()
    d = (got.double() - want).abs()
    bad = d > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((d / tol).max()):.3g} tol, " \
                          f"first at {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("heads,kvh", [(1, 1), (4, 4), (8, 2), (21, 3), (8, 1)])
def test_attention_heads(qt, hd, heads, kvh):
    a = make_attention(heads * hd, [0, 1, 15, 16, 100, 130], [1, 2, 17, 5, 3, 40], heads, kvh, hd, qt)
    close(call_attention(a), *ref_attention(a))


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("lengths,counts,heads,kvh", [
    ([1000], [1], 8, 8),                      # a single token
    ([5000], [1], 8, 1),
    ([0], [1], 2, 1),                         # nothing cached
    ([0, 0, 0], [0, 3, 0], 2, 1),             # requests without rows
    ([127, 128, 129, 255, 256, 257], [1] * 6, 4, 2),   # ends around a tile
    ([63, 64, 65, 111, 112, 113], [16, 17, 33, 1, 64, 65], 4, 1),
    ([777, 3], [300, 129], 4, 4),             # more rows than one tile of queries
    ([20, 4000, 9], [2, 3, 1], 8, 2),         # one long request among short ones
    (list(range(0, 600, 7)), [1 + i % 3 for i in range(86)], 4, 2),
])
def test_attention_lengths(qt, lengths, counts, heads, kvh):
    a = make_attention(len(lengths) + heads, lengths, counts, heads, kvh, 128, qt)
    close(call_attention(a), *ref_attention(a))


@pytest.mark.parametrize("qt", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000])
def test_attention_window(qt, hd, window):
    a = make_attention(window, [0, 30, 300, 515], [3, 20, 70, 1], 4, 2, hd, qt)
    close(call_attention(a, window), *ref_attention(a, window))


@pytest.mark.parametrize("qt", [F32, F16])
def test_attention_without_mask_is_a_chain(qt):
    a = make_attention(3, [40, 0, 200], [50, 260, 1], 4, 2, 64, qt, tree="chain")
    close(call_attention(a, masked=False), *ref_attention(a, masked=False))
    close(call_attention(a, 33, masked=False), *ref_attention(a, 33, masked=False))


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_rows_with_nothing_to_see(qt, hd):
    """Empty masks without a context, rows left out, padded rows behind the
    last request, infinities and NaN where nobody looks."""
    a = make_attention(11, [0, 40, 0, 90], [4, 6, 3, 20], 4, 2, hd, qt, extra=5)
    a["mask"][[1, 11]] = 0           # rows of the requests without cached tokens
    a["pos"][[5, 20]] = -1
    own = a["start"][3] + 7
    a["mask"][a["start"][3]:, 0] &= ~np.uint32(1 << 7)  # nobody sees node 7 of the last request
    t = a["lengths"][3] + 7
    for c, bad in ((a["ck"], math.nan), (a["cv"], math.nan)):
        c[a["tables"][3, t // P], :, t % P] = bad
        last = a["tables"][3, (a["lengths"][3] + 20 - 1) // P]  # the page's unused end
        if (a["lengths"][3] + 20) % P:
            c[last, :, (a["lengths"][3] + 20) % P:] = math.inf
    want, tol = ref_attention(dict(a, ck=a["ck"].nan_to_num(0, 0, 0), cv=a["cv"].nan_to_num(0, 0, 0)))
    out = torch.full_like(a["q"], 7.0)
    got = call_attention(a, out=out)
    close(got[:a["rows"]], want[:a["rows"]], tol[:a["rows"]])
    assert (got[a["rows"]:] == 7.0).all()
    for r in (1, 5, 11, 20):
        assert (got[r] == 0).all()
    assert own < a["rows"]


@pytest.mark.parametrize("qt", [F32, BF16])
def test_attention_bad_pages(qt):
    """Entries outside the cache hide their keys; a context past the table's
    end is cut there."""
    a = make_attention(5, [200, 300, 64], [5, 9, 2], 4, 1, 128, qt)
    a["tables"][0, 3] = -1
    a["tables"][0, 7] = a["ck"].shape[0]
    a["tables"][1, :4] = 1 << 30
    a["tables"][1, 18:] = -(1 << 31)
    a["tables"][2, :] = -5
    close(call_attention(a), *ref_attention(a))
    assert (call_attention(a)[14:] == 0).all()
    b = make_attention(6, [100, 20], [3, 3], 2, 1, 64, qt)
    b["tables"] = b["tables"][:, :4]
    cut = dict(b, tables=np.pad(b["tables"], ((0, 0), (0, 10)), constant_values=-1))
    close(call_attention(b), *ref_attention(cut))


def test_attention_strided_queries_scale_and_streams():
    a = make_attention(8, [50, 333], [7, 1], 8, 2, 128, F16)
    fused = torch.randn(8, 12, 128, device="cuda").to(F16)
    fused[:, 2:10] = a["q"]
    b = dict(a, q=fused[:, 2:10])
    want, tol = ref_attention(a, scale=0.3)
    close(call_attention(b, scale=0.3), want, tol)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call_attention(a, scale=0.3)
    torch.cuda.current_stream().wait_stream(s)
    close(got, want, tol)


def test_attention_extreme_scores():
    """Scores of +-2000 and queries of zeros."""
    a = make_attention(9, [400, 60], [5, 30], 4, 2, 128, F32)
    a["q"] *= 100
    a["q"][3] = 0
    close(call_attention(a), *ref_attention(a))


def test_attention_repeats_exactly():
    a = make_attention(10, [3000, 100, 700], [9, 40, 1], 8, 2, 128, F32)
    first = call_attention(a)
    for _ in range(3):
        assert torch.equal(first, call_attention(a))


@pytest.mark.parametrize("hd,repeats", [(64, 512), (128, 256), (256, 128)])
def test_attention_f32_keeps_its_precision_over_long_contexts(hd, repeats):
    """Tensor products cut their sums off: each addition loses up to 2^-23 of O,
    always towards zero.  No more than 64 may go by before O is added up with
    rounding, so the result is off by 64 x 2^-23 at most for those, whatever the
    context's length, and by 2^-20 for the words of q and P and the scores.  The
    context is 8,192 keys over and over, so its softmax is theirs."""
    a = make_attention(21, [8192], [1], 2, 1, hd, F32)
    a["q"] /= 4 * math.sqrt(hd / 64)
    pages = a["tables"][0, :512]
    k, v = (c[torch.as_tensor(pages, device="cuda")][:, 0].reshape(-1, hd).double() for c in (a["ck"], a["cv"]))
    want = torch.softmax(a["q"][0].double() @ k.T / math.sqrt(hd), -1) @ v
    # the row's own token is left out, so that the pages are all there is
    b = dict(a, tables=np.concatenate([np.tile(pages, repeats), [-1]])[None], lengths=np.array([8192 * repeats]),
             pos=np.array([8192 * repeats]), mask=np.zeros_like(a["mask"]))
    got = call_attention(b)[0].double()
    assert (got - want).norm() <= (64 * 2.0 ** -23 + 2.0 ** -20) * want.norm()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_f32_several_groups_per_cta(hd):
    """Whole groups, and both ends of cut ones, in one CTA, each long enough
    for O to leave TMEM on the way; single query tiles and pairs."""
    rng = np.random.default_rng(hd)
    counts = rng.choice([1, 5, 40, 70], 80)
    a = make_attention(22, rng.integers(900, 2500, 80), counts, 8, 4, hd, F32)
    close(call_attention(a), *ref_attention(a))


@pytest.mark.parametrize("qt", [F16, BF16])
@pytest.mark.parametrize("n,repeats", [(160, 4), (3, 400)])
def test_attention_16_bit_long_contexts(qt, n, repeats):
    """Requests over the same 8,192 keys, several times each: within a rounding
    of the result and of P, and 512 cut-off additions (512 x 2^-23 = 2^-14)."""
    hd, width = 64, 512 * repeats
    a = make_attention(23, [8192], [1], 2, 1, hd, qt)
    pages = a["tables"][0, :512]
    k, v = (c[torch.as_tensor(pages, device="cuda")][:, 0].reshape(-1, hd).double() for c in (a["ck"], a["cv"]))
    w = torch.softmax(a["q"][0].double() @ k.T / math.sqrt(hd), -1)
    want, size = w @ v, w @ v.abs()
    b = dict(a, tables=np.tile(np.concatenate([np.tile(pages, repeats), [-1]]), (n, 1)),
             lengths=np.full(n, 16 * width), start=np.arange(n + 1), pos=np.full(n, 16 * width),
             mask=np.zeros((n, 1), np.uint32), rows=n, q=a["q"].expand(n, 2, hd).contiguous())
    got = call_attention(b).double()
    tol = HALF[qt] * want.abs() + (HALF[qt] + 2.0 ** -14) * size
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("qt", [F32, BF16])
def test_attention_many_requests(qt):
    """More requests than a CTA has threads."""
    rng = np.random.default_rng(1)
    a = make_attention(12, rng.integers(0, 40, 1500), rng.integers(0, 3, 1500), 2, 1, 64, qt)
    close(call_attention(a), *ref_attention(a))


@pytest.mark.parametrize("hd", [32, 128])
def test_attention_small_positions_and_narrow_masks(hd):
    """Positions below the context's length count as it; nodes past the mask's
    width are seen by nobody."""
    a = make_attention(13, [70, 20], [40, 50], 2, 1, hd, F16)
    pos = a["pos"].copy()
    a["pos"] = np.where(np.arange(90) % 3 == 0, 5, pos)
    low = dict(a, pos=np.maximum(a["pos"], np.repeat([70, 20], [40, 50])))
    close(call_attention(a, 30), *ref_attention(low, 30))
    narrow = dict(a, pos=pos, mask=np.ascontiguousarray(a["mask"][:, :1]))
    close(call_attention(narrow), *ref_attention(narrow))


def test_attention_on_two_streams_at_once():
    a, b = (make_attention(s, [900, 40], [20, 3], 8, 2, 128, BF16) for s in (14, 15))
    wa, wb = ref_attention(a), ref_attention(b)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(6):
        with torch.cuda.stream(sa):
            got.append((call_attention(a), wa))
        with torch.cuda.stream(sb):
            got.append((call_attention(b), wb))
    torch.cuda.synchronize()
    for g, w in got:
        close(g, *w)


def test_a_cache_past_32_bit_offsets():
    """Pages whose elements lie beyond 2^32 bytes and 2^31 elements."""
    kvh, hd, pages = 8, 128, 139000  # 2.28e9 elements per cache
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("needs 10 GB")
    a = make_attention(16, [100, 33], [3, 20], 16, kvh, hd, F16)
    used = a["ck"].shape[0]
    big = [torch.empty(pages, kvh, P, hd, dtype=F16, device="cuda") for _ in range(2)]
    for x, small in zip(big, (a["ck"], a["cv"])):
        x[pages - used:] = small
    far = dict(a, ck=big[0], cv=big[1], tables=np.where(a["tables"] >= 0, a["tables"] + pages - used, -1))
    assert torch.equal(call_attention(far), call_attention(a))
    k, v = (torch.randn(2, kvh, hd, device="cuda") for _ in range(2))
    slots = i32([pages * P - 1, (pages - 1) * P])
    ops.kv_append(k, v, slots, *big)
    assert torch.equal(big[0][-1, :, 15], k[0].to(F16)) and torch.equal(big[1][-1, :, 0], v[1].to(F16))
    ops.kv_commit(i32([[pages - 1]]), i32([0]), i32([15]), i32([0, 1]), *big)
    assert torch.equal(big[0][-1, :, 0], k[0].to(F16))


# ------------------------------------------------------------------ logits
def ref_logits(x, rep, pres, freq, made, seen, bias, shut):
    x = x.double().cpu().numpy()
    with np.errstate(all="ignore"):
        y = np.where(seen, np.where(x > 0, x / rep[:, None], x * rep[:, None]), x)
        y = y - np.where(made > 0, freq[:, None] * made + pres[:, None], 0)
        y = y + bias
    y[shut] = -np.inf
    return y


def check_logits(got, want, x, rep, pres, freq, made, bias):
    """Each of the few f32 operations is off by half a step of a value no
    larger than the terms' sizes together; the result by half a step of its type."""
    size = np.abs(x.double().cpu().numpy()) * np.maximum(rep, 1 / rep)[:, None] + np.abs(bias) + \
        np.abs(freq)[:, None] * made + np.abs(pres)[:, None]
    tol = HALF[got.dtype] * np.abs(want) + 8 * HALF[F32] * size
    g = got.double().cpu().numpy()
    same = (g == want) | (np.isnan(g) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        ok = same | (np.abs(g - want) <= tol)
    assert ok.all(), np.argwhere(~ok)[:5]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("rows,V,hist", [(1, 1, 3), (3, 50, 20), (2, 33, 0), (5, 1000, 300), (4, 4096, 50),
                                         (3, 4097, 5000), (2, 32000, 700), (2, 100003, 900)])
def test_logits(dt, rows, V, hist):
    rng = np.random.default_rng(rows * V)
    n = 3
    hl = rng.integers(hist // 2, hist + 1, n)
    hs = np.concatenate([[0], np.cumsum(hl)])
    tok = np.minimum((V * rng.random(hs[-1]) ** 4).astype(int), V - 1)
    pl = rng.integers(0, hl + 1)
    req = rng.integers(-1, n, rows)
    rep, pres, freq = rng.uniform(0.5, 2, rows).astype("f"), rng.normal(0, 1, rows).astype("f"), \
        rng.normal(0, 0.3, rows).astype("f")
    nb = rng.integers(0, min(V, 40) + 1, rows)
    bs = np.concatenate([[0], np.cumsum(nb)])
    bt = rng.integers(0, V, bs[-1])          # now and then twice: the last entry holds
    bv = rng.normal(0, 5, bs[-1]).astype("f")
    W = -(-V // 32)
    masks = rng.integers(0, 2 ** 32, (3, W + 1), dtype=np.uint32)
    masks[2] = 0                              # a mask that leaves nothing
    arow = rng.integers(-1, 3, rows)
    x = torch.from_numpy(rng.normal(0, 4, (rows, V)).astype("f")).cuda().to(dt)
    made, seen, bias = np.zeros((rows, V)), np.zeros((rows, V), bool), np.zeros((rows, V))
    shut = np.zeros((rows, V), bool)
    for r in range(rows):
        if req[r] >= 0:
            h = tok[hs[req[r]]:hs[req[r] + 1]]
            np.add.at(made[r], h[pl[req[r]]:], 1)
            seen[r, h] = True
        for e in range(bs[r], bs[r + 1]):
            bias[r, bt[e]] = bv[e]
        if arow[r] >= 0:
            shut[r] = (masks[arow[r]][np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1 == 0
    want = ref_logits(x, rep, pres, freq, made, seen, bias, shut)
    prm = ops.logit_params(rows, rep, pres, freq, arow)
    kw = dict(history=i32(tok), history_start=i32(hs), prompt_lens=i32(pl), requests=i32(req),
              bias_start=i32(bs), bias_tokens=i32(bt), bias_values=torch.from_numpy(bv).cuda(),
              allowed=i32(masks.view(np.int32)))
    got = ops.process_logits(x, prm, **kw)
    check_logits(got, want, x, rep, pres, freq, made, bias)
    ops.process_logits(x, prm, out=x, **kw)   # in place
    assert torch.equal(x.view(torch.int16 if dt != F32 else torch.int32),
                       got.view(torch.int16 if dt != F32 else torch.int32))


def test_logits_drafts():
    """Tokens on a drafted row's path count as produced."""
    rng = np.random.default_rng(5)
    n, V, counts = 3, 700, np.array([4, 0, 40])
    rows = int(counts.sum()) + 2
    start = np.concatenate([[0], np.cumsum(counts)])
    req = np.concatenate([np.repeat(np.arange(n), counts), [-1, -1]])
    mask = np.zeros((rows, 2), np.uint32)
    for i in range(n):
        for j in range(counts[i]):
            r = start[i] + j
            if j:
                mask[r] = mask[start[i] + rng.integers(0, j)]
            mask[r, j // 32] |= np.uint32(1 << (j % 32))
    tok = rng.integers(0, 9, rows)  # the same ids over and over
    tok[3] = -4                     # ignored, as ids past the vocabulary
    hist, hs, pl = rng.integers(0, 12, 30), [0, 10, 10, 30], [4, 0, 30]
    hist[12] = V + 5
    x = torch.randn(rows, V, device="cuda")
    rep, pres, freq = np.full(rows, 1.3, "f"), np.full(rows, 0.25, "f"), np.full(rows, 0.5, "f")
    made, seen = np.zeros((rows, V)), np.zeros((rows, V), bool)
    for r in range(rows):
        if req[r] < 0:
            continue
        h = [t for t in hist[hs[req[r]]:hs[req[r] + 1]]]
        for q, t in enumerate(h):
            if 0 <= t < V:
                seen[r, t] = True
                made[r, t] += q >= pl[req[r]]
        for c in range(counts[req[r]]):
            t = tok[start[req[r]] + c]
            if mask[r, c // 32] >> np.uint32(c % 32) & 1 and t >= 0:
                made[r, t] += 1
                seen[r, t] = True
    got = ops.process_logits(x, ops.logit_params(rows, rep, pres, freq), history=i32(hist), history_start=i32(hs),
                             prompt_lens=i32(pl), requests=i32(req), draft_tokens=i32(tok),
                             draft_mask=i32(mask.view(np.int32)), row_start=i32(start))
    zero = np.zeros((rows, V))
    check_logits(got, ref_logits(x, rep, pres, freq, made, seen, zero, zero > 1), x, rep, pres, freq, made, zero)


def test_logits_infinities():
    """inf, -inf and NaN go through the rules; a masked place is -inf whatever it held."""
    x = torch.tensor([[math.inf, -math.inf, math.nan, 0.0, -0.0, 3.4e38, -3.4e38, 1.0]], device="cuda")
    x = x.repeat(2, 1)[:, :7]        # rows with a stride
    hist = i32([0, 1, 2, 3, 4, 5, 6])
    kw = dict(history=hist, history_start=i32([0, 7, 7]), requests=i32([0, 0]))
    got = ops.process_logits(x, ops.logit_params(2, 2.0, 0.5, 0.25, [-1, 0]), allowed=i32([[0b1110000]]), **kw)
    assert got[0, 0] == math.inf and got[0, 1] == -math.inf and got[0, 2].isnan()
    assert got[0, 3:7].tolist() == pytest.approx([-0.75, -0.75, 1.7e38, -math.inf])
    assert (got[1, :4] == -math.inf).all() and got[1, 4:].tolist() == got[0, 4:].tolist()


# ------------------------------------------------------------------ together
def run_step(t, q_of, k_of, v_of, logits_of, parents, tokens, prm, hist, cks, free, L):
    """One speculative step: plan, cache writes, attention of two layers,
    rules, greedy picks."""
    rows = parents.shape[0]
    plan = ops.block_tables(t, L, i32([rows - 6, 6]), free[0], free[1], rows, parents=parents, words=1)
    outs = []
    for layer, (ck, cv) in enumerate(cks):
        ops.kv_append(k_of[layer], v_of[layer], plan.slots, ck, cv)
        outs.append(ops.tree_attention(q_of[layer], ck, cv, t, L, plan.row_start, plan.positions, mask=plan.mask))
    y = ops.process_logits(logits_of, prm, history=hist[0], history_start=hist[1], prompt_lens=hist[2],
                           requests=plan.requests, draft_tokens=tokens, draft_mask=plan.mask,
                           row_start=plan.row_start)
    return plan, outs, y, ops.sample(y, 0.0, 0, 1.0, 0.0, params=torch.empty(rows * 16, dtype=torch.uint8, device="cuda"))


def test_a_speculative_step():
    """Drafts verified over the cache give what the same tokens give when each
    accepted path is run as a chain afterwards."""
    rng = np.random.default_rng(2)
    H, kvh, hd, V = 8, 2, 64, 500
    parents = np.array([-1, 0, 0, 1, 2, 4, 4, -1, 0, 1, 0, -1, 4])
    rows = len(parents)
    L = i32([37, 16])
    t = i32([[3, 0, 7, -1, -1], [5, -1, -1, -1, -1]])
    free = (i32([9, 8, 6, 4, 2, 1]), i32([6]))
    cks = [[torch.randn(10, kvh, P, hd, device="cuda").to(F16) for _ in range(2)] for _ in range(2)]
    q, k, v = ([torch.randn(rows, h, hd, device="cuda") for _ in range(2)] for h in (H, kvh, kvh))
    logits = torch.randn(rows, V, device="cuda")
    tokens = i32(rng.integers(0, V, rows))
    hist = (i32(rng.integers(0, V, 53)), i32([0, 37, 53]), i32([20, 16]))
    prm = ops.logit_params(rows, 1.2, 0.1, 0.2)
    plan, outs, y, picks = run_step(t, q, k, v, logits, i32(parents), tokens, prm, hist, cks, free, L)
    assert plan.status.tolist() == [0, 0]
    assert picks.shape == (rows,)
    # request 0 keeps nodes 0, 2, 4, 6; request 1 (rows 7..) keeps 0, 1, 2
    keep = [[0, 2, 4, 6], [0, 1, 2]]
    for layer, (ck, cv) in enumerate(cks):
        ops.kv_commit(t, L, i32(keep[0] + keep[1]), i32([0, 4, 7]), ck, cv)
        path = torch.tensor([0, 2, 4, 6, 7, 8, 9], device="cuda")
        chain = ops.tree_attention(q[layer][path].contiguous(), ck, cv, t, L, i32([0, 4, 7]),
                                   i32([37, 38, 39, 40, 16, 17, 18]))
        # the same keys in another order: a few f32 roundings apart
        torch.testing.assert_close(chain, outs[layer][path], rtol=1e-5, atol=1e-5)
    back = ops.release_pages(t, plan.lengths, L + i32([4, 3]), free[0], plan.free_count)
    assert back.lengths.tolist() == [41, 19] and back.status.tolist() == [0, 0]
    assert back.free_count.item() == 5  # request 1 holds one page more than before
    assert (t >= 0).sum().item() == 5


def test_a_captured_step():
    """The step captured in a graph and replayed on new lengths and drafts."""
    H, kvh, hd, V, rows = 4, 2, 128, 300, 12
    parents = i32([-1, 0, 1, 1, 0, 4, -1, 0, 0, 2, 1, 0])
    L = i32([30, 100])
    t = i32(np.arange(24).reshape(2, 12))
    free = (i32(np.arange(24, 40)), i32([16]))
    cks = [[torch.randn(40, kvh, P, hd, device="cuda").to(F16) for _ in range(2)] for _ in range(2)]
    q, k, v = ([torch.randn(rows, h, hd, device="cuda") for _ in range(2)] for h in (H, kvh, kvh))
    logits, tokens = torch.randn(rows, V, device="cuda"), i32(np.arange(rows))
    hist = (i32(np.arange(100)), i32([0, 50, 100]), i32([20, 50]))
    prm = ops.logit_params(rows, 1.2, 0.1, 0.2)

    def step():
        plan = ops.block_tables(t, L, i32_counts, free[0], free[1], rows, parents=parents, words=1)
        o = []
        for layer, (ck, cv) in enumerate(cks):
            ops.kv_append(k[layer], v[layer], plan.slots, ck, cv)
            o.append(ops.tree_attention(q[layer], ck, cv, t, L, plan.row_start, plan.positions, mask=plan.mask))
        y = ops.process_logits(logits, prm, history=hist[0], history_start=hist[1], prompt_lens=hist[2],
                               requests=plan.requests, draft_tokens=tokens, draft_mask=plan.mask,
                               row_start=plan.row_start)
        return [*plan, *o, y]

    i32_counts = i32([6, 6])
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = step()
    for a, b, par in (([30, 100], [6, 6], None), ([0, 17], [2, 10], [-1, 0, -1, 0, 1, 2, 3, 0, 0, 7, 2, 9]),
                      ([150, 150], [12, 0], [-1] * 12), ([5, 90], [3, 2], None)):
        L.copy_(i32(a))
        i32_counts.copy_(i32(b))
        if par:
            parents.copy_(i32(par))
        logits.normal_()
        for x in q:
            x.normal_()
        g.replay()
        got = [x.clone() for x in held]
        n = sum(b)
        want = step()
        for x, y in zip(got[:9], want[:9]):
            assert torch.equal(x, y)
        for x, y in zip(got[9:11], want[9:11]):
            assert torch.equal(x[:n], y[:n])
        assert torch.equal(got[11], want[11])


def test_engine_rules_on_the_gpu_match_the_host(tiny_models):
    """The batched engine with penalties, biases and a grammar gives the same
    tokens whether the rules and the sampling run on the GPU or on the host."""
    from woolly_b200.engine import BatchEngine, GenerationConfig
    from woolly_b200.model import CudaTransformer
    rng = np.random.default_rng(7)
    prompts = [rng.integers(3, 1024, n).tolist() for n in (5, 9, 3, 12)]
    cfgs = [GenerationConfig(max_tokens=9, eos_below=0, repetition_penalty=1.4, frequency_penalty=0.3),
            GenerationConfig(max_tokens=9, eos_below=0, temperature=0.9, top_k=30, seed=2,
                             logit_bias={t: float(b) for t, b in zip(range(3, 400, 7), rng.normal(0, 2, 57))}),
            GenerationConfig(max_tokens=9, eos_below=0),
            GenerationConfig(max_tokens=9, eos_below=0, temperature=0.7, seed=5, presence_penalty=0.5,
                             allowed=lambda t: range(len(t), 1000, 3) if len(t) < 7 else [])]
    runs = []
    for dev in (False, True):
        m = CudaTransformer(tiny_models["gqa_q4_0"], max_sessions=4, max_context=64, max_batch=4)
        eng = BatchEngine(m, device_sampling=dev)
        ids = [eng.submit(p, c) for p, c in zip(prompts, cfgs)]
        eng.run()
        runs.append([(eng.finished[i].tokens, eng.finished[i].reason) for i in ids])
        eng.close()
        m.close()
    assert runs[0] == runs[1]
    assert runs[0][3][1] == "constraint" and len(runs[0][3][0]) == 7
