"""Measured cases of the serving-step operators: block tables and slot maps,
writes into the paged KV cache, attention of drafted tokens over it, and the
rules applied to logits before sampling.

`run` computes one pass, in elementary torch operations (`own` false) or with
the package's operators (`own` true); `exact` restates each definition in 64
bits.  Pages hold 16 tokens and the cache is [page][kv head][16][head_dim], as
everywhere in the package.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 64 running requests, one token each: the smallest plan
        dict(name="tables_decode", op="tables", mode="decode", n=64, ctx=640, most=1, release=False,
             tight=False),
        # a speculative step: 32 requests with a tree of up to 64 drafted tokens each, whose
        # rejected part is given back to the pool behind it
        dict(name="tables_tree", op="tables", mode="tree", n=32, ctx=4096, most=64, release=True,
             tight=False),
        # prompts of up to 512 tokens of 1024 requests admitted at once, with a pool that runs out
        dict(name="tables_prompts", op="tables", mode="prompts", n=1024, ctx=300, most=512,
             release=False, tight=True),
        # K and V of one decode step of the 7B shape (32 KV heads of 128), 16 requests
        dict(name="cache_decode", op="cache", mode="append", n=16, most=1, ctx=640, kvh=32, hd=128,
             src="f32", cache="f16"),
        # 16 prompts of 512 tokens into a cache of 8 KV heads of 128
        dict(name="cache_prompts", op="cache", mode="append", n=16, most=512, ctx=1, kvh=8, hd=128,
             src="bf16", cache="bf16"),
        # drafted trees written, then the accepted paths moved together
        dict(name="cache_commit", op="cache", mode="commit", n=32, most=64, ctx=1000, kvh=8, hd=128,
             src="f32", cache="f16"),
        # one request of the 7B shape verifying five drafted tokens: the latency of a small call
        dict(name="attn_7b_bs1", op="attention", n=1, most=5, ctx=640, heads=32, kvh=32, hd=128,
             q="f32", cache="f16", window=0, tree=True),
        # 16 ragged requests with odd trees, 8 query heads per KV head of 64
        dict(name="attn_small_heads", op="attention", n=16, most=13, ctx=2048, heads=32, kvh=4, hd=64,
             q="f16", cache="f16", window=0, tree=True),
        # single tokens over long caches, 4 query heads per KV head
        dict(name="attn_long_single", op="attention", n=8, most=1, ctx=32768, heads=32, kvh=8, hd=128,
             q="f16", cache="f16", window=0, tree=False),
        # 32 requests of the 70B shape, trees of 64 tokens over 8192 tokens of context
        dict(name="attn_70b_bs32", op="attention", n=32, most=64, ctx=8192, heads=64, kvh=8, hd=128,
             q="bf16", cache="bf16", window=0, tree=True),
        # a decode step's 16 rows of 32,000 logits, every rule in use
        dict(name="logits_decode", op="logits", n=16, most=1, vocab=32000, hist=600, bias=40, masks=4,
             dtype="f32"),
        # the rows of 16 drafted trees over a large vocabulary and long histories
        dict(name="logits_tree", op="logits", n=16, most=32, vocab=128000, hist=4000, bias=300,
             masks=64, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "cache", "attention", "logits"])
    if op == "tables":
        mode = rng.choice(["decode", "tree", "prompts"])
        most = {"decode": 1, "tree": _log(rng, 2, 64), "prompts": _log(rng, 2, 1024)}[mode]
        n = min(_log(rng, 1, 1024), 524288 // most)
        return dict(op=op, mode=mode, n=n, ctx=_log(rng, 1, 8192), most=most,
                    release=rng.random() < 0.3, tight=rng.random() < 0.3)
    if op == "cache":
        kvh, hd = rng.choice([1, 2, 4, 8, 32]), rng.choice([64, 128, 256])
        src, cache = rng.choice([("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
        mode = rng.choice(["append", "commit"])
        most = _log(rng, 1, 512 if mode == "append" else 64)
        n = min(_log(rng, 1, 64), max(1, 8388608 // (most * kvh * hd)))
        return dict(op=op, mode=mode, n=n, most=most, ctx=_log(rng, 1, 2000), kvh=kvh, hd=hd, src=src,
                    cache=cache)
    if op == "attention":
        kvh, group = rng.choice([1, 2, 4, 8, 32]), rng.choice([1, 2, 3, 4, 7, 8])
        if kvh == 32:
            group = min(group, 2)
        hd = rng.choice([64, 128, 128, 128, 256])
        q, cache = rng.choice([("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
        tree = rng.random() < 0.75
        most = _log(rng, 1, 100) if tree else rng.choice([1, 1, 2, _log(rng, 2, 64)])
        n = _log(rng, 1, 32)
        # keys x rows and cache bytes stay under those of the largest listed case
        room = min(32 * 8192 * 64 * 64 * 128 // (n * most * kvh * group * hd),
                   32 * 8192 * 8 * 128 // (n * kvh * hd), 65536)
        ctx = _log(rng, 1, max(2, room))
        return dict(op=op, n=n, most=most, ctx=ctx, heads=kvh * group, kvh=kvh, hd=hd, q=q, cache=cache,
                    window=rng.choice([0, 0, 0, _log(rng, 4, 4096)]), tree=tree)
    vocab = _log(rng, 50, 152000)
    most = rng.choice([1, 1, _log(rng, 2, 64)])
    n = min(_log(rng, 1, 64), max(1, 65536000 // (vocab * most)))
    return dict(op=op, n=n, most=most, vocab=vocab, hist=_log(rng, 1, 4000),
                bias=min(vocab // 4, _log(rng, 1, 300)), masks=_log(rng, 1, 64),
                dtype=rng.choice(["f32", "f32", "f16", "bf16"]))


# ------------------------------------------------------------------ inputs
def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _i32(a):
    return _dev(np.asarray(a, dtype=np.int32))


def _trees(rng, counts):
    """Parents of the drafted tokens, packed: -1 for a child of the last cached
    token, else the index of an earlier node of the same request."""
    out = []
    for c in counts:
        j = np.arange(c)
        step = np.minimum(j, rng.integers(0, 4, size=c))  # a recent node, now and then the root
        p = j - 1 - step
        p[rng.random(c) < 0.1] = -1
        out.append(np.where(j == 0, -1, np.maximum(p, -1)))
    return np.concatenate(out).astype(np.int32) if out else np.zeros(0, np.int32)


def _depths(parents, counts):
    d, o = np.zeros(len(parents), np.int64), 0
    for c in counts:
        for j in range(c):
            p = parents[o + j]
            d[o + j] = 0 if p < 0 else d[o + p] + 1
        o += c
    return d


def _mask_words(parents, counts, words):
    """Bit c % 32 of word c // 32: node c is the row's own node or an ancestor."""
    m, o = np.zeros((len(parents), words), np.uint32), 0
    for c in counts:
        for j in range(c):
            p = parents[o + j]
            if p >= 0:
                m[o + j] = m[o + p]
            m[o + j, j // 32] |= np.uint32(1 << (j % 32))
        o += c
    return m.view(np.int32)


def _ragged(rng, n, ctx, lo, hi):
    """Context lengths around ctx and row counts in [lo, hi] of n requests: the
    sizes belong to the case (outputs keep their shapes), their order to the seed."""
    sizes = np.random.default_rng([n, ctx, lo, hi])
    lengths = sizes.integers(ctx // 2, ctx + ctx // 2 + 1, size=n)
    counts = sizes.integers(lo, hi + 1, size=n)
    order = rng.permutation(n)
    return lengths[order], counts[order]


def _prepare_tables(case, seed):
    rng = np.random.default_rng(seed)
    n, most = case["n"], case["most"]
    # a decode step and a batch of prompts have idle requests among theirs
    lengths, counts = _ragged(rng, n, case["ctx"], 1 if case["mode"] == "tree" else 0, most)
    rows = n * most if case["mode"] != "prompts" else max(1, int(0.6 * n * most))
    held = -(-lengths // PAGE)
    need = -(-(lengths + counts) // PAGE) - held
    max_pages = int((held + need).max()) + 2
    free = max(1, int(need.sum() * (0.8 if case["tight"] else 1.1)) + (0 if case["tight"] else n))
    pages = rng.permutation(int(held.sum()) + free).astype(np.int32)
    tables = np.full((n, max_pages), -1, np.int32)
    o = 0
    for i in range(n):
        tables[i, :held[i]] = pages[o:o + held[i]]
        o += held[i]
    st = dict(op="tables", case=case, rows=rows, tables=_dev(tables), lengths=_i32(lengths),
              counts=_i32(counts), free_pages=_dev(pages[o:]), free_count=_i32([free]), parents=None,
              words=0, depth=0, max_pages=max_pages)
    if case["mode"] == "tree":
        parents = np.full(rows, -1, np.int32)
        live = _trees(rng, counts)
        parents[:len(live)] = live
        st.update(parents=_dev(parents), words=-(-most // 32),
                  depth=int(_depths(live, counts).max()) + 1)
    if case["release"]:  # every draft is rejected: the requests keep their old tokens
        st["keep"] = st["lengths"]
    return st


def _step(rng, case):
    """Requests with their context, the pages of the context and of the step's rows."""
    n, most = case["n"], case["most"]
    lengths, counts = _ragged(rng, n, case["ctx"], (most + 1) // 2, most)
    pages = -(-(lengths + counts) // PAGE)
    perm = rng.permutation(int(pages.sum()) + 3).astype(np.int32)
    tables = np.full((n, int(pages.max()) + 1), -1, np.int32)
    o = 0
    for i in range(n):
        tables[i, :pages[i]] = perm[o:o + pages[i]]
        o += pages[i]
    start = np.concatenate([[0], np.cumsum(counts)])
    return lengths, counts, start, tables, len(perm)


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _fill_cache(gen, n_pages, kvh, hd, dtype):
    shape = (n_pages, kvh, PAGE, hd)
    return _randn(gen, shape, dtype), _randn(gen, shape, dtype)


def _prepare_cache(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    lengths, counts, start, tables, n_pages = _step(rng, case)
    slots = np.concatenate([[tables[i, p // PAGE] * PAGE + p % PAGE
                             for p in range(lengths[i], lengths[i] + counts[i])]
                            for i in range(case["n"])])
    pad = 3  # rows behind the last request, as a padded batch has them
    rows = len(slots) + pad
    ck, cv = _fill_cache(gen, n_pages, case["kvh"], case["hd"], DTYPES[case["cache"]])
    st = dict(op="cache", case=case, k=_randn(gen, (rows, case["kvh"], case["hd"]), DTYPES[case["src"]]),
              v=_randn(gen, (rows, case["kvh"], case["hd"]), DTYPES[case["src"]]),
              slots=_i32(np.concatenate([slots, [-1] * pad])), live=len(slots), cache_k=ck, cache_v=cv)
    if case["mode"] == "commit":
        acc, acc_start = [], [0]
        for c in counts:
            a = np.sort(rng.choice(c, size=min(int(c), 1 + int(rng.integers(0, 8))), replace=False))
            acc.append(a)
            acc_start.append(acc_start[-1] + len(a))
        st.update(accepted=_i32(np.concatenate(acc)), accepted_start=_i32(acc_start),
                  owner=_dev(np.repeat(np.arange(case["n"]), np.diff(acc_start))),
                  tables=_dev(tables), lengths=_i32(lengths))
    return st


def _prepare_attention(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    lengths, counts, start, tables, n_pages = _step(rng, case)
    rows, words = int(start[-1]), -(-case["most"] // 32)
    parents = _trees(rng, counts)
    if not case["tree"]:
        parents = np.concatenate([np.arange(c) - 1 for c in counts]).astype(np.int32)
    depth = _depths(parents, counts)
    ck, cv = _fill_cache(gen, n_pages, case["kvh"], case["hd"], DTYPES[case["cache"]])
    return dict(op="attention", case=case,
                # queries of trained models give scores of a few units' spread
                q=_randn(gen, (rows, case["heads"], case["hd"]), DTYPES[case["q"]], 2.0),
                cache_k=ck, cache_v=cv, tables=_dev(tables), lengths=_i32(lengths),
                row_start=_i32(start), positions=_i32(np.repeat(lengths, counts) + depth),
                mask=_dev(_mask_words(parents, counts, words)) if case["tree"] else None,
                host_lengths=[int(x) for x in lengths], host_start=[int(x) for x in start])


def _prepare_logits(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    n, V, most = case["n"], case["vocab"], case["most"]
    hist_len, counts = _ragged(rng, n, case["hist"], (most + 1) // 2, most)
    rows = int(counts.sum())
    hist_start = np.concatenate([[0], np.cumsum(hist_len)])
    # token frequencies fall off with rank, as in text
    tokens = np.minimum((V * rng.random(int(hist_len.sum())) ** 3).astype(np.int64), V - 1)
    nb = case["bias"]
    bias = np.concatenate([rng.choice(V, size=nb, replace=False) for _ in range(rows)])
    allowed = rng.integers(0, 2**32, size=(case["masks"], -(-V // 32)), dtype=np.uint32)
    allowed[::2] &= rng.integers(0, 2**32, size=allowed[::2].shape, dtype=np.uint32)
    allowed[:, 0] |= 1  # a token stays open in every mask
    st = dict(op="logits", case=case, logits=_randn(gen, (rows, V), DTYPES[case["dtype"]], 3.0),
              repetition=rng.uniform(0.9, 1.5, rows).astype(np.float32),
              presence=rng.uniform(-0.5, 1.5, rows).astype(np.float32),
              frequency=rng.uniform(-0.2, 0.8, rows).astype(np.float32),
              allowed_row=rng.integers(-1, case["masks"], rows).astype(np.int32),
              history=_i32(tokens), history_start=_i32(hist_start),
              prompt_lens=_i32(rng.integers(0, hist_len + 1)),
              requests=_i32(np.repeat(np.arange(n), counts)),
              bias_start=_i32(np.arange(rows + 1) * nb), bias_tokens=_i32(bias),
              bias_values=_dev(rng.normal(0, 4, rows * nb).astype(np.float32)),
              allowed=_dev(allowed.view(np.int32)), draft_tokens=None, draft_mask=None, row_start=None,
              host_start=[int(x) for x in hist_start], host_req=np.repeat(np.arange(n), counts))
    if most > 1:
        parents = _trees(rng, counts)
        st.update(draft_tokens=_i32(rng.integers(0, V, rows)), host_counts=counts,
                  draft_mask=_dev(_mask_words(parents, counts, -(-most // 32))),
                  row_start=_i32(np.concatenate([[0], np.cumsum(counts)])))
    return st


def prepare(case, seed):
    st = {"tables": _prepare_tables, "cache": _prepare_cache, "attention": _prepare_attention,
          "logits": _prepare_logits}[case["op"]](case, seed)
    if own:
        from woolly_b200 import ops
        if case["op"] == "logits":  # the requests' settings stay on the device between steps
            st["params"] = ops.logit_params(st["logits"].shape[0], repetition=st["repetition"],
                                            presence=st["presence"], frequency=st["frequency"],
                                            allowed_row=st["allowed_row"], device="cuda")
    else:
        if case["op"] == "logits":
            st["params"] = {k: _dev(st[k]) for k in ("repetition", "presence", "frequency", "allowed_row")}
    return st


# ------------------------------------------------------------------ the framework's calls
def _run_own(st):
    from woolly_b200 import ops
    op = st["op"]
    if op == "tables":
        plan = ops.block_tables(st["tables"], st["lengths"], st["counts"], st["free_pages"],
                                st["free_count"], st["rows"], parents=st["parents"], words=st["words"])
        out = dict(row_start=plan.row_start, requests=plan.requests, positions=plan.positions,
                   slots=plan.slots, lengths=plan.lengths, status=plan.status,
                   free_count=plan.free_count)
        if st["parents"] is not None:
            out["mask"] = plan.mask
        if "keep" in st:
            back = ops.release_pages(st["tables"], plan.lengths, st["keep"], st["free_pages"],
                                     plan.free_count)
            out.update(kept=back.lengths, kept_free=back.free_count, kept_status=back.status,
                       free_pages=st["free_pages"])
        out["tables"] = st["tables"]
        return out
    if op == "cache":
        ops.kv_append(st["k"], st["v"], st["slots"], st["cache_k"], st["cache_v"])
        if "accepted" in st:
            ops.kv_commit(st["tables"], st["lengths"], st["accepted"], st["accepted_start"],
                          st["cache_k"], st["cache_v"])
        return st["cache_k"], st["cache_v"]
    if op == "attention":
        return ops.tree_attention(st["q"], st["cache_k"], st["cache_v"], st["tables"], st["lengths"],
                                  st["row_start"], st["positions"], mask=st["mask"],
                                  window=st["case"]["window"])
    return ops.process_logits(st["logits"], st["params"], history=st["history"],
                              history_start=st["history_start"], prompt_lens=st["prompt_lens"],
                              requests=st["requests"], draft_tokens=st["draft_tokens"],
                              draft_mask=st["draft_mask"], row_start=st["row_start"],
                              bias_start=st["bias_start"], bias_tokens=st["bias_tokens"],
                              bias_values=st["bias_values"], allowed=st["allowed"])


# ------------------------------------------------------------------ plain forms
def _pages(tokens):
    return (tokens + (PAGE - 1)) // PAGE


def _plain_tables(st):
    tables, free = st["tables"], st["free_pages"]
    n, max_pages, rows = tables.shape[0], tables.shape[1], st["rows"]
    L, c = st["lengths"].long(), st["counts"].long()
    nf = st["free_count"].long().clamp(0, free.shape[0])
    e = c.clamp(min=0)
    end = torch.cumsum(e, 0)
    row_start = torch.cat([end.new_zeros(1), end]).clamp(max=rows)
    status = torch.where(end > rows, 3, 0)
    status = torch.where(L + c > max_pages * PAGE, 2, status)
    status = torch.where((L < 0) | (c < 0) | ((c > 32 * st["words"]) if st["words"] else (c < 0)), 4, status)
    need = torch.where(status == 0, _pages(L + c) - _pages(L), 0)
    upto = torch.cumsum(need, 0)
    status = torch.where((need > 0) & (upto > nf), 1, status)
    served = status == 0
    taken = torch.where(served, need, 0)
    first = torch.cumsum(taken, 0) - taken
    r = torch.arange(rows, device=tables.device)
    req = torch.searchsorted(row_start[1:].contiguous(), r, right=True)
    live = req < n
    i = req.clamp(max=n - 1)
    j = r - row_start[i]
    ok = live & served[i]
    p = L[i] + j
    # a page of the table, or one taken from the top of the free list
    idx = p // PAGE
    fresh = idx - _pages(L)[i]
    old = tables[i, idx.clamp(0, max_pages - 1)].long()
    new = free[(nf - 1 - first[i] - fresh).clamp(0, max(0, free.shape[0] - 1))].long()
    page = torch.where(fresh >= 0, new, old)
    grows = ok & (fresh >= 0)
    tables[i[grows], idx[grows]] = page[grows].int()
    position, good = p, ok
    out = {}
    if st["parents"] is not None:
        par = st["parents"].long()
        good = good & (par < j) & (par >= -1)
        node, bits = torch.where(good, j, -1), []
        member = torch.zeros((rows, 32 * st["words"]), dtype=torch.bool, device=tables.device)
        depth = torch.full_like(j, -1)
        base = row_start[i]
        for _ in range(st["depth"]):
            on = node >= 0
            member[r[on], node[on]] = True
            depth = depth + on
            node = torch.where(on, par[(base + node).clamp(0, rows - 1)], -1)
        position = L[i] + depth
        w = member.view(rows, st["words"], 32).long() << torch.arange(32, device=tables.device)
        out["mask"] = w.sum(-1).to(torch.int32)
    out.update(row_start=row_start.int(), requests=torch.where(live, req, -1).int(),
               positions=torch.where(good, position, -1).int(),
               slots=torch.where(good & (page >= 0), page * PAGE + p % PAGE, -1).int(),
               lengths=torch.where(served, L + c, L).int(), status=status.int(),
               free_count=(nf - taken.sum()).int())
    if "keep" in st:
        back = _plain_release(tables, out["lengths"], st["keep"], free, out["free_count"])
        out.update(kept=back[0], kept_free=back[1], kept_status=back[2], free_pages=free)
    out["tables"] = tables
    return out


def _plain_release(tables, lengths, keep, free, count):
    n, max_pages = tables.shape
    L, nf = lengths.long(), count.long()
    k = torch.minimum(keep.long(), L)
    col = torch.arange(max_pages, device=tables.device)
    gone = (col >= _pages(k)[:, None]) & (col < _pages(L)[:, None])
    bad = (L < 0) | (k < 0) | (L > max_pages * PAGE)
    status = torch.where(bad, 4, torch.where((gone & (tables < 0)).any(1), 2, 0))
    upto = torch.cumsum(torch.where(status == 0, gone.sum(1), 0), 0)
    status = torch.where((status == 0) & (gone.sum(1) > 0) & (upto > free.shape[0] - nf), 1, status)
    gone = gone & (status == 0)[:, None]
    total = gone.sum()
    g = torch.cumsum(gone.flatten().long(), 0).view_as(gone) - 1
    free[(nf + total - 1 - g)[gone]] = tables[gone]
    tables[gone] = -1
    return torch.where(status == 0, k, L).int(), (nf + total).int(), status.int()


def _plain_cache(st):
    ck, cv = st["cache_k"], st["cache_v"]
    s = st["slots"][:st["live"]].long()
    ck[s // PAGE, :, s % PAGE] = st["k"][:st["live"]].float().to(ck.dtype)
    cv[s // PAGE, :, s % PAGE] = st["v"][:st["live"]].float().to(cv.dtype)
    if "accepted" in st:
        i, a = st["owner"], st["accepted"].long()
        L = st["lengths"].long()[i]
        src = L + a
        dst = L + torch.arange(a.shape[0], device=a.device) - st["accepted_start"].long()[i]
        sp, dp = st["tables"][i, src // PAGE].long(), st["tables"][i, dst // PAGE].long()
        ck[dp, :, dst % PAGE] = ck[sp, :, src % PAGE]
        cv[dp, :, dst % PAGE] = cv[sp, :, src % PAGE]
    return ck, cv


def _plain_attention(st):
    case, q = st["case"], st["q"]
    kvh, hd, group = case["kvh"], case["hd"], case["heads"] // case["kvh"]
    out = torch.empty_like(q)
    for i, L in enumerate(st["host_lengths"]):
        r0, r1 = st["host_start"][i], st["host_start"][i + 1]
        T = r1 - r0
        keys = L + T
        pages = st["tables"][i, :-(-keys // PAGE)].long()
        K = st["cache_k"][pages].float().transpose(0, 1).reshape(kvh, -1, hd)[:, :keys]
        V = st["cache_v"][pages].float().transpose(0, 1).reshape(kvh, -1, hd)[:, :keys]
        x = q[r0:r1].float().view(T, kvh, group, hd).permute(1, 2, 0, 3).reshape(kvh, group * T, hd)
        node = torch.arange(T, device=q.device)
        if st["mask"] is None:
            seen = node[None, :] <= node[:, None]
        else:
            seen = (st["mask"][r0:r1][:, node // 32] >> (node % 32)) & 1 == 1
        pos = st["positions"][r0:r1]
        where = torch.cat([torch.arange(L, device=q.device, dtype=pos.dtype), pos])
        open_ = torch.cat([seen.new_ones(T, L), seen], 1)
        if case["window"] > 0:
            open_ = open_ & (where[None, :] > pos[:, None] - case["window"])
        s = (x @ K.transpose(1, 2)).view(kvh, group, T, keys) * hd ** -0.5
        s = s.masked_fill(~open_, -math.inf)
        e = torch.exp(s - s.amax(-1, keepdim=True))
        o = (e / e.sum(-1, keepdim=True)).view(kvh, group * T, keys) @ V
        out[r0:r1] = o.view(kvh, group, T, hd).permute(2, 0, 1, 3).reshape(T, -1, hd).to(q.dtype)
    return out


def _plain_logits(st):
    x = st["logits"].float()
    rows, V = x.shape
    p, dev = st["params"], x.device
    made = torch.zeros((rows, V), dtype=torch.float32, device=dev)
    seen = torch.zeros((rows, V), dtype=torch.bool, device=dev)
    req = st["requests"].long()
    h = st["history"].long()
    hs = st["history_start"].long()
    owner = torch.searchsorted(hs[1:].contiguous(), torch.arange(h.shape[0], device=dev), right=True)
    is_out = torch.arange(h.shape[0], device=dev) - hs[owner] >= st["prompt_lens"].long()[owner]
    n = st["case"]["n"]
    base = torch.zeros((n, V), dtype=torch.float32, device=dev)
    base.index_put_((owner[is_out], h[is_out]), torch.ones(1, device=dev), accumulate=True)
    have = torch.zeros((n, V), dtype=torch.bool, device=dev)
    have[owner, h] = True
    made += base[req]
    seen |= have[req]
    if st["draft_tokens"] is not None:
        m = st["draft_mask"]
        nodes = torch.arange(32 * m.shape[1], device=dev)
        on = (m[:, nodes // 32] >> (nodes % 32)) & 1 == 1
        r, node = on.nonzero(as_tuple=True)
        tok = st["draft_tokens"].long()[st["row_start"].long()[req[r]] + node]
        made.index_put_((r, tok), torch.ones(1, device=dev), accumulate=True)
        seen[r, tok] = True
    rep = p["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - p["frequency"][:, None] * made
    x = x - p["presence"][:, None] * (made > 0)
    b0 = st["bias_start"].long()
    r = torch.searchsorted(b0[1:].contiguous(), torch.arange(st["bias_tokens"].shape[0], device=dev),
                           right=True)
    x.index_put_((r, st["bias_tokens"].long()), st["bias_values"], accumulate=True)
    a = st["allowed"][p["allowed_row"].clamp(min=0).long()]
    v = torch.arange(V, device=dev)
    shut = ((a[:, v // 32] >> (v % 32)) & 1 == 0) & (p["allowed_row"] >= 0)[:, None]
    return x.masked_fill(shut, -math.inf).to(st["logits"].dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"tables": _plain_tables, "cache": _plain_cache, "attention": _plain_attention,
            "logits": _plain_logits}[state["op"]](state)


# ------------------------------------------------------------------ the definitions in 64 bits
def _up(x):
    return -(-x // PAGE)


def _exact_tables(st):
    T = st["tables"].cpu().numpy().copy()
    L, C = st["lengths"].tolist(), st["counts"].tolist()
    free, nf = st["free_pages"].tolist(), int(st["free_count"][0])
    rows, limit, words = st["rows"], T.shape[1] * PAGE, st["words"]
    par = None if st["parents"] is None else st["parents"].tolist()
    starts, at, want, top = [0], 0, 0, nf
    req, pos, slot = [-1] * rows, [-1] * rows, [-1] * rows
    mask = np.zeros((rows, max(words, 1)), np.uint32)
    new_len, status = [], []
    for i, (l, c) in enumerate(zip(L, C)):
        first, at = at, at + max(c, 0)
        starts.append(min(at, rows))
        if l < 0 or c < 0 or (words and c > 32 * words):
            s = 4
        elif l + c > limit:
            s = 2
        elif at > rows:
            s = 3
        else:
            s, need = 0, _up(l + c) - _up(l)
            want += need
            if need and want > nf:
                s = 1
        if s == 0:
            for k in range(_up(l), _up(l + c)):
                top -= 1
                T[i, k] = free[top]
        status.append(s)
        new_len.append(l + c if s == 0 else l)
        chain, depth = [], []
        for j in range(min(at, rows) - min(first, rows)):
            req[first + j] = i
            if s:
                continue
            p, ok = l + j, True
            if par is None:
                pos[first + j] = p
            else:
                up = par[first + j]
                ok = -1 <= up < j and (up < 0 or chain[up] is not None)
                mine = None
                if ok:
                    mine = ([] if up < 0 else chain[up]) + [j]
                    pos[first + j] = l + len(mine) - 1
                    for b in mine:
                        mask[first + j, b // 32] |= np.uint32(1 << (b % 32))
                chain.append(mine)
            if ok and T[i, p // PAGE] >= 0:
                slot[first + j] = int(T[i, p // PAGE]) * PAGE + p % PAGE
    out = {} if par is None else dict(mask=_dev(mask.view(np.int32)))
    out.update(row_start=_i32(starts), requests=_i32(req), positions=_i32(pos), slots=_i32(slot),
               lengths=_i32(new_len), status=_i32(status), free_count=_i32([top]))
    if "keep" in st:
        stack, order, kept, flag = free[:], [], [], []
        for i, (l, k) in enumerate(zip(new_len, st["keep"].tolist())):
            cols = list(range(_up(min(k, l)), _up(l)))
            bad = 2 if any(T[i, x] < 0 for x in cols) else 0
            if bad == 0 and cols and len(order) + len(cols) > len(stack) - top:
                bad = 1
            if bad == 0:
                order += [(i, x) for x in cols]
            kept.append(min(k, l) if bad == 0 else l)
            flag.append(bad)
        for g, (i, x) in enumerate(order):
            stack[top + len(order) - 1 - g] = int(T[i, x])
            T[i, x] = -1
        out.update(kept=_i32(kept), kept_free=_i32([top + len(order)]), kept_status=_i32(flag),
                   free_pages=_i32(stack))
    out["tables"] = _dev(T)
    return out


def _exact_cache(st):
    out = []
    slots = st["slots"].tolist()
    for src, cache in ((st["k"], st["cache_k"]), (st["v"], st["cache_v"])):
        c = cache.double().transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3]).clone()
        live = [r for r, s in enumerate(slots) if s >= 0]
        c[torch.tensor([slots[r] for r in live], device=c.device)] = src[live].double()
        if "accepted" in st:
            was = c.clone()
            a, a0 = st["accepted"].tolist(), st["accepted_start"].tolist()
            T, L = st["tables"].tolist(), st["lengths"].tolist()
            frm, to = [], []
            for i in range(len(L)):
                for d, node in enumerate(a[a0[i]:a0[i + 1]]):
                    f, t = L[i] + node, L[i] + d
                    frm.append(T[i][f // PAGE] * PAGE + f % PAGE)
                    to.append(T[i][t // PAGE] * PAGE + t % PAGE)
            c[torch.tensor(to, device=c.device)] = was[torch.tensor(frm, device=c.device)]
        out.append(c.view(-1, PAGE, cache.shape[1], cache.shape[3]).transpose(1, 2).contiguous())
    return tuple(out)


def _exact_attention(st):
    case = st["case"]
    kvh, hd, W = case["kvh"], case["hd"], case["window"]
    group = case["heads"] // kvh
    q = st["q"].double()
    out = torch.zeros_like(q)
    for i, L in enumerate(st["host_lengths"]):
        r0, r1 = st["host_start"][i], st["host_start"][i + 1]
        T = r1 - r0
        t = torch.arange(L + T, device=q.device)
        page, off = st["tables"][i].long()[t // PAGE], t % PAGE
        pos = st["positions"][r0:r1].long()
        key_pos = torch.cat([t[:L], pos])
        see = torch.ones(T, L + T, dtype=torch.bool, device=q.device)
        for j in range(T):
            if st["mask"] is None:
                see[j, L + j + 1:] = False
            else:
                w = st["mask"][r0 + j].tolist()
                see[j, L:] = torch.tensor([(w[c // 32] >> (c % 32)) & 1 for c in range(T)],
                                          device=q.device) == 1
            if W > 0:
                see[j] &= key_pos > pos[j] - W
        for h in range(kvh):
            K, V = st["cache_k"][page, h, off].double(), st["cache_v"][page, h, off].double()
            for g in range(group):
                s = torch.einsum("td,kd->tk", q[r0:r1, h * group + g], K) / math.sqrt(hd)
                s[~see] = -math.inf
                p = torch.softmax(s, -1)
                out[r0:r1, h * group + g] = torch.einsum("tk,kd->td", p, V)
    return out


def _exact_logits(st):
    x = st["logits"].double()
    out = torch.empty_like(x)
    V, h, hs = x.shape[1], st["history"].long(), st["host_start"]
    pl = st["prompt_lens"].tolist()
    bs, bt, bv = st["bias_start"].tolist(), st["bias_tokens"].long(), st["bias_values"].double()
    words = None if st["draft_mask"] is None else st["draft_mask"].tolist()
    first = None if words is None else st["row_start"].tolist()
    for r in range(x.shape[0]):
        i = int(st["host_req"][r])
        h0, h1 = hs[i], hs[i + 1]
        made = torch.bincount(h[h0 + pl[i]:h1], minlength=V).double()
        seen = torch.bincount(h[h0:h1], minlength=V) > 0
        if words is not None:
            for c in range(32 * len(words[r])):
                if (words[r][c // 32] >> (c % 32)) & 1:
                    made[st["draft_tokens"][first[i] + c].long()] += 1
        seen = seen | (made > 0)
        y = x[r].clone()
        rep = float(st["repetition"][r])
        y[seen & (x[r] > 0)] /= rep
        y[seen & (x[r] <= 0)] *= rep
        y -= float(st["frequency"][r]) * made + float(st["presence"][r]) * (made > 0).double()
        y[bt[bs[r]:bs[r + 1]]] += bv[bs[r]:bs[r + 1]]
        a = int(st["allowed_row"][r])
        if a >= 0:
            bits = st["allowed"][a].long().repeat_interleave(32)[:V]
            y[(bits >> (torch.arange(V, device=x.device) % 32)) & 1 == 0] = -math.inf
        out[r] = y
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"tables": _exact_tables, "cache": _exact_cache, "attention": _exact_attention,
            "logits": _exact_logits}[case["op"]](st)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    n, most = case["n"], case["most"]
    mean = 1 if most == 1 else 0.75 * most  # rows of a request
    if op == "tables":
        rows = n * most if case["mode"] != "prompts" else max(1, int(0.6 * n * most))
        live = n * (0.5 if most == 1 else most / 2)
        b = 8 * n + 4 + 16 * n + 12 * rows + 8 * live / PAGE
        if case["mode"] == "tree":
            b += 4 * live + 4 * rows * -(-most // 32)
        if case["release"]:
            b += 12 * n + 8 * live / PAGE
        return dict(bytes=int(b), flops=int(4 * rows))
    if op == "cache":
        row = 2 * case["kvh"] * case["hd"]
        rows = n * mean
        b = rows * (4 + row * (SIZES[case["src"]] + SIZES[case["cache"]]))
        if case["mode"] == "commit":
            b += n * min(mean, 4.5) * (4 + 2 * row * SIZES[case["cache"]])
        return dict(bytes=int(b), flops=0)
    if op == "attention":
        H, kvh, hd = case["heads"], case["kvh"], case["hd"]
        rows = n * mean
        ctx = case["ctx"] if case["window"] <= 0 else min(case["ctx"], case["window"])
        b = n * (ctx + mean) * kvh * hd * 2 * 2 + rows * H * hd * 2 * SIZES[case["q"]]
        return dict(bytes=int(b), flops=int(rows * H * hd * 4 * (ctx + mean / 2)))
    rows, V = n * mean, case["vocab"]
    b = rows * V * 2 * SIZES[case["dtype"]] + min(rows, case["masks"]) * V / 8
    b += n * case["hist"] * 4 + rows * (case["bias"] * 8 + 16)
    return dict(bytes=int(b), flops=int(rows * V * 6))
