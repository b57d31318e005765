"""Device ops with the reference's op signatures, on torch CUDA tensors.

torch only provides device memory and the current stream here; every op runs
a kernel of libwoolly_cuda.so and raises if the library or the GPU is missing.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import numpy as np
import torch

from . import _lib
from ._lib import LAYOUT_A, LAYOUT_B, ROPE_NEOX, ROPE_OFF, check, lib


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _dev(t: torch.Tensor, dtype=None, name="tensor") -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def dequantize(data: torch.Tensor, ggml_type: int, nelements: int) -> torch.Tensor:
    """woolly_gguf::dequantize(data, ggml_type, nelements) (dequantize.rs:189)."""
    _dev(data, torch.uint8, "data")
    out = torch.empty(nelements, dtype=torch.float32, device=data.device)
    check(lib().wl_dequantize(int(ggml_type), data.data_ptr(), data.numel(), nelements,
                              out.data_ptr(), _stream()))
    return out


def quantized_matvec(weights: torch.Tensor, ggml_type: int, input: torch.Tensor,
                     output: torch.Tensor, m: int, k: int) -> None:
    """quantization::simd::quantized_matvec(weights, input, output, m, k)
    (woolly-tensor/src/quantization.rs:869): layout A, Q4_0 / Q8_0."""
    _dev(weights, torch.uint8, "weights")
    _dev(input, torch.float32, "input")
    _dev(output, torch.float32, "output")
    if input.numel() < k or output.numel() < m:
        raise ValueError("input/output too small")
    check(lib().wl_quantized_matvec(int(ggml_type), weights.data_ptr(), input.data_ptr(),
                                    output.data_ptr(), m, k, _stream()))


def qgemv(weights: torch.Tensor, ggml_type: int, layout: int, x: torch.Tensor, n: int) -> torch.Tensor:
    """y[b, :] = x[b, :] @ W for quantized W ([K][N] layout B or [N][K] layout A)."""
    _dev(weights, torch.uint8, "weights")
    _dev(x, torch.float32, "x")
    x2 = x.reshape(-1, x.shape[-1])
    B, K = x2.shape
    y = torch.empty(B, n, dtype=torch.float32, device=x.device)
    check(lib().wl_qgemv(int(ggml_type), int(layout), weights.data_ptr(), K, n, x2.data_ptr(), B,
                         y.data_ptr(), _stream()))
    return y.reshape(*x.shape[:-1], n)


def qgemm(weights: torch.Tensor, ggml_type: int, x: torch.Tensor, n: int) -> torch.Tensor:
    """Prefill GEMM y[m, :] = x[m, :] @ W for layout-B W ([K][N] GGUF blocks),
    all rows in one call (tcgen05 tensor cores where the shape allows)."""
    _dev(weights, torch.uint8, "weights")
    _dev(x, torch.float32, "x")
    x2 = x.reshape(-1, x.shape[-1])
    M, K = x2.shape
    y = torch.empty(M, n, dtype=torch.float32, device=x.device)
    check(lib().wl_qgemm(int(ggml_type), weights.data_ptr(), K, n, x2.data_ptr(), M, y.data_ptr(),
                         _stream()))
    return y.reshape(*x.shape[:-1], n)


def split_planes(x: torch.Tensor) -> torch.Tensor:
    """f32 [B, K] -> f16 [2, B, K]: hi = f16(x), lo = f16(x - hi)."""
    hi = x.to(torch.float16)
    return torch.stack([hi, (x - hi.float()).to(torch.float16)]).contiguous()


def qgemv_planes(weights: torch.Tensor, ggml_type: int, planes: torch.Tensor, n: int,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Layout-B GEMV on hi/lo activation planes [2, B, K] (no allocation
    inside the library; capturable in a CUDA graph)."""
    _dev(weights, torch.uint8, "weights")
    _dev(planes, torch.float16, "planes")
    _, B, K = planes.shape
    y = out if out is not None else torch.empty(B, n, dtype=torch.float32, device=planes.device)
    check(lib().wl_qgemv_planes(int(ggml_type), weights.data_ptr(), K, n, planes.data_ptr(), B * K,
                                B, y.data_ptr(), _stream()))
    return y


def qtile(weights: torch.Tensor, ggml_type: int, k: int, n: int) -> torch.Tensor:
    """Tiled decode copy of a layout-B GGUF matrix [k][n] (wl_qtile_repack)."""
    _dev(weights, torch.uint8, "weights")
    nb = lib().wl_qtile_bytes(int(ggml_type), k, n)
    if not nb:
        raise ValueError(f"qtile: unsupported type {ggml_type} or shape {k}x{n}")
    t = torch.empty(nb, dtype=torch.uint8, device=weights.device)
    check(lib().wl_qtile_repack(int(ggml_type), weights.data_ptr(), k, n, t.data_ptr(), _stream()))
    return t


def qgemv_tiled(tiled: torch.Tensor, ggml_type: int, planes: torch.Tensor, n: int,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """qgemv_planes on the tiled copy made by qtile()."""
    _dev(tiled, torch.uint8, "tiled")
    _dev(planes, torch.float16, "planes")
    _, B, K = planes.shape
    y = out if out is not None else torch.empty(B, n, dtype=torch.float32, device=planes.device)
    check(lib().wl_qgemv_tiled(int(ggml_type), tiled.data_ptr(), K, n, planes.data_ptr(), B * K,
                               B, y.data_ptr(), _stream()))
    return y


def qgemm_tiled(tiled: torch.Tensor, ggml_type: int, planes: torch.Tensor, n: int,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """The tcgen05 prefill GEMM on the tiled copy made by qtile(); planes [2, M, K]."""
    _dev(tiled, torch.uint8, "tiled")
    _dev(planes, torch.float16, "planes")
    _, M, K = planes.shape
    y = out if out is not None else torch.empty(M, n, dtype=torch.float32, device=planes.device)
    check(lib().wl_qgemm_tiled(int(ggml_type), tiled.data_ptr(), K, n, planes.data_ptr(), M * K, M,
                               y.data_ptr(), _stream()))
    return y


def rmsnorm_rope(x: torch.Tensor, w: torch.Tensor, eps: float, *, rope: bool = False,
                 positions: torch.Tensor | None = None, head_dim: int = 0, theta: float = 10000.0,
                 out_dtype=torch.float32) -> torch.Tensor:
    """rms_norm (woolly-core tensor_utils.rs:446-480) with an optional fused NeoX
    RoPE of the normalised row (woolly-tensor ops/mod.rs:476-527)."""
    _dev(x, torch.float32, "x")
    _dev(w, torch.float32, "w")
    d = x.shape[-1]
    rows = x.numel() // d
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    pos_ptr = None
    if rope:
        if positions is None:
            raise ValueError("rope needs positions")
        _dev(positions, torch.int32, "positions")
        pos_ptr = positions.data_ptr()
    check(lib().wl_rmsnorm_rope(x.data_ptr(), w.data_ptr(), rows, d, eps,
                                ROPE_NEOX if rope else ROPE_OFF, pos_ptr, head_dim, theta,
                                y.data_ptr(), 1 if out_dtype == torch.float16 else 0, _stream()))
    return y


class TransformerSIMD:
    """woolly_tensor::ops::simd_matmul::TransformerSIMD (simd_matmul.rs:811,1002)."""

    @staticmethod
    def rms_norm(input: torch.Tensor, weight: torch.Tensor, eps: float, output: torch.Tensor) -> None:
        d = weight.numel()
        _dev(output, torch.float32, "output")
        y = rmsnorm_rope(input.reshape(-1, d), weight, eps)
        output.copy_(y.reshape(output.shape))

    @staticmethod
    def swiglu_activation(gate: torch.Tensor, up: torch.Tensor, output: torch.Tensor) -> None:
        _dev(gate, torch.float32, "gate")
        _dev(up, torch.float32, "up")
        _dev(output, torch.float32, "output")
        if gate.numel() != up.numel() or output.numel() != gate.numel():
            raise ValueError("gate, up and output must have the same length")
        check(lib().wl_swiglu(gate.data_ptr(), up.data_ptr(), gate.numel(), output.data_ptr(),
                              _stream()))


class RoPE:
    """woolly_tensor::ops::neural::RoPE (ops/mod.rs:472-527)."""

    @staticmethod
    def apply_f32(input: torch.Tensor, output: torch.Tensor, positions: torch.Tensor, base: float,
                  batch_size: int, seq_len: int, n_heads: int, head_dim: int) -> None:
        _dev(input, torch.float32, "input")
        _dev(output, torch.float32, "output")
        _dev(positions, torch.int32, "positions")
        if input.numel() != batch_size * seq_len * n_heads * head_dim:
            raise ValueError("input size mismatch")
        if positions.numel() != seq_len:
            raise ValueError("positions must have seq_len entries")
        check(lib().wl_rope(input.data_ptr(), output.data_ptr(), positions.data_ptr(), base,
                            batch_size, seq_len, n_heads, head_dim, _stream()))


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, past: int, heads: int,
              kv_heads: int, head_dim: int, window: int = 0) -> torch.Tensor:
    """GQA attention over an f32 KV prefix (lazy_transformer.rs:375-434):
    q [rows, H*hd], k/v [past+rows, KVH*hd]."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _dev(t, torch.float32, n)
    rows = q.numel() // (heads * head_dim)
    out = torch.empty(rows, heads * head_dim, dtype=torch.float32, device=q.device)
    check(lib().wl_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), rows, past, heads, kv_heads,
                             head_dim, window, out.data_ptr(), _stream()))
    return out


__all__ = ["dequantize", "quantized_matvec", "qgemv", "rmsnorm_rope", "TransformerSIMD", "RoPE",
           "attention", "LAYOUT_A", "LAYOUT_B"]


def sample(logits: torch.Tensor, temperature, top_k, top_p, u, out: torch.Tensor | None = None,
           params: torch.Tensor | None = None) -> torch.Tensor:
    """sample_next_token (inference.rs:441-483) for every row of f32 logits
    [rows, vocab] on the GPU; temperature / top_k / top_p / u are per-row
    sequences (or scalars).  `params` (optional): a device buffer of at least
    rows * 16 bytes to stage them in.  Returns int32 token ids [rows]."""
    _dev(logits, torch.float32, "logits")
    rows, V = logits.shape
    rec = sample_params(rows, temperature, top_k, top_p, u)
    src = torch.from_numpy(rec.view(np.uint8))
    if params is None:
        params = src.to(logits.device)
    else:
        params[: src.numel()].copy_(src)
    y = out if out is not None else torch.empty(rows, dtype=torch.int32, device=logits.device)
    check(lib().wl_sample(logits.data_ptr(), rows, V, logits.stride(0), params.data_ptr(),
                          y.data_ptr(), _stream()))
    return y


def sample_params(rows, temperature, top_k, top_p, u) -> "np.ndarray":
    """Per-row knobs as an array of wl_sample_params records."""
    rec = np.zeros(rows, dtype=[("t", "<f4"), ("k", "<i4"), ("p", "<f4"), ("u", "<f4")])
    rec["t"], rec["k"], rec["p"], rec["u"] = temperature, top_k, top_p, u
    return rec


# ---------------------------------------------------------------- a serving step on a paged cache
KV_PAGE = 16  # tokens per page of a KV cache [pages, kv_heads, KV_PAGE, head_dim]
_TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _arg(t, name, dtype=None, shape=None, device=None, rows=False) -> torch.Tensor:
    """A CUDA tensor of the given type, shape (None: any size) and device;
    `rows`: the first dimension may be strided."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if dtype is not None and t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if shape is not None and (t.dim() != len(shape)
                              or any(w is not None and s != w for s, w in zip(t.shape, shape))):
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        if not (rows and t.dim() >= 1 and t.shape[0] > 0 and t[0].is_contiguous() and
                t.stride(0) >= t[0].numel()):
            raise ValueError(f"{name} must be contiguous" + (" within its rows" if rows else ""))
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _ld(t) -> int:
    """Elements from one row to the next."""
    width = t[0].numel() if t.shape[0] else t.numel()
    return t.stride(0) if t.shape[0] > 1 else width


def _on(t):
    """The tensor's device as the current one, so that its current stream is used."""
    return torch.cuda.device(t.device)


class StepPlan(NamedTuple):
    """Device tensors of block_tables (int32); `mask` is None without parents."""
    row_start: torch.Tensor   # [n + 1] first row of each request
    requests: torch.Tensor    # [rows] request of each row, -1 behind the last
    positions: torch.Tensor   # [rows] position, -1 for a row left out
    slots: torch.Tensor       # [rows] slot in the cache, -1 for a row left out
    lengths: torch.Tensor     # [n] tokens held after the step
    status: torch.Tensor      # [n] STEP_OK, STEP_NO_PAGES, ...
    free_count: torch.Tensor  # [1] free pages left
    page_start: torch.Tensor  # [n + 1] pages taken by the requests before each
    mask: torch.Tensor | None  # [rows, words] bits of each row's path


class Released(NamedTuple):
    """Device tensors of release_pages (int32)."""
    lengths: torch.Tensor     # [n] tokens held afterwards
    status: torch.Tensor      # [n]
    free_count: torch.Tensor  # [1] free pages
    page_start: torch.Tensor  # [n + 1] pages given back by the requests before each


def step_plan(n: int, rows: int, words: int = 0, device="cuda") -> StepPlan:
    """Buffers for block_tables' `out`: n requests, `rows` rows, masks of `words` words."""
    def new(*shape):
        return torch.empty(*shape, dtype=torch.int32, device=device)
    return StepPlan(new(n + 1), new(rows), new(rows), new(rows), new(n), new(n), new(1), new(n + 1),
                    new(rows, words) if words else None)


def _tables(tables, n=None, device=None):
    _arg(tables, "tables", torch.int32, (n, None), device, rows=True)
    return tables.shape[0], tables.shape[1], max(_ld(tables), tables.shape[1]), tables.device


def block_tables(tables: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor,
                 free_pages: torch.Tensor, free_count: torch.Tensor, rows: int, *,
                 parents: torch.Tensor | None = None, words: int = 0,
                 out: StepPlan | None = None) -> StepPlan:
    """Block tables, slot maps and positions of a step in which request i,
    holding lengths[i] tokens, adds counts[i] (wl_block_tables; all int32).

    `tables` [n, pages] gets the pages taken, in request order, from the top of
    the stack free_pages[:free_count]; `rows` is the size of the row arrays.
    Requests are served until the first that the stack has too few pages for
    (status STEP_NO_PAGES from there on, for requests that need any); rows of a
    request that is not served, and rows behind the last one, have slot -1.
    parents [rows] (with 32 * words mask bits) makes a request's rows a tree of
    drafted tokens: the index of an earlier node of the request, or -1; the
    plan's `positions` then count depths and its `mask` holds each row's path.
    `out` (step_plan) reuses buffers; its lengths and free_count may be the
    arguments themselves."""
    n, pages, ld, dev = _tables(tables)
    i32 = torch.int32
    _arg(lengths, "lengths", i32, (n,), dev)
    _arg(counts, "counts", i32, (n,), dev)
    _arg(free_pages, "free_pages", i32, (None,), dev)
    _arg(free_count, "free_count", i32, (1,), dev)
    if parents is not None:
        _arg(parents, "parents", i32, (rows,), dev)
    if out is None:
        out = step_plan(n, rows, words, dev)
    else:
        shapes = ((n + 1,), (rows,), (rows,), (rows,), (n,), (n,), (1,), (n + 1,))
        for f, t, shape in zip(StepPlan._fields, out, shapes):
            _arg(t, f"out.{f}", i32, shape, dev)
        if words:
            _arg(out.mask, "out.mask", i32, (rows, words), dev)
    c = _lib.StepPlan(*[_ptr(t) for t in out])
    with _on(tables):
        check(lib().wl_block_tables(tables.data_ptr(), ld, pages, lengths.data_ptr(), counts.data_ptr(), n,
                                    free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(), rows,
                                    _ptr(parents), words, C.byref(c), _stream()))
    return out


def release_pages(tables: torch.Tensor, lengths: torch.Tensor, keep: torch.Tensor,
                  free_pages: torch.Tensor, free_count: torch.Tensor, *,
                  out: Released | None = None) -> Released:
    """Request i keeps its first min(keep[i], lengths[i]) tokens; the pages past
    them go back to the stack, their table entries become -1
    (wl_release_pages).  Releasing what a step took leaves the stack as it was.
    `out`'s lengths and free_count may be the arguments themselves."""
    n, pages, ld, dev = _tables(tables)
    i32 = torch.int32
    _arg(lengths, "lengths", i32, (n,), dev)
    _arg(keep, "keep", i32, (n,), dev)
    _arg(free_pages, "free_pages", i32, (None,), dev)
    _arg(free_count, "free_count", i32, (1,), dev)
    if out is None:
        out = Released(*[torch.empty(s, dtype=i32, device=dev) for s in (n, n, 1, n + 1)])
    else:
        for f, t, s in zip(Released._fields, out, (n, n, 1, n + 1)):
            _arg(t, f"out.{f}", i32, (s,), dev)
    c = _lib.ReleaseResult(*[_ptr(t) for t in out])
    with _on(tables):
        check(lib().wl_release_pages(tables.data_ptr(), ld, pages, lengths.data_ptr(), keep.data_ptr(), n,
                                     free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(),
                                     C.byref(c), _stream()))
    return out


def _caches(cache_k, cache_v):
    _arg(cache_k, "cache_k", (torch.float16, torch.bfloat16), (None, None, KV_PAGE, None))
    _arg(cache_v, "cache_v", cache_k.dtype, tuple(cache_k.shape), cache_k.device)
    return cache_k.shape[0], cache_k.shape[1], cache_k.shape[3], cache_k.device


def kv_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache_k: torch.Tensor,
              cache_v: torch.Tensor) -> None:
    """Writes K and V rows [rows, kv_heads, head_dim] into their slots of a
    paged cache [pages, kv_heads, 16, head_dim] (wl_kv_append).  f32 rows are
    rounded to the cache's f16 or bf16; f16 and bf16 rows go into a cache of
    their type.  Rows may be strided (a slice of a fused projection); slots
    outside the cache, -1 among them, are skipped; slots are distinct."""
    pages, kvh, hd, dev = _caches(cache_k, cache_v)
    _arg(k, "k", tuple(_TYPES), (None, kvh, hd), dev, rows=True)
    _arg(v, "v", k.dtype, tuple(k.shape), dev, rows=True)
    rows = k.shape[0]
    _arg(slots, "slots", torch.int32, (rows,), dev)
    with _on(cache_k):
        check(lib().wl_kv_append(_TYPES[k.dtype], _TYPES[cache_k.dtype], k.data_ptr(), v.data_ptr(),
                                 max(_ld(k), kvh * hd), max(_ld(v), kvh * hd), slots.data_ptr(), rows, kvh,
                                 hd, pages, cache_k.data_ptr(), cache_v.data_ptr(), _stream()))


def kv_commit(tables: torch.Tensor, lengths: torch.Tensor, accepted: torch.Tensor,
              accepted_start: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor) -> None:
    """Moves accepted drafts together (wl_kv_commit): node accepted[start + j]
    of request i, start = accepted_start[i], goes from token lengths[i] + node
    to token lengths[i] + j.  A request's nodes are given in rising order;
    `lengths` are those before the drafts."""
    pages, kvh, hd, dev = _caches(cache_k, cache_v)
    n, max_pages, ld, _ = _tables(tables, device=dev)
    _arg(lengths, "lengths", torch.int32, (n,), dev)
    _arg(accepted, "accepted", torch.int32, (None,), dev)
    _arg(accepted_start, "accepted_start", torch.int32, (n + 1,), dev)
    with _on(cache_k):
        check(lib().wl_kv_commit(_TYPES[cache_k.dtype], tables.data_ptr(), ld, max_pages, lengths.data_ptr(),
                                 n, accepted.data_ptr(), accepted_start.data_ptr(), accepted.numel(), kvh, hd,
                                 pages, cache_k.data_ptr(), cache_v.data_ptr(), _stream()))


def tree_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, tables: torch.Tensor,
                   lengths: torch.Tensor, row_start: torch.Tensor, positions: torch.Tensor, *,
                   mask: torch.Tensor | None = None, window: int = 0, scale: float | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """GQA attention of a step's rows q [rows, heads, head_dim] over a paged
    cache (wl_tree_attention).

    Rows row_start[i] : row_start[i + 1] are request i's tokens; their K and V
    lie in the cache behind its lengths[i] tokens (kv_append at block_tables'
    slots; `lengths` as given to block_tables).  A row attends those lengths[i]
    tokens and the tokens of the step that its mask bits name (block_tables'
    mask); without a mask, the step's earlier tokens and itself, so that one
    row per request is a plain decode step.  `window` > 0 keeps keys at
    positions > positions[r] - window; `scale` defaults to head_dim ** -0.5.
    A row with a negative position or nothing to attend gives zeros; rows
    behind row_start[n] are not written.  q is f32 over an f16 cache, or has
    the cache's type; head_dim 32, 64, 128 or 256."""
    pages, kvh, hd, dev = _caches(cache_k, cache_v)
    _arg(q, "q", tuple(_TYPES), (None, None, hd), dev, rows=True)
    rows, heads = q.shape[0], q.shape[1]
    if q.dtype != cache_k.dtype and not (q.dtype == torch.float32 and cache_k.dtype == torch.float16):
        raise ValueError(f"q must be float32 over a float16 cache or have the cache's type, got {q.dtype} "
                         f"over {cache_k.dtype}")
    n, max_pages, ld, _ = _tables(tables, device=dev)
    i32 = torch.int32
    _arg(lengths, "lengths", i32, (n,), dev)
    _arg(row_start, "row_start", i32, (n + 1,), dev)
    _arg(positions, "positions", i32, (rows,), dev)
    words = 0
    if mask is not None:
        _arg(mask, "mask", i32, (rows, None), dev)
        words = mask.shape[1]
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    else:
        _arg(out, "out", q.dtype, tuple(q.shape), dev)
    qt = _TYPES[q.dtype]
    with _on(q):
        nb = lib().wl_tree_attention_workspace(qt, n, rows, heads, kvh, hd)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        check(lib().wl_tree_attention(qt, q.data_ptr(), max(_ld(q), heads * hd), cache_k.data_ptr(),
                                      cache_v.data_ptr(), pages, tables.data_ptr(), ld, max_pages,
                                      lengths.data_ptr(), row_start.data_ptr(), positions.data_ptr(),
                                      _ptr(mask), words, n, rows, heads, kvh, hd, int(window),
                                      hd ** -0.5 if scale is None else float(scale), out.data_ptr(),
                                      _ptr(ws), nb, _stream()))
    return out


def logit_params(rows: int, repetition=1.0, presence=0.0, frequency=0.0, allowed_row=-1,
                 device="cuda") -> torch.Tensor:
    """Per-row settings of process_logits as a device buffer of wl_logit_params
    records; each argument is a scalar or a sequence of `rows` values."""
    rec = np.zeros(rows, dtype=[("r", "<f4"), ("p", "<f4"), ("f", "<f4"), ("a", "<i4")])
    rec["r"], rec["p"], rec["f"], rec["a"] = repetition, presence, frequency, allowed_row
    if not (np.isfinite(rec["r"]).all() and (rec["r"] > 0).all()):
        raise ValueError("repetition must be positive and finite")
    if not (np.isfinite(rec["p"]).all() and np.isfinite(rec["f"]).all()):
        raise ValueError("presence and frequency must be finite")
    return torch.from_numpy(rec.view(np.uint8)).to(device)


def process_logits(logits: torch.Tensor, params: torch.Tensor, *, history: torch.Tensor | None = None,
                   history_start: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                   requests: torch.Tensor | None = None, draft_tokens: torch.Tensor | None = None,
                   draft_mask: torch.Tensor | None = None, row_start: torch.Tensor | None = None,
                   bias_start: torch.Tensor | None = None, bias_tokens: torch.Tensor | None = None,
                   bias_values: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Penalties for repeated tokens, biases and grammar masks on logits
    [rows, vocab] before sampling (wl_process_logits); params from logit_params.

    history / history_start [n + 1]: the requests' tokens, packed; the first
    prompt_lens[i] of request i are its prompt (repetition only), the others
    were produced (repetition, presence, frequency).  requests [rows]: the
    request of each row (default: row r is request r; -1: none).  draft_tokens
    [rows], draft_mask and row_start (block_tables): the tokens of a drafted
    row's path count as produced.  bias_start [rows + 1], bias_tokens,
    bias_values: additive biases; of several for one token the last holds.
    allowed [masks, words]: bit v % 32 of word v // 32 set means token v may
    follow; params' allowed_row picks the mask of each row.  Integers are
    int32.  `out` may be `logits`."""
    _arg(logits, "logits", tuple(_TYPES), (None, None), rows=True)
    rows, V = logits.shape
    dev, i32 = logits.device, torch.int32
    _arg(params, "params", torch.uint8, (None,), dev)
    if params.numel() < rows * 16:
        raise ValueError(f"params must hold {rows} records")
    c = _lib.LogitContext()
    n = None
    if history_start is not None or history is not None:
        _arg(history_start, "history_start", i32, (None,), dev)
        _arg(history, "history", i32, (None,), dev)
        n = history_start.numel() - 1
        if n < 0:
            raise ValueError("history_start must have one entry more than there are requests")
        c.history, c.history_start, c.history_total = history.data_ptr(), history_start.data_ptr(), history.numel()
    if prompt_lens is not None:
        if n is None:
            raise ValueError("prompt_lens needs a history")
        c.prompt_lens = _arg(prompt_lens, "prompt_lens", i32, (n,), dev).data_ptr()
    if draft_mask is not None or draft_tokens is not None:
        _arg(draft_mask, "draft_mask", i32, (rows, None), dev)
        _arg(draft_tokens, "draft_tokens", i32, (rows,), dev)
        _arg(row_start, "row_start", i32, (None if n is None else n + 1,), dev)
        n = row_start.numel() - 1
        c.draft_mask, c.words = draft_mask.data_ptr(), draft_mask.shape[1]
        c.draft_tokens, c.row_start = draft_tokens.data_ptr(), row_start.data_ptr()
    c.n_history = n or 0
    if requests is not None:
        c.requests = _arg(requests, "requests", i32, (rows,), dev).data_ptr()
    if bias_start is not None or bias_tokens is not None or bias_values is not None:
        _arg(bias_start, "bias_start", i32, (rows + 1,), dev)
        _arg(bias_tokens, "bias_tokens", i32, (None,), dev)
        _arg(bias_values, "bias_values", torch.float32, (bias_tokens.numel(),), dev)
        c.bias_start, c.bias_tokens = bias_start.data_ptr(), bias_tokens.data_ptr()
        c.bias_values, c.bias_total = bias_values.data_ptr(), bias_tokens.numel()
    if allowed is not None:
        _arg(allowed, "allowed", i32, (None, None), dev)
        c.allowed, c.n_allowed, c.allowed_words = allowed.data_ptr(), allowed.shape[0], allowed.shape[1]
    if out is None:
        out = torch.empty((rows, V), dtype=logits.dtype, device=dev)
    else:
        _arg(out, "out", logits.dtype, (rows, V), dev, rows=True)
    with _on(logits):
        check(lib().wl_process_logits(_TYPES[logits.dtype], logits.data_ptr(), max(_ld(logits), V), rows, V,
                                      params.data_ptr(), C.byref(c), out.data_ptr(), max(_ld(out), V),
                                      _stream()))
    return out


__all__ += ["sample", "StepPlan", "Released", "step_plan", "block_tables", "release_pages", "kv_append",
            "kv_commit", "tree_attention", "logit_params", "process_logits", "KV_PAGE"]
