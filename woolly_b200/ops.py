"""Device ops with the reference's op signatures, on torch CUDA tensors.

torch only provides device memory and the current stream here; every op runs
a kernel of libwoolly_cuda.so and raises if the library or the GPU is missing.
"""
from __future__ import annotations

import ctypes as C
import functools
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
# These calls sit between small kernels of a decode step, where the host's time
# per call counts: the checks below read each tensor's attributes once.
KV_PAGE = 16  # tokens per page of a KV cache [pages, kv_heads, KV_PAGE, head_dim]
_TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_I32 = torch.int32


def _refuse(t, name, dtype, shape, index, contiguous=True):
    """Says what is wrong with an argument that failed its check."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if dtype is not None and t.dtype not in dtype:
        raise ValueError(f"{name} must be {' or '.join(map(str, dtype))}, got {t.dtype}")
    if index is not None and t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    if shape is not None and (t.dim() != len(shape)
                              or any(w is not None and s != w for s, w in zip(t.shape, shape))):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{name} must be contiguous" + ("" if contiguous else " within its rows"))


def _i32(t, name, shape, index) -> int:
    """Address of a contiguous int32 tensor of this shape on this device."""
    try:
        if t.dtype is _I32 and t.shape == shape and t.get_device() == index and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _refuse(t, name, (_I32,), shape, index)


def _list32(t, name, index) -> int:
    """The same for one dimension of any size."""
    try:
        if t.dtype is _I32 and t.dim() == 1 and t.get_device() == index and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _refuse(t, name, (_I32,), (None,), index)


def _row_stride(t, name, width) -> int:
    """Elements from one row (of `width` elements, contiguous) to the next."""
    if t.is_contiguous():
        return width
    st, n = t.stride(), 1
    for size, step in zip(t.shape[:0:-1], st[:0:-1]):
        if size != 1 and step != n:
            _refuse(t, name, None, None, None, False)
        n *= size
    if t.shape[0] <= 1:
        return width
    if st[0] < width:
        _refuse(t, name, None, None, None, False)
    return st[0]


def _launch(fn, index, *args):
    """fn(*args, stream) on the device's current stream."""
    if torch._C._cuda_getDevice() == index:
        check(fn(*args, torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(index):
            check(fn(*args, torch._C._cuda_getCurrentRawStream(index)))


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
    b = torch.empty(3 * rows + 4 * n + 3, dtype=_I32, device=device)  # one allocation, cut up
    req, pos, slot, lengths, status, start, pages, free = torch.unsafe_split_with_sizes(
        b, (rows, rows, rows, n, n, n + 1, n + 1, 1))
    return StepPlan(start, req, pos, slot, lengths, status, free, pages,
                    torch.empty((rows, words), dtype=_I32, device=device) if words else None)


def _tables(tables, n, index):
    """Device, requests, pages per row, row stride and address of a block table."""
    try:
        if tables.dtype is _I32 and tables.dim() == 2 and tables.is_cuda:
            rows, pages = tables.shape
            i = tables.get_device()
            if (n is None or n == rows) and (index is None or index == i):
                return i, rows, pages, _row_stride(tables, "tables", pages), tables.data_ptr()
    except AttributeError:
        pass
    _refuse(tables, "tables", (_I32,), (n, None), index)


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
    index, n, pages, ld, at = _tables(tables, None, None)
    each, one = (n,), (1,)
    par = None if parents is None else _i32(parents, "parents", (rows,), index)
    if out is None:
        out = step_plan(n, rows, words, tables.device)
        at0 = out.requests.data_ptr() if rows else out.lengths.data_ptr() if n else out.row_start.data_ptr()
        row0, row1, row2, len0 = at0, at0 + 4 * rows, at0 + 8 * rows, at0 + 12 * rows
        ptrs = (len0 + 8 * n, row0, row1, row2, len0, len0 + 4 * n, len0 + 16 * n + 8, len0 + 12 * n + 4,
                out.mask.data_ptr() if words else None)
    else:
        shapes = ((n + 1,), (rows,), (rows,), (rows,), each, each, one, (n + 1,))
        for f, t, shape in zip(StepPlan._fields, out, shapes):
            _i32(t, f"out.{f}", shape, index)
        if words:
            _i32(out.mask, "out.mask", (rows, words), index)
        ptrs = [t if t is None else t.data_ptr() for t in out]
    o = _lib.StepPlan(*ptrs)
    _launch(lib().wl_block_tables, index, at, ld, pages, _i32(lengths, "lengths", each, index),
            _i32(counts, "counts", each, index), n, _list32(free_pages, "free_pages", index),
            free_pages.numel(), _i32(free_count, "free_count", one, index), rows, par, words, C.byref(o))
    return out


def release_pages(tables: torch.Tensor, lengths: torch.Tensor, keep: torch.Tensor,
                  free_pages: torch.Tensor, free_count: torch.Tensor, *,
                  out: Released | None = None) -> Released:
    """Request i keeps its first min(keep[i], lengths[i]) tokens; the pages past
    them go back to the stack, their table entries become -1
    (wl_release_pages).  Releasing what a step took leaves the stack as it was.
    `out`'s lengths and free_count may be the arguments themselves."""
    index, n, pages, ld, at = _tables(tables, None, None)
    each, one = (n,), (1,)
    if out is None:
        b = torch.empty(3 * n + 2, dtype=_I32, device=tables.device)
        out = Released(*torch.unsafe_split_with_sizes(b, (n, n, 1, n + 1)))
    else:
        for f, t, shape in zip(Released._fields, out, (each, each, one, (n + 1,))):
            _i32(t, f"out.{f}", shape, index)
    o = _lib.ReleaseResult(*[t.data_ptr() for t in out])
    _launch(lib().wl_release_pages, index, at, ld, pages, _i32(lengths, "lengths", each, index),
            _i32(keep, "keep", each, index), n, _list32(free_pages, "free_pages", index),
            free_pages.numel(), _i32(free_count, "free_count", one, index), C.byref(o))
    return out


def _caches(k, v):
    """Device, pages, KV heads, head_dim and type of a pair of caches."""
    try:
        if (k.dtype in (torch.float16, torch.bfloat16) and v.dtype is k.dtype and k.dim() == 4
                and k.is_cuda and k.is_contiguous() and v.is_contiguous() and v.shape == k.shape
                and v.get_device() == k.get_device()):
            pages, kvh, page, hd = k.shape
            if page == KV_PAGE:
                return k.get_device(), pages, kvh, hd, k.dtype
    except AttributeError:
        pass
    for t, name in ((k, "cache_k"), (v, "cache_v")):
        if (not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 4 or t.shape[2] != KV_PAGE
                or t.dtype not in (torch.float16, torch.bfloat16) or not t.is_contiguous()):
            _refuse(t, name, (torch.float16, torch.bfloat16), (None, None, KV_PAGE, None), None)
    _refuse(v, "cache_v", (k.dtype,), tuple(k.shape), k.get_device())


def kv_append(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache_k: torch.Tensor,
              cache_v: torch.Tensor) -> None:
    """Writes K and V rows [rows, kv_heads, head_dim] into their slots of a
    paged cache [pages, kv_heads, 16, head_dim] (wl_kv_append).  f32 rows are
    rounded to the cache's f16 or bf16; f16 and bf16 rows go into a cache of
    their type.  Rows may be strided (a slice of a fused projection); slots
    outside the cache, -1 among them, are skipped; slots are distinct."""
    index, pages, kvh, hd, ct = _caches(cache_k, cache_v)
    try:
        st = _TYPES.get(k.dtype)
        rows = k.shape[0]
        shape = (rows, kvh, hd)
        if st is None or k.shape != shape or k.get_device() != index:
            _refuse(k, "k", tuple(_TYPES), (None, kvh, hd), index)
        if v.dtype is not k.dtype or v.shape != shape or v.get_device() != index:
            _refuse(v, "v", (k.dtype,), shape, index)
    except (AttributeError, IndexError):
        raise ValueError(f"k and v must be CUDA tensors [rows, {kvh}, {hd}]") from None
    width = kvh * hd
    _launch(lib().wl_kv_append, index, st, _TYPES[ct], k.data_ptr(), v.data_ptr(),
            _row_stride(k, "k", width), _row_stride(v, "v", width), _i32(slots, "slots", (rows,), index),
            rows, kvh, hd, pages, cache_k.data_ptr(), cache_v.data_ptr())


def kv_commit(tables: torch.Tensor, lengths: torch.Tensor, accepted: torch.Tensor,
              accepted_start: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor) -> None:
    """Moves accepted drafts together (wl_kv_commit): node accepted[start + j]
    of request i, start = accepted_start[i], goes from token lengths[i] + node
    to token lengths[i] + j.  A request's nodes are given in rising order;
    `lengths` are those before the drafts."""
    index, pages, kvh, hd, ct = _caches(cache_k, cache_v)
    _, n, max_pages, ld, at = _tables(tables, None, index)
    _launch(lib().wl_kv_commit, index, _TYPES[ct], at, ld, max_pages, _i32(lengths, "lengths", (n,), index),
            n, _list32(accepted, "accepted", index), _i32(accepted_start, "accepted_start", (n + 1,), index),
            accepted.numel(), kvh, hd, pages, cache_k.data_ptr(), cache_v.data_ptr())


@functools.lru_cache(maxsize=4096)
def _attention_workspace(index, *sizes) -> int:
    with torch.cuda.device(index):
        return lib().wl_tree_attention_workspace(*sizes)


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
    positions > positions[r] - window (positions below lengths[i] count as it);
    `scale` defaults to head_dim ** -0.5.
    A row with a negative position or nothing to attend gives zeros; rows
    behind row_start[n] are not written.  q is f32 over an f16 cache, or has
    the cache's type; head_dim 32, 64, 128 or 256.  f16 and bf16 round the
    probabilities to their type.  `out` may be a packed q, else it may not
    overlap it."""
    index, pages, kvh, hd, ct = _caches(cache_k, cache_v)
    try:
        qt = q.dtype
        rows, heads, width = q.shape
        if width != hd or q.get_device() != index:
            _refuse(q, "q", None, (None, None, hd), index)
    except (AttributeError, ValueError):
        _refuse(q, "q", None, (None, None, hd), index)
    if qt is not ct and not (qt is torch.float32 and ct is torch.float16):
        raise ValueError(f"q must be float32 over a float16 cache or have the cache's type, got {qt} over {ct}")
    _, n, max_pages, ld, at = _tables(tables, None, index)
    words = m = None
    if mask is not None:
        try:
            words = mask.shape[1]
        except (AttributeError, IndexError):
            _refuse(mask, "mask", (_I32,), (rows, None), index)
        m = _i32(mask, "mask", (rows, words), index)
    if out is None:
        out = torch.empty(q.shape, dtype=qt, device=q.device)
    elif out.dtype is not qt or out.shape != q.shape or out.get_device() != index or not out.is_contiguous():
        _refuse(out, "out", (qt,), tuple(q.shape), index)
    t = _TYPES[qt]
    nb = _attention_workspace(index, t, n, rows, heads, kvh, hd)
    ws = torch.empty(nb, dtype=torch.uint8, device=q.device)
    _launch(lib().wl_tree_attention, index, t, q.data_ptr(), _row_stride(q, "q", heads * hd),
            cache_k.data_ptr(), cache_v.data_ptr(), pages, at, ld, max_pages,
            _i32(lengths, "lengths", (n,), index), _i32(row_start, "row_start", (n + 1,), index),
            _i32(positions, "positions", (rows,), index), m, words or 0, n, rows, heads, kvh, hd,
            min(int(window), 2 ** 31 - 1), hd ** -0.5 if scale is None else float(scale), out.data_ptr(), ws.data_ptr(), nb)
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
    int32.  `out` may be `logits`, else no row of it may overlap one."""
    try:
        lt = _TYPES.get(logits.dtype)
        rows, V = logits.shape
        index = logits.get_device()
        if lt is None or index < 0:
            _refuse(logits, "logits", tuple(_TYPES), (None, None), None)
    except (AttributeError, ValueError):
        _refuse(logits, "logits", tuple(_TYPES), (None, None), None)
    if (params.dtype is not torch.uint8 or params.get_device() != index or not params.is_contiguous()):
        _refuse(params, "params", (torch.uint8,), (None,), index)
    if params.numel() < rows * 16:
        raise ValueError(f"params must hold {rows} records")
    n, every = 0, (rows,)
    h = h0 = hp = req = dt = dm = d0 = bs = bt = bv = al = None
    total = words = nb = na = aw = 0
    if history_start is not None or history is not None:
        h0 = _list32(history_start, "history_start", index)
        h = _list32(history, "history", index)
        total = history.numel()
        n = history_start.numel() - 1
        if n < 0:
            raise ValueError("history_start must have one entry more than there are requests")
    if prompt_lens is not None:
        if history is None:
            raise ValueError("prompt_lens needs a history")
        hp = _i32(prompt_lens, "prompt_lens", (n,), index)
    if draft_mask is not None or draft_tokens is not None:
        if draft_mask is None or draft_tokens is None or row_start is None:
            raise ValueError("drafts need draft_tokens, draft_mask and row_start")
        words = draft_mask.shape[1] if draft_mask.dim() == 2 else 0
        dm = _i32(draft_mask, "draft_mask", (rows, words), index)
        dt = _i32(draft_tokens, "draft_tokens", every, index)
        d0 = _list32(row_start, "row_start", index)
        if history is not None and row_start.numel() != n + 1:
            raise ValueError(f"row_start must have {n + 1} entries, got {row_start.numel()}")
        n = row_start.numel() - 1
    if requests is not None:
        req = _i32(requests, "requests", every, index)
    if bias_start is not None or bias_tokens is not None or bias_values is not None:
        bs = _i32(bias_start, "bias_start", (rows + 1,), index)
        bt = _list32(bias_tokens, "bias_tokens", index)
        nb = bias_tokens.numel()
        if (bias_values is None or bias_values.dtype is not torch.float32 or bias_values.shape != (nb,)
                or bias_values.get_device() != index or not bias_values.is_contiguous()):
            _refuse(bias_values, "bias_values", (torch.float32,), (nb,), index)
        bv = bias_values.data_ptr()
    if allowed is not None:
        try:
            na, aw = allowed.shape
        except (AttributeError, ValueError):
            _refuse(allowed, "allowed", (_I32,), (None, None), index)
        al = _i32(allowed, "allowed", (na, aw), index)
    c = _lib.LogitContext(h, h0, hp, n, total, req, dt, dm, words, d0, bs, bt, bv, nb, al, na, aw)
    if out is None:
        out = torch.empty((rows, V), dtype=logits.dtype, device=logits.device)
    elif out.dtype is not logits.dtype or out.shape != (rows, V) or out.get_device() != index:
        _refuse(out, "out", (logits.dtype,), (rows, V), index, False)
    _launch(lib().wl_process_logits, index, lt, logits.data_ptr(), _row_stride(logits, "logits", V), rows, V,
            params.data_ptr(), C.byref(c), out.data_ptr(), _row_stride(out, "out", V))
    return out


__all__ += ["sample", "StepPlan", "Released", "step_plan", "block_tables", "release_pages", "kv_append",
            "kv_commit", "tree_attention", "logit_params", "process_logits", "KV_PAGE"]
