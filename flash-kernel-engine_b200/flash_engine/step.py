"""The serving step around the paged decode, over CUDA tensors.

* ``plan_paged_step``        -- blocks, block tables, positions and cache slots of a step,
  from request lengths that live on the GPU;
* ``paged_qkv_append``       -- per-head QK norm, rotary embedding and cache write of the
  step's tokens in one pass over their QKV projection;
* ``update_page_bounds``     -- int8 boxes of the keys of the pages the step filled;
* ``sparse_paged_attention`` -- decode attention over the pages whose boxes bound q.k
  highest.

Everything stays on the GPU and on the current stream: no call synchronises, and with
``out=`` buffers none allocates anything a CUDA graph could not keep. As in ``ops``, inputs
must be CUDA tensors (TypeError otherwise) and unsupported shapes raise.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib
from .ops import _on, _paged_shapes, _require_cuda, _workspace

_plan = _lib.lib.fe_plan_paged_step
_append = _lib.lib.fe_paged_qkv_append
_bounds = _lib.lib.fe_update_page_bounds
_sparse = _lib.lib.fe_sparse_paged_attention
_scratch_ints = _lib.lib.fe_sparse_paged_attention_scratch_ints

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_LAYOUTS = {"flat": 0, "vllm": 1}


class PagedStep(NamedTuple):
    """What ``plan_paged_step`` returns (int32, slots int64)."""
    context_lens: torch.Tensor  # [S] tokens each request holds after the step
    cu_seqlens: torch.Tensor    # [S + 1] first token of each request
    positions: torch.Tensor     # [max_tokens] -1 past the step's tokens
    slots: torch.Tensor         # [max_tokens] block * block_size + offset, or -1
    free_state: torch.Tensor    # [4] ring head, ring count, requests served, tokens


class PageBounds(NamedTuple):
    """Boxes of a cache's full pages: ``values`` int8 [num_blocks, Hkv, 2, d] (largest, then
    smallest key value per channel, rounded outwards) in units of ``scales`` float32
    [num_blocks, Hkv], powers of two."""
    values: torch.Tensor
    scales: torch.Tensor


def _raw_stream(t):
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _same_device(first, *ts):
    for t in ts:
        if t.device != first.device:
            raise ValueError("all tensors must be on one device")


def _buffer(t, shape, dtype, like, name):
    if t is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous() or t.device != like.device:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} "
                         f"on {like.device}")
    return t


def plan_paged_step(context_lens, new_lens, block_tables, free_blocks, free_state,
                    block_size: int = 16, *, max_tokens: int | None = None, finished=None,
                    out=None) -> PagedStep:
    """Plans a step of requests that hold ``context_lens`` [S] tokens and add ``new_lens``
    [S] (both int32).

    ``free_blocks`` [num_blocks] int32 is a ring of free block ids whose first is at
    ``free_state[0]`` and whose count is ``free_state[1]`` (int32, 2 or more elements: a
    step's own ``free_state`` serves the next). ``block_tables`` [S, max_blocks] int32 and
    the ring are updated in place. ``finished`` [S] (bool or uint8): requests whose blocks
    go back to the ring; their rows start again at length 0, with new tokens if they have
    any (blocks given back serve from the next step on).

    Requests are served in order until one does not fit ``max_tokens``, the ring or its
    row; that one and those after it get no tokens (``free_state[2]`` counts the served
    ones). Tokens past the step's have position and slot -1, so that a step of fewer
    tokens runs with the same buffers. ``out``: the five tensors of a ``PagedStep`` to write
    into (``max_tokens`` is then their length); they must not be inputs of this call."""
    ts = (context_lens, new_lens, block_tables, free_blocks, free_state)
    _require_cuda(*ts)
    _same_device(*ts)
    for t in ts:
        if t.dtype != torch.int32:
            raise TypeError("lengths, block_tables, free_blocks and free_state must be int32")
    if context_lens.dim() != 1 or new_lens.shape != context_lens.shape or \
            block_tables.dim() != 2 or block_tables.shape[0] != context_lens.shape[0] or \
            free_blocks.dim() != 1 or free_state.dim() != 1 or free_state.shape[0] < 2:
        raise ValueError("context_lens, new_lens [S], block_tables [S, max_blocks], free_blocks "
                         "[num_blocks] and free_state [>= 2] expected")
    S, width = block_tables.shape
    fin = None
    if finished is not None:
        _require_cuda(finished)
        if finished.dtype not in (torch.bool, torch.uint8) or finished.shape != (S,):
            raise ValueError("finished must be a bool or uint8 tensor [S]")
        _same_device(context_lens, finished)
        fin = finished.data_ptr()
    if out is None:
        if max_tokens is None:
            raise ValueError("max_tokens or out must be given")
        out = (None,) * 5
    elif max_tokens is None:
        max_tokens = out[2].shape[0]
    i32 = torch.int32
    r = PagedStep(_buffer(out[0], (S,), i32, context_lens, "context_lens"),
                  _buffer(out[1], (S + 1,), i32, context_lens, "cu_seqlens"),
                  _buffer(out[2], (max_tokens,), i32, context_lens, "positions"),
                  _buffer(out[3], (max_tokens,), torch.int64, context_lens, "slots"),
                  _buffer(out[4], (4,), i32, context_lens, "free_state"))
    if r.context_lens.data_ptr() == context_lens.data_ptr() and S > 0 or \
            r.free_state.data_ptr() == free_state.data_ptr():
        raise ValueError("out must not hold inputs of the same call")
    with _on(context_lens.device):
        st = _plan(context_lens.data_ptr(), new_lens.data_ptr(), fin, block_tables.data_ptr(),
                   free_blocks.data_ptr(), free_state.data_ptr(), r.context_lens.data_ptr(),
                   r.cu_seqlens.data_ptr(), r.positions.data_ptr(), r.slots.data_ptr(),
                   r.free_state.data_ptr(), S, width, free_blocks.shape[0], block_size,
                   max_tokens, _raw_stream(context_lens))
    if st:
        _lib.check(st, "plan_paged_step")
    return r


def _cache_dims(key_cache, block_size, kv_layout):
    """(num_blocks, Hkv, d) of a key cache."""
    if kv_layout == "flat" and key_cache.dim() == 4 and key_cache.shape[2] == block_size:
        return key_cache.shape[0], key_cache.shape[1], key_cache.shape[3]
    if kv_layout == "vllm" and key_cache.dim() == 5 and key_cache.shape[3] == block_size and \
            key_cache.shape[4] == 8:
        return key_cache.shape[0], key_cache.shape[1], key_cache.shape[2] * 8
    raise ValueError("key_cache must be flat [num_blocks, Hkv, block_size, d] or vllm "
                     "[num_blocks, Hkv, d/8, block_size, 8]")


def paged_qkv_append(qkv, key_cache, value_cache, positions, slots, num_heads: int,
                     block_size: int = 16, *, q_weight=None, k_weight=None, eps: float = 1e-6,
                     rope=None, interleaved: bool = True, kv_layout: str = "flat",
                     page_bounds=None, out=None):
    """Norm, rotation and cache write of a step's tokens; returns the queries [T, H, d].

    ``qkv`` [T, (H + 2 Hkv) d] (bfloat16, float16 or float32; rows may be strided): query,
    key and value heads of each token. ``q_weight`` / ``k_weight`` [d] (of qkv's type or
    float32; None = that part is not normalised): RMS norm per head. ``rope=(cos, sin)``:
    float32 tables [max_pos, r / 2], r <= d; queries and keys are rotated at ``positions``
    [T] (int32), pairs (2i, 2i + 1) if ``interleaved`` else (i, i + r / 2). Keys and values
    go to cache slots ``slots`` [T] (int64, block * block_size + offset); a negative slot is
    not cached, a negative position is padding (zero query row, nothing cached).
    ``page_bounds``: also ``update_page_bounds`` of the pages this fills."""
    if not (isinstance(qkv, torch.Tensor) and qkv.is_cuda):
        raise TypeError("qkv must be a CUDA tensor")
    _require_cuda(key_cache, value_cache, positions, slots)
    nb, Hkv, d = _cache_dims(key_cache, block_size, kv_layout)
    dt = _DTYPES.get(qkv.dtype)
    if dt is None:
        raise TypeError(f"unsupported dtype {qkv.dtype}")
    vshape = key_cache.shape if kv_layout == "flat" else (nb, Hkv, d, block_size)
    if key_cache.dtype != qkv.dtype or value_cache.dtype != qkv.dtype or \
            value_cache.shape != vshape:
        raise ValueError("key_cache and value_cache must match, in qkv's dtype")
    if kv_layout == "vllm" and dt == 2:
        raise ValueError("the fp32 cache takes the flat layout")
    if qkv.dim() != 2 or qkv.shape[1] != (num_heads + 2 * Hkv) * d or num_heads < 1:
        raise ValueError("qkv must be [T, (num_heads + 2 Hkv) * d]")
    T = qkv.shape[0]
    if qkv.stride(1) != 1 or (T > 1 and qkv.stride(0) < qkv.shape[1]):
        raise ValueError("the elements of a row of qkv must be contiguous, rows apart")
    if positions.dtype != torch.int32 or slots.dtype != torch.int64 or \
            positions.shape != (T,) or slots.shape != (T,):
        raise ValueError("positions int32 [T] and slots int64 [T] expected")
    _same_device(qkv, key_cache, value_cache, positions, slots)
    wq = wk = rc = rs = None
    f32 = 0
    for w in (q_weight, k_weight):
        if w is not None:
            _require_cuda(w)
            _same_device(qkv, w)
            if w.shape != (d,) or w.dtype not in (qkv.dtype, torch.float32):
                raise ValueError("norm weights must be [d] of qkv's dtype or float32")
            f32 = int(w.dtype == torch.float32)
    if q_weight is not None:
        wq = q_weight.data_ptr()
    if k_weight is not None:
        wk = k_weight.data_ptr()
        if wq is not None and q_weight.dtype != k_weight.dtype:
            raise ValueError("norm weights must share a dtype")
    rd = rmax = 0
    if rope is not None:
        cos, sin = rope
        _require_cuda(cos, sin)
        _same_device(qkv, cos, sin)
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.shape != sin.shape or \
                cos.dim() != 2 or not 1 <= cos.shape[1] <= d // 2:
            raise ValueError("rope tables must be float32 [max_pos, r/2] with r <= d")
        rc, rs, rmax, rd = cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1]
    out = _buffer(out, (T, num_heads, d), qkv.dtype, qkv, "out")
    stride = qkv.stride(0) if T > 1 else qkv.shape[1]
    with _on(qkv.device):
        st = _append(qkv.data_ptr(), stride, out.data_ptr(), key_cache.data_ptr(),
                     value_cache.data_ptr(), positions.data_ptr(), slots.data_ptr(), wq, wk, f32,
                     eps, rc, rs, rd, rmax, int(interleaved), T, num_heads, Hkv, d, block_size,
                     nb, dt, _LAYOUTS[kv_layout], _raw_stream(qkv))
    if st:
        _lib.check(st, "paged_qkv_append")
    if page_bounds is not None:
        update_page_bounds(key_cache, page_bounds, slots, block_size, kv_layout=kv_layout)
    return out


def new_page_bounds(num_blocks: int, num_kv_heads: int, head_dim: int, device) -> PageBounds:
    """Storage for the boxes of a cache of this shape."""
    return PageBounds(torch.zeros((num_blocks, num_kv_heads, 2, head_dim), dtype=torch.int8,
                                  device=device),
                      torch.ones((num_blocks, num_kv_heads), dtype=torch.float32, device=device))


def _check_bounds(page_bounds, nb, Hkv, d, like):
    values, scales = page_bounds
    _require_cuda(values, scales)
    _same_device(like, values, scales)
    if values.dtype != torch.int8 or tuple(values.shape) != (nb, Hkv, 2, d) or \
            scales.dtype != torch.float32 or tuple(scales.shape) != (nb, Hkv):
        raise ValueError("page_bounds must be int8 [num_blocks, Hkv, 2, d] and float32 "
                         "[num_blocks, Hkv]")
    return values, scales


def update_page_bounds(key_cache, page_bounds, slots, block_size: int = 16, *,
                       kv_layout: str = "flat"):
    """Boxes of the pages that the tokens at ``slots`` [T] int64 closed (the slot at a
    page's last place; others are skipped), read from the cache. Call it after the step's
    keys are in the cache, with the step's slots. head_dim 64 or 128, block size 16 or 32.
    Returns page_bounds."""
    _require_cuda(key_cache, slots)
    nb, Hkv, d = _cache_dims(key_cache, block_size, kv_layout)
    dt = _DTYPES.get(key_cache.dtype)
    if dt is None:
        raise TypeError(f"unsupported dtype {key_cache.dtype}")
    values, scales = _check_bounds(page_bounds, nb, Hkv, d, key_cache)
    if slots.dtype != torch.int64 or slots.dim() != 1:
        raise ValueError("slots int64 [T] expected")
    _same_device(key_cache, slots)
    with _on(key_cache.device):
        st = _bounds(key_cache.data_ptr(), values.data_ptr(), scales.data_ptr(),
                     slots.data_ptr(), slots.shape[0], Hkv, d, block_size, nb, dt,
                     _LAYOUTS[kv_layout], _raw_stream(key_cache))
    if st:
        _lib.check(st, "update_page_bounds")
    return page_bounds


def sparse_paged_attention(query, key_cache, value_cache, page_bounds, block_tables, context_lens,
                           num_pages: int, block_size: int = 16, scale: float | None = None, *,
                           keep_first: int = 1, keep_last: int = 1, kv_layout: str = "flat",
                           workspace=None, out=None, selected=None):
    """Paged decode attention over ``num_pages`` pages of each (sequence, KV head).

    ``query`` [S, H, d], caches, ``block_tables``, ``context_lens``, ``scale`` (positive)
    and ``workspace`` as for ``paged_attention`` (bf16, fp16, or fp32 with the flat layout;
    head_dim 64 or 128, block size 16 or 32). ``page_bounds``: the boxes of the full pages
    (``update_page_bounds``). Always attended: the first ``keep_first`` and the last
    ``keep_last`` (>= 1) pages; the rest of ``num_pages`` are those whose box bounds the
    largest q.k of the group's query heads highest, ties to the lower page. The scores are
    exact whole-number arithmetic, so the choice depends on the inputs alone. Sequences of
    at most ``num_pages`` pages are attended whole. Returns (out [S, H, d], selected
    [S, Hkv, num_pages] int32: the pages in ascending order, -1 past their count)."""
    _require_cuda(query, key_cache, value_cache, block_tables, context_lens)
    if query.dim() != 3:
        raise ValueError("query [S, H, d] expected")
    S, H, Hkv, d, nb, maxb = _paged_shapes(query, key_cache, value_cache, block_tables,
                                           context_lens, block_size, kv_layout)
    _same_device(query, key_cache, value_cache, block_tables, context_lens)
    dt = _DTYPES.get(query.dtype)
    if dt is None or key_cache.dtype != query.dtype or value_cache.dtype != query.dtype:
        raise TypeError("query and caches must share a dtype: bfloat16, float16 or float32")
    values, scales = _check_bounds(page_bounds, nb, Hkv, d, query)
    if scale is not None and not scale > 0:
        raise ValueError("scale must be positive")
    if keep_first < 0 or keep_last < 1 or num_pages < keep_first + keep_last:
        raise ValueError("keep_first >= 0, keep_last >= 1 and num_pages >= their sum expected")
    out = _buffer(out, query.shape, query.dtype, query, "out")
    selected = _buffer(selected, (S, Hkv, num_pages), torch.int32, query, "selected")
    scratch = torch.empty(_scratch_ints(S, Hkv, maxb, num_pages), dtype=torch.int32,
                          device=query.device)
    ws, n = _workspace(query, H // Hkv, 1, d, block_size, workspace)
    with _on(query.device):
        st = _sparse(query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
                     out.data_ptr(), values.data_ptr(), scales.data_ptr(),
                     block_tables.data_ptr(), context_lens.data_ptr(), selected.data_ptr(),
                     scratch.data_ptr(), S, H, Hkv, d, block_size, maxb, nb, num_pages,
                     keep_first, keep_last, scale if scale is not None else 1 / math.sqrt(d), dt,
                     _LAYOUTS[kv_layout], ws.data_ptr() if ws is not None else None, n,
                     _raw_stream(query))
    if st:
        _lib.check(st, "sparse_paged_attention")
    return out, selected
