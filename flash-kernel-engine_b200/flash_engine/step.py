"""The serving step around the paged decode, over CUDA tensors.

* ``plan_paged_step``        -- blocks, block tables, positions and cache slots of a step,
  from request lengths that live on the GPU;
* ``paged_qkv_append``       -- per-head QK norm, rotary embedding and cache write of the
  step's tokens in one pass over their QKV projection;
* ``update_page_bounds``     -- int8 boxes of the keys of the pages the step filled;
* ``sparse_paged_attention`` -- decode attention over the pages whose boxes score highest
  for the query.

Everything stays on the GPU and on the current stream: no call synchronises, and all can be
captured in a CUDA graph. With ``out=`` buffers the first three allocate nothing; the sparse
attention takes its scratch (the scores) from torch's allocator at every call. As in ``ops``,
inputs must be CUDA tensors (TypeError otherwise) and unsupported shapes raise.
"""

from __future__ import annotations

import ctypes
import os
from typing import NamedTuple

import torch

from . import _lib
from .ops import _workspace

_native = None


def _load():
    """The native binding, loaded when the first of these operators is called: the others of
    the package do without it."""
    global _native
    try:
        from . import _step_native as native
    except ImportError as e:
        raise ImportError(
            f"the native binding _step_native of {os.path.dirname(__file__)} cannot be loaded; "
            "build it with `make -C flash-kernel-engine_b200/csrc` (or "
            f"__graft_entry__.build()): {e}") from e
    native.bind(*(ctypes.cast(getattr(_lib.lib, n), ctypes.c_void_p).value for n in (
        "fe_plan_paged_step", "fe_paged_qkv_append", "fe_update_page_bounds",
        "fe_sparse_paged_attention", "fe_sparse_paged_attention_scratch_ints")))
    _native = native
    return native


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
    into (``max_tokens`` is then their length); they must share no memory with one another or
    with the inputs of this call (ValueError)."""
    native = _native or _load()
    return PagedStep(*native.plan(context_lens, new_lens, block_tables, free_blocks, free_state,
                                  block_size, max_tokens, finished, out))


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
    ``page_bounds``: also ``update_page_bounds`` of the pages this fills. ``out`` may share no
    memory with qkv or the caches (ValueError)."""
    native = _native or _load()
    return native.append(qkv, key_cache, value_cache, positions, slots, num_heads, block_size,
                         q_weight, k_weight, eps, rope, interleaved, kv_layout, page_bounds, out)


def new_page_bounds(num_blocks: int, num_kv_heads: int, head_dim: int, device) -> PageBounds:
    """Storage for the boxes of a cache of this shape."""
    return PageBounds(torch.zeros((num_blocks, num_kv_heads, 2, head_dim), dtype=torch.int8,
                                  device=device),
                      torch.ones((num_blocks, num_kv_heads), dtype=torch.float32, device=device))


def update_page_bounds(key_cache, page_bounds, slots, block_size: int = 16, *,
                       kv_layout: str = "flat"):
    """Boxes of the pages that the tokens at ``slots`` [T] int64 closed (the slot at a
    page's last place; others are skipped), read from the cache. Call it after the step's
    keys are in the cache, with the step's slots. head_dim 64 or 128, block size 16 or 32.
    Returns page_bounds."""
    (_native or _load()).bounds(key_cache, page_bounds, slots, block_size, kv_layout)
    return page_bounds


def sparse_paged_attention(query, key_cache, value_cache, page_bounds, block_tables, context_lens,
                           num_pages: int, block_size: int = 16, scale: float | None = None, *,
                           keep_first: int = 1, keep_last: int = 1, kv_layout: str = "flat",
                           workspace=None, out=None, selected=None):
    """Paged decode attention over ``num_pages`` pages of each (sequence, KV head).

    ``query`` [S, H, d], caches, ``block_tables``, ``context_lens``, ``scale`` (positive in fp32)
    and ``workspace`` as for ``paged_attention`` (bf16, fp16, or fp32 with the flat layout;
    head_dim 64 or 128, block size 16 or 32). ``page_bounds``: the boxes of the full pages
    (``update_page_bounds``). Always attended: the first ``keep_first`` and the last
    ``keep_last`` (>= 1) pages; the rest of ``num_pages`` are those with the highest scores,
    ties to the lower page. A page's score is the largest product that a key inside its box
    could have with a query head of the group, each head rounded to 8-bit whole numbers and a
    power of two: near an upper bound of the page's q.k, above or below it by the rounding of
    the query, and loose where one channel's keys are far larger than the others', which share
    its exponent. The scores are exact whole-number arithmetic, so the choice depends on the
    inputs alone. Sequences of at most ``num_pages`` pages are attended whole. bf16 and fp16
    round the softmax weights to 16 bits for the product with V, as ``paged_attention`` does.
    Returns (out [S, H, d], selected
    [S, Hkv, num_pages] int32: the pages in ascending order, -1 past their count)."""
    native = _native or _load()
    if workspace is not None or not _fused(query, key_cache, num_pages, kv_layout):
        workspace = _decode_workspace(query, key_cache, block_size, workspace)
    return native.sparse(query, key_cache, value_cache, page_bounds, block_tables, context_lens,
                         num_pages, block_size, scale, keep_first, keep_last, kv_layout,
                         workspace, out, selected)


def _fused(query, key_cache, num_pages, kv_layout):
    """Calls whose attention is not the paged decode, so that they need no workspace (a call
    with neither would take the library's; malformed ones are refused by the native checks)."""
    return (isinstance(query, torch.Tensor) and isinstance(key_cache, torch.Tensor)
            and (query.dim() != 3 or key_cache.dim() < 4
                 or (query.dtype is not torch.float32 and kv_layout == "flat"
                     and num_pages <= 8192 and query.shape[1] <= 16 * key_cache.shape[1])))


def _decode_workspace(query, key_cache, block_size, workspace):
    """The decode's workspace for one KV head a sequence, or None where paged_attention
    would take the library's (or where the native checks will refuse the call)."""
    if not (isinstance(query, torch.Tensor) and isinstance(key_cache, torch.Tensor)
            and query.is_cuda and query.dim() == 3 and key_cache.dim() >= 4) or \
            key_cache.shape[1] == 0 or query.shape[1] % key_cache.shape[1]:
        return workspace
    return _workspace(query, query.shape[1] // key_cache.shape[1], 1, query.shape[2], block_size,
                      workspace)[0]
