"""A serving step over a paged K/V cache, around the paged attention call.

No counterpart in the reference, which has no cache.  In the order of a step:

* ``extend_block_table`` gives the step's new tokens their pages, cache slots,
  positions and offsets, on the GPU, from the requests' lengths;
* ``paged_append`` norms and rotates the new queries and keys
  (``rotary.py``) and writes keys and values into the cache;
* then, with the step's ``seqlens_attended``,
  ``scaled_dot_product_attention_paged`` (``varlen.py``) over all of the
  cache, or attention over a part of it: ``update_page_means`` keeps the mean
  key of every full page, ``select_pages`` scores the pages by it for each
  token and K/V head, and ``scaled_dot_product_attention_paged_sparse``
  attends to the selected pages only.

All are forward only and capture into CUDA graphs: nothing is read back, and
rows of a padded batch behind the last request are left alone.  Indices that
would reach outside a tensor are refused on the GPU (nothing is read or
written there) and set the device status (``_abi.device_status``).
"""

from __future__ import annotations

import math
from numbers import Real
from typing import NamedTuple

import torch

from .rotary import _ptr, check_backend, check_eps, check_table, check_weights, launch, row_arg

# block-table width that select_pages takes (FA_MAX_SELECT_PAGES of include/fa_b200.h)
MAX_SELECT_PAGES = 16384


def _check_page_size(page_size) -> None:
    if isinstance(page_size, bool) or not isinstance(page_size, int) or page_size < 16 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two of at least 16")


def _check_int32(name: str, t, ndim: int, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != torch.int32 or t.ndim != ndim or t.device != device:
        raise ValueError(f"{name} must be a {ndim}-D int32 tensor on the same device as the others")


def _check_cache(name: str, t, dtype, device) -> torch.Size:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    shape = t.shape
    if len(shape) != 4 or 0 in shape:
        raise ValueError(f"{name} must have shape (num_pages, page_size, heads, head_dim); got {tuple(shape)}")
    if not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{name} must be contiguous and start on a 16-byte boundary")
    if shape[0] * shape[1] > 0x7fffffff:
        raise ValueError(f"{name} must have fewer than 2**31 slots")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must have the same dtype and device as the others")
    return shape


def _check_caches(k_cache, v_cache, dtype, device) -> torch.Size:
    shape = _check_cache("k_cache", k_cache, dtype, device)
    if _check_cache("v_cache", v_cache, dtype, device) != shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    return shape


def _check_no_grad(*tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("the paged K/V path is forward only; run it under torch.no_grad()")


class PagedStep(NamedTuple):
    """What ``extend_block_table`` returns; all on the GPU.  ``cu_seqlens_q``
    (requests + 1,), ``seqlens_k`` (requests,), ``positions`` and
    ``slot_mapping`` (total_q,), ``free_next`` (1,) int32; ``fits``
    (requests,) bool."""

    cu_seqlens_q: torch.Tensor
    seqlens_k: torch.Tensor
    positions: torch.Tensor
    slot_mapping: torch.Tensor
    fits: torch.Tensor
    free_next: torch.Tensor

    @property
    def seqlens_attended(self) -> torch.Tensor:
        """``seqlens_k`` for the calls behind the append: 0 where the request
        does not fit, so that its rows, which are in the batch all the same,
        see no key and complete no page.  (One small launch a use; a step
        whose requests are known to fit can pass ``seqlens_k``.)"""
        return self.seqlens_k * self.fits


def extend_block_table(block_table, seqlens_cached, seqlens_new, free_pages, free_start, *, page_size: int,
                       total_q: int) -> PagedStep:
    """Make room in the cache for a step's new tokens.

    ``block_table``: int32 ``(requests, max_pages)``, the first
    ``ceil(seqlens_cached / page_size)`` entries of a row its pages; the new
    ones are appended in place, other entries stay as they are.
    ``seqlens_cached``, ``seqlens_new``: int32 ``(requests,)``, tokens in the
    cache and new ones (either may be 0; negative counts as 0).
    ``free_pages``: int32 page ids; those from entry ``free_start[0]`` on are
    free and are taken in order, ``free_next`` is the start for the next step.
    ``total_q``: rows of the packed batch, at least the sum of
    ``seqlens_new``; rows behind the last request get position 0 and slot -1.

    A request that needs more pages than its row has, or rows behind
    ``total_q``, takes nothing; when the free pages run out, the request that
    lacks them and all after it take nothing.  Such a request has ``fits``
    False, slots of -1 and the ``seqlens_k`` it had, and its rows stay in the
    batch: the calls behind ``paged_append`` take ``seqlens_attended`` of the
    result, with ``seqlens_k`` those rows would stand at the positions of the
    request's last cached tokens."""
    if not isinstance(block_table, torch.Tensor):
        raise TypeError("block_table must be a torch.Tensor")
    dev = block_table.device
    _check_int32("block_table", block_table, 2, dev)
    for name, t in (("seqlens_cached", seqlens_cached), ("seqlens_new", seqlens_new), ("free_pages", free_pages),
                    ("free_start", free_start)):
        _check_int32(name, t, 1, dev)
    requests, width = block_table.shape
    if requests == 0 or width == 0:
        raise ValueError("block_table dimensions must all be greater than zero")
    if not block_table.is_contiguous():
        raise ValueError("block_table must be contiguous (it is extended in place)")
    if seqlens_cached.shape[0] != requests or seqlens_new.shape[0] != requests:
        raise ValueError("seqlens_cached and seqlens_new must have one entry per row of block_table")
    if free_start.shape[0] != 1:
        raise ValueError("free_start must have one entry")
    _check_page_size(page_size)
    if width * page_size > 0x7fffffff:
        raise ValueError("max_pages * page_size must be below 2**31")
    if isinstance(total_q, bool) or not isinstance(total_q, int) or not 0 <= total_q <= 0x7fffffff:
        raise ValueError("total_q must be a non-negative int")
    if dev.type != "cuda":
        raise RuntimeError("B200 CUDA backend is unavailable: the B200 kernel requires a CUDA tensor")
    seqlens_cached, seqlens_new, free_pages = (t.contiguous() for t in (seqlens_cached, seqlens_new, free_pages))
    # one allocation for the int32 outputs
    out = block_table.new_empty(2 * requests + 2 + 2 * total_q)
    cu, sk, pos, slots, nxt = out.split_with_sizes((requests + 1, requests, total_q, total_q, 1))
    fits = torch.empty(requests, device=dev, dtype=torch.bool)
    cu_at = out.data_ptr()
    sk_at = cu_at + 4 * (requests + 1)
    pos_at = sk_at + 4 * requests
    slots_at = pos_at + 4 * total_q
    launch(block_table, "fa_extend_block_table", None, block_table.data_ptr(), seqlens_cached.data_ptr(),
           seqlens_new.data_ptr(), free_pages.data_ptr(), free_start.data_ptr(), cu_at, sk_at, pos_at, slots_at,
           fits.data_ptr(), slots_at + 4 * total_q, requests, width, free_pages.shape[0], page_size, total_q)
    return PagedStep(cu, sk, pos, slots, fits, nxt)


def paged_append(query, key, value, k_cache, v_cache, slot_mapping, table, positions, *, query_weight=None,
                 key_weight=None, eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    """Norm and rotate a step's packed queries and keys as ``qk_norm_rotary``
    does, write keys and values to the cache and return the queries, all in
    one pass.

    ``query``: ``(total, Hq, D)``; ``key``, ``value``: ``(total, Hkv, D)``;
    views of a fused projection are read in place.  ``k_cache``, ``v_cache``:
    contiguous ``(num_pages, page_size, Hkv, D)``, written in place at row
    ``slot_mapping[t]`` (int32, ``page * page_size + row``) of their
    ``num_pages * page_size`` rows; a slot of -1 writes nothing,
    and the token may be at any position (its query is NaN where the table
    has no row for it).  Other slots of one call must differ.  ``positions``: int32 ``(total,)``.  The weights, ``eps``
    and ``interleaved`` as in ``qk_norm_rotary``."""
    for name, t in (("query", query), ("key", key), ("value", value)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        shape = t.shape
        if len(shape) != 3 or 0 in shape:
            raise ValueError(f"{name} must have shape (total, heads, head_dim), no dimension zero; got {tuple(shape)}")
        if t is not query and (t.dtype != query.dtype or t.device != query.device):
            raise ValueError("query, key, and value must have the same dtype and device")
    total, hq, d = query.shape
    dev = query.device
    key_shape = key.shape
    if key_shape != value.shape:
        raise ValueError("key and value must have the same shape")
    if key_shape[0] != total or key_shape[2] != d:
        raise ValueError("query and key must have the same number of rows and head dimension")
    pages, page_size, hkv, cache_d = _check_caches(k_cache, v_cache, query.dtype, dev)
    if hkv != key_shape[1] or cache_d != d:
        raise ValueError("the caches must have the key's heads and head dimension")
    for name, t in (("slot_mapping", slot_mapping), ("positions", positions)):
        _check_int32(name, t, 1, dev)
        if t.shape[0] != total:
            raise ValueError(f"{name} must have one entry per row of query")
    if not isinstance(interleaved, bool):
        raise TypeError("interleaved must be a bool")
    check_eps(eps)
    check_table(table, d, dev)
    check_weights(query_weight, key_weight, query)
    _check_no_grad(query, key, value, query_weight, key_weight)
    check_backend(query)
    q, qp, qs = row_arg(query)
    k, kp, ks = row_arg(key)
    v, vp, vs = row_arg(value)
    slots, pos = slot_mapping.contiguous(), positions.contiguous()
    if query_weight is not None:
        query_weight, key_weight = query_weight.contiguous(), key_weight.contiguous()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    launch(q, "fa_paged_append", q.dtype, qp, kp, vp, out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
           slots.data_ptr(), table.data_ptr(), pos.data_ptr(), _ptr(query_weight), _ptr(key_weight), total, hq, hkv, d,
           pages * page_size, *table.shape, interleaved,
           query_weight is not None and query_weight.dtype == torch.float32, qs.at, ks.at, vs.at, float(eps))
    return out


def _check_step(block_table, cu_seqlens_q, seqlens_k, device) -> torch.Size:
    _check_int32("block_table", block_table, 2, device)
    _check_int32("cu_seqlens_q", cu_seqlens_q, 1, device)
    _check_int32("seqlens_k", seqlens_k, 1, device)
    shape = block_table.shape
    if 0 in shape:
        raise ValueError("block_table dimensions must all be greater than zero")
    if cu_seqlens_q.shape[0] != shape[0] + 1 or seqlens_k.shape[0] != shape[0]:
        raise ValueError("block_table and seqlens_k must have one row per sequence of cu_seqlens_q")
    return shape


def update_page_means(k_cache, page_means, block_table, cu_seqlens_q, seqlens_k, *, total_q: int | None = None):
    """Write the mean key of every page that a step's tokens completed.

    ``k_cache``: contiguous ``(num_pages, page_size, Hkv, D)``, the step's keys
    included; ``page_means``: contiguous ``(num_pages, Hkv, D)`` in the cache's
    type, updated in place at the completed pages and returned.
    ``block_table``, ``cu_seqlens_q``, ``seqlens_k`` as in
    ``scaled_dot_product_attention_paged``: the rows of a sequence are its
    last keys.  ``total_q``: rows of the packed batch when the caller has it;
    None takes room for a step that fills the table.  Means are summed in 64
    bits and do not depend on the order of the sum.  A sequence with more keys
    than its row of ``block_table`` holds is refused on the GPU: no mean of it
    is written."""
    if not isinstance(k_cache, torch.Tensor):
        raise TypeError("k_cache must be a torch.Tensor")
    num_pages, page_size, hkv, d = _check_cache("k_cache", k_cache, k_cache.dtype, k_cache.device)
    _check_page_size(page_size)
    if not isinstance(page_means, torch.Tensor):
        raise TypeError("page_means must be a torch.Tensor")
    if (tuple(page_means.shape) != (num_pages, hkv, d) or page_means.dtype != k_cache.dtype
            or page_means.device != k_cache.device or not page_means.is_contiguous() or page_means.data_ptr() % 16):
        raise ValueError("page_means must be a contiguous (num_pages, heads, head_dim) tensor of the cache's dtype "
                         "and device")
    batch, width = _check_step(block_table, cu_seqlens_q, seqlens_k, k_cache.device)
    if width * page_size > 0x7fffffff:
        raise ValueError("max_pages_per_seq * page_size must be below 2**31")
    if total_q is None:
        total_q = min(batch * width * page_size, 0x7fffffff)
    elif isinstance(total_q, bool) or not isinstance(total_q, int) or not 0 < total_q <= 0x7fffffff:
        raise ValueError("total_q must be a positive int or None")
    _check_no_grad(k_cache, page_means)
    check_backend(k_cache)
    table, cu, lens = block_table.contiguous(), cu_seqlens_q.contiguous(), seqlens_k.contiguous()
    launch(k_cache, "fa_page_means", k_cache.dtype, k_cache.data_ptr(), page_means.data_ptr(), table.data_ptr(),
           cu.data_ptr(), lens.data_ptr(), batch, hkv, d, num_pages, page_size, width, total_q)
    return page_means


def _check_query(query) -> None:
    if not isinstance(query, torch.Tensor):
        raise TypeError("query must be a torch.Tensor")
    if query.ndim != 3:
        raise ValueError(f"query must have shape (total, heads, head_dim); got {tuple(query.shape)}")
    if 0 in query.shape:
        raise ValueError("query dimensions must all be greater than zero")


def select_pages(query, page_means, block_table, cu_seqlens_q, seqlens_k, *, page_size: int, num_selected: int,
                 sink_pages: int = 1, local_pages: int = 1) -> torch.Tensor:
    """Choose the pages that each new token attends to.

    ``query``: packed ``(total_q, Hq, D)``, as it enters the attention;
    ``page_means``: ``update_page_means``'s, up to date for every full page.
    A page's score for a token and K/V head is the highest dot product of one
    of the group's query heads with the page's mean key, summed in 64 bits and
    rounded to fp32.  Kept are the first ``sink_pages`` pages of the sequence,
    the ``local_pages`` up to and with the token's own, and those of the
    highest score (of equal ones the lower page; NaN is the lowest) up to
    ``num_selected`` in all.  Returns int32 ``(total_q, Hkv, num_selected)``:
    page indices in the sequence, ascending, -1 behind the last; all pages up
    to the token's own when there are no more than ``num_selected``."""
    _check_query(query)
    if not isinstance(page_means, torch.Tensor):
        raise TypeError("page_means must be a torch.Tensor")
    total, hq, d = query.shape
    if (page_means.ndim != 3 or 0 in page_means.shape or page_means.shape[2] != d or page_means.dtype != query.dtype
            or page_means.device != query.device or not page_means.is_contiguous() or page_means.data_ptr() % 16):
        raise ValueError("page_means must be a contiguous (num_pages, heads, head_dim) tensor of the query's head "
                         "dimension, dtype and device")
    hkv = page_means.shape[1]
    if hq % hkv:
        raise ValueError("the number of query heads must be divisible by the number of key/value heads")
    batch, width = _check_step(block_table, cu_seqlens_q, seqlens_k, query.device)
    _check_page_size(page_size)
    if width > MAX_SELECT_PAGES:
        raise ValueError(f"block_table may be {MAX_SELECT_PAGES} pages wide for page selection; got {width}")
    if width * page_size > 0x7fffffff or page_means.shape[0] * page_size > 0x7fffffff:
        raise ValueError("page counts times page_size must be below 2**31")
    for name, v, least in (("num_selected", num_selected, 1), ("sink_pages", sink_pages, 0),
                           ("local_pages", local_pages, 1)):
        if isinstance(v, bool) or not isinstance(v, int) or v < least:
            raise ValueError(f"{name} must be an int of at least {least}")
    if sink_pages + local_pages > num_selected:
        raise ValueError("sink_pages + local_pages must not be above num_selected")
    if num_selected * page_size > 0x3fffffff:
        raise ValueError("num_selected * page_size must be below 2**30")
    _check_no_grad(query, page_means)
    check_backend(query)
    q, qp, qs = row_arg(query)
    table, cu, lens = block_table.contiguous(), cu_seqlens_q.contiguous(), seqlens_k.contiguous()
    out = block_table.new_empty((total, hkv, num_selected))
    launch(q, "fa_select_pages", q.dtype, qp, page_means.data_ptr(), table.data_ptr(), cu.data_ptr(), lens.data_ptr(),
           out.data_ptr(), batch, hq, hkv, d, total, page_means.shape[0], page_size, width, num_selected, sink_pages,
           local_pages, qs.at)
    return out


def scaled_dot_product_attention_paged_sparse(query, k_cache, v_cache, block_table, cu_seqlens_q, seqlens_k,
                                              page_indices, *, scale: float | None = None,
                                              enable_gqa: bool = False) -> torch.Tensor:
    """Attention of packed queries over listed pages of a paged K/V cache
    (forward only; made for decode, where each sequence brings one query or a
    few).

    ``query``, the caches, ``block_table``, ``cu_seqlens_q`` and ``seqlens_k``
    as in ``scaled_dot_product_attention_paged`` with ``is_causal=True``: row
    ``i`` of a sequence's ``nq`` sees its keys ``j <= i + nk - nq``.
    ``page_indices``: int32 ``(total_q, Hkv, n)``, for each row and K/V head
    the pages it attends to by their index in the sequence, as
    ``select_pages`` returns them; -1 and pages behind the row's own are
    skipped, and a page listed twice counts twice.  Rows that see no listed
    key, and rows behind the last sequence, get zeros.  Cache rows behind a
    token's position may hold anything.  The default ``scale`` is
    ``D ** -0.5``."""
    _check_query(query)
    if not isinstance(enable_gqa, bool):
        raise TypeError("enable_gqa must be a bool")
    if scale is not None and (not isinstance(scale, Real) or not math.isfinite(float(scale))):
        raise ValueError("scale must be a finite real number or None")
    total, hq, d = query.shape
    dev = query.device
    num_pages, page_size, hkv, cache_d = _check_caches(k_cache, v_cache, query.dtype, dev)
    _check_page_size(page_size)
    if cache_d != d:
        raise ValueError("the caches must have the query's head dimension")
    if hq != hkv and not enable_gqa:
        raise ValueError(
            "query has a different number of heads from key/value; pass "
            "enable_gqa=True to use grouped-query attention")
    if hq % hkv:
        raise ValueError("the number of query heads must be divisible by the number of key/value heads")
    batch, width = _check_step(block_table, cu_seqlens_q, seqlens_k, dev)
    _check_int32("page_indices", page_indices, 3, dev)
    rows, heads, n = page_indices.shape
    if rows != total or heads != hkv or n == 0:
        raise ValueError("page_indices must have shape (total_q, key/value heads, n)")
    if width * page_size > 0x7fffffff or n * page_size > 0x3fffffff:
        raise ValueError("block_table and page_indices are too wide for this page_size")
    _check_no_grad(query, k_cache, v_cache)
    check_backend(query)
    q, qp, qs = row_arg(query)
    table, cu, lens = block_table.contiguous(), cu_seqlens_q.contiguous(), seqlens_k.contiguous()
    pages = page_indices.contiguous()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    launch(q, "fa_fwd_paged_sparse", q.dtype, qp, k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
           table.data_ptr(), cu.data_ptr(), lens.data_ptr(), pages.data_ptr(), batch, hq, hkv, d, total, num_pages,
           page_size, width, n, float(scale) if scale is not None else d ** -0.5, qs.at)
    return out
