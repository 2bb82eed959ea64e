"""A paged K/V cache on the GPU: what fills it, and what a verification step of drafted tokens
does with it.  Not in the reference, whose K/V is contiguous (its README.md:139-141).

The pools are ``[num_pages, page_size, H_kv, D]``; logical row ``r`` of request ``j`` is row
``r % page_size`` of page ``block_table[j, r // page_size]``, and a *slot* is
``page * page_size + row``.  One step of a serving loop:

    plan = paged_block_tables(cached_lens, new_lens, free_pages, page_size=..., num_tokens=T,
                              block_table=block_table)
    mask = paged_tree_mask(parents, plan.cu_seqlens_q, max_nodes=n)   # drafted trees only
    for each layer:
        paged_kv_write(k, v, k_pages, v_pages, plan.slot_mapping)
        out, lse = b200_attn_paged_tree(q, k_pages, v_pages, plan.block_table,
                                        cu_seqlens_q=plan.cu_seqlens_q,
                                        seq_lens=plan.seq_lens, max_seqlen_q=n, tree_mask=mask)
    # after the model has chosen the accepted path of every request, for each layer:
    cached_lens = paged_kv_accept(k_pages, v_pages, plan.block_table, cached_lens, accepted,
                                  cu_seqlens_q=plan.cu_seqlens_q)

Nothing here copies to the host or validates device data: lengths, slots and tables are read by
the kernels, which keep every access inside the tensors that they were given.  With its tensors on
the device (a descale may also be a number) no call waits for the GPU, and every one can be
captured into a CUDA graph.  ``cu_seqlens_q``, ``seq_lens`` and descales of several heads are also
taken from the host; copying those waits for the stream and cannot be captured.
"""

from typing import NamedTuple, Optional

import torch

from . import _lib
from .attn_backend import as_i32, norm_descale, pool_strides, rows16

MAX_TREE_NODES = 4096   # paged_tree_mask: nodes of one tree
MAX_ACCEPT = 1024       # paged_kv_accept: accepted nodes of one request


class PagedPlan(NamedTuple):
    """What :func:`paged_block_tables` returns (all on the device)."""

    block_table: torch.Tensor   # int32 [nseq, max_pages], -1: not owned
    slot_mapping: torch.Tensor  # int64 [num_tokens], -1: no page, or padding
    cu_seqlens_q: torch.Tensor  # int32 [nseq + 1], sums of new_lens
    cu_seqlens_k: torch.Tensor  # int32 [nseq + 1], sums of seq_lens
    seq_lens: torch.Tensor      # int32 [nseq], cached_lens + new_lens
    pages: torch.Tensor         # int32 [2]: pages taken from free_pages, pages not provided


def _check_pools(k_pages, v_pages, *others):
    _lib.require_cuda(k_pages, v_pages, *others)
    assert k_pages.dim() == 4 and k_pages.shape == v_pages.shape, "pools are [pages, page, H_kv, D]"
    assert k_pages.dtype == v_pages.dtype, "the pools must share a dtype"
    assert k_pages.device == v_pages.device, "the pools must be on one device"


def paged_block_tables(cached_lens: torch.Tensor, new_lens: torch.Tensor,
                       free_pages: torch.Tensor, *, page_size: int, num_tokens: int,
                       block_table: Optional[torch.Tensor] = None,
                       max_pages: Optional[int] = None,
                       num_free: Optional[torch.Tensor] = None) -> PagedPlan:
    """Block table and slot map of one step, built on the GPU from the requests' lengths.

    Request ``j`` has ``cached_lens[j]`` tokens in the cache and adds ``new_lens[j]``.  The
    pages that its new tokens fall on and that it does not own yet are taken from
    ``free_pages`` (int32, used from its front) in the order of requests and pages.

    * ``block_table`` (int32 ``[nseq, max_pages]``): the requests' pages so far.  The owned
      pages are the first entries of a row, the rest is negative.  It is not changed.
      ``None``: no request owns a page; ``max_pages`` then gives the table's width.
    * ``num_tokens``: entries of the slot map, the tokens of the step (or more, for a padded
      step).  Entries behind the last request are -1.
    * ``num_free`` (int32 ``[1]``, on the device): entries of ``free_pages`` that are valid;
      ``None``: all.

    Returns a :class:`PagedPlan`.  When ``free_pages`` or a table row is too short, the pages
    that cannot be provided stay -1 in the table, their tokens get slot -1 (no K/V is written
    for them) and ``pages[1]`` counts them.  Sums of lengths must stay below 2^31; negative
    lengths count as 0.
    """
    _lib.require_cuda(cached_lens, new_lens, free_pages, block_table, num_free)
    dev = cached_lens.device
    assert cached_lens.dim() == 1 and cached_lens.shape == new_lens.shape, "lengths are [nseq]"
    nseq = cached_lens.shape[0]
    assert nseq >= 1, "at least one request"
    assert free_pages.dim() == 1, "free_pages is [num_free]"
    assert num_tokens >= 0 and page_size >= 1, "num_tokens >= 0 and page_size >= 1"
    if block_table is not None:
        assert block_table.dim() == 2 and block_table.shape[0] == nseq, "block_table is [nseq, max_pages]"
        assert max_pages is None or max_pages == block_table.shape[1], "max_pages differs from block_table"
        max_pages = block_table.shape[1]
        block_table = as_i32(block_table, dev)
    if max_pages is None:
        raise ValueError("max_pages is required without a block_table")
    if num_free is not None:
        num_free = as_i32(num_free, dev)
        assert num_free.numel() == 1, "num_free is one number"
    cached_lens, new_lens = as_i32(cached_lens, dev), as_i32(new_lens, dev)
    free_pages = as_i32(free_pages, dev)
    table = cached_lens.new_empty((nseq, max_pages))
    slots = cached_lens.new_empty(num_tokens, dtype=torch.int64)
    cu_q, cu_k, lens, pages = cached_lens.new_empty(3 * nseq + 4).unsafe_split_with_sizes(
        (nseq + 1, nseq + 1, nseq, 2))
    with _lib.on_device(dev):
        _lib.check(_lib.load().fa4cp_paged_block_tables(
            cached_lens.data_ptr(), new_lens.data_ptr(), nseq, free_pages.data_ptr(),
            free_pages.numel(), _lib.ptr(num_free), page_size, max_pages, _lib.ptr(block_table),
            table.data_ptr(), slots.data_ptr(), num_tokens, cu_q.data_ptr(), cu_k.data_ptr(),
            lens.data_ptr(), pages.data_ptr(), _lib.stream_of(table)), "paged_block_tables")
    _lib.count_launches()
    return PagedPlan(table, slots, cu_q, cu_k, lens, pages)


def paged_tree_mask(parents: torch.Tensor, cu_seqlens_q: torch.Tensor, *,
                    max_nodes: int) -> torch.Tensor:
    """Visibility bits of drafted trees: int64 ``[T, ceil(max_nodes / 64)]``, where bit ``m``
    of word ``w`` of a row says that the node sees node ``64 w + m`` of its tree (itself and
    its ancestors).

    ``parents`` (int32 ``[T]``): for each node the index of its parent within its own tree, -1
    for a child of the last cached token.  Parents come before their children; a parent that
    does not (or a negative one) counts as none.  ``cu_seqlens_q`` (int32 ``[nseq + 1]``)
    bounds the trees, ascending; ``max_nodes`` (at most 4096) bounds their sizes.  Rows outside
    every tree are 0, and so are those of a tree whose bounds leave the rows.  Built once a step,
    used by every layer."""
    _lib.require_cuda(parents)
    dev = parents.device
    assert parents.dim() == 1 and cu_seqlens_q.dim() == 1, "parents is [T], cu_seqlens_q [nseq + 1]"
    parents, cu = as_i32(parents, dev), as_i32(cu_seqlens_q, dev)
    total = parents.shape[0]
    mask = parents.new_empty((total, (max_nodes + 63) // 64), dtype=torch.int64)
    with _lib.on_device(dev):
        _lib.check(_lib.load().fa4cp_paged_tree_mask(
            parents.data_ptr(), cu.data_ptr(), cu.numel() - 1, total, max_nodes, mask.data_ptr(),
            _lib.stream_of(mask)), "paged_tree_mask")
    _lib.count_launches()
    return mask


def paged_kv_write(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
                   v_pages: torch.Tensor, slot_mapping: torch.Tensor, *,
                   k_descale: Optional[torch.Tensor] = None,
                   v_descale: Optional[torch.Tensor] = None) -> None:
    """Write the rows ``k``, ``v`` (``[T, H_kv, D]``; slices of a fused projection are taken
    as they are) into the page pools at ``slot_mapping`` (int64 ``[T]``), in place.

    Pools of the rows' dtype take copies; e4m3 pools take f16 / bf16 rows as
    ``e4m3(clamp(x / descale))`` with the descales (scalar, ``[H_kv]`` or ``(1, H_kv)``) that
    the attention multiplies back (``None``: 1); the attention reads an e4m3 cache under a bf16 or
    e4m3 q, whichever type the rows came from.  Tokens with a slot outside the pools (-1) are
    skipped.  Slots must differ: two tokens with one slot leave a mixture of their rows."""
    _check_pools(k_pages, v_pages, k, v, slot_mapping)
    num_pages, page_size, h_kv, d = k_pages.shape
    assert k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype, "k and v are [T, H_kv, D]"
    tokens, *row = k.shape
    assert row == [h_kv, d], "the rows and the pools differ in H_kv or D"
    assert slot_mapping.dim() == 1 and slot_mapping.numel() == tokens, "slot_mapping is [T]"
    dev = k_pages.device
    assert k.device == v.device == slot_mapping.device == dev, "tensors must be on the pools' device"
    quant = k_pages.dtype == torch.float8_e4m3fn and k.dtype != torch.float8_e4m3fn
    if not quant and (k_descale is not None or v_descale is not None):
        raise ValueError("descales apply to f16 / bf16 rows written into an e4m3 pool only")
    kd, vd = norm_descale(k_descale, h_kv, dev), norm_descale(v_descale, h_kv, dev)
    ks, vs = pool_strides(k_pages, "k_pages"), pool_strides(v_pages, "v_pages")
    k, v = rows16(k), rows16(v)
    slots = slot_mapping
    if slots.dtype is not torch.int64 or not slots.is_contiguous():
        slots = slots.to(torch.int64).contiguous()
    with _lib.on_device(dev):
        _lib.check(_lib.load().fa4cp_paged_kv_write(
            k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), k_pages.data_ptr(),
            v_pages.data_ptr(), ks, vs, num_pages, page_size, slots.data_ptr(), tokens, h_kv,
            d, _lib.dtype_code(k.dtype), _lib.dtype_code(k_pages.dtype), _lib.ptr(kd),
            _lib.ptr(vd), _lib.stream_of(k_pages)), "paged_kv_write")
    _lib.count_launches()


def paged_kv_accept(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    cached_lens: torch.Tensor, accepted: torch.Tensor, *,
                    cu_seqlens_q: torch.Tensor) -> torch.Tensor:
    """Keep the accepted path of every request: the K/V rows of its nodes, written behind the
    ``cached_lens[j]`` tokens of request ``j`` in tree order, move together in place, and the
    new lengths (int32 ``[nseq]``) are returned.

    ``accepted`` (int32 ``[nseq, A]``, A at most 1024): the accepted nodes of each request from
    the root on.  A row ends at its first entry that is negative, not below the tree's size
    ``cu_seqlens_q[j + 1] - cu_seqlens_q[j]``, or not above the entry before it (nodes of a
    path ascend, since parents come before children).  Row ``cached + i`` becomes what row
    ``cached + accepted[j, i]`` was; the rows behind the path keep what they hold.  Rows
    without a valid page are skipped."""
    _check_pools(k_pages, v_pages, block_table, cached_lens, accepted)
    num_pages, page_size, h_kv, d = k_pages.shape
    dev = k_pages.device
    nseq = cached_lens.shape[0]
    assert cached_lens.dim() == 1 and nseq >= 1, "cached_lens is [nseq]"
    assert block_table.dim() == 2 and block_table.shape[0] == nseq, "block_table is [nseq, max_pages]"
    assert accepted.dim() == 2 and accepted.shape[0] == nseq, "accepted is [nseq, A]"
    assert cu_seqlens_q.numel() == nseq + 1, "cu_seqlens_q is [nseq + 1]"
    ks, vs = pool_strides(k_pages, "k_pages"), pool_strides(v_pages, "v_pages")
    bt, cached = as_i32(block_table, dev), as_i32(cached_lens, dev)
    acc, cu = as_i32(accepted, dev), as_i32(cu_seqlens_q, dev)
    lens = cached.new_empty(nseq)
    with _lib.on_device(dev):
        _lib.check(_lib.load().fa4cp_paged_kv_accept(
            k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, num_pages, page_size, bt.data_ptr(),
            bt.shape[1], cached.data_ptr(), cu.data_ptr(), nseq, acc.data_ptr(), acc.shape[1],
            h_kv, d, _lib.dtype_code(k_pages.dtype), lens.data_ptr(), _lib.stream_of(k_pages)),
            "paged_kv_accept")
    _lib.count_launches()
    return lens
