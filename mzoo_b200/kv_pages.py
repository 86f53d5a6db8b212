"""Pages of a K / V cache, managed on the device: rows written into their pages (``append``),
pages taken for new tokens (``reserve``), shared between sequences (``fork``), released
(``free``), copied (``copy_pages``) and moved together (``compact``).  No counterpart in the
reference; ``mzoo_b200.gqa_attn.decode`` reads what these keep.

State (int32, contiguous, on the device): ``page_table [S, W]`` names the page of each
sequence's positions ``j * page .. (j + 1) * page`` (-1 = none), ``seq_lens [S]``, ``refs [P]``
counts the tables that name a page (0 = free).  A new page is always the lowest free id, in
the order of the sequences that ask.  Nothing here reads from the host: what cannot be done (a
position past the table, an id out of range, no free page) is left out and raised by
``mzoo_b200.check_errors()``, or at once with ``check=True``, as an ``MzbError`` whose ``code`` is
``_lib.MZB_ERR_TABLE``, ``MZB_ERR_PAGES`` or ``MZB_ERR_NO_PAGE`` (of several, the first).

``pools`` is a list of tensors ``[P, ...]`` whose pages ``pool[p]`` are dense (the K and V pools of
every layer, say); each is changed in place.  Tensors that need gradients are refused outside
``torch.no_grad()``.  Kernels: ``csrc/kv_pages.cu``.
"""

import torch

from . import ops
from ._lib import require_cuda


def _state(**tensors):
    first = -1
    for name, t in tensors.items():
        i = t.get_device()
        if first < 0:
            first = i
            require_cuda(t)
        assert i == first and t.dtype == torch.int32 and t.is_contiguous(), \
            f"{name} must be a contiguous int32 tensor on cuda:{first}, got {t.dtype} on {t.device}"
        assert t.dim() == (2 if name == "page_table" else 1), f"{name} has {t.dim()} dimensions: {tuple(t.shape)}"


def _no_grad(what, *tensors):
    assert not (torch.is_grad_enabled() and any([t.requires_grad for t in tensors])), \
        f"{what} has no backward: call it under torch.no_grad()"


def _table(page_table, seq_lens, refs):
    assert seq_lens.shape[0] == page_table.shape[0], \
        f"page_table {tuple(page_table.shape)} and seq_lens {tuple(seq_lens.shape)} name different sequences"
    assert page_table.shape[1] >= 1 and refs.shape[0] >= 1, "the page table and the pool must not be empty"


def _pools(what, pools, pages, dev):
    pools = list(pools)
    _no_grad(what, *pools)
    i = dev.index
    for p in pools:
        shape, step = p.shape, p.stride(0)
        assert p.get_device() == i and len(shape) >= 2 and shape[0] == pages, \
            f"each pool must be [{pages}, ...] on {dev}, got {tuple(shape)} on {p.device}"
        n, size = p.numel() // pages, p.element_size()
        assert (p.is_contiguous() or p[0].is_contiguous()) and (step >= n or pages == 1), \
            "a pool's pages must be dense and apart"
        assert n and not (n * size & 15 or (step * size & 15 and pages > 1) or p.storage_offset() * size & 15), \
            "a pool's pages must be 16-byte aligned and a multiple of 16 bytes"
    return pools


def _rows_ok(t, size, apart=False):
    """Dense rows on 16-byte boundaries (``apart``: no two of them the same memory)."""
    if t.storage_offset() * size & 15:
        return False
    if t.is_contiguous():  # rows are multiples of 16 bytes
        return True
    *outer, last = t.stride()
    if last != 1:
        return False
    for x in outer:
        if x * size & 15 or (apart and not x):
            return not any([n > 1 and (x * size & 15 or (apart and not x)) for n, x in zip(t.shape, outer)])
    return True


def append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
           starts: torch.Tensor, cu: torch.Tensor | None = None, *, check: bool = False) -> None:
    """Write k / v ``[T, Hkv, D]`` into k_pages / v_pages ``[P, Hkv, page, D]`` (any strides over dense
    rows): row i of sequence b, rows ``cu[b] .. cu[b+1]`` (``cu`` None: row b, one token each), goes
    to position ``starts[b] + i``."""
    if cu is None:
        _state(page_table=page_table, starts=starts)
    else:
        _state(page_table=page_table, starts=starts, cu=cu)
    dt, ks, ps = k.dtype, k.shape, k_pages.shape
    i = page_table.get_device()
    for t in (k, v, k_pages, v_pages):
        assert t.dtype == dt and t.get_device() == i, \
            f"k, v and the pools must be {dt} on cuda:{i}, got {t.dtype} on {t.device}"
    _no_grad("append", k, v, k_pages, v_pages)
    assert len(ks) == 3 and ks == v.shape, f"k and v must be [tokens, heads, D], got {tuple(ks)}, {tuple(v.shape)}"
    assert len(ps) == 4 and ps == v_pages.shape and ps[1] == ks[1] and ps[3] == ks[2] and ps[0] and ps[2], \
        f"the pools must be [pages, {ks[1]}, page, {ks[2]}], got {tuple(ps)}, {tuple(v_pages.shape)}"
    B, size, (rows, width) = starts.shape[0], k.element_size(), page_table.shape
    assert B >= 1 and rows == B and width >= 1, \
        f"page_table must have one row for each of the {B} sequences, got {rows} x {width}"
    assert ks[0] == B if cu is None else cu.shape[0] == B + 1, \
        f"rows of {B} sequences: cu must be [{B + 1}], or None with one row each (got {ks[0]} rows)"
    assert ks[2] * size % 16 == 0 and ks[1] >= 1, f"rows must be a multiple of 16 bytes, got {ks[2]} x {dt}"
    assert _rows_ok(k_pages, size, True) and _rows_ok(v_pages, size, True), "the pools need dense, 16-byte aligned rows"
    ops.kv_append(k if _rows_ok(k, size) else k.contiguous(), v if _rows_ok(v, size) else v.contiguous(), k_pages, v_pages,
                  page_table, starts, cu, check)


def reserve(page_table: torch.Tensor, seq_lens: torch.Tensor, refs: torch.Tensor, n_new: torch.Tensor, *, page_size: int,
            check: bool = False) -> torch.Tensor:
    """Room for ``n_new[b]`` more tokens of each sequence: takes the pages, raises seq_lens and returns
    the lengths before (``append``'s ``starts``).  A sequence that cannot have all of them (the
    table is too narrow, no free page) gets none and keeps its length.  Pages are given out in the order of
    the sequences, and none is passed over: behind the first one that the free pages do not
    suffice for, no sequence that needs a page gets one in this call."""
    _state(page_table=page_table, seq_lens=seq_lens, refs=refs, n_new=n_new)
    _table(page_table, seq_lens, refs)
    assert n_new.shape == seq_lens.shape, f"n_new must be {tuple(seq_lens.shape)}, got {tuple(n_new.shape)}"
    assert page_size >= 1, f"page_size must be positive, got {page_size}"
    return ops.kv_reserve(page_table, seq_lens, refs, n_new, int(page_size), check)


def free(page_table: torch.Tensor, seq_lens: torch.Tensor, refs: torch.Tensor, seqs: torch.Tensor, *,
         check: bool = False) -> None:
    """Release the sequences ``seqs``: their entries become -1, their lengths 0, and a page that no
    other table names is free."""
    _state(page_table=page_table, seq_lens=seq_lens, refs=refs, seqs=seqs)
    _table(page_table, seq_lens, refs)
    ops.kv_free(page_table, seq_lens, refs, seqs, check)


def fork(pools, page_table: torch.Tensor, seq_lens: torch.Tensor, refs: torch.Tensor, src: torch.Tensor,
         dst: torch.Tensor, *, page_size: int, check: bool = False) -> None:
    """Make sequence ``dst[i]`` a copy of ``src[i]``: what dst held is released, src's full pages are
    shared and a partly filled last page is copied to a page of its own (without a free page the
    copy ends at the last full one).  ``dst`` names distinct sequences, none of them in ``src``
    (one source may have many copies); other pairs are left out as an error."""
    _state(page_table=page_table, seq_lens=seq_lens, refs=refs, src=src, dst=dst)
    _table(page_table, seq_lens, refs)
    assert src.shape == dst.shape, f"src and dst must have one length, got {src.shape[0]} and {dst.shape[0]}"
    assert page_size >= 1, f"page_size must be positive, got {page_size}"
    ops.kv_fork(_pools("fork", pools, refs.shape[0], refs.device), page_table, seq_lens, refs, src, dst, int(page_size), check)


def compact(pools, page_table: torch.Tensor, refs: torch.Tensor, *, check: bool = False):
    """Move the n pages in use to the ids below n (only pages at or above n move, each into a hole
    below) -> (page_table, refs) after it, as new tensors.  The pools are changed in place, so
    the tables passed in are out of date afterwards."""
    _state(page_table=page_table, refs=refs)
    assert refs.shape[0] >= 1, "the pool must not be empty"
    return ops.kv_compact(_pools("compact", pools, refs.shape[0], refs.device), page_table, refs, check)


def copy_pages(pools, src: torch.Tensor, dst: torch.Tensor, *, check: bool = False) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` of every pool (both -1: nothing).  No destination may be
    named twice or be a source."""
    _state(src=src, dst=dst)
    pools = list(pools)
    assert pools, "copy_pages needs at least one pool"
    assert src.shape == dst.shape, f"src and dst must have one length, got {src.shape[0]} and {dst.shape[0]}"
    assert pools[0].dim() and pools[0].shape[0], "the pools must not be empty"
    ops.kv_copy_pages(_pools("copy_pages", pools, pools[0].shape[0], src.device), src, dst, check)
