"""Pages of a K / V cache, managed on the device: rows written into their pages (``append``),
pages taken for new tokens (``reserve``), shared between sequences (``fork``), released
(``free``), copied (``copy_pages``) and moved together (``compact``).  No counterpart in the
reference; ``mzoo_b200.gqa_attn.decode`` reads what these keep.

State (int32, contiguous, on the device): ``page_table [S, W]`` names the page of each
sequence's positions ``j * page .. (j + 1) * page`` (-1 = none), ``seq_lens [S]``, ``refs [P]``
counts the tables that name a page (0 = free).  A new page is always the lowest free id, in
the order of the sequences that ask.  Nothing here reads from the host: what cannot be done (a
position past the table, an id out of range, no free page) is left out and raised by
``mzoo_b200.check_errors()``, or at once with ``check=True``.

``pools`` is a list of tensors ``[P, ...]`` whose pages ``pool[p]`` are dense (the K and V pools of
every layer, say); each is changed in place.  Kernels: ``csrc/kv_pages.cu``.
"""

import torch

from . import ops
from ._lib import require_cuda


def _state(**tensors):
    require_cuda(*tensors.values())
    dev = next(iter(tensors.values())).device
    for name, t in tensors.items():
        assert t.dtype == torch.int32 and t.is_contiguous() and t.device == dev, \
            f"{name} must be a contiguous int32 tensor on {dev}, got {t.dtype} on {t.device}"
        want = 2 if name == "page_table" else 1
        assert t.dim() == want, f"{name} must have {want} dimension(s), got {tuple(t.shape)}"


def _table(page_table, seq_lens, refs):
    assert seq_lens.shape[0] == page_table.shape[0], \
        f"page_table {tuple(page_table.shape)} and seq_lens {tuple(seq_lens.shape)} name different sequences"
    assert page_table.shape[1] >= 1 and refs.shape[0] >= 1, "the page table and the pool must not be empty"


def _pools(pools, pages, dev):
    pools = list(pools)
    for p in pools:
        require_cuda(p)
        assert p.device == dev and p.dim() >= 2 and p.shape[0] == pages, \
            f"each pool must be [{pages}, ...] on {dev}, got {tuple(p.shape)} on {p.device}"
        assert p[0].is_contiguous() and p.stride(0) >= p[0].numel(), "a pool's pages must be dense and apart"
        n = p.element_size()
        assert p[0].numel() * n % 16 == 0 and p.stride(0) * n % 16 == 0 and p.storage_offset() * n % 16 == 0 and p[0].numel(), \
            "a pool's pages must be 16-byte aligned and a multiple of 16 bytes"
    return pools


def append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
           starts: torch.Tensor, cu: torch.Tensor | None = None, *, check: bool = False) -> None:
    """Write k / v ``[T, Hkv, D]`` into k_pages / v_pages ``[P, Hkv, page, D]`` (any strides over dense
    rows): row i of sequence b, rows ``cu[b] .. cu[b+1]`` (``cu`` None: row b, one token each), goes
    to position ``starts[b] + i``."""
    require_cuda(k, v, k_pages, v_pages)
    _state(page_table=page_table, starts=starts, **({} if cu is None else {"cu": cu}))
    dt, dev = k.dtype, k.device
    for t in (v, k_pages, v_pages):
        assert t.dtype == dt and t.device == dev, f"k, v and the pools must be {dt} on {dev}, got {t.dtype} on {t.device}"
    assert page_table.device == dev, f"page_table must be on {dev}, got {page_table.device}"
    assert k.dim() == 3 and k.shape == v.shape, f"k and v must be [tokens, heads, D], got {tuple(k.shape)}, {tuple(v.shape)}"
    assert k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.shape[1] == k.shape[1] \
        and k_pages.shape[3] == k.shape[2] and k_pages.numel(), \
        f"the pools must be [pages, {k.shape[1]}, page, {k.shape[2]}], got {tuple(k_pages.shape)}, {tuple(v_pages.shape)}"
    B, size = starts.shape[0], k.element_size()
    assert B >= 1 and page_table.shape[0] == B and page_table.shape[1] >= 1, \
        f"page_table must have one row for each of the {B} sequences, got {tuple(page_table.shape)}"
    assert (cu is None and k.shape[0] == B) or (cu is not None and cu.shape[0] == B + 1), \
        f"rows of {B} sequences: cu must be [{B + 1}], or None with one row each (got {k.shape[0]} rows)"
    assert k.shape[2] * size % 16 == 0, f"rows must be a multiple of 16 bytes, got {k.shape[2]} x {dt}"

    def ok(t):
        return t.stride(-1) == 1 and t.storage_offset() * size % 16 == 0 and all(
            n <= 1 or s * size % 16 == 0 for n, s in zip(t.shape[:-1], t.stride()[:-1]))
    for t in (k_pages, v_pages):
        assert ok(t) and all(n <= 1 or s > 0 for n, s in zip(t.shape, t.stride())), \
            "the pools need dense, 16-byte aligned rows"
    ops.kv_append(k if ok(k) else k.contiguous(), v if ok(v) else v.contiguous(), k_pages, v_pages, page_table, starts,
                  cu, check)


def reserve(page_table: torch.Tensor, seq_lens: torch.Tensor, refs: torch.Tensor, n_new: torch.Tensor, *, page_size: int,
            check: bool = False) -> torch.Tensor:
    """Room for ``n_new[b]`` more tokens of each sequence: takes the pages, raises seq_lens and returns
    the lengths before (``append``'s ``starts``).  A sequence that cannot have all of them (the
    table is too narrow, no free page) gets none and keeps its length."""
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
    ops.kv_fork(_pools(pools, refs.shape[0], refs.device), page_table, seq_lens, refs, src, dst, int(page_size), check)


def compact(pools, page_table: torch.Tensor, refs: torch.Tensor, *, check: bool = False):
    """Move the n pages in use to the ids below n (only pages at or above n move, each into a hole
    below) -> (page_table, refs) after it, as new tensors.  The pools are changed in place, so
    the tables passed in are out of date afterwards."""
    _state(page_table=page_table, refs=refs)
    assert refs.shape[0] >= 1, "the pool must not be empty"
    return ops.kv_compact(_pools(pools, refs.shape[0], refs.device), page_table, refs, check)


def copy_pages(pools, src: torch.Tensor, dst: torch.Tensor, *, check: bool = False) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` of every pool (both -1: nothing).  No destination may be
    named twice or be a source."""
    _state(src=src, dst=dst)
    pools = list(pools)
    assert pools, "copy_pages needs at least one pool"
    assert src.shape == dst.shape, f"src and dst must have one length, got {src.shape[0]} and {dst.shape[0]}"
    ops.kv_copy_pages(_pools(pools, pools[0].shape[0], src.device), src, dst, check)
