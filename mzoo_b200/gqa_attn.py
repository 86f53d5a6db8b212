"""Dense causal attention with grouped K / V heads for serving: whole prompts packed one after
another (``prefill``) and one new token per sequence over a paged cache (``decode``).  No
counterpart in the reference's kernel packages: these are the full-attention layers that a
model mixes with the window and sparse ones.

``prefill`` row i of a sequence with nq new tokens and nk keys sees the keys
``j <= i + nk - nq`` (the last token sees all of them, so a prompt can be run in chunks over
keys that grow); head h reads K / V head ``h // (Hq // Hkv)``.  Both return the output in q's
type and the natural-log-sum-exp in fp32; a row that sees no key, or only keys whose scores are
-inf, has output 0 and lse -inf.  An infinite value of v that a row sees makes that channel of its
output infinite in ``prefill``, infinite or NaN in ``decode`` (weights in two parts).
fp32 softmax statistics and accumulation; ``prefill`` rounds each softmax weight to v's type for the
product with v (an error of at most 2^-8 (bf16) or 2^-11 (f16) of sum_j p_j |v_j|), ``decode`` keeps the
weights as two numbers of it; forward only.  The cache's pages are written,
shared and moved by ``mzoo_b200.kv_pages``; the kernels are ``csrc/gqa_prefill.cu`` and
``csrc/gqa_decode.cu``.
"""

import torch

from . import ops
from ._lib import require_cuda

HEAD_DIMS = (64, 96, 128)
PAGE_SIZES = (16, 32, 64, 128)
_TYPES = (torch.bfloat16, torch.float16)


def _check_types(what, q, k, v, *ints):
    dt, i = q.dtype, q.get_device()
    if i < 0 or k.get_device() != i or v.get_device() != i:
        require_cuda(q, k, v, *ints)
        raise AssertionError(f"q, k and v must be on one device, got {q.device}, {k.device}, {v.device}")
    for t in ints:
        if t.get_device() != i:
            require_cuda(t)
            raise AssertionError(f"all tensors must be on {q.device}, got one on {t.device}")
    assert dt in _TYPES, f"{what} supports bf16 / f16, got {dt}"
    assert k.dtype == dt and v.dtype == dt, f"q, k and v must have one type, got {dt}, {k.dtype}, {v.dtype}"
    assert not ((q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled()), \
        f"{what} has no backward: call it under torch.no_grad()"


def _check_heads(qs, hkv):
    assert len(qs) == 3 and qs[2] in HEAD_DIMS, f"q must be [tokens, heads, D in {HEAD_DIMS}], got {tuple(qs)}"
    hq = qs[1]
    assert hq >= 1 and hkv >= 1 and hq % hkv == 0 and hq // hkv <= 128, \
        f"query heads must be a multiple (at most 128) of the K / V heads, got {hq} and {hkv}"


def _aligned(t: torch.Tensor) -> bool:
    """Whether the kernels can address t in place: dense rows, 16-byte aligned (the base address of
    foreign storage is checked by the library), no broadcast dimension."""
    if t.storage_offset() & 7:
        return False
    if t.is_contiguous():  # head dims are multiples of 8
        return True
    *outer, last = t.stride()
    if last != 1:
        return False
    for x in outer:
        if x & 7 or not x:
            return not any([n > 1 and (x & 7 or not x) for n, x in zip(t.shape, outer)])
    return True


def _int32(name, t, *shape):
    """An int32 tensor with as many dimensions as `shape` and its first size (None: any), dense."""
    got = t.shape
    assert t.dtype == torch.int32, f"{name} must be int32, got {t.dtype}"
    assert len(got) == len(shape) and shape[0] in (None, got[0]), \
        f"{name} has shape {tuple(got)}, not {shape}"
    return t if t.is_contiguous() else t.contiguous()


def prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor | None = None, *,
            causal: bool = True, softmax_scale: float | None = None, check: bool = False):
    """-> (o ``[Tq, Hq, D]``, lse fp32 ``[Tq, Hq]``).

    q ``[Tq, Hq, D]``, k / v ``[Tk, Hkv, D]`` bf16 or f16 (slices of a fused projection are read in
    place); ``cu_q`` / ``cu_k`` int32 ``[B + 1]`` on the device, from 0 ascending: sequence b is
    rows ``cu_q[b] .. cu_q[b+1]`` of q and ``cu_k[b] .. cu_k[b+1]`` of k / v (``cu_k`` None: the
    same as q's).  Rows of q from ``cu_q[B]`` on (a batch padded to a fixed size) belong to no
    sequence: output 0, lse -inf.  softmax_scale defaults to ``D ** -0.5``."""
    if cu_k is None:
        _check_types("prefill", q, k, v, cu_q)
    else:
        _check_types("prefill", q, k, v, cu_q, cu_k)
    qs, ks = q.shape, k.shape
    assert len(ks) == 3 and ks == v.shape and ks[2] == qs[-1], \
        f"k and v must be [tokens, heads, {qs[-1]}], got {tuple(ks)} and {tuple(v.shape)}"
    _check_heads(qs, ks[1])
    cu_q = _int32("cu_q", cu_q, None)
    n = cu_q.shape[0]
    assert n >= 2, "cu_q needs at least one sequence"
    if cu_k is None:
        assert ks[0] == qs[0], f"without cu_k, k must have q's {qs[0]} tokens, got {ks[0]}"
        cu_k = cu_q
    else:
        cu_k = _int32("cu_k", cu_k, n)
    return ops.gqa_prefill(q if _aligned(q) else q.contiguous(), k if _aligned(k) else k.contiguous(),
                           v if _aligned(v) else v.contiguous(), cu_q, cu_k, causal,
                           qs[2] ** -0.5 if softmax_scale is None else float(softmax_scale), check)


def decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
           seq_lens: torch.Tensor, *, softmax_scale: float | None = None, check: bool = False):
    """-> (o ``[B, Hq, D]``, lse fp32 ``[B, Hq]``).

    q ``[B, Hq, D]``; k_pages / v_pages ``[P, Hkv, page, D]`` of q's type, any strides over a dense
    last dimension (a ``[P, page, Hkv, D]`` pool as ``pool.transpose(1, 2)``); page_table int32
    ``[B, W]``; seq_lens int32 ``[B]`` (the new token's key included; 0 = empty slot).  Lengths past
    ``W * page`` are cut there.  What the pages hold past a sequence's length is not used.  A page id
    outside the pool within a length (-1: a sequence without all its pages) is raised by
    ``mzoo_b200.check_errors()``, or at once with ``check=True``."""
    _check_types("decode", q, k_pages, v_pages, page_table, seq_lens)
    qs, ks = q.shape, k_pages.shape
    assert len(ks) == 4 and ks == v_pages.shape and ks[3] == qs[-1] and ks[0], \
        f"the pools must be [pages, heads, page, {qs[-1]}], got {tuple(ks)} and {tuple(v_pages.shape)}"
    assert ks[2] in PAGE_SIZES, f"page size must be one of {PAGE_SIZES}, got {ks[2]}"
    _check_heads(qs, ks[1])
    assert _aligned(k_pages) and _aligned(v_pages), \
        "the pools need dense, 16-byte aligned rows (they are not copied)"
    return ops.gqa_decode(q if _aligned(q) else q.contiguous(), k_pages, v_pages,
                          _int32("page_table", page_table, qs[0], None), _int32("seq_lens", seq_lens, qs[0]),
                          qs[2] ** -0.5 if softmax_scale is None else float(softmax_scale), check)
