"""Dense causal attention with grouped K / V heads for serving: whole prompts packed one after
another (``prefill``) and one new token per sequence over a paged cache (``decode``).  No
counterpart in the reference's kernel packages: these are the full-attention layers that a
model mixes with the window and sparse ones.

``prefill`` row i of a sequence with nq new tokens and nk keys sees the keys
``j <= i + nk - nq`` (the last token sees all of them, so a prompt can be run in chunks over
keys that grow); head h reads K / V head ``h // (Hq // Hkv)``.  Both return the output in q's
type and the natural-log-sum-exp in fp32; a row that sees no key has output 0 and lse -inf.
fp32 softmax statistics and accumulation; forward only.  The cache's pages are written,
shared and moved by ``mzoo_b200.kv_pages``; the kernels are ``csrc/gqa_prefill.cu`` and
``csrc/gqa_decode.cu``.
"""

import torch

from . import ops
from ._lib import require_cuda

HEAD_DIMS = (64, 96, 128)
PAGE_SIZES = (16, 32, 64, 128)
_TYPES = (torch.bfloat16, torch.float16)


def _check_qkv(what, q, k, v, *rest):
    require_cuda(q, k, v, *rest)
    assert q.dtype in _TYPES, f"{what} supports bf16 / f16, got {q.dtype}"
    assert q.dtype == k.dtype == v.dtype, f"q, k and v must have one type, got {q.dtype}, {k.dtype}, {v.dtype}"
    for t in (k, v, *rest):
        assert t.device == q.device, f"all tensors must be on {q.device}, got one on {t.device}"
    assert q.dim() == 3 and q.shape[2] in HEAD_DIMS, f"q must be [tokens, heads, D in {HEAD_DIMS}], got {tuple(q.shape)}"
    assert not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)), \
        f"{what} has no backward: call it under torch.no_grad()"


def _heads(q, hkv):
    hq = q.shape[1]
    assert hq >= 1 and hkv >= 1 and hq % hkv == 0 and hq // hkv <= 128, \
        f"query heads must be a multiple (at most 128) of the K / V heads, got {hq} and {hkv}"


def _aligned(t: torch.Tensor) -> bool:
    """Whether the kernels can address t in place: dense rows, 16-byte aligned (the base address of
    foreign storage is checked by the library), no broadcast dimension."""
    return t.stride(-1) == 1 and t.storage_offset() % 8 == 0 and all(
        n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1]))


def _int32(name, t, *shape):
    assert t.dtype == torch.int32, f"{name} must be int32, got {t.dtype}"
    assert t.dim() == len(shape) and all(s is None or s == n for s, n in zip(shape, t.shape)), \
        f"{name} has shape {tuple(t.shape)}, not {shape}"
    return t.contiguous()


def prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor | None = None, *,
            causal: bool = True, softmax_scale: float | None = None, check: bool = False):
    """-> (o ``[Tq, Hq, D]``, lse fp32 ``[Tq, Hq]``).

    q ``[Tq, Hq, D]``, k / v ``[Tk, Hkv, D]`` bf16 or f16 (slices of a fused projection are read in
    place); ``cu_q`` / ``cu_k`` int32 ``[B + 1]`` on the device, from 0 ascending: sequence b is
    rows ``cu_q[b] .. cu_q[b+1]`` of q and ``cu_k[b] .. cu_k[b+1]`` of k / v (``cu_k`` None: the
    same as q's).  softmax_scale defaults to ``D ** -0.5``."""
    _check_qkv("prefill", q, k, v, cu_q, *(() if cu_k is None else (cu_k,)))
    assert k.dim() == 3 and k.shape == v.shape and k.shape[2] == q.shape[2], \
        f"k and v must be [tokens, heads, {q.shape[2]}], got {tuple(k.shape)} and {tuple(v.shape)}"
    _heads(q, k.shape[1])
    cu_q = _int32("cu_q", cu_q, None)
    assert cu_q.shape[0] >= 2, "cu_q needs at least one sequence"
    if cu_k is None:
        assert k.shape[0] == q.shape[0], f"without cu_k, k must have q's {q.shape[0]} tokens, got {k.shape[0]}"
        cu_k = cu_q
    else:
        cu_k = _int32("cu_k", cu_k, cu_q.shape[0])
    q, k, v = (t if _aligned(t) else t.contiguous() for t in (q, k, v))
    return ops.gqa_prefill(q, k, v, cu_q, cu_k, causal, q.shape[2] ** -0.5 if softmax_scale is None else float(softmax_scale),
                           check)


def decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
           seq_lens: torch.Tensor, *, softmax_scale: float | None = None, check: bool = False):
    """-> (o ``[B, Hq, D]``, lse fp32 ``[B, Hq]``).

    q ``[B, Hq, D]``; k_pages / v_pages ``[P, Hkv, page, D]`` of q's type, any strides over a dense
    last dimension (a ``[P, page, Hkv, D]`` pool as ``pool.transpose(1, 2)``); page_table int32
    ``[B, W]``; seq_lens int32 ``[B]`` (the new token's key included; 0 = empty slot).  Lengths past
    ``W * page`` are cut there.  What the pages hold past a sequence's length is not used."""
    _check_qkv("decode", q, k_pages, v_pages, page_table, seq_lens)
    assert k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.shape[3] == q.shape[2] and k_pages.shape[0], \
        f"the pools must be [pages, heads, page, {q.shape[2]}], got {tuple(k_pages.shape)} and {tuple(v_pages.shape)}"
    assert k_pages.shape[2] in PAGE_SIZES, f"page size must be one of {PAGE_SIZES}, got {k_pages.shape[2]}"
    _heads(q, k_pages.shape[1])
    for t in (k_pages, v_pages):
        assert _aligned(t), "the pools need dense, 16-byte aligned rows (they are not copied)"
    page_table, seq_lens = _int32("page_table", page_table, q.shape[0], None), _int32("seq_lens", seq_lens, q.shape[0])
    return ops.gqa_decode(q if _aligned(q) else q.contiguous(), k_pages, v_pages, page_table, seq_lens,
                          q.shape[2] ** -0.5 if softmax_scale is None else float(softmax_scale), check)
