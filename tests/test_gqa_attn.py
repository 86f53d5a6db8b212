"""Dense grouped-head attention (``mzoo_b200.gqa_attn``) against the definition in 64 bits.

Tolerances, from the arithmetic: with u the unit roundoff of the output type (2^-8 bf16,
2^-11 f16) the kernels may round each softmax weight and the output once, so an element is
off by at most u (sum_j p_j |v_j| + |o|); fp32 scores, exponentials and sums add a relative
2^-14 of sum_j p_j |v_j|, and f16 weights below 2^-14 an absolute 2^-25 each.  The fp32
log-sum-exp is within 2e-5 + 2e-6 |lse|."""

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mzoo_b200 import gqa_attn, ops

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _attend(q, k, v, seen, scale):
    """One head in doubles -> (o, lse, sum p |v|, sum |v|) over the keys `seen` [nq, nk]; keys that no
    row sees do not enter, whatever they hold."""
    o = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
    lse = torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    mag, tiny = torch.zeros_like(o), torch.zeros_like(o)
    for i in range(q.shape[0]):
        j = torch.nonzero(seen[i])[:, 0]
        if len(j):
            x = k[j] @ q[i] * scale
            lse[i] = torch.logsumexp(x, 0)
            p = torch.exp(x - lse[i])
            o[i], mag[i], tiny[i] = p @ v[j], p @ v[j].abs(), v[j].abs().sum(0)
    return o, lse, mag, tiny


def _compare(o, lse, ro, rl, mag, tiny, dt):
    o, lse = o.double().cpu(), lse.double().cpu()
    assert torch.equal(torch.isnan(o), torch.isnan(ro)) and torch.equal(torch.isinf(lse), torch.isinf(rl))
    bound = U[dt] * (mag + ro.abs()) * 1.01 + 2.0 ** -14 * mag + (2.0 ** -25 * tiny if dt == torch.float16 else 0) + 1e-30
    fine = torch.isfinite(ro)
    assert torch.equal(o[~fine & ~torch.isnan(ro)], ro[~fine & ~torch.isnan(ro)])
    worst = ((o - ro).abs() / bound)[fine]
    assert not worst.numel() or float(worst.max()) <= 1.0, f"o is off by {float(worst.max()):.2f} of its bound"
    empty = torch.isinf(rl)
    assert torch.equal(lse[empty], rl[empty]) and not o[empty].any()
    some = torch.isfinite(rl)
    assert ((lse - rl).abs()[some] <= 2e-5 + 2e-6 * rl.abs()[some]).all()


def _cu(lens):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32)


def _prefill_ref(q, k, v, new, keys, causal, scale):
    q, k, v = (t.double().cpu() for t in (q, k, v))
    out = [torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64), torch.zeros_like(q), torch.zeros_like(q)]
    a = b = 0
    for n, m in zip(new, keys):
        i, j = torch.arange(n)[:, None], torch.arange(m)[None, :]
        seen = (j <= i + m - n) if causal else (j < m).expand(n, m)
        for h in range(q.shape[1]):
            kh = h // (q.shape[1] // k.shape[1])
            got = _attend(q[a:a + n, h], k[b:b + m, kh], v[b:b + m, kh], seen, scale)
            for t, g in zip(out, got):
                t[a:a + n, h] = g
        a, b = a + n, b + m
    return out


def _randn(g, dt, *shape):
    return torch.randn(*shape, generator=g).to(dt)


def _prefill(dev, dt, hq, hkv, d, new, keys, causal=True, scale=None, seed=0, edit=None, fused=False):
    g = torch.Generator().manual_seed(seed)
    if fused:
        q, k, v = _randn(g, dt, sum(new), hq + 2 * hkv, d).split([hq, hkv, hkv], 1)
    else:
        q, k, v = _randn(g, dt, sum(new), hq, d), _randn(g, dt, sum(keys), hkv, d), _randn(g, dt, sum(keys), hkv, d)
    if edit:
        edit(q, k, v)
    if fused:
        base = torch.cat([q, k, v], 1).to(dev)
        qd, kd, vd = base.split([hq, hkv, hkv], 1)
    else:
        qd, kd, vd = q.to(dev), k.to(dev), v.to(dev)
    cu_k = None if new == keys else _cu(keys).to(dev)
    o, lse = gqa_attn.prefill(qd, kd, vd, _cu(new).to(dev), cu_k, causal=causal, softmax_scale=scale, check=True)
    assert o.shape == q.shape and o.dtype == dt and lse.shape == q.shape[:2] and lse.dtype == torch.float32
    _compare(o, lse, *_prefill_ref(q, k, v, new, keys, causal, d ** -0.5 if scale is None else scale), dt)
    return qd, kd, vd, o, lse


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (8, 2), (6, 1), (10, 2), (16, 1)])
def test_prefill_packed(cuda, dt, d, hq, hkv):
    new = [1, 130, 17, 64, 0, 257, 2]
    _prefill(cuda, dt, hq, hkv, d, new, new)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(64, 1), (128, 1), (96, 2), (127, 1), (7, 7)])
def test_prefill_wide_groups(cuda, hq, hkv):
    _prefill(cuda, torch.bfloat16, hq, hkv, 64, [5, 40, 1], [5, 40, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 15, 16, 31, 32, 33, 63, 65, 127, 128, 129, 255, 256, 300, 513])
def test_prefill_lengths(cuda, n):
    _prefill(cuda, torch.bfloat16, 4, 1, 128, [n], [n], seed=n)
    _prefill(cuda, torch.bfloat16, 2, 2, 64, [n], [n], seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("new,keys", [([3, 70], [200, 131]), ([128], [384]), ([1, 1, 1], [1, 129, 300]),
                                      ([40, 5], [3, 0]), ([5], [0]), ([300], [20]), ([0, 9, 0], [50, 9, 0]), ([200], [129])])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_other_key_lengths(cuda, new, keys, causal):
    """Chunks over earlier keys, and fewer keys than tokens: rows that see no key."""
    _prefill(cuda, torch.bfloat16, 6, 2, 64, new, keys, causal=causal)
    _prefill(cuda, torch.float16, 4, 4, 128, new, keys, causal=causal)


@pytest.mark.gpu
def test_prefill_long_rows(cuda):
    """Many key tiles; a few rows of a long prompt."""
    _prefill(cuda, torch.bfloat16, 2, 1, 128, [3], [5000])
    _prefill(cuda, torch.float16, 2, 1, 64, [200], [2300])


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [32, 33, 64, 301])
def test_prefill_many_sequences(cuda, seqs):
    g = torch.Generator().manual_seed(seqs)
    new = torch.randint(0, 40, (seqs,), generator=g).tolist()
    keys = [n + int(p) for n, p in zip(new, torch.randint(0, 30, (seqs,), generator=g))]
    _prefill(cuda, torch.bfloat16, 4, 2, 64, new, new)
    _prefill(cuda, torch.float16, 3, 1, 64, new, keys)


@pytest.mark.gpu
def test_prefill_no_tokens_and_wild_offsets(cuda):
    """No tokens; offsets that leave the tensors touch nothing outside them."""
    none = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=cuda)
    o, lse = gqa_attn.prefill(none, none, none, torch.zeros(2, dtype=torch.int32, device=cuda), check=True)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    big = torch.randn(3000, 4, 64, device=cuda).to(torch.bfloat16)
    q = big[1000:1100]
    wild = torch.tensor([-50, 60, 2 ** 30, 40, 5000], dtype=torch.int32, device=cuda)
    gqa_attn.prefill(q, big[:200], big[:200], wild, wild, check=True)
    want = gqa_attn.prefill(q[:60], big[:60], big[:60], _cu([60]).to(cuda))[0]
    wild = torch.tensor([-9, 60, 100], dtype=torch.int32, device=cuda)
    got = gqa_attn.prefill(q, big[:200], big[:200], wild, wild, check=True)[0]
    assert torch.equal(got[:60], want)


@pytest.mark.gpu
def test_prefill_offsets_past_32_bits(cuda):
    """Outputs behind 2^31 elements; thousands of sequences."""
    T, hq, n = 270000, 64, 100
    q = torch.empty(T, hq, 128, dtype=torch.bfloat16, device=cuda)
    q.copy_(torch.randn(hq, 128, device=cuda, generator=torch.Generator(device=cuda).manual_seed(0)))
    q[-n:] = torch.randn(n, hq, 128, device=cuda).to(torch.bfloat16)
    k, v = (torch.randn(T, 1, 128, device=cuda).to(torch.bfloat16) for _ in range(2))
    cu = torch.arange(0, T + 1, n, dtype=torch.int32, device=cuda)
    o, lse = gqa_attn.prefill(q, k, v, cu, check=True)
    want = gqa_attn.prefill(q[-n:].clone(), k[-n:], v[-n:], _cu([n]).to(cuda), check=True)
    assert o.numel() > 2 ** 31 and torch.equal(o[-n:], want[0]) and torch.equal(lse[-n:], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 64), (12, 2, 96), (8, 8, 128), (40, 1, 128)])
@pytest.mark.parametrize("new,keys", [([1], [1537]), ([2, 5, 1], [1600, 3, 4000]), ([9], [8 * 128]), ([33, 0, 7], [1800, 2000, 0]),
                                      ([3000], [900]), ([20], [12 * 128 + 7])])
def test_prefill_few_rows_many_keys(cuda, hq, hkv, d, new, keys):
    """Key ranges cut into parts and joined, rows without keys among them."""
    if sum(new) * hq > 4000:
        hq = hkv
    _prefill(cuda, torch.bfloat16, hq, hkv, d, new, keys)
    _prefill(cuda, torch.float16, hq, hkv, d, new, keys, causal=False, scale=-0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 64), (12, 2, 96), (16, 1, 128)])
def test_prefill_many_parts(cuda, hq, hkv, d):
    """As many parts that several warps share a row of them; sequences of one part and of none beside."""
    _prefill(cuda, torch.bfloat16, hq, hkv, d, [3, 17, 5, 0], [9000, 70, 2, 700])

    def edit(q, k, v):
        v[8998, :, 3] = math.nan   # seen by the last two of the three
        v[40, :, 5] = -math.inf
    _prefill(cuda, torch.float16, hq, hkv, d, [3], [9000], edit=edit)


@pytest.mark.gpu
def test_prefill_parts_keep_nan_apart(cuda):
    """In a cut key range, values that a row does not see stay out of it and those it sees arrive."""
    def edit(q, k, v):
        v[2990, :, 3] = math.inf   # token 2 of 12 new ones and later see it
        v[2995] = math.nan
        v[100, :, 7] = -math.inf   # in the first part, seen by all
    _prefill(cuda, torch.bfloat16, 4, 2, 128, [12], [3000], edit=edit)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 0.5, -0.3])
def test_prefill_scale_and_fused_projection(cuda, scale):
    _prefill(cuda, torch.bfloat16, 6, 2, 128, [50, 131], [50, 131], scale=scale, fused=True)


@pytest.mark.gpu
def test_prefill_growing_scores(cuda):
    """Each tile's scores are far above the tiles before it (and far below, reversed): the running
    maximum has to be followed."""
    def up(q, k, v):
        k *= torch.linspace(0.1, 12.0, k.shape[0])[:, None, None].to(k.dtype)
        q.copy_(q.abs())
        k.copy_(k.abs())

    def down(q, k, v):
        up(q, k, v)
        k.copy_(k.flip(0))
    for edit in (up, down):
        _prefill(cuda, torch.bfloat16, 2, 1, 128, [300], [600], edit=edit)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_neighbours_and_future_stay_apart(cuda, bad, d):
    """A NaN or infinity in one sequence's keys or values, or in a token that a row does not see, does
    not reach that row; the rows that see an infinite value get it."""
    new = [70, 33, 140]

    def in_v(q, k, v):
        v[70:103] = bad   # the whole middle sequence
        v[103 + 100, :, 5] = bad  # one channel of one token of the last one
    _prefill(cuda, torch.bfloat16, 4, 2, d, new, new, edit=in_v)

    def in_k(q, k, v):
        k[70:103] = bad
    g = torch.Generator().manual_seed(0)
    q, k, v = (_randn(g, torch.bfloat16, sum(new), h, d) for h in (4, 2, 2))
    clean = gqa_attn.prefill(q.to(cuda), k.to(cuda), v.to(cuda), _cu(new).to(cuda))
    in_k(q, k, v)
    k[242] = bad  # the last token of the last sequence
    got = gqa_attn.prefill(q.to(cuda), k.to(cuda), v.to(cuda), _cu(new).to(cuda), check=True)
    for a, b in zip(clean, got):
        assert torch.equal(a[:70], b[:70]) and torch.equal(a[103:242], b[103:242])


@pytest.mark.gpu
def test_prefill_same_bits_twice_on_another_stream(cuda):
    g = torch.Generator().manual_seed(3)
    q, k, v = (_randn(g, torch.bfloat16, 700, h, 128).to(cuda) for h in (8, 2, 2))
    cu = _cu([300, 1, 399]).to(cuda)
    first = gqa_attn.prefill(q, k, v, cu)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        again = gqa_attn.prefill(q, k, v, cu)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
def test_prefill_strides(cuda):
    """Rows apart by odd strides, a sliced head range, broadcast K / V and a misaligned start are the
    same as their dense copies."""
    g = torch.Generator().manual_seed(5)
    base = _randn(g, torch.bfloat16, 90, 9, 200).to(cuda)
    q, k, v = base[:, :4, 8:72], base[:, 4:6, 64:128], base[:, 6:8, 128:192]
    cu = _cu([41, 49]).to(cuda)
    want = gqa_attn.prefill(q.contiguous(), k.contiguous(), v.contiguous(), cu, check=True)
    for x, y, z in ((q, k, v), (base[:, :4, 8:72], k.transpose(0, 1).contiguous().transpose(0, 1), v)):
        got = gqa_attn.prefill(x, y, z, cu, check=True)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    odd = base[:, :4, 3:67]  # 2-byte aligned only: copied
    got = gqa_attn.prefill(odd, k, v, cu, check=True)
    assert all(torch.equal(a, b) for a, b in zip(gqa_attn.prefill(odd.contiguous(), k, v, cu), got))
    one = k[:, :1]
    got = gqa_attn.prefill(q, one.expand(-1, 2, -1), one.expand(-1, 2, -1), cu, check=True)
    assert all(torch.equal(a, b) for a, b in zip(gqa_attn.prefill(q, one, one, cu), got))


# ------------------------------------------------------------------ decode

def _pages(g, dt, hkv, d, page, lens, fill=None, width=None, extra=3):
    need = [-(-n // page) for n in lens]
    P, W = sum(need) + extra, width or max(1, max(need))
    kp, vp = _randn(g, dt, P, hkv, page, d), _randn(g, dt, P, hkv, page, d)
    order = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((len(lens), W), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    if fill is not None:  # everything that no sequence covers
        live = torch.zeros(P, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for t in range(n):
                live[table[b, t // page], t % page] = True
        kp[(~live)[:, None].expand(-1, hkv, -1)] = fill
        vp[(~live)[:, None].expand(-1, hkv, -1)] = fill
    return kp, vp, table


def _decode(dev, dt, hq, hkv, d, page, lens, scale=None, seed=0, fill=math.nan, cut=None):
    g = torch.Generator().manual_seed(seed)
    q = _randn(g, dt, len(lens), hq, d)
    kp, vp, table = _pages(g, dt, hkv, d, page, lens, fill)
    o, lse = gqa_attn.decode(q.to(dev), kp.to(dev), vp.to(dev), table.to(dev),
                             torch.tensor(cut or lens, dtype=torch.int32, device=dev), softmax_scale=scale, check=True)
    assert o.shape == q.shape and o.dtype == dt and lse.shape == q.shape[:2]
    ref = [torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)]
    ref += [torch.zeros_like(ref[0]), torch.zeros_like(ref[0])]
    grp = hq // hkv
    for b, n in enumerate(lens):
        ids = table[b, :-(-n // page)].long()
        k, v = (t[ids].transpose(0, 1).flatten(1, 2)[:, :n].double() for t in (kp, vp))
        for h in range(hq):
            got = _attend(q[b, h:h + 1].double(), k[h // grp], v[h // grp], torch.ones(1, n, dtype=torch.bool),
                          d ** -0.5 if scale is None else scale)
            for t, x in zip(ref, got):
                t[b, h] = x[0]
    _compare(o, lse, *ref, dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_decode_lengths(cuda, dt, d, page):
    """Lengths 0, 1 and around page and tile ends, NaN in every slot past them."""
    _decode(cuda, dt, 8, 2, d, page, [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (8, 8), (14, 2), (16, 1), (17, 1), (32, 1), (40, 1), (64, 1), (128, 1),
                                    (96, 2)])
def test_decode_heads(cuda, hq, hkv):
    _decode(cuda, torch.bfloat16, hq, hkv, 128, 64, [130, 5, 700, 0, 64])


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[9000], [1], [20000, 3, 5000], [700] * 40, [1] * 300, [0, 0, 0], [33] * 150 + [6000]])
def test_decode_splits(cuda, lens):
    """Few long, many short and mixed sequences: how the work is cut does not show."""
    _decode(cuda, torch.bfloat16, 4, 2, 64, 32, lens, fill=None if sum(lens) > 9000 else math.inf)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(12, 4, 64), (36, 4, 128), (16, 8, 96), (22, 2, 96)])
@pytest.mark.parametrize("lens", [[0, 256, 1, 0, 130] * 17, [0] * 50 + [200, 255, 3] + [0] * 40, [128] * 37, [0, 300, 1, 129] * 24])
def test_decode_short_tables(cuda, hq, hkv, d, lens):
    """More (sequence, head)s than blocks, none of their rows cut, runs that begin in empty sequences;
    tables just above, with cut rows; one and two head tiles, full and not."""
    _decode(cuda, torch.bfloat16, hq, hkv, d, 16, lens, fill=None)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (11, 1, 64), (40, 2, 96)])
def test_decode_query_rows_at_any_even_offset(cuda, hq, hkv, d):
    """Query rows that are only 4-byte aligned, as the library takes them."""
    from mzoo_b200 import ops
    g = torch.Generator().manual_seed(3)
    lens = [200, 0, 33, 900]
    kp, vp, table = _pages(g, torch.bfloat16, hkv, d, 32, lens)
    rest = [t.to(cuda) for t in (kp, vp, table, torch.tensor(lens, dtype=torch.int32))]
    wide = _randn(g, torch.bfloat16, 4 * (hq * (d + 2) + 6) + 2).to(cuda)
    q = wide[2:].as_strided((4, hq, d), (hq * (d + 2) + 6, d + 2, 1), 2)
    want = gqa_attn.decode(q.contiguous(), *rest, check=True)
    got = ops.gqa_decode(q, *rest, d ** -0.5, True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_decode_scale_and_wide_scores(cuda):
    _decode(cuda, torch.bfloat16, 4, 1, 128, 16, [500, 77], scale=2.0)
    _decode(cuda, torch.float16, 4, 1, 128, 16, [500, 77], scale=0.0)


@pytest.mark.gpu
def test_decode_length_past_the_table_is_cut(cuda):
    _decode(cuda, torch.bfloat16, 4, 2, 64, 16, [64, 64], cut=[1000, 64])


@pytest.mark.gpu
def test_decode_token_major_pool_and_wild_ids(cuda):
    """A [P, page, heads, D] pool through transposed views, K and V in one tensor, and table entries
    past the lengths that name no page."""
    g = torch.Generator().manual_seed(1)
    q = _randn(g, torch.bfloat16, 3, 8, 128).to(cuda)
    kp, vp, table = _pages(g, torch.bfloat16, 2, 128, 32, [40, 0, 100], width=9)
    lens = torch.tensor([40, 0, 100], dtype=torch.int32, device=cuda)
    want = gqa_attn.decode(q, kp.to(cuda), vp.to(cuda), table.to(cuda), lens, check=True)
    both = torch.stack([kp, vp], 1).transpose(2, 3).contiguous().to(cuda)  # [P, 2, page, heads, D]
    wild = torch.where(table < 0, torch.tensor([2 ** 31 - 1, -2 ** 31, -7] * 3, dtype=torch.int32), table)
    got = gqa_attn.decode(q, both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), wild.to(cuda), lens, check=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_decode_offsets_past_32_bits_and_empty_batches(cuda):
    g = torch.Generator().manual_seed(9)
    P, hkv, page, d = 18000, 8, 128, 128
    kp, vp = (torch.empty(P, hkv, page, d, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    assert kp.numel() > 2 ** 31
    few = [_randn(g, torch.bfloat16, 3, hkv, page, d).to(cuda) for _ in range(2)]
    for pool, x in zip((kp, vp), few):
        pool[P - 3:] = x
    q, lens = _randn(g, torch.bfloat16, 1, 16, d).to(cuda), torch.tensor([300], dtype=torch.int32, device=cuda)
    table = torch.tensor([[P - 1, P - 3, P - 2]], dtype=torch.int32, device=cuda)
    got = gqa_attn.decode(q, kp, vp, table, lens, check=True)
    want = gqa_attn.decode(q, *few, table - (P - 3), lens, check=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    o, lse = gqa_attn.decode(q[:0], *few, table[:0], lens[:0], check=True)
    assert o.shape == (0, 16, d) and lse.shape == (0, 16)
    o, lse = gqa_attn.decode(q, *few, table[:, :0], lens, check=True)
    assert not o.any() and bool((lse == -math.inf).all())


@pytest.mark.gpu
def test_decode_step_in_a_graph(cuda):
    """A captured step (cache write and attention) follows the lengths and tables of its replay."""
    from mzoo_b200 import kv_pages
    g = torch.Generator().manual_seed(4)
    B, hq, hkv, d, page, W = 5, 8, 2, 64, 16, 40
    q, k, v = (_randn(g, torch.bfloat16, B, h, d).to(cuda) for h in (hq, hkv, hkv))
    kp, vp = (_randn(g, torch.bfloat16, B * W, hkv, page, d).to(cuda) for _ in range(2))
    table = torch.randperm(B * W, generator=g).view(B, W).to(torch.int32).to(cuda)
    lens = torch.tensor([1, 17, 600, 0, 40], dtype=torch.int32, device=cuda)

    def step():
        kv_pages.append(k, v, kp, vp, table, lens)
        return gqa_attn.decode(q, kp, vp, table, lens + 1)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(cuda).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in ([3, 90, 620, 5, 0], [0, 0, 639, 16, 15]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        table.copy_(table.flip(0))
        q.copy_(q.flip(0))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
def test_decode_equals_prefill_of_one_token(cuda):
    """The last row of a prompt, by both operators."""
    g = torch.Generator().manual_seed(2)
    n, page = 333, 64
    q, k, v = (_randn(g, torch.float16, n, h, 128).to(cuda) for h in (8, 2, 2))
    o, lse = gqa_attn.prefill(q, k, v, _cu([n]).to(cuda))
    P = -(-n // page)
    pools = [torch.zeros(P * page, 2, 128, dtype=torch.float16, device=cuda) for _ in range(2)]
    for pool, x in zip(pools, (k, v)):
        pool[:n] = x
    kp, vp = (p.view(P, page, 2, 128).transpose(1, 2) for p in pools)
    od, ld = gqa_attn.decode(q[-1:], kp, vp, torch.arange(P, dtype=torch.int32, device=cuda)[None],
                             torch.tensor([n], dtype=torch.int32, device=cuda), check=True)
    # both are within u (mag + |o|) of the value; mag <= max |v|
    assert (od[0].float() - o[-1].float()).abs().max() <= 2 * 2.0 ** -11 * 2 * v.float().abs().max()
    assert (ld[0] - lse[-1]).abs().max() <= 4e-5


# ------------------------------------------------------------------ refusals, tracing

def test_cpu_tensors_are_refused():
    q, k = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="CUDA tensors only"):
        gqa_attn.prefill(q, k, k, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(AssertionError, match="CUDA tensors only"):
        gqa_attn.decode(q, k[None], k[None], torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))


def _t(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="cuda:0")


def _i(*shape):
    return _t(*shape, dtype=torch.int32)


def test_prefill_refusals_and_shapes():
    with FakeTensorMode():
        o, lse = gqa_attn.prefill(_t(9, 6, 96), _t(20, 2, 96), _t(20, 2, 96), _i(3), _i(3))
        assert o.shape == (9, 6, 96) and o.dtype == torch.bfloat16 and lse.shape == (9, 6)
        grad = _t(4, 2, 64).requires_grad_()
        for args, word in (((_t(4, 2, 80), _t(4, 2, 80), _t(4, 2, 80), _i(2)), "D in"),
                           ((_t(4, 2, 64), _t(4, 2, 64, dtype=torch.float16), _t(4, 2, 64), _i(2)), "one type"),
                           ((_t(4, 2, 64, dtype=torch.float32),) * 3 + (_i(2),), "bf16 / f16"),
                           ((_t(4, 3, 64), _t(4, 2, 64), _t(4, 2, 64), _i(2)), "multiple"),
                           ((_t(4, 129, 64), _t(4, 1, 64), _t(4, 1, 64), _i(2)), "multiple"),
                           ((_t(4, 2, 64), _t(5, 2, 64), _t(5, 2, 64), _i(2)), "without cu_k"),
                           ((_t(4, 2, 64), _t(5, 2, 64), _t(4, 2, 64), _i(2), _i(2)), "k and v"),
                           ((_t(4, 2, 64), _t(5, 2, 64), _t(5, 2, 64), _i(2), _i(3)), "cu_k"),
                           ((_t(4, 2, 64),) * 3 + (_t(2, dtype=torch.int64),), "int32"),
                           ((_t(4, 2, 64),) * 3 + (_i(1),), "at least one sequence"),
                           ((grad, _t(4, 2, 64), _t(4, 2, 64), _i(2)), "no backward")):
            with pytest.raises(AssertionError, match=word):
                gqa_attn.prefill(*args)
        with torch.no_grad():
            assert gqa_attn.prefill(grad, _t(4, 2, 64), _t(4, 2, 64), _i(2))[0].shape == (4, 2, 64)


def test_decode_refusals_and_shapes():
    with FakeTensorMode():
        pool = _t(7, 2, 64, 128)
        assert gqa_attn.decode(_t(3, 8, 128), pool, pool, _i(3, 5), _i(3))[1].shape == (3, 8)
        for args, word in (((_t(3, 8, 128), _t(7, 2, 48, 128), _t(7, 2, 48, 128), _i(3, 5), _i(3)), "page size"),
                           ((_t(3, 8, 64), pool, pool, _i(3, 5), _i(3)), "pools"),
                           ((_t(3, 7, 128), pool, pool, _i(3, 5), _i(3)), "multiple"),
                           ((_t(3, 8, 128), pool, pool, _i(2, 5), _i(3)), "page_table"),
                           ((_t(3, 8, 128), pool, pool, _i(3, 5), _i(4)), "seq_lens"),
                           ((_t(3, 8, 128), pool, pool, _t(3, 5, dtype=torch.int64), _i(3)), "int32"),
                           ((_t(3, 8, 128), _t(7, 2, 128, 64).transpose(2, 3), pool, _i(3, 5), _i(3)), "dense")):
            with pytest.raises(AssertionError, match=word):
                gqa_attn.decode(*args)


def test_default_path_does_not_sync(monkeypatch):
    def boom(*a, **k):
        raise AssertionError("host synchronisation on the default path")
    with FakeTensorMode():
        for name in ("item", "tolist", "__int__", "__float__", "__index__"):
            monkeypatch.setattr(torch.Tensor, name, boom)
        monkeypatch.setattr(torch.cuda, "synchronize", boom)
        pool = _t(7, 2, 64, 128)
        gqa_attn.decode(_t(3, 8, 128), pool, pool, _i(3, 5), _i(3))
        gqa_attn.prefill(_t(4, 2, 64), _t(4, 2, 64), _t(4, 2, 64), _i(2))


def test_c_entry_refusals():
    """Sizes the kernels are not built for are refused before any launch."""
    from mzoo_b200 import _lib
    lib = _lib.lib()
    pre = lambda D=64, hq=4, hkv=2, dt=1, B=1: lib.mzb_gqa_prefill(  # noqa: E731
        0, 0, 0, 0, 0, 0, 0, 0, 8, 8, B, hq, hkv, D, dt, 256, 64, 128, 64, 128, 64, 1, 1.0, None, None)
    assert pre(D=80) == _lib.MZB_ERR_UNSUPPORTED and b"head dim" in lib.mzb_last_error()
    assert pre(hq=5) == _lib.MZB_ERR_SHAPE and pre(dt=0) == _lib.MZB_ERR_UNSUPPORTED and pre(B=0) == _lib.MZB_ERR_SHAPE
    assert pre() == _lib.MZB_ERR_SHAPE and b"error word" in lib.mzb_last_error()
    dec = lambda page=64, W=4, P=9: lib.mzb_gqa_decode(  # noqa: E731
        0, 0, 0, 0, 0, 0, 0, 0, 1, 4, 2, 64, 1, page, P, W, 256, 64, 8192, 4096, 64, 8192, 4096, 64, 1.0, None, None)
    assert dec(page=48) == _lib.MZB_ERR_UNSUPPORTED and dec(P=0) == _lib.MZB_ERR_SHAPE
    assert dec(W=1 << 30) == _lib.MZB_ERR_SHAPE and dec() == _lib.MZB_ERR_SHAPE


def test_ops_are_registered():
    """Schemas and fake implementations at import, the C++ kernels once the libraries are built."""
    from mzoo_b200 import _lib, build
    names = {"gqa_prefill", "gqa_decode", "kv_append", "kv_reserve", "kv_fork", "kv_free", "kv_compact", "kv_copy_pages"}
    assert names <= set(dir(torch.ops.mzb))
    build.build()
    _lib.load_torch_ops()
    assert all(torch._C._dispatch_has_kernel_for_dispatch_key(f"mzb::{n}", "CUDA") for n in names)


def test_errors_keep_their_kinds():
    """A status of the C ABI that comes through the C++ ops is the exception the other ops raise."""
    from mzoo_b200 import _lib
    for status, kind in ((_lib.MZB_ERR_SHAPE, AssertionError), (_lib.MZB_ERR_ALIGN, AssertionError),
                         (_lib.MZB_ERR_UNSUPPORTED, AssertionError), (_lib.MZB_ERR_LAUNCH, _lib.MzbError)):
        with pytest.raises(kind, match="gqa: why"):
            ops._failed(RuntimeError(f"gqa: why [mzb status {status}]"))
    with pytest.raises(RuntimeError, match="another"):
        ops._failed(RuntimeError("another"))


@pytest.mark.gpu
def test_library_refusals_are_assertions(cuda):
    """What only the library can see: a misaligned base address of foreign storage."""
    raw = torch.zeros(4 * 2 * 64 + 8, dtype=torch.bfloat16, device=cuda)
    odd = torch.empty(0, dtype=torch.bfloat16, device=cuda).set_(raw.untyped_storage()[2:], 0, (4, 2, 64))
    with pytest.raises(AssertionError, match="aligned"):
        gqa_attn.prefill(odd, odd, odd, _cu([4]).to(cuda))
