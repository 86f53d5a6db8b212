"""Edges of the dense serving operators: rows of no sequence, infinite scores, broken tables, error words,
tracing."""

import math

import pytest
import torch

import mzoo_b200
from mzoo_b200 import _lib, gqa_attn
from test_gqa_attn import _cu, _pages, _prefill, _randn


def _soil(dev, numbers):
    """Free blocks of the allocator that hold large numbers, of the sizes that a call takes next."""
    for n in numbers:
        del_me = torch.full((max(1, n),), 0x3fffffff, dtype=torch.int32, device=dev)
        del del_me


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,new,keys", [(16, 1, 128, [16], [4000]), (16, 1, 128, [3], [30000]), (4, 2, 64, [2, 0, 5], [1600, 9, 4000]),
                                               (8, 2, 96, [130, 1, 64], [130, 1, 64]), (2, 1, 64, [7] * 40, [9] * 40),
                                               (3, 1, 128, [5], [0]), (4, 4, 64, [0], [700])])
@pytest.mark.parametrize("pad", [1, 16, 300])
def test_prefill_padded_batch(cuda, hq, hkv, d, new, keys, pad):
    """Rows behind cu_q[B], with and without cut key ranges, as few and as many parts: 0 and -inf; the
    rows of sequences are those of the call without padding."""
    g = torch.Generator().manual_seed(pad)
    n = sum(new)
    q = _randn(g, torch.bfloat16, n + pad, hq, d).to(cuda)
    k, v = (_randn(g, torch.bfloat16, max(1, sum(keys)) + 3, hkv, d).to(cuda) for _ in range(2))
    cu_q, cu_k = _cu(new).to(cuda), _cu(keys).to(cuda)
    rows = (n + pad) * hq
    _soil(cuda, [rows * (s * (d + 1) + 1) for s in (1, 2, 4, 9, 16, 37, 74)])
    o, lse = gqa_attn.prefill(q, k, v, cu_q, cu_k, check=True)
    assert not o[n:].any() and bool((lse[n:] == -math.inf).all())
    if n:
        want = gqa_attn.prefill(q[:n], k, v, cu_q, cu_k, check=True)
        # the number of parts may differ: each row is within a rounding of the output's type
        assert (o[:n].float() - want[0].float()).abs().max() <= 2.0 ** -6 * v.float().abs().max()
        assert torch.equal(torch.isinf(lse[:n]), torch.isinf(want[1]))
        some = torch.isfinite(want[1])
        assert (lse[:n] - want[1])[some].abs().max() <= 1e-4 if some.any() else True


@pytest.mark.gpu
def test_prefill_padding_beside_the_definition(cuda):
    """A padded call against 64 bits: the keys of the padding's rows are nobody's."""
    dt = torch.float16
    g = torch.Generator().manual_seed(1)
    q, k, v = (_randn(g, dt, 40, h, 64).to(cuda) for h in (4, 2, 2))
    k[25:], v[25:] = math.nan, math.nan
    o, lse = gqa_attn.prefill(q, k, v, _cu([9, 16]).to(cuda), check=True)
    want = gqa_attn.prefill(q[:25], k[:25], v[:25], _cu([9, 16]).to(cuda), check=True)
    assert torch.equal(o[:25], want[0]) and torch.equal(lse[:25], want[1])
    assert not o[25:].any() and bool((lse[25:] == -math.inf).all())
    _prefill(cuda, dt, 4, 2, 64, [9, 16], [9, 16], seed=1)


@pytest.mark.parametrize("tokens,hq,hkv,pairs", [(16, 16, 1, 1), (64, 32, 8, 1), (128, 16, 2, 4), (32, 16, 1, 2), (17, 16, 1, 2), (1, 1, 1, 1)])
def test_one_sequence_is_cut_for_all_sms(tokens, hq, hkv, pairs):
    """The number of parts (from the workspace's size) is what 148 SMs can take of the sequence's items, also
    where its tokens fill them exactly."""
    from mzoo_b200 import _lib
    floats = _lib.lib().mzb_gqa_prefill_ws(tokens, 60000, 1, hq, hkv, 64)
    parts = floats // (tokens * hq * 65)
    assert parts == 148 // (pairs * hkv)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,width,at", [([40, 0, 100], None, (2, 3)), ([40, 0, 100], None, (0, 0)), ([200, 256], 8, (1, 7)),
                                           ([30000, 9], None, (0, 700)), ([30000, 9], None, (1, 0)), ([5000] * 70, None, (69, 156))])
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 2 ** 31 - 1, "P"])
def test_decode_reports_ids_outside_the_pool(cuda, lens, width, at, bad):
    """Within a sequence's length they are an error, in whichever block's run they lie; other sequences are
    right.  Behind the length they are nobody's."""
    g = torch.Generator().manual_seed(0)
    q = _randn(g, torch.bfloat16, len(lens), 4, 64).to(cuda)
    kp, vp, table = _pages(g, torch.bfloat16, 2, 64, 32, lens, width=width)
    rest = [t.to(cuda) for t in (kp, vp)]
    n = torch.tensor(lens, dtype=torch.int32, device=cuda)
    want = gqa_attn.decode(q, *rest, table.to(cuda), n, check=True)
    table[at] = kp.shape[0] if bad == "P" else bad
    with pytest.raises(_lib.MzbError, match="id out of range"):
        gqa_attn.decode(q, *rest, table.to(cuda), n, check=True)
    o, lse = gqa_attn.decode(q, *rest, table.to(cuda), n)
    with pytest.raises(_lib.MzbError, match="page"):
        mzoo_b200.check_errors()
    others = torch.arange(len(lens)) != at[0]
    assert torch.equal(o[others], want[0][others]) and torch.equal(lse[others], want[1][others])
    n[at[0]] = 32 * at[1]  # now it lies behind the length
    gqa_attn.decode(q, *rest, table.to(cuda), n, check=True)


def _sink(g, nq, n, at, bits):
    """q rows and n keys whose scores (scale 1) lie around 0 but for key `at`, `bits` bits above; its value is 0."""
    q, k = torch.zeros(nq, 1, 64), torch.zeros(n, 1, 64)
    q[:, :, 0], q[:, :, 1] = 1.0, torch.rand(nq, 1, generator=g) + 0.5
    k[:, :, 1] = torch.randn(n, 1, generator=g) * 0.5
    k[at, :, 0], k[at, :, 1] = bits * math.log(2.0), 0.0
    v = torch.rand(n, 1, 64, generator=g) + 0.5
    v[at] = 0.0
    return q.half(), k.half(), v.half()


def _near(o, lse, q, k, v, seen):
    """f16 results against 64 bits: each weight and the output are rounded to 11 bits once, weights below 2^-14 of
    2^8 times the largest to multiples of 2^-32 of it, and fp32 arithmetic adds 2^-14."""
    q, k, v = q[:, 0].double(), k[:, 0].double(), v[:, 0].double()
    x = (q @ k.T).masked_fill(~seen, -math.inf)
    rl = torch.logsumexp(x, 1)
    p = torch.exp(x - rl[:, None])
    ro, mag, tiny = p @ v, p @ v.abs(), seen.double() @ v.abs()
    bound = 2.0 ** -11 * (mag + ro.abs()) * 1.01 + 2.0 ** -14 * mag + 2.0 ** -33 * tiny + 2.0 ** -25
    assert ((o.double().cpu()[:, 0] - ro).abs() / bound).max() <= 1
    assert ((lse.double().cpu()[:, 0] - rl).abs() <= 2e-5 + 2e-6 * rl.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [10, 20, 26, 30])
@pytest.mark.parametrize("at", [0, 30000, 59990])
def test_f16_weights_beside_a_sink(cuda, bits, at):
    """One key takes nearly all of the weight and has no value: the rest of a long context, some 2^-26 each, is
    the output.  Prefill with few rows (cut key ranges) and with many, and decode."""
    n = 60000
    g = torch.Generator().manual_seed(bits)
    for nq in (3, 300):
        q, k, v = _sink(g, nq, n, at, bits)
        qs = q.expand(-1, 1 if nq == 3 else 64, -1).contiguous()  # 64 heads of the same rows: no cuts
        o, lse = gqa_attn.prefill(qs.to(cuda), k.to(cuda), v.to(cuda), _cu([nq]).to(cuda), _cu([n]).to(cuda),
                                  softmax_scale=1.0, check=True)
        seen = torch.arange(n)[None] <= torch.arange(nq)[:, None] + n - nq
        _near(o[:, -1:], lse[:, -1:], q, k, v, seen)
    pools = [t.view(n // 32, 32, 1, 64).transpose(1, 2).to(cuda) for t in (k, v)]
    o, lse = gqa_attn.decode(qs[:2].to(cuda), *pools, torch.arange(n // 32, dtype=torch.int32, device=cuda).expand(2, -1),
                             torch.tensor([n, n - 7], dtype=torch.int32, device=cuda), softmax_scale=1.0, check=True)
    seen = torch.arange(n)[None] < torch.tensor([[n], [n - 7]])
    _near(o[:, -1:], lse[:, -1:], q[:2], k, v, seen)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step", [0.0, 4.0, 5.5, 8.0, 11.0])
@pytest.mark.parametrize("base", [0.0, 3000.0, -8.4e6, 5.0e7, 3.0e8])
def test_scores_that_grow_by_a_few_bits_a_tile(cuda, dt, step, base):
    """Maxima that grow by about as much as a reference waits for, at small and very large scores: weights stay
    in the type's range and every part of the sum has its share."""
    n, tile = 1024, 128
    q, k, v = torch.zeros(1, 1, 64), torch.zeros(n, 1, 64), torch.ones(n, 1, 64)
    q[:, :, 0], k[:, :, 0] = 1.0, (torch.arange(n) // tile).float()[:, None] * step
    q[:, :, 1], k[:, :, 1] = 2.0 ** 12, base / 2 ** 12 if abs(base) < 1e8 else math.copysign(2.0 ** 14, base)
    q, k, v = (t.to(dt) for t in (q, k, v))
    scale = math.log(2.0)
    x = q[:, 0].double() @ k[:, 0].double().T * scale
    o, lse = gqa_attn.prefill(q.to(cuda), k.to(cuda), v.to(cuda), _cu([1]).to(cuda), _cu([n]).to(cuda), softmax_scale=scale, check=True)
    pools = [t.view(n // 64, 64, 1, 64).transpose(1, 2).to(cuda) for t in (k, v)]
    od, ld = gqa_attn.decode(q.to(cuda), *pools, torch.arange(n // 64, dtype=torch.int32, device=cuda)[None],
                             torch.tensor([n], dtype=torch.int32, device=cuda), softmax_scale=scale, check=True)
    want = torch.logsumexp(x, 1)
    # all values are 1, so the output is whatever the weights are; the scores are fp32 sums, off by some 2^-23 of the base
    for a, b in ((o, lse), (od, ld)):
        assert torch.isfinite(a).all() and (a.float() - 1).abs().max() <= 2.0 ** -6
        assert abs(float(b) - float(want)) <= 1e-3 + 2.0 ** -21 * abs(float(want))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,n", [(64, 4, 200), (128, 2, 5), (96, 2, 200), (64, 1, 6000), (128, 40, 6000)])
def test_scores_of_minus_infinity(cuda, dt, d, hq, n):
    """Keys whose scores are -inf have no weight; rows that see no others are 0 and -inf, whether the key range
    is cut or not."""
    g = torch.Generator().manual_seed(n)
    q, k, v = _randn(g, dt, 3, hq, d), _randn(g, dt, n, 1, d), _randn(g, dt, n, 1, d)
    q[:, :, 0] = 1.0
    cu = [_cu([3]).to(cuda), _cu([n]).to(cuda)]
    pools = lambda x: torch.cat([x, torch.zeros(-n % 16, 1, d, dtype=dt)]).view(-1, 16, 1, d).transpose(1, 2).to(cuda)  # noqa: E731
    table = torch.arange(-(-n // 16), dtype=torch.int32, device=cuda).expand(3, -1)
    lens = torch.tensor([n, n, 0], dtype=torch.int32, device=cuda)

    def both(k):
        return (gqa_attn.prefill(q.to(cuda), k.to(cuda), v.to(cuda), *cu, causal=False, check=True),
                gqa_attn.decode(q.to(cuda), pools(k), pools(v), table, lens, check=True))
    some, kept = k.clone(), torch.rand(n, generator=g) < 0.3
    kept[n // 2] = True
    some[~kept, :, 0] = -math.inf
    (o, lse), (od, ld) = both(some)
    x = torch.einsum("qhd,kd->qhk", q.double(), k[:, 0].double()) * d ** -0.5
    p = torch.softmax(x.masked_fill(~kept, -math.inf), -1)
    want, mag = p @ v[:, 0].double(), p @ v[:, 0].double().abs()
    # a rounding of each weight, one of the output, fp32 arithmetic (as in test_gqa_attn.py)
    bound = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dt] * (mag + want.abs()) * 1.01 + 2.0 ** -14 * mag
    assert ((o.double().cpu() - want).abs() <= bound).all() and ((od.double().cpu() - want)[:2].abs() <= bound[:2]).all()
    k[:, :, 0] = -math.inf
    for a, b in both(k):
        assert not a.any() and bool((b == -math.inf).all())


# ------------------------------------------------------------------ error words, tracing, types of tensors

def _traced(fn, *args, **more):
    """fn as a graph made on fake tensors."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    mode = FakeTensorMode()
    with mode:
        fakes = [torch.empty(a, dtype=d, device="cuda:0") for a, d in args]
        graph = make_fx(fn, **more)(*fakes)
    return graph


_BF, _I32 = torch.bfloat16, torch.int32


def _step(q, k, v, kp, vp, table, lens, refs, ones):
    """A step through five of the operators."""
    from mzoo_b200 import kv_pages
    starts = kv_pages.reserve(table, lens, refs, ones, page_size=16)
    kv_pages.append(k, v, kp, vp, table, starts)
    o, lse = gqa_attn.decode(q, kp, vp, table, lens)
    table, refs = kv_pages.compact([kp, vp], table, refs)
    return o, lse, table, refs, gqa_attn.decode(q, kp, vp, table, lens)[0]


_STEP = [((3, 4, 64), _BF), ((3, 2, 64), _BF), ((3, 2, 64), _BF), ((20, 2, 16, 64), _BF), ((20, 2, 16, 64), _BF), ((3, 5), _I32),
         ((3,), _I32), ((20,), _I32), ((3,), _I32)]


def test_traced_graphs_hold_no_tensor_of_the_trace():
    """Neither a fake error word nor any other constant; also where the checks are asked for."""
    for fn in (_step, lambda q, k, v, *rest: gqa_attn.prefill(q, k, v, torch.ops.aten.cumsum(rest[-1], 0, dtype=_I32), check=True)):
        args = _STEP if fn is _step else [((3, 4, 64), _BF), ((3, 2, 64), _BF), ((3, 2, 64), _BF), ((2,), _I32)]
        graph = _traced(fn, *args)
        assert any("gqa" in str(n.target) for n in graph.graph.nodes)
        assert not [n for n in graph.graph.nodes if n.op == "get_attr"]


def _state(dev):
    g = torch.Generator().manual_seed(0)
    x = [_randn(g, dt, *shape).to(dev) if dt == _BF else torch.zeros(*shape, dtype=dt, device=dev) for shape, dt in _STEP]
    x[5].fill_(-1)
    x[8].copy_(torch.tensor([1, 30, 16]))
    return x


@pytest.mark.gpu
def test_traced_graph_runs_and_reports(cuda):
    """A graph traced on fake tensors is the eager call, and its errors reach check_errors()."""
    graph = _traced(_step, *_STEP)
    a, b = _state(cuda), _state(cuda)
    for x, y in zip(_step(*a), graph(*b)):
        assert torch.equal(x, y)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    mzoo_b200.check_errors()
    b = _state(cuda)
    b[8].fill_(1000)  # past the table
    graph(*b)
    with pytest.raises(_lib.MzbError, match="past its page table"):
        mzoo_b200.check_errors()


@pytest.mark.gpu
def test_exported_program_runs(cuda):
    class Attend(torch.nn.Module):
        def forward(self, q, k, v, cu):
            return gqa_attn.prefill(q, k, v, cu)

    g = torch.Generator().manual_seed(0)
    q, k, v = (_randn(g, _BF, 30, h, 64).to(cuda) for h in (4, 2, 2))
    args = (q, k, v, _cu([13, 17]).to(cuda))
    with torch.no_grad():
        program = torch.export.export(Attend(), args, strict=False)
        for x, y in zip(program.module()(*args), gqa_attn.prefill(*args)):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_parameters_and_subclasses_are_tensors(cuda):
    class Named(torch.Tensor):
        pass

    from mzoo_b200 import kv_pages
    want = _step(*_state(cuda))
    for kind in (lambda t: torch.nn.Parameter(t, requires_grad=False), lambda t: t.as_subclass(Named)):
        x = [kind(t) for t in _state(cuda)]
        got = _step(*x)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        q, k, v = x[:3]
        gqa_attn.prefill(q, k, v, kind(_cu([1, 2]).to(cuda)), check=True)
        ids = kind(torch.tensor([0], dtype=_I32, device=cuda))
        kv_pages.copy_pages([x[3]], ids, ids + 1, check=True)
        kv_pages.fork([x[3]], x[5], x[6], x[7], ids, ids + 1, page_size=16, check=True)
        kv_pages.free(x[5], x[6], x[7], ids, check=True)
    with pytest.raises(_lib.MzbError, match="out of range"):
        kv_pages.free(x[5], x[6], x[7], ids + 99, check=True)
    mzoo_b200.check_errors()  # a checked call's error is its own


@pytest.mark.gpu
def test_ops_refuse_what_a_kernel_would_misread(cuda):
    """The ops themselves, without the wrappers' checks: tensors of another device or type, other shapes and
    strides are refused before a launch."""
    from mzoo_b200 import ops
    z = lambda *shape, dt=_BF, dev=cuda: torch.zeros(*shape, dtype=dt, device=dev)  # noqa: E731
    i = lambda *shape, dt=_I32, dev=cuda: torch.zeros(*shape, dtype=dt, device=dev)  # noqa: E731
    q, k, cu, pool, table, lens, refs = z(4, 4, 64), z(4, 2, 64), i(2), z(9, 2, 16, 64), i(4, 3) - 1, i(4), i(9)
    half = lambda t: t.to(torch.float16)  # noqa: E731
    good = {"gqa_prefill": (q, k, k, cu, cu, True, 1.0), "gqa_decode": (q, pool, pool, table, lens, 1.0),
            "kv_append": (k, k, pool, pool, i(4, 3), lens, None), "kv_reserve": (table, lens, refs, lens, 16), "kv_free": (table, lens, refs, cu),
            "kv_copy_pages": ([pool], cu - 1, cu - 1), "kv_fork": ([pool], table, lens, refs, cu[:0], cu[:0], 16),
            "kv_compact": ([pool], table, refs)}

    def others(name, t, at):  # what may stand in the place of t, and must not
        if isinstance(t, list):
            yield from ([x] for x in (t[0].cpu(), t[0].transpose(1, 2)))
            if name != "kv_copy_pages":  # (there any number of pages will do)
                yield from ([x] for x in (t[0][:5], t[0][0]))
        elif t.dtype == _I32:
            yield from (x for x in (t.cpu(), t.long(), t[None], t[..., None].expand(*t.shape, 2)[..., 0].transpose(0, -1)) if x is not t)
            if t.numel() > 1 and t.dim() == 1:
                yield t.repeat_interleave(2)[::2]
        else:
            yield from (t.cpu(), t[..., :32], t[0], t.transpose(-1, -2))
            if at:
                yield half(t)
    for name, args in good.items():
        getattr(ops, name)(*args, True)
        tried = 0
        for at, t in enumerate(args):
            if not isinstance(t, (torch.Tensor, list)):
                continue
            for x in others(name, t, at):
                if isinstance(x, torch.Tensor) and x.shape == t.shape and x.dtype == t.dtype and x.device == t.device and \
                        (x.is_contiguous() or (t.dtype != _I32 and x.stride(-1) == 1)):
                    continue  # as good as t
                tried += 1
                with pytest.raises((AssertionError, NotImplementedError)):  # (no CUDA tensor first: no such kernel)
                    getattr(ops, name)(*args[:at], x, *args[at + 1:], True)
        assert tried >= 4
    with pytest.raises(AssertionError, match="int32"):
        ops.gqa_prefill(q, k, k, cu, i(3), True, 1.0, True)
    with pytest.raises(AssertionError, match="apart"):
        ops.kv_copy_pages([pool[:1].expand(9, -1, -1, -1)], cu, cu, True)
    torch.cuda.synchronize()


def test_cache_writes_refuse_tensors_that_need_gradients():
    """As the attention does: a gradient would be lost without a word."""
    from mzoo_b200 import kv_pages
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        t = lambda *shape, dt=_BF: torch.empty(*shape, dtype=dt, device="cuda:0")  # noqa: E731
        table, lens, refs, ids = t(3, 4, dt=_I32), t(3, dt=_I32), t(9, dt=_I32), t(2, dt=_I32)
        for at in range(4):
            args = [t(3, 2, 64), t(3, 2, 64), t(9, 2, 16, 64), t(9, 2, 16, 64)]
            args[at].requires_grad_()
            with pytest.raises(AssertionError, match="append has no backward"):
                kv_pages.append(*args, table, lens)
            with torch.no_grad():
                kv_pages.append(*args, table, lens)
        pools = [t(9, 2, 16, 64), t(9, 2, 16, 64).requires_grad_()]
        for name, rest in (("fork", (table, lens, refs, ids, ids)), ("compact", (table, refs)), ("copy_pages", (ids, ids))):
            more = {"page_size": 16} if name == "fork" else {}
            with pytest.raises(AssertionError, match=f"{name} has no backward"):
                getattr(kv_pages, name)(pools, *rest, **more)
            with torch.no_grad():
                getattr(kv_pages, name)(pools, *rest, **more)


@pytest.mark.gpu
def test_compiled_step_is_the_eager_one(cuda):
    """torch.compile around the wrappers (the eager backend behind AOT autograd: no kernels of its own)."""
    a, b = _state(cuda), _state(cuda)
    with torch.no_grad():
        want = _step(*a)
        got = torch.compile(_step, backend="aot_eager")(*b)
    assert all(torch.equal(x, y) for x, y in zip(want, got)) and all(torch.equal(x, y) for x, y in zip(a, b))
    mzoo_b200.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_prefill_wild_offsets_of_cut_key_ranges(cuda, seed):
    """Offsets that do not ascend or leave the tensors, where key ranges are cut (test_gqa_items.py shows that
    rows, keys and parts stay inside): no error, and a sequence that overlaps no other is right."""
    g = torch.Generator().manual_seed(seed)
    q, k, v = (_randn(g, torch.bfloat16, *shape).to(cuda) for shape in ((32, 16, 64), (4000, 1, 64), (4000, 1, 64)))
    wild = [int(x) for x in torch.randint(-50, 4100, (3,), generator=g)] + [2 ** 31 - 1, -2 ** 31, 0]
    cu_k = torch.tensor([0, 3000, *wild], dtype=torch.int32, device=cuda)
    cu_q = torch.tensor([0, 16, 32, *wild[::-1][:-1]], dtype=torch.int32, device=cuda)
    cu_q[3:] = cu_q[3:].masked_fill(cu_q[3:].abs() < 32, 40)  # (none comes back to the first sequence's rows)
    o, lse = gqa_attn.prefill(q, k, v, cu_q, cu_k, check=True)
    want = gqa_attn.prefill(q[:16], k[:3000], v[:3000], _cu([16]).to(cuda), _cu([3000]).to(cuda), check=True)
    # the number of parts may differ: two results within 2^-8 (mag + |o|) of the value, both at most max |v|
    assert (o[:16].float() - want[0].float()).abs().max() <= 2.0 ** -6 * v.float().abs().max()
