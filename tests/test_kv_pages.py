"""Pages of a K / V cache (``mzoo_b200.kv_pages``) against a plain model in Python lists.  Every
result is a whole number or a copied row, so all comparisons are exact."""

import random

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mzoo_b200
from mzoo_b200 import _lib, kv_pages


def _int(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Model:
    """The state as lists, with the operations' definitions."""

    def __init__(self, S, W, P, page):
        self.table, self.lens, self.refs = [[-1] * W for _ in range(S)], [0] * S, [0] * P
        self.W, self.page = W, page
        self.data = list(range(P))  # what each page holds

    def lowest(self):
        return next((p for p, r in enumerate(self.refs) if r == 0), None)

    def reserve(self, n_new):
        starts, full = list(self.lens), False
        for b, n in enumerate(n_new):
            cols = range(-(-self.lens[b] // self.page), -(-(self.lens[b] + n) // self.page))
            if self.lens[b] + n > self.W * self.page:
                continue
            if len(cols) and (full or len(cols) > self.refs.count(0)):
                full = True  # the ones after it are not served either
                continue
            for j in cols:
                p = self.lowest()
                self.table[b][j], self.refs[p] = p, 1
            self.lens[b] += n
        return starts

    def free(self, seqs):
        for s in seqs:
            for j, p in enumerate(self.table[s]):
                if p >= 0:
                    self.refs[p] -= 1
                self.table[s][j] = -1
            self.lens[s] = 0

    def fork(self, src, dst):
        self.free(dst)
        for a, b in zip(src, dst):
            for j in range(self.lens[a] // self.page):
                self.table[b][j] = self.table[a][j]
                self.refs[self.table[a][j]] += 1
        for a, b in zip(src, dst):
            self.lens[b] = self.lens[a]
            if self.lens[a] % self.page:
                p, j = self.lowest(), self.lens[a] // self.page
                if p is None:
                    self.lens[b] = j * self.page
                    continue
                self.table[b][j], self.refs[p] = p, 1
                self.data[p] = self.data[self.table[a][j]]

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        to = list(range(len(self.refs)))
        for p in range(n, len(self.refs)):
            if self.refs[p]:
                q = self.lowest()
                to[p], self.refs[q], self.refs[p], self.data[q] = q, self.refs[p], 0, self.data[p]
        self.table = [[to[p] if p >= 0 else -1 for p in row] for row in self.table]


class Device:
    def __init__(self, m, dev, shapes=((2, 8), (3, 4, 16))):
        self.table, self.lens, self.refs = _int(m.table, dev), _int(m.lens, dev), _int(m.refs, dev)
        P = len(m.refs)
        self.pools = [torch.arange(P, device=dev, dtype=torch.int32).view(P, *[1] * len(s)).expand(P, *s).contiguous()
                      for s in shapes]

    def same(self, m):
        assert self.table.tolist() == m.table and self.lens.tolist() == m.lens and self.refs.tolist() == m.refs
        for pool in self.pools:
            want = _int(m.data, pool.device).view(-1, *[1] * (pool.dim() - 1))
            used = self.refs > 0
            assert torch.equal(pool[used], want.expand_as(pool)[used])


@pytest.mark.gpu
@pytest.mark.parametrize("S,W,P,page,seed", [(3, 4, 20, 16, 0), (40, 9, 300, 16, 1), (7, 130, 1100, 32, 2), (130, 3, 5000, 64, 3),
                                             (1, 1, 1, 16, 4), (1500, 4, 4000, 16, 5)])
def test_random_life_of_a_cache(cuda, S, W, P, page, seed):
    """Reserve, fork, free and compact in a random order, exhaustion among them."""
    rng = random.Random(seed)
    m = Model(S, W, P, page)
    d = Device(m, cuda)
    for _ in range(14):
        what = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        if what == "reserve":
            n = [rng.choice([0, 1, 1, 3, page, rng.randint(0, W * page)]) for _ in range(S)]
            starts = m.reserve(n)
            assert kv_pages.reserve(d.table, d.lens, d.refs, _int(n, cuda), page_size=page).tolist() == starts
        elif what == "free":
            seqs = rng.sample(range(S), rng.randint(0, S))
            kv_pages.free(d.table, d.lens, d.refs, _int(seqs + seqs[:2], cuda))  # a sequence named twice is freed once
            m.free(seqs)
        elif what == "fork" and S > 1:
            cut = rng.randint(1, S - 1)
            names = rng.sample(range(S), S)
            dst = names[cut:][:rng.randint(1, S)]
            src = [rng.choice(names[:cut]) for _ in dst]
            kv_pages.fork(d.pools, d.table, d.lens, d.refs, _int(src, cuda), _int(dst, cuda), page_size=page)
            m.fork(src, dst)
        elif what == "compact":
            d.table, d.refs = kv_pages.compact(d.pools, d.table, d.refs)
            m.compact()
            n = sum(r > 0 for r in m.refs)
            assert not any(m.refs[n:])
        d.same(m)
    try:
        mzoo_b200.check_errors()  # an exhausted pool or table is an error that was left out
    except _lib.MzbError as e:
        assert "no free page" in str(e)


@pytest.mark.gpu
def test_exhaustion_is_an_error(cuda):
    m = Model(3, 4, 5, 16)
    d = Device(m, cuda)
    n = [33, 48, 16]  # 3 pages, 3 pages (2 left), 1 page: behind the one that failed
    with pytest.raises(_lib.MzbError, match="no free page"):
        kv_pages.reserve(d.table, d.lens, d.refs, _int(n, cuda), page_size=16, check=True)
    m.reserve(n)
    d.same(m)
    with pytest.raises(_lib.MzbError, match="past its page table"):
        kv_pages.reserve(d.table, d.lens, d.refs, _int([40, 0, 0], cuda), page_size=16, check=True)
    m.reserve([40, 0, 0])
    d.same(m)
    m.reserve([0, 20, 0])
    kv_pages.reserve(d.table, d.lens, d.refs, _int([0, 20, 0], cuda), page_size=16, check=True)
    with pytest.raises(_lib.MzbError, match="no free page"):
        kv_pages.fork(d.pools, d.table, d.lens, d.refs, _int([0], cuda), _int([2], cuda), page_size=16, check=True)
    m.fork([0], [2])
    assert m.lens[2] == 32
    d.same(m)


@pytest.mark.gpu
def test_fork_leaves_bad_pairs_out(cuda):
    m = Model(6, 3, 30, 16)
    m.reserve([20, 40, 3, 0, 0, 0])
    d = Device(m, cuda)
    # dst 3 twice, dst 0 is a source, ids out of range: only 1 -> 5 is taken
    src, dst = [0, 1, 1, 1, 9, 0], [3, 3, 0, 5, 4, -1]
    with pytest.raises(_lib.MzbError, match="out of range"):
        kv_pages.fork(d.pools, d.table, d.lens, d.refs, _int(src, cuda), _int(dst, cuda), page_size=16, check=True)
    m.fork([1], [5])
    d.same(m)
    with pytest.raises(_lib.MzbError, match="out of range"):
        kv_pages.free(d.table, d.lens, d.refs, _int([6, -1, 2], cuda), check=True)
    m.free([2])
    d.same(m)


@pytest.mark.gpu
def test_empty_calls(cuda):
    m = Model(2, 2, 4, 16)
    m.reserve([5, 0])
    d = Device(m, cuda)
    none = _int([], cuda)
    kv_pages.fork(d.pools, d.table, d.lens, d.refs, none, none, page_size=16, check=True)
    kv_pages.free(d.table, d.lens, d.refs, none, check=True)
    kv_pages.copy_pages(d.pools, none, none, check=True)
    kv_pages.append(torch.zeros(0, 1, 8, device=cuda), torch.zeros(0, 1, 8, device=cuda), torch.zeros(4, 1, 16, 8, device=cuda),
                    torch.zeros(4, 1, 16, 8, device=cuda), d.table, d.lens, _int([0, 0, 0], cuda), check=True)
    d.same(m)


@pytest.mark.gpu
@pytest.mark.parametrize("P,live", [(1, 0), (1, 1), (50, 0), (50, 50), (1023, 400), (1025, 1000), (70000, 30000)])
def test_compact_sizes(cuda, P, live):
    g = torch.Generator().manual_seed(P)
    order = torch.randperm(P, generator=g)
    refs = torch.zeros(P, dtype=torch.int32)
    refs[order[:live]] = torch.randint(1, 5, (live,), generator=g, dtype=torch.int32)
    table = torch.full((3, max(1, live)), -1, dtype=torch.int32)
    table[1, :live] = order[:live].to(torch.int32)
    pool = torch.arange(P, dtype=torch.int32)[:, None].expand(P, 4).contiguous().to(cuda)
    new_table, new_refs = kv_pages.compact([pool], table.to(cuda), refs.to(cuda), check=True)
    assert bool((new_refs[:live] > 0).all()) and not bool((new_refs[live:]).any())
    assert bool((new_table[0] == -1).all()) and bool((new_table[2] == -1).all())
    got = new_table[1, :live].long()
    assert torch.equal(pool[got, 0].cpu(), order[:live].to(torch.int32))  # each entry still finds its page's data
    assert torch.equal(new_refs[got].cpu(), refs[order[:live]])
    stay = order[:live] < live
    assert torch.equal(got.cpu()[stay], order[:live][stay])


@pytest.mark.gpu
def test_compact_reports_a_table_that_names_a_free_page(cuda):
    pool = torch.zeros(4, 4, device=cuda)
    with pytest.raises(_lib.MzbError, match="page"):
        kv_pages.compact([pool], _int([[0, 2]], cuda), _int([1, 0, 0, 0], cuda), check=True)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dt", [((8,), torch.bfloat16), ((2, 33, 8), torch.float16), ((64, 64, 128), torch.uint8),
                                      ((5, 16, 96), torch.float32)])
def test_copy_pages(cuda, shape, dt):
    g = torch.Generator().manual_seed(0)
    base = torch.randint(0, 200, (24, 2, *shape), generator=g).to(dt).to(cuda)
    pools = [base[:, 0], base[:, 1], torch.randint(0, 200, (24, 16), generator=g).to(torch.uint8).to(cuda)]
    want = [p.clone() for p in pools]
    for p in want:
        p[torch.tensor([3, 20, 7], device=cuda)] = p[torch.tensor([1, 1, 23], device=cuda)]
    kv_pages.copy_pages(pools, _int([1, -1, 1, 23], cuda), _int([3, -1, 20, 7], cuda), check=True)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    with pytest.raises(_lib.MzbError, match="out of range"):
        kv_pages.copy_pages(pools, _int([1, 2], cuda), _int([24, -1], cuda), check=True)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


@pytest.mark.gpu
def test_many_pools(cuda):
    pools = [torch.arange(6, device=cuda)[:, None].repeat(1, 2) + 100 * i for i in range(150)]
    kv_pages.copy_pages(pools, _int([5], cuda), _int([0], cuda), check=True)
    for i, p in enumerate(pools):
        assert p[:, 0].tolist() == [100 * i + x for x in (5, 1, 2, 3, 4, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt,hkv,d,page", [(torch.bfloat16, 8, 128, 64), (torch.float16, 1, 64, 16), (torch.bfloat16, 3, 96, 32),
                                           (torch.float32, 2, 100, 16), (torch.uint8, 4, 128, 128)])
@pytest.mark.parametrize("token_major", [False, True])
def test_append(cuda, dt, hkv, d, page, token_major):
    g = torch.Generator().manual_seed(0)
    new, starts, W, P = [1, 0, 70, 200, 3], [0, 5, 31, 0, 99], 16, 60
    table = torch.randperm(P, generator=g)[:5 * 9].view(5, 9).to(torch.int32)
    table = torch.cat([table, torch.full((5, W - 9), -1, dtype=torch.int32)], 1)
    shape = (P, page, hkv, d) if token_major else (P, hkv, page, d)
    kp, vp = (torch.randint(0, 99, shape, generator=g).to(dt).to(cuda) for _ in range(2))
    if token_major:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    if page == 16:  # 200 tokens do not fit nine pages of 16
        new[3] = 140
    qkv = torch.randint(100, 200, (sum(new), 3 * hkv, d), generator=g).to(dt).to(cuda)
    k, v = qkv[:, hkv:2 * hkv], qkv[:, 2 * hkv:]
    want = [kp.clone(), vp.clone()]
    at = 0
    for b, n in enumerate(new):
        for i in range(n):
            p, s = table[b, (starts[b] + i) // page], (starts[b] + i) % page
            for w, x in zip(want, (k, v)):
                w[p, :, s] = x[at]
            at += 1
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda)
    kv_pages.append(k, v, kp, vp, table.to(cuda), _int(starts, cuda), cu, check=True)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


@pytest.mark.gpu
def test_append_leaves_rows_without_a_page_out(cuda):
    kp, vp = torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=cuda), torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=cuda)
    k = torch.ones(6, 2, 64, dtype=torch.float16, device=cuda)
    table = _int([[1, 3], [2, -1], [7, 0], [0, 0], [-2 ** 31, 0], [0, 0]], cuda)
    starts = _int([5, 16, 0, 32, 2, -1], cuda)  # only the first row has a place
    with pytest.raises(_lib.MzbError, match="past its page table"):
        kv_pages.append(k, k, kp, vp, table, starts, check=True)
    assert float(kp.float().sum()) == 128 and bool((kp[1, :, 5] == 1).all()) and torch.equal(kp, vp)


@pytest.mark.gpu
def test_large_offsets(cuda):
    """Rows and pages past 2^31 elements."""
    P, page = 5000, 128
    pool = torch.zeros(P, 8, page, 512, dtype=torch.uint8, device=cuda)  # 2.6e9 bytes
    k = torch.full((1, 8, 512), 7, dtype=torch.uint8, device=cuda)
    kv_pages.append(k, k, pool, pool, _int([[P - 1]], cuda), _int([127], cuda), check=True)
    assert int(pool[P - 1, :, 127].min()) == 7 and int(pool[P - 1, :, 126].max()) == 0
    kv_pages.copy_pages([pool], _int([P - 1], cuda), _int([P - 2], cuda), check=True)
    assert torch.equal(pool[P - 1], pool[P - 2]) and int(pool[:P - 2].max()) == 0


def _t(*shape, dtype=torch.int32):
    return torch.empty(*shape, dtype=dtype, device="cuda:0")


def test_refusals():
    cpu = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="CUDA tensors only"):
        kv_pages.free(cpu, cpu[0], cpu[0], cpu[0])
    bf = torch.bfloat16
    with FakeTensorMode():
        table, lens, refs, ids, pool = _t(3, 4), _t(3), _t(9), _t(2), _t(9, 2, 16, 64, dtype=bf)
        kv_pages.fork([pool], table, lens, refs, ids, ids, page_size=16)
        assert kv_pages.reserve(table, lens, refs, lens, page_size=16).shape == (3,)
        assert [t.shape for t in kv_pages.compact([pool], table, refs)] == [(3, 4), (9,)]
        k = _t(3, 2, 64, dtype=bf)
        kv_pages.append(k, k, pool, pool, table, lens)
        for call, word in ((lambda: kv_pages.fork([_t(8, 64)], table, lens, refs, ids, ids, page_size=16), "pool must be"),
                           (lambda: kv_pages.fork([pool[:, :, :, ::2]], table, lens, refs, ids, ids, page_size=16), "dense"),
                           (lambda: kv_pages.fork([_t(9, 3, dtype=bf)], table, lens, refs, ids, ids, page_size=16), "16 bytes"),
                           (lambda: kv_pages.fork([pool], table, lens, refs, ids, lens, page_size=16), "one length"),
                           (lambda: kv_pages.fork([pool], table, _t(4), refs, ids, ids, page_size=16), "different sequences"),
                           (lambda: kv_pages.fork([pool], table, lens, refs, ids, ids, page_size=0), "page_size"),
                           (lambda: kv_pages.free(table, lens, refs, _t(2, dtype=torch.int64)), "int32"),
                           (lambda: kv_pages.reserve(table, lens, refs, ids, page_size=16), "n_new"),
                           (lambda: kv_pages.reserve(table[:, ::2], lens, refs, lens, page_size=16), "contiguous"),
                           (lambda: kv_pages.copy_pages([], ids, ids), "at least one pool"),
                           (lambda: kv_pages.append(k, k, pool, pool, table, ids), "one row for each"),
                           (lambda: kv_pages.append(_t(5, 2, 64, dtype=bf), _t(5, 2, 64, dtype=bf), pool, pool, table, lens), "cu must be"),
                           (lambda: kv_pages.append(k.half(), k.half(), pool, pool, table, lens), "must be"),
                           (lambda: kv_pages.append(_t(3, 2, 32, dtype=bf), _t(3, 2, 32, dtype=bf), pool, pool, table, lens), "pools must be")):
            with pytest.raises(AssertionError, match=word):
                call()
