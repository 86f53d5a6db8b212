"""Page operations raise exactly where a plain model says that something could not be done, and with that cause."""

import random

import pytest
import torch

import mzoo_b200
from mzoo_b200 import _lib, kv_pages
from test_kv_pages import Device, Model, _int

TABLE, IDS, NO_PAGE = _lib.MZB_ERR_TABLE, _lib.MZB_ERR_PAGES, _lib.MZB_ERR_NO_PAGE


def _expect(causes, call):
    """call raises with one of the causes, or, where there is none, does not."""
    try:
        call()
    except _lib.MzbError as e:
        assert e.code in causes, f"{e} (expected {causes})"
    else:
        assert not causes, f"no error, expected {causes}"


@pytest.mark.gpu
@pytest.mark.parametrize("S,W,P,page,seed", [(3, 4, 20, 16, 0), (40, 9, 120, 16, 1), (7, 130, 500, 32, 2), (130, 3, 150, 64, 3),
                                             (1, 1, 1, 16, 4), (1500, 4, 2500, 16, 5), (6, 5, 400, 16, 6)])
def test_errors_of_a_random_life(cuda, S, W, P, page, seed):
    rng = random.Random(100 + seed)
    m = Model(S, W, P, page)
    d = Device(m, cuda)
    mzoo_b200.check_errors()
    for _ in range(25):
        what = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        if what == "reserve":
            n = [rng.choice([0, 1, 1, 3, page, rng.randint(0, W * page // 2)]) for _ in range(S)]
            was = m.reserve(n)
            causes = {TABLE if x + k > W * page else NO_PAGE for x, k, now in zip(was, n, m.lens) if now != x + k}
            _expect(causes, lambda: kv_pages.reserve(d.table, d.lens, d.refs, _int(n, cuda), page_size=page, check=True))
        elif what == "free":
            seqs, bad = rng.sample(range(S), rng.randint(0, S)), rng.choice([[], [S], [-1]])
            m.free(seqs)
            _expect({IDS} if bad else set(), lambda: kv_pages.free(d.table, d.lens, d.refs, _int(seqs + bad, cuda), check=True))
        elif what == "fork" and S > 1:
            cut = rng.randint(1, S - 1)
            names = rng.sample(range(S), S)
            dst = names[cut:][:rng.randint(1, S)]
            src = [rng.choice(names[:cut]) for _ in dst]
            m.fork(src, dst)
            causes = {NO_PAGE for a, b in zip(src, dst) if m.lens[a] != m.lens[b]}
            _expect(causes, lambda: kv_pages.fork(d.pools, d.table, d.lens, d.refs, _int(src, cuda), _int(dst, cuda), page_size=page,
                                                  check=True))
        elif what == "compact":
            d.table, d.refs = kv_pages.compact(d.pools, d.table, d.refs, check=True)
            m.compact()
        d.same(m)
    mzoo_b200.check_errors()  # the checked calls kept their errors to themselves


@pytest.mark.gpu
def test_append_causes_and_the_first_of_several(cuda):
    pool, k = torch.zeros(4, 1, 16, 64, device=cuda), torch.ones(1, 1, 64, device=cuda)
    for entry, start, cause in ((0, 16, TABLE), (0, -1, TABLE), (0, 2 ** 31 - 1, TABLE), (-1, 3, IDS), (4, 3, IDS), (3, 15, None)):
        args = (k, k, pool, pool.clone(), _int([[entry]], cuda), _int([start], cuda))
        _expect({cause} - {None}, lambda: kv_pages.append(*args, check=True))
        kv_pages.append(*args)
        kv_pages.free(_int([[-1]], cuda), _int([0], cuda), _int([0], cuda), _int([7], cuda))  # another error behind it
        with pytest.raises(_lib.MzbError) as e:
            mzoo_b200.check_errors()
        assert e.value.code == (cause or IDS)
        mzoo_b200.check_errors()


def test_messages_name_the_cause_first():
    from mzoo_b200 import ops
    for code, text in ((TABLE, "past its page table"), (IDS, "id out of range"), (NO_PAGE, "no free page")):
        with pytest.raises(_lib.MzbError, match=rf"^kv: a?n?o? ?.*{text} \(") as e:
            ops._raise_code(code, "kv")
        assert e.value.code == code
    ops._raise_code(0, "kv")
