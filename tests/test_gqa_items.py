"""Work items of the prefill kernel, on the host: ``csrc/gqa_items.cuh`` compiled with fibers for a warp's
lanes (``gqa_items_host.cpp``).  The items of all block numbers cover every token once, each with
the key tiles that it sees, and the join finds the number of parts that the items have."""

import os
import random
import subprocess

import pytest

from conftest import ROOT

TILE = 128


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("items") / "items")
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "mzoo_b200", "csrc"),
                    os.path.join(ROOT, "tests", "gqa_items_host.cpp"), "-o", exe], check=True)

    def run(cu_q, cu_k, ntok, causal, splits, Tq, Tk, seed=-1):
        text = " ".join(map(str, [len(cu_q) - 1, ntok, int(causal), splits, Tq, Tk, seed, *cu_q, *cu_k]))
        out = subprocess.run([exe], input=text, capture_output=True, text=True, check=True, timeout=300).stdout.split("\n")
        items = [tuple(map(int, x.split()[1:])) for x in out if x.startswith("item")]
        return items, [int(x.split()[1]) for x in out if x.startswith("token")]
    return run


def _check(items, parts, cu_q, cu_k, ntok, causal, splits, Tq):
    """Against the definition, for ascending offsets from 0."""
    assert len(parts) == Tq
    got = {}
    for who, tok0, tok_end, k0, nk, n0, n1, part, of in items:
        for t in (0, 1):
            for tok in range(tok0 + t * ntok, min(tok0 + (t + 1) * ntok, tok_end)):
                assert (tok, part) not in got, f"token {tok} twice"
                got[tok, part] = (k0, nk, n1 if t else n0, of)
    b = 0
    for tok in range(Tq):
        while b < len(cu_q) - 1 and tok >= cu_q[b + 1]:
            b += 1
        if b == len(cu_q) - 1:  # padding: no keys, one part
            assert got.pop((tok, 0))[2:] == (0, 1) and parts[tok] == 1
            continue
        nq, keys, i = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b], tok - cu_q[b]
        sees = max(0, min(keys, i + keys - nq + 1)) if causal else keys
        of, at = parts[tok], cu_k[b]
        assert 1 <= of <= splits
        for part in range(of):
            k0, nk, n, said = got.pop((tok, part))
            assert said == of and k0 == at and nk >= 0
            # tiles of the part hold what the token sees of it
            assert max(0, min(nk, cu_k[b] + sees - k0)) <= n * TILE
            at += nk
        assert at >= cu_k[b] + sees and at <= cu_k[b + 1]
    assert not got


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


CASES = [([32], [4000], 8, 16), ([16], [4000], 8, 16), ([1], [1537], 128, 74), ([2, 5, 1], [1600, 3, 4000], 10, 9),
         ([33, 0, 7], [1800, 2000, 0], 3, 5), ([300], [20], 42, 1), ([64, 0, 1, 129], [64, 0, 1, 129], 32, 1),
         ([0, 0], [50, 0], 16, 4), ([3] * 33, [700] * 33, 4, 3), ([7, 0, 90] * 30, [9, 4, 300] * 30, 16, 1)]


@pytest.mark.parametrize("new,keys,ntok,splits", CASES)
@pytest.mark.parametrize("pad", [0, 1, 16, 50])
@pytest.mark.parametrize("causal", [True, False])
def test_items_cover_every_row_once(host, new, keys, ntok, splits, pad, causal):
    cu_q, cu_k = _cu(new), _cu(keys)
    Tq = cu_q[-1] + pad
    if Tq:
        items, parts = host(cu_q, cu_k, ntok, causal, splits, Tq, cu_k[-1])
        _check(items, parts, cu_q, cu_k, ntok, causal, splits, Tq)


@pytest.mark.parametrize("seed", range(30))
def test_parts_stay_in_bounds_whatever_the_offsets_hold(host, seed):
    """Offsets that do not ascend or leave the tensors: rows, keys and part counts stay inside."""
    rng = random.Random(seed)
    B, Tq, Tk, splits = rng.randint(1, 40), rng.randint(1, 60), rng.randint(1, 5000), rng.randint(1, 40)
    cu_q, cu_k = ([rng.choice([rng.randint(-9, t + 9), -2 ** 31, 2 ** 31 - 1, 0, t]) for _ in range(B + 1)] for t in (Tq, Tk))
    items, parts = host(cu_q, cu_k, rng.choice([1, 3, 8, 128]), seed % 2, splits, Tq, Tk)
    assert len(parts) == Tq and all(1 <= n <= splits for n in parts)
    for who, tok0, tok_end, k0, nk, n0, n1, part, of in items:
        assert 0 <= tok0 and tok_end <= Tq and 0 <= k0 and k0 + max(nk, 0) <= Tk and 0 <= part < of <= splits


@pytest.mark.parametrize("new,keys,ntok,splits", CASES[-2:] + [([5, 0, 300] * 25, [5, 2, 300] * 25, 8, 1), CASES[6]])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_block_numbers_in_any_order(host, new, keys, ntok, splits, seed):
    """A running block takes over numbers of others, in whatever order they come."""
    cu_q, cu_k = _cu(new), _cu(keys)
    items, parts = host(cu_q, cu_k, ntok, True, splits, cu_q[-1] + 9, cu_k[-1], seed)
    _check(items, parts, cu_q, cu_k, ntok, True, splits, cu_q[-1] + 9)
