"""The serving example end to end: prompts, shared pages, single-token steps, release, compaction."""

import os
import sys

import pytest
import torch

from conftest import ROOT

sys.path.insert(0, os.path.join(ROOT, "examples"))


@pytest.mark.gpu
def test_cached_steps_equal_a_run_without_a_cache(cuda):
    import mzoo_b200
    import paged_serving as ps
    from mzoo_b200 import kv_pages
    model, texts, logits, cache = ps.serve(lengths=(5, 40, 17, 16, 1), answers=3, steps=20)
    # the two runs round attention outputs to bf16 in different places: 2 layers of unit-variance
    # residuals and a head of unit-variance logits leave some 2^-8 * sqrt(layers) of each
    want = ps.whole(model, texts)
    assert float((logits.float() - want.float()).norm() / want.float().norm()) < 4 * 2.0 ** -8
    refs = cache.refs.clone()
    assert cache.lens.tolist() == [len(t) for t in texts]
    # the 40-token prompt's two full pages are shared by its three answers
    assert cache.table[[1, 6, 11], :2].unique(dim=0).shape[0] == 1 and int(refs[cache.table[1, 0].long()]) == 3

    # release two answers of every prompt, move the rest together: the next step is unchanged
    keep, gone = torch.arange(10, 15), torch.arange(0, 10, dtype=torch.int32, device=cuda)
    token = logits.argmax(-1)
    with torch.no_grad():
        before = ps.step(model, cache, token)[keep]
    kv_pages.free(cache.table, cache.lens, cache.refs, gone)
    cache.table, cache.refs = kv_pages.compact(cache.pools, cache.table, cache.refs)
    live = int((cache.refs > 0).sum())
    assert live == sum(-(-int(n) // ps.PAGE) for n in cache.lens) and not bool(cache.refs[live:].any())
    cache.lens[keep.to(cuda)] -= 1  # run the same token once more
    with torch.no_grad():
        cache.table, cache.lens = cache.table[10:].contiguous(), cache.lens[10:].contiguous()
        after = ps.step(model, cache, token[keep])
    mzoo_b200.check_errors()
    assert torch.equal(before, after)
