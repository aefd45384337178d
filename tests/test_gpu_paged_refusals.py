"""What the paged cache refuses on the device does no harm, and what it can do
it does: tokens without room, rows that no slot claims, heads and rows whose
strides have no meaning."""
import numpy as np
import pytest
import torch

from oracle import paged_cache as O
from test_gpu_paged_cache import agree, both_store, i32, make, paired, pc, queries, same  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layer", [None, 1])
@pytest.mark.parametrize("ps", [16, 64])
def test_refused_tokens_are_not_stored(pc, ps, layer):
    """extend, store, extend, store, ... with a pool that is soon full: a slot that got no room keeps its tokens, whatever
    rows are stored for it, in both forms of store, until it is given room again."""
    rng = np.random.default_rng(ps)
    cache, sim = paired(pc, 5, 5, 4 * ps, ps=ps)
    n = cache.slots

    def step(counts):
        sim.extend(counts)
        cache.extend(i32(counts))
        both_store(cache, sim, [0] + np.cumsum(np.maximum(counts, 0)).tolist(), rng, layer)
        same(cache, sim)

    step([ps, ps - 2, 3, ps, 5])                    # every page is taken
    before = cache.pool.clone()
    step([1, 0, ps + 4, 2, -3])                     # no room for any, a count out of range
    assert torch.equal(cache.pool.view(torch.int16), before.view(torch.int16))
    assert cache.status.tolist() == [2, 0, 2, 2, 1]
    # the decode form, a row for every slot: only those that asked for nothing or were given room
    k, v = queries(n, 2, 64, cache.dtype, 3), queries(n, 2, 64, cache.dtype, 4)
    for counts in ([1, 1, 1, 1, 1], [1, 1, 0, 1, 0]):
        sim.extend(counts)
        cache.extend(i32(counts))
        sim.store(k[None], v[None], list(range(n + 1)), [0])
        cache.store(k.cuda(), v.cuda(), layer=0)
        same(cache, sim)
    assert sim.refused == [True, False, False, True, False]
    # released, and taken over from another slot: the slots are written again
    for mask, source in (([True] + [False] * 4, [1] + [-1] * 4), ([False] * 2 + [True] + [False] * 2, [-1, -1, -1, 2, -1])):
        sim.free(mask)
        cache.free(torch.tensor(mask, device="cuda"))
        sim.fork(source, deep=True)
        cache.fork(i32(source), deep=True)
        sim.store(k[None], v[None], [0, 1, 2, 3, 4, 5] if sim.lengths[2] else [0, 1, 2, 2, 2, 3], [1])
        cache.store(k.cuda(), v.cuda(), layer=1, offsets=None if sim.lengths[2] else i32([0, 1, 2, 2, 2, 3]))
        same(cache, sim)
