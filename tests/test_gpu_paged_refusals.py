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


def odd(t, *sizes):
    """t's values with other strides: dimensions of one with sizes[i] as theirs."""
    st = list(t.stride())
    for dim, stride in sizes:
        assert t.shape[dim] == 1
        st[dim] = stride
    return torch.as_strided(t, t.shape, st)


@pytest.mark.parametrize("prompt", [False, True])
def test_one_head_and_one_row_of_any_stride(pc, prompt):
    """A single head's stride, a single row's, a single layer's and a single slot's have no meaning."""
    lengths = [40, 57, 3]
    cache, pool, table = make(pc, lengths, hkv=1, layers=1)
    q = queries(3, 1, 64, torch.bfloat16)
    offsets = [0, 1, 2, 3]
    ref = O.attention(pool, table, lengths, 0, q, offsets)
    args = dict(offsets=i32(offsets)) if prompt else {}
    got, lse = cache.attend(0, odd(q.cuda(), (1, 7)), out=odd(torch.empty(3, 1, 64, dtype=q.dtype, device="cuda"), (1, 3)),
                            return_lse=True, **args)
    agree(got, lse, ref, torch.bfloat16, 57)
    one, pool, table = make(pc, [57], hkv=2, layers=1)
    q = queries(1, 4, 64, torch.bfloat16)
    mask = torch.rand(1, one.table_pages * 16, generator=torch.Generator().manual_seed(1)) < 0.5
    ref = O.attention(pool, table, [57], 0, q, [0, 1], key_mask=mask)
    args = dict(offsets=i32([0, 1])) if prompt else {}
    got, lse = one.attend(0, odd(q.cuda(), (0, 3)), key_mask=odd(mask.cuda(), (0, 5)), return_lse=True, **args)
    agree(got, lse, ref, torch.bfloat16, 57)


@pytest.mark.parametrize("hkv,rows,form", [(1, 3, "layer"), (2, 1, "layer"), (1, 3, "all"), (2, 1, "all")])
def test_stores_of_any_stride(pc, hkv, rows, form):
    cache, sim = paired(pc, 8, rows, 64, layers=1, hkv=hkv)
    sim.extend([5] * rows)
    cache.extend(i32([5] * rows))
    k, v = queries(rows, hkv, 64, cache.dtype, 3), queries(rows, hkv, 64, cache.dtype, 4)
    sim.store(k[None], v[None], list(range(rows + 1)), [0])
    dims = [(1, 9)] if hkv == 1 else [(0, 11)]
    if form == "layer":
        cache.store(odd(k.cuda(), *dims), odd(v.cuda(), *dims), layer=0)
    else:
        dims = [(0, 13)] + [(d + 1, s) for d, s in dims]
        cache.store(odd(k.cuda()[None], *dims), odd(v.cuda()[None], *dims))
    same(cache, sim)


@pytest.mark.parametrize("d,group", [(64, 1), (128, 3)])
@pytest.mark.parametrize("before,after", [(0, 5), (300, 0), (3, 700), (0, 0)])
def test_rows_that_no_slot_has(pc, before, after, d, group):
    """Offsets that begin after the first row or end before the last: those rows get 0 and -inf, whatever was there."""
    lengths, new = [300, 40, 0, 9], [290, 0, 0, 9]
    cache, pool, table = make(pc, lengths, 2, d)
    offsets = (before + np.cumsum([0] + new)).tolist()
    rows = offsets[-1] + after
    q = queries(rows, 2 * group, d, torch.bfloat16)
    ref = O.attention(pool, table, lengths, 0, q, offsets)
    out = torch.full((rows, 2 * group + 1, d), float("nan"), dtype=q.dtype, device="cuda")
    trash = torch.full((rows, 2 * group), 7.0, device="cuda")   # where the call's lse will probably lie
    del trash
    got, lse = cache.attend(0, q.cuda(), out=out[:, :2 * group], offsets=i32(offsets), return_lse=True)
    agree(got, lse, ref, torch.bfloat16, 300)
    assert torch.isnan(out[:, 2 * group]).all()
    free = torch.ones(rows, dtype=torch.bool)
    free[before:offsets[-1]] = False
    assert (got.cpu()[free] == 0).all() and (lse.cpu()[free] == float("-inf")).all()
    none = cache.attend(0, q.cuda(), offsets=i32([rows] * 5))
    assert (none == 0).all()
