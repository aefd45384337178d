"""Forms of a 4-bit cache's attention that come together in a serving step: windows, sinks
and masked keys on the line of tiles (more units than clusters run at once), and
prefixes shared by slots, in both types, with and without a window.

Tolerances: of the single tokens that of test_gpu_paged_4bit.py.  Of a shared prefix,
against the cache's values with the prefix's rounded once to its type: its keys are two
numbers of the type, right to k = 2^-16 (bf16) or 2^-21 (f16; half a subnormal step
of the second is 2^-21 of keys above 2^-4, and all that is below adds at most 2^-25 |q|), so a score is off by
k scale sum |q| |k| more, and its probabilities are rounded once, u sum p |v|."""
import numpy as np
import pytest
import torch

from oracle import paged_cache as O
from test_gpu_paged_4bit import TYPES, check, some_keys, values
from test_gpu_paged_4bit_values import step_tolerance
from test_gpu_paged_cache import U, i32, pc, queries  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,group,window,sinks", [(64, 1, 60, 9), (64, 2, 20, 0), (64, 4, 33, 40), (64, 16, 70, 5), (128, 1, 48, 17),
                                                  (128, 4, 100, 0), (128, 8, 50, 20)])
def test_masked_windows_of_many_slots(pc, d, group, window, sinks):  # noqa: F811
    """1020 units, where at most 740 clusters of a CTA run at once (five CTAs of 96 registers a thread an SM).  Masked keys hold
    NaN; slot 1 sees nothing, slot 2 begins with 40 masked keys, some slots are empty."""
    lengths = np.random.default_rng(window).integers(0, 200, 340).tolist()
    lengths[1], lengths[2] = 90, 130
    check(pc, lengths, hkv=3, d=d, group=group, window=window, sinks=sinks, mask=some_keys, seed=window, dtype=TYPES[window // 10 % 2])


PREFIX, PS = 160, 16


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", [(64, 1), (64, 4), (128, 2), (128, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, PREFIX), (9, PREFIX + 3), (24, 100)])
def test_shared_prefix(pc, dtype, d, group, window, sinks):  # noqa: F811
    """Under a window a prefix is shared while it lies among the sinks; sinks 100: each slot by itself."""
    hkv, own = 2, [0, 3, 1, 20, 40, 17, 0, 30, 2]
    cache = pc.PagedCache.allocate(200, 9, 320, 2, hkv, d, PS, dtype, bits=4)
    cache.pool.fill_(0xff)                               # NaN, but for what is stored
    cache.extend(i32([PREFIX + 5] + [0] * 8))
    x = values((2, 2, PREFIX + 5, hkv, d), dtype, 2).cuda()
    cache.store(x[0], x[1], offsets=i32([0] + [PREFIX + 5] * 9))
    cache.fork(i32([-1, 0, 0, 0, 0, 0, 0, -1, 0]))
    cache.extend(i32(own))
    y = values((2, 2, sum(own), hkv, d), dtype, 3).cuda()
    cache.store(y[0], y[1], offsets=i32([0] + np.cumsum(own).tolist()))
    assert (cache.status == 0).all()
    groups = pc.PrefixGroups(cache, [(0, PREFIX + 5, [0, 1, 2, 3, 4, 5, 6, 8])], q_heads=hkv * group)
    groups._c.shared_tokens = 0                          # not known: the pass is made however small it is
    q = queries(9, hkv * group, d, dtype, 4)
    got, lse = (t.cpu().double() for t in cache.attend_shared(1, q.cuda(), groups, window=window, sinks=sinks, return_lse=True))
    pool, lengths, table = cache.pool.cpu(), cache.lengths.tolist(), cache.page_table.cpu()
    held, scale = O.held(pool, dtype), d ** -0.5
    shared = window == 0 or sinks >= PREFIX
    if shared:
        pages = table[0, :PREFIX // PS].long()
        held[pages, :, 1] = held[pages, :, 1].to(dtype).double()
    ref = O.attention(held, table, lengths, 1, q, list(range(10)), window, sinks)
    tol, tol_lse = step_tolerance(pool, table, lengths, 1, q, ref, dtype, scale, window, sinks)
    if shared:
        key = held[:, 1, 0].nan_to_num(0).abs().amax()
        size = q.double().abs().sum(-1, keepdim=True) * scale
        delta = (2.0 ** -16 * key if dtype is torch.bfloat16 else 2.0 ** -21 * key + 2.0 ** -25) * size
        members = torch.tensor([[[float(s != 7)]] for s in range(9)])
        tol = tol + members * 1.1 * ((U[dtype] + torch.expm1(2 * delta)) * ref[2] + 2.0 ** -25 * max(lengths))
        tol_lse = tol_lse + delta[..., 0]
    assert torch.isfinite(got).all() and torch.isfinite(lse).all()
    assert ((got - ref[0]).abs() <= tol).all(), ((got - ref[0]).abs() / tol).max()
    assert ((lse - ref[1]).abs() <= tol_lse).all(), ((lse - ref[1]).abs() / tol_lse).max()


@pytest.mark.parametrize("bits", [4, 16])
def test_load_of_both_into_one_tensor(pc, bits):  # noqa: F811
    """It holds the values, whatever the warps' order."""
    cache = pc.PagedCache.allocate(40, 4, 128, 3, 2, 64, 16, bits=bits)
    cache.extend(i32([100, 128, 3, 60]))
    offsets = i32([0, 100, 228, 231, 291])
    x = values((2, 3, 291, 2, 64), torch.bfloat16, 1).cuda()
    cache.store(x[0], x[1], offsets=offsets)
    _, want = cache.load(291, offsets=offsets)
    for _ in range(5):
        both = torch.zeros_like(want)
        cache.load(291, offsets=offsets, k=both, v=both)
        assert torch.equal(both, want)
