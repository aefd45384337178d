"""The prompt kernel's bounded waits: their bounds grow with the work that they
wait for; a kernel that gives up says whose rows it left, and the GPU goes on as
if nothing had happened."""
import ctypes

import numpy as np
import pytest
import torch

from magpie_tts_rt_b200 import _lib as L
from test_gpu_paged_cache import agree, i32, make, pc, queries, voices_and_members  # noqa: F401
from oracle import paged_cache as O

pytestmark = pytest.mark.gpu


def call(cache, q, wait_ns, offsets=None, groups=None, starve=False, layer=0):
    """The attention calls with bounds of their own; (out, lse).  starve: the kernel waits for keys that never come."""
    args, out, lse = cache._attention(layer, q, None, 0, 0, None, True, None)
    if offsets is not None:
        args.offsets = offsets.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    space = cache._workspace(stream, None, q.shape[1], q.shape[0]) if groups is None else groups._workspace(stream, None)
    assert L.lib.mtt_b200_launch_test_paged_attention(cache._ref, ctypes.byref(args), None if groups is None else groups._ref,
                                                      wait_ns, starve, space[0], space[1], stream) == L.STATUS_OK
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("d,hkv", [(64, 8), (128, 4)])
def test_units_longer_than_the_limit(pc, d, hkv):
    """Each CTA's share is a part of one unit after another of some 5,000 key tiles, about 10 ms each: waits that last as
    long as a unit outlive a bound of 2 ms that would not grow with the share.  The slot's pages are 64 that its table names again and
    again, so that a key's weight in the reference is how often it occurs."""
    ps, distinct, rows = 128, 64, 16384 // hkv
    length = 1_480_000
    used = -(-length // ps)
    g = torch.Generator().manual_seed(4)
    pool = torch.randn(distinct, 1, 2, hkv, ps, d, generator=g).to(torch.bfloat16)
    table = torch.randint(0, distinct, (1, used), generator=g, dtype=torch.int32)
    cache = pc.PagedCache(pool.cuda(), table.cuda(), i32([length]), torch.ones(distinct, dtype=torch.int32, device="cuda"))
    q = queries(rows, hkv, d, torch.bfloat16)
    out, lse = call(cache, q.cuda(), 2_000_000, i32([0, rows]))
    assert int(cache.status) == 0
    k, v = (pool[:, 0, i].permute(1, 0, 2, 3).reshape(hkv, distinct * ps, d).double() for i in range(2))
    for r in (0, 255, 256, rows // 2 + 3, rows - 1):
        p = length - rows + r
        full = p // ps
        times = torch.bincount(table[0, :full].long(), minlength=distinct).double()[:, None].expand(distinct, ps).clone()
        times[table[0, full], :p % ps + 1] += 1
        s = torch.einsum("hd,hkd->hk", q[r].double(), k) * d ** -0.5 + times.reshape(-1).log()
        w = torch.softmax(s, -1)
        ref = tuple(torch.einsum("hk,hkd->hd", w, x)[None] for x in (v, v.abs()))
        agree(out[r:r + 1], lse[r:r + 1], (ref[0], torch.logsumexp(s, -1)[None], ref[1]), torch.bfloat16, 1)


def test_prompt_that_gives_up(pc):
    """Every CTA waits for its first keys in vain: all slots with rows are marked, no other, and the next call is right."""
    new = [1, 0, 300, 40, 0, 129, 7]
    lengths = [n + 100 * (i % 3) for i, n in enumerate(new)]
    cache, pool, table = make(pc, lengths, 12)
    q = queries(sum(new), 12, 64, torch.bfloat16)
    offsets = [0] + np.cumsum(new).tolist()
    call(cache, q.cuda(), 2_000_000, i32(offsets), starve=True)
    assert cache.status.tolist() == [4 if n else 0 for n in new]
    cache.status.zero_()
    got, lse = call(cache, q.cuda(), 200_000_000, i32(offsets))
    agree(got, lse, O.attention(pool, table, lengths, 0, q, offsets), torch.bfloat16, max(lengths))
    assert (cache.status == 0).all()


def test_prefix_pass_that_gives_up(pc):
    """Its members are attended on their own: marked, and right."""
    cache, groups = voices_and_members(pc, [640, 96], [[1, 5, 9], [2, 30, 4]])
    plan = pc.PrefixGroups(cache, groups, q_heads=4)
    plan._c.shared_tokens = 0                       # the prefix pass in any case
    q = queries(cache.slots, 4, 64, torch.bfloat16)
    lengths = cache.lengths.tolist()
    ref = O.attention(cache.pool.cpu(), cache.page_table.cpu(), lengths, 0, q, list(range(cache.slots + 1)))
    for starve, status in ((True, [0, 0] + [4] * 6), (False, [0] * 8)):
        cache.status.zero_()
        got, lse = call(cache, q.cuda(), 2_000_000, groups=plan, starve=starve)
        agree(got, lse, ref, torch.bfloat16, max(lengths))
        assert cache.status.tolist() == status
