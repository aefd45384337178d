"""The paged cache on several streams: what a queued call reads stays its own
until the call is done, and streams do not share workspaces."""
import pytest
import torch

from oracle import paged_cache as O
from test_gpu_paged_cache import agree, i32, make, pc, queries, voices_and_members  # noqa: F401

pytestmark = pytest.mark.gpu


def busy(stream):
    """Some tens of milliseconds of work on the stream."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(100_000_000)


def reused(size, device, at):
    """Whether the allocator gives the memory at the addresses to new tensors of the size."""
    new = [torch.empty(size, dtype=torch.int32, device=device) for _ in range(4096)]
    return any(t.data_ptr() in at for t in new)


@pytest.mark.parametrize("how", ["given", "current"])
def test_groups_dropped_while_a_call_is_queued(pc, how):
    cache, groups = voices_and_members(pc, [640, 96], [[1, 5, 9], [2, 30, 4]])
    q = queries(cache.slots, 4, 64, torch.bfloat16)
    ref = O.attention(cache.pool.cpu(), cache.page_table.cpu(), cache.lengths.tolist(), 0, q, list(range(cache.slots + 1)))
    dev = q.cuda()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    plan = pc.PrefixGroups(cache, groups, q_heads=4)
    plan._c.shared_tokens = 0               # the prefix pass in any case
    size, at = plan._data.numel(), {plan._data.data_ptr()}
    busy(side)
    if how == "given":
        got, lse = cache.attend_shared(0, dev, plan, return_lse=True, stream=side)
    else:
        with torch.cuda.stream(side):
            got, lse = cache.attend_shared(0, dev, plan, return_lse=True)
    del plan
    assert not side.query() and not reused(size, cache.device, at)
    side.synchronize()
    agree(got, lse, ref, torch.bfloat16, 700)


def test_cache_dropped_while_a_call_is_queued(pc):
    cache, _, _ = make(pc, [100, 700])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    size, at = cache.slots, {t.data_ptr() for t in (cache.status, cache.lengths)}
    busy(side)
    cache.extend(i32([1, 1]), stream=side)
    del cache
    assert not side.query() and not reused(size, "cuda", at)
    side.synchronize()


def test_two_streams_read_at_once(pc):
    """Long calls of every form on two streams, over and over, with nothing between them: each result is the one that the
    call gives alone."""
    lengths, new = [3000, 17, 900, 2500], [700, 17, 300, 40]
    cache, _, _ = make(pc, lengths, 12, spare=9)
    one, many = queries(4, 12, 64, torch.bfloat16).cuda(), queries(sum(new), 12, 64, torch.bfloat16, 2).cuda()
    offsets = i32([0, 700, 717, 1017, 1057])
    calls = [lambda s: cache.attend(1, one, stream=s), lambda s: cache.attend(0, many, offsets=offsets, stream=s),
             lambda s: cache.attend(0, many, offsets=offsets, window=300, sinks=16, stream=s)]
    alone = [c(None).clone() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [(k, calls[k](s)) for _ in range(20) for k in range(3) for s in streams]
    torch.cuda.synchronize()
    assert all(torch.equal(g, alone[k]) for k, g in got) and (cache.status == 0).all()
