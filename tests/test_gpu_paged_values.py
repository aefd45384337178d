"""What the paged cache's attention makes of its values: those that no query can
see do not matter, and small probabilities count."""
import numpy as np
import pytest
import torch

from oracle import paged_cache as O
from test_gpu_paged_cache import U, agree, i32, make, pc, queries, voices_and_members  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 16), (64, 130), (129, 1), (250, 0)])
@pytest.mark.parametrize("new", [[300, 1, 5], [40, 257, 64], [1, 1, 1]])
@pytest.mark.parametrize("d,group,bad", [(64, 1, float("nan")), (128, 4, float("inf")), (64, 16, float("nan"))])
def test_prompt_nothing_out_of_sight_counts(pc, window, sinks, new, d, group, bad):
    """Keys and values that every query's window has left behind are not finite: the result is what it is without them."""
    lengths = [700, 610, 333]
    cache, pool, table = make(pc, lengths, 2, d)
    q = queries(sum(new), 2 * group, d, torch.bfloat16)
    offsets = [0] + np.cumsum(new).tolist()
    ref = O.attention(pool, table, lengths, 0, q, offsets, window, sinks)
    for i, n in enumerate(lengths):
        for j in range(sinks, n - new[i] - window + 1):
            cache.pool[table[i, j // 16], :, :, :, j % 16] = bad
    got, lse = cache.attend(0, q.cuda(), offsets=i32(offsets), window=window, sinks=sinks, return_lse=True)
    agree(got, lse, ref, torch.bfloat16, 700)


# one cluster's keys, several clusters', the line of tiles; one and sixteen query heads per key head
@pytest.mark.parametrize("keys,slots", [(2, 1), (466, 2), (1000, 1), (700, 60)])
@pytest.mark.parametrize("dtype,d,group", [(torch.bfloat16, 64, 1), (torch.float16, 64, 16), (torch.bfloat16, 128, 16),
                                           (torch.float16, 128, 1)])
def test_step_weights_are_finer_than_the_caches_type(pc, keys, slots, dtype, d, group):
    """Half of the values are 1, the others -1 with weights a little smaller (by less than 16 bits can tell): the
    difference is what is left.  Tolerance: the result's rounding, 1.1 u |o|, and 2^-16 of sum p|v| for weights held to
    2^-17 or better and f32 sums and exponentials."""
    cache, pool, table = make(pc, [keys] * slots, 1, d, dtype=dtype)
    pool.fill_(0.0)
    delta = torch.tensor(0.002 if dtype == torch.bfloat16 else 0.0002).to(dtype)
    for i in range(slots):
        for j in range(keys):
            at = pool[table[i, j // 16], 1, :, 0, j % 16]
            at[0, 0] = 0 if j % 2 else -delta
            at[1] = 1 if j % 2 else -1
    cache.pool.copy_(pool)
    q = torch.zeros(slots, group, d, dtype=dtype)
    q[:, :, 0] = torch.linspace(0.7, 1.3, group)[None].to(dtype)
    out, ref_lse, weight = O.attention(pool, table, [keys] * slots, 1, q, list(range(slots + 1)), scale=1.0)
    got, lse = cache.attend(1, q.cuda(), scale=1.0, return_lse=True)
    tol = 1.1 * U[dtype] * out.abs() + 2.0 ** -16 * weight
    err = (got.cpu().double() - out).abs()
    assert (err <= tol).all(), (err / tol).max().item()
    assert (lse.cpu().double() - ref_lse).abs().max().item() <= 5e-4


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [6.4, 13.4, 20.4, 24.4, 27.4])
@pytest.mark.parametrize("form,slots", [("step", 2), ("step", 1200), ("prompt", 1200), ("shared", 400)])
@pytest.mark.parametrize("sink_at", [0, 40000])
def test_many_small_probabilities(pc, dtype, bits, form, slots, sink_at):
    """One key whose value is zero takes nearly all, 65,536 others 2^-bits of it each: the result is theirs alone.  Slots
    enough that most keep their keys together (each part of a slot has a largest probability of its own).
    Tolerance: the formulas of agree(), without its allowance for small f16 probabilities but with the 2^-33 of the
    largest that such a one may lose below 2^-22 of it, and the smallest step of the result's type."""
    n, d, ps = 65536, 64, 128
    g = torch.Generator().manual_seed(int(bits))
    pool = torch.zeros(n // ps, 1, 2, 1, ps, d)
    pool[:, :, 1] = 1 + torch.rand(pool[:, :, 1].shape, generator=g)
    pool[sink_at // ps, 0, 0, 0, sink_at % ps, 0] = bits * 0.6931 / 8
    pool[sink_at // ps, 0, 1, 0, sink_at % ps] = 0
    pool = pool.to(dtype)
    table = torch.arange(n // ps, dtype=torch.int32).expand(slots, n // ps).contiguous()    # all slots hold all pages
    cache = pc.PagedCache(pool.cuda(), table.cuda(), i32([n] * slots), i32([slots] * (n // ps)))
    q = torch.zeros(slots, 1, d, dtype=dtype)
    q[:, :, 0] = 8
    out, ref_lse, weight = O.attention(pool, table[:1], [n], 0, q[:1], [0, 1], scale=1.0)
    if form == "shared":
        plan = pc.PrefixGroups(cache, [(0, n, [i]) for i in range(slots)], q_heads=1)
        plan._c.shared_tokens = 0
        got, lse = cache.attend_shared(0, q.cuda(), plan, scale=1.0, return_lse=True)
    else:
        offsets = i32(list(range(slots + 1))) if form == "prompt" else None
        got, lse = cache.attend(0, q.cuda(), offsets=offsets, scale=1.0, return_lse=True)
    tol = 1.1 * U[dtype] * (out.abs() + weight)
    if dtype == torch.float16:
        tol += 2.0 ** -33 * 2 * n + 2.0 ** -25
    err = (got.cpu().double() - out).abs()
    assert (err <= tol).all(), (err / tol).max().item()
    assert (lse.cpu().double() - ref_lse).abs().max().item() <= 5e-4
    assert (cache.status == 0).all()
