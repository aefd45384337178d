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
