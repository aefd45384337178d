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
