"""The paged cache at sizes of which its other tests have only one side: many
query heads per key head in prompts, page tables much wider than their slots,
pools of several rounds of the plans that walk them."""
import numpy as np
import pytest
import torch

from oracle import paged_cache as O
from test_gpu_paged_cache import agree, check_attend, i32, make, paired, pc, queries, same  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [5, 13, 24, 48, 64])
@pytest.mark.parametrize("hkv,d,dtype,window", [(2, 64, torch.bfloat16, 0), (1, 128, torch.float16, 90)])
def test_prompt_many_heads(pc, group, hkv, d, dtype, window):
    check_attend(pc, [300, 0, 17, 64, 500], [57, 0, 17, 1, 130], group=group, hkv=hkv, d=d, dtype=dtype, window=window,
                 sinks=20 if window else 0)


@pytest.mark.parametrize("lengths,hkv,group,d", [([467, 40], 12, 1, 64), ([467, 0, 1, 33], 2, 4, 128),
                                                 ([100 + 7 * i for i in range(40)], 12, 1, 64), ([5000, 3], 1, 13, 64)])
@pytest.mark.parametrize("table_pages", [400, 4096, 40000])
def test_wide_tables(pc, lengths, hkv, group, d, table_pages):
    """Slots that could hold up to 640,000 tokens and hold a few: both forms of the step, and the prompt."""
    cache, pool, table = make(pc, lengths, hkv, d, table_pages=table_pages)
    q = queries(len(lengths), hkv * group, d, torch.bfloat16)
    ref = O.attention(pool, table, lengths, 1, q, list(range(len(lengths) + 1)))
    for offsets in (None, i32(list(range(len(lengths) + 1)))):
        got, lse = cache.attend(1, q.cuda(), offsets=offsets, return_lse=True)
        agree(got, lse, ref, torch.bfloat16, max(lengths))
    assert (cache.status == 0).all()


def test_upkeep_of_a_large_pool(pc):
    """60,000 pages: free ones past several rounds of the list, moved ones from and to everywhere."""
    cache, sim = paired(pc, 60000, 18, 4096 * 16, layers=1, hkv=1)

    def extend(counts):
        sim.extend(counts)
        cache.extend(i32(counts))
        same(cache, sim)

    def free(slots):
        mask = [i in slots for i in range(18)]
        sim.free(mask)
        cache.free(torch.tensor(mask, device="cuda"))

    def compact():
        assert sim.compact() == (cache.compact(), int(cache.live))[1]
        same(cache, sim)

    extend([65536] * 14 + [0] * 4)              # 57,344 pages in use: what is free lies at the end
    extend([0] * 14 + [20000, 30000, 1, 0])     # enough for the first alone
    assert cache.status.tolist()[14:17] == [0, 2, 2]
    free([1, 4, 5, 11])
    sim.fork([-1] * 17 + [14], deep=True)
    cache.fork(i32([-1] * 17 + [14]), deep=True)
    extend([0, 33, 0, 0, 65536, 17] + [0] * 9 + [5000, 0, 0])
    compact()
    free([0, 2, 3, 6, 7, 8, 9, 10])             # mostly free now
    extend([1] * 13 + [0] * 5)
    free([4, 14])
    compact()
