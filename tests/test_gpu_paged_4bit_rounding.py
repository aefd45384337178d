"""Prompts over a 4-bit cache round a probability once.

Keys and values here are held as they are (groups without a spread), values are
1, -1 or 0, and each key's score is chosen (two groups of 64 dims add up to it), so
that rounding the probabilities to u = finfo.eps / 2 moves the result by nearly all that
it may: one rounding stays below u (sum_j p_j |v_j| + |out|), the tolerance of a 16-bit
cache, and a second one of the same weights, down as the first, goes past it (1.2 to
1.3 times, worked out in 64 bits)."""
import math

import numpy as np
import pytest
import torch

from oracle import paged_cache as O
from test_gpu_paged_4bit import TYPES, token_bytes
from test_gpu_paged_cache import agree, i32, pc  # noqa: F401

pytestmark = pytest.mark.gpu

D, PS = 128, 16


def plain_keys(pc, scores, signs, dtype):  # noqa: F811
    """A cache of one slot and key head whose key j gives `scores[j]` for a query of ones in dims 0 and 64, value signs[j]."""
    n = len(scores)
    pages = -(-n // PS)
    pool = torch.full((pages, 1, 2, 1, PS, token_bytes(D)), 0xff, dtype=torch.uint8)
    s = torch.tensor(scores, dtype=torch.float64)
    near = s.to(dtype)
    rest = (s - near.double()).to(dtype)
    for j in range(n):
        k = torch.cat([near[j].expand(64), rest[j].expand(64)])
        O.put4(pool[j // PS, 0, 0], j % PS, k[None])
        O.put4(pool[j // PS, 0, 1], j % PS, torch.full((1, D), float(signs[j]), dtype=dtype))
    table = torch.arange(pages, dtype=torch.int32)[None]
    return pc.PagedCache(pool.cuda(), table.cuda(), i32([n]), torch.ones(pages, dtype=torch.int32, device="cuda"), dtype=dtype), pool, table


def held_to_one_rounding(pc, scores, signs, new, sizes, dtype, window=0):  # noqa: F811
    """sizes: of the query heads, which share the key head."""
    cache, pool, table = plain_keys(pc, scores, signs, dtype)
    n = len(scores)
    q = torch.zeros(new, len(sizes), D, dtype=dtype)
    q[:, :, 0] = q[:, :, 64] = torch.tensor(sizes, dtype=dtype)
    ln2 = math.log(2)                                   # scores are in powers of two
    held = O.held(pool, dtype)
    ref = O.attention(held, table, [n], 0, q, [0, new], window, 0, ln2)
    got, lse = cache.attend(0, q.cuda(), offsets=i32([0, new]), window=window, scale=ln2, return_lse=True)
    agree(got, lse, ref, dtype, n)


def close(dtype):
    """Exponents just above a power of two that round down to it, and up from it."""
    u = torch.finfo(dtype).eps / 2
    return math.log2(1 + 0.97 * u), math.log2(1 + 1.03 * u)


def halves(dtype):
    """32 keys of which one has the largest weight and 31 half of it, 32 keys of nearly twice that: weights of the first are
    cut by the factor's rounding as by their own."""
    down, up = close(dtype)
    b = 1 - down
    return [0.] + [b * -1.] * 31 + [b] + [b - 1 + up] * 14 + [-30.] * 17, [1.] * 32 + [-1.] * 32


@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_beside_one_whose_maximum_rises(pc, dtype):  # noqa: F811
    """The second head's scores are 40 times the first one's: its maximum has to be looked for at keys 32 to 63."""
    scores, signs = halves(dtype)
    held_to_one_rounding(pc, scores, signs, 1, [1., 40.], dtype)
    held_to_one_rounding(pc, scores, signs, 1, [1.], dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_beside_one_that_has_seen_nothing(pc, dtype):  # noqa: F811
    """Under a window the last row's keys begin where the first one's second 32 do (of which key 0 is out of reach)."""
    scores, signs = halves(dtype)
    scores[:2] = [-30., 0.]
    held_to_one_rounding(pc, scores + [-30.] * 32, signs + [0.] * 32, 32, [1.], dtype, window=64)


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_as_large_as_they_may_become(pc, dtype):  # noqa: F811
    """After a tile of small weights, 32 keys whose weights are just not too large for the maximum before, and 32 that are."""
    down, up = close(dtype)
    bias = 8. if dtype is torch.float16 else 0.         # of the weights, in powers of two
    top = 15 - down - bias
    scores = [0.] * 128 + [9 + down - bias] * 32 + [top] + [top - 6 + up] * 31 + [-30.] * 64
    signs = [0.] * 128 + [1.] * 32 + [0.] + [-1.] * 31 + [0.] * 64
    held_to_one_rounding(pc, scores, signs, 1, [1.], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [0, 64])
def test_rising_scores(pc, dtype, window):  # noqa: F811
    """Every 32 keys by some 0.3 to 20 powers of two more than the ones before: the maximum is looked for all the time."""
    rng = np.random.default_rng(1)
    scores = np.repeat(np.cumsum(rng.uniform(0.3, 20, 20)), 32) + rng.uniform(-3, 0, 640)
    signs = rng.choice([-1., 1.], 640)
    held_to_one_rounding(pc, list(scores), list(signs), 40, [1., 0.25, -1.], dtype, window)
