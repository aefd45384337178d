"""Attention over a 4-bit cache whose groups are awkward: as large as the type goes,
constant, with steps that are subnormal, of steps without codes.  What load gives finite
is attended to as that.

Tolerance of a single token's attention, derived, key by key.  A score is scale times
the sum over groups of step (q.(16 + c) - 16 sum q) + low sum q in f32, off by
delta_j <= (2 D + 16) 2^-24 scale sum_d |q_d| (47 step_j + |low_j|); a weighted mean by
(e^{2 delta} - 1) sum_j p_j |v_j| then.  The weights p step are two bf16 numbers, off by
2^-16, and a value by 2^-16 sum_j p_j 31 step_j of its group.  The exponentials
(2^-22 each) and the sums in f32 are allowed for by 2^-16 of sum_j p_j (31 step_j +
|low_j|) again, the result is rounded once, and a tenth is added."""
import numpy as np
import pytest
import torch

from oracle import paged_cache as O
from test_gpu_paged_4bit import TYPES, make4, values, values_rounded
from test_gpu_paged_cache import agree, i32, pc, queries  # noqa: F401

pytestmark = pytest.mark.gpu

LARGE = {torch.bfloat16: 1.2e38, torch.float16: 3e4}    # 31 steps, and 16 below the smallest, are past single precision


def put(pool, table, slot, token, kv, x):
    """x [heads, d] becomes a token's keys or values in every layer."""
    ps = pool.shape[4]
    for layer in range(pool.shape[1]):
        O.put4(pool[table[slot, token // ps], layer, kv], token % ps, x)


def large(heads, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (2 * torch.rand(heads, d // 64, 64, generator=g) - 1) * LARGE[dtype]
    x[..., 5], x[..., 9] = LARGE[dtype], -LARGE[dtype]
    return x.reshape(heads, d).to(dtype)


def awkward(heads, d, dtype, seed):
    """Groups without a spread, of subnormal steps, of steps that have no codes; a token each."""
    x = values((4, heads, d), dtype, seed)
    x[0] = 0.625
    x[1] = (x[1].float() * 1e-7).to(dtype)
    x[2] = ((torch.arange(d) % 5) * (2.0 ** -130 if dtype is torch.bfloat16 else 2.0 ** -24)).to(dtype)
    x[3] = torch.where(torch.arange(d) % 2 == 0, -0.0, 0.0).to(dtype)
    return x


def pairs_of(pool, dtype):
    """step and low of every dim in 64 bits, laid out as the values."""
    ps, d = pool.shape[4], pool.shape[5] * 16 // 9
    flat = pool.reshape(*pool.shape[:4], -1)
    p = flat[..., ps * d // 2:].contiguous().view(dtype).double().reshape(*pool.shape[:4], ps, d // 64, 2)
    return p[..., 0].repeat_interleave(64, -1), p[..., 1].repeat_interleave(64, -1)


def step_tolerance(pool, table, lengths, layer, q, ref, dtype, scale, window=0, sinks=0):
    """(of each output, of each log-sum-exp); see above."""
    held, (step, low) = O.held(pool, dtype), pairs_of(pool, dtype)
    out, lse, weight = ref
    hkv, ps, d = held.shape[3:]
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for i, n in enumerate(lengths):
        if n == 0:
            continue
        j = np.arange(n)
        if window:
            j = j[(n - 1 - j < window) | (j < sinks)]
        page = torch.as_tensor(np.asarray(table[i])[j // ps], dtype=torch.long)
        at = lambda x, kv: x[page, layer, kv, :, j % ps]    # noqa: E731  [n, hkv, d]
        x = q[i].double().reshape(hkv, -1, d)
        p = torch.softmax(torch.einsum("hgd,khd->hgk", x, at(held, 0)) * scale, -1)
        delta = (2 * d + 16) * 2.0 ** -24 * scale * torch.einsum("hgd,khd->hgk", x.abs(), 47 * at(step, 0) + at(low, 0).abs()).amax(-1)
        mass = torch.einsum("hgk,khd->hgd", p, 31 * at(step, 1))
        more = mass + torch.einsum("hgk,khd->hgd", p, at(low, 1).abs())
        off = torch.expm1(2 * delta)[..., None] * weight[i].reshape(mass.shape) + 2.0 ** -16 * (mass + more)
        tol[i] = off.reshape(-1, d) + torch.finfo(dtype).eps / 2 * out[i].abs()
        tol_lse[i] = delta.reshape(-1)
    smallest = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return 1.1 * tol + smallest, 1.1 * tol_lse + 2.0 ** -18 * (1 + lse.abs().nan_to_num(0, 0, 0))


def check(cache, pool, table, lengths, q, new, dtype):
    """attend against the 64-bit form of what is held."""
    held, scale = O.held(pool, dtype), cache.head_dim ** -0.5
    if new is None:
        ref = O.attention(held, table, lengths, 1, q, list(range(len(lengths) + 1)))
        got, lse = cache.attend(1, q.cuda(), return_lse=True)
        tol, tol_lse = step_tolerance(pool, table, lengths, 1, q, ref, dtype, scale)
        got, lse = got.cpu().double(), lse.cpu().double()
        assert torch.isfinite(got).all() and not torch.isnan(lse).any()
        err = (got - ref[0]).abs()
        assert (err <= tol).all(), (err / tol).max().item()
        fin = torch.isfinite(ref[1])
        assert torch.equal(torch.isfinite(lse), fin) and ((lse - ref[1]).abs()[fin] <= tol_lse[fin]).all()
        return
    offsets = [0] + np.cumsum(new).tolist()
    ref = O.attention(values_rounded(held, dtype), table, lengths, 1, q, offsets)
    got, lse = cache.attend(1, q.cuda(), offsets=i32(offsets), return_lse=True)
    agree(got, lse, ref, dtype, max(lengths))


LENGTHS = [12, 40, 1, 0, 150]
NEW = [3, 20, 1, 0, 40]
WAYS = [(None, None), (None, 4096), (NEW, None)]        # clusters, the line of tiles, a prompt


def filled(pc, d, hkv, dtype, table_pages):  # noqa: F811
    cache, pool, table = make4(pc, LENGTHS, hkv, d, 16, dtype=dtype, seed=3, table_pages=table_pages)
    return cache, pool, table


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,table_pages", WAYS, ids=["clusters", "line", "prompt"])
@pytest.mark.parametrize("d,group", [(64, 1), (64, 2), (64, 4), (64, 8), (64, 16), (128, 1), (128, 4), (128, 8), (128, 16)])
def test_large_values(pc, dtype, new, table_pages, d, group):  # noqa: F811
    """One value of a slot is as large as single precision's sums allow; queries are small, so that its weight is near the others'."""
    cache, pool, table = filled(pc, d, 2, dtype, table_pages)
    for i, token in ((0, 5), (1, 17), (4, 100), (2, 0)):
        put(pool, table, i, token, 1, large(2, d, dtype, i))
    cache.pool.copy_(pool)
    q = (0.1 * queries(sum(new) if new else len(LENGTHS), 2 * group, d, torch.float32, 4)).to(dtype)
    check(cache, pool, table, LENGTHS, q, new, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,table_pages", WAYS, ids=["clusters", "line", "prompt"])
@pytest.mark.parametrize("d,group", [(64, 1), (64, 2), (64, 4), (64, 8), (64, 16), (128, 1), (128, 4), (128, 8), (128, 16)])
def test_large_keys(pc, dtype, new, table_pages, d, group):  # noqa: F811
    """Queries so small that scores of the largest keys are ordinary ones."""
    cache, pool, table = filled(pc, d, 2, dtype, table_pages)
    for i, token in ((0, 2), (0, 5), (1, 17), (1, 18), (4, 0), (4, 100), (4, 129), (2, 0)):
        put(pool, table, i, token, 0, large(2, d, dtype, 7 * i + token))
    cache.pool.copy_(pool)
    q = (queries(sum(new) if new else len(LENGTHS), 2 * group, d, torch.float32, 4) / LARGE[dtype]).to(dtype)
    check(cache, pool, table, LENGTHS, q, new, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,table_pages", WAYS, ids=["clusters", "line", "prompt"])
@pytest.mark.parametrize("d,group", [(64, 1), (64, 2), (64, 4), (128, 8), (128, 16)])
def test_awkward_groups(pc, dtype, new, table_pages, d, group):  # noqa: F811
    cache, pool, table = filled(pc, d, 2, dtype, table_pages)
    x = awkward(2, d, dtype, 5)
    for n in range(4):
        for i, token in ((0, 2), (1, 17), (4, 100)):
            put(pool, table, i, token + 2 * n, 0, x[n])
            put(pool, table, i, token + 2 * n + 1, 1, x[n])
    put(pool, table, 2, 0, 1, x[1])
    cache.pool.copy_(pool)
    check(cache, pool, table, LENGTHS, queries(sum(new) if new else len(LENGTHS), 2 * group, d, dtype, 4), new, dtype)


@pytest.mark.parametrize("table_pages", [None, 4096], ids=["clusters", "line"])
@pytest.mark.parametrize("d,group", [(64, 1), (64, 2), (64, 4), (64, 8), (64, 16), (128, 1), (128, 4), (128, 8), (128, 16)])
def test_small_values_of_wide_groups(pc, table_pages, d, group):  # noqa: F811
    """Dims that are 0 beside -8 and 7: their error goes by the steps, u |out| + 2^-16 sum_j p_j 31 step_j as the header
    says (in f16, whose u is small), scores and f32 sums apart; of 2^-16 sum_j p_j |v_j| nothing would be left for them."""
    dtype, scale = torch.float16, d ** -0.5
    cache, pool, table = filled(pc, d, 2, dtype, table_pages)
    g = torch.Generator().manual_seed(2)
    for i, n in enumerate(LENGTHS):
        for token in range(n):
            x = torch.randint(-8, 8, (2, d), generator=g).to(dtype)
            x[:, ::8], x[:, 1::64], x[:, 2::64] = 0, -8, 7
            put(pool, table, i, token, 1, x)
    cache.pool.copy_(pool)
    q = (0.05 * queries(len(LENGTHS), 2 * group, d, torch.float32, 4)).to(dtype)
    held, (step, low) = O.held(pool, dtype), pairs_of(pool, dtype)
    assert (held[table[1, 0], 1, 1, 0, 0, ::8] == 0).all() and step[table[1, 0], 1, 1, 0, 0, 0] == 1
    out, _, weight = O.attention(held, table, LENGTHS, 1, q, list(range(len(LENGTHS) + 1)))
    got = cache.attend(1, q.cuda()).cpu().double()
    for i, n in enumerate(LENGTHS):
        if n == 0:
            continue
        j = np.arange(n)
        page = torch.as_tensor(np.asarray(table[i])[j // 16], dtype=torch.long)
        size = 47 * step[page, 1, 0, :, j % 16] + low[page, 1, 0, :, j % 16].abs()
        delta = (2 * d + 16) * 2.0 ** -24 * scale * torch.einsum("hgd,khd->hgk", q[i].double().reshape(2, -1, d).abs(), size).amax()
        sums = 2.0 ** -20 * 39                          # exponentials and sums in f32, of p (31 step + |low|)
        tol = 1.1 * (2.0 ** -16 * 31 + 2.0 ** -11 * out[i].abs()) + torch.expm1(2 * delta) * weight[i] + sums
        assert ((got[i] - out[i]).abs() <= tol).all()
