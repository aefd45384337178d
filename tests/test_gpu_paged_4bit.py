"""The paged cache in 4 bits on the GPU against its plain restatement
(oracle/paged_cache.py): what store writes exact to the bit, what load gives
within its one rounding, attention within the rounding of its operands.

Tolerance of a single token's attention, derived.  Scores are sums of products
of 16-bit numbers in f32, step (q.(16 + c)) + off sum q: with S = scale sum_d
|q_d| (31 step + |off|) at most 2 D + 16 roundings of 2^-24 each, so a score is off by
delta <= (2 D + 16) 2^-24 S, and a weighted mean by (e^{2 delta} - 1) sum p |v|.  The
weights p step are two bf16 numbers, off by 2^-16 p step (16 + c) <= 2^-16 p 31 step.
The result is rounded once: u |o|, u = finfo.eps / 2.  Sums in f32 and the
exponential's own error (2^-22 each) are allowed for by n 2^-22 of the weight for n
keys, n at most 64 (parts are summed pairwise by warps and joined), and a tenth.

Prompts take keys as they are held, too, and round the held values once to the
cache's type: with values rounded so, they are held to the tolerance of a 16-bit
cache."""
import math

import numpy as np
import pytest
import torch

from oracle import paged_cache as O
from test_gpu_paged_cache import agree, i32, pc, queries  # noqa: F401
from test_gpu_paged_waits import call

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def token_bytes(d):
    return d // 2 + d // 16


def values(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    d = shape[-1]
    size, off = torch.exp(0.5 * torch.randn(d, generator=g)), 0.5 * torch.randn(d, generator=g)
    return (torch.randn(shape, generator=g) * size + off).to(dtype)


def make4(pc, lengths, hkv=2, d=64, ps=16, layers=2, dtype=torch.bfloat16, seed=0, table_pages=None, spare=3):
    """A cache with slots of the given lengths on shuffled pages; whatever is not a stored token is 0xff: codes of 15
    and pairs that are NaN."""
    need = [-(-n // ps) for n in lengths]
    pages = sum(need) + spare
    table_pages = table_pages or max(max(need), 1) + 1
    pool = torch.full((pages, layers, 2, hkv, ps, token_bytes(d)), 0xff, dtype=torch.uint8)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), table_pages), -1, dtype=torch.int32)
    for i, n in enumerate(lengths):
        mine, order = order[:need[i]], order[need[i]:]
        if n:
            table[i, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
        for j, p in enumerate(mine):
            x = values((min(ps, n - j * ps), layers, 2, hkv, d), dtype, seed + 97 * i + j)
            for t in range(x.shape[0]):
                O.put4(pool[p].view(layers * 2 * hkv, ps, -1), t, x[t].reshape(-1, d))
    refs = torch.zeros(pages, dtype=torch.int32)
    for p in table[table >= 0].tolist():
        refs[p] += 1
    cache = pc.PagedCache(pool.cuda(), table.cuda(), i32(lengths), refs.cuda(), dtype=dtype)
    return cache, pool, table


def values_rounded(held, dtype):
    held = held.clone()
    held[:, :, 1] = held[:, :, 1].to(dtype).double()
    return held


def spoil(cache, table, i, j, value=0xff):
    """Token j of slot i gets codes and pairs that are NaN."""
    ps, d = cache.page_size, cache.head_dim
    flat = cache.pool[table[i, j // ps]].view(cache.layers, 2, cache.kv_heads, -1)
    t = j % ps
    flat[..., t * d // 2:(t + 1) * d // 2] = value
    flat[..., ps * d // 2 + t * d // 16:ps * d // 2 + (t + 1) * d // 16] = value


def step_tolerance(pool, table, lengths, layer, q, ref, dtype, scale):
    """Of each output (see above): the slots' largest 31 step + |off| stand for every key."""
    out, _, weight = ref
    ps, d = pool.shape[4], pool.shape[5] * 16 // 9
    flat = pool.reshape(*pool.shape[:4], -1)
    pairs = flat[..., ps * d // 2:].contiguous().view(dtype).double().reshape(*pool.shape[:4], ps, d // 64, 2)
    tol = torch.zeros_like(out)
    heads, hkv = q.shape[1], pool.shape[3]
    for i, n in enumerate(lengths):
        if n == 0:
            continue
        j = np.arange(n)
        page = torch.as_tensor(np.asarray(table[i])[j // ps], dtype=torch.long)
        big = []
        for kv in range(2):
            p = pairs[page, layer, kv, :, j % ps]                         # [n, hkv, groups, 2]
            step, off = p[..., 0], p[..., 1] - 16 * p[..., 0]
            big.append(((31 * step + off.abs()).nan_to_num(0).amax(0), (31 * step).nan_to_num(0).amax(0)))
        spread = lambda x: x.repeat_interleave(heads // hkv, 0).repeat_interleave(64, -1)  # noqa: E731  [heads, d]
        size = scale * (q[i].double().abs() * spread(big[0][0])).sum(-1, keepdim=True)
        delta = (2 * d + 16) * 2.0 ** -24 * size
        mass = spread(big[1][0])
        tol[i] = (torch.expm1(2 * delta) * weight[i] + (2.0 ** -16 + 64 * 2.0 ** -22) * mass) + \
            torch.finfo(dtype).eps / 2 * out[i].abs()
    return 1.1 * tol + 1e-7


def check(pc, lengths, new=None, group=1, hkv=2, d=64, ps=16, dtype=torch.bfloat16, window=0, sinks=0, mask=None, seed=0,
          scale=None, table_pages=None):
    cache, pool, table = make4(pc, lengths, hkv, d, ps, dtype=dtype, seed=seed, table_pages=table_pages)
    n = len(lengths)
    offsets = list(range(n + 1)) if new is None else [0] + np.cumsum(new).tolist()
    q = queries(offsets[-1], hkv * group, d, dtype, seed + 1)
    key_mask = None
    if mask is not None:
        key_mask = mask(n, cache.table_pages * ps)
        for i in range(n):      # masked keys hold NaN: none of it may come through
            for j in range(lengths[i]):
                if not key_mask[i, j]:
                    spoil(cache, table, i, j)
    held = O.held(pool, dtype)
    if new is not None:
        held = values_rounded(held, dtype)
    ref = O.attention(held, table, lengths, 1, q, offsets, window, sinks, scale, key_mask)
    got, lse = cache.attend(1, q.cuda(), offsets=None if new is None else i32(offsets), window=window, sinks=sinks,
                            scale=scale, key_mask=None if key_mask is None else key_mask.cuda(), return_lse=True)
    torch.cuda.synchronize()
    if new is not None:
        agree(got, lse, ref, dtype, max(max(lengths), 1))
        return
    tol = step_tolerance(pool, table, lengths, 1, q, ref, dtype, d ** -0.5 if scale is None else scale)
    err = (got.cpu().double() - ref[0]).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), (err / tol).max().item()
    lse = lse.cpu().double()
    assert torch.equal(torch.isinf(lse), torch.isinf(ref[1])) and not torch.isnan(lse).any()
    fin = torch.isfinite(ref[1])
    if fin.any():
        assert (lse[fin] - ref[1][fin]).abs().max().item() <= 1e-3     # delta of these sizes: D = 128, S < 60


# ---------------------------------------------------------------------------
# rows in and out
# ---------------------------------------------------------------------------

def awkward(rows, heads, d, dtype, seed):
    """Rows whose groups are constant, tiny, as large as the type goes, of two values, or not finite."""
    x = values((rows, heads, d), dtype, seed)
    top = torch.finfo(dtype).max
    g = x.view(rows, heads, -1, 64)
    g[0, 0, 0] = 0.75                                   # no spread
    g[1 % rows, 0, 0] = 0
    g[2 % rows, 0, 0] = x.view(-1)[:64] * 1e-7          # subnormal steps in f16
    g[3 % rows, 0, 0, ::2], g[3 % rows, 0, 0, 1::2] = top / 4, -top / 4
    g[4 % rows, 0, 0, 5] = float("inf")
    g[5 % rows, 0, 0, 7] = float("nan")
    g[6 % rows, 0, 0] = 100 + torch.arange(64, dtype=torch.float64).to(dtype) / 256
    g[7 % rows, 0, 0] = torch.where(torch.arange(64) % 2 == 0, torch.tensor(-0.0), torch.tensor(0.0)).to(dtype)
    if dtype is torch.bfloat16:
        g[8 % rows, 0, 0, ::2], g[8 % rows, 0, 0, 1::2] = top, -top            # a spread past single precision
        g[9 % rows, 0, 0] = (torch.arange(64) % 5).to(dtype) * 2.0 ** -130      # a step below 2^-126
    return x


def same_pool(cache, data):
    """Bit for bit, but that a pair's NaN is any NaN and a zero of either sign."""
    ps, d = cache.page_size, cache.head_dim
    a, b = (t.reshape(*t.shape[:4], -1) for t in (cache.pool.cpu(), data))
    pa, pb = (t[..., ps * d // 2:].contiguous().view(cache.dtype) for t in (a, b))
    codes = (a[..., :ps * d // 2] != b[..., :ps * d // 2]).nonzero()
    pairs = (~((pa == pb) | (pa.isnan() & pb.isnan()))).nonzero()
    assert not len(codes), (len(codes), codes[:4].tolist())
    assert not len(pairs), (len(pairs), pairs[:4].tolist(), [(pa[tuple(i)].item(), pb[tuple(i)].item()) for i in pairs[:4]])
    return True


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,ps,hkv,layers", [(64, 16, 12, 2), (128, 64, 3, 1), (64, 32, 1, 3), (128, 16, 8, 2)])
def test_store_to_the_bit_and_load(pc, dtype, d, ps, hkv, layers):
    lengths, new = [0, 1, ps, ps + 1, 3 * ps + 5], [0, 1, ps - 2, 3, 2 * ps + 7]
    cache, pool, table = make4(pc, lengths, hkv, d, ps, layers, dtype)
    sim = O.ListCache(pool.clone(), len(lengths), cache.table_pages, dtype)
    sim.rows, sim.lengths = [[p for p in r if p >= 0] for r in table.tolist()], list(lengths)
    offsets = [0] + np.cumsum(new).tolist()
    wide = awkward(offsets[-1] * layers, 2 * hkv, d, dtype, 5).view(layers, offsets[-1], 2 * hkv, d)
    k, v = wide[:, :, :hkv], wide[:, :, hkv:]           # views: strides past the heads
    sim.store(k, v, offsets, range(layers))
    on = wide.cuda()
    cache.store(on[:, :, :hkv], on[:, :, hkv:], offsets=i32(offsets))
    torch.cuda.synchronize()
    assert same_pool(cache, sim.data)
    # and what it stands for: every row, each layer by itself, and into rows of the caller's
    got_k, got_v = cache.load(offsets[-1], offsets=i32(offsets))
    one_k, one_v = cache.load(offsets[-1], layer=layers - 1, offsets=i32(offsets))
    out = torch.zeros(offsets[-1], 2 * hkv, d, dtype=dtype, device="cuda")
    cache.load(offsets[-1], layer=0, offsets=i32(offsets), k=out[:, :hkv], v=out[:, hkv:])
    torch.cuda.synchronize()
    held = O.held(sim.data, dtype).to(dtype)
    for i, n in enumerate(lengths):
        for r in range(offsets[i], offsets[i + 1]):
            t = n - offsets[i + 1] + r
            for kv, got in enumerate((got_k, got_v)):
                want = held[table[i, t // ps], :, kv, :, t % ps]
                assert torch.equal(got[:, r].cpu().nan_to_num(7), want.nan_to_num(7))
    assert torch.equal(one_k.nan_to_num(7), got_k[-1].nan_to_num(7)) and torch.equal(one_v.nan_to_num(7), got_v[-1].nan_to_num(7))
    assert torch.equal(out.nan_to_num(7), torch.cat([got_k[0], got_v[0]], 1).nan_to_num(7))


def test_values_are_near_what_was_stored(pc):
    """A held value is off by half a step, and by what rounding the step to its type adds: 15 of them, 2^-8 each."""
    for dtype in TYPES:
        cache = pc.PagedCache.allocate(8, 2, 64, 1, 4, 128, 16, dtype, bits=4)
        cache.extend(i32([40, 9]))
        x = values((49, 4, 128), dtype, 3).cuda()
        cache.store(x, -x, layer=0, offsets=i32([0, 40, 49]))
        k, v = cache.load(49, layer=0, offsets=i32([0, 40, 49]))
        g = x.double().view(49, 4, 2, 64)
        step = (g.amax(-1) - g.amin(-1))[..., None] / 15
        u = torch.finfo(dtype).eps / 2
        tol = step * (0.5 + 15 * u) * (1 + 2 * u) + u * (g.abs() + step)
        for got, want in ((k, g), (v, -g)):
            assert ((got.double().view(49, 4, 2, 64) - want).abs() <= tol).all()


@pytest.mark.parametrize("bits", [4, 16])
def test_load_of_rows_that_are_not_there(pc, bits):
    cache = pc.PagedCache.allocate(8, 4, 64, 2, 2, 64, 16, bits=bits)
    cache.extend(i32([20, 0, 3, 1]))
    x = values((24, 2, 64), torch.bfloat16, 1).cuda()
    for layer in range(2):
        cache.store(x, x, layer=layer, offsets=i32([0, 20, 20, 23, 24]))
    # slot 2 is asked for more tokens than it has, and rows before the first and after the last slot
    k, v = cache.load(40, layer=1, offsets=i32([2, 22, 22, 30, 31]))
    assert (k[:2] == 0).all() and (k[22:30] == 0).all() and (k[31:] == 0).all() and (v[31:] == 0).all()
    ref, _ = cache.load(24, layer=1, offsets=i32([0, 20, 20, 23, 24]))
    assert torch.equal(k[2:22], ref[:20]) and torch.equal(k[30], ref[23])
    # the decode form: a row for each slot
    k, v = cache.load(4, layer=1)
    assert torch.equal(k[0], ref[19]) and (k[1] == 0).all() and torch.equal(v[2], ref[22]) and torch.equal(k[3], ref[23])
    if bits == 16:
        assert torch.equal(ref, x)
    cache.page_table[0, 1] = -1                         # a page that is gone
    k, _ = cache.load(4, layer=1)
    assert (k[0] == 0).all()


@pytest.mark.parametrize("ps,d,seed", [(16, 64, 0), (64, 128, 1), (128, 64, 2), (32, 128, 3)])
def test_upkeep_random_sequence(pc, ps, d, seed):
    """extend, store, fork (shallow and deep), free and compact on a pool near its limit: tables and bytes as restated."""
    rng = np.random.default_rng(seed)
    slots, pages, dtype = 6, 24, TYPES[seed % 2]
    cache = pc.PagedCache.allocate(pages, slots, 6 * ps, 2, 3, d, ps, dtype, bits=4)
    cache.pool.fill_(17)
    sim = O.ListCache(cache.pool.cpu().clone(), slots, cache.table_pages, dtype)
    for step in range(15):
        counts = np.where(rng.random(slots) < 0.7, rng.integers(0, 2 * ps, slots), 0).tolist()
        sim.extend(counts)
        cache.extend(i32(counts))
        offsets = [0] + np.cumsum(counts).tolist()
        x = values((2, 2, offsets[-1], 3, d), dtype, seed * 100 + step)
        sim.store(x[0], x[1], offsets, range(2))
        cache.store(x[0].cuda(), x[1].cuda(), offsets=i32(offsets))
        if step % 3 == 1:
            source = np.where(rng.random(slots) < 0.5, rng.integers(-1, slots, slots), -1).tolist()
            sim.fork(source, deep=step % 2 == 0)
            cache.fork(i32(source), deep=step % 2 == 0)
        if step % 3 == 2:
            mask = rng.random(slots) < 0.6
            sim.free(mask.tolist())
            cache.free(torch.tensor(mask, device="cuda"))
            sim.compact()
            cache.compact()
        torch.cuda.synchronize()
        assert cache.page_table.cpu().tolist() == sim.table() and cache.lengths.cpu().tolist() == sim.lengths
        assert cache.refs.cpu().tolist() == sim.refs() and cache.status.cpu().tolist() == sim.status
        assert same_pool(cache, sim.data)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 47, 64, 65, 100, 129, 200]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,ps", [(64, 16), (64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("wide", [False, True])
def test_step_lengths(pc, dtype, d, ps, wide):
    """wide: a table so wide that the line of tiles is taken; else a cluster for each slot and head."""
    check(pc, LENGTHS, d=d, ps=ps, dtype=dtype, seed=d + ps, table_pages=65536 // ps if wide else None)


@pytest.mark.parametrize("group", [2, 3, 7, 8, 9, 16, 20])
@pytest.mark.parametrize("d,wide", [(64, False), (64, True), (128, False), (128, True)])
def test_step_groups(pc, group, d, wide):
    check(pc, [0, 5, 130, 77], group=group, d=d, hkv=1 + group % 3, dtype=TYPES[group % 2], seed=group,
          table_pages=4096 if wide else None)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 3), (40, 16), (64, 33), (1000, 5), (1, 200)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("wide", [False, True])
def test_step_windows(pc, window, sinks, d, wide):
    check(pc, [0, 1, 16, 63, 150, 211], d=d, group=2, window=window, sinks=sinks, seed=window, dtype=TYPES[window % 2],
          table_pages=4096 if wide and window > 900 else None)


def some_keys(n, keys):
    g = torch.Generator().manual_seed(9)
    m = torch.rand(n, keys, generator=g) < 0.7
    m[1] = False                                        # a row that sees nothing
    if n > 2:
        m[2, :40] = False                               # a padded beginning
    return m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,wide", [(64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("window", [0, 50])
def test_step_masks(pc, dtype, d, wide, window):
    check(pc, [70, 33, 129, 16, 0, 1], d=d, mask=some_keys, window=window, sinks=8 if window else 0, dtype=dtype, hkv=3,
          group=3, table_pages=4096 if wide else None)


@pytest.mark.parametrize("d,group,window,sinks", [(64, 1, 17, 3), (64, 2, 40, 33), (64, 8, 100, 0), (128, 2, 64, 16), (128, 4, 1, 20),
                                                  (128, 1, 90, 5)])
def test_step_windows_of_many_slots(pc, d, group, window, sinks):
    """More slots and heads than there are clusters: the line of tiles, whose shares begin and end inside windows."""
    lengths = np.random.default_rng(window).integers(0, 260, 330).tolist()
    check(pc, lengths, d=d, group=group, window=window, sinks=sinks, seed=window, dtype=TYPES[window % 2])


def test_step_many_slots_and_scale(pc):
    rng = np.random.default_rng(3)
    check(pc, rng.integers(0, 90, 300).tolist(), hkv=1, scale=0.37, table_pages=600)
    check(pc, [1000, 3, 700], hkv=2, d=128, group=4, ps=64, dtype=torch.float16, scale=1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,ps,group", [(64, 16, 1), (64, 128, 4), (128, 64, 2), (128, 16, 8)])
def test_prompt_lengths(pc, dtype, d, ps, group):
    check(pc, [0, 1, 17, 64, 130, 200, 300], new=[0, 1, 17, 10, 130, 3, 290], d=d, ps=ps, group=group, dtype=dtype,
          seed=d + ps)


@pytest.mark.parametrize("window,sinks", [(1, 0), (30, 0), (100, 17), (200, 130)])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_windows(pc, window, sinks, d):
    check(pc, [40, 129, 400], new=[40, 2, 260], d=d, window=window, sinks=sinks, group=2, dtype=TYPES[window % 2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,window", [(64, 0), (64, 60), (128, 0)])
def test_prompt_masks(pc, dtype, d, window):
    check(pc, [70, 33, 200, 16], new=[70, 20, 150, 1], d=d, mask=some_keys, window=window, sinks=9 if window else 0,
          dtype=dtype, group=3)


def test_prompt_more_slots_than_ctas(pc):
    rng = np.random.default_rng(5)
    lengths = rng.integers(1, 60, 200)
    check(pc, lengths.tolist(), new=[int(rng.integers(0, n + 1)) for n in lengths], hkv=2, group=2)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_long_line(pc, dtype):
    """Units cut between CTAs, hundreds of rounds of the ring."""
    check(pc, [5000], new=[3], hkv=2, group=4, d=128, ps=64, dtype=dtype)
    check(pc, [2500, 700], new=[400, 700], hkv=1, group=1, d=64, ps=32, dtype=dtype)


@pytest.mark.parametrize("d,group,known", [(64, 1, False), (128, 4, False), (64, 2, True)])
def test_shared_prefix(pc, d, group, known):
    """Members forked from a voice: the prefix pass over the 4-bit pool, and each slot's own tokens."""
    dtype, ps, hkv, prefix = torch.bfloat16, 16, 2, 160
    cache = pc.PagedCache.allocate(200, 9, 320, 2, hkv, d, ps, dtype, bits=4)
    counts = [prefix + 5] + [0] * 8
    cache.extend(i32(counts))
    x = values((2, 2, prefix + 5, hkv, d), dtype, 2).cuda()
    offsets = i32([0] + [prefix + 5] * 9)
    cache.store(x[0], x[1], offsets=offsets)
    cache.fork(i32([-1, 0, 0, 0, 0, 0, 0, -1, 0]))
    own = [0, 3, 1, 20, 40, 17, 0, 30, 2]
    cache.extend(i32(own))
    y = values((2, 2, sum(own), hkv, d), dtype, 3).cuda()
    cache.store(y[0], y[1], offsets=i32([0] + np.cumsum(own).tolist()))
    assert (cache.status == 0).all()
    groups = pc.PrefixGroups(cache, [(0, prefix + 5, [0, 1, 2, 3, 4, 5, 6, 8])], q_heads=hkv * group)
    if not known:
        groups._c.shared_tokens = 0                      # not known: the pass is made however small it is
    q = queries(9, hkv * group, d, dtype, 4)
    got, lse = cache.attend_shared(1, q.cuda(), groups, return_lse=True)
    alone, _ = cache.attend(1, q.cuda(), return_lse=True)
    torch.cuda.synchronize()
    held = O.held(cache.pool.cpu(), dtype)
    lengths, table = cache.lengths.tolist(), cache.page_table.cpu()
    ref = O.attention(values_rounded(held, dtype), table, lengths, 1, q, list(range(10)))
    plain = O.attention(held, table, lengths, 1, q, list(range(10)))
    # a prefix's values are rounded once, the others not at all: between the two references, which differ by that rounding
    out, ref_lse, weight = ref
    tol = 1.1 * 2.0 ** -8 * (out.abs() + weight) + (plain[0] - out).abs() * 2 + 1e-4
    assert ((got.cpu().double() - out).abs() <= tol).all()
    fin = torch.isfinite(ref_lse)
    assert ((lse.cpu().double() - ref_lse).abs()[fin] <= 1e-3 + 2 * (plain[1] - ref_lse).abs()[fin]).all()
    assert (alone.cpu().double() - plain[0]).abs().max() < 0.05


@pytest.mark.parametrize("d,ps", [(64, 16), (128, 128)])
def test_places_past_32_bits(pc, d, ps):
    """A pool of more than 4 GB whose last pages are in use: what a small pool gives, bit for bit."""
    hkv, group, dtype, lengths = 8, 2, torch.bfloat16, [300, 1, 77]
    block = 2 * hkv * ps * (d // 2 + d // 16)
    many = (5 << 30) // block
    x = values((2, sum(lengths), hkv, d), dtype, 1).cuda()
    q, rows = queries(3, hkv * group, d, dtype, 2).cuda(), queries(sum(lengths), hkv * group, d, dtype, 3).cuda()
    offsets = i32([0] + np.cumsum(lengths).tolist())
    got = []
    for pages in (64, many):
        cache = pc.PagedCache.allocate(pages, 3, 320, 1, hkv, d, ps, dtype, bits=4)
        cache.refs[:pages - 64] = 1                      # all but the last are taken
        cache.extend(i32(lengths))
        cache.store(x[0], x[1], layer=0, offsets=offsets)
        first = cache.page_table[0, 0].item()
        assert first == pages - 64
        got.append([*cache.load(sum(lengths), layer=0, offsets=offsets), cache.attend(0, q), cache.attend(0, q, window=40, sinks=3),
                    cache.attend(0, rows, offsets=offsets), cache.status])
        torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_voice_sessions_in_4_bits(pc):
    """The example on a 4-bit cache: prefill, forks, shared-prefix steps, sessions ended, compaction, new ones; no call is
    refused, and a prefix stays to the bit what it was when it was stored."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    from voice_sessions import REFERENCE_PREFIX, WIDTH, VoiceServer
    server = VoiceServer(6, REFERENCE_PREFIX + 32, layers=2, window=24, bits=4)
    g = torch.Generator(device="cuda").manual_seed(3)
    draw = lambda *s: torch.randn(*s, WIDTH, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    server.prefill(draw(4, REFERENCE_PREFIX))
    cache, n = server.cache, REFERENCE_PREFIX
    offsets = i32([n * min(s, 4) for s in range(cache.slots + 1)])
    before = cache.load(4 * n, offsets=offsets)
    server.start(range(6), [s % 2 for s in range(6)])
    x = draw(cache.slots)
    for step in range(10):
        if step == 5:
            server.end([0, 2, 4])
            server.start([0, 4], [1, 1])
        x = server.step(x)
    torch.cuda.synchronize()
    assert cache.bits == 4 and (cache.status == 0).all()
    live = torch.tensor([s for s in range(4, cache.slots) if server.open[(s - 4) // 2]], device="cuda")
    assert torch.isfinite(x[live].float()).all()
    after = cache.load(4 * n, offsets=offsets)
    assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1])


# ---------------------------------------------------------------------------
# bounded waits (the converters' among them)
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128])
def test_prompt_that_gives_up(pc, d):
    """No key tile is ever converted: all slots with rows are marked, no other, and the next call is right."""
    new = [1, 0, 300, 40, 0, 129, 7]
    lengths = [n + 100 * (i % 3) for i, n in enumerate(new)]
    cache, pool, table = make4(pc, lengths, 2, d)
    q = queries(sum(new), 4, d, torch.bfloat16)
    offsets = [0] + np.cumsum(new).tolist()
    call(cache, q.cuda(), 2_000_000, i32(offsets), starve=True)
    assert cache.status.tolist() == [4 if n else 0 for n in new]
    cache.status.zero_()
    got, lse = call(cache, q.cuda(), 200_000_000, i32(offsets))
    agree(got, lse, O.attention(values_rounded(O.held(pool, torch.bfloat16), torch.bfloat16), table, lengths, 0, q, offsets),
          torch.bfloat16, max(lengths))
    assert (cache.status == 0).all()


def test_prefix_pass_that_gives_up(pc):
    """Its members are attended on their own: marked, and right."""
    cache = pc.PagedCache.allocate(60, 5, 320, 1, 2, 64, bits=4)
    cache.extend(i32([160, 0, 0, 0, 0]))
    x = values((160, 2, 64), torch.bfloat16, 2).cuda()
    cache.store(x, -x, layer=0, offsets=i32([0] + [160] * 5))
    cache.fork(i32([-1, 0, 0, 0, -1]))
    cache.extend(i32([0, 3, 1, 20, 0]))
    y = values((24, 2, 64), torch.bfloat16, 3).cuda()
    cache.store(y, y, layer=0, offsets=i32([0, 0, 3, 4, 24, 24]))
    plan = pc.PrefixGroups(cache, [(0, 160, [1, 2, 3])], q_heads=4)
    plan._c.shared_tokens = 0
    q = queries(5, 4, 64, torch.bfloat16).cuda()
    for starve, status in ((True, [0, 4, 4, 4, 0]), (False, [0] * 5)):
        cache.status.zero_()
        got, lse = call(cache, q, 2_000_000, groups=plan, starve=starve)
        assert cache.status.tolist() == status
        held = O.held(cache.pool.cpu(), torch.bfloat16)
        ref = O.attention(held, cache.page_table.cpu(), cache.lengths.tolist(), 0, q.cpu(), list(range(6)))
        # a prefix's values are rounded once more (2^-8 of the weight), as are its weights and the result
        assert ((got.cpu().double() - ref[0]).abs() <= 1.1 * 2.0 ** -8 * (ref[0].abs() + 2 * ref[2]) + 1e-4).all()
        if starve:      # single tokens: the result's rounding, scores and weights right to 2^-12 (see above)
            assert ((got.cpu().double() - ref[0]).abs() <= 2.0 ** -8 * ref[0].abs() + 2.0 ** -12 * (ref[2] + 1)).all()


def test_units_longer_than_the_limit(pc):
    """As in test_gpu_paged_waits.py: a unit lasts far longer than a bound that would not grow with the share."""
    d, hkv, ps, distinct, rows, length, dtype = 128, 4, 128, 64, 4096, 700_000, torch.bfloat16
    used = -(-length // ps)
    g = torch.Generator().manual_seed(4)
    pool = torch.randint(0, 256, (distinct, 1, 2, hkv, ps, token_bytes(d)), generator=g, dtype=torch.uint8)
    pairs = torch.stack([torch.full((2,), 0.25), torch.full((2,), -2.0)], -1).to(dtype)     # values -2 .. 1.75
    pool.view(distinct, 1, 2, hkv, -1)[..., ps * d // 2:] = pairs.view(torch.uint8).flatten().repeat(ps)
    table = torch.randint(0, distinct, (1, used), generator=g, dtype=torch.int32)
    cache = pc.PagedCache(pool.cuda(), table.cuda(), i32([length]), torch.ones(distinct, dtype=torch.int32, device="cuda"), dtype=dtype)
    q = queries(rows, hkv, d, dtype)
    out, lse = call(cache, q.cuda(), 2_000_000, i32([0, rows]))
    assert int(cache.status) == 0
    k, v = (x.permute(1, 0, 2, 3).reshape(hkv, distinct * ps, d) for x in O.held(pool, dtype)[:, 0].unbind(1))
    for r in (0, 255, 256, rows // 2 + 3, rows - 1):
        p = length - rows + r
        full = p // ps
        times = torch.bincount(table[0, :full].long(), minlength=distinct).double()[:, None].expand(distinct, ps).clone()
        times[table[0, full], :p % ps + 1] += 1
        s = torch.einsum("hd,hkd->hk", q[r].double(), k) * d ** -0.5 + times.reshape(-1).log()
        w = torch.softmax(s, -1)
        ref = tuple(torch.einsum("hk,hkd->hd", w, x)[None] for x in (v, v.abs()))
        agree(out[r:r + 1], lse[r:r + 1], (ref[0], torch.logsumexp(s, -1)[None], ref[1]), dtype, 1)
