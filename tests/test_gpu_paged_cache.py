"""The paged key/value cache and its attention on the GPU against their plain
restatement (oracle/paged_cache.py): upkeep exact to the bit, attention within
the rounding of its operands.

Tolerance of an attention output, derived: probabilities are rounded once to
the operands' type (relative error u each, so u * sum p|v| in the sum) and the
result once more (u |o|), u = 2^-8 for bf16 and 2^-11 for f16; probabilities
below f16's normal range lose at most 2^-25 each against a largest one of 1;
f32 sums add far less than 2^-11 of u, allowed for by a tenth.  A log-sum-exp
is off by at most the f32 dot product's error, d 2^-24 sum|q k| scale < 5e-4
for these inputs."""
import numpy as np
import pytest
import torch

from oracle import paged_cache as O

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def pc():
    from magpie_tts_rt_b200 import paged_cache
    return paged_cache


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(pc, lengths, hkv=2, d=64, ps=16, layers=2, dtype=torch.bfloat16, seed=0, table_pages=None, spare=3):
    """A cache with slots of the given lengths on shuffled pages; everything
    that is not a stored token is NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // ps) for n in lengths]
    pages = sum(need) + spare
    table_pages = table_pages or max(max(need), 1) + 1
    pool = torch.full((pages, layers, 2, hkv, ps, d), float("nan"), dtype=dtype)
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lengths), table_pages), -1, dtype=torch.int32)
    for i, n in enumerate(lengths):
        mine, order = order[:need[i]], order[need[i]:]
        for j, p in enumerate(mine):
            table[i, j] = p
            t = min(ps, n - j * ps)
            pool[p, :, :, :, :t] = torch.randn(layers, 2, hkv, t, d, generator=g).to(dtype)
    refs = torch.zeros(pages, dtype=torch.int32)
    for p in table[table >= 0].tolist():
        refs[p] += 1
    cache = pc.PagedCache(pool.cuda(), table.cuda(), i32(lengths), refs.cuda())
    return cache, pool, table


def queries(rows, heads, d, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (1.5 * torch.randn(rows, heads, d, generator=g)).to(dtype)


def agree(got, lse, ref, dtype, keys):
    out, ref_lse, weight = ref
    u = U[dtype]
    tol = 1.1 * u * (out.abs() + weight) + keys * 2.0 ** -25 * 4 + 1e-6
    err = (got.cpu().double() - out).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), (err / tol).max().item()
    if lse is not None:
        lse = lse.cpu().double()
        assert torch.equal(torch.isinf(lse), torch.isinf(ref_lse)) and not torch.isnan(lse).any()
        fin = torch.isfinite(ref_lse)
        assert (lse[fin] - ref_lse[fin]).abs().max().item() <= 5e-4 if fin.any() else True


def check_attend(pc, lengths, new=None, group=1, hkv=2, d=64, ps=16, dtype=torch.bfloat16, window=0, sinks=0,
                 mask=None, seed=0, scale=None):
    cache, pool, table = make(pc, lengths, hkv, d, ps, dtype=dtype, seed=seed)
    n = len(lengths)
    offsets = list(range(n + 1)) if new is None else [0] + np.cumsum(new).tolist()
    q = queries(offsets[-1], hkv * group, d, dtype, seed + 1)
    key_mask = None
    if mask is not None:
        key_mask = mask(n, cache.table_pages * ps)
        for i in range(n):      # masked keys hold NaN: none of it may come through
            for j in range(lengths[i]):
                if not key_mask[i, j]:
                    cache.pool[table[i, j // ps], :, :, :, j % ps] = float("nan")
    ref = O.attention(pool, table, lengths, 1, q, offsets, window, sinks, scale, key_mask)
    got, lse = cache.attend(1, q.cuda(), offsets=None if new is None else i32(offsets), window=window, sinks=sinks,
                            scale=scale, key_mask=None if key_mask is None else key_mask.cuda(), return_lse=True)
    torch.cuda.synchronize()
    agree(got, lse, ref, dtype, max(max(lengths), 1))
    return cache


# ---------------------------------------------------------------------------
# upkeep
# ---------------------------------------------------------------------------

def same(cache, sim):
    torch.cuda.synchronize()
    assert cache.page_table.cpu().tolist() == sim.table()
    assert cache.lengths.cpu().tolist() == sim.lengths
    assert cache.refs.cpu().tolist() == sim.refs()
    assert cache.status.cpu().tolist() == sim.status
    assert torch.equal(cache.pool.cpu().view(torch.int16), sim.data.view(torch.int16))


def paired(pc, pages, slots, max_tokens, layers=2, hkv=2, d=64, ps=16, dtype=torch.bfloat16, seed=0):
    cache = pc.PagedCache.allocate(pages, slots, max_tokens, layers, hkv, d, ps, dtype)
    cache.pool.copy_(torch.randn(cache.pool.shape, generator=torch.Generator().manual_seed(seed)).to(dtype))
    return cache, O.ListCache(cache.pool.cpu().clone(), slots, cache.table_pages)


def both_store(cache, sim, offsets, rng, layer=None):
    shape = (cache.layers if layer is None else 1, offsets[-1], cache.kv_heads, cache.head_dim)
    g = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
    k, v = (torch.randn(shape, generator=g).to(cache.dtype) for _ in range(2))
    sim.store(k, v, offsets, range(cache.layers) if layer is None else [layer])
    if layer is None:
        cache.store(k.cuda(), v.cuda(), offsets=i32(offsets))
    else:
        cache.store(k[0].cuda(), v[0].cuda(), layer=layer, offsets=i32(offsets))


@pytest.mark.parametrize("ps,slots,pages,seed", [(16, 7, 60, 0), (32, 33, 150, 1), (64, 12, 70, 2), (128, 5, 20, 3),
                                                 (16, 1500, 5000, 4)])
def test_upkeep_random_sequence(pc, ps, slots, pages, seed):
    """Random calls, the pool kept near its limit so that refusals occur."""
    rng = np.random.default_rng(seed)
    small = slots > 1000
    cache, sim = paired(pc, pages, slots, 6 * ps, layers=1 if small else 2, hkv=1 if small else 2, ps=ps, seed=seed)
    for step in range(12):
        kind = step % 6
        if kind in (0, 1):
            counts = np.where(rng.random(slots) < 0.7, rng.integers(0, 3 * ps, slots), 0)
            before = list(sim.lengths)
            sim.extend(counts.tolist())
            cache.extend(i32(counts.tolist()))
            grown = [b - a for a, b in zip(before, sim.lengths)]
            both_store(cache, sim, [0] + np.cumsum(grown).tolist(), rng, layer=None if kind else 0)
        elif kind == 2:
            source = np.where(rng.random(slots) < 0.5, rng.integers(0, slots, slots), -1)
            sim.fork(source.tolist())
            cache.fork(i32(source.tolist()))
        elif kind == 3:
            mask = rng.random(slots) < 0.4
            sim.free(mask)
            cache.free(torch.from_numpy(mask).cuda())
        elif kind == 4:
            source = np.where(rng.random(slots) < 0.2, rng.integers(0, slots, slots), -1)
            sim.fork(source.tolist(), deep=True)
            cache.fork(i32(source.tolist()), deep=True)
        else:
            live = sim.compact()
            cache.compact()
            assert int(cache.live) == live
        same(cache, sim)


def test_fork_permutes_all_slots_at_once(pc):
    cache, sim = paired(pc, 40, 4, 96)
    counts = [5, 16, 33, 0]
    sim.extend(counts)
    cache.extend(i32(counts))
    both_store(cache, sim, [0, 5, 21, 54, 54], np.random.default_rng(0))
    for source in ([1, 2, 0, 3], [3, -1, 0, 2], [2, 2, 2, 2]):
        sim.fork(source)
        cache.fork(i32(source))
        same(cache, sim)


def test_refusals_on_the_device(pc):
    cache, sim = paired(pc, 6, 5, 64)
    for counts in ([16, -1, 65, 40, 17], [0, 2**31 - 1, 64, 0, 0], [1, 1, 1, 1, 1]):
        sim.extend(counts)
        cache.extend(i32(counts))
        same(cache, sim)
    for source in ([1, 7, -2, -1, 3], [4, 4, 4, 4, -1]):
        sim.fork(source)
        cache.fork(i32(source))
        same(cache, sim)
    # the table's last page, and a pool without any free page
    sim.free([True] * 5)
    cache.free(torch.ones(5, dtype=torch.bool, device="cuda"))
    sim.extend([64, 32, 0, 0, 1])
    cache.extend(i32([64, 32, 0, 0, 1]))
    same(cache, sim)
    sim.compact()
    cache.compact()
    same(cache, sim)


def test_store_skips_what_does_not_fit(pc):
    cache, sim = paired(pc, 20, 4, 64)
    sim.extend([32, 16, 0, 3])
    cache.extend(i32([32, 16, 0, 3]))
    sim.fork([-1, -1, 0, -1])
    cache.fork(i32([-1, -1, 0, -1]))        # slots 0 and 2 share both pages
    rng = np.random.default_rng(1)
    both_store(cache, sim, [0, 2, 3, 3, 7], rng)   # slot 0: shared pages; slot 3: four rows for three tokens
    same(cache, sim)
    assert sim.status == [3, 0, 0, 1]


def test_store_of_last_tokens_and_strided_rows(pc):
    """A decode step's keys and values as they lie in a fused q|k|v row; closed slots are skipped."""
    cache, sim = paired(pc, 20, 4, 64, hkv=12)
    sim.extend([7, 0, 16, 33])
    cache.extend(i32([7, 0, 16, 33]))
    qkv = torch.randn(4, 3 * 12 * 64, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    k, v = qkv[:, 768:1536].view(4, 12, 64), qkv[:, 1536:].view(4, 12, 64)
    keep = [0, 2, 3]
    sim.store(k[None, keep], v[None, keep], [0, 1, 1, 2, 3], [1])
    dev = qkv.cuda()
    cache.store(dev[:, 768:1536].view(4, 12, 64), dev[:, 1536:].view(4, 12, 64), layer=1)
    same(cache, sim)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hkv,group,d,ps", [(12, 1, 64, 16), (2, 4, 128, 64), (1, 8, 64, 32), (3, 3, 128, 16),
                                            (1, 16, 128, 128), (2, 13, 64, 16), (1, 64, 64, 16)])
def test_step_heads(pc, dtype, hkv, group, d, ps):
    check_attend(pc, [1, 467, 16, 0, 65, 130, 33], hkv=hkv, group=group, d=d, ps=ps, dtype=dtype)


@pytest.mark.parametrize("lengths", [[0], [1], [0, 0, 0], [15], [16], [17], [2049], [5, 3000, 1, 0, 64, 700] * 8])
def test_step_lengths(pc, lengths):
    check_attend(pc, lengths)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 5), (100, 16), (64, 100), (7, 218), (2000, 4),
                                          (128, 4000), (2**31 - 1, 2**31 - 1)])
def test_step_window(pc, window, sinks):
    check_attend(pc, [1, 16, 17, 99, 467, 0, 1000], window=window, sinks=sinks, ps=32)


def holes(n, width):
    m = torch.rand(n, width, generator=torch.Generator().manual_seed(9)) < 0.6
    m[0] = False                # a row that sees nothing
    if n > 1:
        m[1, :100] = False      # a padded beginning
    if n > 2:
        m[2] = True
    if n > 3:
        m[3] = False
        m[3, 40] = True         # one key alone
    return m


@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 20)])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_step_masks_and_nan_behind_them(pc, window, sinks, d, dtype):
    check_attend(pc, [50, 130, 467, 41, 300], mask=holes, window=window, sinks=sinks, d=d, dtype=dtype, group=2)


# few slots: clusters of 64, 32, 16, 8 and 4 warps for each unit, up to and past their longest caches; many slots
FORMS = [([480, 33, 0, 1, 511], 2, 1, 64), ([1000, 33, 0, 1, 513], 2, 1, 64), ([8000, 130, 0, 1], 1, 1, 64),
         ([8192, 17], 1, 1, 64), ([300, 0, 1, 257], 2, 4, 128), ([3900, 33, 64, 1], 2, 4, 128), ([4097, 5], 1, 3, 128),
         ([2100, 33, 0, 1], 1, 16, 128), ([2500, 40], 2, 13, 64), ([700, 33, 0, 1, 64, 257, 16], 12, 1, 64),
         ([700, 33, 0, 1, 64, 257] * 4, 12, 1, 64), ([90, 33, 0, 1, 64, 257] * 8, 6, 2, 128),
         ([90, 33, 0, 1, 64, 240] * 16, 3, 1, 128), ([90, 33, 0, 1, 64, 500] * 16, 2, 16, 64),
         ([90, 33, 0, 1, 64, 300] * 16, 6, 1, 64), ([90, 33, 0, 1, 64, 700] * 16, 6, 1, 64)]


@pytest.mark.parametrize("lengths,hkv,group,d", FORMS)
@pytest.mark.parametrize("window,sinks,masked", [(0, 0, False), (40, 20, True), (0, 0, True)])
def test_step_forms(pc, lengths, hkv, group, d, window, sinks, masked):
    check_attend(pc, lengths, hkv=hkv, group=group, d=d, window=window, sinks=sinks, mask=holes if masked else None)


def test_step_forms_agree(pc):
    """Slot 0's row alone, among few slots and among many: the same up to the order of its sums, and each form's bits
    are the same in every call."""
    lengths = [467, 40] + [100 + i for i in range(30)]
    cache, pool, table = make(pc, lengths, hkv=12)
    q = queries(32, 12, 64, torch.bfloat16)
    ref = O.attention(pool, table, lengths, 1, q, list(range(33)))
    for rows in (1, 2, 32):
        got = [cache.attend(1, q[:rows].cuda()) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(got[0], g) for g in got)
        agree(got[0], None, tuple(r[:rows] for r in ref), torch.bfloat16, 467)


PROMPTS = [([1], [1]), ([218], [218]), ([128], [128]), ([129], [1]), ([300, 0, 17, 64], [257, 0, 17, 1]),
           ([1000, 33, 513], [3, 33, 400]), ([131] * 5, [131, 130, 129, 128, 127])]


@pytest.mark.parametrize("lengths,new", PROMPTS)
@pytest.mark.parametrize("dtype,hkv,group,d,ps", [(torch.bfloat16, 2, 1, 64, 16), (torch.float16, 2, 4, 128, 64),
                                                  (torch.bfloat16, 1, 3, 128, 32), (torch.float16, 1, 16, 64, 128)])
def test_prompt(pc, lengths, new, dtype, hkv, group, d, ps):
    check_attend(pc, lengths, new, hkv=hkv, group=group, d=d, ps=ps, dtype=dtype)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 3), (100, 16), (64, 218), (129, 1), (5000, 7), (2**31 - 1, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_window(pc, window, sinks, d):
    check_attend(pc, [700, 90, 5, 400], [600, 90, 2, 33], window=window, sinks=sinks, group=2, d=d)


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 30)])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_prompt_masks_and_nan_behind_them(pc, window, sinks, d, dtype):
    check_attend(pc, [200, 300, 467, 150, 77], [200, 250, 30, 150, 77], mask=holes, window=window, sinks=sinks, d=d,
                 dtype=dtype)


@pytest.mark.parametrize("window,sinks,masked", [(0, 0, False), (300, 16, True), (64, 0, False)])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_many_units_per_sm(pc, window, sinks, masked, d):
    """More units than SMs, many with an empty second tile: every SM walks several, whole and cut."""
    new = [1, 7, 130, 2, 255, 3, 40, 129, 5, 1, 300, 64] * 2
    lengths = [n + (i * 97) % 500 for i, n in enumerate(new)]
    cache = check_attend(pc, lengths, new, hkv=12, d=d, window=window, sinks=sinks, mask=holes if masked else None)
    assert (cache.status == 0).all()


@pytest.mark.parametrize("slots", [383, 384, 1100])
def test_prompt_many_slots(pc, slots):
    """Up to as many pairs of Q tiles as the kernel has threads, and more."""
    new = [(7 * i) % 23 for i in range(slots)]
    cache = check_attend(pc, [n + (5 * i) % 40 for i, n in enumerate(new)], new, hkv=1)
    assert (cache.status == 0).all()


def test_prompt_calls_back_to_back(pc):
    """Hundreds of calls of many units each: no wait inside the kernel gives up, the result never changes."""
    new = [1, 7, 130, 2, 255, 3, 40, 129, 5, 1, 300, 64] * 2
    lengths = [n + (i * 97) % 500 for i, n in enumerate(new)]
    cache, _, _ = make(pc, lengths, 12)
    q = queries(sum(new), 12, 64, torch.bfloat16).cuda()
    offsets = i32([0] + np.cumsum(new).tolist())
    out = torch.empty_like(q)
    first = cache.attend(0, q, offsets=offsets, window=300, sinks=16).clone()
    for _ in range(400):
        cache.attend(0, q, out=out, offsets=offsets, window=300, sinks=16)
    assert torch.equal(out, first) and (cache.status == 0).all()


def test_prompt_offsets_that_do_not_fit(pc):
    """More rows than tokens: those rows get 0 and -inf, the others are unharmed."""
    cache, pool, table = make(pc, [20, 40, 7])
    q = queries(60, 2, 64, torch.bfloat16)
    offsets = [0, 25, 55, 60]
    ref = O.attention(pool, table, [20, 40, 7], 0, q, offsets)
    got, lse = cache.attend(0, q.cuda(), offsets=i32(offsets), return_lse=True)
    agree(got, lse, ref, torch.bfloat16, 40)
    assert (got[:25] == 0).all() and torch.isinf(lse[:25]).all()


def test_step_is_the_prompts_last_row(pc):
    lengths = [100, 257, 31]
    cache, pool, table = make(pc, lengths, group := 2)
    q = queries(3, 4, 64, torch.bfloat16)
    ref = O.attention(pool, table, lengths, 0, q, [0, 1, 2, 3])
    for offsets in (None, i32([0, 1, 2, 3])):
        agree(*cache.attend(0, q.cuda(), offsets=offsets, return_lse=True), ref, torch.bfloat16, 257)


def test_strided_rows_scale_and_out(pc):
    lengths = [100, 257, 31]
    cache, pool, table = make(pc, lengths, 12)
    qkv = queries(3, 36, 64, torch.bfloat16)
    ref = O.attention(pool, table, lengths, 1, qkv[:, :12], [0, 1, 2, 3], scale=0.3)
    wide = torch.full((3, 20, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    got = cache.attend(1, qkv.cuda()[:, :12], out=wide[:, 4:16], scale=0.3)
    assert got.data_ptr() == wide[:, 4:16].data_ptr()
    agree(got, None, ref, torch.bfloat16, 257)
    assert (wide[:, :4] == 7).all() and (wide[:, 16:] == 7).all()


@pytest.mark.parametrize("group,d", [(1, 64), (3, 128), (4, 64)])
def test_prompt_strided_and_repeated_rows(pc, group, d):
    """Rows inside wider ones, and one row broadcast over all (a stride of 0)."""
    lengths, new = [300, 40], [290, 33]
    cache, pool, table = make(pc, lengths, 2, d)
    rows, heads = sum(new), 2 * group
    offsets = [0, 290, 323]
    wide = queries(rows, heads + 5, d, torch.bfloat16)
    ref = O.attention(pool, table, lengths, 0, wide[:, 2:2 + heads], offsets)
    got = cache.attend(0, wide.cuda()[:, 2:2 + heads], offsets=i32(offsets))
    agree(got, None, ref, torch.bfloat16, 300)
    one = queries(1, heads, d, torch.bfloat16)
    ref = O.attention(pool, table, lengths, 0, one.expand(rows, heads, d), offsets)
    got = cache.attend(0, one.cuda().expand(rows, heads, d), offsets=i32(offsets))
    agree(got, None, ref, torch.bfloat16, 300)


def test_large_scores_and_infinities(pc):
    """Scores far apart (one key takes all), scores of the same huge size, and -inf and +inf among the values'
    masked neighbours."""
    cache, pool, table = make(pc, [300, 64])
    q = (queries(2, 2, 64, torch.bfloat16).float() * 300).to(torch.bfloat16)
    ref = O.attention(pool, table, [300, 64], 0, q, [0, 1, 2])
    got = cache.attend(0, q.cuda())
    # here the dot product's f32 error (4e-4 * 300) moves probabilities by up to that share
    tol = (2.0 ** -8 + 0.12) * (ref[0].abs() + ref[2]) + 1e-5
    assert ((got.cpu().double() - ref[0]).abs() <= tol).all()
    mask = torch.ones(2, cache.table_pages * 16, dtype=torch.bool)
    mask[:, 10:20] = False
    q = queries(2, 2, 64, torch.bfloat16)
    ref = O.attention(pool, table, [300, 64], 0, q, [0, 1, 2], key_mask=mask)
    for i in range(2):
        for j in range(10, 20):
            cache.pool[table[i, j // 16], :, :, :, j % 16] = float("inf") * (1 if j % 2 else -1)
    got, lse = cache.attend(0, q.cuda(), key_mask=mask.cuda(), return_lse=True)
    agree(got, lse, ref, torch.bfloat16, 300)


@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16)])
def test_prompt_scores_that_climb(pc, d, dtype):
    """Scores that grow along the keys, slowly and in jumps far past the range of an f16 or an f32 exponential:
    the running maximum has to move again and again."""
    n = 700
    cache, pool, table = make(pc, [n], 2, d, dtype=dtype)
    rise = torch.cat([torch.linspace(0, 6, 400), torch.linspace(20, 60, 200), torch.full((100,), 200.0)])
    for j in range(n):
        pool[table[0, j // 16], :, 0, :, j % 16] = (pool[table[0, j // 16], :, 0, :, j % 16] * 0.1).to(dtype)
        pool[table[0, j // 16], :, 0, :, j % 16, 0] = rise[j].to(dtype)
    cache.pool.copy_(pool)
    q = (0.1 * queries(n, 2, d, dtype).float()).to(dtype)
    q[:, :, 0] = 2.0
    ref = O.attention(pool, table, [n], 0, q, [0, n], scale=0.7)
    got, lse = cache.attend(0, q.cuda(), offsets=i32([0, n]), scale=0.7, return_lse=True)
    agree(got, lse, ref, dtype, n)


def test_same_bits_every_time(pc):
    """Work is split and joined in an order that does not depend on timing."""
    cache, _, _ = make(pc, [3000, 17, 900, 2500], 2, seed=3)
    q = queries(4, 8, 64, torch.bfloat16).cuda()
    offsets = i32([0, 1, 2, 3, 4])
    first = [cache.attend(0, q).clone(), cache.attend(0, q, offsets=offsets).clone()]
    for _ in range(20):
        assert torch.equal(cache.attend(0, q), first[0])
        assert torch.equal(cache.attend(0, q, offsets=offsets), first[1])


def test_pool_past_32_bit_offsets(pc):
    """More than 2^32 elements: pages at the far end, copied and read."""
    ps, hkv, d = 128, 8, 128
    pages = (1 << 32) // (2 * hkv * ps * d) + 40
    cache = pc.PagedCache.allocate(pages, 2, 1024, 1, hkv, d, ps)
    assert cache.pool.numel() > 1 << 32
    cache.refs[:pages - 9] = 1             # as if held by others
    cache.extend(i32([130, 0]))
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(1, 130, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    cache.store(k.cuda(), v.cuda(), offsets=i32([0, 130, 130]))
    cache.fork(i32([-1, 0]))
    q = queries(2, 16, d, torch.bfloat16)
    got, lse = cache.attend(0, q.cuda(), return_lse=True)
    tail = pages - 9
    small = cache.pool[tail:].cpu()
    table = cache.page_table.cpu()
    assert table[0, :2].tolist() == [tail, tail + 1] and table[1, :2].tolist() == [tail, tail + 2]
    ref = O.attention(small, (table - tail).clamp(min=0), [130, 130], 0, q, [0, 1, 2])
    agree(got, lse, ref, torch.bfloat16, 130)
    got, lse = cache.attend(0, q.cuda(), offsets=i32([0, 1, 2]), return_lse=True)
    agree(got, lse, ref, torch.bfloat16, 130)


def test_side_stream(pc):
    """Everything on a stream of its own, while the default stream is busy."""
    lengths = [100, 700]
    cache, pool, table = make(pc, lengths)
    q = queries(2, 2, 64, torch.bfloat16)
    ref = O.attention(pool, table, lengths, 0, q, [0, 1, 2])
    dev = q.cuda()
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    for _ in range(4):
        busy = busy @ busy * 1e-2
    outs = [cache.attend(0, dev, stream=side, return_lse=True) for _ in range(3)]
    with torch.cuda.stream(side):
        outs.append(cache.attend(0, dev, return_lse=True))
    side.synchronize()
    for got, lse in outs:
        agree(got, lse, ref, torch.bfloat16, 700)


def test_in_a_cuda_graph(pc):
    lengths = [100, 700, 0]
    cache, pool, table = make(pc, lengths, spare=9)
    q = queries(3, 2, 64, torch.bfloat16).cuda()
    out = torch.empty_like(q)
    counts = i32([1, 1, 0])
    kv = queries(3, 2, 64, torch.bfloat16, 7).cuda()
    cache.attend(0, q, out=out)             # workspaces exist before the capture
    cache.extend(i32([0, 0, 0]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    cache.attend(0, q, out=out, stream=side)
    cache.extend(i32([0, 0, 0]), stream=side)
    with torch.cuda.graph(graph, stream=side):
        cache.extend(counts)
        cache.store(kv, kv, layer=0)
        cache.attend(0, q, out=out)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert cache.lengths.tolist() == [103, 703, 0]
    ref = O.attention(cache.pool.cpu(), cache.page_table.cpu(), [103, 703, 0], 0, q.cpu(), [0, 1, 2, 3])
    agree(out, None, ref, torch.bfloat16, 703)


# ---------------------------------------------------------------------------
# shared prefixes
# ---------------------------------------------------------------------------

def voices_and_members(pc, prefixes, suffixes, hkv=2, d=64, ps=16, dtype=torch.bfloat16, seed=0):
    """Slots: the voices, then for each voice its members, forked from it and
    extended by suffixes[voice]; everything not stored is NaN."""
    n = len(prefixes) + sum(len(s) for s in suffixes)
    longest = max(p + max(s, default=0) for p, s in zip(prefixes, suffixes))
    pages = sum(-(-p // ps) for p in prefixes) + sum(2 + x // ps for s in suffixes for x in s) + 4
    cache = pc.PagedCache.allocate(pages, n, longest + 1, 1, hkv, d, ps, dtype)
    cache.pool.fill_(float("nan"))
    g = torch.Generator().manual_seed(seed)

    def add(counts):
        rows = sum(counts)
        cache.extend(i32(counts))
        k, v = (torch.randn(1, rows, hkv, d, generator=g).to(dtype).cuda() for _ in range(2))
        cache.store(k, v, offsets=i32([0] + np.cumsum(counts).tolist()))

    add(list(prefixes) + [0] * (n - len(prefixes)))
    source, more, groups, at = [-1] * len(prefixes), [0] * len(prefixes), [], len(prefixes)
    for v, s in enumerate(suffixes):
        groups.append((v, prefixes[v], list(range(at, at + len(s)))))
        source += [v] * len(s)
        more += s
        at += len(s)
    cache.fork(i32(source))
    add(more)
    assert (cache.status == 0).all()
    return cache, groups


def check_shared(pc, cache, groups, group=1, window=0, sinks=0, rows=None, seed=5):
    lengths = cache.lengths.cpu().tolist()
    rows = len(lengths) if rows is None else rows
    q = queries(rows, cache.kv_heads * group, cache.head_dim, cache.dtype, seed)
    ref = O.attention(cache.pool.cpu(), cache.page_table.cpu(), lengths[:rows], 0, q, list(range(rows + 1)), window,
                      sinks)
    plan = pc.PrefixGroups(cache, groups, q_heads=q.shape[1])
    for shared_tokens in (plan._c.shared_tokens, 0):    # by the rule on sizes, and shared in any case
        plan._c.shared_tokens = shared_tokens
        got, lse = cache.attend_shared(0, q.cuda(), plan, window=window, sinks=sinks, return_lse=True)
        agree(got, lse, ref, cache.dtype, max(lengths))
    assert (cache.status == 0).all()


@pytest.mark.parametrize("prefixes,suffixes", [
    ([208], [[1, 5, 17, 40, 100, 249, 3, 64]]), ([16], [[1]]), ([48], [[0, 0, 1]]), ([218, 37], [[1, 30], [2, 9, 200]]),
    ([1000], [[7] * 3]), ([64, 128, 256], [[1 + i % 7 for i in range(130)], [3], [2] * 270]), ([5], [[1, 2, 3]])])
@pytest.mark.parametrize("group,d,dtype", [(1, 64, torch.bfloat16), (4, 128, torch.float16)])
def test_shared(pc, prefixes, suffixes, group, d, dtype):
    cache, groups = voices_and_members(pc, prefixes, suffixes, d=d, dtype=dtype)
    check_shared(pc, cache, groups, group)


def test_shared_many_groups(pc):
    """More groups than the prefix pass's kernel has threads."""
    cache, groups = voices_and_members(pc, [16 + 16 * (i % 3) for i in range(400)], [[1 + i % 5] for i in range(400)])
    check_shared(pc, cache, groups)


@pytest.mark.parametrize("hkv,group,d,ps", [(12, 1, 64, 16), (1, 13, 64, 32), (2, 64, 128, 128), (3, 3, 128, 64)])
def test_shared_heads(pc, hkv, group, d, ps):
    cache, groups = voices_and_members(pc, [3 * ps + 5, 640], [[1, 70, 9], [2, 33]], hkv=hkv, d=d, ps=ps)
    check_shared(pc, cache, groups, group)


def test_shared_long_prefix_is_cut(pc):
    """Few members and a long prefix: the prefix's key tiles are dealt over the SMs and joined."""
    cache, groups = voices_and_members(pc, [9000, 4096], [[1, 2, 3], [5] * 140], hkv=1, d=128)
    check_shared(pc, cache, groups, group=2)


@pytest.mark.parametrize("window,sinks", [(30, 208), (30, 300), (1, 218), (500, 208), (30, 100), (30, 0)])
def test_shared_window(pc, window, sinks):
    """sinks below the prefix's length: attended slot by slot."""
    cache, groups = voices_and_members(pc, [218], [[1, 5, 40, 100, 249]])
    check_shared(pc, cache, groups, group=2, window=window, sinks=sinks)


def test_shared_slots_change_hands(pc):
    """Members closed, reopened from another voice or too short, and a voice among its members."""
    cache, groups = voices_and_members(pc, [64, 96], [[1, 5, 9], [2, 30, 4]])
    n = cache.slots
    groups = [(v, p, [v] + m) for v, p, m in groups]
    check_shared(pc, cache, groups)
    mask = torch.zeros(n, dtype=torch.bool, device="cuda")
    mask[groups[0][2][1]] = True
    mask[groups[1][2][2]] = True
    cache.free(mask)
    source = [-1] * n
    source[groups[0][2][2]] = 1             # a member of voice 0 now speaks with voice 1
    source[groups[1][2][3]] = 0             # and the other way round: shorter than its group's prefix
    cache.fork(i32(source))
    check_shared(pc, cache, groups)
    check_shared(pc, cache, groups, rows=n - 2)
    check_shared(pc, cache, groups[:1])
    check_shared(pc, cache, [])
    cache.compact()
    check_shared(pc, cache, groups)
    mask.zero_()
    mask[1] = True                          # a voice closed under its members
    cache.free(mask)
    check_shared(pc, cache, groups)


def test_shared_refusals(pc):
    cache, groups = voices_and_members(pc, [64, 96], [[1, 5, 9], [2, 30, 4]])
    other, _ = voices_and_members(pc, [64], [[1]])
    plan = pc.PrefixGroups(cache, groups, q_heads=4)
    q = queries(cache.slots, 4, 64, torch.bfloat16).cuda()
    bad = [lambda: pc.PrefixGroups(cache, [(0, 64, [2, 3]), (1, 96, [3])], 4),
           lambda: pc.PrefixGroups(cache, [(99, 64, [2])], 4), lambda: pc.PrefixGroups(cache, [(0, 64, [-1])], 4),
           lambda: pc.PrefixGroups(cache, [(0, 64, [99])], 4), lambda: pc.PrefixGroups(cache, [(0, 1 << 20, [2])], 4),
           lambda: pc.PrefixGroups(cache, groups, 3), lambda: other.attend_shared(0, q[:2], plan),
           lambda: cache.attend_shared(0, q[:, :2], plan), lambda: cache.attend_shared(0, torch.cat([q, q]), plan),
           lambda: cache.attend_shared(0, q, plan, window=-1), lambda: cache.attend_shared(1, q, plan),
           lambda: cache.attend_shared(0, q, plan, scale=0.0)]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {n} was accepted")


# ---------------------------------------------------------------------------
# refusals on the host
# ---------------------------------------------------------------------------

def test_host_refusals(pc):
    cache, _, _ = make(pc, [20, 30])
    q = queries(2, 4, 64, torch.bfloat16).cuda()
    kv = queries(2, 2, 64, torch.bfloat16).cuda()
    bad = [
        lambda: cache.attend(2, q), lambda: cache.attend(-1, q), lambda: cache.attend(0, q[:, :3]),
        lambda: cache.attend(0, q.half()), lambda: cache.attend(0, q.cpu()), lambda: cache.attend(0, q[..., :32]),
        lambda: cache.attend(0, torch.cat([q, q])), lambda: cache.attend(0, q, window=-1),
        lambda: cache.attend(0, q, sinks=-1), lambda: cache.attend(0, q, out=q[:1]),
        lambda: cache.attend(0, q, offsets=i32([0, 1])), lambda: cache.attend(0, q, offsets=torch.tensor([0, 1, 2])),
        lambda: cache.attend(0, q, key_mask=torch.ones(2, 16, dtype=torch.bool, device="cuda")),
        lambda: cache.attend(0, q.transpose(0, 1)),
        lambda: cache.attend(0, torch.cat([q, q], 1).view(2, 64, 8).transpose(1, 2)[:, :, :64].reshape(2, 8, 64)[:, ::2]),
        lambda: cache.attend(0, torch.empty(2 * 256 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 4, 64)),
        lambda: cache.extend(i32([1])), lambda: cache.extend(torch.tensor([1, 1], device="cuda")),
        lambda: cache.extend(torch.tensor([1, 1], dtype=torch.int32)), lambda: cache.fork(i32([0, 1, 2])),
        lambda: cache.free(i32([0, 1])), lambda: cache.store(kv, kv[:1], layer=0),
        lambda: cache.store(kv, kv, layer=2), lambda: cache.store(kv, kv), lambda: cache.store(kv.half(), kv, layer=0),
        lambda: cache.store(torch.cat([kv, kv]), torch.cat([kv, kv]), layer=0),
        lambda: pc.PagedCache.allocate(4, 2, 64, 1, 2, 96), lambda: pc.PagedCache.allocate(4, 2, 64, 1, 2, 64, 24),
        lambda: pc.PagedCache.allocate(4, 2, 0, 1, 2, 64),
        lambda: pc.PagedCache.allocate(4, 2, 64, 1, 2, 64, dtype=torch.float32),
        lambda: pc.PagedCache(cache.pool, cache.page_table.long(), cache.lengths, cache.refs),
        lambda: pc.PagedCache(cache.pool, cache.page_table, cache.lengths[:1], cache.refs),
        lambda: pc.PagedCache(cache.pool, cache.page_table, cache.lengths, cache.refs[1:]),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {n} was accepted")
    assert cache.attend(0, q[:0]).shape == (0, 4, 64)
    cache.store(kv[:0], kv[:0], layer=0)
