"""Norm and position rotation of heads (rotary.Rotation) and the append that
rotates (PagedCache.append) on the GPU.

Tolerance of a rotated value, derived: f32 arithmetic on a pair (a, b) loses at
most (D + 24) 2^-24 (|a| + |b|): the mean of D squares in f32, a reciprocal square root
and two products (8 roundings), cosine and sine (the reduced angle right to 2^-22, the
functions to 2^-21: 12 of these units), two products and a sum.  The result is rounded once:
u |y|, u = finfo.eps / 2."""
import math

import numpy as np
import pytest
import torch

from oracle import paged_cache as O
from test_gpu_paged_4bit import check, make4, same_pool, token_bytes, values  # noqa: F401
from test_gpu_paged_cache import i32, make, pc, queries  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def rotary():
    from magpie_tts_rt_b200 import rotary
    return rotary


def near(got, ref, dtype, d):
    y, size = ref
    tol = torch.finfo(dtype).eps / 2 * y.abs() + (d + 24) * 2.0 ** -24 * size + 1e-30
    if dtype is torch.float16:
        tol = tol + 2.0 ** -25                          # half of its smallest number
    err = (got.cpu().double() - y).abs()
    assert (err <= tol).all(), (err / tol).max().item()


def radians(base, rot):
    return [base ** (-2.0 * i / rot) for i in range(rot // 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rot", [(64, 64), (64, 16), (64, 48), (128, 128), (128, 64), (128, 96), (128, 112)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_rotate(rotary, dtype, d, rot, interleaved, norm):
    rows, heads, kv = 37, 5, 3
    x = values((rows, heads + kv, d), dtype, d + rot)
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(s))) for s in (1, 2))
    pos = torch.tensor([0, 1, 2, -1, 131071, 2 ** 20 + 3, -77] + list(range(30)), dtype=torch.int32)
    r = rotary.Rotation(d, rot, base=5e5, interleaved=interleaved, q_norm=qw if norm else None, k_norm=kw if norm else None)
    y = x.cuda()
    q, k = r.rotate(y[:, :heads], y[:, heads:], pos.cuda())
    for got, src, w in ((q, x[:, :heads], qw), (k, x[:, heads:], kw)):
        near(got, O.rotated(src, pos, rot, radians(5e5, rot), interleaved, w if norm else None), dtype, d)
    # in place, and alone, the same bits
    assert torch.equal(r.rotate(y[:, :heads], None, pos.cuda())[0], q)
    only = r.rotate(None, y[:, heads:], pos.cuda())
    assert only[0] is None and torch.equal(only[1], k)
    r.rotate(y[:, :heads], y[:, heads:], pos.cuda(), q_out=y[:, :heads], k_out=y[:, heads:])
    assert torch.equal(y, torch.cat([q, k], 1))


@pytest.mark.parametrize("rows,heads,kv", [(1, 1, 1), (1, 64, 8), (3, 12, 12), (5000, 1, 1), (700, 40, 5), (0, 4, 4)])
def test_rotate_sizes(rotary, rows, heads, kv):
    d, dtype = 128, torch.bfloat16
    x = values((rows, heads + kv, d), dtype, rows)
    pos = torch.randint(0, 1 << 20, (rows,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    w = 1 + 0.1 * torch.randn(d, generator=torch.Generator().manual_seed(3)).to(dtype)
    r = rotary.Rotation(d, q_norm=w)
    q, k = r.rotate(x[:, :heads].cuda(), x[:, heads:].cuda(), pos.cuda())
    near(q, O.rotated(x[:, :heads], pos, d, radians(1e4, d), weight=w), dtype, d)
    near(k, O.rotated(x[:, heads:], pos, d, radians(1e4, d)), dtype, d)


def test_rotate_far_positions_and_given_frequencies(rotary):
    """Positions to the ends of 32 bits: the angle is kept to 2^-22 of a turn and less."""
    d, f = 64, torch.linspace(1.0, 3.0, 32, dtype=torch.float64)
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 12345678], dtype=torch.int32)
    x = values((4, 2, d), torch.float16, 1)
    got, _ = rotary.Rotation(d, frequencies=f).rotate(x.cuda(), None, pos.cuda())
    y, size = O.rotated(x, pos, d, f.tolist())
    tol = 2.0 ** -11 * y.abs() + 2 * math.pi * 2.0 ** -21 * size + (d + 24) * 2.0 ** -24 * size + 2.0 ** -25
    assert ((got.cpu().double() - y).abs() <= tol).all()


def test_rotate_keeps_lengths_and_inverts(rotary):
    """Turning back by the negative position gives the input, within two roundings."""
    d, dtype = 128, torch.float16
    x = values((50, 4, d), dtype, 5).cuda()
    pos = torch.arange(50, dtype=torch.int32, device="cuda") * 1000
    r = rotary.Rotation(d, 96)
    back, _ = r.rotate(r.rotate(x, None, pos)[0], None, -pos)
    size = (x.double().unflatten(-1, (-1, 16)).abs().amax((-1, -2), keepdim=True) * 2).flatten(-2)
    assert ((back.double() - x.double()).abs() <= 2.5 * 2.0 ** -11 * size + 1e-6).all()
    assert torch.equal(back[..., 96:], x[..., 96:])


def test_rotate_values_beside_infinities(rotary):
    """A dim past rotary_dim keeps its bits; an infinity or NaN reaches its own pair only (and its head where there is a norm)."""
    x = values((3, 2, 64), torch.bfloat16, 1)
    x[1, 0, 3], x[1, 1, 40], x[2, 0, 63] = float("inf"), float("nan"), -float("inf")
    got, _ = rotary.Rotation(64, 32).rotate(x.cuda(), None, i32([5, 6, 7]))
    got = got.cpu()
    bad = ~torch.isfinite(got)
    assert bad.nonzero().tolist() == [[1, 0, 3], [1, 0, 19], [1, 1, 40], [2, 0, 63]]
    assert torch.equal(got[..., 32:].view(torch.int16), x[..., 32:].view(torch.int16))


def test_rotation_made_on_a_busy_stream(rotary):
    """Weights that a stream has yet to write: the rotation is there for any stream at once."""
    side = torch.cuda.Stream()
    x, pos = values((4, 2, 64), torch.bfloat16, 1).cuda(), i32([0, 1, 2, 3])
    weight, given = torch.ones(64, device="cuda"), torch.rand(64, device="cuda") + 0.5
    ref, _ = rotary.Rotation(64, q_norm=given).rotate(x, None, pos)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        weight.copy_(given)
        r = rotary.Rotation(64, q_norm=weight)
    got, _ = r.rotate(x, None, pos)
    assert torch.equal(got, ref)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def filled(pc, bits, lengths, hkv, d, ps, dtype, layers=2):
    if bits == 4:
        return make4(pc, lengths, hkv, d, ps, layers, dtype)[0]
    return make(pc, lengths, hkv, d, ps, layers, dtype)[0]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rot,interleaved", [(64, 64, False), (64, 48, False), (64, 32, True), (128, 128, False),
                                               (128, 96, False), (128, 128, True), (128, 48, False)])
@pytest.mark.parametrize("prompt", [False, True])
def test_append_is_rotate_and_store(pc, rotary, bits, dtype, d, rot, interleaved, prompt):
    """Bit for bit, in the queries and in the pool, with positions from the cache and with given ones."""
    lengths, hkv, ps, heads = [0, 1, 17, 40, 64, 3], 3, 16, 9
    new = [0, 1, 9, 40, 3, 2] if prompt else [1] * 6
    offsets = [0] + np.cumsum(new).tolist()
    rows = offsets[-1]
    y = values((rows, heads + 2 * hkv, d), dtype, 3).cuda()
    q, k, v = y[:, :heads], y[:, heads:heads + hkv], y[:, heads + hkv:]
    w = [1 + 0.2 * torch.randn(d, generator=torch.Generator().manual_seed(s)) for s in (1, 2)]
    r = rotary.Rotation(d, rot, interleaved=interleaved, q_norm=w[0], k_norm=w[1])
    at = i32(offsets) if prompt else None
    place = torch.tensor([max(n - m + j, 0) for n, m in zip(lengths, new) for j in range(m)], dtype=torch.int32).cuda()
    given = torch.arange(rows, dtype=torch.int32, device="cuda") * 7919
    for positions in (None, given):
        one, two = (filled(pc, bits, lengths, hkv, d, ps, dtype) for _ in range(2))
        got = one.append(1, q, k, v, r, offsets=at, positions=positions)
        want, turned = r.rotate(q, k, place if positions is None else positions)
        two.store(turned, v, layer=1, offsets=at)
        torch.cuda.synchronize()
        if not prompt:
            want[0] = 0                                 # slot 0 has no token
        assert torch.equal(got, want)
        assert torch.equal(one.pool.view(torch.uint8), two.pool.view(torch.uint8))
        assert one.status.tolist() == two.status.tolist()


@pytest.mark.parametrize("bits", [16, 4])
def test_append_refused_and_unfit_rows(pc, rotary, bits):
    """Rows of no slot, of slots that were refused their tokens, of more tokens than there are, and on shared pages."""
    d, hkv = 64, 2
    r = rotary.Rotation(d)
    cache = pc.PagedCache.allocate(4, 5, 64, 1, hkv, d, 16, bits=bits)
    cache.pool.view(torch.uint8).fill_(1)
    cache.extend(i32([16, 16, 10, 0, 0]))
    cache.fork(i32([-1, -1, -1, 0, -1]))                # slot 3 shares slot 0's page
    cache.extend(i32([0, 20, 0, 0, 5]))                 # slot 1: no room for 2 pages; slot 4: the last page
    assert cache.status.tolist() == [0, 2, 0, 0, 0] or cache.status.tolist()[1] == 2
    refused = cache.refused.tolist()
    before = cache.pool.clone()
    offsets = i32([1, 2, 4, 16, 17, 19])                # a row before the first; 12 rows of slot 2, which has 10 tokens
    x = values((21, 6, d), torch.bfloat16, 1).cuda()
    cache.status.zero_()
    got = cache.append(0, x[:, :2], x[:, 2:4], x[:, 4:], r, offsets=offsets)
    torch.cuda.synchronize()
    status = cache.status.tolist()
    assert refused[1] == 1 and status[1] == 0 and status[2] == 1 and status[0] == 3 and status[3] == 3
    zero = [0] + [2, 3] + list(range(4, 16)) + [19, 20] + ([17, 18] if refused[4] else [])
    for row in range(21):
        assert (got[row] == 0).all() == (row in zero), row
    # a shared page's token is turned, not stored
    want, _ = r.rotate(x[:, :2], None, i32([0, 15] + [0] * 14 + [15] + [0] * 4))
    assert torch.equal(got[1], want[1]) and torch.equal(got[16], want[16])
    kept = cache.page_table[0, 0].item(), cache.page_table[1, 0].item(), cache.page_table[2, 0].item()
    for p in kept:
        assert torch.equal(cache.pool[p].view(torch.uint8), before[p].view(torch.uint8))


def test_append_without_queries_and_in_place(pc, rotary):
    lengths, d = [5, 33], 128
    r = rotary.Rotation(d, k_norm=torch.ones(d))
    y = values((2, 6, d), torch.bfloat16, 2).cuda()
    one, two = (filled(pc, 16, lengths, 2, d, 16, torch.bfloat16) for _ in range(2))
    assert one.append(0, None, y[:, 2:4], y[:, 4:], r) is None
    q = two.append(0, y[:, :2], y[:, 2:4], y[:, 4:], r)
    assert torch.equal(one.pool.view(torch.int16), two.pool.view(torch.int16))
    again = y.clone()
    same = two.append(0, again[:, :2], again[:, 2:4], again[:, 4:], r, q_out=again[:, :2])
    assert torch.equal(same, q) and torch.equal(again[:, 2:], y[:, 2:])


@pytest.mark.parametrize("slots", [1, 2, 31, 32, 33, 500, 1024, 1025, 3000])
def test_rows_find_their_slots(pc, slots):
    """Ragged rows, empty slots among them, of many slots: each row goes to its own."""
    rng = np.random.default_rng(slots)
    new = np.where(rng.random(slots) < 0.6, rng.integers(1, 4, slots), 0)
    new[-1] = 2
    cache = pc.PagedCache.allocate(2 * slots, slots, 32, 1, 1, 64, 16)
    cache.extend(i32(new.tolist()))
    offsets = [0] + np.cumsum(new).tolist()
    x = values((offsets[-1], 1, 64), torch.bfloat16, 3).cuda()
    cache.store(x, -x, layer=0, offsets=i32(offsets))
    k, v = cache.load(offsets[-1], layer=0, offsets=i32(offsets))
    assert torch.equal(k, x) and torch.equal(v, -x)
    last = [offsets[i + 1] - 1 for i in range(slots) if new[i]]
    k, _ = cache.load(slots, layer=0)
    assert torch.equal(k[torch.tensor(new > 0, device="cuda")], x[last])


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("graph", [False, True])
def test_a_decoder_with_rotation(pc, rotary, bits, graph):
    """Prompt, fork, steps with append and attention, sessions closed and the pool compacted, on another stream than the
    default one, the steps replayed from a CUDA graph: attention over what the cache then holds, in 64 bits."""
    d, hkv, heads, ps, dtype, layers = 64, 2, 4, 16, torch.bfloat16, 2
    stream = torch.cuda.Stream()
    cache = pc.PagedCache.allocate(64, 5, 96, layers, hkv, d, ps, dtype, bits=bits)
    w = 1 + 0.1 * torch.randn(d, generator=torch.Generator().manual_seed(1))
    r = rotary.Rotation(d, base=1e4, q_norm=w, k_norm=w)
    seen = {i: [] for i in range(5)}                     # what each slot was given: (layer, position) -> rows
    with torch.cuda.stream(stream):
        new = [30, 0, 21, 0, 0]
        offsets = i32([0] + np.cumsum(new).tolist())
        cache.extend(i32(new))
        x = values((layers, sum(new), heads + 2 * hkv, d), dtype, 1).cuda()
        for layer in range(layers):
            q = cache.append(layer, x[layer, :, :heads], x[layer, :, heads:heads + hkv], x[layer, :, heads + hkv:], r, offsets=offsets)
            out = cache.attend(layer, q, offsets=offsets)
        for i, (a, b) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
            seen[i] = [x[:, t].cpu() for t in range(a, b)]
        cache.fork(i32([-1, 0, -1, 2, -1]))
        seen[1], seen[3] = list(seen[0]), list(seen[2])
        one = i32([1, 1, 1, 1, 0])
        y = torch.empty(layers, 5, heads + 2 * hkv, d, dtype=dtype, device="cuda")
        outs = torch.empty(layers, 5, heads, d, dtype=dtype, device="cuda")

        def step():
            cache.extend(one)
            for layer in range(layers):
                q = cache.append(layer, y[layer, :, :heads], y[layer, :, heads:heads + hkv], y[layer, :, heads + hkv:], r)
                cache.attend(layer, q, out=outs[layer])

        captured = None
        for n in range(6):
            y.copy_(values((layers, 5, heads + 2 * hkv, d), dtype, 10 + n))
            if graph and n >= 1:
                if captured is None:
                    captured = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(captured, stream=stream):
                        step()
                captured.replay()
            else:
                step()
            for i in (0, 1, 2, 3) if n <= 2 else (0, 1, 3):
                seen[i].append(y[:, i].cpu())
            if n == 2:
                cache.free(torch.tensor([False, False, True, False, False], device="cuda"))
                cache.compact()
                seen[2] = []
                one[2] = 0
    stream.synchronize()
    assert (cache.status == 0).all()
    assert cache.lengths.tolist() == [len(seen[i]) for i in range(5)]
    # the references: rows as rotate leaves them, held in 4 bits where the cache does, attention in 64 bits
    for i in (0, 1, 3):
        n = len(seen[i])
        rows = torch.stack(seen[i], 1)                   # [layers, n, heads + 2 hkv, d]
        pos = torch.arange(n, dtype=torch.int32, device="cuda")
        for layer in range(layers):
            q, k = (t.cpu() for t in r.rotate(rows[layer, :, :heads].cuda(), rows[layer, :, heads:heads + hkv].cuda(), pos))
            v = rows[layer, :, heads + hkv:]
            if bits == 4:
                blocks = torch.zeros(2, hkv, n, token_bytes(d), dtype=torch.uint8)
                for t in range(n):
                    O.put4(blocks[0], t, k[t])
                    O.put4(blocks[1], t, v[t])
                k, v = (b.transpose(0, 1) for b in O.held(blocks[None, None], dtype)[0, 0])
            p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[-1].double().view(hkv, -1, d), k.double()) / 8, -1)
            want = torch.einsum("hgn,nhd->hgd", p, v.double()).reshape(heads, d)
            weight = torch.einsum("hgn,nhd->hgd", p, v.double().abs()).reshape(heads, d)
            # the result's rounding; scores and weights are right to 2^-12 (see test_gpu_paged_4bit.py)
            tol = 2.0 ** -8 * want.abs() + 2.0 ** -12 * (weight + 1)
            err = (outs[layer, i].cpu().double() - want).abs()
            assert (err <= tol).all(), (i, layer, (err / tol).max().item())
