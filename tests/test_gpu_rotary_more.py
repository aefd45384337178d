"""The rotation and the append that rotates: which slots are refused is said in full, and a
rotation's inverse and lengths are held pair by pair."""
import pytest
import torch

from oracle import paged_cache as O
from test_gpu_paged_4bit import TYPES, values
from test_gpu_paged_cache import i32, pc  # noqa: F401
from test_gpu_rotary import rotary  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", TYPES)
def test_append_to_refused_slots(pc, rotary, bits, dtype):  # noqa: F811
    """Slot 1 asks for two pages where one is free, and slot 4 comes after it: both are refused.  Statuses, refusals and
    the rows of zeros are those of the plain restatement."""
    d, hkv = 64, 2
    r = rotary.Rotation(d)
    cache = pc.PagedCache.allocate(4, 5, 64, 1, hkv, d, 16, dtype, bits=bits)
    cache.pool.view(torch.uint8).fill_(1)
    sim = O.ListCache(cache.pool.cpu().clone(), 5, cache.table_pages, dtype if bits == 4 else None)
    for counts in ([16, 16, 10, 0, 0], [0, 20, 0, 0, 5]):
        cache.extend(i32(counts))
        sim.extend(counts)
        if counts[0]:
            cache.fork(i32([-1, -1, -1, 0, -1]))         # slot 3 shares slot 0's page
            sim.fork([-1, -1, -1, 0, -1])
    assert sim.status == [0, 2, 0, 0, 2] and sim.refused == [False, True, False, False, True]
    assert cache.status.tolist() == sim.status and cache.refused.bool().tolist() == sim.refused
    assert cache.lengths.tolist() == [16, 16, 10, 16, 0] == sim.lengths
    offsets = [1, 2, 4, 10, 11, 13]                     # a row before the first and two behind the last
    x = values((15, 6, d), dtype, 1)
    y = x.cuda()
    cache.status.zero_()
    sim.status = [0] * 5
    got = cache.append(0, y[:, :2], y[:, 2:4], y[:, 4:], r, offsets=i32(offsets))
    place = torch.tensor([0, 15, 0, 0] + list(range(4, 10)) + [15] + [0] * 4, dtype=torch.int32)
    q, k = r.rotate(y[:, :2], y[:, 2:4], place.cuda())
    sim.store(k.cpu()[None], x[None, :, 4:], offsets, [0])
    zero = [0, 2, 3, 11, 12, 13, 14]
    for row in range(15):
        assert torch.equal(got[row], torch.zeros_like(got[row]) if row in zero else q[row]), row
    assert cache.status.tolist() == sim.status == [3, 0, 0, 3, 0]
    assert torch.equal(cache.pool.cpu().view(torch.uint8), sim.data.view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rot,interleaved", [(64, 64, False), (128, 96, False), (128, 128, True), (64, 48, True)])
def test_lengths_and_inverse_pair_by_pair(rotary, dtype, d, rot, interleaved):  # noqa: F811
    """A turned value is off by u |y| for its rounding and (d + 24) 2^-24 (|a| + |b|) for its arithmetic, at most e = (u + (d +
    24) 2^-24) (|a| + |b|), and half of the type's smallest number: a pair's length by twice that, and turning back adds the same
    to what the first errors become, e (|cos| + |sin|) <= 1.5 e each.  Small pairs stand beside large ones."""
    x = values((50, 4, d), dtype, 5) * torch.exp2(torch.randint(-9, 1, (50, 4, d), generator=torch.Generator().manual_seed(1)).float())
    x = x.to(dtype).cuda()
    pos = torch.arange(50, dtype=torch.int32, device="cuda") * 1000 - 7
    r = rotary.Rotation(d, rot, interleaved=interleaved)
    turned, _ = r.rotate(x, None, pos)
    back, _ = r.rotate(turned, None, -pos)
    assert torch.equal(turned[..., rot:], x[..., rot:]) and torch.equal(back[..., rot:], x[..., rot:])

    def pairs(t):
        t = t[..., :rot].double()
        return t.unflatten(-1, (-1, 2)) if interleaved else t.unflatten(-1, (2, -1)).transpose(-1, -2)
    a, b, c = pairs(x), pairs(turned), pairs(back)
    u = torch.finfo(dtype).eps / 2
    e = (u + (d + 24) * 2.0 ** -24) * a.abs().sum(-1) + torch.finfo(dtype).smallest_normal * u
    assert ((b.norm(dim=-1) - a.norm(dim=-1)).abs() <= 2 * e).all()
    assert ((c - a).abs() <= 1.01 * (1.5 + 1) * e[..., None]).all()
