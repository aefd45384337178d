"""Outputs of load and rotate that share memory are refused, on the host and before
any launch: every way that rows, layers and tensors can lie in one another, against
sets of the elements that they cover.  The library is a stand-in, the tensors are on the CPU."""
import random

import pytest
import torch

from test_paged_cache_python import lib, on_host  # noqa: F401
from test_rotary_host import turner

H, D = 2, 64
BLOCK = H * D


def covered(base, shape, strides, block=BLOCK):
    """Elements of the blocks at base + sum i strides, or None where two of them share some."""
    starts = [base]
    for n, s in zip(shape, strides):
        starts = [a + i * s for a in starts for i in range(n)]
    seen = set()
    for a in starts:
        here = set(range(a, a + block))
        if seen & here:
            return None
        seen |= here
    return seen


def strided(storage, at, shape, strides):
    return torch.as_strided(storage, (*shape, H, D), (*strides, D, 1), at)


LAYOUTS = [(layers, rows, 8 * a, 8 * b) for layers, rows in ((2, 3), (3, 2), (4, 5), (2, 1), (1, 3), (3, 7))
           for a, b in ((16, 16), (16, 32), (16, 48), (48, 16), (80, 16), (32, 48), (48, 32), (33, 24), (40, 17), (8, 16), (0, 16), (64, 24),
                        (17, 51), (112, 16), (40, 64))]


@pytest.mark.parametrize("layers,rows,layer,row", LAYOUTS)
def test_load_into_layers(lib, layers, rows, layer, row):  # noqa: F811
    cache = on_host(slots=8, layers=layers)
    storage = torch.zeros(20000, dtype=torch.bfloat16)
    storage = storage[(-storage.data_ptr() // 2) % 8:]
    x = strided(storage, 0, (layers, rows), (layer, row))
    fine = torch.zeros(layers, rows, H, D, dtype=torch.bfloat16)
    apart = covered(0, (layers, rows), (layer, row)) is not None
    for kw in (dict(k=x, v=fine), dict(k=fine, v=x)):
        if apart:
            cache.load(rows, **kw)
        else:
            with pytest.raises(ValueError):
                cache.load(rows, **kw)
    assert len(lib.calls) == (2 if apart else 0)


def test_load_of_no_rows(lib):  # noqa: F811
    cache = on_host()
    none = torch.zeros(1, 0, H, D, dtype=torch.bfloat16).expand(2, 0, H, D)
    cache.load(0, k=none, v=none)
    assert len(lib.calls) == 1


def two_layouts(n):
    """Pairs of layouts in one storage whose own rows are apart: most of them views of a buffer of wider rows."""
    rng, found = random.Random(5), []
    while len(found) < n:
        layers, rows = rng.choice([(1, 1), (1, 4), (2, 3), (3, 2), (4, 1), (3, 5)])
        strides = [8 * rng.randint(16, 60) if rng.random() < 0.5 else rng.choice([128, 256, 384, 512, 768, 1024, 1536]) for _ in range(2)]
        other = strides if rng.random() < 0.7 else [8 * rng.randint(16, 100) for _ in range(2)]
        at = 8 * rng.randint(0, 120) if rng.random() < 0.5 else 128 * rng.randint(0, 12)
        a, b = covered(0, (layers, rows), strides), covered(at, (layers, rows), other)
        if a is not None and b is not None:
            found.append((layers, rows, strides, other, at, bool(a & b)))
    return found


@pytest.mark.parametrize("swap", [False, True])
def test_keys_and_values_into_one_storage(lib, swap):  # noqa: F811
    storage = torch.zeros(20000, dtype=torch.bfloat16)
    storage = storage[(-storage.data_ptr() // 2) % 8:]
    found = two_layouts(600)
    assert 100 < sum(share for *_, share in found) < 500
    for layers, rows, strides, other, at, share in found:
        cache = on_host(slots=8, layers=layers)
        x, y = strided(storage, 0, (layers, rows), strides), strided(storage, at, (layers, rows), other)
        if at == 0 and x.stride() == y.stride():
            continue                                    # one tensor: see below
        k, v = (y, x) if swap else (x, y)
        before = len(lib.calls)
        if share:
            with pytest.raises(ValueError):
                cache.load(rows, k=k, v=v)
        else:
            cache.load(rows, k=k, v=v)
        assert len(lib.calls) == before + (not share)
        if layers == 1:                                 # the same, one layer by itself
            if share:
                with pytest.raises(ValueError):
                    cache.load(rows, layer=0, k=k[0], v=v[0])
            else:
                cache.load(rows, layer=0, k=k[0], v=v[0])


def test_one_tensor_for_keys_and_values(lib, monkeypatch):  # noqa: F811
    """The values go there, the keys elsewhere."""
    from magpie_tts_rt_b200 import paged_cache as pc
    made = []
    real = pc.L.CacheRows
    monkeypatch.setattr(pc.L, "CacheRows", lambda: made.append(real()) or made[-1])
    cache, x = on_host(), torch.zeros(2, 3, 2, H, D, dtype=torch.bfloat16)[:, :, 0]
    k, v = cache.load(3, k=x, v=x)
    assert k is x and v is x and made[-1].v == x.data_ptr() and made[-1].v_row_stride == x.stride(1)
    low, high = x.data_ptr(), x.data_ptr() + 2 * (x.stride(0) + 2 * x.stride(1) + BLOCK)
    size = 2 * (made[-1].k_layer_stride + 2 * made[-1].k_row_stride + BLOCK)
    assert made[-1].k + size <= low or made[-1].k >= high
    assert len(lib.calls) == 1


def test_queries_and_keys_into_one_storage(lib):  # noqa: F811
    """Of other numbers of heads, too."""
    r, rng = turner(), random.Random(7)
    storage = torch.zeros(20000, dtype=torch.bfloat16)
    storage = storage[(-storage.data_ptr() // 2) % 8:]
    shared = 0
    for _ in range(600):
        rows, heads = rng.choice([1, 2, 5]), (rng.choice([1, 2, 4]), rng.choice([1, 2]))
        row = [rng.choice([64 * h, 256, 384, 8 * rng.randint(8 * h, 60)]) for h in heads]
        row[1] = row[0] if rng.random() < 0.6 and row[0] >= 64 * heads[1] else row[1]
        at = 8 * rng.randint(0, 80) if rng.random() < 0.5 else 64 * rng.randint(0, 12)
        a, b = (covered(x, (rows,), (s,), 64 * h) for x, s, h in zip((0, at), row, heads))
        if a is None or b is None:
            continue
        outs = [torch.as_strided(storage, (rows, h, D), (s, D, 1), x) for x, s, h in zip((0, at), row, heads)]
        q, k = (torch.zeros(rows, h, D, dtype=torch.bfloat16) for h in heads)
        before, pos = len(lib.calls), torch.zeros(rows, dtype=torch.int32)
        if a & b:
            shared += 1
            with pytest.raises(ValueError):
                r.rotate(q, k, pos, q_out=outs[0], k_out=outs[1])
        else:
            r.rotate(q, k, pos, q_out=outs[0], k_out=outs[1])
        assert len(lib.calls) == before + (not a & b)
    assert shared > 50


def test_rotating_in_place(lib):  # noqa: F811
    """Queries and keys of one projection's rows, where they are."""
    y, r = torch.zeros(3, 5, D, dtype=torch.bfloat16), turner()
    q, k = y[:, :3], y[:, 3:]
    got = r.rotate(q, k, torch.zeros(3, dtype=torch.int32), q_out=q, k_out=k)
    assert got[0] is q and got[1] is k and len(lib.calls) == 1
    for bad in (y[:, 2:4], y[:, :2], q[:, 1:]):
        with pytest.raises(ValueError):
            r.rotate(q, k, torch.zeros(3, dtype=torch.int32), q_out=q, k_out=bad)
    assert len(lib.calls) == 1
