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
