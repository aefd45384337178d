"""Host side of the position rotation, the append that rotates, load and the 4-bit
cache, without a GPU: the C structs as the header lays them out, the calls'
refusals, and on which device and stream the Python calls are made (the library
is a stand-in that notes each call, the tensors are on the CPU)."""
import ctypes
import os
import subprocess
import types

import pytest
import torch

from magpie_tts_rt_b200 import _lib as L
from magpie_tts_rt_b200 import paged_cache as pc
from magpie_tts_rt_b200 import rotary
from test_paged_cache_host import BAD_CACHES, attention, cache, rows
from test_paged_cache_python import HOST, lib, on_host  # noqa: F401

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD = L.STATUS_INVALID_ARGUMENT
FOUR = L.CACHE_4BIT


def test_struct_layouts(tmp_path):
    structs = {"mtt_b200_rotation_t": L.Rotation, "mtt_b200_rotate_rows_t": L.RotateRows}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "magpie_tts_rt_b200.h"', "int main(void) {"]
    expected = [FOUR]
    lines.append('  printf("%d\\n", MTT_B200_CACHE_4BIT);')
    for name, struct in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        expected.append(ctypes.sizeof(struct))
        for field, _ in struct._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({name}, {field}));')
            expected.append(getattr(struct, field).offset)
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}", ""]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(REPO, "include"), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout
    assert [int(x) for x in out.split()] == expected


def rotation(**over):
    r = L.Rotation(64, 64, 0, L.DTYPE_BF16, 1 << 20, None, None, 1e-6, 0)
    for k, v in over.items():
        setattr(r, k, v)
    return ctypes.byref(r)


def rotate_rows(**over):
    r = L.RotateRows(8, 4, 4, 0, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 256, 256, 256, 256, 256, 1 << 20, None)
    for k, v in over.items():
        setattr(r, k, v)
    return ctypes.byref(r)


BAD_ROTATIONS = [dict(head_dim=96), dict(rotary_dim=0), dict(rotary_dim=8), dict(rotary_dim=24), dict(rotary_dim=80), dict(dtype=2),
                 dict(dtype=FOUR), dict(turns=None), dict(turns=(1 << 20) + 4), dict(q_weight=(1 << 20) + 4),
                 dict(k_weight=(1 << 20) + 8), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf"))]


@pytest.mark.parametrize("bad", BAD_ROTATIONS, ids=str)
def test_bad_rotations(bad):
    assert L.lib.mtt_b200_launch_rotate_heads(rotation(**bad), rotate_rows(), None) == BAD
    assert L.lib.mtt_b200_launch_paged_cache_append(cache(), rotation(**bad), rotate_rows(), None) == BAD


SHARED_ROWS = [dict(rows=-1), dict(rows=(1 << 22) + 1), dict(q_heads=-1), dict(q_heads=65537), dict(q=None), dict(q=(1 << 20) + 8),
               dict(q_row_stride=252), dict(q_out=None), dict(q_out=(1 << 20) + 2), dict(q_out_row_stride=4), dict(k=None),
               dict(k=(1 << 20) + 4), dict(k_row_stride=4)]


@pytest.mark.parametrize("bad", SHARED_ROWS + [dict(kv_heads=-1), dict(kv_heads=65537), dict(k_out=None), dict(k_out=(1 << 20) + 8),
                                               dict(k_out_row_stride=1), dict(positions=None)], ids=str)
def test_bad_rotate_rows(bad):
    assert L.lib.mtt_b200_launch_rotate_heads(rotation(), rotate_rows(**bad), None) == BAD


@pytest.mark.parametrize("bits", [0, FOUR])
@pytest.mark.parametrize("bad", SHARED_ROWS + [dict(kv_heads=3), dict(layer=-1), dict(layer=2), dict(v=None), dict(v=(1 << 20) + 8),
                                               dict(v_row_stride=12), dict(rows=9)], ids=str)
def test_bad_append_rows(bad, bits):
    c = cache(dtype=L.DTYPE_BF16 | bits)
    assert L.lib.mtt_b200_launch_paged_cache_append(c, rotation(), rotate_rows(**bad), None) == BAD


def test_append_wants_the_caches_heads_and_type():
    assert L.lib.mtt_b200_launch_paged_cache_append(cache(), rotation(head_dim=128), rotate_rows(), None) == BAD
    assert L.lib.mtt_b200_launch_paged_cache_append(cache(), rotation(dtype=L.DTYPE_F16), rotate_rows(), None) == BAD
    assert L.lib.mtt_b200_launch_paged_cache_append(cache(dtype=FOUR | L.DTYPE_F16), rotation(), rotate_rows(), None) == BAD
    for args in ((None, rotation(), rotate_rows()), (cache(), None, rotate_rows()), (cache(), rotation(), None)):
        assert L.lib.mtt_b200_launch_paged_cache_append(*args, None) == BAD
    assert L.lib.mtt_b200_launch_rotate_heads(None, rotate_rows(), None) == BAD
    assert L.lib.mtt_b200_launch_rotate_heads(rotation(), None, None) == BAD


@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(n_layers=0), dict(layer=1, n_layers=2), dict(rows=-1),
                                 dict(rows=9), dict(k=None), dict(v=None), dict(k=(1 << 20) + 8), dict(k_row_stride=4),
                                 dict(v_layer_stride=3)], ids=str)
@pytest.mark.parametrize("bits", [0, FOUR])
def test_bad_loads_and_4bit_stores(bad, bits):
    c = cache(dtype=L.DTYPE_F16 | bits)
    assert L.lib.mtt_b200_launch_paged_cache_load(c, ctypes.byref(rows(**bad)), None) == BAD
    assert L.lib.mtt_b200_launch_paged_cache_store(c, ctypes.byref(rows(**bad)), None) == BAD


@pytest.mark.parametrize("bad", [b for b in BAD_CACHES if "dtype" not in b] + [dict(dtype=2 | FOUR), dict(dtype=2 * FOUR),
                                                                              dict(dtype=-1)], ids=str)
def test_bad_4bit_caches(bad):
    c = cache(**dict(dict(dtype=FOUR | L.DTYPE_BF16), **bad))
    assert L.lib.mtt_b200_paged_cache_workspace_size(c, 4, 8) == 0
    assert L.lib.mtt_b200_launch_paged_cache_load(c, ctypes.byref(rows()), None) == BAD
    assert L.lib.mtt_b200_launch_paged_cache_store(c, ctypes.byref(rows()), None) == BAD
    assert L.lib.mtt_b200_launch_paged_attention(c, ctypes.byref(attention()), 1 << 20, 1 << 40, None) == BAD


def test_nothing_to_do_is_done():
    assert L.lib.mtt_b200_launch_paged_cache_load(cache(), ctypes.byref(rows(rows=0, k=None, v=None)), None) == 0
    assert L.lib.mtt_b200_launch_paged_cache_store(cache(dtype=FOUR), ctypes.byref(rows(rows=0, k=None, v=None)), None) == 0
    nothing = dict(rows=0, q=None, k=None, v=None, q_out=None, k_out=None, positions=None)
    assert L.lib.mtt_b200_launch_rotate_heads(rotation(), rotate_rows(**nothing), None) == 0
    assert L.lib.mtt_b200_launch_paged_cache_append(cache(), rotation(), rotate_rows(**nothing), None) == 0
    assert L.lib.mtt_b200_launch_rotate_heads(rotation(), rotate_rows(q_heads=0, kv_heads=0), None) == 0
    assert 0 < L.lib.mtt_b200_paged_cache_workspace_size(cache(dtype=FOUR), 4, 8) < 1 << 27


# ---------------------------------------------------------------------------
# Python
# ---------------------------------------------------------------------------

def turner(**kw):
    r = rotary.Rotation(64, device="cpu", **kw)
    r._raw, r._streams = lambda index: 0, {0, 7}
    return r


def heads(rows=3, n=2, d=64, dtype=torch.bfloat16):
    return torch.zeros(rows, n, d, dtype=dtype)


@pytest.mark.parametrize("bad", [dict(head_dim=96), dict(rotary_dim=0), dict(rotary_dim=24), dict(rotary_dim=80), dict(eps=-1e-9),
                                 dict(eps=float("nan")), dict(base=0.0), dict(base=float("inf")),
                                 dict(frequencies=torch.zeros(31)), dict(frequencies=torch.zeros(32, dtype=torch.complex64)),
                                 dict(q_norm=torch.ones(32)), dict(k_norm=torch.ones(64, dtype=torch.int32))], ids=str)
def test_rotation_refuses(bad):
    with pytest.raises(ValueError):
        rotary.Rotation(**dict(dict(head_dim=64, device="cpu"), **bad))


def test_rotation_keeps_its_own():
    """Weights and frequencies are copied; frequencies in radians become turns."""
    w, f = torch.ones(64), torch.linspace(0, 1, 32)
    r = rotary.Rotation(64, frequencies=f, q_norm=w, device="cpu")
    assert torch.allclose(r.turns * 2 * torch.pi, f.double())
    w.zero_()
    assert (r.q_norm == 1).all() and r.k_norm is None
    assert rotary.Rotation(128, 32, base=7.0, device="cpu").turns.shape == (16,)


POS = torch.zeros(3, dtype=torch.int32)


@pytest.mark.parametrize("args,kw", [
    ((None, None, POS), {}), ((heads(), heads(4), POS), {}), ((heads(), None, POS[:2]), {}), ((heads(), None, POS.long()), {}),
    ((heads(), None, torch.zeros(6, dtype=torch.int32)[::2]), {}), ((heads(d=128), None, POS), {}),
    ((heads(dtype=torch.float32), None, POS), {}), ((heads(), heads(dtype=torch.float16), POS), {}),
    ((heads()[0], None, POS), {}), ((heads(n=4)[:, ::2], None, POS), {}), ((heads(d=65)[..., 1:], None, POS), {}),
    ((heads(), None, POS), dict(k_out=heads())), ((heads(), None, POS), dict(q_out=heads(4))),
    ((heads(), None, POS), dict(q_out=heads(dtype=torch.float16))),
    ((heads(), None, POS), dict(stream=types.SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=7)))],
    ids=range(15))
def test_rotate_refuses(lib, args, kw):  # noqa: F811
    with pytest.raises(ValueError):
        turner().rotate(*args, **kw)
    assert lib.calls == []


def test_calls_are_made_on_the_tensors_device(lib):  # noqa: F811
    cache, r = on_host(), turner()
    kv = heads()
    r.rotate(kv, kv, POS)
    cache.append(0, kv, kv, kv, r)
    cache.append(1, None, kv, kv, r, positions=POS)
    cache.load(3, layer=0)
    cache.load(3)
    assert [d for _, d in lib.calls] == [HOST] * 5 and lib.device == 0
    stream = types.SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=7)
    for call in (lambda: cache.append(0, kv, kv, kv, r, q_out=kv, stream=stream),
                 lambda: cache.load(3, layer=0, k=kv, v=kv, stream=stream)):
        with pytest.raises(ValueError):
            call()
    assert len(lib.calls) == 5


@pytest.mark.parametrize("call", [
    lambda c, r: c.append(2, heads(), heads(), heads(), r), lambda c, r: c.append(0, heads(4), heads(), heads(), r),
    lambda c, r: c.append(0, heads(), heads(n=3), heads(n=3), r), lambda c, r: c.append(0, heads(), heads(), heads(2), r),
    lambda c, r: c.append(0, heads(n=129), heads(), heads(), r), lambda c, r: c.append(0, heads(4), heads(4), heads(4), r),
    lambda c, r: c.append(0, heads(dtype=torch.float16), heads(), heads(), r),
    lambda c, r: c.append(0, None, heads(), heads(), r, q_out=heads()),
    lambda c, r: c.append(0, heads(), heads(), heads(), r, q_out=heads(2)),
    lambda c, r: c.append(0, heads(), heads(), heads(), r, positions=POS.long()),
    lambda c, r: c.append(0, heads(), heads(), heads(), r, offsets=POS),
    lambda c, r: c.append(0, heads(), heads(), heads(), rotary.Rotation(128, device="cpu")),
    lambda c, r: c.load(4, layer=0), lambda c, r: c.load(-1), lambda c, r: c.load(3, layer=2), lambda c, r: c.load(3, layer=0, k=heads()),
    lambda c, r: c.load(2, layer=0, k=heads(), v=heads()), lambda c, r: c.load(3, layer=0, k=heads(n=3), v=heads(n=3))],
    ids=range(18))
def test_append_and_load_refuse(lib, call):  # noqa: F811
    with pytest.raises(ValueError):
        call(on_host(), turner())
    assert lib.calls == []


def test_overlapping_rows_are_not_written(lib):  # noqa: F811
    """Outputs whose rows (or layers) share memory are refused; inputs may be broadcast."""
    cache, r = on_host(), turner()
    one, x = heads(1).expand(3, 2, 64), heads()
    layers = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16).expand(2, 3, 2, 64)
    for call in (lambda: r.rotate(x, None, POS, q_out=one), lambda: r.rotate(x, x, POS, k_out=one),
                 lambda: cache.append(0, x, x, x, r, q_out=one), lambda: cache.load(3, layer=0, k=one, v=x),
                 lambda: cache.load(3, layer=0, k=x, v=one), lambda: cache.load(3, k=layers, v=torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            call()
    assert lib.calls == []
    r.rotate(one, one, POS)
    cache.append(0, one, one, one, r)
    rows = torch.zeros(3, 2, 2, 64, dtype=torch.bfloat16).transpose(0, 1)  # layers side by side in a row
    cache.load(3, k=rows, v=rows)
    assert len(lib.calls) == 3


def test_4bit_pools_are_looked_at():
    """Without a GPU a cache cannot be made; that a pool is on a CUDA device is the first thing asked for."""
    pool = torch.zeros(2, 1, 2, 1, 16, 36, dtype=torch.uint8)
    i32 = torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(ValueError):
        pc.PagedCache(pool, i32, i32[:, 0], i32[:, 0], dtype=torch.bfloat16)
    for bad in (dict(bits=8), dict(bits=4, head_dim=80)):
        with pytest.raises(ValueError):
            pc.PagedCache.allocate(**dict(dict(pages=2, slots=2, max_tokens=16, layers=1, kv_heads=1, head_dim=64, device="cpu"), **bad))
