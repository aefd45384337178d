"""Host side of the paged cache without a GPU: the C structs as the header lays
them out, the calls' refusals, and workspace sizes."""
import ctypes
import os
import subprocess

import pytest

from magpie_tts_rt_b200 import _lib as L

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STRUCTS = {"mtt_b200_paged_cache_t": L.PagedCache, "mtt_b200_cache_rows_t": L.CacheRows,
           "mtt_b200_cache_attention_t": L.CacheAttention, "mtt_b200_prefix_groups_t": L.PrefixGroups}


def test_struct_layouts(tmp_path):
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "magpie_tts_rt_b200.h"', "int main(void) {"]
    expected = []
    for name, struct in STRUCTS.items():
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


def cache(**over):
    """A cache whose addresses are never read here."""
    c = L.PagedCache(100, 2, 4, 16, 64, L.DTYPE_BF16, 8, 10, 1 << 20, 1 << 20, 1 << 20, 1 << 20, None, None)
    for k, v in over.items():
        setattr(c, k, v)
    return ctypes.byref(c)


BAD_CACHES = [dict(pages=0), dict(layers=0), dict(kv_heads=0), dict(page_size=24), dict(page_size=256), dict(head_dim=96),
              dict(dtype=2), dict(slots=0), dict(slots=16385), dict(table_pages=0), dict(pool=None), dict(pool=(1 << 20) + 64),
              dict(page_table=None), dict(lengths=None), dict(refs=None), dict(refs=(1 << 20) + 4),
              dict(table_pages=1 << 26), dict(pages=1 << 30), dict(slots=16384, table_pages=1 << 20)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches(bad):
    c = cache(**bad)
    assert L.lib.mtt_b200_paged_cache_workspace_size(c, 4, 8) == 0
    assert L.lib.mtt_b200_paged_shared_workspace_size(c, 4, 8) == 0
    ws, size = 1 << 20, 1 << 40
    assert L.lib.mtt_b200_launch_paged_cache_extend(c, 16, ws, size, None) == L.STATUS_INVALID_ARGUMENT
    assert L.lib.mtt_b200_launch_paged_cache_fork(c, 16, 0, ws, size, None) == L.STATUS_INVALID_ARGUMENT
    assert L.lib.mtt_b200_launch_paged_cache_free(c, 16, None) == L.STATUS_INVALID_ARGUMENT
    assert L.lib.mtt_b200_launch_paged_cache_compact(c, ws, size, None) == L.STATUS_INVALID_ARGUMENT
    assert L.lib.mtt_b200_launch_paged_cache_store(c, ctypes.byref(rows()), None) == L.STATUS_INVALID_ARGUMENT
    assert L.lib.mtt_b200_launch_paged_attention(c, ctypes.byref(attention()), ws, size, None) == L.STATUS_INVALID_ARGUMENT


def rows(**over):
    r = L.CacheRows(0, 1, 8, 0, 1 << 20, 1 << 20, 256, 256, 0, 0, None)
    for k, v in over.items():
        setattr(r, k, v)
    return r


def attention(**over):
    a = L.CacheAttention(0, 4, 8, 0, 0, 0.125, 1 << 20, 256, 1 << 20, 256, None, None, None, 0)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_null_arguments():
    ws, size = 1 << 20, 1 << 40
    bad = L.STATUS_INVALID_ARGUMENT
    assert L.lib.mtt_b200_paged_cache_workspace_size(None, 4, 8) == 0
    assert L.lib.mtt_b200_launch_paged_cache_extend(cache(), None, ws, size, None) == bad
    assert L.lib.mtt_b200_launch_paged_cache_extend(None, 16, ws, size, None) == bad
    assert L.lib.mtt_b200_launch_paged_cache_fork(cache(), None, 0, ws, size, None) == bad
    assert L.lib.mtt_b200_launch_paged_cache_free(cache(), None, None) == bad
    assert L.lib.mtt_b200_launch_paged_cache_store(cache(), None, None) == bad
    assert L.lib.mtt_b200_launch_paged_attention(cache(), None, ws, size, None) == bad
    assert L.lib.mtt_b200_launch_paged_attention_shared(cache(), ctypes.byref(attention()), None, ws, size, None) == bad


@pytest.mark.parametrize("bad", [dict(layer=-1), dict(layer=2), dict(n_layers=0), dict(layer=1, n_layers=2), dict(rows=-1),
                                 dict(rows=9), dict(k=None), dict(v=None), dict(k=(1 << 20) + 8), dict(k_row_stride=4),
                                 dict(v_layer_stride=3)], ids=str)
def test_bad_rows(bad):
    assert L.lib.mtt_b200_launch_paged_cache_store(cache(), ctypes.byref(rows(**bad)), None) == L.STATUS_INVALID_ARGUMENT


BAD_ATTENTION = [dict(layer=2), dict(layer=-1), dict(q_heads=0), dict(q_heads=6), dict(q_heads=260), dict(rows=-1), dict(rows=9),
                 dict(rows=(1 << 22) + 1, offsets=16), dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0),
                 dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(out=None), dict(q=(1 << 20) + 2),
                 dict(q_row_stride=12), dict(out_row_stride=4), dict(key_mask=16, mask_stride=159)]


@pytest.mark.parametrize("bad", BAD_ATTENTION, ids=str)
def test_bad_attention(bad):
    a = ctypes.byref(attention(**bad))
    ws, size = 1 << 20, 1 << 40
    assert L.lib.mtt_b200_launch_paged_attention(cache(), a, ws, size, None) == L.STATUS_INVALID_ARGUMENT
    groups = L.PrefixGroups()
    assert L.lib.mtt_b200_launch_paged_attention_shared(cache(), a, ctypes.byref(groups), ws, size,
                                                        None) == L.STATUS_INVALID_ARGUMENT


@pytest.mark.parametrize("bad", [dict(n_groups=-1), dict(n_groups=9), dict(n_members=-1), dict(n_members=(1 << 22) + 1),
                                 dict(n_groups=1, n_members=1)], ids=str)
def test_bad_groups(bad):
    groups = L.PrefixGroups()
    for k, v in bad.items():
        setattr(groups, k, v)
    assert L.lib.mtt_b200_launch_paged_attention_shared(cache(), ctypes.byref(attention()), ctypes.byref(groups), 1 << 20,
                                                        1 << 40, None) == L.STATUS_INVALID_ARGUMENT


def test_workspaces():
    size = L.lib.mtt_b200_paged_cache_workspace_size(cache(), 4, 8)
    assert 0 < size < 1 << 27
    assert L.lib.mtt_b200_paged_cache_workspace_size(cache(), 4, 1 << 16) > size
    assert L.lib.mtt_b200_paged_shared_workspace_size(cache(), 4, 8) > size
    for q_heads, n in ((0, 8), (6, 8), (260, 8), (4, -1), (4, (1 << 22) + 1)):
        assert L.lib.mtt_b200_paged_cache_workspace_size(cache(), q_heads, n) == 0
    a = ctypes.byref(attention())
    bad = L.STATUS_INVALID_ARGUMENT
    assert L.lib.mtt_b200_launch_paged_attention(cache(), a, 1 << 20, size - 1, None) == bad
    assert L.lib.mtt_b200_launch_paged_attention(cache(), a, None, size, None) == bad
    assert L.lib.mtt_b200_launch_paged_attention(cache(), a, (1 << 20) + 16, size, None) == bad
    assert L.lib.mtt_b200_launch_paged_cache_extend(cache(), 16, 1 << 20, 64, None) == bad


def test_nothing_to_do_is_done():
    assert L.lib.mtt_b200_launch_paged_attention(cache(), ctypes.byref(attention(rows=0, q=None, out=None)), None, 0, None) == 0
    assert L.lib.mtt_b200_launch_paged_cache_store(cache(), ctypes.byref(rows(rows=0, k=None, v=None)), None) == 0
