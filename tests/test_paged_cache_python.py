"""The Python side of the paged cache without a GPU: on which device its calls
are made.  The library is a stand-in that notes each call, the tensors are on
the CPU."""
import types

import pytest
import torch

from magpie_tts_rt_b200 import paged_cache as pc

HOST = -1  # the index that tensors on the CPU report


class Library:
    """Notes (call, device current at it)."""

    def __init__(self):
        self.calls, self.device = [], 0

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_size"):
                return 256
            self.calls.append((name, self.device))
            return pc.L.STATUS_OK
        return call


@pytest.fixture
def lib(monkeypatch):
    lib = Library()

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, lib.device = lib.device, self.index

        def __exit__(self, *exc):
            lib.device = self.before

    monkeypatch.setattr(pc.L, "lib", lib)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(pc, "_current_device", lambda: lib.device, raising=False)
    return lib


def on_host(slots=3, pages=4, layers=2, heads=2, ps=16, d=64):
    cache = pc.PagedCache.__new__(pc.PagedCache)
    cache.pool = torch.zeros(pages, layers, 2, heads, ps, d, dtype=torch.bfloat16)
    cache.device, cache._index, cache._raw, cache.dtype = torch.device("cpu"), HOST, lambda index: 0, torch.bfloat16
    cache.pages, cache.layers, cache.kv_heads, cache.page_size, cache.head_dim = pages, layers, heads, ps, d
    cache.slots, cache.table_pages, cache._scale = slots, 2, d ** -0.5
    cache._c = pc.L.PagedCache()
    cache._ref = pc.ctypes.byref(cache._c)
    cache._streams, cache._spaces, cache._outgrown = {0, 7}, {}, []
    cache._keep = lambda stream, *tensors: None     # a matter of CUDA memory
    return cache


def every_call(cache, stream=None):
    """The public calls that launch something."""
    i32 = torch.zeros(cache.slots, dtype=torch.int32)
    kv = torch.zeros(cache.slots, cache.kv_heads, cache.head_dim, dtype=torch.bfloat16)
    groups = pc.PrefixGroups(cache, [(0, 16, [1, 2])], q_heads=cache.kv_heads)
    return [lambda: cache.extend(i32, stream=stream), lambda: cache.fork(i32, stream=stream),
            lambda: cache.free(i32.bool(), stream=stream), lambda: cache.compact(stream=stream),
            lambda: cache.store(kv, kv, layer=0, stream=stream), lambda: cache.attend(0, kv, stream=stream),
            lambda: cache.attend_shared(0, kv, groups, stream=stream)]


@pytest.mark.parametrize("call", range(7))
def test_calls_are_made_on_the_pools_device(lib, call):
    """Another device is current: each launch is made with the pool's, and the other is current again after it."""
    every_call(on_host())[call]()
    assert len(lib.calls) == 1 and lib.calls[0][1] == HOST
    assert lib.device == 0


@pytest.mark.parametrize("call", range(7))
def test_streams_of_another_device_are_refused(lib, call):
    stream = types.SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=7)
    with pytest.raises(ValueError):
        every_call(on_host(), stream)[call]()
    assert lib.calls == []


@pytest.mark.parametrize("window,sinks,groups,shared", [
    (0, 0, 3, 16 * 2 + 48 * 3 + 96 * 1), (9, 96, 3, 16 * 2 + 48 * 3 + 96 * 1), (9, 95, 3, 16 * 2 + 48 * 3),
    (9, 48, 3, 16 * 2 + 48 * 3), (9, 16, 3, 16 * 2), (9, 15, 0, None), (9, 0, 0, None), (0, 15, 3, 16 * 2 + 48 * 3 + 96 * 1)])
@pytest.mark.parametrize("known", [True, False])
def test_groups_that_a_window_does_not_share(lib, monkeypatch, window, sinks, groups, shared, known):
    """The prefix pass is asked for by the groups that it can serve: those whose prefix is among the sinks."""
    cache = on_host(slots=8)
    cache.table_pages = 8
    plan = pc.PrefixGroups(cache, [(0, 50, [1, 2, 3]), (0, 16, [4, 5]), (0, 96, [6]), (0, 7, [7])], q_heads=2)
    if not known:
        plan._c.shared_tokens = 0
    seen = []
    monkeypatch.setattr(cache, "_call", lambda name, *args: seen.append(args[2]._obj))
    q = torch.zeros(8, 2, 64, dtype=torch.bfloat16)
    cache.attend_shared(0, q, plan, window=window, sinks=sinks)
    assert seen[0].n_groups == groups
    if groups:
        assert seen[0].shared_tokens == (shared if known else 0) and seen[0].n_members == 6
        assert [getattr(seen[0], f) for f in ("voice", "tokens", "offsets", "members")] == [
            getattr(plan._c, f) for f in ("voice", "tokens", "offsets", "members")]


@pytest.mark.parametrize("value", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 63 - 1, 2 ** 70])
@pytest.mark.parametrize("name", ["window", "sinks"])
def test_windows_past_32_bits(lib, monkeypatch, name, value):
    """A window or number of sinks that no slot reaches is all of a slot, however large it is given."""
    cache = on_host()
    seen = []
    monkeypatch.setattr(cache, "_call", lambda call, *args: seen.append(args[1]._obj))
    cache.attend(0, torch.zeros(3, 2, 64, dtype=torch.bfloat16), **{name: value})
    assert getattr(seen[0], name) >= 1 << 30
