"""The voice-sessions example end to end against dense attention in 64 bits:
prefill, fork, shared-prefix steps with a window, sessions closed and reopened,
compaction between steps."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


class Dense:
    """Each slot's keys and values as plain lists of rows, per layer, on the CPU."""

    def __init__(self, slots, layers):
        self.k = [[[] for _ in range(slots)] for _ in range(layers)]
        self.v = [[[] for _ in range(slots)] for _ in range(layers)]

    def copy(self, to, source):
        for kv in (self.k, self.v):
            for layer in kv:
                layer[to] = list(layer[source])

    def attend(self, layer, slot, q, pos, window, sinks):
        j = torch.arange(pos + 1)
        if window:
            j = j[(pos - j < window) | (j < sinks)]
        k = torch.stack(self.k[layer][slot])[j].double()
        v = torch.stack(self.v[layer][slot])[j].double()
        p = torch.softmax(torch.einsum("hd,khd->hk", q.double(), k) * q.shape[-1] ** -0.5, -1)
        return torch.einsum("hk,khd->hd", p, v), torch.einsum("hk,khd->hd", p, v.abs())


@pytest.mark.parametrize("window", [0, 24])
def test_sessions_against_dense_attention(window):
    """Layer by layer: the attention that the server's rows got equals dense
    attention over the keys and values that it stored for those slots.  The
    tolerance is that of one attention call (tests/test_gpu_paged_cache.py)."""
    from voice_sessions import REFERENCE_PREFIX, WIDTH, VoiceServer
    from magpie_tts_rt_b200.main_decoder import HEAD_DIM, HEADS

    layers, sessions = 2, 6
    server = VoiceServer(sessions, REFERENCE_PREFIX + 32, layers=layers, window=window)
    cache = server.cache
    dense = Dense(cache.slots, layers)
    g = torch.Generator().manual_seed(3)
    seen = []

    def watch(name):
        call = getattr(cache, name)

        def wrapped(layer, q, *args, **kw):
            out = call(layer, q, *args, **kw)
            seen.append((layer, q.cpu(), out.cpu()))
            return out
        setattr(cache, name, wrapped)

    store = cache.store

    def watched_store(k, v, layer=None, offsets=None):
        at = offsets.tolist()
        for s in range(cache.slots):
            for r in range(at[s], at[s + 1]):
                dense.k[layer][s].append(k[r].cpu())
                dense.v[layer][s].append(v[r].cpu())
        store(k, v, layer=layer, offsets=offsets)

    watch("attend")
    watch("attend_shared")
    cache.store = watched_store

    def check(rows, window, sinks):
        for layer, q, out in seen:
            for row, slot, pos in rows:
                ref, weight = dense.attend(layer, slot, q[row], pos, window, sinks)
                tol = 1.1 * 2.0 ** -8 * (ref.abs() + weight) + 1e-4
                assert ((out[row].double() - ref).abs() <= tol).all(), (layer, row)
        seen.clear()

    draw = lambda *s: torch.randn(*s, WIDTH, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    server.prefill(draw(4, REFERENCE_PREFIX))
    n = REFERENCE_PREFIX
    check([(v * n + p, v, p) for v in range(4) for p in (0, 1, 100, n - 1)], 0, 0)
    server.start(range(sessions), [s % 2 for s in range(sessions)])
    for s in range(sessions):
        for r in range(2):
            dense.copy(4 + 2 * s + r, 2 * (s % 2) + r)
    x = draw(cache.slots)
    for step in range(30):
        if step == 20:
            server.end([1, 2, 5])
            server.start([1, 5], [0, 0])
            for s in (1, 5):
                for r in range(2):
                    dense.copy(4 + 2 * s + r, r)
        x = server.step(x)
        if step in (0, 5, 19, 20, 29):
            lengths = cache.lengths.tolist()
            live = [s for s in range(4, cache.slots) if lengths[s]]
            assert len(live) == (12 if step < 20 else 10)
            check([(s, s, lengths[s] - 1) for s in live], window, REFERENCE_PREFIX if window else 0)
        seen.clear()
    assert (cache.status == 0).all()
    assert HEADS * HEAD_DIM == WIDTH


def test_example_runs(capsys, monkeypatch):
    import voice_sessions
    monkeypatch.setattr(sys, "argv", ["voice_sessions.py", "--sessions", "8", "--steps", "12", "--window", "16"])
    voice_sessions.main()
    assert "outputs finite" in capsys.readouterr().out
