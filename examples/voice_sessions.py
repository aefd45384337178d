"""Many speech sessions from a few prefilled voices, on one paged cache.

    python examples/voice_sessions.py [--sessions 64] [--steps 48] [--window 64]

The decoder here is the self-attention part of the Main Decoder's layers (its
width, heads and weights; LayerNorm and projections in torch): what matters is
how the cache is used.

1. Two voices, each with a conditional and an unconditional row, are prefilled:
   218 tokens each, keys and values stored layer by layer, prompt attention.
2. Every session is forked from a voice: two slots that share the voice's full
   pages and own a copy of its last, partial one.
3. Decode steps: room for one token in every open slot, its keys and values,
   attention in which each voice's prefix is read once for all its sessions.
   With a window only the voice and the last tokens stay visible, so a step's
   cost no longer grows with the speech.
4. Halfway, every second session ends: its slots are closed, the pool is
   compacted, and new sessions take their place.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from magpie_tts_rt_b200.main_decoder import HEADS, HEAD_DIM, REFERENCE_PREFIX, WIDTH, make_main_decoder_weights  # noqa: E402
from magpie_tts_rt_b200.paged_cache import PagedCache, PrefixGroups  # noqa: E402


class VoiceServer:
    """Slots 0..3: voices 0 and 1, conditional and unconditional rows; session
    i: slots 4 + 2 i (conditional) and 5 + 2 i."""

    def __init__(self, sessions: int, max_tokens: int, layers: int = 4, window: int = 0, seed: int = 0, page_size=16):
        self.sessions, self.layers, self.window = sessions, layers, window
        slots = 4 + 2 * sessions
        # the voices once, and for each slot its own tokens and a copy of a partial page
        pages = 4 * -(-REFERENCE_PREFIX // page_size) + 2 * sessions * (2 + (max_tokens - REFERENCE_PREFIX) // page_size)
        self.cache = PagedCache.allocate(pages, slots, max_tokens, layers, HEADS, HEAD_DIM, page_size)
        self.weights = make_main_decoder_weights(seed, positions=8, layers=layers).to(device="cuda")
        self.open = [False] * sessions
        self.voice = [0] * sessions
        self.groups = None

    def _slots(self, values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device="cuda")

    def _layer(self, x, layer, attend, store):
        """One layer for rows x [rows, 768]: q, k, v views of one product, no copies."""
        w = self.weights
        y = torch.nn.functional.layer_norm(x, (WIDTH,), w.ln_self[layer])
        qkv = (y @ w.qkv[layer].T).view(-1, 3 * HEADS, HEAD_DIM)
        store(qkv[:, HEADS:2 * HEADS], qkv[:, 2 * HEADS:], layer)
        return x + attend(layer, qkv[:, :HEADS]).reshape(-1, WIDTH) @ w.o[layer].T

    def prefill(self, tokens: torch.Tensor) -> torch.Tensor:
        """tokens [4, 218, 768]: the voices' rows."""
        n = tokens.shape[1]
        counts = [n] * 4 + [0] * (2 * self.sessions)
        offsets = [0]
        for c in counts:
            offsets.append(offsets[-1] + c)
        offsets = self._slots(offsets)
        self.cache.extend(self._slots(counts))
        x = tokens.reshape(-1, WIDTH)
        for layer in range(self.layers):
            x = self._layer(x, layer, lambda l, q: self.cache.attend(l, q, offsets=offsets),
                            lambda k, v, l: self.cache.store(k, v, layer=l, offsets=offsets))
        return x.view(4, n, WIDTH)

    def start(self, sessions, voices) -> None:
        """Opens sessions (numbers) with voices (0 or 1 each)."""
        source = [-1] * self.cache.slots
        for s, v in zip(sessions, voices):
            source[4 + 2 * s], source[5 + 2 * s] = 2 * v, 2 * v + 1
            self.open[s], self.voice[s] = True, v
        self.cache.fork(self._slots(source))
        self._regroup()

    def end(self, sessions) -> None:
        mask = [False] * self.cache.slots
        for s in sessions:
            mask[4 + 2 * s] = mask[5 + 2 * s] = True
            self.open[s] = False
        self.cache.free(self._slots(mask, torch.bool))
        self.cache.compact()
        self._regroup()

    def _regroup(self) -> None:
        rows = [(2 * v + r, REFERENCE_PREFIX, [4 + 2 * s + r for s in range(self.sessions)
                                               if self.open[s] and self.voice[s] == v])
                for v in range(2) for r in range(2)]
        self.groups = PrefixGroups(self.cache, rows, q_heads=HEADS)
        one_more = [0] * 4 + [1 if self.open[s // 2] else 0 for s in range(2 * self.sessions)]
        self.one_more = self._slots(one_more)
        # rows of the voices themselves store nothing: their last tokens are shared pages or already there
        self.live = self._slots([s for s, n in enumerate(one_more) if n], torch.int64)
        self.offsets = self._slots([sum(one_more[:s]) for s in range(len(one_more) + 1)])

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """x [slots, 768]: one token's input per slot (closed slots' rows are ignored)."""
        self.cache.extend(self.one_more)
        sinks = REFERENCE_PREFIX if self.window else 0
        for layer in range(self.layers):
            x = self._layer(x, layer,
                            lambda l, q: self.cache.attend_shared(l, q, self.groups, window=self.window, sinks=sinks),
                            lambda k, v, l: self.cache.store(k[self.live], v[self.live], layer=l, offsets=self.offsets))
        return x


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--sessions", type=int, default=64)
    ap.add_argument("--steps", type=int, default=48)
    ap.add_argument("--window", type=int, default=64)
    a = ap.parse_args()
    server = VoiceServer(a.sessions, REFERENCE_PREFIX + a.steps + 1, window=a.window)
    g = torch.Generator(device="cuda").manual_seed(1)
    draw = lambda *s: torch.randn(*s, WIDTH, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    server.prefill(draw(4, REFERENCE_PREFIX))
    server.start(range(a.sessions), [s % 2 for s in range(a.sessions)])
    x = draw(server.cache.slots)
    for step in range(a.steps):
        if step == a.steps // 2:
            server.end(range(0, a.sessions, 2))
            print(f"step {step}: every second session ended, {int(server.cache.live)} of {server.cache.pages} pages in use")
            server.start(range(0, a.sessions, 4), [1] * len(range(0, a.sessions, 4)))
        x = server.step(x)
    torch.cuda.synchronize()
    assert (server.cache.status == 0).all(), "a call was refused"
    lengths = server.cache.lengths.tolist()
    print(f"{sum(server.open)} sessions open, tokens per slot {min(lengths[4:])}..{max(lengths[4:])}, "
          f"outputs {'finite' if torch.isfinite(x.float()).all() else 'NOT FINITE'}")


if __name__ == "__main__":
    main()
