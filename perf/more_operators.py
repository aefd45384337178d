"""Workloads of position rotation, of the append that rotates, and of the cache held in 4 bits.

Five operators, as a serving program calls them (``magpie_tts_rt_b200.rotary`` and
``magpie_tts_rt_b200.paged_cache``):

* ``rotate``   norms of the queries and keys of each head and their position rotation, in one pass;
* ``append``   the same on the way into a 16-bit paged cache: keys normed, rotated and stored with
               their values, queries normed and rotated;
* ``store4``   keys and values stored in 4 bits, and read back as the values they stand for;
* ``step4``    attention of one new token per slot over a cache held in 4 bits (a decode step);
* ``prompt4``  the same for runs of new tokens of each slot, causal.

Rotation: dims i and i + rotary_dim / 2 (or 2 i and 2 i + 1, ``interleaved``) of a head are turned
by position * base^(-2 i / rotary_dim); dims past rotary_dim stay.  The norm before it is
x / sqrt(mean x^2 + eps) * weight over a head.

The 4-bit format: 64 dims of a token's head share a (step, low) pair of the cache's 16-bit type,
value = low + step * code, code 0..15; low is the smallest of the 64, step the spread / 15, and the
code is chosen in single precision: rint((x - low) * (1 / step)).  A block (page, layer, keys or
values, head) of the pool [pages, layers, 2, kv_heads, page_size, head_dim / 2 + head_dim / 16]
bytes holds the codes of its page_size tokens, then their pairs.  Every 8 dims are a 32-bit word: the
codes of dims 0, 2, 4, 6, then those of 1, 3, 5, 7, from the lowest bits up.

With ``own`` false every operator is computed in its plain form (elementary torch operations
in 32 bits, rounded once at the end); with ``own`` true by the framework's kernels.
"""
import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
GROUP = 64


# --------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------

def listed():
    return [
        # one session (its two CFG rows), one layer of a decode step: latency
        dict(name="rotate_one_session", op="rotate", dtype="bf16", rows=2, q_heads=12, kv_heads=12, head_dim=64,
             rotary_dim=64, interleaved=False, base=1e4, norm=True, far=467),
        # a long prompt with shared key heads, queries and keys views of one projection's rows
        dict(name="rotate_prompt", op="rotate", dtype="bf16", rows=8192, q_heads=32, kv_heads=8, head_dim=128,
             rotary_dim=128, interleaved=False, base=5e5, norm=True, far=131072),
        # one session's decode step into the cache
        dict(name="append_one_session", op="append", dtype="bf16", slots=2, q_heads=12, kv_heads=12, head_dim=64,
             page_size=16, rotary_dim=64, interleaved=False, base=1e4, norm=True, low=450, high=467, idle=0, prompt=False,
             given=False),
        # 512 slots' decode step, a few of them closed; no norms, half of each head turned
        dict(name="append_sessions", op="append", dtype="bf16", slots=512, q_heads=12, kv_heads=12, head_dim=64,
             page_size=16, rotary_dim=32, interleaved=True, base=1e4, norm=False, low=8, high=512, idle=16, prompt=False,
             given=False),
        # ragged prompts of 24 slots on large pages, shared key heads
        dict(name="append_prompts", op="append", dtype="f16", slots=24, q_heads=32, kv_heads=8, head_dim=128,
             page_size=64, rotary_dim=128, interleaved=False, base=1e6, norm=True, low=1, high=2001, idle=0, prompt=True,
             given=False),
        # one session's decode step, every layer of the decoder at once
        dict(name="store4_one_session", op="store4", dtype="bf16", slots=2, kv_heads=12, head_dim=64, page_size=16,
             layers=12, low=1, high=1, context=450),
        # prompts of 96 slots, several layers at once
        dict(name="store4_prompts", op="store4", dtype="f16", slots=96, kv_heads=8, head_dim=128, page_size=64,
             layers=8, low=33, high=513, context=101),
        # one session near the decoder's cache capacity: one layer's latency
        dict(name="step4_one_session", op="step4", dtype="bf16", slots=2, q_heads=12, kv_heads=12, head_dim=64,
             page_size=16, layers=2, low=450, high=467, window=0, sinks=0, masked=False, idle=0),
        # 256 sessions of long speech: the 218-token voice prefix stays visible, the rest slides;
        # some keys masked, a few slots closed
        dict(name="step4_sessions", op="step4", dtype="bf16", slots=512, q_heads=12, kv_heads=12, head_dim=64,
             page_size=16, layers=1, low=218, high=2048, window=1024, sinks=218, masked=True, idle=16),
        # few very long caches with shared key heads: the split over the long axis
        dict(name="step4_long", op="step4", dtype="f16", slots=8, q_heads=32, kv_heads=8, head_dim=128,
             page_size=64, layers=1, low=30001, high=65536, window=0, sinks=0, masked=False, idle=0),
        # ragged continued prompts of many sessions, windowed, with masked keys and a slot that sees nothing
        dict(name="prompt4_ragged", op="prompt4", dtype="f16", slots=24, q_heads=12, kv_heads=12, head_dim=64,
             page_size=16, layers=1, low=1, high=509, context=1531, window=512, sinks=16, masked=True),
        # one long prompt with shared key heads: the arithmetic bound
        dict(name="prompt4_long", op="prompt4", dtype="bf16", slots=1, q_heads=32, kv_heads=8, head_dim=128,
             page_size=64, layers=1, low=8192, high=8192, context=0, window=0, sinks=0, masked=False),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["rotate", "append", "store4", "step4", "prompt4"])
    head_dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 12])
    q_heads = kv * rng.choice([1, 1, 2, 3, 4, 6, 8])
    common = dict(op=op, dtype=rng.choice(["bf16", "f16"]), kv_heads=kv, head_dim=head_dim)
    if op in ("rotate", "append"):
        common.update(q_heads=q_heads, rotary_dim=16 * rng.randint(1, head_dim // 16), interleaved=rng.random() < 0.5,
                      base=rng.choice([1e4, 5e5, 1e6]), norm=rng.random() < 0.6)
    if op == "rotate":
        return dict(common, rows=_log(rng, 1, max(1, 8192 * 40 * 128 // ((q_heads + kv) * head_dim * 2))),
                    far=_log(rng, 1, 1 << 20))
    page_size = rng.choice([16, 32, 64])
    common.update(page_size=page_size)
    if op == "append":
        prompt = rng.random() < 0.5
        slots, high = _log(rng, 1, 64 if prompt else 512), _log(rng, 1, 2001 if prompt else 512)
        while slots * (high + page_size) * (kv + q_heads) * head_dim > 1e8:
            slots, high = max(1, slots * 2 // 3), max(1, high * 4 // 5)
        return dict(common, slots=slots, low=_log(rng, 1, high), high=high, idle=0 if prompt else rng.choice([0, 7]),
                    prompt=prompt, given=rng.random() < 0.3)
    if op == "store4":
        layers = _log(rng, 1, 12)
        slots, high, context = _log(rng, 1, 96), _log(rng, 1, 513), _log(rng, 1, 200) - 1
        while slots * (high + context + page_size) * layers * kv * head_dim > 1e8:
            slots, high = max(1, slots * 2 // 3), max(1, high * 4 // 5)
        return dict(common, layers=layers, slots=slots, low=_log(rng, 1, high), high=high, context=context)
    common.update(q_heads=q_heads, layers=rng.choice([1, 2]))
    window = rng.choice([0, 0, _log(rng, 1, 4096 if op == "step4" else 2048)])
    common.update(window=window, sinks=_log(rng, 1, 256) if window else 0, masked=rng.random() < 0.3)
    if op == "step4":
        slots, high = _log(rng, 1, 512), _log(rng, 1, 65536)
        while slots * high * kv * head_dim * 4 > 1.2e9:
            slots, high = max(1, slots * 2 // 3), max(1, high * 4 // 5)
        return dict(common, slots=slots, low=_log(rng, 1, high), high=high, idle=rng.choice([0, 0, 7]))
    slots, high, context = _log(rng, 1, 32), _log(rng, 1, 4096), _log(rng, 1, 8192) - 1
    while slots * q_heads * high * (high + context) > 1.5e9:
        slots, high, context = max(1, slots // 2), max(1, high * 4 // 5), context * 4 // 5
    return dict(common, slots=slots, low=_log(rng, 1, high), high=high, context=context)


def spread(low, high, n):
    """n whole numbers from low to high, even over their logarithm: the same for every seed."""
    if n == 1:
        return np.array([high], np.int64)
    return np.rint(low * (high / low) ** (np.arange(n) / (n - 1))).astype(np.int64)


def _step_lengths(case):
    lengths = spread(case["low"], case["high"], case["slots"])
    if case["idle"]:
        lengths[case["idle"] // 2::case["idle"]] = 0
    return lengths


def _prompt_lengths(case):
    """New tokens of each slot, and those it had before."""
    n = case["slots"]
    new = spread(case["low"], case["high"], n)
    most = case.get("context", case.get("high", 0))
    context = (np.arange(n) * 7 % n) * most // max(1, n - 1) if n > 1 else np.array([most])
    return new, context


def _seen(length, first, window, sinks):
    """How many keys each query at positions first..length-1 sees."""
    p = np.arange(first, length, dtype=np.int64)
    if not window:
        return p + 1
    low = np.maximum(p + 1 - window, 0)
    return p + 1 - low + np.minimum(sinks, low)


def token_bytes(head_dim):
    """Of one token's keys, or values, of one head in 4 bits."""
    return head_dim // 2 + 4 * (head_dim // GROUP)


def work(case):
    kv, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "rotate":
        heads = case["q_heads"] + kv
        return {"bytes": float(case["rows"] * (heads * d * 4 + 4)), "flops": 7.0 * case["rows"] * heads * d}
    if case["op"] == "append":
        rows = int(_prompt_lengths(case)[0].sum()) if case["prompt"] else int((_step_lengths(case) > 0).sum())
        return {"bytes": float(rows * (case["q_heads"] + 2 * kv) * d * 4),
                "flops": 7.0 * rows * (case["q_heads"] + kv) * d}
    if case["op"] == "store4":
        # keys and values in, their 4 bits out, and the values that these stand for
        n = case["layers"] * int(_prompt_lengths(case)[0].sum()) * 2 * kv
        return {"bytes": float(n * (4 * d + token_bytes(d))), "flops": 6.0 * n * d}
    key = 2 * kv * token_bytes(d)
    row = 2 * case["q_heads"] * d * 2
    pair = 4.0 * case["q_heads"] * d
    if case["op"] == "step4":
        lengths = _step_lengths(case)
        seen = sum(int(_seen(t, t - 1, case["window"], case["sinks"])[0]) for t in lengths if t)
        return {"bytes": float(seen * key + len(lengths) * row), "flops": pair * seen}
    new, context = _prompt_lengths(case)
    pairs = read = 0
    for m, c in zip(new, context):
        s = _seen(c + m, c, case["window"], case["sinks"])
        pairs += int(s.sum())
        read += int(min(c + m, s[0] + m - 1 + (case["sinks"] if case["window"] else 0)))
    return {"bytes": float(read * key + int(new.sum()) * row), "flops": pair * pairs}


# --------------------------------------------------------------------------------------
# what a serving program has in hand before the call
# --------------------------------------------------------------------------------------

def _cuda(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(device="cuda", dtype=dtype)


def _normal(gen, *shape):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=gen)


def _channels(gen, *shape):
    """Keys and values as projections leave them: some dims of a head are larger than others, some off zero."""
    return torch.exp(0.5 * _normal(gen, *shape)), 0.5 * _normal(gen, *shape)


def _pages(rng, lengths, page_size):
    """Shuffled pages for slots of these lengths: (page_table, pages in the pool)."""
    need = -(-lengths // page_size)
    table = np.full((len(lengths), int(max(need.max(), 1))), -1, np.int64)
    pages = int(need.sum()) + int(need.sum()) // 8 + 1
    order = rng.permutation(pages)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, pages


def _rotation(state, case, gen):
    d, dtype = case["head_dim"], DTYPES[case["dtype"]]
    state.update(rotary_dim=case["rotary_dim"], interleaved=case["interleaved"], base=case["base"], q_norm=None, k_norm=None)
    if case["norm"]:
        state["q_norm"], state["k_norm"] = ((1 + 0.2 * _normal(gen, d)).to(dtype) for _ in range(2))
    if own:
        from magpie_tts_rt_b200.rotary import Rotation
        state["rotation"] = Rotation(d, rotary_dim=case["rotary_dim"], base=case["base"], interleaved=case["interleaved"],
                                     q_norm=state["q_norm"], k_norm=state["k_norm"], eps=EPS)


def _projection(state, case, rows, gen):
    """q, k, v: views of one product's rows."""
    h, kv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    size, off = _channels(gen, h + 2 * kv, d)
    y = (_normal(gen, rows, h + 2 * kv, d) * size + off).to(DTYPES[case["dtype"]])
    state.update(q=y[:, :h], k=y[:, h:h + kv], v=y[:, h + kv:])


def _pool4(case, pages, gen):
    """A pool in 4 bits, every page filled, a piece at a time."""
    layers, kv, ps, d = case["layers"], case["kv_heads"], case["page_size"], case["head_dim"]
    size, off = _channels(gen, layers, 2, kv, 1, d)
    pool = torch.empty(pages, layers, 2, kv, ps, token_bytes(d), dtype=torch.uint8, device="cuda")
    step = max(1, int(2e8) // (layers * 2 * kv * ps * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = _normal(gen, n, layers, 2, kv, ps, d).mul_(size).add_(off).to(DTYPES[case["dtype"]])
        codes, pairs = _quantised(x)
        _blocks(pool[p:p + n]).copy_(torch.cat([_packed(codes).flatten(-2), _raw(pairs).flatten(-3)], -1))
    return pool


def _blocks(pool):
    return pool.view(*pool.shape[:4], -1)


def _raw(pairs):
    """The bytes of (step, low) pairs [..., groups, 2]."""
    return pairs.contiguous().view(torch.uint8)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    state = dict(op=op)
    if op == "rotate":
        _rotation(state, case, gen)
        _projection(state, case, case["rows"], gen)
        state["positions"] = _cuda(rng.integers(0, case["far"], case["rows"]))
        return state
    ps, d, kv = case["page_size"], case["head_dim"], case["kv_heads"]
    state.update(offsets=None)
    if op == "step4" or (op == "append" and not case["prompt"]):
        lengths = rng.permutation(_step_lengths(case))
        rows = len(lengths)
    else:
        new, context = _prompt_lengths(case)
        order = rng.permutation(len(new))
        new, context = new[order], context[order]
        lengths = new + context
        offsets = np.concatenate([[0], np.cumsum(new)])
        rows = int(offsets[-1])
        state.update(offsets=_cuda(offsets), longest=int(new.max()))
    table, pages = _pages(rng, lengths, ps)
    state.update(page_table=_cuda(table), lengths=_cuda(lengths), rows=rows,
                 refs=_cuda(np.bincount(table[table >= 0], minlength=pages)), longest_key=int(lengths.max()))
    if op == "append":
        _rotation(state, case, gen)
        _projection(state, case, rows, gen)
        state["pool"] = _normal(gen, pages, 1, 2, kv, ps, d).to(dtype)
        state["positions"] = _cuda(rng.integers(0, 1 << 20, rows)) if case["given"] else None
    elif op == "store4":
        size, off = _channels(gen, 2, case["layers"], 1, kv, d)
        y = (_normal(gen, 2, case["layers"], rows, kv, d) * size + off).to(dtype)
        state.update(k=y[0], v=y[1], head_dim=d,
                     pool=torch.zeros(pages, case["layers"], 2, kv, ps, token_bytes(d), dtype=torch.uint8, device="cuda"))
    else:
        state.update(layer=case["layers"] - 1, window=case["window"], sinks=case["sinks"], key_mask=None,
                     pool=_pool4(case, pages, gen), q=(1.5 * _normal(gen, rows, case["q_heads"], d)).to(dtype))
        if case["masked"]:
            mask = rng.random((len(lengths), table.shape[1] * ps)) < 0.9
            if len(lengths) > 3:
                mask[3] = False                                     # a slot whose rows see nothing
                mask[1, :int(lengths[1]) // 2] = False              # a padded beginning
            state["key_mask"] = _cuda(mask, torch.bool)
    if own:
        from magpie_tts_rt_b200.paged_cache import PagedCache
        state["cache"] = PagedCache(pool=state["pool"], page_table=state["page_table"], lengths=state["lengths"],
                                    refs=state["refs"], dtype=dtype)
    return state


# --------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------

def run(state):
    op = state["op"]
    if own:
        return _run_own(state)
    if op == "rotate":
        return {"q": _plain_rotate(state, state["q"], state["q_norm"], state["positions"]),
                "k": _plain_rotate(state, state["k"], state["k_norm"], state["positions"])}
    if op == "append":
        return _plain_append(state)
    if op == "store4":
        return _plain_store(state)
    if op == "prompt4":
        return _plain_prompt(state)
    pos = state["lengths"].long()[:, None] - 1
    out, lse = _plain_attention(state, state["q"][:, None], pos)
    return {"out": out[:, 0].to(state["q"].dtype), "lse": lse[:, 0]}


def _run_own(state):
    op = state["op"]
    if op == "rotate":
        q, k = state["rotation"].rotate(state["q"], state["k"], state["positions"])
        return {"q": q, "k": k}
    cache = state["cache"]
    if op == "append":
        q = cache.append(0, state["q"], state["k"], state["v"], state["rotation"], offsets=state["offsets"],
                         positions=state["positions"])
        return {"q": q, "pool": cache.pool}
    if op == "store4":
        cache.store(state["k"], state["v"], offsets=state["offsets"])
        k, v = cache.load(state["rows"], offsets=state["offsets"])
        return {"k": k, "v": v}
    out, lse = cache.attend(state["layer"], state["q"], offsets=state["offsets"], window=state["window"],
                            sinks=state["sinks"], key_mask=state["key_mask"], return_lse=True)
    return {"out": out, "lse": lse}


def _plain_rotate(state, x, weight, positions):
    rot, d = state["rotary_dim"], x.shape[-1]
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    i = torch.arange(rot // 2, device=x.device)
    angle = positions.double()[:, None] * state["base"] ** (-2.0 * i.double() / rot)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    first, second = (2 * i, 2 * i + 1) if state["interleaved"] else (i, i + rot // 2)
    out = y.clone()
    out[..., first] = y[..., first] * cos - y[..., second] * sin
    out[..., second] = y[..., second] * cos + y[..., first] * sin
    return out.to(x.dtype)


def _places(state):
    """Of each row: its slot and position (-1: no such token)."""
    lengths = state["lengths"].long()
    row = torch.arange(state["rows"], device=lengths.device)
    if state["offsets"] is None:
        return row, lengths - 1
    offsets = state["offsets"].long()
    slot = torch.searchsorted(offsets, row, right=True) - 1
    return slot, lengths[slot] - offsets[slot + 1] + row


def _plain_append(state):
    pool, ps = state["pool"], state["pool"].shape[4]
    slot, pos = _places(state)
    at = pos if state["positions"] is None else state["positions"].long()
    there = pos >= 0
    q = _plain_rotate(state, state["q"], state["q_norm"], at)
    k = _plain_rotate(state, state["k"], state["k_norm"], at)
    page = state["page_table"][slot, pos.clamp(min=0) // ps].long()[there]
    pool[page, 0, 0, :, pos[there] % ps] = k[there]
    pool[page, 0, 1, :, pos[there] % ps] = state["v"][there]
    return {"q": torch.where(there[:, None, None], q, torch.zeros_like(q)), "pool": pool}


def _quantised(x):
    """(codes [..., d] uint8, pairs [..., groups, 2] of x's type)."""
    g = x.unflatten(-1, (-1, GROUP)).float()
    low, high = torch.aminmax(g, dim=-1)
    step = ((high - low) / torch.full_like(low, 15)).to(x.dtype)
    inverse = torch.where(step == 0, torch.zeros_like(low), 1 / step.float())
    code = torch.round((g - low[..., None]) * inverse[..., None]).clamp_(0, 15).to(torch.uint8)
    return code.flatten(-2), torch.stack([step, low.to(x.dtype)], -1)


def _packed(codes):
    c = codes.unflatten(-1, (-1, 4, 2)).transpose(-1, -2).flatten(-2)      # of each 8: 0, 2, 4, 6, 1, 3, 5, 7
    return (c[..., 0::2] | c[..., 1::2] << 4).flatten(-2)


def _unpacked(blocks, ps, d, dtype):
    """blocks [..., bytes] -> values [..., ps, d] in f32."""
    codes = blocks[..., :ps * d // 2].unflatten(-1, (ps, d // 2))
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    codes = codes.unflatten(-1, (-1, 2, 4)).transpose(-1, -2).flatten(-3)
    pairs = blocks[..., ps * d // 2:].contiguous().view(dtype).unflatten(-1, (ps, d // GROUP, 2)).float()
    values = codes.unflatten(-1, (-1, GROUP)).float()
    return values.mul_(pairs[..., 0:1]).add_(pairs[..., 1:2]).flatten(-2)


def _plain_store(state):
    pool, d = state["pool"], state["head_dim"]
    blocks, ps, layers, kv = _blocks(pool), pool.shape[4], pool.shape[1], pool.shape[3]
    slot, pos = _places(state)
    page = state["page_table"][slot, pos // ps].long()
    t = pos % ps
    place = page[:, None, None, None], torch.arange(layers, device=page.device)[:, None, None], \
        torch.arange(kv, device=page.device)[None, :, None]
    code_at = t[:, None, None, None] * (d // 2) + torch.arange(d // 2, device=page.device)
    pair_at = ps * d // 2 + t[:, None, None, None] * (d // 16) + torch.arange(d // 16, device=page.device)
    for n, x in enumerate((state["k"], state["v"])):
        codes, pairs = _quantised(x.transpose(0, 1))                       # [rows, layers, kv, ...]
        blocks[place[0], place[1], n, place[2], code_at] = _packed(codes)
        blocks[place[0], place[1], n, place[2], pair_at] = _raw(pairs).flatten(-2)
    out = []
    for n in range(2):
        got = torch.cat([blocks[place[0], place[1], n, place[2], at] for at in (code_at, pair_at)], -1)
        out.append(_unpacked(got, 1, d, state["k"].dtype)[..., 0, :].transpose(0, 1).to(state["k"].dtype))
    return {"k": out[0], "v": out[1]}


def _plain_attention(state, q, pos):
    """q [slots, m, q_heads, D], pos [slots, m] (below 0: no such row) -> out [slots, m, q_heads, D], lse, in f32."""
    pool, layer = state["pool"], state["layer"]
    n, m, heads, d = q.shape
    hkv, ps = pool.shape[3], pool.shape[4]
    used = -(-max(state["longest_key"], 1) // ps)
    blocks = _blocks(pool)[:, layer][state["page_table"][:, :used].long().clamp(min=0)]    # [n, pages, 2, hkv, bytes]
    blocks = blocks.permute(2, 0, 3, 1, 4)
    k = _unpacked(blocks[0], ps, d, q.dtype).reshape(n, hkv, used * ps, d)
    j = torch.arange(used * ps, device=q.device)
    there = j < state["lengths"].long()[:, None]                               # [n, keys]
    if state["key_mask"] is not None:
        there = there & state["key_mask"][:, :used * ps]
    seen = there[:, None] & (j <= pos[..., None])                              # [n, m, keys]
    if state["window"]:
        seen = seen & ((pos[..., None] - j < state["window"]) | (j < state["sinks"]))
    qg = q.float().reshape(n, m, hkv, heads // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    s = torch.matmul(qg, k.transpose(2, 3)).reshape(n, hkv, heads // hkv, m, used * ps)
    del k
    s = (s * d ** -0.5).masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    e = s.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    v = _unpacked(blocks[1], ps, d, q.dtype).reshape(n, hkv, used * ps, d).masked_fill_(~there[:, None, :, None], 0.0)
    o = torch.matmul(e.reshape(n, hkv, -1, used * ps), v).reshape(n, hkv, heads // hkv, m, d)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + total.log())[..., 0]
    return o.permute(0, 3, 1, 2, 4).reshape(n, m, heads, d), lse.permute(0, 3, 1, 2).reshape(n, m, heads)


def _plain_prompt(state):
    q, offsets, m = state["q"], state["offsets"].long(), state["longest"]
    counts = offsets[1:] - offsets[:-1]
    i = torch.arange(m, device=q.device)
    row = (offsets[:-1, None] + i).clamp(max=q.shape[0] - 1)
    real = i < counts[:, None]
    pos = torch.where(real, state["lengths"].long()[:, None] - counts[:, None] + i, torch.full_like(row, -1))
    out, lse = _plain_attention(state, q[row], pos)
    return {"out": out[real].to(q.dtype), "lse": lse[real]}


# --------------------------------------------------------------------------------------
# the definitions, in 64 bits
# --------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotate":
        at = state["positions"]
        return {"q": _turned(case, state["q"], state["q_norm"], at), "k": _turned(case, state["k"], state["k_norm"], at)}
    if case["op"] == "append":
        return _exact_append(case, state)
    if case["op"] == "store4":
        return {"k": _stands_for(state["k"]), "v": _stands_for(state["v"])}
    return _exact_attention(case, state)


def _turned(case, x, weight, at):
    """Each pair of dims as a complex number, times e^(i angle)."""
    rot = case["rotary_dim"]
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.double()
    head, rest = y[..., :rot], y[..., rot:]
    pair = head.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    frequency = torch.tensor([case["base"] ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.ones_like(frequency).expand(len(at), -1), at.double()[:, None] * frequency)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn[:, None])
    z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, rest], -1)


def _exact_append(case, state):
    table, lengths = state["page_table"].cpu().numpy(), state["lengths"].cpu().numpy()
    ps = case["page_size"]
    offsets = np.arange(len(lengths) + 1) if state["offsets"] is None else state["offsets"].cpu().numpy()
    at = np.zeros(state["rows"], np.int64)
    pages, places, rows = [], [], []
    for i, length in enumerate(lengths):
        if length == 0:
            continue
        for r in range(offsets[i], offsets[i + 1]):
            t = int(length) - int(offsets[i + 1]) + r
            at[r] = t
            rows.append(r)
            pages.append(int(table[i, t // ps]))
            places.append(t % ps)
    at = _cuda(at, torch.int64) if state["positions"] is None else state["positions"]
    rows, pages, places = (torch.tensor(x, device="cuda", dtype=torch.int64) for x in (rows, pages, places))
    q = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    q[rows] = _turned(case, state["q"][rows], state["q_norm"], at[rows])
    pool = state["pool"].double()
    pool[pages, 0, 0, :, places] = _turned(case, state["k"][rows], state["k_norm"], at[rows])
    pool[pages, 0, 1, :, places] = state["v"][rows].double()
    return {"q": q, "pool": pool}


def _stands_for(x):
    """What 4 bits hold of x.  Pair and code are fixed by the format in x's type and in single precision: every operation
    is carried out in 64 bits and rounded to those."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for l in range(x.shape[0]):
        g = x[l].double().reshape(*x.shape[1:-1], -1, GROUP)
        low = g.min(-1, keepdim=True).values
        step = ((g.max(-1, keepdim=True).values - low).float().double() / 15).to(x.dtype).double()
        inverse = torch.where(step > 0, step.reciprocal().float().double(), step)
        code = ((g - low).float().double() * inverse).float().double().round().clamp(0, 15)
        out[l] = (low + step * code).reshape(x.shape[1:])
    return out


def _held(case, blocks):
    """The values of blocks [n, heads, bytes] in 64 bits: [n, heads, ps, d]."""
    ps, d = case["page_size"], case["head_dim"]
    n, h = blocks.shape[:2]
    byte = blocks[..., :ps * d // 2].reshape(n, h, ps, d // 2).long()
    code = torch.empty(n, h, ps, d, dtype=torch.float64, device=blocks.device)
    for dim, (b, above) in enumerate([(0, 1), (2, 1), (0, 16), (2, 16), (1, 1), (3, 1), (1, 16), (3, 16)]):
        code[..., dim::8] = (byte[..., b::4] // above % 16).double()
    pair = blocks[..., ps * d // 2:].contiguous().view(DTYPES[case["dtype"]]).double().reshape(n, h, ps, d // GROUP, 2)
    return pair[..., 1].repeat_interleave(GROUP, -1) + pair[..., 0].repeat_interleave(GROUP, -1) * code


def _exact_attention(case, state):
    table, lengths = state["page_table"].cpu().numpy(), state["lengths"].cpu().numpy()
    q, pool, layer = state["q"], state["pool"], state["layer"]
    hkv, ps, d = case["kv_heads"], case["page_size"], case["head_dim"]
    group = q.shape[1] // hkv
    offsets = np.arange(len(lengths) + 1) if state["offsets"] is None else state["offsets"].cpu().numpy()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=q.device)
    flat = pool.reshape(*pool.shape[:4], -1)
    for i, length in enumerate(lengths):
        a, b = int(offsets[i]), int(offsets[i + 1])
        length = int(length)
        if length == 0 or b == a:
            continue
        pages = _cuda(table[i, :-(-length // ps)], torch.int64)
        key = torch.arange(length, device=q.device)[None]
        pos = torch.arange(length - (b - a), length, device=q.device)[:, None]
        see = key <= pos
        if case["window"]:
            see &= (key > pos - case["window"]) | (key < case["sinks"])
        if state["key_mask"] is not None:
            see &= state["key_mask"][i, :length]
        heads_at_once = hkv if (b - a) * length * q.shape[1] < 5e7 else 1
        for h in range(0, hkv, heads_at_once):
            hs = slice(h, h + heads_at_once)
            k, v = (_held(case, flat[pages, layer, n, hs]).transpose(0, 1).flatten(1, 2)[:, :length] for n in range(2))
            rows = slice(h * group, (h + heads_at_once) * group)
            x = q[a:b, rows].double().reshape(b - a, heads_at_once, group, d)
            score = torch.einsum("mhgd,hkd->mhgk", x, k) / d ** 0.5
            score = torch.where(see[:, None, None], score, torch.full_like(score, float("-inf")))
            some = see.any(1)[:, None, None, None]
            p = torch.where(some, torch.softmax(score, -1), torch.zeros_like(score))
            out[a:b, rows] = torch.einsum("mhgk,hkd->mhgd", p, v).reshape(b - a, -1, d)
            lse[a:b, rows] = torch.logsumexp(score, -1).reshape(b - a, -1)
    return {"out": out, "lse": lse}
