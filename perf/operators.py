"""Workloads of the paged key/value cache and of the attention that reads it.

Four operators, as a serving program calls them (``magpie_tts_rt_b200.paged_cache``):

* ``step``    attention of one new token per slot over its cached tokens, with an optional
              sliding window and a few first tokens that stay visible (a decode step);
* ``prompt``  the same for runs of new tokens of each slot, causal (prefill, continued prefill);
* ``shared``  one new token per slot where groups of slots share a long prefix (sessions
              started from one prefilled voice), the prefix computed once for the group;
* ``pages``   closing, forking, extending, storing and compacting: the cache's own upkeep
              between decode steps.

The cache is one pool of pages ``[pages, layers, 2, kv_heads, page_size, head_dim]`` (keys at
index 0, values at 1), a table of page numbers per slot (-1: none), a length per slot and a
reference count per page.

With ``own`` false every operator is computed in its plain form (elementary torch operations
in 32 bits, rounded once at the end); with ``own`` true by the framework's kernels.
"""
import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# --------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------

def listed():
    return [
        # one session (its two CFG rows) near the decoder's cache capacity: one layer's latency
        dict(name="step_one_session", op="step", dtype="bf16", slots=2, q_heads=12, kv_heads=12, head_dim=64,
             page_size=16, layers=2, low=450, high=467, window=0, sinks=0, masked=False, idle=0),
        # 256 sessions of long speech: the 218-token voice prefix stays visible, the rest slides;
        # some keys masked, a few slots closed
        dict(name="step_sessions", op="step", dtype="bf16", slots=512, q_heads=12, kv_heads=12, head_dim=64,
             page_size=16, layers=1, low=218, high=2048, window=1024, sinks=218, masked=True, idle=16),
        # few very long caches with shared key heads: the split over the long axis
        dict(name="step_long", op="step", dtype="f16", slots=8, q_heads=32, kv_heads=8, head_dim=128,
             page_size=64, layers=1, low=30001, high=65536, window=0, sinks=0, masked=False, idle=0),
        # the prefill of one voice prefix of the decoder's own size
        dict(name="prompt_voice", op="prompt", dtype="bf16", slots=1, q_heads=12, kv_heads=12, head_dim=64,
             page_size=16, layers=2, low=218, high=218, context=0, window=0, sinks=0, masked=False),
        # ragged continued prompts of many sessions, windowed, with masked keys and a slot that sees nothing
        dict(name="prompt_ragged", op="prompt", dtype="f16", slots=24, q_heads=12, kv_heads=12, head_dim=64,
             page_size=16, layers=1, low=1, high=509, context=1531, window=512, sinks=16, masked=True),
        # one long prompt with shared key heads: the arithmetic bound
        dict(name="prompt_long", op="prompt", dtype="bf16", slots=1, q_heads=32, kv_heads=8, head_dim=128,
             page_size=64, layers=1, low=8192, high=8192, context=0, window=0, sinks=0, masked=False),
        # four sessions (eight CFG rows) of one voice: the smallest group
        dict(name="shared_one_voice", op="shared", dtype="bf16", voices=1, members=8, q_heads=12, kv_heads=12,
             head_dim=64, page_size=16, layers=1, prefix=208, low=1, high=249, window=0, sinks=0),
        # 1024 sessions with CFG rows over four voices, each row 1 to 249 tokens past its voice
        dict(name="shared_sessions", op="shared", dtype="bf16", voices=4, members=512, q_heads=12, kv_heads=12,
             head_dim=64, page_size=16, layers=1, prefix=208, low=1, high=249, window=192, sinks=208),
        # a long common context with shared key heads
        dict(name="shared_long", op="shared", dtype="f16", voices=1, members=64, q_heads=32, kv_heads=8,
             head_dim=128, page_size=64, layers=1, prefix=32768, low=1, high=2001, window=0, sinks=0),
        # one session opened from a voice, all decoder layers: the upkeep's latency
        dict(name="pages_one_session", op="pages", dtype="bf16", voices=2, children=2, kv_heads=12, head_dim=64,
             page_size=16, layers=12, prefix=218, low=1, high=3),
        # 128 sessions opened, advanced, half of them closed, the pool compacted
        dict(name="pages_sessions", op="pages", dtype="bf16", voices=8, children=256, kv_heads=12, head_dim=64,
             page_size=16, layers=12, prefix=218, low=1, high=40),
        # large pages of shared key heads, long stores
        dict(name="pages_large", op="pages", dtype="f16", voices=4, children=96, kv_heads=8, head_dim=128,
             page_size=64, layers=8, prefix=1001, low=33, high=513),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["step", "prompt", "shared", "pages"])
    dtype = rng.choice(["bf16", "f16"])
    head_dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 12])
    q_heads = kv * rng.choice([1, 1, 2, 3, 4, 6, 8])
    page_size = rng.choice([16, 32, 64])
    common = dict(op=op, dtype=dtype, kv_heads=kv, head_dim=head_dim, page_size=page_size)
    if op == "pages":
        layers = _log(rng, 1, 12)
        voices, children = _log(rng, 1, 8), _log(rng, 1, 256)
        prefix, high = _log(rng, 1, 1001), _log(rng, 1, 513)
        per_token = layers * 2 * kv * head_dim * 2
        while (voices * prefix + children * (page_size + high)) * per_token > 1.5e9:
            children = max(1, children // 2)
            high = max(1, high * 2 // 3)
        return dict(common, layers=layers, voices=voices, children=children, prefix=prefix, low=_log(rng, 1, high),
                    high=high)
    common.update(q_heads=q_heads, layers=rng.choice([1, 2]))
    if op == "step":
        slots, high = _log(rng, 1, 512), _log(rng, 1, 65536)
        while slots * high * kv * head_dim * 4 > 1.2e9:
            slots, high = max(1, slots * 2 // 3), max(1, high * 4 // 5)
        window = rng.choice([0, 0, _log(rng, 1, 4096)])
        return dict(common, slots=slots, low=_log(rng, 1, high), high=high, window=window,
                    sinks=_log(rng, 1, 256) if window else 0, masked=rng.random() < 0.3, idle=rng.choice([0, 0, 7]))
    if op == "prompt":
        slots, high, context = _log(rng, 1, 32), _log(rng, 1, 4096), _log(rng, 1, 8192) - 1
        while slots * q_heads * high * (high + context) > 1.5e9:
            slots, high, context = max(1, slots // 2), max(1, high * 4 // 5), context * 4 // 5
        window = rng.choice([0, 0, _log(rng, 1, 2048)])
        return dict(common, slots=slots, low=_log(rng, 1, high), high=high, context=context, window=window,
                    sinks=_log(rng, 1, 256) if window else 0, masked=rng.random() < 0.3)
    voices, members = _log(rng, 1, 8), _log(rng, 1, 512)
    prefix, high = page_size * _log(rng, 1, 32768 // page_size), _log(rng, 1, 2001)
    while voices * members * (prefix + high) * kv * head_dim > 1.5e9:
        members, prefix = max(1, members // 2), max(page_size, prefix * 2 // 3 // page_size * page_size)
    window = rng.choice([0, _log(rng, 1, 512)])
    return dict(common, voices=voices, members=members, prefix=prefix, low=_log(rng, 1, high), high=high, window=window,
                sinks=prefix if window else 0)


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
    n = case["slots"]
    new = spread(case["low"], case["high"], n)
    context = (np.arange(n) * 7 % n) * case["context"] // max(1, n - 1) if n > 1 else np.array([case["context"]])
    return new, context


def _seen(length, first, window, sinks):
    """How many keys each query at positions first..length-1 sees."""
    p = np.arange(first, length, dtype=np.int64)
    if not window:
        return p + 1
    low = np.maximum(p + 1 - window, 0)
    return p + 1 - low + np.minimum(sinks, low)


def work(case):
    size, d = 2, case["head_dim"]
    if case["op"] == "pages":
        token = case["layers"] * 2 * case["kv_heads"] * d * size  # one token's keys and values of all layers
        c, ps = case["children"], case["page_size"]
        stored = int(spread(case["low"], case["high"], c).sum())
        copied = c * (case["prefix"] % ps)
        # half of the children's pages stay, and half of those lie past the live count
        pages = c * (case["prefix"] % ps > 0) + stored // ps
        return {"bytes": 2.0 * token * (stored + copied + pages * ps / 4), "flops": 0.0}
    key = 2 * case["kv_heads"] * d * size
    row = 2 * case["q_heads"] * d * size
    pair = 4.0 * case["q_heads"] * d
    if case["op"] == "step":
        lengths = _step_lengths(case)
        seen = sum(int(_seen(t, t - 1, case["window"], case["sinks"])[0]) for t in lengths if t)
        return {"bytes": float(seen * key + len(lengths) * row), "flops": pair * seen}
    if case["op"] == "prompt":
        new, context = _prompt_lengths(case)
        pairs = read = 0
        for m, c in zip(new, context):
            s = _seen(c + m, c, case["window"], case["sinks"])
            pairs += int(s.sum())
            read += int(min(c + m, s[0] + m - 1 + (case["sinks"] if case["window"] else 0)))
        return {"bytes": float(read * key + int(new.sum()) * row), "flops": pair * pairs}
    n = case["voices"] * case["members"]
    suffix = spread(case["low"], case["high"], n)
    if case["window"]:
        suffix = np.minimum(suffix, case["window"])
    keys = case["voices"] * case["prefix"] + int(suffix.sum())
    n += case["voices"]  # a voice's own slot has a row too
    return {"bytes": float(keys * key + n * row), "flops": pair * (n * case["prefix"] + int(suffix.sum()))}


# --------------------------------------------------------------------------------------
# what a serving program has in hand before the call
# --------------------------------------------------------------------------------------

def _pool(case, pages, gen):
    shape = (pages, case["layers"], 2, case["kv_heads"], case["page_size"], case["head_dim"])
    return torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=gen)


def _cuda(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(device="cuda", dtype=dtype)


def _own_cache(state):
    from magpie_tts_rt_b200.paged_cache import PagedCache
    return PagedCache(pool=state["pool"], page_table=state["page_table"], lengths=state["lengths"], refs=state["refs"])


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "pages":
        return _prepare_pages(case, rng, gen)
    ps = case["page_size"]
    state = dict(op=case["op"], layer=case["layers"] - 1, window=case["window"], sinks=case["sinks"], key_mask=None)
    shared_pages = 0
    if case["op"] == "step":
        lengths = rng.permutation(_step_lengths(case))
        rows = len(lengths)
    elif case["op"] == "prompt":
        new, context = _prompt_lengths(case)
        order = rng.permutation(len(new))
        new, context = new[order], context[order]
        lengths = new + context
        offsets = np.concatenate([[0], np.cumsum(new)])
        rows = int(offsets[-1])
        state.update(offsets=_cuda(offsets), longest=int(new.max()))
    else:
        # slots: the voices, then their members, dealt out in turn
        voices, members = case["voices"], case["members"]
        shared_pages = case["prefix"] // ps
        suffix = rng.permutation(spread(case["low"], case["high"], voices * members))
        lengths = np.concatenate([np.full(voices, case["prefix"]), case["prefix"] + suffix])
        voice_of = np.concatenate([np.arange(voices), np.arange(voices * members) % voices])
        rows = len(lengths)
    need = -(-lengths // ps)
    table_pages = int(max(need.max(), 1))
    table = np.full((len(lengths), table_pages), -1, np.int64)
    private = need - shared_pages
    if shared_pages:
        private[:voices] = need[:voices]
    total = int(private.sum())
    pages = total + total // 8 + 1
    order = rng.permutation(pages)
    first = np.concatenate([[0], np.cumsum(private)])
    for i in range(len(lengths)):
        mine = order[first[i]:first[i + 1]]
        if shared_pages and i >= voices:
            table[i, :shared_pages] = table[voice_of[i], :shared_pages]
            table[i, shared_pages:shared_pages + len(mine)] = mine
        else:
            table[i, :len(mine)] = mine
    refs = np.bincount(table[table >= 0], minlength=pages)
    dtype = DTYPES[case["dtype"]]
    q = torch.empty(rows, case["q_heads"], case["head_dim"], dtype=torch.float32, device="cuda").normal_(generator=gen)
    state.update(pool=_pool(case, pages, gen), page_table=_cuda(table), lengths=_cuda(lengths), refs=_cuda(refs),
                 q=(1.5 * q).to(dtype), longest_key=int(lengths.max()))
    if case.get("masked"):
        mask = rng.random((len(lengths), table_pages * ps)) < 0.9
        if len(lengths) > 3:
            mask[3] = False                                     # a slot whose rows see nothing
            mask[1, :int(lengths[1]) // 2] = False              # a padded beginning
        state["key_mask"] = _cuda(mask, torch.bool)
    if own:
        cache = state["cache"] = _own_cache(state)
        if case["op"] == "shared":
            from magpie_tts_rt_b200.paged_cache import PrefixGroups
            groups = [(v, case["prefix"], np.flatnonzero(voice_of == v).tolist()) for v in range(voices)]
            state["groups"] = PrefixGroups(cache, groups, q_heads=case["q_heads"])
    return state


def _prepare_pages(case, rng, gen):
    ps, voices, children = case["page_size"], case["voices"], case["children"]
    prefix = case["prefix"]
    voice_pages = -(-prefix // ps)
    counts = rng.permutation(spread(case["low"], case["high"], children))
    slots = voices + children
    table_pages = -(-(prefix + case["high"]) // ps) + 1
    live = voices * voice_pages
    pages = live + children + int((-(-(prefix % ps + counts) // ps)).sum()) + 1
    table = np.full((slots, table_pages), -1, np.int64)
    table[:voices, :voice_pages] = rng.permutation(live).reshape(voices, voice_pages)
    lengths = np.concatenate([np.full(voices, prefix), np.zeros(children, np.int64)])
    refs = np.concatenate([np.ones(live, np.int64), np.zeros(pages - live, np.int64)])
    child = np.arange(slots) >= voices
    source = np.where(child, rng.integers(0, voices, slots), -1)
    extend = np.concatenate([np.zeros(voices, np.int64), counts])
    offsets = np.concatenate([[0], np.cumsum(extend)])
    dtype = DTYPES[case["dtype"]]
    kv = torch.empty(2, case["layers"], int(offsets[-1]), case["kv_heads"], case["head_dim"], dtype=dtype,
                     device="cuda").normal_(generator=gen)
    state = dict(op="pages", pool=_pool(case, pages, gen), page_table=_cuda(table), lengths=_cuda(lengths),
                 refs=_cuda(refs), closing=_cuda(child, torch.bool), source=_cuda(source), counts=_cuda(extend),
                 offsets=_cuda(offsets), k=kv[0], v=kv[1], ended=_cuda(child & (np.arange(slots) % 2 == 0), torch.bool))
    if own:
        state["cache"] = _own_cache(state)
    return state


# --------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "pages":
        return _plain_pages(state)
    if state["op"] == "prompt":
        return _plain_prompt(state)
    pos = state["lengths"].long()[:, None] - 1
    out, lse = _plain_attention(state, state["q"][:, None], pos)
    return {"out": out[:, 0].to(state["q"].dtype), "lse": lse[:, 0]}


def _run_own(state):
    cache = state["cache"]
    if state["op"] == "pages":
        cache.free(state["closing"])
        cache.fork(state["source"])
        cache.extend(state["counts"])
        cache.store(state["k"], state["v"], offsets=state["offsets"])
        cache.free(state["ended"])
        cache.compact()
        return {"pool": cache.pool, "page_table": cache.page_table, "lengths": cache.lengths, "refs": cache.refs}
    if state["op"] == "shared":
        out, lse = cache.attend_shared(state["layer"], state["q"], state["groups"], window=state["window"],
                                       sinks=state["sinks"], return_lse=True)
    else:
        out, lse = cache.attend(state["layer"], state["q"], offsets=state.get("offsets"), window=state["window"],
                                sinks=state["sinks"], key_mask=state["key_mask"], return_lse=True)
    return {"out": out, "lse": lse}


def _plain_attention(state, q, pos):
    """q [slots, m, q_heads, D], pos [slots, m] (below 0: no such row) -> out [slots, m, q_heads, D], lse, in f32."""
    pool, layer = state["pool"], state["layer"]
    n, m, heads, d = q.shape
    hkv, ps = pool.shape[3], pool.shape[4]
    used = -(-max(state["longest_key"], 1) // ps)
    kv = pool[:, layer][state["page_table"][:, :used].long().clamp(min=0)]     # [n, pages, 2, hkv, ps, D]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, n, hkv, used * ps, d)
    j = torch.arange(used * ps, device=q.device)
    there = j < state["lengths"].long()[:, None]                               # [n, keys]
    if state["key_mask"] is not None:
        there = there & state["key_mask"][:, :used * ps]
    seen = there[:, None] & (j <= pos[..., None])                              # [n, m, keys]
    if state["window"]:
        seen = seen & ((pos[..., None] - j < state["window"]) | (j < state["sinks"]))
    k = kv[0].float()
    qg = q.float().reshape(n, m, hkv, heads // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    s = torch.matmul(qg, k.transpose(2, 3)).reshape(n, hkv, heads // hkv, m, used * ps)
    del k
    s = (s * d ** -0.5).masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    e = s.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    v = kv[1].float().masked_fill(~there[:, None, :, None], 0.0)
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


def _ranked(free, need, able):
    """Which of the slots in order get their new pages, lowest free page first: (granted, first page's rank)."""
    need = torch.where(able, need, torch.zeros_like(need))
    upto = need.cumsum(0)
    return able & ((need == 0) | (upto <= free.numel())), upto - need


def _plain_free(state, mask):
    table, refs = state["page_table"], state["refs"]
    gone = table[mask].long()
    gone = gone[gone >= 0]
    refs.sub_(torch.bincount(gone, minlength=refs.numel()).to(refs.dtype))
    table[mask] = -1
    state["lengths"][mask] = 0


def _plain_fork(state, source):
    pool, table, refs, lengths = state["pool"], state["page_table"], state["refs"], state["lengths"]
    ps, slots = pool.shape[4], table.shape[0]
    d = torch.arange(slots, device=table.device)
    able = (source >= 0) & (source < slots) & (source != d)
    src = source.long().clamp(0, slots - 1)
    new_len = lengths[src].long()
    free = (refs == 0).nonzero()[:, 0]
    granted, rank = _ranked(free, (new_len % ps != 0).long(), able)
    rows = table[src].clone()
    old = table[granted].long()
    part = granted & (new_len % ps != 0)
    at = new_len[part] // ps
    fresh = free[rank[part]]
    pool[fresh] = pool[rows[part, at].long()]
    rows[part, at] = fresh.to(rows.dtype)
    got = rows[granted].long()
    refs.add_(torch.bincount(got[got >= 0], minlength=refs.numel()).to(refs.dtype))
    refs.sub_(torch.bincount(old[old >= 0], minlength=refs.numel()).to(refs.dtype))
    table[granted] = rows[granted]
    lengths[granted] = new_len[granted].to(lengths.dtype)


def _plain_extend(state, counts):
    table, refs, lengths, ps = state["page_table"], state["refs"], state["lengths"], state["pool"].shape[4]
    have = -(-lengths.long() // ps)
    want = -(-(lengths + counts).long() // ps)
    able = (counts >= 0) & (want <= table.shape[1])
    free = (refs == 0).nonzero()[:, 0]
    granted, rank = _ranked(free, want - have, able)
    column = torch.arange(table.shape[1], device=table.device)
    new = granted[:, None] & (column >= have[:, None]) & (column < want[:, None])
    page = free[(rank[:, None] + column - have[:, None])[new]]
    table[new] = page.to(table.dtype)
    refs[page] = 1
    lengths.add_(torch.where(granted, counts, torch.zeros_like(counts)))


def _plain_store(state, k, v, offsets):
    pool, ps = state["pool"], state["pool"].shape[4]
    offsets = offsets.long()
    row = torch.arange(k.shape[1], device=k.device)
    slot = torch.searchsorted(offsets, row, right=True) - 1
    pos = state["lengths"].long()[slot] - offsets[slot + 1] + row
    page = state["page_table"][slot, pos // ps].long()
    pool[page, :, 0, :, pos % ps] = k.transpose(0, 1)
    pool[page, :, 1, :, pos % ps] = v.transpose(0, 1)


def _plain_compact(state):
    pool, table, refs = state["pool"], state["page_table"], state["refs"]
    used = refs > 0
    page = torch.arange(refs.numel(), device=refs.device)
    live = used.sum()
    moved = (used & (page >= live)).nonzero()[:, 0]
    holes = (~used & (page < live)).nonzero()[:, 0]
    pool[holes] = pool[moved]
    refs[holes] = refs[moved]
    refs[moved] = 0
    to = page.clone()
    to[moved] = holes
    table.copy_(torch.where(table >= 0, to[table.long().clamp(min=0)].to(table.dtype), table))


def _plain_pages(state):
    _plain_free(state, state["closing"])
    _plain_fork(state, state["source"])
    _plain_extend(state, state["counts"])
    _plain_store(state, state["k"], state["v"], state["offsets"])
    _plain_free(state, state["ended"])
    _plain_compact(state)
    return {"pool": state["pool"], "page_table": state["page_table"], "lengths": state["lengths"], "refs": state["refs"]}


# --------------------------------------------------------------------------------------
# the definitions, in 64 bits
# --------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "pages":
        return _exact_pages(state)
    table, lengths = state["page_table"].cpu().numpy(), state["lengths"].cpu().numpy()
    q, pool, layer = state["q"], state["pool"], state["layer"]
    hkv, ps, d = pool.shape[3], pool.shape[4], pool.shape[5]
    group = q.shape[1] // hkv
    offsets = state["offsets"].cpu().numpy() if case["op"] == "prompt" else np.arange(len(lengths) + 1)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=q.device)
    for i, length in enumerate(lengths):
        a, b = int(offsets[i]), int(offsets[i + 1])
        if length == 0 or b == a:
            continue
        j = np.arange(length)
        where = _cuda(table[i][j // ps], torch.int64), _cuda(j % ps, torch.int64)
        pos = _cuda(length - (b - a) + np.arange(b - a), torch.int64)[:, None]
        key = _cuda(j, torch.int64)[None]
        see = key <= pos
        if case["window"]:
            see &= (key > pos - case["window"]) | (key < case["sinks"])
        if state["key_mask"] is not None:
            see &= state["key_mask"][i, :int(length)]
        heads_at_once = hkv if (b - a) * length * q.shape[1] < 5e7 else 1
        for h in range(0, hkv, heads_at_once):
            hs = slice(h, h + heads_at_once)
            k = pool[where[0], layer, 0, hs, where[1]].double().transpose(0, 1)        # [h, keys, D]
            v = pool[where[0], layer, 1, hs, where[1]].double().transpose(0, 1)
            rows = slice(h * group, (h + heads_at_once) * group)
            x = q[a:b, rows].double().reshape(b - a, heads_at_once, group, d)
            score = torch.einsum("mhgd,hkd->mhgk", x, k) / d ** 0.5
            score = torch.where(see[:, None, None], score, torch.full_like(score, float("-inf")))
            some = see.any(1)[:, None, None, None]
            p = torch.where(some, torch.softmax(score, -1), torch.zeros_like(score))
            out[a:b, rows] = torch.einsum("mhgk,hkd->mhgd", p, v).reshape(b - a, -1, d)
            lse[a:b, rows] = torch.logsumexp(score, -1).reshape(b - a, -1)
    return {"out": out, "lse": lse}


def _exact_pages(state):
    """The pass page by page with lists and sets; None where the pool is large."""
    pool = state["pool"]
    if pool.numel() > 3e7:
        return None
    data = pool.double().cpu().numpy().copy()
    rows = [[int(p) for p in r if p >= 0] for r in state["page_table"].cpu().numpy()]
    lengths = [int(t) for t in state["lengths"].cpu().numpy()]
    k, v = state["k"].double().cpu().numpy(), state["v"].double().cpu().numpy()
    closing, ended = state["closing"].cpu().numpy(), state["ended"].cpu().numpy()
    source, counts, offsets = (state[x].cpu().numpy() for x in ("source", "counts", "offsets"))
    pages, ps = data.shape[0], data.shape[4]

    def close(mask):
        for i in np.flatnonzero(mask):
            rows[i], lengths[i] = [], 0

    def lowest(taken):
        return next(p for p in range(pages) if p not in taken)

    def taken():
        return {p for r in rows for p in r}

    close(closing)
    used, before, old_lengths = taken(), [list(r) for r in rows], list(lengths)
    for i, s in enumerate(source):
        if 0 <= s != i:
            rows[i], lengths[i] = list(before[s]), old_lengths[s]
            if lengths[i] % ps:
                p = lowest(used)
                used.add(p)
                data[p] = data[rows[i][-1]]
                rows[i][-1] = p
    used = taken()
    for i, c in enumerate(counts):
        lengths[i] += int(c)
        while len(rows[i]) * ps < lengths[i]:
            rows[i].append(lowest(used))
            used.add(rows[i][-1])
        for r in range(offsets[i], offsets[i + 1]):
            t = lengths[i] - int(offsets[i + 1]) + r
            data[rows[i][t // ps], :, 0, :, t % ps] = k[:, r]
            data[rows[i][t // ps], :, 1, :, t % ps] = v[:, r]
    close(ended)
    used = taken()
    to = dict(zip(sorted(p for p in used if p >= len(used)), (p for p in range(len(used)) if p not in used)))
    for p, hole in to.items():
        data[hole] = data[p]
    rows = [[to.get(p, p) for p in r] for r in rows]
    table = np.full(tuple(state["page_table"].shape), -1, np.int64)
    refs = np.zeros(pages, np.int64)
    for i, r in enumerate(rows):
        table[i, :len(r)] = r
        for p in r:
            refs[p] += 1
    return {"pool": torch.from_numpy(data), "page_table": torch.from_numpy(table),
            "lengths": torch.tensor(lengths), "refs": torch.from_numpy(refs)}
