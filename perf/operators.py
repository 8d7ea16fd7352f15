"""Timing cases of windowed attention, rotated cache appends and shared-prefix decode.

A case is a dict of plain values. ``listed()`` gives the fixed ones, ``draw(rng)`` one more of the same ranges,
``prepare(case, seed)`` what a program holds before the call, ``run(state)`` one pass, ``work(case)`` the bytes and
operations that a pass cannot do without and ``exact(case, seed)`` the outputs in float64. With ``own`` false a
pass is the operators' plain form in elementary torch operations; with ``own`` true it makes the package's calls.

Kinds:
- ``decode``: one query token per sequence over a cache of one length, of which the last ``window`` tokens and the
  first ``sinks`` are visible (the registered attention's call for a sliding layer).
- ``ragged``: the same for sequences of different lengths.
- ``prefill``: a chunk of new tokens on a cache, or a whole prompt, under the same window, layer after layer.
- ``rope_append``: one sequence's new tokens go into every layer of a paged cache, their keys rotated to their
  positions on the way.
- ``paged_step``: a step of several sequences on a paged cache, layer after layer: the new tokens' keys and queries
  are rotated, the rows written, and (one token a sequence) the window attended.
- ``shared``: one query token per sequence over a prefix that all sequences share and each one's own tokens.
- ``shared_paged``: the same on a paged cache whose sequences were forked from one, layer after layer.
"""
import math

import numpy as np
import torch

own = False

D = 128
SCALE = D ** -0.5
DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
TURN = 512  # tokens that a sequence of a paged cache receives before the next one gets some


def listed():
    return [
        # The smallest call: one token of one conversation, a window of 1024 (32 query heads over 8 KV heads).
        dict(name="decode_window_1024", kind="decode", batch=1, q_heads=32, kv_heads=8, tokens=10240, window=1024,
             sinks=4, dtype="fp16"),
        # Sixteen conversations of 1k to 32k tokens, a window of 4096: some shorter than it.
        dict(name="decode_window_ragged_16", kind="ragged", batch=16, q_heads=32, kv_heads=8, tokens=32768,
             shortest=1024, window=4096, sinks=16, dtype="bf16"),
        # The engine's chunk of 2048 tokens on the 7716 that a prune kept.
        dict(name="prefill_window_chunk", kind="prefill", layers=4, batch=1, q_heads=32, kv_heads=8, queries=2048,
             past=7716, window=4096, sinks=4, dtype="fp16"),
        # A long prompt with a short window, no sinks (16 query heads over 8 KV heads, an odd length).
        dict(name="prefill_window_prompt", kind="prefill", layers=2, batch=1, q_heads=16, kv_heads=8, queries=8191,
             past=0, window=1000, sinks=0, dtype="bf16"),
        # A tool result of 333 tokens goes into every layer of a paged cache.
        dict(name="rope_append_333", kind="rope_append", layers=28, kv_heads=8, tokens=5001, queries=333,
             page_tokens=64, dtype="bf16"),
        # A prompt of 6620 tokens.
        dict(name="rope_append_6620", kind="rope_append", layers=24, kv_heads=8, tokens=100, queries=6620,
             page_tokens=64, dtype="fp16"),
        # A decode step of eight sequences at odd lengths: rotation, cache rows and windowed attention of every layer.
        dict(name="paged_step_8", kind="paged_step", layers=16, batch=8, q_heads=32, kv_heads=8, tokens=9001,
             queries=1, window=2048, sinks=4, page_tokens=64, dtype="fp16"),
        # The rotation and cache rows of a chunk of two sequences at different lengths.
        dict(name="paged_rows_2x700", kind="paged_step", layers=12, batch=2, q_heads=32, kv_heads=8, tokens=3001,
             queries=700, window=0, sinks=0, page_tokens=32, dtype="bf16"),
        # Four branches of one conversation, a short shared prompt.
        dict(name="shared_4x2000", kind="shared", batch=4, q_heads=32, kv_heads=8, prefix=2000, tokens=200,
             shortest=1, dtype="fp16"),
        # Sixty-four requests behind a long common prompt, eight query heads a KV head.
        dict(name="shared_64x16384", kind="shared", batch=64, q_heads=64, kv_heads=8, prefix=16384, tokens=1500,
             shortest=100, dtype="bf16"),
        # Twenty-four forked sequences on pages, every layer of a token.
        dict(name="shared_paged_24", kind="shared_paged", layers=12, batch=24, q_heads=32, kv_heads=8, prefix=8200,
             tokens=900, shortest=30, page_tokens=64, dtype="fp16"),
    ]


def _span(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["decode", "ragged", "prefill", "prefill", "rope_append", "paged_step", "paged_step", "shared",
                       "shared", "shared_paged"])
    q_heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 8), (8, 8), (64, 8), (8, 2), (16, 4)])
    c = dict(kind=kind, q_heads=q_heads, kv_heads=kv_heads, dtype=rng.choice(["fp16", "bf16"]))
    sinks = rng.choice([0, 1, 4, 4, 16, 100])
    if kind == "decode":
        c.update(batch=rng.choice([1, 1, 2, 5, 16]), tokens=_span(rng, 40, 32000), window=_span(rng, 16, 8192),
                 sinks=sinks)
    elif kind == "ragged":
        top = _span(rng, 500, 32768)
        c.update(batch=rng.randint(2, 16), tokens=top, shortest=_span(rng, 1, top // 2), window=_span(rng, 64, 8192),
                 sinks=sinks)
    elif kind == "prefill":
        chunk = rng.random() < 0.6
        c.update(queries=_span(rng, 2, 2048) if chunk else _span(rng, 20, 8191),
                 past=_span(rng, 100, 9000) if chunk else 0, batch=rng.choice([1, 1, 2]), layers=rng.randint(1, 4),
                 window=_span(rng, 16, 8192), sinks=sinks)
        while c["batch"] * c["q_heads"] * c["queries"] * (c["queries"] + c["past"]) > 1 << 30 or work(c)["flops"] > 5e11:
            c["queries"] = c["queries"] // 2 + 1
    elif kind == "rope_append":
        c.update(layers=rng.randint(1, 24), tokens=_span(rng, 1, 20000), queries=_span(rng, 1, 6620),
                 page_tokens=rng.choice([16, 32, 64, 64, 128]))
        del c["q_heads"]
    elif kind == "paged_step":
        one = rng.random() < 0.6
        c.update(layers=rng.randint(2, 16), batch=_span(rng, 1, 16), tokens=_span(rng, 60, 9000),
                 queries=1 if one else _span(rng, 2, 700), window=_span(rng, 64, 4096) if one else 0,
                 sinks=sinks if one else 0, page_tokens=rng.choice([16, 32, 64, 64, 128]))
    elif kind == "shared":
        top = _span(rng, 4, 1500)
        c.update(batch=_span(rng, 2, 64), prefix=_span(rng, 64, 16384), tokens=top, shortest=rng.randint(0, top))
    else:
        top = _span(rng, 4, 900)
        c.update(layers=rng.randint(2, 12), batch=_span(rng, 2, 24), prefix=_span(rng, 64, 8200), tokens=top,
                 shortest=rng.randint(1, top), page_tokens=rng.choice([16, 32, 64, 64, 128]))
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _randn(gen, shape, case):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(DTYPES[case["dtype"]])


def _rows(gen, case, batch, heads, n):
    """Projections of n new tokens as a model hands them over: [b, heads, n, d], a transposed view."""
    return _randn(gen, (batch, n, heads, D), case).transpose(1, 2)


def _cache(gen, case, batch, heads, n):
    """A cache's n tokens as a view of a buffer with room for more."""
    return _randn(gen, (batch, heads, n + 64, D), case)[:, :, :n]


def _inv_freq():
    return (1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))).float().to(DEV)


def _inputs(case, seed):
    """Every random tensor of a case, from the seed alone."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kind, hkv, n = case["kind"], case["kv_heads"], case.get("tokens", 0)
    hq, layers, b = case.get("q_heads", 0), case.get("layers", 1), case.get("batch", 1)
    x = {"lens": [n] * b}
    if "shortest" in case:  # one of them as long as they get
        x["lens"] = torch.randint(case["shortest"], n + 1, (b,), generator=g, device=DEV).tolist()
        x["lens"][b // 2] = n
    elif kind == "paged_step":  # between half and all of `tokens`
        x["lens"] = torch.randint(n - n // 2, n + 1, (b,), generator=g, device=DEV).tolist()
    total = n + (case["past"] + case["queries"] if kind == "prefill" else 0)
    x["k"] = [_cache(g, case, b, hkv, total) for _ in range(layers)]
    x["v"] = [_cache(g, case, b, hkv, total) for _ in range(layers)]
    if "prefix" in case:
        x["kp"] = [_cache(g, case, 1, hkv, case["prefix"]) for _ in range(layers)]
        x["vp"] = [_cache(g, case, 1, hkv, case["prefix"]) for _ in range(layers)]
    if kind in ("rope_append", "paged_step"):
        x["kn"] = [_rows(g, case, b, hkv, case["queries"]) for _ in range(layers)]
        x["vn"] = [_rows(g, case, b, hkv, case["queries"]) for _ in range(layers)]
    if kind != "rope_append":
        x["q"] = [_rows(g, case, b, hq, case.get("queries", 1)) for _ in range(layers)]
    return x


def _layout(case, lens):
    """Pages of the pools, and for each sequence the (page, slot) of its tokens, shared ones first, and of the step's
    new ones: pages are taken in order, a prefix first, then a turn of each sequence after the other's."""
    P, prefix, new = case["page_tokens"], case.get("prefix", 0), case.get("queries", 0)
    used = -(-prefix // P)
    head = [(t // P, t % P) for t in range(prefix)]
    mine = [[] for _ in lens]
    last = [None] * len(lens)

    def take(i, count):
        nonlocal used
        for _ in range(count):
            if last[i] is None or last[i][1] == P - 1:
                last[i] = (used, 0)
                used += 1
            else:
                last[i] = (last[i][0], last[i][1] + 1)
            mine[i].append(last[i])

    for at in range(0, max(lens), TURN):
        for i, n in enumerate(lens):
            take(i, max(0, min(n, at + TURN) - at))
    for i in range(len(lens)):
        take(i, new)
    old = [np.array(head + m[:n], dtype=np.int64).reshape(-1, 2) for m, n in zip(mine, lens)]
    fresh = [np.array(m[n:], dtype=np.int64).reshape(-1, 2) for m, n in zip(mine, lens)]
    return -(-prefix // P) + len(lens) * -(-(case["tokens"] + new) // P), old, fresh


def _pools(case, pages):
    shape = (pages, case["kv_heads"], case["page_tokens"], D)
    return [torch.zeros(shape, device=DEV, dtype=DTYPES[case["dtype"]]) for _ in range(case["layers"])]


def _put(pools, slots, rows):
    """rows: per layer [heads, n, d] of one sequence, into its slots."""
    at = torch.from_numpy(slots).to(DEV)
    for pool, r in zip(pools, rows):
        pool[at[:, 0], :, at[:, 1]] = r.transpose(0, 1)


def prepare(case, seed):
    x = _inputs(case, seed)
    kind, b = case["kind"], case.get("batch", 1)
    st = {"case": case, "q": x.get("q"), "kn": x.get("kn"), "vn": x.get("vn")}
    if kind in ("decode", "prefill"):
        st.update(k=x["k"], v=x["v"])
        return st
    lens = x["lens"]
    if kind in ("ragged", "shared"):
        st.update(q=x["q"][0].reshape(b, case["kv_heads"], -1, D), k=x["k"][0], v=x["v"][0],
                  lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        if kind == "shared":
            st.update(kp=x["kp"][0], vp=x["vp"][0])
        return st
    # The paged kinds: pools with the cached rows in place, and the tables that a paged cache keeps.
    pages, old, fresh = _layout(case, lens)
    st.update(inv_freq=_inv_freq(), counts=[len(o) for o in old])
    if own:
        from threadcut_amd import paged

        cache = paged.PagedKV(case["layers"], case["kv_heads"], pages, case["page_tokens"], batch=b,
                              dtype=DTYPES[case["dtype"]], device=DEV)
        if "prefix" in case:
            cache.append(0, [t[0] for t in x["kp"]], [t[0] for t in x["vp"]])
            for i in range(1, b):
                cache.fork(0, i)
        for at in range(0, max(lens), TURN):
            for i, n in enumerate(lens):
                if at < n:
                    cache.append(i, [t[i, :, at:min(n, at + TURN)] for t in x["k"]],
                                 [t[i, :, at:min(n, at + TURN)] for t in x["v"]])
        st["cache"] = cache
        return st
    st.update(kpool=_pools(case, pages), vpool=_pools(case, pages))
    shared = case.get("prefix", 0)
    for name, head in (("k", "kp"), ("v", "vp")):
        if shared:
            _put(st[name + "pool"], old[0][:shared], [t[0] for t in x[head]])
        for i, n in enumerate(lens):
            _put(st[name + "pool"], old[i][shared:], [t[i, :, :n] for t in x[name]])
    if kind == "shared_paged":  # [b, longest] slots of each sequence's own tokens
        most = max(lens)
        table = np.zeros((b, most, 2), dtype=np.int64)
        for i, n in enumerate(lens):
            table[i, :n] = old[i][shared:]
        st.update(head=torch.from_numpy(old[0][:shared]).to(DEV), table=torch.from_numpy(table).to(DEV),
                  lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        return st
    st.update(slots=torch.from_numpy(np.stack(fresh)).to(DEV),
              pos=torch.tensor(lens, device=DEV)[:, None] + torch.arange(case["queries"], device=DEV))
    if case.get("window"):  # the visible slots of each sequence, -1 past them; the new token is the last one
        seen = [np.concatenate((np.concatenate((o, f))[:case["sinks"]],
                                np.concatenate((o, f))[max(len(o) + 1 - case["window"], case["sinks"]):]))
                for o, f in zip(old, fresh)]
        table = np.full((b, max(len(s) for s in seen), 2), -1, dtype=np.int64)
        for i, s in enumerate(seen):
            table[i, :len(s)] = s
        st["seen"] = torch.from_numpy(table).to(DEV)
    return st


# ---------------------------------------------------------------------------
# The plain form: elementary torch operations in float32
# ---------------------------------------------------------------------------

def _weights(s):
    """Softmax over the last dim of scores in which -inf is hidden; a row with nothing visible weighs nothing."""
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _attend(q, k, v, seen):
    """q [b, hq, t, d] on k/v [b, hkv, n, d], seen a bool that broadcasts to [b, 1, t, n] or None -> [b, t, hq, d]."""
    b, hq, t, d = q.shape
    hkv = k.shape[1]
    s = (q.float().reshape(b, hkv, -1, d) @ k.float().transpose(2, 3)) * SCALE
    if seen is not None:
        s = s.view(b, hkv, hq // hkv, t, -1).masked_fill_(~seen[:, :, None], float("-inf")).view(s.shape)
    out = _weights(s) @ v.float()
    return out.reshape(b, hq, t, d).transpose(1, 2).to(q.dtype)


def _band(t, n, window, sinks, device):
    """bool [1, 1, t, n]: what t queries at the end of n keys see."""
    p = torch.arange(n - t, n, device=device)[:, None]
    j = torch.arange(n, device=device)[None]
    return ((j <= p) & ((j > p - window) | (j < sinks)))[None, None]


def _rotated(x, pos, inv_freq):
    """x [b, heads, t, d] moved to positions pos [b, t]: the angles in 64 bits (far positions), the rest in 32."""
    angle = pos[..., None].double() * inv_freq.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    lo, hi = x.float().split(D // 2, -1)
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1).to(x.dtype)


def _shared(q, kp, vp, k, v, lens):
    """q [b, hkv, g, d] on a prefix kp/vp [hkv, p, d] and own keys k/v [b, hkv, n, d] of lens tokens."""
    b, hkv, g, d = q.shape
    qf = q.float()
    head = (qf.transpose(0, 1).reshape(hkv, b * g, d) @ kp.float().transpose(1, 2)).view(hkv, b, g, -1).transpose(0, 1)
    mine = qf @ k.float().transpose(2, 3)
    hidden = torch.arange(k.shape[2], device=q.device) >= lens[:, None]
    mine = mine.masked_fill(hidden[:, None, None], float("-inf"))
    w_head, w_mine = _weights(torch.cat((head, mine), -1) * SCALE).split((head.shape[-1], mine.shape[-1]), -1)
    out = (w_head.transpose(0, 1).reshape(hkv, b * g, -1) @ vp.float()).view(hkv, b, g, d).transpose(0, 1)
    return (out + w_mine @ v.float()).to(q.dtype)


def _at(pool, table):
    """Rows of a pool by [..., n, 2] slots: [..., heads, n, d]."""
    return pool[table[..., 0], :, table[..., 1]].transpose(-2, -3)


def _plain(st):
    case = st["case"]
    kind = case["kind"]
    window, sinks = case.get("window"), case.get("sinks")
    if kind == "decode":
        k, v, n = st["k"][0], st["v"][0], case["tokens"]
        lo = max(n - window, 0)
        first = min(sinks, lo)
        return _attend(st["q"][0], torch.cat((k[:, :, :first], k[:, :, lo:]), 2),
                       torch.cat((v[:, :, :first], v[:, :, lo:]), 2), None)
    if kind == "ragged":
        q, lens = st["q"], st["lens"][:, None]
        j = torch.arange(case["tokens"], device=q.device)[None]
        seen = (j < lens) & ((j >= lens - window) | (j < sinks))
        return _attend(q.reshape(q.shape[0], -1, 1, D), st["k"], st["v"], seen[:, None, None]).reshape(q.shape)
    if kind == "prefill":
        n = case["past"] + case["queries"]
        seen = _band(case["queries"], n, window, sinks, DEV)
        return [_attend(q, k, v, seen) for q, k, v in zip(st["q"], st["k"], st["v"])]
    if kind == "shared":
        return _shared(st["q"], st["kp"][0], st["vp"][0], st["k"], st["v"], st["lens"])
    if kind == "shared_paged":
        b, hkv = case["batch"], case["kv_heads"]
        return [_shared(q.reshape(b, hkv, -1, D), _at(kp, st["head"]), _at(vp, st["head"]), _at(kp, st["table"]),
                        _at(vp, st["table"]), st["lens"]) for q, kp, vp in zip(st["q"], st["kpool"], st["vpool"])]
    page, slot = st["slots"][..., 0], st["slots"][..., 1]
    outs = []
    for i, (kn, vn) in enumerate(zip(st["kn"], st["vn"])):
        kp, vp = st["kpool"][i], st["vpool"][i]
        kp[page, :, slot] = _rotated(kn, st["pos"], st["inv_freq"]).transpose(1, 2)
        vp[page, :, slot] = vn.transpose(1, 2)
        if kind == "paged_step":
            q = _rotated(st["q"][i], st["pos"], st["inv_freq"])
            if window:
                seen = (st["seen"][..., 0] >= 0)[:, None, None]
                at = st["seen"].clamp(min=0)
                q = _attend(q, _at(kp, at), _at(vp, at), seen)
            outs.append(q)
    return {"k": st["kpool"], "v": st["vpool"], "out": outs}


# ---------------------------------------------------------------------------
# The package's calls
# ---------------------------------------------------------------------------

def _own(st):
    from threadcut_amd import attention, flash_decode
    from threadcut_amd.match import Split

    case = st["case"]
    kind = case["kind"]
    window, sinks = case.get("window"), case.get("sinks")
    if kind in ("decode", "prefill"):
        outs = [attention.attention(None, q, k, v, None, scaling=SCALE, sliding_window=window, sink_tokens=sinks)[0]
                for q, k, v in zip(st["q"], st["k"], st["v"])]
        return outs[0] if kind == "decode" else outs
    if kind == "ragged":
        return flash_decode.decode_attention_batched(st["q"], st["k"], st["v"], SCALE, lens=st["lens"], window=window,
                                                     sink_tokens=sinks)
    if kind == "shared":
        return flash_decode.decode_attention_shared(st["q"], st["kp"], st["vp"], st["k"], st["v"], SCALE,
                                                    lens=st["lens"])
    cache, hkv = st["cache"], case["kv_heads"]
    if kind == "shared_paged":
        return [cache.decode(i, q.reshape(q.shape[0], hkv, -1, D), SCALE) for i, q in enumerate(st["q"])]
    outs = []
    if kind == "rope_append":
        cache.append(0, st["kn"], st["vn"], inv_freq=st["inv_freq"])
    else:
        cache.reserve_step(case["queries"])
        for i, (q, kn, vn) in enumerate(zip(st["q"], st["kn"], st["vn"])):
            q = cache.write_step(i, kn, vn, inv_freq=st["inv_freq"], query=q)
            if window:
                b = q.shape[0]
                q = cache.decode(i, q.reshape(b, hkv, -1, D), SCALE, window=window,
                                 sink_tokens=sinks).reshape(b, 1, -1, D)
            outs.append(q)
    for i, n in reversed(list(enumerate(st["counts"]))):  # the tokens are taken back, the last page taken first
        cache.prune(i, Split(n, cache.length(i), 0), st["inv_freq"])
    return {"k": cache.k_pools, "v": cache.v_pools, "out": outs}


def run(st):
    return _own(st) if own else _plain(st)


# ---------------------------------------------------------------------------
# What a pass has to read, write and compute
# ---------------------------------------------------------------------------

def _visible(n, window, sinks):
    """Keys that the last of n tokens sees."""
    return min(n, window) + min(sinks, max(0, n - window))


def work(case):
    kind, hkv, hq = case["kind"], case["kv_heads"], case.get("q_heads", 0)
    layers, b, n = case.get("layers", 1), case.get("batch", 1), case.get("tokens", 0)
    window, sinks = case.get("window"), case.get("sinks")
    row = 2 * D  # bytes of one head's row
    if kind == "prefill":
        t, past = case["queries"], case["past"]
        pairs = sum(_visible(p + 1, window, sinks) for p in range(past, past + t))
        first = max(0, past + 1 - window)
        keys = past + t - first + min(sinks, first)
        return {"bytes": layers * b * (2 * hkv * keys + 2 * hq * t) * row, "flops": layers * 4 * D * hq * b * pairs}
    if kind in ("rope_append", "paged_step"):
        t = case["queries"]
        moved = 4 * hkv * t + (2 * hq * t if kind == "paged_step" else 0)
        keys = _visible(n - n // 4 + 1, window, sinks) if window else 0
        return {"bytes": layers * b * (moved + 2 * hkv * keys) * row,
                "flops": layers * b * (3 * D * (hkv + hq) * t + 4 * D * hq * keys)}
    if kind == "decode":
        keys, pairs = b * _visible(n, window, sinks), b * _visible(n, window, sinks)
    elif kind == "ragged":
        low = case["shortest"]
        steps = [low + (n - low) * i // 64 for i in range(65)]
        keys = pairs = _visible(n, window, sinks) + (b - 1) * sum(_visible(m, window, sinks) for m in steps) // 65
    else:
        mine = n + (b - 1) * (n + case["shortest"]) // 2
        keys, pairs = case["prefix"] + mine, b * case["prefix"] + mine
    return {"bytes": layers * (2 * hkv * keys + 2 * hq * b) * row, "flops": layers * 4 * D * hq * pairs}


# ---------------------------------------------------------------------------
# The definition in float64, sequence by sequence and head by head
# ---------------------------------------------------------------------------

def _one(q, k, v, seen=None):
    """float64 softmax(q k^T) v of one head: q [t, d], k/v [n, d], seen bool [t, n] or None."""
    s = torch.mm(q.double(), k.double().t().contiguous()) * SCALE
    if seen is not None:
        s[~seen] = -math.inf
    return torch.softmax(s, 1).nan_to_num(0.0).mm(v.double())


def _turned(x, start, inv_freq):
    """x [heads, t, d] as complex pairs times exp(i pos f), pos = start .. start + t."""
    x = x.double()
    pair = torch.complex(x[..., :D // 2], x[..., D // 2:])
    pos = start + torch.arange(x.shape[1], dtype=torch.float64, device=x.device)
    pair = pair * torch.polar(torch.ones((), dtype=torch.float64, device=x.device), torch.outer(pos, inv_freq.double()))
    return torch.cat((pair.real, pair.imag), -1)


def exact(case, seed):
    x = _inputs(case, seed)
    kind, hkv, b = case["kind"], case["kv_heads"], case.get("batch", 1)
    g = case.get("q_heads", hkv) // hkv
    window, sinks, lens = case.get("window"), case.get("sinks"), x["lens"]
    if kind == "prefill":
        t, n = case["queries"], case["past"] + case["queries"]
        ahead = torch.arange(n, device=DEV) - torch.arange(n - t, n, device=DEV)[:, None]  # key - query
        seen = (ahead <= 0) & (ahead > -window)
        seen[:, :sinks] |= ahead[:, :sinks] <= 0
        return [torch.stack([torch.stack([_one(q[i, h], k[i, h // g], v[i, h // g], seen) for h in range(hkv * g)], 1)
                             for i in range(b)]) for q, k, v in zip(x["q"], x["k"], x["v"])]

    def keys_of(k, i, n):
        """Sequence i's visible rows of n tokens [hkv, n, d]."""
        first = max(n - window, 0)
        return torch.cat((k[i, :, :min(sinks, first)], k[i, :, first:n]), 1)

    if kind in ("decode", "ragged"):
        out = torch.stack([torch.stack([_one(x["q"][0][i, h], keys_of(x["k"][0], i, n)[h // g],
                                             keys_of(x["v"][0], i, n)[h // g])[0] for h in range(hkv * g)])
                           for i, n in enumerate(lens)])
        return out[:, None] if kind == "decode" else out.view(b, hkv, g, D)
    if kind in ("shared", "shared_paged"):
        outs = []
        for q, kp, vp, k, v in zip(x["q"], x["kp"], x["vp"], x["k"], x["v"]):
            outs.append(torch.stack([torch.stack([_one(q[i, h], torch.cat((kp[0, h // g], k[i, h // g, :n])),
                                                       torch.cat((vp[0, h // g], v[i, h // g, :n])))[0]
                                                  for h in range(hkv * g)]) for i, n in enumerate(lens)]).view(b, hkv, g, D))
        return outs[0] if kind == "shared" else outs
    pages, old, fresh = _layout(case, lens)
    inv_freq = _inv_freq()
    pools = {"k": [], "v": [], "out": []}
    for layer in range(case["layers"]):
        k, v = x["k"][layer], x["v"][layer]
        kp = torch.zeros((pages, hkv, case["page_tokens"], D), dtype=torch.float64, device=DEV)
        vp = torch.zeros_like(kp)
        outs = []
        for i, n in enumerate(lens):
            kn, vn = _turned(x["kn"][layer][i], n, inv_freq), x["vn"][layer][i].double()
            rows = torch.from_numpy(np.concatenate((old[i], fresh[i]))).to(DEV)
            kp[rows[:, 0], :, rows[:, 1]] = torch.cat((k[i, :, :n].double(), kn), 1).transpose(0, 1)
            vp[rows[:, 0], :, rows[:, 1]] = torch.cat((v[i, :, :n].double(), vn), 1).transpose(0, 1)
            if kind == "paged_step":
                q = _turned(x["q"][layer][i], n, inv_freq)
                if window:
                    # The attention reads keys and queries as they are stored: rounded to the cache's type.
                    kn, q = (t.to(DTYPES[case["dtype"]]).double() for t in (kn, q))
                    both = [torch.cat((t[i, :, :n].double(), new), 1)[None] for t, new in ((k, kn), (v, vn))]
                    ks, vs = (keys_of(t, 0, n + 1) for t in both)
                    q = torch.stack([_one(q[h], ks[h // g], vs[h // g])[0] for h in range(hkv * g)])[None]
                outs.append(q)
        pools["k"].append(kp)
        pools["v"].append(vp)
        if outs:
            pools["out"].append(torch.stack(outs))
    return pools
