"""The serving operators next to the KV transfers, as they are measured: slot
mappings from request lengths, rotary positions, and the attention of a batch
that shares a prefix.

A case is a dict of plain values.  `kind` names the call:

  slots         block tables, slot mapping and positions of a batch
                (build_slot_mapping)
  rotary        queries and keys rotated to or from their positions
                (rotary_embedding)
  rotary_paged  the same with keys and values written to their paged caches
                (rotary_embedding_to_paged)
  attention     tokens of a batch whose requests share a prefix, over the
                paged caches (shared_prefix_attention)
"""

import math
import os
import sys

import torch

# False: run() computes the operators in plain torch operations; true: it
# calls the library.
own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _slots(name, requests, query, context, block, free, pad=0, wide=False):
    return {"name": name, "kind": "slots", "requests": requests, "query": query, "context": context, "block": block,
            "free": free, "pad": pad, "wide": wide}


def _rotary(name, tokens, heads, kv_heads, dim, rot, offset, neox, dtype, scaling, context, inverse=False):
    return {"name": name, "kind": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "offset": offset, "neox": neox, "dtype": dtype, "scaling": scaling, "context": context,
            "inverse": inverse}


def _paged(name, tokens, heads, kv_heads, dim, rot, offset, neox, dtype, scaling, context, block, pad):
    return dict(_rotary(name, tokens, heads, kv_heads, dim, rot, offset, neox, dtype, scaling, context),
                kind="rotary_paged", block=block, pad=pad)


def _attention(name, requests, query, heads, kv_heads, dim, prefix, suffix, block, dtype, pad=0):
    return {"name": name, "kind": "attention", "requests": requests, "query": query, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "prefix": prefix, "suffix": suffix, "block": block, "dtype": dtype,
            "pad": pad}


def listed():
    return [
        # A decode step of 64 requests in 16-token blocks: one token each, a
        # new block for the few whose last one is full.  Latency.
        _slots("slots_decode", 64, 1, 4096, 16, True),
        # Ragged prompts on top of loaded prefixes, their blocks taken from
        # the free list, the batch padded.
        _slots("slots_prefill_ragged", 48, 2047, 8192, 128, True, pad=37),
        # The tokens of 256 long requests whose tables are there already: the
        # slot mapping a connector stores them by.
        _slots("slots_store_long", 256, 4096, 32768, 64, False, wide=True),
        # A decode step of 64 requests, 32 query and 8 KV heads.  Latency.
        _rotary("rotary_decode", 64, 32, 8, 128, 128, 0, True, "bf16", "none", 8192),
        # Interleaved pairs in the last half of each head, an odd prompt, a
        # context scaled in part of the frequencies.
        _rotary("rotary_part_interleaved", 1009, 28, 4, 128, 64, 64, False, "f16", "yarn", 131072),
        # The backward direction (gradients, or keys stripped of their
        # positions) over a long sequence.
        _rotary("rotary_backward", 8192, 32, 8, 128, 128, 0, True, "bf16", "llama3", 131072, inverse=True),
        # A decode step that writes its new rows, some of its tokens padding.
        _paged("rotary_paged_decode", 48, 16, 2, 96, 96, 0, True, "f16", "none", 4096, 16, 0.1),
        # A 16384-token prefill, rotated and written to its pages in one pass.
        _paged("rotary_paged_prefill", 16384, 32, 8, 128, 128, 0, True, "bf16", "linear", 65536, 128, 0.05),
        # Four requests behind a system prompt: the smallest decode step.
        _attention("attention_small", 4, 1, 32, 8, 128, 1000, 200, 16, "bf16"),
        # 64 requests over one loaded document.
        _attention("attention_decode", 64, 1, 32, 8, 128, 4096, 1024, 128, "bf16"),
        # Several tokens a request to verify, ragged, small heads, padding at
        # the batch's end and a prefix that ends inside a page.
        _attention("attention_verify", 17, 5, 16, 2, 64, 8197, 777, 64, "f16", pad=3),
        # 256 requests over a prefix of 16384 tokens: the matrix products.
        _attention("attention_large", 256, 1, 32, 8, 128, 16384, 1024, 128, "bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["slots", "rotary", "rotary_paged", "attention", "attention"])
    block = rng.choice([16, 64, 128])
    if kind == "slots":
        requests = _log(rng, 1, 1024)
        query = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(4096, 256 * 4096 // requests)))
        c = _slots("", requests, query, _log(rng, 1, 32768), block, rng.random() < 0.6, rng.choice([0, rng.randint(1, 64)]),
                   rng.random() < 0.5)
    elif kind != "attention":
        dim = rng.choice([64, 96, 128])
        rot = rng.choice([dim, dim, dim // 2])
        offset = rng.choice([0, dim - rot])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        tokens = _log(rng, 1, 8192 if dtype == "f32" else 16384)
        args = (tokens, heads, kv_heads, dim, rot, offset, rng.random() < 0.6, dtype,
                rng.choice(["none", "linear", "llama3", "yarn"]), _log(rng, 2048, 262144))
        if kind == "rotary":
            c = _rotary("", *args, inverse=rng.random() < 0.4)
        else:
            c = _paged("", *args, block, rng.choice([0.0, 0.05]))
    else:
        requests = _log(rng, 1, 256)
        query = 1 if rng.random() < 0.6 else rng.randint(1, max(1, min(8, 256 // requests)))
        dim = rng.choice([64, 96, 128])
        kv_heads, group = rng.choice([(8, 4), (4, 7), (2, 8), (8, 1), (1, 16), (1, 5)])
        c = _attention("", requests, query, kv_heads * group, kv_heads, dim, _log(rng, 1, 16384), _log(rng, query, 1024),
                       block, rng.choice(["bf16", "bf16", "f16"]), rng.choice([0, rng.randint(1, 4)]))
    c.pop("name")
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"slots": _slots_state, "rotary": _rotary_state, "rotary_paged": _paged_state, "attention": _attention_state}
    return dict(make[case["kind"]](case, gen), case=case)


def _below(gen, high, n):
    """n whole numbers in [0, high)."""
    return torch.randint(0, max(1, int(high)), (n,), generator=gen, device="cuda")


def _lens(case):
    """New tokens of each request: evenly from 1 to `query`, so that every
    seed has the same number of tokens; a few of many requests are done."""
    R, Q = case["requests"], case["query"]
    done = R // 16 if case["kind"] == "slots" else 0
    return [0 if r < done else 1 + r * Q // R for r in range(R)]


def _shuffled(case, gen):
    lens = torch.tensor(_lens(case), device="cuda")
    return lens[torch.randperm(lens.numel(), generator=gen, device="cuda")]


def _slots_state(case, gen):
    """Requests of 0 to `context` tokens so far; pages in random order."""
    R, Q, C, BS = case["requests"], case["query"], case["context"], case["block"]
    context = _below(gen, C + 1, R)
    query = _shuffled(case, gen)
    width = -(-(C + Q) // BS)
    have, need = (context + BS - 1) // BS, (context + query + BS - 1) // BS
    pages = R * width + 64
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = order[: R * width].view(R, width).clone()
    there = have if case["free"] else need
    table[torch.arange(width, device="cuda")[None, :] >= there[:, None]] = -1
    total = int(query.sum()) + case["pad"]
    new = int((need - have).sum())
    lens = torch.int64 if case["wide"] else torch.int32
    i32 = {"dtype": torch.int32, "device": "cuda"}
    i64 = {"dtype": torch.int64, "device": "cuda"}
    state = {"query_lens": query.to(lens), "context_lens": context.to(lens), "table": table,
             "slots": torch.empty(total, **i64), "positions": torch.empty(total, **i64),
             "query_start_loc": torch.empty(R + 1, **i32), "seq_lens": torch.empty(R, **i32)}
    if case["free"]:
        at = int(_below(gen, 50, 1))
        state["free"] = torch.randperm(pages, generator=gen, device="cuda")[: at + new + 10].to(torch.int32)
        state["cursor"] = torch.tensor([at], **i64)
        state["next_cursor"] = torch.empty(1, **i64)
    return state


def _inv_freq(rot, scaling):
    """64-bit frequencies (radians a position) and the factor on cos and sin."""
    base = 500000.0 if scaling == "llama3" else 10000.0
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "linear":
        return inv / 4.0, 1.0
    if scaling == "llama3":
        # Wavelengths over 8192 positions eight times as long, those under
        # 2048 as they are, those between by a blend.
        turns = 8192.0 * inv / (2.0 * math.pi)
        keep = ((turns - 1.0) / 3.0).clamp(0.0, 1.0)
        return inv * keep + inv / 8.0 * (1.0 - keep), 1.0
    if scaling == "yarn":
        # Frequencies of more than 32 turns in 4096 positions kept, of less
        # than one divided by 32, a ramp between.
        def dim_of(turns):
            return rot * math.log(4096.0 / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(0, math.floor(dim_of(32.0))), min(rot - 1, math.ceil(dim_of(1.0)))
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return inv / 32.0 * ramp + inv * (1.0 - ramp), 0.1 * math.log(32.0) + 1.0
    return inv, 1.0


def _rotary_state(case, gen):
    """Rows of one fused projection [q | k | v]; runs of positions from a
    random place in the context, as requests of a batch have them."""
    T, D, dt = case["tokens"], case["dim"], DTYPES[case["dtype"]]
    wq, wk = case["heads"] * D, case["kv_heads"] * D
    qkv = torch.randn((T, wq + 2 * wk), generator=gen, device="cuda").to(dt)
    runs = _below(gen, case["context"], -(-T // 256))
    positions = (runs[:, None] + torch.arange(256, device="cuda")[None, :]).reshape(-1)[:T] % case["context"]
    inv, scale = _inv_freq(case["rot"], case["scaling"])
    return {"query": qkv[:, :wq], "key": qkv[:, wq: wq + wk], "value": qkv[:, wq + wk:],
            "positions": positions.contiguous(), "inv_freq": inv.cuda(), "scale": scale,
            "query_out": torch.empty((T, wq), dtype=dt, device="cuda"),
            "key_out": torch.empty((T, wk), dtype=dt, device="cuda")}


def _paged_state(case, gen):
    """One request's rows: its pages in random order, some tokens padding."""
    s = _rotary_state(case, gen)
    T, BS, dt = case["tokens"], case["block"], DTYPES[case["dtype"]]
    used = -(-T // BS)
    pages = used + used // 4 + 1
    order = torch.randperm(pages, generator=gen, device="cuda")[:used]
    slots = (order[:, None] * BS + torch.arange(BS, device="cuda")[None, :]).reshape(-1)[:T]
    drop = torch.rand(T, generator=gen, device="cuda") < case["pad"]
    s["slots"] = torch.where(drop, torch.full_like(slots, -1), slots).contiguous()
    shape = (pages, BS, case["kv_heads"], case["dim"])
    s["caches"] = tuple(torch.randn(shape, generator=gen, device="cuda").to(dt) for _ in range(2))
    s.pop("key_out")
    return s


def _attention_state(case, gen):
    """Each request: the shared prefix, its own tokens (the newest `query` or
    fewer asked for now), and pages in random order; with `pad`, rows behind
    the last request and a request that is no longer there."""
    R, Q, P, S, BS = case["requests"], case["query"], case["prefix"], case["suffix"], case["block"]
    dt = DTYPES[case["dtype"]]
    lens = _shuffled(case, gen)
    own_tokens = torch.maximum(1 + _below(gen, S, R), lens)
    seq = P + own_tokens
    if case["pad"]:
        seq[R // 2] = 0
    start = torch.zeros(R + 1, dtype=torch.int64, device="cuda")
    start[1:] = lens.cumsum(0)
    T = int(start[-1]) + case["pad"]
    # A page that the prefix ends in is each request's own behind that point.
    width = -(-(P + S) // BS)
    first = P // BS
    shared = -(-P // BS)
    pages = shared + R * (width - first) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.empty((R, width), dtype=torch.int32, device="cuda")
    table[:, :first] = order[:first]
    table[:, first:] = order[shared: shared + R * (width - first)].view(R, width - first)
    shape = (pages, BS, case["kv_heads"], case["dim"])
    caches = tuple(torch.randn(shape, generator=gen, device="cuda", dtype=dt) for _ in range(2))
    q = torch.randn((T, case["heads"], case["dim"]), generator=gen, device="cuda")
    return {"query": (1.5 * q).to(dt), "caches": caches, "shared": order[:shared].clone(), "table": table,
            "seq_lens": seq.to(torch.int32), "query_start_loc": start.to(torch.int32),
            "scale": case["dim"] ** -0.5,
            "output": (0.02 * torch.randn(q.shape, generator=gen, device="cuda")).to(dt),
            "lse": torch.randn(q.shape[:2], generator=gen, device="cuda")}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"slots": _plain_slots, "rotary": _plain_rotary, "rotary_paged": _plain_paged,
            "attention": _plain_attention}[state["case"]["kind"]](state)


def _run_own(s):
    c = s["case"]
    ops = _library()
    if c["kind"] == "slots":
        ops.build_slot_mapping(s["query_lens"], s["context_lens"], s["table"], c["block"], s["slots"], s["positions"],
                               s["query_start_loc"], s["seq_lens"], s.get("free"), s.get("cursor"), s.get("next_cursor"))
        return _slots_out(s)
    if c["kind"] == "rotary":
        ops.rotary_embedding(s["positions"], s["query"], s["key"], c["dim"], s["inv_freq"], is_neox=c["neox"],
                             rotary_offset=c["offset"], scale=s["scale"], inverse=c["inverse"],
                             query_out=s["query_out"], key_out=s["key_out"])
        return {"query": s["query_out"], "key": s["key_out"]}
    if c["kind"] == "rotary_paged":
        ops.rotary_embedding_to_paged(s["positions"], s["query"], s["key"], s["value"], s["caches"], s["slots"],
                                      c["dim"], s["inv_freq"], is_neox=c["neox"], rotary_offset=c["offset"],
                                      scale=s["scale"], query_out=s["query_out"])
        return {"query": s["query_out"], "key_cache": s["caches"][0], "value_cache": s["caches"][1]}
    ops.shared_prefix_attention(s["query"], s["caches"], s["shared"], c["prefix"], s["table"], s["seq_lens"],
                                s["query_start_loc"], s["scale"], s["output"], s["lse"])
    return {"output": s["output"], "lse": s["lse"]}


def _library():
    global _ops
    if _ops is None:
        sys.path.insert(0, os.path.join(ROOT, "lmcache-ascend_amd"))
        from lmcache_amd import c_ops

        _ops = c_ops
    return _ops


_ops = None


def _slots_out(s):
    names = ("slots", "positions", "query_start_loc", "seq_lens") + (("table", "next_cursor") if "free" in s else ())
    return {n: s[n] for n in names}


def _plain_slots(s):
    BS, table = s["case"]["block"], s["table"]
    R, width = table.shape
    query, context = s["query_lens"].to(torch.int64), s["context_lens"].to(torch.int64)
    end = query.cumsum(0)
    start = end - query
    out = {"query_start_loc": torch.cat((start[:1], end)).to(torch.int32), "seq_lens": (context + query).to(torch.int32)}
    if "free" in s:
        have, need = (context + BS - 1) // BS, (context + query + BS - 1) // BS
        new = need - have
        taken = new.cumsum(0)
        col = torch.arange(width, device=table.device)[None, :]
        at = s["cursor"] + (taken - new - have)[:, None] + col
        fresh = (col >= have[:, None]) & (col < need[:, None])
        table.copy_(torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], table))
        out["table"] = table
        out["next_cursor"] = s["cursor"] + taken[-1:]
    t = torch.arange(s["slots"].numel(), device=table.device)
    r = torch.searchsorted(end, t, right=True)
    there = r < R
    r = r.clamp(max=R - 1)
    pos = torch.where(there, context[r] + t - start[r], 0)
    page = table[r, (pos // BS).clamp(max=width - 1)].to(torch.int64)
    out["positions"] = pos
    out["slots"] = torch.where(there & (page >= 0), page * BS + pos % BS, -1)
    return out


def _rotate(x, cos, sin, case):
    """Rows [T, heads * dim] in their own type, rotated in 32 bits."""
    D, rot, off = case["dim"], case["rot"], case["offset"]
    y = x.float().reshape(x.shape[0], -1, D).clone()
    part = y[..., off: off + rot]
    if case["neox"]:
        a, b = part[..., : rot // 2], part[..., rot // 2:]
    else:
        a, b = part[..., 0::2], part[..., 1::2]
    u, v = a * cos - b * sin, b * cos + a * sin
    a.copy_(u)
    b.copy_(v)
    return y.reshape(x.shape).to(x.dtype)


def _angles(s):
    """cos and sin [T, 1, rot / 2]: the angle in 64 bits, far positions need
    them."""
    angle = s["positions"].double()[:, None, None] * s["inv_freq"]
    sign = -1.0 if s["case"]["inverse"] else 1.0
    return (angle.cos() * s["scale"]).float(), (angle.sin() * (sign * s["scale"])).float()


def _plain_rotary(s):
    cos, sin = _angles(s)
    return {"query": _rotate(s["query"], cos, sin, s["case"]), "key": _rotate(s["key"], cos, sin, s["case"])}


def _plain_paged(s):
    cos, sin = _angles(s)
    key = _rotate(s["key"], cos, sin, s["case"])
    # Padding goes to a row behind the cache, which is cut off again.
    out = {"query": _rotate(s["query"], cos, sin, s["case"])}
    for name, cache, rows in (("key_cache", s["caches"][0], key), ("value_cache", s["caches"][1], s["value"])):
        flat = cache.reshape(-1, rows.shape[1])
        n = flat.shape[0]
        more = torch.cat((flat, flat[:1]))
        more.index_copy_(0, torch.where(s["slots"] >= 0, s["slots"], n), rows)
        out[name] = more[:n].reshape(cache.shape)
    return out


def _plain_attention(s):
    c, table = s["case"], s["table"]
    P, BS, H, D = c["prefix"], c["block"], c["kv_heads"], c["dim"]
    q = s["query"]
    T, G = q.shape[0], q.shape[1] // H
    start, seq = s["query_start_loc"].to(torch.int64), s["seq_lens"].to(torch.int64)
    t = torch.arange(T, device=q.device)
    r = torch.searchsorted(start[1:], t, right=True)
    there = r < seq.numel()
    r = r.clamp(max=seq.numel() - 1)
    pos = torch.where(there, seq[r] - start[r + 1] + t, -1)
    # Shared keys once for all rows, each token's own behind them.
    j = torch.arange(P, device=q.device)
    own_j = P + torch.arange(c["suffix"], device=q.device)
    page, own_page = s["shared"].to(torch.int64)[j // BS], table.to(torch.int64)[r][:, own_j // BS]
    qf = q.float().view(T, H, G, D) * s["scale"]
    k = s["caches"][0][page, j % BS].float()
    own_k = s["caches"][0][own_page, own_j % BS].float()
    flat = qf.permute(1, 0, 2, 3).reshape(H, T * G, D).contiguous()
    a = torch.bmm(flat, k.permute(1, 2, 0).contiguous()).view(H, T, G, P).permute(1, 0, 2, 3)
    b = torch.matmul(qf, own_k.permute(0, 2, 3, 1).contiguous())
    score = torch.cat((a, b), dim=-1)
    hidden = torch.cat((j, own_j))[None, :] > pos[:, None]
    score = score.masked_fill(hidden[:, None, None, :], float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(dim=-1, keepdim=True)
    v = s["caches"][1][page, j % BS].float().permute(1, 0, 2).contiguous()
    own_v = s["caches"][1][own_page, own_j % BS].float().permute(0, 2, 1, 3).contiguous()
    o = torch.bmm(p[..., :P].permute(1, 0, 2, 3).reshape(H, T * G, P).contiguous(), v).view(H, T, G, D).permute(1, 0, 2, 3)
    o = o + torch.matmul(p[..., P:].contiguous(), own_v)
    o = torch.where(total > 0, o / total, 0.0).reshape(T, H * G, D).to(q.dtype)
    lse = (torch.log(total) + top).reshape(T, H * G)
    return {"output": torch.where(there[:, None, None], o, s["output"]), "lse": torch.where(there[:, None], lse, s["lse"])}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    if case["kind"] == "slots":
        R = case["requests"]
        tokens = sum(_lens(case))
        pages = tokens / case["block"] + R / 2
        ids = (16 if case["wide"] else 8) * R
        return {"bytes": ids + 4 * pages * (3 if case["free"] else 1) + 16 * (tokens + case["pad"]) + 8 * R, "flops": 0}
    es = 4 if case.get("dtype") == "f32" else 2
    if case["kind"] == "rotary":
        elems = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * es * elems + 8 * case["tokens"], "flops": 3 * elems * case["rot"] // case["dim"]}
    if case["kind"] == "rotary_paged":
        rows = case["heads"] + 2 * case["kv_heads"] * (1 - case["pad"])
        elems = case["tokens"] * rows * case["dim"]
        return {"bytes": 2 * es * elems + 16 * case["tokens"],
                "flops": 3 * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rot"]}
    tokens = sum(_lens(case))
    own_tokens = (1 + case["suffix"]) / 2
    keys = case["prefix"] + case["requests"] * own_tokens
    rows = tokens * case["heads"]
    return {"bytes": 2 * es * keys * case["kv_heads"] * case["dim"] + rows * (2 * es * case["dim"] + 4),
            "flops": 4 * rows * case["dim"] * (case["prefix"] + own_tokens)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "slots":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_attention(s) if case["kind"] == "attention" else _exact_rotary(s)


def _exact_turned(x, s):
    """Pairs as complex numbers, times scale * exp(i * angle)."""
    c = s["case"]
    D, rot, off = c["dim"], c["rot"], c["offset"]
    y = x.double().reshape(c["tokens"], -1, D).clone()
    at = torch.arange(rot // 2, device=x.device)
    first = off + (at if c["neox"] else 2 * at)
    second = first + (rot // 2 if c["neox"] else 1)
    angle = s["positions"].double()[:, None] * s["inv_freq"][None, :]
    turn = torch.polar(torch.full_like(angle, s["scale"]), -angle if c["inverse"] else angle)
    z = torch.complex(y[..., first], y[..., second]) * turn[:, None, :]
    y[..., first], y[..., second] = z.real, z.imag
    return y.reshape(x.shape)


def _exact_rotary(s):
    if s["case"]["kind"] == "rotary":
        return {"query": _exact_turned(s["query"], s), "key": _exact_turned(s["key"], s)}
    out = {"query": _exact_turned(s["query"], s)}
    keep = s["slots"] >= 0
    for name, cache, rows in (("key_cache", s["caches"][0], _exact_turned(s["key"], s)),
                              ("value_cache", s["caches"][1], s["value"].double())):
        full = cache.double()
        full.view(-1, rows.shape[1])[s["slots"][keep]] = rows[keep]
        out[name] = full
    return out


def _exact_attention(s):
    """Request by request, its keys gathered in order."""
    c = s["case"]
    H, D, P, BS = c["kv_heads"], c["dim"], c["prefix"], c["block"]
    G = c["heads"] // H
    K, V = s["caches"]
    out, lse = s["output"].double(), s["lse"].double()
    start, seq = s["query_start_loc"].tolist(), s["seq_lens"].tolist()
    j = torch.arange(P, device=K.device)
    page = s["shared"].long()[j // BS]
    head_k, head_v = (x[page, j % BS].double().permute(1, 0, 2).contiguous() for x in (K, V))
    for r, n in enumerate(seq):
        t0, t1 = start[r], start[r + 1]
        if n <= 0:
            out[t0:t1], lse[t0:t1] = 0.0, float("-inf")
            continue
        j = torch.arange(P, max(P, n), device=K.device)
        page = s["table"][r].long()[j // BS]
        k, v = (torch.cat((head, x[page, j % BS].double().permute(1, 0, 2)), dim=1)[:, :n].contiguous()
                for head, x in ((head_k, K), (head_v, V)))
        q = s["query"][t0:t1].double().view(t1 - t0, H, G, D).permute(1, 0, 2, 3).reshape(H, -1, D).contiguous()
        score = torch.bmm(q, k.transpose(1, 2).contiguous()).view(H, t1 - t0, G, n) * s["scale"]
        last = n - (t1 - t0) + torch.arange(t1 - t0, device=K.device)
        hidden = torch.arange(n, device=K.device)[None, :] > last[:, None]
        score.masked_fill_(hidden[None, :, None, :], float("-inf"))
        row = torch.logsumexp(score, dim=-1)
        p = torch.exp(score - row[..., None]).reshape(H, -1, n)
        o = torch.bmm(p, v).view(H, t1 - t0, G, D)
        out[t0:t1] = o.permute(1, 0, 2, 3).reshape(t1 - t0, H * G, D)
        lse[t0:t1] = row.permute(1, 0, 2).reshape(t1 - t0, H * G)
    return {"output": out, "lse": lse}
