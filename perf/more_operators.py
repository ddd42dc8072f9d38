"""The operators of drafting and branching over the paged caches, as they are
measured: trees of drafted tokens, their attention, and the pages and rows
that a step copies, moves and gives back.

A case is a dict of plain values.  `kind` names the call:

  tree       masks and positions of drafted trees (build_draft_tree)
  attention  drafted tokens over their requests' caches (tree_attention)
  copy       pages copied in every layer, as forks do (copy_kv_pages)
  compact    kept rows moved together in every layer (compact_kv)
  release    pages given back to the free list (release_pages)
"""

import math
import os
import sys

import torch

# False: run() computes the operators in plain torch operations; true: it
# calls the library.
own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _tree(name, requests, drafts, context, even, pad=0):
    return {"name": name, "kind": "tree", "requests": requests, "drafts": drafts, "context": context, "even": even, "pad": pad}


def _attention(name, requests, drafts, heads, kv_heads, dim, context, block, dtype, even, pad=0):
    return {"name": name, "kind": "attention", "requests": requests, "drafts": drafts, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "context": context, "block": block, "dtype": dtype, "even": even, "pad": pad}


def _copy(name, pairs, layers, kv_heads, dim, block, dtype, head_major=False):
    return {"name": name, "kind": "copy", "pairs": pairs, "layers": layers, "kv_heads": kv_heads, "dim": dim,
            "block": block, "dtype": dtype, "head_major": head_major}


def _compact(name, requests, base, held, keep, layers, kv_heads, dim, block, dtype, head_major=False):
    return {"name": name, "kind": "compact", "requests": requests, "base": base, "held": held, "keep": keep,
            "layers": layers, "kv_heads": kv_heads, "dim": dim, "block": block, "dtype": dtype, "head_major": head_major}


def _release(name, requests, held, drop, block, pages, forked):
    return {"name": name, "kind": "release", "requests": requests, "held": held, "drop": drop, "block": block,
            "pages": pages, "forked": forked}


def listed():
    return [
        # A few requests with eight drafted tokens each.  Latency.
        _tree("tree_small", 4, 8, 2000, True),
        # A large batch with trees of up to 100 tokens (two words a row), padded.
        _tree("tree_large", 256, 100, 16384, False, pad=21),
        # Two requests of short contexts: the smallest verification step.  Latency.
        _attention("attention_small", 2, 8, 32, 8, 128, 2000, 16, "bf16", True),
        # 32 requests that draft 16 tokens: the bytes of their caches.
        _attention("attention_batch", 32, 16, 32, 8, 128, 8192, 128, "bf16", True),
        # Wide trees (two words a row) of small heads, seven a KV head, in small
        # blocks; padding, a request that is gone and rows that see no draft.
        _attention("attention_ragged", 13, 77, 28, 4, 64, 4999, 16, "f16", False, pad=5),
        # 32 requests with trees of 64 tokens over long contexts: the matrix products.
        _attention("attention_large", 32, 64, 32, 8, 128, 16384, 128, "bf16", True),
        # Beams that fork: the last, partly filled page of each in 32 layers.
        _copy("copy_forks", 8, 32, 8, 128, 16, "bf16"),
        # Many forks of long pages, heads before tokens in a page.
        _copy("copy_many", 256, 8, 8, 128, 128, "bf16", head_major=True),
        # The accepted path of each request's 16 drafted tokens moves behind its
        # context, in 32 layers.
        _compact("compact_accepted", 64, 700, 16, 6, 32, 8, 128, 16, "bf16"),
        # Half of each context's tokens are dropped.
        _compact("compact_dropped", 8, 0, 8000, 4000, 8, 8, 128, 128, "bf16"),
        # The pages of refused drafts go back.  Latency.
        _release("release_drafts", 64, 4096, 64, 16, 20000, 0.0),
        # Requests end, some of them forks that share their pages.
        _release("release_finished", 256, 16384, 16384, 16, 300000, 0.25),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["tree", "attention", "attention", "attention", "copy", "compact", "release"])
    block = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    dim = rng.choice([64, 96, 128, 128])
    if kind == "tree":
        c = _tree("", _log(rng, 1, 256), _log(rng, 1, 100), _log(rng, 100, 100000), rng.random() < 0.5,
                  rng.choice([0, rng.randint(1, 40)]))
    elif kind == "attention":
        kv_heads, group = rng.choice([(8, 4), (8, 4), (4, 7), (2, 8), (8, 1), (1, 16), (5, 2)])
        drafts = 1 if rng.random() < 0.15 else _log(rng, 2, 100)
        requests = _log(rng, 1, max(1, min(128, 4096 // drafts)))
        most = min(16384, 2**29 // (requests * kv_heads * dim), 2**29 // (requests * drafts * kv_heads * group))
        c = _attention("", requests, drafts, kv_heads * group, kv_heads, dim, _log(rng, 1, max(1, most)), block, dtype,
                       rng.random() < 0.6, rng.choice([0, 0, rng.randint(1, 6)]))
    elif kind == "copy":
        layers, kv_heads = _log(rng, 1, 64), rng.choice([1, 2, 4, 8])
        most = 2**28 // (layers * kv_heads * dim * block)
        c = _copy("", _log(rng, 1, max(1, min(256, most))), layers, kv_heads, dim, block, dtype, rng.random() < 0.3)
    elif kind == "compact":
        layers, kv_heads = _log(rng, 1, 32), rng.choice([1, 2, 4, 8])
        if rng.random() < 0.5:
            requests, held = _log(rng, 1, 64), rng.randint(1, 48)
            base = rng.randint(0, 700)
        else:
            requests, base = _log(rng, 1, 8), rng.choice([0, 0, 77])
            held = _log(rng, 64, max(64, min(8192, 2**28 // (layers * kv_heads * dim * requests))))
        c = _compact("", requests, base, held, max(1, int(held * rng.uniform(0.1, 1.0))), layers, kv_heads, dim, block, dtype,
                     rng.random() < 0.3)
    else:
        requests, held = _log(rng, 1, 256), _log(rng, 16, 16384)
        need = requests * -(-held // block) + 1
        c = _release("", requests, held, _log(rng, 1, held), block, need + rng.randint(0, 100000), rng.choice([0.0, 0.25, 0.5]))
    c.pop("name")
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"tree": _tree_state, "attention": _attention_state, "copy": _copy_state, "compact": _compact_state,
            "release": _release_state}
    return dict(make[case["kind"]](case, gen), case=case)


def _perm(gen, n):
    return torch.randperm(n, generator=gen, device="cuda")


def _spread(gen, low, high, n):
    """n whole numbers evenly from low to high, in random order: every seed
    has the same sum."""
    values = torch.tensor([low + (high - low) * (i + 1) // n for i in range(n)], device="cuda")
    return values[_perm(gen, n)]


def _lens(case):
    """Drafted tokens of the requests: as many each, or evenly from one on."""
    R, Q = case["requests"], case["drafts"]
    return [Q if case["even"] else max(1, Q * (r + 1) // R) for r in range(R)]


def _drafts(case, gen):
    """(query_start_loc, drafted tokens of each request, parents, index of each
    token in its request): trees whose tokens follow one of the eight before."""
    R = case["requests"]
    lens = torch.tensor(_lens(case), device="cuda")[_perm(gen, R)]
    start = torch.zeros(R + 1, dtype=torch.int64, device="cuda")
    start[1:] = lens.cumsum(0)
    T = int(start[-1])
    at = torch.arange(T, device="cuda") - start[:-1].repeat_interleave(lens)
    back = (torch.rand(T, generator=gen, device="cuda") * (at + 1).clamp(max=8)).long()
    parents = torch.cat((at - 1 - back, torch.randint(-5, 200, (case["pad"],), generator=gen, device="cuda")))
    return start.to(torch.int32), lens, parents.to(torch.int32), at


def _tree_state(case, gen):
    start, lens, parents, _ = _drafts(case, gen)
    seq = _spread(gen, 0, case["context"], case["requests"]) + lens
    N, W = parents.numel(), -(-case["drafts"] // 64)
    i64 = {"dtype": torch.int64, "device": "cuda"}
    return {"parents": parents, "query_start_loc": start, "seq_lens": seq.to(torch.int32),
            "tree_mask": torch.empty((N, W), **i64), "positions": torch.empty(N, **i64)}


def _pages(gen, requests, width, spare):
    """A table of different pages in random order, and how many there are."""
    pages = requests * width + spare
    return _perm(gen, pages)[: requests * width].view(requests, width).to(torch.int32).contiguous(), pages


def _attention_state(case, gen):
    """Contexts of up to `context` tokens with the drafted ones behind them,
    the pages in random order; with `pad`, rows behind the last request, one of
    several requests no longer there, and rows that see no drafted token."""
    R, C, BS = case["requests"], case["context"], case["block"]
    dt = DTYPES[case["dtype"]]
    start, lens, parents, _ = _drafts(case, gen)
    context = _spread(gen, 0, C, R)
    seq = context + lens
    if case["pad"] and R > 1:
        seq[R // 2] = 0
    N, W = parents.numel(), -(-case["drafts"] // 64)
    bits, _ = _ancestors(parents, start, case["drafts"], W)
    if case["pad"]:
        bits[::9] = 0
    table, pages = _pages(gen, R, -(-(C + case["drafts"]) // BS), 3)
    shape = (pages, BS, case["kv_heads"], case["dim"])
    caches = tuple(torch.randn(shape, generator=gen, device="cuda", dtype=dt) for _ in range(2))
    q = torch.randn((N, case["heads"], case["dim"]), generator=gen, device="cuda")
    return {"query": (1.5 * q).to(dt), "caches": caches, "table": table, "seq_lens": seq.to(torch.int32),
            "query_start_loc": start, "tree_mask": bits, "scale": case["dim"] ** -0.5,
            "output": (0.02 * torch.randn(q.shape, generator=gen, device="cuda")).to(dt),
            "lse": torch.randn(q.shape[:2], generator=gen, device="cuda")}


def _all_layers(case, gen, pages):
    """K and V of every layer in one allocation each, and the layers' caches
    as an engine holds them."""
    L, BS, H, D = case["layers"], case["block"], case["kv_heads"], case["dim"]
    shape = (L, pages, H, BS, D) if case["head_major"] else (L, pages, BS, H, D)
    both = tuple(torch.randn(shape, generator=gen, device="cuda", dtype=DTYPES[case["dtype"]]) for _ in range(2))
    k, v = (x.transpose(2, 3) if case["head_major"] else x for x in both)
    state = {"key": k, "value": v}
    if own:
        state["layers"] = _library().prepare_kv_pages([(k[i], v[i]) for i in range(L)])
    return state


def _copy_state(case, gen):
    n = case["pairs"]
    pages = 2 * n + 5
    order = _perm(gen, pages)[: 2 * n]
    s = _all_layers(case, gen, pages)
    # Several forks of one page: a quarter of the sources are others' too.
    source, target = order[:n].clone(), order[n:]
    again = n // 4
    source[:again] = source[n - again:] if again else source[:0]
    s["pages"] = torch.stack((source, target), dim=1).contiguous()
    return s


def _compact_state(case, gen):
    """Each request keeps up to `keep` of the `held` rows behind its first
    `base` ones."""
    R, n, m = case["requests"], case["held"], case["keep"]
    kept = _spread(gen, 0, m, R)
    chosen = torch.rand((R, n), generator=gen, device="cuda").argsort(dim=1)[:, :m]
    col = torch.arange(m, device="cuda")
    keep = torch.where(col < kept[:, None], chosen, n + col).sort(dim=1).values
    table, pages = _pages(gen, R, -(-(case["base"] + n) // case["block"]), 2)
    s = _all_layers(case, gen, pages)
    base = _spread(gen, 0, case["base"], R)
    i32 = torch.int32
    s.update(table=table, base_lens=base.to(i32), keep=keep.to(i32).contiguous(), keep_lens=kept.to(i32),
             seq_lens=torch.empty(R, dtype=i32, device="cuda"))
    return s


def _release_state(case, gen):
    """Requests give up to `drop` of their last tokens back; `forked` of them
    hold the pages of the request before them, which count a holder more."""
    R, BS, P = case["requests"], case["block"], case["pages"]
    width = -(-case["held"] // BS)
    held = _spread(gen, 0, case["held"], R).clamp(min=1)
    keep = (held - _spread(gen, 0, case["drop"], R)).clamp(min=0)
    table = _perm(gen, P)[: R * width].view(R, width).clone()
    forks = int(case["forked"] * R)
    refs = torch.zeros(P, dtype=torch.int64, device="cuda")
    if forks:
        child = 1 + 2 * torch.arange(min(forks, R // 2), device="cuda")
        table[child] = table[child - 1]
        refs[table[child].reshape(-1)] = 1
    cursor = R * width + 7
    i64 = {"dtype": torch.int64, "device": "cuda"}
    return {"table": table.to(torch.int32).contiguous(), "held_lens": held.to(torch.int32), "keep_lens": keep.to(torch.int32),
            "page_refs": refs.to(torch.int32), "free": _perm(gen, P + 7).to(torch.int32),
            "cursor": torch.tensor([cursor], **i64), "next_cursor": torch.empty(1, **i64)}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"tree": _plain_tree, "attention": _plain_attention, "copy": _plain_copy, "compact": _plain_compact,
            "release": _plain_release}[state["case"]["kind"]](state)


def _run_own(s):
    kind = s["case"]["kind"]
    ops = _library()
    if kind == "tree":
        ops.build_draft_tree(s["parents"], s["query_start_loc"], s["seq_lens"], s["tree_mask"], s["positions"])
        return {"tree_mask": s["tree_mask"], "positions": s["positions"]}
    if kind == "attention":
        ops.tree_attention(s["query"], s["caches"], s["table"], s["seq_lens"], s["query_start_loc"], s["tree_mask"],
                           s["scale"], s["output"], s["lse"])
        return {"output": s["output"], "lse": s["lse"]}
    if kind == "copy":
        ops.copy_kv_pages(s["layers"], s["pages"])
        return {"key": s["key"], "value": s["value"]}
    if kind == "compact":
        ops.compact_kv(s["layers"], s["table"], s["base_lens"], s["keep"], s["keep_lens"], s["seq_lens"])
        return {"key": s["key"], "value": s["value"], "seq_lens": s["seq_lens"]}
    ops.release_pages(s["table"], s["held_lens"], s["keep_lens"], s["case"]["block"], s["page_refs"], s["free"], s["cursor"],
                      s["next_cursor"])
    return {"page_refs": s["page_refs"], "free": s["free"], "next_cursor": s["next_cursor"]}


def _library():
    global _ops
    if _ops is None:
        sys.path.insert(0, os.path.join(ROOT, "lmcache-ascend_amd"))
        from lmcache_amd import c_ops

        _ops = c_ops
    return _ops


_ops = None


def _places(start, total):
    """Request and index in it of each of `total` rows, and which are one's."""
    start = start.to(torch.int64)
    t = torch.arange(total, device=start.device)
    r = torch.searchsorted(start[1:], t, right=True)
    there = r < start.numel() - 1
    r = r.clamp(max=start.numel() - 2)
    return r, t - start[r], there


def _ancestors(parents, start, most, words):
    """(bits [T, words], ancestors with the token itself): the closure of the
    parents by squaring, a request's tokens padded to `most`."""
    R = start.numel() - 1
    r, at, there = _places(start, parents.numel())
    p = parents.to(torch.int64)
    good = there & (p >= 0) & (p < at)
    a = torch.eye(most + 1, device=start.device).repeat(R, 1, 1)
    # (row and column `most` take what is no token's)
    a[r, torch.where(there, at, most).clamp(max=most), torch.where(good, p, most).clamp(max=most)] = 1.0
    a[:, most, :] = 0.0
    a[:, :, most] = 0.0
    for _ in range(max(1, most).bit_length()):
        a = (torch.bmm(a, a) > 0).float()
    rows = torch.where(there[:, None], a[r, at.clamp(max=most - 1), :most], 0.0).to(torch.int64)
    rows = torch.nn.functional.pad(rows, (0, words * 64 - most)).view(-1, words, 64)
    return (rows << torch.arange(64, device=start.device)).sum(dim=-1), rows.sum(dim=(1, 2))


def _plain_tree(s):
    c = s["case"]
    start = s["query_start_loc"]
    bits, count = _ancestors(s["parents"], start, c["drafts"], s["tree_mask"].shape[1])
    r, _, there = _places(start, s["parents"].numel())
    first = s["seq_lens"].to(torch.int64) - (start[1:] - start[:-1])
    return {"tree_mask": bits, "positions": torch.where(there, first[r] + count - 1, 0)}


def _plain_attention(s):
    """Each request's drafted tokens padded to the most, its keys to the table's."""
    c, table = s["case"], s["table"]
    BS, H, D, Q, R = c["block"], c["kv_heads"], c["dim"], c["drafts"], c["requests"]
    q = s["query"]
    N, G = q.shape[0], q.shape[1] // H
    start, seq = s["query_start_loc"].to(torch.int64), s["seq_lens"].to(torch.int64)
    lens = start[1:] - start[:-1]
    n = c["context"] + Q
    i, j = torch.arange(Q, device=q.device), torch.arange(n, device=q.device)
    row = (start[:-1, None] + i).clamp(max=N - 1)                            # [R, Q]
    page = table.to(torch.int64)[:, j // BS]
    k, v = (x[page, j % BS].float().permute(0, 2, 1, 3) for x in s["caches"])  # [R, H, n, D]
    rows = q[row].float().view(R, Q, H, G, D).permute(0, 2, 1, 3, 4).reshape(R * H, Q * G, D) * s["scale"]
    score = torch.bmm(rows, k.reshape(R * H, n, D).transpose(1, 2).contiguous()).view(R, H, Q, G, n)
    draft = j - (seq - lens)[:, None]                                        # [R, n]
    word = s["tree_mask"][row].gather(2, (draft.clamp(0, Q - 1) // 64)[:, None, :].expand(R, Q, n))
    bit = (word >> (draft.clamp(min=0) % 64)[:, None, :]) & 1
    seen = (draft < 0)[:, None] | ((bit != 0) & (draft >= 0)[:, None])
    seen = seen & (j < seq[:, None])[:, None]
    score.masked_fill_(~seen[:, None, :, None], float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score.sub_(torch.where(top == float("-inf"), 0.0, top)))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.bmm(p.view(R * H, Q * G, n), v.reshape(R * H, n, D)).view(R, H, Q, G, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(R, Q, H * G, D)
    lse = (torch.log(total) + top).permute(0, 2, 1, 3, 4).reshape(R, Q, H * G)
    r, at, there = _places(s["query_start_loc"], N)
    at = at.clamp(max=Q - 1)
    return {"output": torch.where(there[:, None, None], o[r, at].to(q.dtype), s["output"]),
            "lse": torch.where(there[:, None], lse[r, at], s["lse"])}


def _plain_copy(s):
    src, dst = s["pages"].unbind(1)
    for x in (s["key"], s["value"]):
        x[:, dst] = x[:, src]
    return {"key": s["key"], "value": s["value"]}


def _plain_compact(s):
    BS, table = s["case"]["block"], s["table"].to(torch.int64)
    base, count = s["base_lens"].to(torch.int64)[:, None], s["keep_lens"].to(torch.int64)[:, None]
    keep = s["keep"].to(torch.int64)
    col = torch.arange(keep.shape[1], device=keep.device)
    # What is past a list moves its first entry again; an empty list, nothing.
    there = col < count
    src = base + torch.where(there, keep, torch.where(count > 0, keep[:, :1], 0))
    dst = base + torch.where(there, col, 0)
    a, b = ((torch.gather(table, 1, x // BS), x % BS) for x in (src, dst))
    for x in (s["key"], s["value"]):
        x[:, b[0], b[1]] = x[:, a[0], a[1]]
    s["seq_lens"].copy_((base + count)[:, 0])
    return {"key": s["key"], "value": s["value"], "seq_lens": s["seq_lens"]}


def _plain_release(s):
    BS, table, refs, free = s["case"]["block"], s["table"].to(torch.int64), s["page_refs"], s["free"]
    P = refs.numel()
    col = torch.arange(table.shape[1], device=table.device)
    first, stop = ((s[n].to(torch.int64) + BS - 1) // BS for n in ("keep_lens", "held_lens"))
    given = (col >= first[:, None]) & (col < stop[:, None]) & (table >= 0) & (table < P)
    lost = torch.zeros(P + 1, dtype=torch.int32, device=table.device)
    lost.index_add_(0, torch.where(given, table, P).reshape(-1), torch.ones(table.numel(), dtype=torch.int32, device=table.device))
    left = refs - lost[:P]
    freed = left < 0
    rank = freed.to(torch.int64).cumsum(0)
    s["next_cursor"].copy_(s["cursor"] - rank[-1])
    at = torch.where(freed, s["next_cursor"] + rank - 1, free.numel())
    more = torch.cat((free, free[:1]))
    more[at] = torch.arange(P, dtype=torch.int32, device=table.device)
    free.copy_(more[:-1])
    refs.copy_(left.clamp(min=0))
    return {"page_refs": refs, "free": free, "next_cursor": s["next_cursor"]}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def _sum(low, high, n):
    return sum(low + (high - low) * (i + 1) // n for i in range(n))


def work(case):
    R = case.get("requests", 0)
    if case["kind"] in ("tree", "attention"):
        tokens = sum(_lens(case))
        words = -(-case["drafts"] // 64)
        if case["kind"] == "tree":
            return {"bytes": tokens * (4 + 8 * words + 8) + 8 * R, "flops": 0}
        context = _sum(0, case["context"], R)
        rows = tokens * case["heads"]
        return {"bytes": 4 * (context + tokens) * case["kv_heads"] * case["dim"] + rows * (4 * case["dim"] + 4) +
                8 * words * tokens,
                "flops": 4 * rows * case["dim"] * context // R}
    if case["kind"] == "release":
        entries = _sum(0, case["drop"], R) / case["block"]
        # (the tables' released entries, and each of their pages' counts and places)
        return {"bytes": 16 * entries + 4 * case["pages"] + 8 * R, "flops": 0}
    row = 2 * case["layers"] * case["kv_heads"] * case["dim"] * 2
    if case["kind"] == "copy":
        n = case["pairs"]
        return {"bytes": row * case["block"] * (n + n - n // 4) + 16 * n, "flops": 0}
    kept = _sum(0, case["keep"], R)
    return {"bytes": 2 * row * kept + 4 * kept + 16 * R, "flops": 0}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    if case["kind"] in ("tree", "release"):
        return None  # whole numbers
    s = prepare(case, seed)
    return {"attention": _exact_attention, "copy": _exact_copy, "compact": _exact_compact}[case["kind"]](s)


def _exact_attention(s):
    """Request by request: its keys in order, each token's from its mask."""
    c, table = s["case"], s["table"].long()
    H, D, BS = c["kv_heads"], c["dim"], c["block"]
    G = c["heads"] // H
    out, lse = s["output"].double(), s["lse"].double()
    start, seq = s["query_start_loc"].tolist(), s["seq_lens"].tolist()
    for r, n in enumerate(seq):
        t0, t1 = start[r], start[r + 1]
        q = t1 - t0
        if n <= 0:
            out[t0:t1], lse[t0:t1] = 0.0, float("-inf")
            continue
        j = torch.arange(n, device=table.device)
        k, v = (x[table[r, j // BS], j % BS].double().permute(1, 0, 2).contiguous() for x in s["caches"])
        words = s["tree_mask"][t0:t1]
        bits = torch.stack([(words[:, i // 64] >> (i % 64)) & 1 for i in range(q)], dim=1) != 0
        hidden = torch.zeros((q, n), dtype=torch.bool, device=table.device)
        hidden[:, n - q:] = ~bits
        for h in range(H):
            rows = s["query"][t0:t1, h * G: (h + 1) * G].double().reshape(q * G, D)
            score = (rows @ k[h].t().contiguous()).view(q, G, n) * s["scale"]
            score.masked_fill_(hidden[:, None, :], float("-inf"))
            low = torch.logsumexp(score, dim=-1)
            p = torch.exp(score - low.clamp(min=-1e300)[..., None])
            out[t0:t1, h * G: (h + 1) * G] = (p.view(q * G, n) @ v[h]).view(q, G, D)
            lse[t0:t1, h * G: (h + 1) * G] = low
    return {"output": out, "lse": lse}


def _exact_copy(s):
    out = {}
    for name in ("key", "value"):
        x = s[name]
        y = x.double()
        for a, b in s["pages"].tolist():
            y[:, b] = x[:, a].double()
        out[name] = y
    return out


def _exact_compact(s):
    BS, table = s["case"]["block"], s["table"].long()
    base, count = s["base_lens"].tolist(), s["keep_lens"].tolist()
    out = {"seq_lens": None}
    for name in ("key", "value"):
        x = s[name]
        y = x.double()
        for r, n in enumerate(count):
            src = base[r] + s["keep"][r, :n].long()
            dst = base[r] + torch.arange(n, device=src.device)
            y[:, table[r, dst // BS], dst % BS] = x[:, table[r, src // BS], src % BS].double()
        out[name] = y
    return out
