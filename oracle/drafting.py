"""CPU oracle for drafting and branching over the paged caches: trees of
drafted tokens, their attention, and pages copied, compacted and given back,
from their definitions.  TEST INFRASTRUCTURE ONLY."""

from __future__ import annotations

import numpy as np
import torch


def draft_tree(parents, starts, seq_lens, n_tokens, words):
    """(mask rows as Python integers below 2^(64 words), positions)."""
    mask, positions = [0] * n_tokens, [0] * n_tokens
    for r, n in enumerate(seq_lens):
        t0, t1 = int(starts[r]), int(starts[r + 1])
        above = {}
        for t in range(t0, t1):
            i, p = t - t0, int(parents[t])
            above[i] = (above[p] if 0 <= p < i else frozenset()) | {i}
            if t < n_tokens:
                fits = i < 64 * words
                mask[t] = sum(1 << j for j in above[i]) if fits else 0
                positions[t] = int(n) - (t1 - t0) + (len(above[i]) - 1 if fits else 0)
    return mask, positions


def words_of(mask, words):
    """[T, words] int64 of integers."""
    out = np.zeros((len(mask), words), np.uint64)
    for t, m in enumerate(mask):
        for w in range(words):
            out[t, w] = (m >> (64 * w)) & (2**64 - 1)
    return torch.from_numpy(out.view(np.int64))


def mask_of(rows):
    """The integers of [T, words] int64."""
    return [sum((int(x) & (2**64 - 1)) << (64 * w) for w, x in enumerate(row)) for row in rows.tolist()]


def tree_attention(q, k_cache, v_cache, table, seq_lens, starts, mask, scale, output, lse, dtype):
    """(output, lse, their tolerances) in float64; mask: integers.  k_cache,
    v_cache: [pages, block, heads, dim] tensors; rows behind the last request
    keep what `output` and `lse` hold."""
    T, Hq, D = q.shape
    pages, block, H, _ = k_cache.shape
    G = Hq // H
    out, low = output.double().numpy().copy(), lse.double().numpy().copy()
    tol_o, tol_l = np.zeros_like(out), np.zeros_like(low)
    k_cache, v_cache, qd = k_cache.double().numpy(), v_cache.double().numpy(), q.double().numpy()
    half = torch.finfo(dtype).eps / 2
    for r, n in enumerate(seq_lens):
        t0, t1 = int(starts[r]), min(int(starts[r + 1]), T)
        context = int(n) - (int(starts[r + 1]) - t0)
        there = []
        for j in range(min(int(n), len(table[r]) * block)):
            page = int(table[r][j // block])
            if 0 <= page < pages:
                there.append((j, page, j % block))
        for t in range(t0, t1):
            rows = [(p, a) for j, p, a in there if j < context or (mask[t] >> (j - context)) & 1]
            if not rows:
                out[t], low[t] = 0.0, -np.inf
                continue
            pg, at = np.array(rows).T
            k, v = k_cache[pg, at], v_cache[pg, at]              # [n, H, D]
            for h in range(Hq):
                kh, vh = k[:, h // G], v[:, h // G]
                s = kh @ qd[t, h] * scale
                # 32-bit sums of D products, and the exponent's argument.
                ds = scale * D * 2.0**-24 * (np.abs(kh) @ np.abs(qd[t, h])).max() + 2.0**-21 * np.abs(s).max()
                m = s.max()
                e = np.exp(s - m)
                p = e / e.sum()
                low[t, h] = m + np.log(e.sum())
                out[t, h] = p @ vh
                spread = p @ np.abs(vh)
                # p is rounded to the type once (fp16 below 2^-14 by 2^-25
                # of the largest), the result once; sums in 32 bits.
                tol_o[t, h] = (half + 2.2 * ds + 2.0**-18) * spread + half * np.abs(out[t, h])
                if dtype == torch.float16:
                    tol_o[t, h] += 2.0**-25 * (np.abs(vh).sum(0) / e.sum() + 1.0)
                tol_l[t, h] = ds + 2.0**-18 * (1.0 + abs(low[t, h]))
    return out, low, tol_o, tol_l


def copy_pages(planes, pairs):
    """Planes ([layers, pages, ...] tensors) after the copies."""
    out = [x.clone() for x in planes]
    for a, b in pairs:
        for x, y in zip(planes, out):
            if 0 <= a < x.shape[1] and 0 <= b < x.shape[1]:
                y[:, b] = x[:, a]
    return out


def compact(planes, table, base, keep, keep_lens):
    """Planes ([layers, pages, block, ...] tensors) after the moves."""
    out = [x.clone() for x in planes]
    pages, block = planes[0].shape[1:3]

    def place(r, pos):
        if pos < 0 or pos // block >= len(table[r]) or not 0 <= table[r][pos // block] < pages:
            return None
        return int(table[r][pos // block]), pos % block

    for r, n in enumerate(keep_lens):
        for i in range(min(max(0, int(n)), len(keep[r]))):
            a, b = place(r, int(base[r]) + int(keep[r][i])), place(r, int(base[r]) + i)
            if a and b:
                for x, y in zip(planes, out):
                    y[:, b[0], b[1]] = x[:, a[0], a[1]]
    return out


def release(table, held, keep, block, refs, free, cursor):
    """(refs, free, next cursor)."""
    refs, free = list(refs), list(free)
    for row, h, k in zip(table, held, keep):
        for j in range(-(-max(0, k) // block), min(len(row), -(-max(0, h) // block))):
            if 0 <= row[j] < len(refs):
                refs[row[j]] -= 1
    given = [p for p, n in enumerate(refs) if n < 0]
    cursor = min(cursor, len(free))
    for i, p in enumerate(given):
        refs[p] = 0
        if 0 <= cursor - len(given) + i < len(free):
            free[cursor - len(given) + i] = p
    return refs, free, cursor - len(given)
