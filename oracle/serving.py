"""CPU oracle for the serving operators: slot mappings, rotary positions and
shared-prefix attention, from their definitions, in 64 bits, one request or
token at a time.  TEST INFRASTRUCTURE ONLY."""

from __future__ import annotations

import numpy as np
import torch

I32_MAX = 2**31 - 1


def slot_mapping(query, context, table, block, n_tokens, free=None, cursor=0):
    """(slots, positions, query_start_loc, seq_lens, table, next_cursor)."""
    query = [max(0, int(x)) for x in query]
    context = [max(0, int(x)) for x in context]
    table = np.array(table, dtype=np.int64, copy=True)
    width = table.shape[1]
    slots = np.full(n_tokens, -1, np.int64)
    positions = np.zeros(n_tokens, np.int64)
    starts, at = [0], cursor
    for r, (q, c) in enumerate(zip(query, context)):
        if free is not None:
            have, need = min(width, -(-c // block)), min(width, -(-(c + q) // block))
            for j in range(have, need):
                table[r, j] = free[at] if 0 <= at < len(free) else -1
                at += 1
        for i in range(min(q, max(0, n_tokens - starts[-1]))):
            t, pos = starts[-1] + i, c + i
            positions[t] = pos
            if pos // block < width and table[r, pos // block] >= 0:
                slots[t] = table[r, pos // block] * block + pos % block
        starts.append(min(I32_MAX, starts[-1] + q))
    seq = [min(I32_MAX, c + q) for q, c in zip(query, context)]
    return slots, positions, np.array(starts), np.array(seq), table, at


def rotate(x, positions, inv_freq, dim, neox, offset=0, scale=1.0, inverse=False):
    """Rows [T, heads * dim] (float64) turned; also |x1| + |x2| of each
    rotated element's pair (0 elsewhere), which bounds its rounding."""
    y = np.array(x, np.float64).reshape(x.shape[0], -1, dim)
    size = np.zeros_like(y)
    n = len(inv_freq)
    a = offset + (np.arange(n) if neox else 2 * np.arange(n))
    b = a + (n if neox else 1)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)[None, :]
    c, s = scale * np.cos(angle)[:, None], scale * np.sin(angle)[:, None] * (-1.0 if inverse else 1.0)
    x1, x2 = y[:, :, a].copy(), y[:, :, b].copy()
    y[:, :, a], y[:, :, b] = x1 * c - x2 * s, x2 * c + x1 * s
    size[:, :, a] = size[:, :, b] = (np.abs(x1) + np.abs(x2)) * abs(scale)
    return y.reshape(x.shape), size.reshape(x.shape)


def rotary_tolerance(want, size, dtype):
    """One rounding to the type (half a step; 2^-25 below fp16's normal
    range), and in 32 bits: cos and sin to 1.3e-7 and their product with scale
    2^-24, the two products and the sum 2^-24 each of what they join, the
    angle's 64 bits nothing beside these: under 4.5e-7 of |x1| + |x2|."""
    return torch.finfo(dtype).eps / 2 * np.abs(want) + 4.5e-7 * size + (2.0**-25 if dtype == torch.float16 else 0.0)


def attention(q, k_cache, v_cache, shared, shared_len, table, seq_lens, starts, scale, output, lse, dtype):
    """(output, lse, their tolerances) in float64.  k_cache, v_cache: [pages,
    block, heads, dim] tensors; rows behind the last request keep what
    `output` and `lse` hold."""
    T, Hq, D = q.shape
    pages, block, H, _ = k_cache.shape
    G = Hq // H
    out, low = output.double().numpy().copy(), lse.double().numpy().copy()
    tol_o, tol_l = np.zeros_like(out), np.zeros_like(low)
    k_cache, v_cache, qd = k_cache.double().numpy(), v_cache.double().numpy(), q.double().numpy()
    half = torch.finfo(dtype).eps / 2
    for r, n in enumerate(seq_lens):
        t0, t1 = int(starts[r]), int(starts[r + 1])
        for t in range(t0, t1):
            last = int(n) - (t1 - t0) + (t - t0)
            rows = []
            for j in range(last + 1):
                b = j // block
                if j < shared_len:
                    page = int(shared[b])
                else:
                    page = int(table[r][b]) if b < len(table[r]) else -1
                if 0 <= page < pages:
                    rows.append((page, j % block))
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
