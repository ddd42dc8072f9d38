"""shared_prefix_attention where its work is cut into long and into many parts,
over blocks of any size, and captured with every head size: against softmax
attention in 64 bits (tolerances: oracle.serving.attention, derived there)."""

import numpy as np
import pytest
import torch

from oracle import serving as osv

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    import lmcache_amd

    return lmcache_amd.c_ops


def _case(seed, q_lens, own, P, block, Hq, Hk, dim, dtype=BF16, table_keys=0, pad=0):
    """Requests of `own` keys behind P shared ones (own < 0: inside the prefix;
    None: not there).  The table spans `table_keys` keys at least, blocks are
    dealt to the requests as far as they reach, and rows that no token sees
    hold NaN."""
    gen = torch.Generator().manual_seed(seed)
    seq = [0 if n is None else P + n for n in own]
    n_shared = -(-P // block)
    width = -(-max([P, 1, table_keys] + seq) // block)
    first = P // block
    need = [max(0, -(-n // block) - first) for n in seq]
    pages = n_shared + sum(need) + 3
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    shared = order[:n_shared].clone()
    table = torch.randint(-5, 2 * pages, (len(seq), width), generator=gen, dtype=torch.int32)
    k, v = (torch.full((pages, block, Hk, dim), float("nan"), dtype=dtype) for _ in range(2))
    flat_k, flat_v = k.view(-1, Hk, dim), v.view(-1, Hk, dim)

    def fill(blocks, lo, hi):
        j = torch.arange(lo, hi)
        at = blocks.long()[j // block] * block + j % block
        for x in (flat_k, flat_v):
            x[at] = torch.randn((len(j), Hk, dim), generator=gen).to(dtype)

    fill(shared, 0, P)
    at = n_shared
    for r, n in enumerate(seq):
        table[r, first: first + need[r]] = order[at: at + need[r]]
        at += need[r]
        if n > P:
            fill(table[r], P, n)
    starts = torch.zeros(len(seq) + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(q_lens, dtype=torch.int32).cumsum(0)
    T = int(starts[-1]) + pad
    return {"q": torch.randn((T, Hq, dim), generator=gen).to(dtype), "k": k, "v": v, "shared": shared, "P": P, "table": table,
            "seq": torch.tensor(seq, dtype=torch.int32), "starts": starts, "scale": dim ** -0.5,
            "out": torch.randn((T, Hq, dim), generator=gen).to(dtype), "lse": torch.randn((T, Hq), generator=gen), "dtype": dtype}


def _device(c):
    return {n: x.to(DEV) if torch.is_tensor(x) else x for n, x in c.items()}


def _call(ops, d):
    ops.shared_prefix_attention(d["q"], (d["k"], d["v"]), d["shared"], d["P"], d["table"], d["seq"], d["starts"], d["scale"],
                                d["out"], d["lse"])


def _want(c):
    return osv.attention(c["q"], c["k"], c["v"], c["shared"], c["P"], c["table"].tolist(), c["seq"].tolist(),
                         c["starts"].tolist(), c["scale"], c["out"], c["lse"], c["dtype"])


def _hold(want, out, lse):
    o, low, tol_o, tol_l = want
    err = np.abs(out.double().cpu().numpy() - o)
    assert not np.isnan(err).any() and (err <= tol_o).all(), (np.nanmax(err - tol_o), np.isnan(err).sum())
    got, fine = lse.double().cpu().numpy(), np.isfinite(low)
    assert np.array_equal(got[~fine], low[~fine])
    over = np.abs(got[fine] - low[fine]) - tol_l[fine]
    assert (over <= 0).all(), np.nanmax(over)


def _check(ops, c):
    d = _device(c)
    _call(ops, d)
    torch.cuda.synchronize()
    _hold(_want(c), d["out"], d["lse"])
    return d


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_wide_tiles_over_several_parts(ops, dtype, dim):
    """160 rows a KV head over five parts of 320 shared keys, the last one
    short; requests inside the prefix, and one that is not there."""
    rng = np.random.default_rng(dim)
    own = [int(x) for x in rng.integers(1, 90, 80)]
    own[3], own[17], own[40], own[60] = None, -1, -700, -1499
    _check(ops, _case(dim, [1] * 80, own, 1511, 16, 4, 2, dim, dtype, pad=2))


# Many requests of which most have no new token: their own keys are taken to
# be most of the work, so the prefix is one part.
def _sparse(n, R=600):
    q = [0] * R
    for i in range(n):
        q[i * R // n] = 1
    return q


def _own(q, most, seed):
    rng = np.random.default_rng(seed)
    return [int(rng.integers(1, most)) if n else None for n in q]


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 128)])
@pytest.mark.parametrize("holes", [False, True])
def test_one_wide_part_of_thousands_of_keys(ops, dtype, dim, holes):
    """More than two times the 1024 keys of a part whose blocks are looked up
    at once; with blocks outside the caches behind the first 1024."""
    q = _sparse(80)
    c = _case(1, q, _own(q, 40, 1), 2317, 16, 4, 4, dim, dtype, table_keys=2317 + 1100)
    if holes:
        c["shared"][[70, 71, 100, 128, 144]] = torch.tensor([-1, c["k"].shape[0], -7, 2**31 - 1, -1], dtype=torch.int32)
    _check(ops, c)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 192])
def test_wide_tiles_with_blocks_outside_the_caches(ops, dtype, dim):
    c = _case(2, [1] * 80, [1 + i % 50 for i in range(80)], 700, 16, 4, 2, dim, dtype)
    for i, page in ((0, -1), (5, c["k"].shape[0]), (6, 2**31 - 1), (30, -3), (43, -1)):
        c["shared"][i] = page
    c["table"][::7, 44] = -1
    _check(ops, c)
    c["shared"][:] = -1
    _check(ops, c)


@pytest.mark.parametrize("dim", [64, 128])
def test_narrow_prefix_parts_of_several_blocks_a_wave(ops, dim):
    """60 rows a KV head: three parts of 512 keys; one part of 5120 keys, more
    than the 4096 that are looked up at once."""
    _check(ops, _case(3, [1] * 60, [1 + i for i in range(60)], 1403, 16, 8, 8, dim, table_keys=2500))
    q = _sparse(60, 1300)
    c = _case(4, q, _own(q, 30, 4), 5003, 16, 4, 4, dim, table_keys=6100)
    c["shared"][[260, 300]] = -1
    _check(ops, c)


def test_own_parts_of_more_keys_than_are_looked_up_at_once(ops):
    """9000 own keys in eight parts of some 1150, blocks outside the caches
    among the late ones; the other requests are short."""
    own = [1 + i % 20 for i in range(64)]
    own[11], own[40] = 9000, 2500
    c = _case(5, [1] * 64, own, 100, 16, 8, 8, 64, table_keys=9200)
    c["table"][11, [20, 75, 76, 150, 560]] = -1
    _check(ops, c)


@pytest.mark.parametrize("block", [1, 8, 24, 40, 17])
@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 96), (BF16, 128)])
def test_blocks_that_are_no_multiple_of_16_keys(ops, block, dtype, dim):
    """Looked up key by key: a narrow tile, several tokens a request, and wide
    tiles, with blocks outside the caches in all of them."""
    for seed, q, own, P, Hq, Hk in ((6, [1, 3, 1], [70, 41, 5], 203, 4, 2), (7, [1] * 70, [1 + i % 40 for i in range(70)], 330, 2, 2)):
        c = _case(seed, q, own, P, block, Hq, Hk, dim, dtype, pad=1)
        _check(ops, c)
        c["shared"][150 // block] = -1
        c["table"][0, (P + 20) // block] = c["k"].shape[0]
        _check(ops, c)


def test_several_parts_give_the_same_each_time(ops):
    c = _case(8, [1] * 70, [1 + 3 * i for i in range(70)], 1800, 16, 8, 2, 128)
    want = _want(c)
    first = None
    for _ in range(4):
        d = _device(c)
        _call(ops, d)
        torch.cuda.synchronize()
        _hold(want, d["out"], d["lse"])
        if first is not None:
            assert torch.equal(d["out"], first["out"]) and torch.equal(d["lse"], first["lse"])
        first = d


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("R", [5, 70])
def test_captured_calls_of_every_head_size(ops, dim, R):
    """Narrow and wide tiles, each replayed several times on the rows and
    lengths of its time, with eager calls between."""
    c = _case(dim + R, [1] * R, [20 + i % 30 for i in range(R)], 600, 16, 4, 2, dim)
    d = _device(c)
    _call(ops, d)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _call(ops, d)
    for turn in range(3):
        now = dict(c, q=torch.randn(c["q"].shape, generator=torch.Generator().manual_seed(turn)).to(c["dtype"]),
                   seq=(c["seq"] - 5 * turn).clamp(min=c["P"] + 1))
        d["q"].copy_(now["q"])
        d["seq"].copy_(now["seq"])
        g.replay()
        torch.cuda.synchronize()
        eager = _device(now)
        _call(ops, eager)
        torch.cuda.synchronize()
        assert torch.equal(eager["out"], d["out"]) and torch.equal(eager["lse"], d["lse"])
        _hold(_want(now), d["out"], d["lse"])


@pytest.mark.parametrize("dim", [64, 128])
def test_one_token_of_a_projection_of_odd_width(ops, dim):
    """The stride of a dim of one entry is not used: one token, one head."""
    c = _case(9, [1], [37], 90, 16, 4, 1, dim)
    d = _device(c)
    wide = torch.zeros((1, 4 * dim + 3), dtype=BF16, device=DEV)
    wide[:, : 4 * dim] = d["q"].view(1, -1)
    d["q"] = torch.as_strided(wide, (1, 4, dim), (4 * dim + 3, dim, 1))
    d["out"] = torch.as_strided(d["out"], (1, 4, dim), (5, dim, 1))
    for x in "kv":
        d[x] = torch.as_strided(d[x], d[x].shape, (16 * dim, dim, 7, 1))
    _call(ops, d)
    torch.cuda.synchronize()
    _hold(_want(c), d["out"], d["lse"])
