"""tree_attention against softmax attention in 64 bits, one token and head at a
time (tolerances: oracle.drafting.tree_attention, derived there)."""

import numpy as np
import pytest
import torch

from oracle import drafting as od

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops():
    import lmcache_amd

    return lmcache_amd.c_ops


def _case(seed, q_lens, contexts, block, Hq, Hk, dim, dtype=torch.bfloat16, fmt="separate", pad=0, words=None, spread=1.0,
          density=0.4):
    """Caches, tables and rows on the CPU; masks with any bits, those of other
    tokens and those past the request's among them.  Rows of the caches that
    no token sees hold NaN."""
    gen = torch.Generator().manual_seed(seed)
    R = len(q_lens)
    seq = [c + q for c, q in zip(contexts, q_lens)]
    width = max(1, -(-max([0] + seq) // block))
    words = words if words is not None else max(1, -(-max(q_lens) // 64))
    pages = R * width + 3
    table = torch.randperm(pages, generator=gen).to(torch.int32)[: R * width].reshape(R, width).clone()
    starts = torch.zeros(R + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(q_lens, dtype=torch.int32).cumsum(0)
    T = int(starts[-1]) + pad
    bits = torch.rand((T, words * 64), generator=gen) < density
    for r, n in enumerate(q_lens):
        for i in range(n):
            if i < words * 64 and (i + r) % 5:
                bits[int(starts[r]) + i, i] = True
    mask = [sum(1 << int(j) for j in row.nonzero().flatten()) for row in bits]
    k, v = (torch.full((pages, block, Hk, dim), NAN, dtype=dtype) for _ in range(2))
    for r, n in enumerate(seq):
        for j in range(n):
            i = j - contexts[r]
            if i >= 0 and not any((mask[int(starts[r]) + x] >> i) & 1 for x in range(q_lens[r])):
                continue
            page, at = int(table[r, j // block]), j % block
            k[page, at] = (spread * torch.randn((Hk, dim), generator=gen)).to(dtype)
            v[page, at] = torch.randn((Hk, dim), generator=gen).to(dtype)
        # Tables past a request's end hold anything.
        used = -(-max(0, n) // block)
        table[r, used:] = torch.randint(-5, 2 * pages, (width - used,), generator=gen, dtype=torch.int32)
    q = torch.randn((T, Hq, dim), generator=gen).to(dtype)
    return {"q": q, "k": k, "v": v, "table": table, "seq": torch.tensor(seq, dtype=torch.int32), "starts": starts,
            "mask": mask, "words": words, "scale": dim ** -0.5, "fmt": fmt, "dtype": dtype,
            "out": torch.randn((T, Hq, dim), generator=gen).to(dtype), "lse": torch.randn((T, Hq), generator=gen)}


def _device_caches(c):
    k, v, fmt = c["k"], c["v"], c["fmt"]
    if fmt == "separate":
        return (k.to(DEV), v.to(DEV)), {}
    if fmt == "head_major":
        return tuple(x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for x in (k, v)), {}
    if fmt == "merged":
        return torch.stack((k, v), dim=1).to(DEV), {"kvcache_format_raw": 1}
    return torch.stack((k, v), dim=0).to(DEV), {"kvcache_format_raw": 1, "vllm_two_major": True}


def _call(ops, c, caches, kw, q, out, lse):
    ops.tree_attention(q, caches, c["table"].to(DEV), c["seq"].to(DEV), c["starts"].to(DEV),
                       od.words_of(c["mask"], c["words"]).to(DEV), c["scale"], out, lse, **kw)


def _want(c):
    return od.tree_attention(c["q"], c["k"], c["v"], c["table"].tolist(), c["seq"].tolist(), c["starts"].tolist(),
                             c["mask"], c["scale"], c["out"], c["lse"], c["dtype"])


def _hold(out, lse, want):
    o, low, tol_o, tol_l = want
    err = np.abs(out.double().cpu().numpy() - o)
    assert not np.isnan(err).any() and (err <= tol_o).all(), (np.nanmax(err - tol_o), np.isnan(err).sum())
    if lse is not None:
        got = lse.double().cpu().numpy()
        fine = np.isfinite(low)
        assert np.array_equal(got[~fine], low[~fine])
        assert (np.abs(got[fine] - low[fine]) <= tol_l[fine]).all(), np.nanmax(np.abs(got[fine] - low[fine]) - tol_l[fine])


def _check(ops, c, with_lse=True):
    caches, kw = _device_caches(c)
    out, lse = c["out"].to(DEV), c["lse"].to(DEV) if with_lse else None
    _call(ops, c, caches, kw, c["q"].to(DEV), out, lse)
    torch.cuda.synchronize()
    _hold(out, lse, _want(c))
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("contexts,block", [([0, 0, 0], 16), ([1, 63, 0], 16), ([64, 65, 57], 64), ([300, 3, 129], 48),
                                            ([517, 0, 255], 128)])
def test_lengths_and_dims(ops, dtype, dim, contexts, block):
    _check(ops, _case(dim + sum(contexts), [8, 1, 5], contexts, block, 4, 2, dim, dtype))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (8, 8), (8, 2), (7, 1), (10, 2), (33, 1)])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [3, 0, 5, 1], [40, 2], [0, 0], [66]])
def test_heads_and_tree_sizes(ops, dim, Hq, Hk, q_lens):
    _check(ops, _case(Hq, q_lens, [70 + 13 * i for i in range(len(q_lens))], 16, Hq, Hk, dim, pad=2))


@pytest.mark.parametrize("fmt", ["head_major", "merged", "two_major"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cache_layouts(ops, fmt, dtype):
    _check(ops, _case(5, [9, 4, 20], [150, 97, 31], 16, 8, 2, 128, dtype, fmt, pad=1))


@pytest.mark.parametrize("block", [1, 5, 24, 200])
def test_blocks_that_are_not_whole_groups(ops, block):
    _check(ops, _case(block, [6, 17], [120, 33], block, 4, 1, 64))


@pytest.mark.parametrize("Hq,Hk,dim", [(16, 1, 64), (8, 2, 128), (4, 1, 96)])
@pytest.mark.parametrize("q_lens,contexts", [([70, 1, 90], [200, 900, 10]), ([130, 65, 257], [64, 1, 500])])
def test_wide_trees_and_several_row_tiles(ops, Hq, Hk, dim, q_lens, contexts):
    """Rows of a request and KV head over one tile, of 128 and of 256 rows."""
    _check(ops, _case(7, q_lens, contexts, 32, Hq, Hk, dim))


@pytest.mark.parametrize("words", [0, 1, 2, 4])
def test_masks_narrower_and_wider_than_the_trees(ops, words):
    _check(ops, _case(words, [100, 3], [90, 64], 16, 4, 2, 64, words=words))


@pytest.mark.parametrize("Hk", [1, 3, 8])
def test_long_contexts_are_cut_and_joined(ops, Hk):
    """One long request, many pieces a tile; then one among short ones."""
    _check(ops, _case(1, [6], [4100], 16, Hk, Hk, 64))
    _check(ops, _case(2, [3, 5, 2, 4], [1, 2900, 0, 130], 32, 2 * Hk, Hk, 64, torch.float16))


def test_many_requests(ops):
    gen = torch.Generator().manual_seed(3)
    q_lens = torch.randint(0, 4, (600,), generator=gen).tolist()
    contexts = torch.randint(0, 100, (600,), generator=gen).tolist()
    _check(ops, _case(3, q_lens, contexts, 16, 2, 1, 64, pad=3))


def test_rows_that_see_nothing(ops):
    c = _case(11, [4, 3, 2], [0, 30, 0], 16, 4, 2, 64)
    c["mask"][0] = c["mask"][4] = c["mask"][8] = 0
    c["mask"][2] = 1 << 40                      # a bit past the request's tokens
    c["seq"][2] = 0                             # a request that is no longer there
    out = _check(ops, c)
    assert (out[0] == 0).all() and (out[2] == 0).all() and (out[7:9] == 0).all() and (out[4] != 0).any()


def test_drafts_before_the_caches_first_row(ops):
    """seq_lens under the drafted tokens: the first of them have no row."""
    c = _case(12, [6, 5], [3, 0], 16, 2, 2, 64)
    c["seq"] = torch.tensor([4, 2], dtype=torch.int32)
    c["k"].nan_to_num_(0.5)
    c["v"].nan_to_num_(0.25)
    _check(ops, c)


def test_sequences_longer_than_the_table(ops):
    c = _case(13, [5, 4], [60, 40], 16, 2, 2, 64)
    c["seq"] += 2000
    c["k"].nan_to_num_(0.5)
    c["v"].nan_to_num_(0.25)
    _check(ops, c)


@pytest.mark.parametrize("bad", [-1, -(2**31), 2**31 - 1, 10**6])
def test_blocks_outside_the_caches_are_unseen(ops, bad):
    c = _case(14, [7, 3], [100, 200], 16, 4, 2, 128)
    c["table"][0, 2] = bad
    c["table"][1, 0] = bad
    c["table"][1, 12] = bad                     # with drafted tokens
    _check(ops, c)


@pytest.mark.parametrize("odd", [INF, -INF, NAN])
def test_what_a_row_does_not_see_is_not_used(ops, odd):
    """Infinities and NaN in rows of K and V that some rows see and others do
    not: only those that see them get them."""
    c = _case(15, [6], [50], 16, 2, 1, 64, density=0.0)
    c["mask"] = [1 << i | (1 if i % 2 else 0) for i in range(6)]
    c["k"].nan_to_num_(0.5)                     # (every drafted token's row is seen)
    c["v"].nan_to_num_(0.25)
    page, at = int(c["table"][0, 3]), 2         # key 50: the first drafted token
    c["v"][page, at, 0, 5] = odd
    caches, kw = _device_caches(c)
    out = c["out"].to(DEV)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, None)
    torch.cuda.synchronize()
    got = out.float().cpu()
    sees = torch.tensor([True if i % 2 or i == 0 else False for i in range(6)])
    assert torch.isfinite(got[~sees]).all()
    column = got[sees][:, :, 5]
    assert torch.isnan(column).all() if odd != odd else (column == odd).all()
    c["v"][page, at, 0, 5] = 0.0
    rest = _want(c)
    keep = np.ones(64, bool)
    keep[5] = False
    err = np.abs(got.double().numpy() - rest[0])
    assert (err[:, :, keep] <= rest[2][:, :, keep]).all()
    assert (err[~sees.numpy()] <= rest[2][~sees.numpy()]).all()


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("q,Hq", [(40, 1), (60, 2), (60, 4)])
@pytest.mark.parametrize("odd", [INF, NAN])
def test_odd_values_anywhere_in_a_block(ops, dim, q, Hq, odd):
    """Tiles of every shape: each of several drafted keys, odd in one dim, is
    seen by one token alone."""
    c = _case(30 + dim, [q], [45], 16, Hq, 1, dim, density=0.0)
    c["k"].nan_to_num_(0.5)
    c["v"].nan_to_num_(0.25)
    c["mask"] = [1 << i for i in range(q)]
    put = {0: 0, 7: dim - 1, 18: dim // 2, 19: dim // 2 - 1, q - 1: 31, q - 9: dim - 33}
    for i, d in put.items():
        c["v"][int(c["table"][0, (45 + i) // 16]), (45 + i) % 16, 0, d] = odd
    caches, kw = _device_caches(c)
    out = c["out"].to(DEV)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, None)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    for i, d in put.items():
        c["v"][int(c["table"][0, (45 + i) // 16]), (45 + i) % 16, 0, d] = 0.0
    want, _, tol, _ = _want(c)
    hit = np.zeros_like(got, dtype=bool)
    for i, d in put.items():
        hit[i, :, d] = True
    assert (np.isnan(got[hit]) if odd != odd else got[hit] == INF).all()
    assert (np.abs(got - want)[~hit] <= tol[~hit]).all()


@pytest.mark.parametrize("R", [63, 64, 65, 256, 257])
def test_numbers_of_requests(ops, R):
    """Up to 64 requests are summed up in another way than more."""
    gen = torch.Generator().manual_seed(R)
    q_lens = torch.randint(0, 4, (R,), generator=gen).tolist()
    contexts = torch.randint(0, 90, (R,), generator=gen).tolist()
    contexts[R // 2] = 1200
    _check(ops, _case(R, q_lens, contexts, 16, 2, 2, 64, pad=1))


def test_a_key_of_infinities_hidden_from_some(ops):
    c = _case(16, [4], [20], 16, 2, 1, 64, density=0.0)
    c["mask"] = [1, 2, 4, 8]
    c["k"].nan_to_num_(0.5)                     # (every drafted token's row is seen)
    c["v"].nan_to_num_(0.25)
    c["k"][int(c["table"][0, 1]), 5] = INF      # key 21: seen by token 1 alone
    caches, kw = _device_caches(c)
    out, lse = c["out"].to(DEV), c["lse"].to(DEV)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, lse)
    torch.cuda.synchronize()
    c["k"][int(c["table"][0, 1]), 5] = 0.0
    want = _want(c)
    others = [0, 2, 3]
    assert (np.abs(out.double().cpu().numpy() - want[0])[others] <= want[2][others]).all()


def test_scores_of_minus_infinity(ops):
    """A token whose every score is -infinity: zeros, and an lse of -infinity."""
    c = _case(17, [2, 1], [10, 4], 16, 1, 1, 64)
    c["q"].fill_(1.0)
    for j in range(4 + 1):
        c["k"][int(c["table"][1, 0]), j] = -INF
    caches, kw = _device_caches(c)
    out, lse = c["out"].to(DEV), c["lse"].to(DEV)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, lse)
    torch.cuda.synchronize()
    assert (out[2] == 0).all() and (lse[2] == -INF).all()


def test_no_weight_beside_infinite_values(ops):
    """Scores of -infinity leave zeros, whatever the values that go with them."""
    c = _case(25, [1, 3], [20, 4], 16, 1, 1, 64)
    c["q"].fill_(1.0)
    c["k"].nan_to_num_(0.5)
    c["v"].nan_to_num_(0.25)
    for j in range(7):
        c["k"][int(c["table"][1, 0]), j] = -INF
    c["v"][int(c["table"][1, 0]), 5] = INF
    c["mask"][1:] = [1, 3, 7]
    caches, kw = _device_caches(c)
    out, lse = c["out"].to(DEV), c["lse"].to(DEV)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, lse)
    torch.cuda.synchronize()
    assert (out[1:] == 0).all() and (lse[1:] == -INF).all()


def test_two_calls_at_once(ops):
    """Calls on two streams work in scratch of their own."""
    cases = [_case(26 + i, [40, 9], [700, 1500], 16, 8, 2, 64) for i in range(2)]
    args = [(_device_caches(c)[0], c["q"].to(DEV), c["out"].to(DEV), c["lse"].to(DEV)) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, (caches, q, out, lse), s in zip(cases, args, streams):
            with torch.cuda.stream(s):
                _call(ops, c, caches, {}, q, out, lse)
    torch.cuda.synchronize()
    for c, (_, _, out, lse) in zip(cases, args):
        _hold(out, lse, _want(c))


def test_large_scores(ops):
    _check(ops, _case(18, [9, 70], [200, 64], 16, 8, 2, 128, spread=20.0))


def test_a_chain_is_what_shared_prefix_attention_gives(ops):
    c = _case(19, [5, 1, 9], [100, 30, 64], 16, 8, 2, 128, density=0.0)
    c["k"].nan_to_num_(0.5)
    c["v"].nan_to_num_(0.25)
    at = [i for n in (5, 1, 9) for i in range(n)]
    c["mask"] = [(1 << (i + 1)) - 1 for i in at]
    out = _check(ops, c)
    causal = torch.empty_like(out)
    caches, _ = _device_caches(c)
    ops.shared_prefix_attention(c["q"].to(DEV), caches, torch.zeros(0, dtype=torch.int32, device=DEV), 0, c["table"].to(DEV),
                                c["seq"].to(DEV), c["starts"].to(DEV), c["scale"], causal)
    want = _want(c)
    assert (np.abs(causal.double().cpu().numpy() - want[0]) <= want[2]).all()


def test_strided_rows_and_output_over_the_query(ops):
    c = _case(20, [9, 30], [70, 33], 16, 4, 2, 64, pad=2)
    T = c["q"].shape[0]
    caches, kw = _device_caches(c)
    want = _want(c)
    # Columns of a fused projection, the output beside the query.
    wide = torch.zeros((T, 4, 3, 64), dtype=c["dtype"], device=DEV)
    wide[:, :, 0], wide[:, :, 1], wide[:, :, 2] = c["q"].to(DEV), c["out"].to(DEV), 5.0
    low = torch.zeros((4, T), device=DEV).t()
    low.copy_(c["lse"])
    _call(ops, c, caches, kw, wide[:, :, 0], wide[:, :, 1], low)
    torch.cuda.synchronize()
    _hold(wide[:, :, 1], low, want)
    assert (wide[:, :, 2] == 5.0).all() and torch.equal(wide[:, :, 0].cpu(), c["q"])
    over = c["q"].to(DEV)
    _call(ops, c, caches, kw, over, over, None)
    torch.cuda.synchronize()
    n = int(c["starts"][-1])
    assert torch.equal(over[:n], wide[:n, :, 1]) and torch.equal(over[n:].cpu(), c["q"][n:])


def test_masks_as_columns_of_a_buffer(ops):
    c = _case(21, [70, 5], [40, 3], 16, 2, 1, 64)
    space = torch.full((75, 5), -1, dtype=torch.int64, device=DEV)
    space[:, 1:3] = od.words_of(c["mask"], 2).to(DEV)
    caches, _ = _device_caches(c)
    out, lse = c["out"].to(DEV), c["lse"].to(DEV)
    ops.tree_attention(c["q"].to(DEV), caches, c["table"].to(DEV), c["seq"].to(DEV), c["starts"].to(DEV), space[:, 1:3],
                       c["scale"], out, lse)
    torch.cuda.synchronize()
    _hold(out, lse, _want(c))


def test_the_same_call_gives_the_same_bits(ops):
    c = _case(22, [30, 5, 64], [900, 2000, 10], 16, 8, 2, 128)
    a = _check(ops, c)
    assert torch.equal(a, _check(ops, c))


@pytest.mark.parametrize("dim,Hq,q_lens", [(64, 4, [6, 2]), (96, 8, [40, 30]), (128, 4, [8, 5]), (192, 2, [3, 3]), (256, 2, [2, 2])])
def test_captured_with_other_work_between_the_replays(ops, dim, Hq, q_lens):
    c = _case(23, q_lens, [300, 90], 16, Hq, 1, dim)
    caches, _ = _device_caches(c)
    q, table, seq, starts = (c[n].to(DEV) for n in ("q", "table", "seq", "starts"))
    mask = od.words_of(c["mask"], c["words"]).to(DEV)
    out, lse = torch.zeros_like(c["out"], device=DEV), torch.zeros_like(c["lse"], device=DEV)

    def call(o, e):
        ops.tree_attention(q, caches, table, seq, starts, mask, c["scale"], o, e)

    call(out, lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, lse)
    gen = torch.Generator().manual_seed(1)
    for n in range(4):
        q.copy_(torch.randn(q.shape, generator=gen).to(q.dtype))
        seq.copy_(c["seq"] - torch.tensor([37 * n, 11 * n], dtype=torch.int32))
        caches[0].nan_to_num_(0.5)
        caches[1].nan_to_num_(0.25)
        out.fill_(7.0)
        graph.replay()
        o, e = torch.zeros_like(out), torch.zeros_like(lse)
        call(o, e)
        torch.cuda.synchronize()
        assert torch.equal(out, o) and torch.equal(lse, e)


def test_on_another_stream(ops):
    c = _case(24, [6, 6], [500, 20], 16, 4, 2, 64)
    caches, kw = _device_caches(c)
    out, q = c["out"].to(DEV), c["q"].to(DEV)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        _call(ops, c, caches, kw, q, out, None)
    s.synchronize()
    _hold(out, None, _want(c))


def test_nothing_to_do(ops):
    cache = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    q = torch.zeros((0, 4, 64), dtype=torch.bfloat16, device=DEV)
    ops.tree_attention(q, (cache, cache.clone()), torch.zeros((2, 3), **i32), torch.zeros(2, **i32), torch.zeros(3, **i32),
                       torch.zeros((0, 1), dtype=torch.int64, device=DEV), 1.0, torch.zeros_like(q))
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device=DEV)
    out = q.clone()
    ops.tree_attention(q, (cache, cache.clone()), torch.zeros((0, 3), **i32), torch.zeros(0, **i32), torch.zeros(1, **i32),
                       torch.zeros((3, 1), dtype=torch.int64, device=DEV), 1.0, out)
    torch.cuda.synchronize()
    assert torch.equal(out, q)
    # A table without pages: nobody sees anything.
    ops.tree_attention(q, (cache, cache.clone()), torch.zeros((1, 0), **i32), torch.full((1,), 9, **i32),
                       torch.tensor([0, 3], **i32), torch.full((3, 1), -1, dtype=torch.int64, device=DEV), 1.0, out)
    torch.cuda.synchronize()
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,Hq", [(64, 1), (64, 2), (96, 2), (128, 1), (128, 2), (192, 1), (256, 1)])
@pytest.mark.parametrize("context", [0, 64])
@pytest.mark.parametrize("odd", [INF, -INF, NAN])
def test_odd_values_of_a_rows_first_keys(ops, dtype, dim, Hq, context, odd):
    """Tokens that see themselves alone (and the context), the values of some
    odd: nothing is summed up in their row, or the piece of it, before."""
    q = 100
    c = _case(40 + dim, [q], [context], 16, Hq, 1, dim, dtype, density=0.0)
    c["k"].nan_to_num_(0.5)
    c["v"].nan_to_num_(0.25)
    c["mask"] = [1 << i for i in range(q)]
    put = {0: 1, 5: dim - 1, 31: 3, 32: 0, 47: dim // 2, 63: 7, 64: 2, 95: dim - 2, 96: 33, 99: 4}
    for i, d in put.items():
        c["v"][int(c["table"][0, (context + i) // 16]), (context + i) % 16, 0, d] = odd
    caches, kw = _device_caches(c)
    out = c["out"].to(DEV)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, None)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    for i, d in put.items():
        c["v"][int(c["table"][0, (context + i) // 16]), (context + i) % 16, 0, d] = 0.0
    want, _, tol, _ = _want(c)
    hit = np.zeros_like(got, dtype=bool)
    for i, d in put.items():
        hit[i, :, d] = True
    assert (np.isnan(got[hit]) if odd != odd else got[hit] == odd).all(), np.argwhere(hit & np.isnan(got))
    assert (np.abs(got - want)[~hit] <= tol[~hit]).all()


def _spread_pages(c, pages, at):
    """The case's pages at page `at(p)` of caches of `pages` pages of NaN."""
    caches = []
    for x in (c["k"], c["v"]):
        big = torch.full((pages, *x.shape[1:]), NAN, dtype=x.dtype, device=DEV)
        big[torch.tensor([at(p) for p in range(x.shape[0])], device=DEV)] = x.to(DEV)
        caches.append(big)
    return tuple(caches)


@pytest.mark.parametrize("Hq,dim,block", [(4, 128, 16), (4, 64, 24)])
def test_caches_past_4_gib(ops, Hq, dim, block):
    """Pages on both sides of 2^31 and 2^32 bytes."""
    c = _case(31, [20, 7], [150, 40], block, Hq, 2, dim)
    page = block * 2 * dim * 2
    pages = (2**32 + 2**31) // page + 100
    caches = _spread_pages(c, pages, lambda p: pages - 1 - p * ((pages - 1) // c["k"].shape[0]))
    table = c["table"].clone()
    for r, n in enumerate(c["seq"].tolist()):
        for j in range(-(-n // block)):
            table[r, j] = pages - 1 - int(table[r, j]) * ((pages - 1) // c["k"].shape[0])
    out, lse = c["out"].to(DEV), c["lse"].to(DEV)
    ops.tree_attention(c["q"].to(DEV), caches, table.to(DEV), c["seq"].to(DEV), c["starts"].to(DEV),
                       od.words_of(c["mask"], c["words"]).to(DEV), c["scale"], out, lse)
    torch.cuda.synchronize()
    _hold(out, lse, _want(c))


@pytest.mark.parametrize("dim,q_lens", [(64, [20, 7]), (128, [70, 80])])
def test_rows_far_apart(ops, dim, q_lens):
    """Cache rows 2^27 - 16 bytes apart, the most that is taken (a group of 16
    spans 2 GiB); query, output, lse and masks of rows hundreds of MB apart."""
    c = _case(32, q_lens, [60, 35], 16, 2, 1, dim)
    pages, step = c["k"].shape[0], (2**27 - 16) // 2
    caches = []
    for x in (c["k"], c["v"]):
        space = torch.empty(15 * step + pages * dim, dtype=x.dtype, device=DEV)
        far = space.as_strided((pages, 16, 1, dim), (dim, step, dim, 1))
        far.copy_(x.to(DEV))
        caches.append(far)
    T = c["q"].shape[0]

    def apart(x, row):
        space = torch.empty((T - 1) * row + x[0].numel(), dtype=x.dtype, device=DEV)
        far = space.as_strided(x.shape, (row, *x.stride()[1:]))
        far.copy_(x.to(DEV))
        return far

    q, out, lse = apart(c["q"], 2**33 // T // 16 * 8), apart(c["out"], 2**33 // T // 16 * 8), apart(c["lse"], 2**32 // T)
    mask = apart(od.words_of(c["mask"], c["words"]), 2**32 // T // 2)
    ops.tree_attention(q, tuple(caches), c["table"].to(DEV), c["seq"].to(DEV), c["starts"].to(DEV), mask, c["scale"], out, lse)
    torch.cuda.synchronize()
    _hold(out, lse, _want(c))
