"""shared_prefix_attention against softmax attention in 64 bits, one token and
head at a time (tolerances: oracle.serving.attention, derived there)."""

import numpy as np
import pytest
import torch

from oracle import serving as osv

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    import lmcache_amd

    return lmcache_amd.c_ops


def _case(seed, q_lens, seq_lens, P, block, Hq, Hk, dim, dtype=torch.bfloat16, fmt="separate", pad=0, extra_pages=3,
          spread=1.0):
    """Caches, tables and rows on the CPU.  Rows of the caches that no token
    sees hold NaN."""
    gen = torch.Generator().manual_seed(seed)
    R = len(q_lens)
    longest = max([P, 1] + list(seq_lens))
    width = -(-longest // block)
    n_shared = -(-P // block)
    pages = n_shared + R * width + extra_pages
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    shared = order[:n_shared].clone()
    table = order[n_shared: n_shared + R * width].reshape(R, width).clone()
    k, v = (torch.full((pages, block, Hk, dim), float("nan"), dtype=dtype) for _ in range(2))

    def fill(page, at):
        k[page, at] = (spread * torch.randn((Hk, dim), generator=gen)).to(dtype)
        v[page, at] = torch.randn((Hk, dim), generator=gen).to(dtype)

    for j in range(P):
        fill(int(shared[j // block]), j % block)
    for r, n in enumerate(seq_lens):
        for j in range(P, n):
            fill(int(table[r, j // block]), j % block)
    # Tables past a request's end hold anything.
    for r, n in enumerate(seq_lens):
        table[r, -(-max(0, n) // block):] = torch.randint(-5, 2 * pages, (width - -(-max(0, n) // block),), generator=gen,
                                                          dtype=torch.int32)
    starts = torch.zeros(R + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(q_lens, dtype=torch.int32).cumsum(0)
    T = int(starts[-1]) + pad
    q = torch.randn((T, Hq, dim), generator=gen).to(dtype)
    return {"q": q, "k": k, "v": v, "shared": shared, "P": P, "table": table, "seq": torch.tensor(seq_lens, dtype=torch.int32),
            "starts": starts, "scale": dim ** -0.5, "fmt": fmt, "out": torch.randn((T, Hq, dim), generator=gen).to(dtype),
            "lse": torch.randn((T, Hq), generator=gen), "dtype": dtype}


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
    ops.shared_prefix_attention(q, caches, c["shared"].to(DEV), c["P"], c["table"].to(DEV), c["seq"].to(DEV),
                                c["starts"].to(DEV), c["scale"], out, lse, **kw)


def _want(c):
    return osv.attention(c["q"], c["k"], c["v"], c["shared"], c["P"], c["table"].tolist(), c["seq"].tolist(),
                         c["starts"].tolist(), c["scale"], c["out"], c["lse"], c["dtype"])


def _hold(c, out, lse, want=None):
    o, low, tol_o, tol_l = want or _want(c)
    err = np.abs(out.double().cpu().numpy() - o)
    assert not np.isnan(err).any() and (err <= tol_o).all(), (np.nanmax(err - tol_o), np.isnan(err).sum())
    if lse is not None:
        got = lse.double().cpu().numpy()
        fine = np.isfinite(low)
        assert np.array_equal(got[~fine], low[~fine])
        assert (np.abs(got - low)[fine] <= tol_l[fine]).all(), np.nanmax(np.abs(got - low)[fine] - tol_l[fine])


def _check(ops, c, with_lse=True):
    caches, kw = _device_caches(c)
    out, lse = c["out"].to(DEV), c["lse"].to(DEV) if with_lse else None
    _call(ops, c, caches, kw, c["q"].to(DEV), out, lse)
    torch.cuda.synchronize()
    _hold(c, out, lse)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("P,block", [(0, 16), (1, 16), (31, 16), (64, 16), (65, 64), (300, 48), (517, 128)])
def test_lengths_and_dims(ops, dtype, dim, P, block):
    seq = [P + 1, P + 40, P + 17, P + 130]
    _check(ops, _case(dim + P, [1, 1, 1, 1], seq, P, block, 4, 2, dim, dtype))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (8, 8), (32, 8), (7, 1), (10, 2), (16, 1), (33, 1), (80, 2)])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [3, 0, 5, 1], [17, 2], [1]])
def test_heads_and_several_tokens(ops, dim, Hq, Hk, q_lens):
    P = 70
    seq = [P + n + 3 * i for i, n in enumerate(q_lens)]
    _check(ops, _case(Hq, q_lens, seq, P, 16, Hq, Hk, dim, pad=2))


@pytest.mark.parametrize("fmt", ["head_major", "merged", "two_major"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_cache_layouts(ops, fmt, dtype):
    _check(ops, _case(5, [1, 4, 2], [150, 97, 131], 90, 16, 8, 2, 128, dtype, fmt, pad=1))


@pytest.mark.parametrize("R", [40, 150])
def test_many_rows(ops, R):
    """Rows enough for full tiles, some requests shorter than the prefix (or
    not there), ragged own parts."""
    rng = np.random.default_rng(R)
    P = 260
    seq = [int(P + rng.integers(1, 90)) for _ in range(R)]
    seq[3], seq[7], seq[11] = 0, 12, P - 1
    _check(ops, _case(R, [1] * R, seq, P, 16, 8, 2, 64, pad=3))


def test_long_prefix_few_rows(ops):
    _check(ops, _case(1, [1, 2], [3000, 2950], 2900, 64, 4, 1, 128))


def test_long_own_part(ops):
    """No prefix: the own parts split over workgroups."""
    _check(ops, _case(2, [1, 1], [2500, 13], 0, 16, 4, 1, 64))
    _check(ops, _case(3, [2], [3001], 5, 16, 2, 2, 128))


def test_requests_that_end_inside_the_prefix(ops):
    """Several tokens whose positions lie in the shared blocks: each sees what
    is before it."""
    _check(ops, _case(4, [20, 5, 9], [50, 64, 9], 64, 16, 4, 2, 64))


def test_more_tokens_than_keys(ops):
    """The first of 6 tokens of a request with 2 keys see nothing."""
    out = _check(ops, _case(6, [6, 1], [2, 40], 1, 16, 4, 2, 64))
    assert (out[:4] == 0).all()


def test_blocks_outside_the_caches(ops):
    c = _case(7, [1, 3, 1], [200, 180, 150], 100, 16, 4, 2, 64)
    c["shared"][2] = -1
    c["shared"][5] = c["k"].shape[0]
    c["table"][0, 8] = -7
    c["table"][1, 11] = 2**31 - 1
    c["table"][2, 6:] = -1            # its whole own part
    _check(ops, c)
    c["shared"][:] = -1
    _check(ops, c)                     # request 2 sees nothing at all


def test_table_shorter_than_the_request(ops):
    c = _case(8, [1, 1], [200, 90], 60, 16, 4, 2, 64)
    c["table"] = c["table"][:, :9].contiguous()
    _check(ops, c)


@pytest.mark.parametrize("R", [1, 40])
def test_tables_much_wider_than_the_requests(ops, R):
    """Tables as wide as the longest context: most parts of the own keys are
    empty, and what lies in the tables behind a request is not read."""
    c = _case(17, [1] * R, [290 + 5 * r for r in range(R)], 270, 16, 8, 2, 64)
    wide = torch.full((R, 4000), 2**30, dtype=torch.int32)
    wide[:, : c["table"].shape[1]] = c["table"]
    c["table"] = wide
    _check(ops, c)


def test_lengths_far_past_the_table(ops):
    """A request said to be 2^31 - 1 long ends where its table's row ends."""
    c = _case(16, [1, 2, 1], [96, 80, 64], 40, 16, 4, 2, 64)
    c["seq"][0] = 2**31 - 1
    c["seq"][1] = -(2**31)
    caches, kw = _device_caches(c)
    out, lse = c["out"].to(DEV), c["lse"].to(DEV)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, lse)
    torch.cuda.synchronize()
    _hold(c, out, lse, _want(dict(c, seq=torch.tensor([96, 0, 64]))))


def test_unseen_infinities_among_several_tokens(ops):
    """A later token's key and value hold NaN and infinity: earlier tokens of
    the request do not see them, the later one does."""
    c = _case(9, [4, 4], [104, 90], 70, 16, 4, 2, 64)
    page, at = int(c["table"][0, 103 // 16]), 103 % 16
    c["v"][page, at] = float("nan")
    c["v"][page, at, :, 1::2] = float("inf")
    caches, kw = _device_caches(c)
    out, lse = c["out"].to(DEV), c["lse"].to(DEV)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, lse)
    torch.cuda.synchronize()
    assert torch.isinf(out[3, :, 1::2]).all() and torch.isnan(out[3, :, 0::2]).all()
    clean = dict(c, v=torch.nan_to_num(c["v"], nan=0.0, posinf=0.0, neginf=0.0), k=torch.nan_to_num(c["k"], nan=0.0))
    want = _want(clean)
    rows = [0, 1, 2, 4, 5, 6, 7]
    err = np.abs(out.double().cpu().numpy() - want[0])[rows]
    assert (err <= want[2][rows]).all()
    # The same with the key.
    c["v"][page, at] = 1.0
    c["k"][page, at] = float("nan")
    caches, kw = _device_caches(c)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, lse)
    torch.cuda.synchronize()
    assert torch.isnan(out[3]).all() and torch.isnan(lse[3]).all()
    err = np.abs(out.double().cpu().numpy() - want[0])[rows]
    assert (err <= want[2][rows]).all()


def test_unseen_infinity_inside_the_prefix(ops):
    """The same within the shared blocks: a request whose tokens end there."""
    c = _case(10, [5, 1], [40, 100], 64, 16, 2, 1, 128)
    page, at = int(c["shared"][38 // 16]), 38 % 16
    c["v"][page, at, :, ::3] = float("-inf")
    caches, kw = _device_caches(c)
    out = c["out"].to(DEV)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, None)
    torch.cuda.synchronize()
    clean = dict(c, v=torch.nan_to_num(c["v"], nan=0.0, neginf=0.0), k=torch.nan_to_num(c["k"], nan=0.0))
    want = _want(clean)
    got = out.double().cpu().numpy()
    # Keys 0 .. 35 + i: token 3 is the first that sees key 38.
    for t in (0, 1, 2):
        assert (np.abs(got[t] - want[0][t]) <= want[2][t]).all()
    for t in (3, 4, 5):
        assert np.isneginf(got[t][:, ::3]).all() and np.isfinite(got[t][:, 1::3]).all()


def test_large_scores(ops):
    """Scores of hundreds: one key takes all, and none overflows."""
    c = _case(11, [1, 2, 1], [300, 290, 280], 200, 16, 4, 2, 64, spread=60.0)
    _check(ops, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_strided_rows_and_no_lse(ops, dtype):
    """query a slice of a fused projection, output with a padded row."""
    c = _case(12, [1, 3, 2], [120, 99, 103], 80, 16, 6, 2, 96, dtype)
    caches, kw = _device_caches(c)
    T, H, D = c["q"].shape
    wide = torch.zeros((T, H * D + 64), dtype=dtype, device=DEV)
    wide[:, : H * D] = c["q"].reshape(T, H * D).to(DEV)
    q = wide[:, : H * D].view(T, H, D)
    buf = torch.full((T, H, D + 32), 7.0, dtype=dtype, device=DEV)
    _call(ops, c, caches, kw, q, buf[:, :, :D], None)
    torch.cuda.synchronize()
    _hold(c, buf[:, :, :D], None)
    assert (buf[:, :, D:] == 7.0).all()


def test_results_do_not_change_between_calls(ops):
    c = _case(13, [1] * 30, [900 + 7 * i for i in range(30)], 800, 16, 8, 2, 128)
    caches, kw = _device_caches(c)
    first = None
    for _ in range(4):
        out, lse = c["out"].to(DEV), c["lse"].to(DEV)
        _call(ops, c, caches, kw, c["q"].to(DEV), out, lse)
        torch.cuda.synchronize()
        if first is not None:
            assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
        first = (out, lse)


def test_replays_beside_eager_calls_on_another_stream(ops):
    """Two captured calls of different sizes, each replayed several times with
    eager calls between, on lengths and rows of the replay's time."""
    cases = [_case(s, [1] * n, [p + 5 + 3 * i for i in range(n)], p, 16, 8, 2, 64) for s, n, p in ((1, 12, 300), (2, 3, 64))]
    held = []
    for c in cases:
        caches, kw = _device_caches(c)
        s = {"q": c["q"].to(DEV), "out": c["out"].to(DEV), "lse": c["lse"].to(DEV), "shared": c["shared"].to(DEV),
             "table": c["table"].to(DEV), "seq": c["seq"].to(DEV), "starts": c["starts"].to(DEV)}

        def call(s=s, caches=caches, kw=kw, c=c):
            ops.shared_prefix_attention(s["q"], caches, s["shared"], c["P"], s["table"], s["seq"], s["starts"], c["scale"],
                                        s["out"], s["lse"], **kw)

        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        held.append((c, s, g, caches, kw))
    side = torch.cuda.Stream()
    for turn in range(3):
        for c, s, g, caches, kw in held:
            c = dict(c, q=torch.randn(c["q"].shape, generator=torch.Generator().manual_seed(turn)).to(c["dtype"]),
                     seq=(c["seq"] - turn).clamp(min=c["P"] + 1))
            s["q"].copy_(c["q"])
            s["seq"].copy_(c["seq"])
            torch.cuda.synchronize()
            g.replay()
            eager = c["out"].to(DEV)
            with torch.cuda.stream(side):
                _call(ops, c, caches, kw, c["q"].to(DEV), eager, None)
            torch.cuda.synchronize()
            assert torch.equal(eager, s["out"])
            _hold(c, s["out"], s["lse"])


def test_cache_rows_past_32_bits(ops):
    """Blocks more than 4 GiB into the caches."""
    block, H, D = 128, 8, 128
    pages = (5 << 30) // (block * H * D * 2)
    c = _case(14, [1, 1], [300, 290], 200, block, 8, 8, D, torch.bfloat16)
    small = c["k"].shape[0]
    caches = tuple(torch.zeros((pages, block, H, D), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for big, x in zip(caches, (c["k"], c["v"])):
        big[pages - small:] = x.to(DEV)
    out, lse = c["out"].to(DEV), c["lse"].to(DEV)
    moved = dict(c, shared=c["shared"] + (pages - small), table=c["table"] + (pages - small))
    _call(ops, moved, caches, {}, c["q"].to(DEV), out, lse)
    torch.cuda.synchronize()
    _hold(c, out, lse)


def test_no_tokens(ops):
    c = _case(15, [1], [10], 4, 16, 2, 1, 64)
    caches, kw = _device_caches(c)
    empty = torch.empty((0, 2, 64), dtype=c["dtype"], device=DEV)
    ops.shared_prefix_attention(empty, caches, c["shared"].to(DEV), 4, torch.empty((0, 1), dtype=torch.int32, device=DEV),
                                torch.empty(0, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV),
                                1.0, empty.clone())
    out = c["out"].to(DEV)
    ops.shared_prefix_attention(c["q"].to(DEV), caches, c["shared"].to(DEV), 4, torch.empty((0, 1), dtype=torch.int32, device=DEV),
                                torch.empty(0, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV),
                                1.0, out)
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), c["out"])


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_unseen_infinity_in_a_prefix_of_many_rows(ops, dim):
    """Tiles of 128 rows: one request ends before a key whose value holds
    infinities, the others see it."""
    P, R, short, key = 300, 80, 5, 150
    seq = [P + 1 + r % 7 for r in range(R)]
    seq[short] = 100
    c = _case(dim, [1] * R, seq, P, 16, 4, 2, dim)
    page, at = int(c["shared"][key // 16]), key % 16
    c["v"][page, at, :, ::3] = float("inf")
    caches, kw = _device_caches(c)
    out = c["out"].to(DEV)
    _call(ops, c, caches, kw, c["q"].to(DEV), out, None)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    others = [r for r in range(R) if r != short]
    assert np.isposinf(got[others][:, :, ::3]).all() and np.isfinite(got[others][:, :, 1::3]).all()
    c["v"] = torch.nan_to_num(c["v"], nan=0.0, posinf=0.0)
    c["k"] = torch.nan_to_num(c["k"], nan=0.0)
    want = _want(c)
    assert (np.abs(got[short] - want[0][short]) <= want[2][short]).all()
    assert (np.abs(got - want[0]) <= want[2])[:, :, 1::3].all()


@pytest.mark.parametrize("P", [0, 100])
def test_prompts_in_chunks(ops, P):
    """Hundreds of tokens a request: several tiles of 32 rows each over the
    request's own keys."""
    q_lens = [130, 0, 257, 1]
    _check(ops, _case(21 + P, q_lens, [P + n + 9 for n in q_lens], P, 16, 6, 2, 64, pad=3))


@pytest.mark.parametrize("R", [3, 50])
def test_output_over_the_query(ops, R):
    c = _case(22, [1] * R, [90 + i for i in range(R)], 70, 16, 8, 2, 64)
    caches, kw = _device_caches(c)
    q, lse = c["q"].to(DEV), c["lse"].to(DEV)
    _call(ops, c, caches, kw, q, q, lse)
    torch.cuda.synchronize()
    _hold(c, q, lse)


def test_output_and_lse_as_columns_of_one_buffer(ops):
    c = _case(23, [1, 2, 1], [90, 85, 77], 70, 16, 8, 2, 64)
    caches, kw = _device_caches(c)
    T, H, D = c["q"].shape
    rows = torch.zeros((T, H * (D * 2 + 4) + 16), dtype=torch.uint8, device=DEV)
    out = rows.view(torch.bfloat16)[:, : H * D].view(T, H, D)
    lse = rows.view(torch.float32)[:, H * D // 2: H * D // 2 + H]
    _call(ops, c, caches, kw, c["q"].to(DEV), out, lse)
    torch.cuda.synchronize()
    _hold(c, out, lse)
    assert (rows[:, H * (D * 2 + 4):] == 0).all()


def test_two_streams_at_once(ops):
    """Each call works in scratch of its own."""
    cases = [_case(s, [1] * 40, [420 + 3 * i for i in range(40)], 400, 16, 8, 2, 64) for s in (24, 25)]
    held = [(c, _device_caches(c), c["q"].to(DEV), c["out"].to(DEV), c["lse"].to(DEV), torch.cuda.Stream()) for c in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, (caches, kw), q, out, lse, stream in held:
            with torch.cuda.stream(stream):
                _call(ops, c, caches, kw, q, out, lse)
    torch.cuda.synchronize()
    for c, _, _, out, lse, _ in held:
        _hold(c, out, lse)


def test_one_block_several_times(ops):
    """Requests that own one block together, and one that has it twice."""
    c = _case(26, [1, 1, 2], [112, 112, 112], 64, 16, 4, 2, 128)
    c["table"][1] = c["table"][0]
    c["table"][2, 5] = c["table"][2, 4]
    _check(ops, c)


def test_one_request_with_one_key(ops):
    """Its value, whatever the query, and an lse of the score."""
    for P in (0, 1):
        c = _case(27, [1], [1], P, 16, 2, 1, 64)
        out = _check(ops, c)
        page = int(c["shared"][0]) if P else int(c["table"][0, 0])
        assert torch.equal(out[0].cpu(), c["v"][page, 0].expand(2, 64))
