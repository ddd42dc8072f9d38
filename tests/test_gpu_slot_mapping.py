"""build_slot_mapping against the definition, request by request: whole
numbers, so equal."""

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


def _run(ops, query, context, table, block, n, free=None, cursor=None, lens=torch.int32, table_pad=0):
    R = len(query)
    wide = torch.full((R, table.shape[1] + table_pad), -77, dtype=torch.int32, device=DEV)
    tb = wide[:, : table.shape[1]]
    tb.copy_(torch.from_numpy(table.astype(np.int32)))
    out = {
        "slots": torch.full((n,), -99, dtype=torch.int64, device=DEV),
        "positions": torch.full((n,), -99, dtype=torch.int64, device=DEV),
        "starts": torch.full((R + 1,), -99, dtype=torch.int32, device=DEV),
        "seq": torch.full((R,), -99, dtype=torch.int32, device=DEV),
    }
    extra = {}
    if free is not None:
        extra["free_blocks"] = torch.tensor(free, dtype=torch.int32, device=DEV)
        extra["next_cursor"] = torch.full((1,), -99, dtype=torch.int64, device=DEV)
        if cursor is not None:
            extra["free_cursor"] = torch.tensor([cursor], dtype=torch.int64, device=DEV)
    ops.build_slot_mapping(torch.tensor(query, dtype=lens, device=DEV), torch.tensor(context, dtype=lens, device=DEV), tb,
                           block, out["slots"], out["positions"], out["starts"], out["seq"], **extra)
    torch.cuda.synchronize()
    want = osv.slot_mapping(query, context, table, block, n, free, cursor or 0)
    got = [out[k].cpu().numpy() for k in ("slots", "positions", "starts", "seq")]
    for name, g, w in zip(("slots", "positions", "query_start_loc", "seq_lens"), got, want):
        assert np.array_equal(g, w), name
    assert np.array_equal(tb.cpu().numpy(), want[4])
    if table_pad:
        assert (wide[:, table.shape[1]:] == -77).all()
    if free is not None:
        assert extra["next_cursor"].item() == want[5]


def _batch(seed, R, q_max, c_max, block, grow, zero=0.1):
    rng = np.random.default_rng(seed)
    query = rng.integers(1, q_max + 1, R)
    query[rng.random(R) < zero] = 0
    context = rng.integers(0, c_max + 1, R)
    width = int(-(-(c_max + q_max) // block))
    order = rng.permutation(R * width + 100).astype(np.int64)
    table = order[: R * width].reshape(R, width).copy()
    have = -(-context // block)
    if grow:
        for r in range(R):
            table[r, have[r]:] = -1
    free = order[R * width:].tolist() + rng.permutation(5000).tolist()
    return query.tolist(), context.tolist(), table, free


@pytest.mark.parametrize("lens", [torch.int32, torch.int64])
@pytest.mark.parametrize("grow", [False, True])
@pytest.mark.parametrize("R,q_max,c_max,block", [
    (1, 1, 0, 16), (1, 1, 15, 16), (1, 1000, 100, 16), (3, 70, 50, 1), (64, 1, 4096, 16), (65, 1, 300, 128),
    (256, 3, 40, 48), (257, 5, 64, 64), (300, 200, 100, 7), (1025, 2, 33, 16), (2500, 1, 20, 16)])
def test_against_the_definition(ops, R, q_max, c_max, block, grow, lens):
    query, context, table, free = _batch(R + block, R, q_max, c_max, block, grow)
    total = sum(query)
    for n in {total, total + 37, max(0, total - 5)}:
        _run(ops, query, context, table, block, n, free if grow else None, 11 if grow else None, lens, table_pad=3)


def test_largest_batch(ops):
    """16384 requests, the most a call takes (two sums of 64 KiB in LDS)."""
    query, context, table, free = _batch(5, 16384, 2, 17, 16, True)
    _run(ops, query, context, table, 16, sum(query) + 1, free, 3)


def test_free_list_ends(ops):
    query, context, table, _ = _batch(9, 40, 60, 100, 16, True)
    _run(ops, query, context, table, 16, sum(query), [5, 3, 1000000, 2**31 - 1], 1)
    _run(ops, query, context, table, 16, sum(query), [], None)
    _run(ops, query, context, table, 16, sum(query), list(range(50)), -3)


def test_negative_lengths_and_rows_without_pages(ops):
    table = np.full((4, 3), -1, np.int64)
    table[1] = [4, -1, 2]
    # Past the table's row: no page; a negative length counts as none.
    _run(ops, [5, 60, -4, 3], [-2, 10, 7, 2**31 - 2], table, 16, 80)
    _run(ops, [5, 60, -4, 3], [-2, 10, 7, 2**40], table, 16, 80, lens=torch.int64)
    _run(ops, [5, 60, -4, 3], [-2, 10, 7, 2**40], table, 16, 80, list(range(10)), 0, torch.int64)


def test_lengths_whose_sum_passes_32_bits(ops):
    table = np.zeros((3, 2), np.int64)
    _run(ops, [3, 2**31 - 1, 2**31 - 1], [0, 0, 5], table, 8, 100)
    _run(ops, [3, 2**40, 7], [0, 2**62, 5], table, 8, 100, lens=torch.int64)


def test_short_and_long_requests_in_one_batch(ops):
    """Requests of 7, 8 and 9 new tokens, of none and of thousands, next to
    each other and behind the first 256."""
    for seed, R in ((1, 40), (2, 700)):
        rng = np.random.default_rng(seed)
        query = rng.choice([0, 1, 7, 8, 9, 10, 65, 2000 if R < 100 else 300], R).tolist()
        context = rng.integers(0, 200, R)
        width = (200 + 2001) // 16 + 1
        table = rng.permutation(R * width).reshape(R, width)
        _run(ops, query, context.tolist(), table, 16, sum(query) + 11)
        for r in range(R):
            table[r, -(-context[r] // 16):] = -1
        _run(ops, query, context.tolist(), table, 16, sum(query) + 11, rng.permutation(R * width).tolist(), 5)


def test_contexts_at_the_top_of_64_bits(ops):
    table = np.arange(6).reshape(2, 3)
    for q in (3, 40):
        _run(ops, [q, 2], [2**63 - 1 - q, 4], table, 8, q + 5, lens=torch.int64)


def test_slots_past_32_bits(ops):
    table = np.array([[2**31 - 1, 2**30]], np.int64)
    _run(ops, [20], [0], table, 16, 20)


def test_no_requests_and_no_tokens(ops):
    _run(ops, [], [], np.zeros((0, 4), np.int64), 16, 10)
    _run(ops, [4, 5], [0, 3], np.arange(8).reshape(2, 4), 16, 0, [9], 0)
    _run(ops, [4, 5], [0, 3], np.zeros((2, 0), np.int64), 16, 9)


def test_optional_outputs(ops):
    q = torch.tensor([3, 2], dtype=torch.int32, device=DEV)
    c = torch.tensor([0, 20], dtype=torch.int32, device=DEV)
    table = torch.tensor([[7, 8], [1, 2]], dtype=torch.int32, device=DEV)
    slots = torch.empty(5, dtype=torch.int64, device=DEV)
    ops.build_slot_mapping(q, c, table, 16, slots)
    assert slots.tolist() == [112, 113, 114, 36, 37]


def test_replays_read_the_lengths_of_their_time(ops):
    """A captured call on new lengths, eager work between the replays."""
    R, block, n = 40, 16, 500
    q = torch.zeros(R, dtype=torch.int32, device=DEV)
    c = torch.zeros(R, dtype=torch.int32, device=DEV)
    tb = torch.zeros((R, 12), dtype=torch.int32, device=DEV)
    free = torch.arange(1000, 2000, dtype=torch.int32, device=DEV)
    cur, nxt = (torch.zeros(1, dtype=torch.int64, device=DEV) for _ in range(2))
    slots, pos = (torch.empty(n, dtype=torch.int64, device=DEV) for _ in range(2))
    starts = torch.empty(R + 1, dtype=torch.int32, device=DEV)

    def call():
        ops.build_slot_mapping(q, c, tb, block, slots, pos, starts, None, free, cur, nxt)

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for seed in range(4):
        query, context, table, _ = _batch(seed, R, 12, 150, block, True)
        table = table[:, :12].copy() if table.shape[1] >= 12 else np.pad(table, ((0, 0), (0, 12 - table.shape[1])), constant_values=-1)
        q.copy_(torch.tensor(query))
        c.copy_(torch.tensor(context))
        tb.copy_(torch.from_numpy(table.astype(np.int32)))
        cur.fill_(seed * 7)
        g.replay()
        torch.cuda.synchronize()
        want = osv.slot_mapping(query, context, table, block, n, list(range(1000, 2000)), seed * 7)
        assert np.array_equal(slots.cpu().numpy(), want[0])
        assert np.array_equal(pos.cpu().numpy(), want[1])
        assert np.array_equal(tb.cpu().numpy(), want[4])
        assert nxt.item() == want[5]


def test_two_streams_at_once(ops):
    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = [_batch(s, 200, 50, 300, 16, False) for s in (1, 2)]
    outs = []
    torch.cuda.synchronize()
    for s, (query, context, table, _) in zip(streams, cases):
        with torch.cuda.stream(s):
            slots = torch.empty(sum(query), dtype=torch.int64, device=DEV)
            ops.build_slot_mapping(torch.tensor(query, device=DEV), torch.tensor(context, device=DEV),
                                   torch.from_numpy(table.astype(np.int32)).to(DEV), 16, slots)
            outs.append(slots)
    torch.cuda.synchronize()
    for slots, (query, context, table, _) in zip(outs, cases):
        assert np.array_equal(slots.cpu().numpy(), osv.slot_mapping(query, context, table, 16, sum(query))[0])
