"""The serving operators at the ends of their sizes, eager and captured."""

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


@pytest.mark.parametrize("T", [1, 2047, 2048, 2049])
@pytest.mark.parametrize("n_freq", [4096, 2500])
def test_rotary_heads_of_8192_dims(ops, T, n_freq):
    """The longest angles' rows, one and two tokens' of them in a workgroup."""
    dim = 8192
    gen = torch.Generator().manual_seed(T)
    x = torch.randn((T, dim), generator=gen).to(torch.bfloat16)
    pos = torch.randint(0, 100000, (T,), generator=gen)
    inv = 10000.0 ** (-torch.arange(n_freq, dtype=torch.float64) / n_freq)
    got = x.to(DEV)
    ops.rotary_embedding(pos.to(DEV), got, None, dim, inv.to(DEV))
    torch.cuda.synchronize()
    want, size = osv.rotate(x.double().numpy(), pos.numpy(), inv.numpy(), dim, True)
    assert (np.abs(got.double().cpu().numpy() - want) <= osv.rotary_tolerance(want, size, x.dtype)).all()


@pytest.mark.parametrize("R", [6200, 16384])
def test_captured_slot_mapping_of_many_requests(ops, R):
    """Two sums of more than 48 KiB in a workgroup, replayed on the lengths of
    each replay's time."""
    rng = np.random.default_rng(R)
    block, width, n = 16, 6, 2 * R + 5
    q, c = (torch.zeros(R, dtype=torch.int32, device=DEV) for _ in range(2))
    table = torch.zeros((R, width), dtype=torch.int32, device=DEV)
    free = torch.from_numpy(rng.permutation(3 * R).astype(np.int32)).to(DEV)
    cursor, following = (torch.zeros(1, dtype=torch.int64, device=DEV) for _ in range(2))
    slots, pos = (torch.empty(n, dtype=torch.int64, device=DEV) for _ in range(2))
    starts, seq = torch.empty(R + 1, dtype=torch.int32, device=DEV), torch.empty(R, dtype=torch.int32, device=DEV)

    def call():
        ops.build_slot_mapping(q, c, table, block, slots, pos, starts, seq, free, cursor, following)

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for turn in range(3):
        query, context = rng.integers(0, 4, R), rng.integers(0, 60, R)
        pages = rng.permutation(R * width).reshape(R, width)
        q.copy_(torch.from_numpy(query.astype(np.int32)))
        c.copy_(torch.from_numpy(context.astype(np.int32)))
        table.copy_(torch.from_numpy(pages.astype(np.int32)))
        cursor.fill_(turn)
        g.replay()
        torch.cuda.synchronize()
        want = osv.slot_mapping(query, context, pages, block, n, free.tolist(), turn)
        for got, w in zip((slots, pos, starts, seq, table), want):
            assert np.array_equal(got.cpu().numpy(), w)
        assert following.item() == want[5]


@pytest.mark.parametrize("q", [1, 5, 8, 9, 300])
@pytest.mark.parametrize("grow", [False, True])
def test_positions_past_64_bits(ops, q, grow):
    """A request whose positions pass 2^63 - 1 stops there, without pages, and
    its neighbours are as they would be; a cursor next to 2^63 - 1 finds no
    block."""
    top = 2**63 - 1
    lens = torch.tensor([2, q, 3], dtype=torch.int64, device=DEV)
    for back in (0, 1, 4):
        context = torch.tensor([1, top - back, 4], dtype=torch.int64, device=DEV)
        table = torch.tensor([[7, 3], [1, 2], [5, 6]], dtype=torch.int32, device=DEV)
        slots, pos = (torch.full((q + 6,), -99, dtype=torch.int64, device=DEV) for _ in range(2))
        more = {}
        if grow:
            more = {"free_blocks": torch.tensor([11, 12], dtype=torch.int32, device=DEV),
                    "free_cursor": torch.tensor([top - 1], dtype=torch.int64, device=DEV)}
        ops.build_slot_mapping(lens, context, table, 4, slots, pos, **more)
        torch.cuda.synchronize()
        far = [min(top, top - back + i) for i in range(q)]
        assert pos.tolist() == [1, 2] + far + [4, 5, 6, 0]
        own = [-1, -1, -1] if grow else [6 * 4, 6 * 4 + 1, 6 * 4 + 2]      # block 1 of request 2 is new
        assert slots.tolist() == [7 * 4 + 1, 7 * 4 + 2] + [-1] * q + own + [-1]
        assert table[2, 1].item() == (-1 if grow else 6)


@pytest.mark.parametrize("T,H", [(1, 3), (70, 4), (3000, 2)])
def test_rotary_of_heads_dealt_in_turn(ops, T, H):
    """q, k and v of a head beside each other: q and k in place, and k and v
    to their pages with q in place."""
    dim, block = 64, 16
    gen = torch.Generator().manual_seed(T)
    x = torch.randn((T, H, 3, dim), generator=gen).to(torch.bfloat16)
    pos = torch.randint(0, 5000, (T,), generator=gen)
    inv = 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))

    def holds(got, part):
        src = x[:, :, part].reshape(T, H * dim)
        want, size = osv.rotate(src.double().numpy(), pos.numpy(), inv.numpy(), dim, True)
        err = np.abs(got.reshape(T, H * dim).double().cpu().numpy() - want)
        assert (err <= osv.rotary_tolerance(want, size, x.dtype)).all()

    d = x.to(DEV)
    ops.rotary_embedding(pos.to(DEV), d[:, :, 0], d[:, :, 1], dim, inv.to(DEV))
    torch.cuda.synchronize()
    holds(d[:, :, 0], 0)
    holds(d[:, :, 1], 1)
    assert torch.equal(d[:, :, 2].cpu(), x[:, :, 2])
    d = x.to(DEV)
    caches = torch.zeros((-(-T // block) + 1, block, H, 2, dim), dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(T, device=DEV)
    ops.rotary_embedding_to_paged(pos.to(DEV), d[:, :, 0], d[:, :, 1], d[:, :, 2], (caches[:, :, :, 0], caches[:, :, :, 1]),
                                  slots, dim, inv.to(DEV))
    torch.cuda.synchronize()
    holds(d[:, :, 0], 0)
    assert torch.equal(d[:, :, 1:].cpu(), x[:, :, 1:])
    rows = caches.view(-1, H, 2, dim)
    holds(rows[:T, :, 0], 1)
    assert torch.equal(rows[:T, :, 1].cpu(), x[:, :, 2])
    assert (rows[T:] == 0).all()
