"""copy_kv_pages, compact_kv and release_pages against their definitions, page
by page and row by row: the same bytes, everywhere else as before."""

import pytest
import torch

from oracle import drafting as od

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    import lmcache_amd

    return lmcache_amd.c_ops


class Caches:
    """All layers on the GPU in one of the layouts, and the planes ([layers,
    pages, block, ...]) of each on the CPU."""

    def __init__(self, ops, fmt, layers, pages, block, heads, dim, dtype=torch.bfloat16, seed=0):
        gen = torch.Generator().manual_seed(seed)

        def make(*shape):
            if dtype.itemsize == 1:
                return torch.randint(0, 255, shape, generator=gen, dtype=torch.uint8).view(dtype)
            return torch.randn(shape, generator=gen).to(dtype)

        def on_gpu(x):
            return x.view(torch.uint8).to(DEV).view(dtype) if dtype.itemsize == 1 else x.to(DEV)

        L, kw = layers, {}
        if fmt in ("separate", "head_major", "padded"):
            planes = [make(L, pages, block, heads, dim) for _ in range(2)]
            if fmt == "head_major":
                gpu = [on_gpu(x.transpose(2, 3).contiguous()).transpose(2, 3) for x in planes]
            elif fmt == "padded":
                gpu = []
                for x in planes:
                    wide = torch.zeros((L, pages, block + 1, heads + 1, dim + 8), dtype=dtype, device=DEV)
                    wide[:, :, :block, :heads, :dim] = x.to(DEV)
                    gpu.append(wide[:, :, :block, :heads, :dim])
            else:
                gpu = [on_gpu(x) for x in planes]
            self.layers = [(gpu[0][i], gpu[1][i]) for i in range(L)]
            self.gpu = gpu
        elif fmt in ("merged", "two_major"):
            planes = [make(L, pages, block, heads, dim) for _ in range(2)]
            at = 2 if fmt == "merged" else 1
            both = on_gpu(torch.stack(planes, dim=at))
            self.layers = [both[i] for i in range(L)]
            self.gpu = [both.select(at, p) for p in range(2)]
            kw = {"kvcache_format_raw": 1, "vllm_two_major": fmt == "two_major"}
        elif fmt == "index":
            planes = [make(L, pages, block, dim)]
            gpu = [on_gpu(x) for x in planes]
            self.layers, self.gpu, kw = [gpu[0][i] for i in range(L)], gpu, {"kvcache_format_raw": 6}
        else:
            widths = [dim, dim // 2, dim // 4][: 3 if fmt == "dsa" else 2]
            planes = [make(L, pages, block, 1, w) for w in widths]
            gpu = [on_gpu(x) for x in planes]
            self.layers = [tuple(x[i] for x in gpu) for i in range(L)]
            self.gpu, kw = gpu, {"kvcache_format_raw": {"mla": 3, "dsa": 4}[fmt]}
        self.planes = planes
        self.state = ops.prepare_kv_pages(self.layers, **kw)

    def hold(self, want):
        torch.cuda.synchronize()
        for x, y in zip(self.gpu, want):
            a, b = x.cpu().contiguous(), y.contiguous()
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


FORMATS = ["separate", "head_major", "padded", "merged", "two_major", "mla", "dsa", "index"]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("block,heads,dim", [(16, 2, 64), (1, 1, 8), (7, 3, 40), (128, 8, 128)])
@pytest.mark.parametrize("wide", [True, False])
def test_copies(ops, fmt, block, heads, dim, wide):
    c = Caches(ops, fmt, 3, 12, block, heads, dim)
    pairs = [(3, 7), (3, 0), (11, 11), (-1, 4), (5, -1), (12, 2), (1, 12), (2**31 - 1, 6), (9, 10), (4, -(2**31))]
    c_pairs = torch.tensor(pairs, dtype=torch.int64 if wide else torch.int32, device=DEV)
    ops.copy_kv_pages(c.state, c_pairs)
    c.hold(od.copy_pages(c.planes, pairs))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.uint8, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("heads,dim", [(1, 5), (3, 6), (2, 12), (4, 64)])
def test_dtypes_and_odd_widths(ops, dtype, heads, dim):
    c = Caches(ops, "separate", 2, 9, 16, heads, dim, dtype)
    pairs = [(0, 8), (2, 1), (2, 3)]
    ops.copy_kv_pages(c.state, torch.tensor(pairs, device=DEV))
    want = od.copy_pages([x.view(torch.uint8) for x in c.planes], pairs)
    table, base, keep, lens = [[4, 5, 6, 7]], [3], [[0, 2, 3, 9, 20, 40, 41]], [7]
    ops.compact_kv(c.state, *(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (table, base, keep, lens)))
    c.hold(od.compact(want, table, base, keep, lens))


def test_pairs_with_a_stride_and_none(ops):
    c = Caches(ops, "separate", 1, 20, 16, 2, 64)
    wide = torch.zeros((3, 5), dtype=torch.int64, device=DEV)
    wide[:, 1:3] = torch.tensor([[1, 2], [3, 4], [5, 6]])
    ops.copy_kv_pages(c.state, wide[:, 1:3])
    c.hold(od.copy_pages(c.planes, [(1, 2), (3, 4), (5, 6)]))
    ops.copy_kv_pages(c.state, wide[:0, 1:3])


def test_states_that_are_refused(ops):
    k, v = (torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    with pytest.raises(ValueError, match="no layers"):
        ops.prepare_kv_pages([])
    with pytest.raises(ValueError, match="given twice"):
        ops.prepare_kv_pages([(k, v), (k, v)])
    with pytest.raises(ValueError, match="number of their caches"):
        ops.prepare_kv_pages([(k, v), (k.clone(),)])
    with pytest.raises(ValueError, match="shape, dtype"):
        ops.prepare_kv_pages([(k, v), (k.half(), v.half())])
    with pytest.raises(ValueError, match="shape, dtype"):
        ops.prepare_kv_pages([(k, v), (k.transpose(1, 2).contiguous().transpose(1, 2), v.clone())])
    with pytest.raises(ValueError, match="overlap"):
        ops.prepare_kv_pages([(k[:3], k[1:])])
    wide = torch.zeros((4, 16, 2, 64 + 4), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="alignment"):
        ops.prepare_kv_pages([(wide[..., :64], wide.clone()[..., :64]), (wide.clone()[..., 4:], wide.clone()[..., :64])])
    with pytest.raises(ValueError, match="GPU"):
        ops.prepare_kv_pages([(k.cpu(), v.cpu())])
    with pytest.raises(RuntimeError, match="neither a Tensor"):
        ops.prepare_kv_pages([[k, v]])


def test_many_pairs(ops):
    c = Caches(ops, "two_major", 5, 900, 16, 2, 32)
    order = torch.randperm(900, generator=torch.Generator().manual_seed(1))
    pairs = torch.stack((order[torch.arange(600) % 300], order[300:]), dim=1)
    ops.copy_kv_pages(c.state, pairs.to(DEV))
    c.hold(od.copy_pages(c.planes, pairs.tolist()))


def _lists(gen, R, held, most, pages, block, width):
    """Lists that keep from none to all of the rows, of any density."""
    table = torch.randperm(pages, generator=gen)[: R * width].view(R, width)
    keep = torch.full((R, most), 2**31 - 1, dtype=torch.int64)
    lens = []
    for r in range(R):
        n = [0, most, 1, most // 2, most - 1][r % 5]
        n = min(n, held)
        lens.append(n)
        keep[r, :n] = torch.randperm(held, generator=gen)[:n].sort().values
    base = torch.randint(0, width * block - held + 1, (R,), generator=gen)
    return table, base, keep, torch.tensor(lens)


def _compact(ops, c, table, base, keep, lens, planes=None):
    i32 = [x.to(torch.int32).to(DEV) for x in (table, base, keep, lens)]
    seq = torch.full((len(lens),), -7, dtype=torch.int32, device=DEV)
    ops.compact_kv(c.state, *i32, seq)
    want = od.compact(planes or c.planes, table.tolist(), base.tolist(), keep.tolist(), lens.tolist())
    c.hold(want)
    assert seq.tolist() == [int(b) + min(max(0, int(n)), keep.shape[1]) for b, n in zip(base, lens)]
    return want


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("held,most", [(16, 6), (40, 40), (300, 150)])
def test_rows_move_together(ops, fmt, held, most):
    gen = torch.Generator().manual_seed(held)
    c = Caches(ops, fmt, 2, 130, 16, 3, 40, seed=held)
    _compact(ops, c, *_lists(gen, 6, held, most, 130, 16, 20))


@pytest.mark.parametrize("layers,heads,dim,block", [(1, 1, 8, 16), (1, 8, 128, 128), (40, 8, 128, 16), (3, 1, 576, 64)])
@pytest.mark.parametrize("R", [1, 33])
def test_sizes_of_rows_and_batches(ops, layers, heads, dim, block, R):
    gen = torch.Generator().manual_seed(R)
    width = -(-64 // block) + 1
    c = Caches(ops, "separate", layers, R * width + 1, block, heads, dim)
    _compact(ops, c, *_lists(gen, R, 33, 20, R * width, block, width))


@pytest.mark.parametrize("R", [1, 3])
def test_long_lists(ops, R):
    """Thousands of rows in place, what is read ahead of what is written."""
    gen = torch.Generator().manual_seed(R)
    c = Caches(ops, "separate", 2, R * 300, 16, 2, 64)
    table, base, keep, lens = _lists(gen, R, 4500, 3000, R * 300, 16, 300)
    lens[0] = 3000
    keep[0] = torch.randperm(4500, generator=gen)[:3000].sort().values
    _compact(ops, c, table, base, keep, lens)


def test_one_row_dropped_moves_all_behind_it(ops):
    c = Caches(ops, "head_major", 1, 140, 16, 4, 64)
    keep = torch.tensor([[i for i in range(2200) if i != 0], [i for i in range(2200) if i != 1100]])
    table = torch.randperm(140, generator=torch.Generator().manual_seed(1))[: 2 * 70].view(2, 70)
    # (70 pages hold 1120 rows: the rest has no page)
    _compact(ops, c, table, torch.tensor([0, 0]), keep, torch.tensor([2199, 2199]))


def test_rows_without_a_page_stay(ops):
    gen = torch.Generator().manual_seed(5)
    c = Caches(ops, "separate", 2, 60, 16, 2, 64)
    table, base, keep, lens = _lists(gen, 5, 60, 40, 60, 16, 8)
    table[1, 2], table[2, 0], table[3, 1], table[4, 3] = -1, 60, 2**31 - 1, -(2**31)
    base[1], base[2], base[3] = 120, -5, 0
    lens[1], lens[2], lens[3], lens[4] = 40, 41, -3, 1000
    for r in (1, 2, 4):
        keep[r] = torch.randperm(60, generator=gen)[:40].sort().values
    _compact(ops, c, table, base, keep, lens)


def test_lists_that_do_not_increase_stay_in_their_rows(ops):
    """Which rows such a list leaves is not said; the others are as before."""
    c = Caches(ops, "separate", 1, 20, 16, 2, 64)
    table = torch.tensor([[3, 4, 5], [9, 8, 7]])
    keep = torch.tensor([[5, 3, 3, 0, 40, -9, 2**31 - 1, -(2**31)], [0, 0, 0, 0, 0, 0, 0, 0]])
    ops.compact_kv(c.state, *(x.to(torch.int32).to(DEV) for x in (table, torch.tensor([16, 2]), keep, torch.tensor([8, 8]))))
    torch.cuda.synchronize()
    for x, y in zip(c.gpu, c.planes):
        x, y = x.cpu().clone(), y.clone()
        x[:, 4, :8] = y[:, 4, :8] = 0
        x[:, 9, 2:10] = y[:, 9, 2:10] = 0
        assert torch.equal(x, y)


def test_captured_copies_and_moves(ops):
    c = Caches(ops, "separate", 3, 80, 16, 2, 64)
    gen = torch.Generator().manual_seed(2)
    pairs = torch.zeros((4, 2), dtype=torch.int64, device=DEV)
    args = [torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((3, 8), (3,), (3, 30), (3,), (3,))]

    def call():
        ops.copy_kv_pages(c.state, pairs)
        ops.compact_kv(c.state, *args)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    planes = c.planes
    for n in range(4):
        table, base, keep, lens = _lists(gen, 3, 50, 30, 60, 16, 8)
        lens = torch.tensor([30, n, 17])
        for r in range(3):
            keep[r] = torch.randperm(50, generator=gen)[:30].sort().values
        some = torch.randperm(20, generator=gen)[:8].view(4, 2) + 60
        pairs.copy_(some)
        for a, x in zip(args, (table, base, keep, lens)):
            a.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        planes = od.compact(od.copy_pages(planes, some.tolist()), table.tolist(), base.tolist(), keep.tolist(), lens.tolist())
        c.hold(planes)


def test_places_past_2_gib(ops):
    """Rows and pages that lie more than 2^32 bytes into a layer."""
    pages = 2200
    k, v = (torch.zeros((pages, 128, 8, 1024), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    state = ops.prepare_kv_pages([(k, v)])
    for x in (k, v):
        x[5].normal_()
        x[2190].normal_()
    a, b = k[5].clone(), v[2190].clone()
    ops.copy_kv_pages(state, torch.tensor([[5, 2199], [2190, 0]], device=DEV))
    assert torch.equal(k[2199], a) and torch.equal(v[0], b)
    i32 = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([[2198, 2199]], [100], [[30, 40, 150]], [3])]
    ops.compact_kv(state, *i32)
    torch.cuda.synchronize()
    assert torch.equal(k[2198, 100], a[2]) and torch.equal(k[2198, 101], a[12]) and torch.equal(k[2198, 102], a[122])


def _release(ops, table, held, keep, block, refs, free, cursor, strided=False):
    R, W = len(table), len(table[0]) if table else 0
    i32 = dict(dtype=torch.int32, device=DEV)
    t = torch.tensor(table, **i32).view(R, W)
    if strided:
        t = torch.cat((t, torch.full((R, 3), 1, **i32)), dim=1)[:, :W]
    refs_d, free_d = torch.tensor(refs, **i32), torch.tensor(free, **i32)
    cur, nxt = (torch.tensor([x], dtype=torch.int64, device=DEV) for x in (cursor, -99))
    ops.release_pages(t, torch.tensor(held, **i32), torch.tensor(keep, **i32), block, refs_d, free_d, cur, nxt)
    torch.cuda.synchronize()
    want = od.release(table, held, keep, block, refs, free, cursor)
    assert refs_d.tolist() == want[0]
    assert nxt.item() == want[2] and cur.item() == cursor
    assert free_d.tolist() == want[1]
    assert t.tolist() == table


@pytest.mark.parametrize("block", [1, 16, 100])
@pytest.mark.parametrize("pages", [40, 4096, 4097, 30000])
def test_pages_are_given_back(ops, block, pages):
    gen = torch.Generator().manual_seed(pages + block)
    R, W = 9, 4
    table = torch.randperm(pages, generator=gen)[: R * W].view(R, W).tolist()
    held = torch.randint(0, W * block + 1, (R,), generator=gen).tolist()
    keep = [int(h * x) for h, x in zip(held, torch.rand(R, generator=gen).tolist())]
    free = torch.randperm(pages, generator=gen).tolist()
    _release(ops, table, held, keep, block, [0] * pages, free, R * W, strided=True)


def test_shared_pages_stay_until_their_last_holder(ops):
    refs = [0] * 50
    refs[3], refs[4], refs[5] = 1, 2, 1
    # 3: both holders; 4: two of three; 5: one of two; 6: twice without a count.
    table = [[3, 4, 5, 6], [3, 4, 6, 9], [20, 21, 22, 23]]
    _release(ops, table, [64, 64, 40], [0, 0, 17], 16, refs, list(range(100, 150)), 20)


def test_lengths_and_entries_that_say_nothing(ops):
    table = [[1, -1, 50, 2], [2**31 - 1, -(2**31), 7, 8], [9, 10, 11, 12], [13, 14, 15, 16]]
    _release(ops, table, [64, 2**31 - 1, -5, 30], [0, -(2**31), -9, 40], 16, [0] * 50, [0] * 50, 12)


def test_a_list_without_room(ops):
    table = [[1, 2, 3, 4]]
    _release(ops, table, [64], [0], 16, [0] * 9, [99] * 9, 2)       # two of the four fit
    _release(ops, table, [64], [0], 16, [0] * 9, [99] * 2, 4)       # the list ends before
    _release(ops, table, [64], [0], 16, [0] * 9, [], 4)
    _release(ops, table, [64], [0], 16, [0] * 9, [99] * 9, -3)
    _release(ops, table, [64], [0], 16, [0] * 9, [99] * 9, 2**40)


def test_counts_below_zero_are_given_back(ops):
    _release(ops, [[1, 2]], [32], [16], 16, [0, 0, -4, -1, 5], [9] * 9, 6)


def test_no_requests_and_no_pages(ops):
    _release(ops, [], [], [], 16, [0] * 10, [9] * 9, 4)
    _release(ops, [[1, 2]], [32], [0], 16, [], [9] * 9, 4)


def test_many_pages(ops):
    gen = torch.Generator().manual_seed(8)
    P, R, W = 70000, 100, 500
    table = torch.randperm(P, generator=gen)[: R * W].view(R, W)
    table[1::2, :200] = table[0::2, :200]
    refs = torch.zeros(P, dtype=torch.int64)
    refs[table[1::2, :150].reshape(-1)] = 1
    held = torch.randint(0, W * 16 + 1, (R,), generator=gen)
    keep = (held * torch.rand(R, generator=gen)).long()
    _release(ops, table.tolist(), held.tolist(), keep.tolist(), 16, refs.tolist(), list(range(P)), 60000)


def test_release_in_a_graph_gives_back_at_each_replay(ops):
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.arange(40, **i32).view(4, 10)
    held, keep = torch.zeros(4, **i32), torch.zeros(4, **i32)
    refs, free = torch.zeros(9000, **i32), torch.zeros(100, **i32)
    cur, nxt = torch.full((1,), 60, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)

    def call():
        ops.release_pages(table, held, keep, 16, refs, free, cur, nxt)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for n in range(4):
        h, k = [160, 100 + n, 16 * n, 0], [16 * n, 20, 0, 0]
        held.copy_(torch.tensor(h, dtype=torch.int32))
        keep.copy_(torch.tensor(k, dtype=torch.int32))
        refs.zero_()
        refs[5] = 1
        before = free.tolist()
        start = refs.tolist()
        graph.replay()
        torch.cuda.synchronize()
        want = od.release(table.tolist(), h, k, 16, start, before, 60)
        assert (refs.tolist(), free.tolist(), nxt.item()) == want


def test_given_back_pages_are_taken_again(ops):
    """release_pages and build_slot_mapping on one list."""
    i32, i64 = dict(dtype=torch.int32, device=DEV), dict(dtype=torch.int64, device=DEV)
    free = torch.randperm(64, generator=torch.Generator().manual_seed(3)).to(torch.int32).to(DEV)
    table = torch.full((2, 20), -1, **i32)
    cur, nxt = torch.zeros(1, **i64), torch.zeros(1, **i64)
    refs, seq = torch.zeros(64, **i32), torch.zeros(2, **i32)
    context = torch.zeros(2, **i32)
    for step, (q, keep) in enumerate([([100, 40], [90, 0]), ([30, 70], [0, 65]), ([17, 1], [17, 66])]):
        slots = torch.empty(sum(q), **i64)
        ops.build_slot_mapping(torch.tensor(q, **i32), context, table, 16, slots, seq_lens=seq, free_blocks=free,
                               free_cursor=cur, next_cursor=nxt)
        assert (slots >= 0).all() and slots.unique().numel() == slots.numel()
        cur.copy_(nxt)
        context = torch.tensor(keep, **i32)
        ops.release_pages(table, seq, context, 16, refs, free, cur, nxt)
        cur.copy_(nxt)
        torch.cuda.synchronize()
        used = sum(-(-k // 16) for k in keep)
        assert cur.item() == used
        assert sorted(free[used:].tolist() + [int(x) for r in range(2) for x in table[r, : -(-keep[r] // 16)]]) == list(range(64))


@pytest.mark.parametrize("cursor", [9, 10, 13, 2**31, 2**63 - 1])
@pytest.mark.parametrize("pages", [9, 5000])
def test_places_past_the_list_were_never_handed_out(ops, cursor, pages):
    """A cursor past the list's end, as build_slot_mapping leaves it when pages
    run short: the pages go below the list's end, none is lost."""
    table = [[1, 2, 3, 4], [8, -1, -1, -1]]
    _release(ops, table, [64, 64], [16, 0], 16, [0] * pages, [99] * 9, cursor)
    i32, i64 = dict(dtype=torch.int32, device=DEV), dict(dtype=torch.int64, device=DEV)
    free, nxt = torch.full((9,), 99, **i32), torch.zeros(1, **i64)
    ops.release_pages(torch.tensor(table, **i32), torch.tensor([64, 64], **i32), torch.tensor([16, 0], **i32), 16,
                      torch.zeros(pages, **i32), free, torch.tensor([cursor], **i64), nxt)
    torch.cuda.synchronize()
    assert nxt.item() == 5 and free.tolist() == [99] * 5 + [2, 3, 4, 8]


@pytest.mark.parametrize("pages,lens", [(4, [96, 0]), (4, [40, 70]), (7, [160, 160]), (1, [16, 17])])
def test_no_page_is_lost_when_the_list_runs_short(ops, pages, lens):
    """More pages asked for than there are, time and again: what is given back
    is the whole list each time, every page in it once."""
    i32, i64 = dict(dtype=torch.int32, device=DEV), dict(dtype=torch.int64, device=DEV)
    free = torch.arange(pages, **i32).flip(0).contiguous()
    cur, nxt, refs = torch.zeros(1, **i64), torch.zeros(1, **i64), torch.zeros(pages, **i32)
    none, seq = torch.zeros(2, **i32), torch.zeros(2, **i32)
    asked = sum(-(-n // 16) for n in lens)
    assert asked > pages
    for _ in range(3):
        table, slots = torch.full((2, 12), -1, **i32), torch.empty(sum(lens), **i64)
        ops.build_slot_mapping(torch.tensor(lens, **i32), none, table, 16, slots, seq_lens=seq, free_blocks=free,
                               free_cursor=cur, next_cursor=nxt)
        assert nxt.item() == asked and (table >= 0).sum() == pages
        cur.copy_(nxt)
        # Half of the first request's tokens first, then the rest.
        half = torch.tensor([lens[0] // 2, lens[1]], **i32)
        ops.release_pages(table, seq, half, 16, refs, free, cur, nxt)
        cur.copy_(nxt)
        ops.release_pages(table, half, none, 16, refs, free, cur, nxt)
        cur.copy_(nxt)
        torch.cuda.synchronize()
        assert cur.item() == 0 and sorted(free.tolist()) == list(range(pages)) and refs.sum() == 0


def test_caches_without_pages(ops):
    """Caches that hold nothing have no address: they are not one cache."""
    none = torch.zeros((0, 16, 2, 64), dtype=torch.bfloat16, device=DEV)
    state = ops.prepare_kv_pages([(none, none.clone()), (none.clone(), none.clone())])
    ops.copy_kv_pages(state, torch.tensor([[0, 1]], device=DEV))
    i32 = dict(dtype=torch.int32, device=DEV)
    seq = torch.zeros(2, **i32)
    ops.compact_kv(state, torch.zeros((2, 3), **i32), torch.tensor([3, 4], **i32), torch.tensor([[1, 2], [0, 5]], **i32),
                   torch.tensor([2, 1], **i32), seq)
    torch.cuda.synchronize()
    assert seq.tolist() == [5, 5]


def test_layers_over_each_other_are_refused(ops):
    both = torch.zeros((2, 9, 16, 2, 64), dtype=torch.bfloat16, device=DEV)
    k, v = both[0], both[1]
    with pytest.raises(ValueError, match="two of the layers' caches overlap"):
        ops.prepare_kv_pages([(k[:4], v[:4]), (k[2:6], v[4:8])])
    with pytest.raises(ValueError, match="two of the layers' caches overlap"):
        ops.prepare_kv_pages([both[:, :5], both[:, 4:]], 1, True)
    with pytest.raises(ValueError, match="two of the layers' caches overlap"):
        ops.prepare_kv_pages([(k[:4].view(torch.float8_e4m3fn), v[:4].view(torch.float8_e4m3fn)),
                              (k[3:7].view(torch.float8_e4m3fn), v[4:8].view(torch.float8_e4m3fn))])


def test_layers_in_turn_in_one_buffer(ops):
    """Pages that hold every layer's K and V beside each other."""
    gen = torch.Generator().manual_seed(8)
    x = torch.randn((12, 3, 2, 16, 2, 64), generator=gen).to(torch.bfloat16)
    gpu = x.to(DEV)
    state = ops.prepare_kv_pages([(gpu[:, i, 0], gpu[:, i, 1]) for i in range(3)])
    pairs = [(3, 7), (0, 11)]
    ops.copy_kv_pages(state, torch.tensor(pairs, device=DEV))
    i32 = [torch.tensor(a, dtype=torch.int32, device=DEV) for a in ([[4, 5, 6]], [3], [[0, 2, 20]], [3])]
    ops.compact_kv(state, *i32)
    torch.cuda.synchronize()
    planes = [x[:, :, p].transpose(0, 1) for p in range(2)]
    want = od.compact(od.copy_pages(planes, pairs), [[4, 5, 6]], [3], [[0, 2, 20]], [3])
    assert torch.equal(gpu.cpu(), torch.stack([w.transpose(0, 1) for w in want], dim=2))


@pytest.mark.parametrize("direct", [False, True])
def test_lists_in_the_caches_of_any_layer_are_refused(ops, monkeypatch, direct):
    if direct:
        monkeypatch.setattr(ops, "_ext", None)
    space = torch.zeros(4 * 4096 * 2 + 64, dtype=torch.int32, device=DEV)
    whole = space[: 4 * 4096].view(torch.bfloat16).view(4, 4, 16, 2, 64)
    k, v = whole[:2], whole[2:]
    state = ops.prepare_kv_pages([(k[i], v[i]) for i in range(2)])
    assert state.ranges.shape == (1, 2)
    i32 = dict(dtype=torch.int32, device=DEV)
    fine = [torch.zeros(s, **i32) for s in ((2, 3), (2,), (2, 3), (2,), (2,))]
    behind = space[4 * 4096:]
    # Beside the caches in their buffer.
    ops.copy_kv_pages(state, behind[:6].view(3, 2))
    ops.compact_kv(state, *fine[:4], behind[6:8])
    torch.cuda.synchronize()
    for layer in (k[0], k[1], v[0], v[1]):
        inside = layer.view(-1)[-16:].view(torch.int32)
        with pytest.raises(ValueError, match="overlap the paged caches"):
            ops.copy_kv_pages(state, inside[:6].view(3, 2))
        for i, t in enumerate(fine):
            args = list(fine)
            args[i] = inside[: t.numel()].view(t.shape)
            with pytest.raises(ValueError, match="overlap the paged caches"):
                ops.compact_kv(state, *args)


def test_lengths_without_layers(ops):
    """No layer moves a row, seq_lens is written all the same."""
    c = Caches(ops, "separate", 2, 6, 16, 2, 64)
    c.state.layer_ptrs = c.state.layer_ptrs[:0]
    i32 = dict(dtype=torch.int32, device=DEV)
    seq = torch.full((3,), -7, **i32)
    ops.compact_kv(c.state, torch.tensor([[0, 1]] * 3, **i32), torch.tensor([3, 4, 2**31 - 1], **i32),
                   torch.tensor([[1, 2]] * 3, **i32), torch.tensor([2, 9, 1], **i32), seq)
    ops.copy_kv_pages(c.state, torch.tensor([[0, 1]], device=DEV))
    c.hold(c.planes)
    assert seq.tolist() == [5, 6, 2**31 - 1]


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("pages", [5, 1023, 1025, 5000])
def test_counts_off_a_16_byte_boundary(ops, offset, pages):
    gen = torch.Generator().manual_seed(pages + offset)
    i32 = dict(dtype=torch.int32, device=DEV)
    n = min(pages, 400)
    table = torch.randperm(pages, generator=gen)[:n].view(1, n)
    refs = torch.randint(0, 2, (pages,), generator=gen).tolist()
    space = torch.full((pages + 8,), -50, **i32)
    refs_d = space[offset: offset + pages]
    refs_d.copy_(torch.tensor(refs, dtype=torch.int32))
    free, cur, nxt = torch.full((n,), 99, **i32), torch.tensor([n], device=DEV), torch.tensor([0], device=DEV)
    ops.release_pages(table.to(**i32), torch.tensor([16 * n], **i32), torch.tensor([0], **i32), 16, refs_d, free, cur, nxt)
    torch.cuda.synchronize()
    want = od.release(table.tolist(), [16 * n], [0], 16, refs, [99] * n, n)
    assert (refs_d.tolist(), free.tolist(), nxt.item()) == want
    assert (space[:offset] == -50).all() and (space[offset + pages:] == -50).all()


@pytest.mark.parametrize("direct", [False, True])
def test_prepared_under_a_default_device(ops, monkeypatch, direct):
    """The ranges that the calls look up on the host stay there."""
    if direct:
        monkeypatch.setattr(ops, "_ext", None)
    k = torch.zeros((3, 4, 16, 2, 64), dtype=torch.bfloat16, device=DEV)
    torch.set_default_device(DEV)
    try:
        state = ops.prepare_kv_pages([(k[i], k[i].clone()) for i in range(3)])
    finally:
        torch.set_default_device(None)
    assert state.ranges.device.type == "cpu" and state.layer_ptrs.is_cuda
    ops.copy_kv_pages(state, torch.tensor([[0, 1]], device=DEV))
    torch.cuda.synchronize()
