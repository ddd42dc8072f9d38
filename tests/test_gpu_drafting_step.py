"""The operators of drafting and branching as a step uses them, beside the
slot maps, rotary positions and the KV transfers: drafts get slots and a tree's
positions, attend, the accepted path moves together, and the pages behind it go
back; requests fork and end."""

import numpy as np
import pytest
import torch

from oracle import drafting as od
from oracle import serving as osv

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HQ, HK, D, BS, LAYERS = 8, 2, 64, 16, 3
DT = torch.bfloat16
I32, I64 = dict(dtype=torch.int32, device=DEV), dict(dtype=torch.int64, device=DEV)


@pytest.fixture(scope="module")
def ops():
    import lmcache_amd

    return lmcache_amd.c_ops


class Engine:
    """What an engine keeps: every layer's caches, tables, the free list, and
    buffers for R requests that draft at most T tokens."""

    def __init__(self, ops, R, T, pages, seed):
        gen = torch.Generator().manual_seed(seed)
        self.ops, self.R, self.T, self.pages = ops, R, T, pages
        self.k, self.v = (torch.zeros((LAYERS, pages, BS, HK, D), dtype=DT, device=DEV) for _ in range(2))
        self.state = ops.prepare_kv_pages([(self.k[i], self.v[i]) for i in range(LAYERS)])
        self.free = torch.randperm(pages, generator=gen).to(**I32)
        self.table = torch.full((R, 24), -1, **I32)
        self.refs = torch.zeros(pages, **I32)
        self.cursor, self.next_cursor = torch.zeros(1, **I64), torch.zeros(1, **I64)
        self.context, self.lens = torch.zeros(R, **I32), torch.zeros(R, **I32)
        self.slots, self.unused, self.positions = (torch.zeros(T, **I64) for _ in range(3))
        self.starts, self.seq = torch.zeros(R + 1, **I32), torch.zeros(R, **I32)
        self.parents, self.mask = torch.zeros(T, **I32), torch.zeros((T, 1), **I64)
        self.qkv = torch.zeros((LAYERS, T, (HQ + 2 * HK) * D), dtype=DT, device=DEV)
        self.out = torch.zeros((LAYERS, T, HQ, D), dtype=DT, device=DEV)
        self.lse = torch.zeros((LAYERS, T, HQ), device=DEV)
        self.keep, self.keep_lens, self.after = torch.zeros((R, 8), **I32), torch.zeros(R, **I32), torch.zeros(R, **I32)
        from lmcache_amd import formats

        self.inv, self.scale = formats.rotary_inv_freq(D, 10000.0)
        self.inv_dev = self.inv.to(DEV)

    def verify(self):
        """Drafts to slots, masks and positions, and every layer's attention."""
        o = self.ops
        o.build_slot_mapping(self.lens, self.context, self.table, BS, self.slots, self.unused, self.starts, self.seq,
                             self.free, self.cursor, self.next_cursor)
        o.build_draft_tree(self.parents, self.starts, self.seq, self.mask, self.positions)
        for i in range(LAYERS):
            q, k, v = self.qkv[i].split([HQ * D, HK * D, HK * D], dim=1)
            caches = (self.k[i], self.v[i])
            o.rotary_embedding_to_paged(self.positions, q, k, v, caches, self.slots, D, self.inv_dev, scale=self.scale)
            o.tree_attention(q.view(self.T, HQ, D), caches, self.table, self.seq, self.starts, self.mask, D ** -0.5,
                             self.out[i], self.lse[i])
        self.cursor.copy_(self.next_cursor)

    def accept(self):
        """The accepted paths behind their contexts, the pages behind them back."""
        o = self.ops
        o.compact_kv(self.state, self.table, self.context, self.keep, self.keep_lens, self.after)
        o.release_pages(self.table, self.seq, self.after, BS, self.refs, self.free, self.cursor, self.next_cursor)
        self.context.copy_(self.after)
        self.cursor.copy_(self.next_cursor)

    def prepare(self, lens, gen):
        parents = [int(torch.randint(-1, i, (1,), generator=gen)) if i else -1 for n in lens for i in range(n)]
        self.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        self.parents.zero_()
        self.parents[: len(parents)] = torch.tensor(parents, **I32)
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=gen).to(DT))
        return parents


def _path(parents, leaf):
    path = []
    while leaf >= 0:
        path.append(leaf)
        leaf = parents[leaf]
    return path[::-1]


@pytest.mark.parametrize("captured", [False, True])
def test_drafting_steps(ops, captured):
    R, T = 5, 60
    e = Engine(ops, R, T, 90, 1)
    gen = torch.Generator().manual_seed(2)
    graphs = None
    if captured:
        e.verify()
        e.accept()
        torch.cuda.synchronize()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for g, f in zip(graphs, (e.verify, e.accept)):
            with torch.cuda.graph(g):
                f()
    context = [0] * R
    rows = [[[] for _ in range(R)] for _ in range(LAYERS)]  # (k, v) rows that the pages must hold
    for step, lens in enumerate([[20, 3, 17, 0, 9], [8, 8, 8, 8, 8], [1, 12, 5, 30, 2], [8, 1, 8, 8, 8]]):
        parents = e.prepare(lens, gen)
        before = e.qkv.clone().cpu()
        out0 = e.out.clone().cpu()
        graphs[0].replay() if graphs else e.verify()
        torch.cuda.synchronize()
        starts = e.starts.tolist()
        total = starts[-1]
        assert starts == [0] + np.cumsum(lens).tolist() and e.seq.tolist() == [c + n for c, n in zip(context, lens)]
        slots = e.slots[:total]
        assert (slots >= 0).all() and slots.unique().numel() == total
        mask, pos = od.draft_tree(parents + [0] * (T - total), starts, e.seq.tolist(), T, 1)
        assert od.mask_of(e.mask.cpu()) == mask and e.positions.tolist() == pos
        for i in range(LAYERS):
            # Rotated to the tree's positions, one rounding away; attention over what the pages hold.
            want_k, size = osv.rotate(before[i, :, HQ * D: (HQ + HK) * D].double().numpy(), pos, e.inv.numpy(), D, True, 0, e.scale)
            flat_k, flat_v = (x[i].reshape(-1, HK * D) for x in (e.k, e.v))
            got = flat_k[slots].double().cpu().numpy()
            assert (np.abs(got - want_k[:total]) <= osv.rotary_tolerance(want_k, size, DT)[:total]).all()
            assert torch.equal(flat_v[slots].cpu(), before[i, :total, (HQ + HK) * D:])
            q = e.qkv[i, :, : HQ * D].cpu().reshape(T, HQ, D)
            want = od.tree_attention(q, e.k[i].cpu(), e.v[i].cpu(), e.table.tolist(), e.seq.tolist(), starts, mask, D ** -0.5,
                                     out0[i], e.lse[i].cpu(), DT)
            assert (np.abs(e.out[i].double().cpu().numpy() - want[0]) <= want[2]).all()
            assert torch.equal(e.out[i, total:].cpu(), out0[i, total:])
        # A path of each tree is accepted.
        paths = []
        for r, n in enumerate(lens):
            leaf = int(torch.randint(-1, n, (1,), generator=gen)) if n else -1
            paths.append(_path(parents[starts[r]: starts[r + 1]], leaf)[:8])
            for i in range(LAYERS):
                for x in paths[r]:
                    s = int(slots[starts[r] + x])
                    rows[i][r].append((e.k[i].reshape(-1, HK * D)[s].clone(), e.v[i].reshape(-1, HK * D)[s].clone()))
        e.keep.zero_()
        for r, p in enumerate(paths):
            e.keep[r, : len(p)] = torch.tensor(p, **I32)
        e.keep_lens.copy_(torch.tensor([len(p) for p in paths], dtype=torch.int32))
        graphs[1].replay() if graphs else e.accept()
        torch.cuda.synchronize()
        context = [c + len(p) for c, p in zip(context, paths)]
        assert e.context.tolist() == context
        held = [int(x) for r in range(R) for x in e.table[r, : -(-context[r] // BS)]]
        assert e.cursor.item() == len(held)
        assert sorted(held + e.free[len(held):].tolist()) == list(range(e.pages))
        for i in range(LAYERS):
            for r in range(R):
                for j, (k, v) in enumerate(rows[i][r]):
                    page, at = int(e.table[r, j // BS]), j % BS
                    assert torch.equal(e.k[i, page, at].reshape(-1), k) and torch.equal(e.v[i, page, at].reshape(-1), v)


def test_forks_share_pages_and_end(ops):
    """A request forks (whole pages shared, the last one copied), both go on
    differently, and end; the pages go to memory objects and back to the list."""
    e = Engine(ops, 2, 40, 40, 3)
    gen = torch.Generator().manual_seed(4)
    e.prepare([40, 0], gen)
    e.parents.copy_(torch.arange(-1, 39))      # a prompt is a chain
    e.verify()
    e.context.copy_(e.seq)
    # The fork: 2 whole pages shared, the third (8 rows) copied to a page of the list.
    e.table[1] = e.table[0]
    e.refs[e.table[0, :2].long()] += 1
    at = int(e.cursor)
    e.table[1, 2] = e.free[at]
    e.cursor += 1
    e.context[1] = e.context[0]
    ops.copy_kv_pages(e.state, torch.stack((e.table[0, 2:3], e.table[1, 2:3]), dim=1))
    assert torch.equal(e.k[:, int(e.table[0, 2]), :8], e.k[:, int(e.table[1, 2]), :8])
    prefix = e.k[:, e.table[0, :2].long()].clone()
    # Both draft the same tokens after the same context: the same attention.
    e.prepare([6, 6], gen)
    e.qkv[:, 6:12] = e.qkv[:, :6]
    e.parents[6:12] = e.parents[:6]
    e.verify()
    torch.cuda.synchronize()
    assert torch.equal(e.out[:, :6], e.out[:, 6:12])
    # They accept different ones.
    paths = [[0], [0, 1, 5]]
    for r, p in enumerate(paths):
        e.keep[r, : len(p)] = torch.tensor(p, **I32)
    e.keep_lens.copy_(torch.tensor([1, 3], dtype=torch.int32))
    e.accept()
    torch.cuda.synchronize()
    assert e.context.tolist() == [41, 43] and torch.equal(e.k[:, e.table[0, :2].long()], prefix)
    # A request's rows to a memory object, by the slots of all its tokens.
    one = torch.full((1,), 43, **I32)
    slots = torch.empty(43, **I64)
    ops.build_slot_mapping(one, torch.zeros_like(one), e.table[1:2], BS, slots)
    obj = torch.zeros((2, LAYERS, 43, HK * D), dtype=DT, device=DEV)
    ptrs = torch.tensor([x.data_ptr() for i in range(LAYERS) for x in (e.k[i], e.v[i])], **I64)
    ops.multi_layer_kv_transfer(obj, ptrs, slots, torch.device(DEV), e.pages * BS, True, False, 2)
    torch.cuda.synchronize()
    assert torch.equal(obj[0], e.k.view(LAYERS, -1, HK * D)[:, slots])
    # The first ends: the shared pages stay.
    held = e.context.clone()
    none = torch.zeros(2, **I32)
    none[1] = 43
    ops.release_pages(e.table, held, none, BS, e.refs, e.free, e.cursor, e.next_cursor)
    e.cursor.copy_(e.next_cursor)
    torch.cuda.synchronize()
    assert e.refs.sum() == 0 and e.cursor.item() == 3
    assert sorted(e.free[3:].tolist() + e.table[1, :3].tolist()) == list(range(e.pages))
    # Then the second.
    held[0] = none[1] = 0
    ops.release_pages(e.table, held, none, BS, e.refs, e.free, e.cursor, e.next_cursor)
    torch.cuda.synchronize()
    assert e.next_cursor.item() == 0 and sorted(e.free.tolist()) == list(range(e.pages))


def test_the_ctypes_path_gives_the_same(ops, monkeypatch):
    """Without the C++ binding the same functions are called through ctypes."""
    results = []
    for direct in (False, True):
        if direct:
            monkeypatch.setattr(ops, "_ext", None)
        e = Engine(ops, 3, 30, 50, 5)
        gen = torch.Generator().manual_seed(6)
        e.prepare([9, 5, 12], gen)
        e.verify()
        e.keep[:, :3] = torch.tensor([[0, 2, 3], [1, 2, 4], [0, 5, 11]], **I32)
        e.keep_lens.fill_(3)
        e.accept()
        ops.copy_kv_pages(e.state, torch.tensor([[int(e.table[0, 0]), int(e.free[40])]], device=DEV))
        torch.cuda.synchronize()
        results.append([x.clone() for x in (e.mask, e.positions, e.out, e.lse, e.k, e.v, e.free, e.refs, e.cursor, e.context)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
