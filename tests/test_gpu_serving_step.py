"""The serving operators as a step uses them, one after the other, beside the
KV transfers: lengths to slots, slots to rotated keys in their pages, pages to
attention, and the pages to a memory object."""

import numpy as np
import pytest
import torch

from oracle import serving as osv

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HQ, HK, D, BS = 8, 2, 64, 16
DT = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    import lmcache_amd

    return lmcache_amd.c_ops


class Step:
    """What an engine keeps: one layer's caches, tables, and buffers for R
    requests and at most T new tokens."""

    def __init__(self, ops, R, T, prefix, pages, seed):
        gen = torch.Generator().manual_seed(seed)
        self.ops, self.R, self.T, self.P = ops, R, T, prefix
        self.caches = tuple(torch.zeros((pages, BS, HK, D), dtype=DT, device=DEV) for _ in range(2))
        order = torch.randperm(pages, generator=gen).to(torch.int32)
        n = -(-prefix // BS)
        self.shared, self.free = order[:n].to(DEV), order[n:].contiguous().to(DEV)
        width = 40
        self.table = torch.full((R, width), -1, dtype=torch.int32, device=DEV)
        self.table[:, : prefix // BS] = self.shared[: prefix // BS]   # prefix ends on a block here
        i32, i64 = dict(dtype=torch.int32, device=DEV), dict(dtype=torch.int64, device=DEV)
        self.query_lens, self.context_lens = torch.zeros(R, **i32), torch.full((R,), prefix, **i32)
        self.slots, self.positions = torch.zeros(T, **i64), torch.zeros(T, **i64)
        self.starts, self.seq = torch.zeros(R + 1, **i32), torch.zeros(R, **i32)
        self.cursor, self.next_cursor = torch.zeros(1, **i64), torch.zeros(1, **i64)
        self.qkv = torch.zeros((T, (HQ + 2 * HK) * D), dtype=DT, device=DEV)
        self.out, self.lse = torch.zeros((T, HQ, D), dtype=DT, device=DEV), torch.zeros((T, HQ), device=DEV)
        from lmcache_amd import formats

        self.inv, self.scale = formats.rotary_inv_freq(D, 10000.0, {"rope_type": "linear", "factor": 2.0})
        self.inv_dev = self.inv.to(DEV)

    def __call__(self):
        q, k, v = self.qkv.split([HQ * D, HK * D, HK * D], dim=1)
        self.ops.build_slot_mapping(self.query_lens, self.context_lens, self.table, BS, self.slots, self.positions,
                                    self.starts, self.seq, self.free, self.cursor, self.next_cursor)
        self.ops.rotary_embedding_to_paged(self.positions, q, k, v, self.caches, self.slots, D, self.inv_dev,
                                           scale=self.scale)
        self.ops.shared_prefix_attention(q.view(self.T, HQ, D), self.caches, self.shared, self.P, self.table, self.seq,
                                         self.starts, D ** -0.5, self.out, self.lse)
        # For the next step.
        self.context_lens.copy_(self.seq)
        self.cursor.copy_(self.next_cursor)


def _fill_prefix(s, seed):
    """The prefix's rows, as a retrieve leaves them in the shared blocks."""
    gen = torch.Generator().manual_seed(seed)
    obj = torch.randn((2, 1, s.P, HK * D), generator=gen).to(DT)
    slots = (s.shared.long()[:, None] * BS + torch.arange(BS, device=DEV)).reshape(-1)[: s.P].contiguous()
    ptrs = torch.tensor([c.data_ptr() for c in s.caches], dtype=torch.int64, device=DEV)
    pages = s.caches[0].shape[0]
    s.ops.multi_layer_kv_transfer(obj.to(DEV), ptrs, slots, torch.device(DEV), pages * BS, False, False, 2)
    return obj


@pytest.mark.parametrize("prefix", [64, 160])
@pytest.mark.parametrize("captured", [False, True])
def test_prefill_and_decode_steps(ops, prefix, captured):
    R, T = 6, 70
    s = Step(ops, R, T, prefix, 200, prefix)
    obj = _fill_prefix(s, 1)
    steps = [[9, 1, 30, 0, 17, 3], [1, 1, 1, 0, 1, 1], [1, 2, 1, 20, 1, 0], [1] * 6]
    graph = None
    context = [prefix] * R
    rows = [[] for _ in range(R)]     # each request's own (k, v), rotated, in 64 bits
    table, cursor = s.table.cpu().numpy().astype(np.int64), 0
    if captured:
        s()                           # once before capture, with no tokens
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s()
    for n, lens in enumerate(steps):
        gen = torch.Generator().manual_seed(100 + n)
        qkv = torch.randn(s.qkv.shape, generator=gen).to(DT)
        s.qkv.copy_(qkv)
        s.query_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        before = s.out.clone()
        graph.replay() if graph else s()
        torch.cuda.synchronize()
        slots, pos, starts, seq, table, cursor = osv.slot_mapping(lens, context, table, BS, T, s.free.tolist(), cursor)
        assert np.array_equal(s.slots.cpu().numpy(), slots) and np.array_equal(s.positions.cpu().numpy(), pos)
        assert np.array_equal(s.table.cpu().numpy(), table) and s.cursor.item() == cursor
        total = int(starts[-1])
        # The rotated rows in the pages, to one rounding.
        want_k, size = osv.rotate(qkv[:, HQ * D: (HQ + HK) * D].double().numpy(), pos, s.inv.numpy(), D, True, 0, s.scale)
        flat_k, flat_v = (c.reshape(-1, HK * D) for c in s.caches)
        at = torch.from_numpy(slots[:total]).to(DEV)
        got_k = flat_k[at].double().cpu().numpy()
        tol = osv.rotary_tolerance(want_k, size, DT)
        assert (np.abs(got_k - want_k[:total]) <= tol[:total]).all()
        assert torch.equal(flat_v[at].cpu(), qkv[:total, (HQ + HK) * D:])
        # Attention over what the pages hold.
        q = s.qkv[:, : HQ * D].cpu().view(T, HQ, D)
        want = osv.attention(q, s.caches[0].cpu(), s.caches[1].cpu(), s.shared.tolist(), prefix, table.tolist(), seq.tolist(),
                             starts.tolist(), D ** -0.5, before.cpu(), s.lse.cpu(), DT)
        assert (np.abs(s.out.double().cpu().numpy() - want[0]) <= want[2]).all()
        assert torch.equal(s.out[total:], before[total:])
        context = seq.tolist()
    # A request's pages to a memory object, by the slots of all its tokens.
    r = 2
    n = context[r]
    one = torch.full((1,), n, dtype=torch.int32, device=DEV)
    slots = torch.empty(n, dtype=torch.int64, device=DEV)
    ops.build_slot_mapping(one, torch.zeros_like(one), s.table[r: r + 1], BS, slots)
    out = torch.zeros((2, 1, n, HK * D), dtype=DT, device=DEV)
    ptrs = torch.tensor([c.data_ptr() for c in s.caches], dtype=torch.int64, device=DEV)
    ops.multi_layer_kv_transfer(out, ptrs, slots, torch.device(DEV), s.caches[0].shape[0] * BS, True, False, 2)
    torch.cuda.synchronize()
    assert torch.equal(out[:, :, :prefix].cpu(), obj)
    assert torch.equal(out[0, 0, prefix:], s.caches[0].reshape(-1, HK * D)[slots[prefix:]])


def test_the_ctypes_path_gives_the_same(ops, monkeypatch):
    """Without the C++ binding the same functions are called through ctypes."""
    results = []
    for direct in (False, True):
        if direct:
            monkeypatch.setattr(ops, "_ext", None)
        s = Step(ops, 5, 40, 64, 120, 3)
        obj = torch.randn((2, 1, 64, HK * D), generator=torch.Generator().manual_seed(2)).to(DT).to(DEV)
        slots = (s.shared.long()[:, None] * BS + torch.arange(BS, device=DEV)).reshape(-1).contiguous()
        for c, rows in zip(s.caches, obj):
            c.view(-1, HK * D)[slots] = rows[0]
        s.qkv.copy_(torch.randn(s.qkv.shape, generator=torch.Generator().manual_seed(4)).to(DT))
        s.query_lens.copy_(torch.tensor([9, 0, 20, 1, 1], dtype=torch.int32))
        s()
        k = s.qkv[:, HQ * D: (HQ + HK) * D].contiguous()
        s.ops.rotary_embedding(s.positions, None, k, D, s.inv_dev, inverse=True)
        torch.cuda.synchronize()
        results.append([x.clone() for x in (s.slots, s.table, *s.caches, s.out, s.lse, k)])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_attention_of_a_prefix_by_itself_joins_with_the_rest(ops):
    """lse joins attention over two key ranges into attention over both."""
    s = Step(ops, 4, 4, 64, 120, 5)
    for c in s.caches:
        c.copy_(torch.randn(c.shape, generator=torch.Generator().manual_seed(6)).to(DT))
    s.query_lens.fill_(1)
    s.qkv.copy_(torch.randn(s.qkv.shape, generator=torch.Generator().manual_seed(7)).to(DT))
    s()
    q = s.qkv[:, : HQ * D].reshape(4, HQ, D)
    far = torch.full((4,), 64, dtype=torch.int32, device=DEV)
    a, la = torch.empty_like(s.out), torch.empty_like(s.lse)
    ops.shared_prefix_attention(q, s.caches, s.shared, 64, s.table, far, s.starts, D ** -0.5, a, la)
    # The one own key's attention is its value.
    v = s.caches[1].reshape(-1, HK, D)[s.slots].repeat_interleave(HQ // HK, dim=1)
    k = s.caches[0].reshape(-1, HK, D)[s.slots].repeat_interleave(HQ // HK, dim=1)
    lb = (q.float() * k.float()).sum(-1) * D ** -0.5
    w = torch.sigmoid(lb - la)[..., None]
    joined = a.float() * (1 - w) + v.float() * w
    # Two roundings to bfloat16 of each side and the weights' own.
    assert (joined - s.out.float()).abs().max() <= 3 * 2.0**-8 * max(1.0, joined.abs().max().item())
    assert torch.allclose(torch.logaddexp(la, lb), s.lse, atol=1e-4)
