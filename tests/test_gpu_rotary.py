"""rotary_embedding and rotary_embedding_to_paged against the rotation in 64
bits (tolerance: oracle.serving.rotary_tolerance, one rounding to the type and
a few in 32 bits)."""

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


def _inv(n, base=10000.0):
    return base ** (-torch.arange(n, dtype=torch.float64) / n)


def _rows(seed, T, width, dtype):
    return torch.randn((T, width), generator=torch.Generator().manual_seed(seed)).to(dtype)


def _pos(seed, T, high=1 << 20):
    p = torch.randint(0, high, (T,), generator=torch.Generator().manual_seed(seed))
    p[: min(T, 3)] = torch.tensor([0, 1, high - 1])[: min(T, 3)]
    return p


def _close(got, x, pos, inv, dim, neox, offset, scale, inverse):
    want, size = osv.rotate(x.double().numpy(), pos.numpy(), inv.numpy(), dim, neox, offset, scale, inverse)
    err = np.abs(got.double().cpu().numpy() - want)
    tol = osv.rotary_tolerance(want, size, x.dtype)
    assert (err <= tol).all(), (err - tol).max()
    # The dims that are not rotated pass through.
    keep = size == 0
    assert (err[keep & (np.abs(want) > 0)] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,dim,rot,offset", [
    (1, 1, 1, 64, 64, 0), (3, 4, 1, 128, 128, 0), (7, 8, 2, 96, 96, 0), (5, 3, 3, 128, 64, 64), (130, 28, 4, 128, 64, 0),
    (2, 2, 1, 80, 20, 6), (9, 1, 1, 6, 2, 3), (4, 2, 1, 192, 64, 128), (2500, 2, 1, 64, 32, 16), (1, 64, 8, 256, 256, 0)])
def test_out_of_place_and_in_place(ops, dtype, neox, inverse, T, Hq, Hk, dim, rot, offset):
    inv, pos = _inv(rot // 2), _pos(T, T)
    q, k = _rows(1, T, Hq * dim, dtype), _rows(2, T, Hk * dim, dtype)
    scale = 1.3
    dq, dk, di, dp = q.to(DEV), k.to(DEV), inv.to(DEV), pos.to(DEV)
    qo, ko = torch.empty_like(dq), torch.empty_like(dk)
    ops.rotary_embedding(dp, dq, dk, dim, di, neox, offset, scale, inverse, qo, ko)
    torch.cuda.synchronize()
    assert torch.equal(dq.cpu(), q) and torch.equal(dk.cpu(), k)
    _close(qo, q, pos, inv, dim, neox, offset, scale, inverse)
    _close(ko, k, pos, inv, dim, neox, offset, scale, inverse)
    ops.rotary_embedding(dp.to(torch.int32), dq, dk, dim, di, neox, offset, scale, inverse)
    torch.cuda.synchronize()
    assert torch.equal(dq, qo) and torch.equal(dk, ko)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_slices_of_a_projection_and_three_dims(ops, dtype):
    """q and k as column slices of one buffer, in place; guard columns stay;
    [T, heads, dim] and head-major views give the same."""
    T, Hq, Hk, dim = 33, 6, 2, 64
    inv, pos = _inv(32), _pos(3, T)
    w = Hq * dim + 2 * Hk * dim + 8
    buf = _rows(4, T, w, dtype)
    d = buf.to(DEV)
    q, k = d[:, : Hq * dim], d[:, Hq * dim: (Hq + Hk) * dim]
    ops.rotary_embedding(pos.to(DEV), q, k, dim, inv.to(DEV))
    torch.cuda.synchronize()
    assert torch.equal(d[:, (Hq + Hk) * dim:].cpu(), buf[:, (Hq + Hk) * dim:])
    _close(q, buf[:, : Hq * dim], pos, inv, dim, True, 0, 1.0, False)
    _close(k, buf[:, Hq * dim: (Hq + Hk) * dim], pos, inv, dim, True, 0, 1.0, False)
    src = buf[:, : Hq * dim].reshape(T, Hq, dim).to(DEV)
    major = src.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty((Hq, T, dim), dtype=dtype, device=DEV).transpose(0, 1)
    ops.rotary_embedding(pos.to(DEV), major, None, dim, inv.to(DEV), query_out=out)
    torch.cuda.synchronize()
    assert torch.equal(out.reshape(T, Hq * dim), q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shift", [1, 2, 4])
@pytest.mark.parametrize("neox", [True, False])
def test_rows_off_a_16_byte_boundary(ops, dtype, shift, neox):
    T, H, dim = 11, 3, 64
    inv, pos = _inv(32), _pos(5, T)
    x = _rows(6, T, H * dim, dtype)
    flat = torch.zeros(T * (H * dim + shift) + shift, dtype=dtype, device=DEV)
    v = torch.as_strided(flat, (T, H * dim), (H * dim + shift, 1), shift)
    v.copy_(x)
    ops.rotary_embedding(pos.to(DEV), None, v, dim, inv.to(DEV), neox)
    torch.cuda.synchronize()
    _close(v, x, pos, inv, dim, neox, 0, 1.0, False)


def test_far_and_negative_positions(ops):
    """new - old positions re-rotate; angles past 2^24 turns keep their
    place.  The 64-bit product of position and frequency is off by 2^-52 of
    its turns, in the oracle too: 2^31 / 2 pi turns, 1e-6 of a radian."""
    T, dim = 64, 64
    inv = _inv(32)
    pos = torch.randint(-(2**31), 2**31 - 1, (T,), generator=torch.Generator().manual_seed(0))
    x = _rows(7, T, dim, torch.float32)
    d = x.to(DEV)
    ops.rotary_embedding(pos.to(DEV), None, d, dim, inv.to(DEV))
    torch.cuda.synchronize()
    want, size = osv.rotate(x.double().numpy(), pos.numpy(), inv.numpy(), dim, True)
    assert (np.abs(d.double().cpu().numpy() - want) <= osv.rotary_tolerance(want, size, x.dtype) + 1e-6 * size).all()


def test_inverse_is_the_gradient(ops):
    """The gradient of sum(g * rotate(x)) is the inverse rotation of g, by the
    formula and by differences of the oracle's rotation."""
    T, dim, rot, off, scale = 6, 32, 16, 8, 1.7
    inv, pos = _inv(rot // 2), _pos(8, T, 5000)
    x, g = _rows(8, T, 2 * dim, torch.float32), _rows(9, T, 2 * dim, torch.float32)
    d = g.to(DEV)
    ops.rotary_embedding(pos.to(DEV), d, None, dim, inv.to(DEV), False, off, scale, True)
    torch.cuda.synchronize()
    _close(d, g, pos, inv, dim, False, off, scale, True)
    xn, gn = x.double().numpy(), g.double().numpy()
    got = d.double().cpu().numpy()
    for t, e in [(0, 0), (1, 8), (2, 9), (3, 23), (4, 45), (5, 63)]:
        step = np.zeros_like(xn)
        step[t, e] = 1.0
        hi, _ = osv.rotate(xn + step, pos.numpy(), inv.numpy(), dim, False, off, scale)
        lo, _ = osv.rotate(xn - step, pos.numpy(), inv.numpy(), dim, False, off, scale)
        assert abs((gn * (hi - lo)).sum() / 2 - got[t, e]) <= 1e-5 * (1 + abs(got[t, e]))


def _caches(fmt, pages, block, heads, dim, dtype, seed):
    """(what the op takes, K view, V view, kwargs), each [pages, block, heads, dim]."""
    gen = torch.Generator().manual_seed(seed)

    def make(shape):
        return torch.randn(shape, generator=gen).to(dtype).to(DEV)

    if fmt == "separate":
        k, v = make((pages, block, heads, dim)), make((pages, block, heads, dim))
        return (k, v), k, v, {}
    if fmt == "head_major":
        k, v = (make((pages, heads, block, dim)).transpose(1, 2) for _ in range(2))
        return (k, v), k, v, {}
    if fmt == "merged":
        c = make((pages, 2, block, heads, dim))
        return c, c[:, 0], c[:, 1], {"kvcache_format_raw": 1}
    c = make((2, pages, block, heads, dim))
    return c, c[0], c[1], {"kvcache_format_raw": 1, "vllm_two_major": True}


@pytest.mark.parametrize("fmt", ["separate", "head_major", "merged", "two_major"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,Hq,Hk,dim,rot,offset,block", [
    (1, 4, 1, 128, 128, 0, 16), (77, 6, 2, 96, 96, 0, 16), (200, 4, 4, 64, 32, 32, 48), (3000, 2, 1, 64, 64, 0, 128)])
def test_to_paged(ops, fmt, dtype, T, Hq, Hk, dim, rot, offset, block):
    pages = -(-T // block) + 3
    caches, kc, vc, kw = _caches(fmt, pages, block, Hk, dim, dtype, T)
    inv, pos = _inv(rot // 2), _pos(10, T)
    qkv = _rows(11, T, (Hq + 2 * Hk) * dim, dtype)
    d = qkv.to(DEV)
    q, k, v = d.split([Hq * dim, Hk * dim, Hk * dim], dim=1)
    slots = torch.randperm(pages * block, generator=torch.Generator().manual_seed(12))[:T]
    if T > 2:
        slots[T // 2] = -1
        slots[T // 3] = pages * block
        slots[2] = 2**40
    before_k, before_v = kc.clone(), vc.clone()
    qo = torch.empty((T, Hq * dim), dtype=dtype, device=DEV)
    ops.rotary_embedding_to_paged(pos.to(DEV), q, k, v, caches, slots.to(DEV), dim, inv.to(DEV), True, offset, 0.9, qo, **kw)
    torch.cuda.synchronize()
    assert torch.equal(d.cpu(), qkv)
    _close(qo, qkv[:, : Hq * dim], pos, inv, dim, True, offset, 0.9, False)
    there = (slots >= 0) & (slots < pages * block)
    rows_k = kc.reshape(pages * block, Hk * dim)[slots[there].to(DEV)]
    rows_v = vc.reshape(pages * block, Hk * dim)[slots[there].to(DEV)]
    _close(rows_k, qkv[there, Hq * dim: (Hq + Hk) * dim], pos[there], inv, dim, True, offset, 0.9, False)
    assert torch.equal(rows_v.cpu(), qkv[there, (Hq + Hk) * dim:])
    rest = torch.ones(pages * block, dtype=torch.bool)
    rest[slots[there]] = False
    for now, before in ((kc, before_k), (vc, before_v)):
        a, b = (x.reshape(pages * block, -1)[rest.to(DEV)] for x in (now, before))
        assert torch.equal(a, b)
    # Without a query, 32-bit slots (those past 32 bits among the skipped).
    kc.copy_(before_k)
    vc.copy_(before_v)
    ops.rotary_embedding_to_paged(pos.to(DEV), None, k, v, caches, slots.clamp(-1, 2**31 - 1).to(DEV, torch.int32), dim,
                                  inv.to(DEV), True, offset, 0.9, **kw)
    torch.cuda.synchronize()
    assert torch.equal(kc.reshape(pages * block, Hk * dim)[slots[there].to(DEV)], rows_k)


def test_cache_rows_past_32_bits(ops):
    """Rows more than 4 GiB into a cache."""
    block, heads, dim = 128, 8, 128
    pages = (5 << 30) // (block * heads * dim * 2)
    kc, vc = (torch.zeros((pages, block, heads, dim), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    T = 4
    slots = torch.tensor([0, pages * block - 1, pages * block - 130, (pages - 2) * block])
    k, v = _rows(1, T, heads * dim, torch.bfloat16), _rows(2, T, heads * dim, torch.bfloat16)
    inv, pos = _inv(64), _pos(3, T)
    ops.rotary_embedding_to_paged(pos.to(DEV), None, k.to(DEV), v.to(DEV), (kc, vc), slots.to(DEV), dim, inv.to(DEV))
    torch.cuda.synchronize()
    _close(kc.view(-1, heads * dim)[slots.to(DEV)], k, pos, inv, dim, True, 0, 1.0, False)
    assert torch.equal(vc.view(-1, heads * dim)[slots.to(DEV)].cpu(), v)


def test_replays_and_a_second_stream(ops):
    T, H, dim = 50, 4, 64
    inv = _inv(32).to(DEV)
    pos = torch.zeros(T, dtype=torch.int64, device=DEV)
    q = torch.zeros((T, H * dim), dtype=torch.bfloat16, device=DEV)
    out, want = torch.empty_like(q), torch.empty_like(q)
    ops.rotary_embedding(pos, q, None, dim, inv, query_out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.rotary_embedding(pos, q, None, dim, inv, query_out=out)
    side = torch.cuda.Stream()
    for seed in range(4):
        pos.copy_(_pos(seed, T))
        q.copy_(_rows(seed, T, H * dim, torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            ops.rotary_embedding(pos, q, None, dim, inv, query_out=want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_infinities_and_nans_stay_in_their_pairs(ops):
    T, dim = 4, 64
    x = _rows(1, T, dim, torch.bfloat16)
    y = x.clone()
    y[1, 3], y[2, 40] = float("nan"), float("inf")
    inv, pos = _inv(32).to(DEV), _pos(2, T).to(DEV)
    a, b = x.to(DEV), y.to(DEV)
    ops.rotary_embedding(pos, a, None, dim, inv)
    ops.rotary_embedding(pos, b, None, dim, inv)
    torch.cuda.synchronize()
    differ = (a != b).cpu()
    for t, e in ((1, 3), (1, 35), (2, 8), (2, 40)):
        differ[t, e] = False
    assert not differ.any()
    assert torch.isnan(b[1, 3]) and torch.isnan(b[1, 35])


def test_two_tokens_with_one_slot(ops):
    """Either's row, whole: K and V are each one token's."""
    T, H, dim, block = 600, 2, 64, 16
    inv, pos = _inv(32).to(DEV), torch.zeros(T, dtype=torch.int64, device=DEV)
    rows = torch.arange(T, device=DEV, dtype=torch.float32)[:, None].expand(T, H * dim).contiguous()
    caches = tuple(torch.full((2, block, H, dim), -1.0, device=DEV) for _ in range(2))
    slots = torch.full((T,), 5, dtype=torch.int64, device=DEV)
    slots[::2] = 21
    ops.rotary_embedding_to_paged(pos, None, rows, rows.clone(), caches, slots, dim, inv)
    torch.cuda.synchronize()
    for c in caches:
        flat = c.view(2 * block, H * dim).cpu()
        for slot, odd in ((5, 1), (21, 0)):
            assert set(flat[slot].long().tolist()) <= set(range(odd, T, 2))
        flat[[5, 21]] = -1.0
        assert (flat == -1.0).all()
