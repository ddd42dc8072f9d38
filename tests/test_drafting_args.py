"""Refusals of the operators of drafting and branching (CPU: the checks run
before any device call; descriptors carry addresses that nothing reads), and
their oracle against closed forms."""

import ctypes
import math

import numpy as np
import pytest
import torch

from lmcache_amd import _lib, c_ops
from oracle import drafting as od

L = _lib.load()


def _t(dtype, *shape, device=0, data=None, strides=None):
    d = _lib.LmcTensor()
    _t.next += 1 << 34
    d.data = data or _t.next
    d.dtype, d.device, d.ndim = dtype, device, len(shape)
    step = 1
    for i in reversed(range(len(shape))):
        d.sizes[i], d.strides[i] = shape[i], step if strides is None else strides[i]
        step *= shape[i]
    return d


_t.next = 1 << 40

U8, I32, I64, BF16, F16, F32 = _lib.U8, _lib.I32, _lib.I64, _lib.BF16, _lib.F16, _lib.F32


def _refuses(status, text):
    assert status == _lib.ERR_VALUE, (status, L.lmc_last_error())
    assert text.encode() in L.lmc_last_error(), L.lmc_last_error()
    with pytest.raises(ValueError):
        _lib.raise_for(status)


def _ptr(t):
    return None if t is None else ctypes.byref(t)


def _caches(n=2, pages=6, block=16, heads=2, dim=64, dtype=BF16, device=0, strides=None):
    return [_t(dtype, pages, block, heads, dim, device=device, strides=strides) for _ in range(n)]


def _array(caches):
    return (_lib.LmcTensor * max(1, len(caches)))(*caches)


# --- build_draft_tree ------------------------------------------------------


def _tree(**over):
    a = dict(parents=_t(I32, 9), starts=_t(I32, 4), seq=_t(I32, 3), mask=_t(I64, 9, 2), pos=_t(I64, 9))
    a.update(over)
    return L.lmc_build_draft_tree(*(_ptr(a[n]) for n in ("parents", "starts", "seq", "mask", "pos")), None)


_PARENTS = _t(I32, 9)
_MASK = _t(I64, 9, 2)


@pytest.mark.parametrize("over,text", [
    ({"parents": None}, "parents is null"),
    ({"starts": None}, "query_start_loc is null"),
    ({"seq": None}, "seq_lens is null"),
    ({"mask": None}, "tree_mask is null"),
    ({"mask": _t(I64, 9, 2, device=-1)}, "tree_mask is not on a GPU"),
    ({"mask": _t(I32, 9, 2)}, "tree_mask has a dtype"),
    ({"mask": _t(I64, 8, 2)}, "tree_mask must be"),
    ({"mask": _t(I64, 18)}, "tree_mask must be"),
    ({"mask": _t(I64, 9, 0)}, "1 to 16 words"),
    ({"mask": _t(I64, 9, 17)}, "1 to 16 words"),
    ({"mask": _t(I64, 9, 2, strides=[4, 2])}, "rows must be contiguous"),
    ({"mask": _t(I64, 9, 2, strides=[1, 1])}, "overlapping rows"),
    ({"parents": _t(I64, 9)}, "parents has a dtype"),
    ({"parents": _t(I32, 9, strides=[2])}, "parents must be 1-D"),
    ({"parents": _t(I32, 9, device=1)}, "parents is not on the GPU"),
    ({"starts": _t(I32, 3)}, "query_start_loc must have"),
    ({"seq": _t(I64, 3)}, "seq_lens has a dtype"),
    ({"pos": _t(I32, 9)}, "positions has a dtype"),
    ({"pos": _t(I64, 8)}, "differ in length"),
    ({"mask": _MASK, "pos": _t(I64, 9, data=_MASK.data + 8)}, "positions and tree_mask overlap"),
    ({"parents": _PARENTS, "pos": _t(I64, 9, data=_PARENTS.data)}, "overlaps what it is computed from"),
    ({"parents": _PARENTS, "mask": _t(I64, 9, 2, data=_PARENTS.data + 32)}, "overlaps what it is computed from"),
])
def test_draft_tree_refusals(over, text):
    _refuses(_tree(**over), text)


# --- tree_attention ----------------------------------------------------------


def _attend(sizes_only=False, **over):
    a = dict(q=_t(BF16, 9, 8, 64), caches=_caches(), table=_t(I32, 3, 5), seq=_t(I32, 3), starts=_t(I32, 4),
             mask=_t(I64, 9, 1), scale=0.125, out=_t(BF16, 9, 8, 64), lse=_t(F32, 9, 8), ws=_t(U8, 1 << 33), fmt=2)
    a.update(over)
    size = ctypes.c_int64(-1)
    st = L.lmc_tree_attention(_ptr(a["q"]), _array(a["caches"]), len(a["caches"]), _ptr(a["table"]), _ptr(a["seq"]),
                              _ptr(a["starts"]), _ptr(a["mask"]), a["scale"], _ptr(a["out"]), _ptr(a["lse"]),
                              _ptr(a["ws"]), ctypes.byref(size) if sizes_only else None, a["fmt"], 0, None)
    return (st, size.value) if sizes_only else st


_Q = _t(BF16, 9, 8, 64)
_ROWS = _t(BF16, 9, 8, 64)
_FIVE = _t(I32, 3, 5)
_KV = _caches()


@pytest.mark.parametrize("over,text", [
    ({"q": None}, "query is null"),
    ({"out": None}, "output is null"),
    ({"table": None}, "block_table is null"),
    ({"mask": None}, "tree_mask is null"),
    ({"ws": None}, "workspace is null"),
    ({"caches": _caches(dtype=F32), "q": _t(F32, 9, 8, 64), "out": _t(F32, 9, 8, 64)}, "tree_attention takes bfloat16 or float16"),
    ({"caches": _caches(dim=72), "q": _t(BF16, 9, 8, 72), "out": _t(BF16, 9, 8, 72)}, "tree_attention takes heads of"),
    ({"caches": _caches(n=1)}, "takes two caches"),
    ({"caches": _caches(device=-1)}, "not on a GPU"),
    ({"fmt": 3}, "K and V caches of equal shape"),
    ({"q": _t(F16, 9, 8, 64)}, "query has a dtype"),
    ({"out": _t(BF16, 9, 4, 64)}, "differ in shape"),
    ({"q": _t(BF16, 9, 7, 64), "out": _t(BF16, 9, 7, 64), "lse": None}, "not a multiple"),
    ({"q": _t(BF16, 9, 8, 64, strides=[512, 64, 2])}, "must be adjacent"),
    ({"out": _t(BF16, 9, 8, 64, strides=[0, 64, 1])}, "output has overlapping rows"),
    ({"out": _t(BF16, 9, 8, 64, strides=[516, 64, 1])}, "16-byte boundaries"),
    ({"mask": _t(I32, 9, 1)}, "tree_mask has a dtype"),
    ({"mask": _t(I64, 8, 1)}, "tree_mask must be"),
    ({"mask": _t(I64, 9)}, "tree_mask must be"),
    ({"mask": _t(I64, 9, 2, strides=[4, 2])}, "tree_mask rows must be contiguous"),
    ({"mask": _t(I64, 9, 1, strides=[-1, 1])}, "negative strides"),
    ({"mask": _t(I64, 9, 1, device=1)}, "tree_mask is not on the GPU"),
    ({"mask": _t(I64, 9, (1 << 20) + 1)}, "2^20 words"),
    ({"starts": _t(I32, 3)}, "query_start_loc must have"),
    ({"seq": _t(I64, 3)}, "seq_lens has a dtype"),
    ({"table": _t(I32, 4, 5)}, "block_table must be"),
    ({"table": _t(I32, 3, 1 << 27)}, "spans more than 2^30 keys"),
    ({"scale": 0.0}, "scale must be positive"),
    ({"scale": -1.0}, "scale must be positive"),
    ({"scale": math.inf}, "scale must be positive"),
    ({"scale": math.nan}, "scale must be positive"),
    ({"lse": _t(F32, 9, 7)}, "lse must be"),
    ({"lse": _t(BF16, 9, 8)}, "lse has a dtype"),
    ({"lse": _t(F32, 9, 8, strides=[0, 1])}, "lse has overlapping rows"),
    ({"ws": _t(U8, 100)}, "at least"),
    ({"ws": _t(U8, 1 << 33, data=(1 << 50) + 8)}, "16-byte boundary"),
    ({"ws": _t(I32, 1 << 31)}, "workspace has a dtype"),
    ({"q": _Q, "out": _t(BF16, 9, 8, 64, data=_Q.data + 1024)}, "output overlaps query"),
    ({"q": _Q, "out": _t(BF16, 9, 8, 64, data=_Q.data, strides=[64, 576, 1])}, "output overlaps query"),
    ({"q": _Q, "lse": _t(F32, 9, 8, data=_Q.data + 64)}, "lse overlaps query"),
    ({"out": _ROWS, "lse": _t(F32, 9, 8, data=_ROWS.data + 64)}, "output and lse overlap"),
    ({"table": _FIVE, "lse": _t(F32, 9, 8, data=_FIVE.data)}, "overlap the tables"),
    ({"caches": _KV, "out": _t(BF16, 9, 8, 64, data=_KV[1].data)}, "overlap the paged caches"),
    ({"q": _Q, "ws": _t(U8, 1 << 33, data=_Q.data)}, "workspace overlaps query"),
    ({"q": _t(BF16, 1 << 22, 8, 64), "out": _t(BF16, 1 << 22, 8, 64), "lse": None, "mask": _t(I64, 1 << 22, 1)}, "too many rows"),
])
def test_tree_attention_refusals(over, text):
    _refuses(_attend(**over), text)


def test_tree_attention_workspace_sizes():
    st, size = _attend(True)
    assert st == _lib.OK and size > 0
    assert _attend(True, q=_t(BF16, 0, 8, 64), out=_t(BF16, 0, 8, 64), lse=None, mask=_t(I64, 0, 1)) == (_lib.OK, 0)
    assert _attend(True, table=_t(I32, 0, 5), seq=_t(I32, 0), starts=_t(I32, 1)) == (_lib.OK, 0)
    # By the tensors' sizes alone: one for the largest lengths.
    assert _attend(True)[1] == size
    # At most two tiles of 256 rows for each of the 512 places.
    big = _attend(True, q=_t(BF16, 8192, 32, 128), out=_t(BF16, 8192, 32, 128), lse=None, mask=_t(I64, 8192, 1),
                  caches=_caches(heads=8, dim=128), table=_t(I32, 3, 1 << 20))
    assert big[0] == _lib.OK and big[1] <= 512 * 2 * 256 * (128 * 4 + 8) + 512 * 16


# --- pages -------------------------------------------------------------------


def _copy(**over):
    a = dict(ptrs=_t(I64, 3, 2), caches=_caches(), pages=_t(I64, 5, 2), fmt=2)
    a.update(over)
    return L.lmc_copy_kv_pages(_ptr(a["ptrs"]), _array(a["caches"]), len(a["caches"]), _ptr(a["pages"]), a["fmt"], 0, None)


@pytest.mark.parametrize("over,text", [
    ({"ptrs": None}, "layer_ptrs is null"),
    ({"pages": None}, "pages is null"),
    ({"ptrs": _t(I32, 3, 2)}, "layer_ptrs has a dtype"),
    ({"ptrs": _t(I64, 3, 3)}, "layer_ptrs must be"),
    ({"ptrs": _t(I64, 6)}, "layer_ptrs must be"),
    ({"ptrs": _t(I64, 3, 2, strides=[4, 1])}, "layer_ptrs must be contiguous"),
    ({"ptrs": _t(I64, 3, 2, device=-1)}, "layer_ptrs is not on the GPU"),
    ({"ptrs": _t(I64, 70000, 2)}, "more than 65535 layers"),
    ({"ptrs": _t(I64, 40000, 2)}, "too many pages"),
    ({"pages": _t(I64, 5, 3)}, "pages must be"),
    ({"pages": _t(I64, 10)}, "pages must be"),
    ({"pages": _t(F32, 5, 2)}, "pages has a dtype"),
    ({"pages": _t(I64, 5, 2, strides=[1, 5])}, "must be adjacent"),
    ({"pages": _t(I64, 5, 2, device=1)}, "pages is not on the GPU"),
    ({"pages": _t(I64, 1 << 31, 2)}, "too many pairs"),
    ({"caches": _caches(n=1)}, "takes two caches"),
    ({"caches": _caches(device=-1)}, "not on a GPU"),
    ({"caches": _caches(strides=[100, 128, 64, 1])}, "overlapping rows"),
    ({"caches": [_KV[0], _KV[0]]}, "K and V caches overlap"),
    ({"caches": _KV, "pages": _t(I64, 5, 2, data=_KV[0].data + 64)}, "overlap the paged caches"),
    ({"fmt": 9}, "is not a KV cache format"),
    ({"fmt": 3, "caches": [_t(BF16, 6, 16, 1, 64), _t(BF16, 6, 8, 1, 32)]}, "differ in pages, block"),
    ({"fmt": 3, "caches": [_t(BF16, 96, 64), _t(BF16, 96, 32)]}, "caches of this format are"),
    ({"fmt": 6, "ptrs": _t(I64, 3, 4), "caches": [_t(BF16, 6, 16, 32) for _ in range(4)]}, "at most 3 caches"),
    ({"fmt": 6, "ptrs": _t(I64, 3, 2), "caches": [_KV[0], _KV[0]]}, "a layer's caches overlap"),
])
def test_copy_refusals(over, text):
    _refuses(_copy(**over), text)


def _compact(**over):
    a = dict(ptrs=_t(I64, 3, 2), caches=_caches(), table=_t(I32, 4, 5), base=_t(I32, 4), keep=_t(I32, 4, 7), lens=_t(I32, 4),
             seq=_t(I32, 4), fmt=2)
    a.update(over)
    return L.lmc_compact_kv(_ptr(a["ptrs"]), _array(a["caches"]), len(a["caches"]), _ptr(a["table"]), _ptr(a["base"]),
                            _ptr(a["keep"]), _ptr(a["lens"]), _ptr(a["seq"]), a["fmt"], 0, None)


_BASE = _t(I32, 4)


@pytest.mark.parametrize("over,text", [
    ({"table": None}, "block_table is null"),
    ({"base": None}, "base_lens is null"),
    ({"keep": None}, "keep is null"),
    ({"lens": None}, "keep_lens is null"),
    ({"table": _t(I64, 4, 5)}, "block_table has a dtype"),
    ({"table": _t(I32, 3, 5)}, "block_table must be"),
    ({"table": _t(I32, 4, 5, strides=[5, 2])}, "block_table rows must be contiguous"),
    ({"table": _t(I32, 4, 1 << 28)}, "spans 2^31 positions"),
    ({"base": _t(I64, 4)}, "base_lens has a dtype"),
    ({"keep": _t(I64, 4, 7)}, "keep has a dtype"),
    ({"keep": _t(I32, 28)}, "keep must be"),
    ({"keep": _t(I32, 3, 7)}, "keep must be"),
    ({"keep": _t(I32, 4, 7, strides=[14, 2])}, "lists must be contiguous"),
    ({"keep": _t(I32, 4, 7, strides=[-7, 1])}, "negative strides"),
    ({"lens": _t(I32, 5)}, "keep_lens must have"),
    ({"seq": _t(I32, 3)}, "seq_lens must have"),
    ({"seq": _t(I64, 4)}, "seq_lens has a dtype"),
    ({"base": _BASE, "seq": _BASE}, "seq_lens overlaps"),
    ({"caches": _KV, "keep": _t(I32, 4, 7, data=_KV[1].data)}, "overlap the paged caches"),
    ({"table": _t(I32, 70000, 5), "base": _t(I32, 70000), "keep": _t(I32, 70000, 7), "lens": _t(I32, 70000), "seq": None},
     "more than 65535 requests"),
])
def test_compact_refusals(over, text):
    _refuses(_compact(**over), text)


def _release(**over):
    a = dict(table=_t(I32, 4, 5), held=_t(I32, 4), keep=_t(I32, 4), block=16, refs=_t(I32, 90), free=_t(I32, 90),
             cursor=_t(I64, 1), following=_t(I64, 1), ws=_t(U8, 1 << 12), size=None)
    a.update(over)
    return L.lmc_release_pages(_ptr(a["table"]), _ptr(a["held"]), _ptr(a["keep"]), a["block"], _ptr(a["refs"]),
                               _ptr(a["free"]), _ptr(a["cursor"]), _ptr(a["following"]), _ptr(a["ws"]), a["size"], None)


_CURSOR = _t(I64, 1)
_LIST = _t(I32, 90)


@pytest.mark.parametrize("over,text", [
    ({"table": None}, "block_table is null"),
    ({"refs": None}, "page_refs is null"),
    ({"cursor": None}, "free_cursor is null"),
    ({"following": None}, "next_cursor is null"),
    ({"ws": None}, "workspace is null"),
    ({"refs": _t(I32, 90, device=-1)}, "page_refs is not on a GPU"),
    ({"refs": _t(I64, 90)}, "page_refs has a dtype"),
    ({"refs": _t(I32, 90, strides=[2])}, "page_refs must be 1-D"),
    ({"refs": _t(I32, 2**31 - 1)}, "too many entries"),
    ({"table": _t(I64, 4, 5)}, "block_table has a dtype"),
    ({"table": _t(I32, 3, 5)}, "block_table must be"),
    ({"table": _t(I32, 4, 5, strides=[10, 2])}, "block_table rows must be contiguous"),
    ({"held": _t(I64, 4)}, "held_lens has a dtype"),
    ({"keep": _t(I32, 5)}, "differ in length"),
    ({"block": 0}, "block_size must be positive"),
    ({"block": 2**31}, "block_size must be positive"),
    ({"free": _t(I64, 90)}, "free_blocks has a dtype"),
    ({"cursor": _t(I64, 2)}, "free_cursor must have one entry"),
    ({"cursor": _t(I32, 1)}, "free_cursor has a dtype"),
    ({"following": _t(I64, 2)}, "next_cursor must have one entry"),
    ({"cursor": _CURSOR, "following": _CURSOR}, "overlaps what it is computed from"),
    ({"refs": _LIST, "free": _LIST}, "two outputs overlap"),
    ({"ws": _t(U8, 3)}, "at least 4 bytes"),
    ({"ws": _t(U8, 1 << 12, data=(1 << 50) + 2)}, "4-byte boundary"),
])
def test_release_refusals(over, text):
    _refuses(_release(**over), text)


def test_release_workspace_size():
    size = ctypes.c_int64(-1)
    assert _release(ws=None, size=ctypes.byref(size), refs=_t(I32, 5000)) == _lib.OK and size.value == 20
    assert _release(ws=None, size=ctypes.byref(size), refs=_t(I32, 0)) == _lib.OK and size.value == 4


def test_cpu_tensors_are_refused():
    i32, i64 = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError):
        c_ops.build_draft_tree(i32, i32, i32[:1], torch.zeros((2, 1), dtype=torch.int64))
    with pytest.raises(ValueError):
        c_ops.release_pages(i32.view(1, 2), i32[:1], i32[:1], 16, i32, i32, i64, i64)
    q = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        c_ops.tree_attention(q, (q, q), i32.view(1, 2), i32[:1], i32, torch.zeros((2, 1), dtype=torch.int64), 1.0, q)
    with pytest.raises(ValueError):
        c_ops.prepare_kv_pages([(q, q.clone())])


# --- the oracle --------------------------------------------------------------


def test_oracle_trees():
    mask, pos = od.draft_tree([-1, 0, 0, 2, 9, -1], [0, 5, 6], [25, 8], 8, 1)
    assert mask == [1, 0b11, 0b101, 0b1101, 0b10000, 1, 0, 0] and pos == [20, 21, 21, 22, 20, 7, 0, 0]
    chain, pos = od.draft_tree(range(-1, 69), [0, 70], [70], 70, 1)
    assert chain[63] == 2**64 - 1 and chain[64] == 0 and pos[63] == 63 and pos[64] == 0
    rows = [5, 2**127, 2**64 - 1, 0]
    assert od.mask_of(od.words_of(rows, 2)) == rows


def test_oracle_attention():
    """Equal scores: the mean of the values that are seen."""
    k = torch.zeros((3, 4, 1, 2))
    v = torch.arange(24.0).view(3, 4, 1, 2)
    out, low, _, _ = od.tree_attention(torch.ones((2, 1, 2)), k, v, [[2, 0]], [5], [0, 2], [0b01, 0b10], 1.0,
                                       torch.zeros((2, 1, 2)), torch.zeros((2, 1)), torch.float32)
    first = v[2, :3, 0].double().numpy()
    assert np.allclose(out[0, 0], np.concatenate((first, v[2, 3:4, 0].double().numpy())).mean(0))
    assert np.allclose(out[1, 0], np.concatenate((first, v[0, 0:1, 0].double().numpy())).mean(0))
    assert np.allclose(low, math.log(4))


def test_oracle_pages():
    x = torch.arange(12).view(1, 3, 4, 1)
    assert od.copy_pages([x], [(0, 2), (1, -1), (3, 0)])[0].flatten().tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 0, 1, 2, 3]
    moved = od.compact([x], [[2, 0]], [1], [[1, 3, 4]], [3])[0].flatten().tolist()
    assert moved == [0, 1, 2, 3, 4, 5, 6, 7, 8, 10, 0, 1]
    assert od.release([[3, 1], [3, 2]], [8, 5], [4, 0], 4, [0, 0, 0, 1, 0], [9] * 5, 4) == ([0, 0, 0, 0, 0], [9, 9, 1, 2, 9], 2)


def test_oracle_catches_a_planted_mistake():
    """A tree that forgets its tokens' own bits, and a release that leaves out
    the last page, are not what the definitions give."""
    mask, _ = od.draft_tree([-1, 0, 1], [0, 3], [3], 3, 1)
    assert [m & ~(1 << i) for i, m in enumerate(mask)] != mask
    right = od.release([[1, 2]], [8], [0], 4, [0] * 3, [9] * 3, 3)
    assert od.release([[1, 2]], [7], [0], 8, [0] * 3, [9] * 3, 3) != right


def test_oracle_release_past_the_list():
    """Places behind the list's end were never handed out: pages go below it."""
    assert od.release([[0, 1, 2, -1], [3, -1, -1, -1]], [64, 32], [0, 0], 16, [0] * 4, [9] * 4, 6) == ([0] * 4, [0, 1, 2, 3], 0)
    assert od.release([[0, 1]], [32], [16], 16, [0] * 4, [9] * 4, 6) == ([0] * 4, [9, 9, 9, 1], 3)


def _layers_check(caches):
    return L.lmc_check_layers_apart(_array(caches), len(caches), None, None)


def _at(data, *shape, strides=None, dtype=BF16, device=0):
    return _t(dtype, *shape, data=data, strides=strides, device=device)


_BASE_AT = 1 << 50
_ROW = 16 * 2 * 64                       # elements of a page of 16 tokens, 2 heads of 64 dims


@pytest.mark.parametrize("caches", [
    # Layers of one buffer that begin two pages after each other.
    [_at(_BASE_AT, 4, 16, 2, 64), _at(_BASE_AT + 2 * 2 * _ROW, 4, 16, 2, 64)],
    # A last row that is the next layer's first, with others between them.
    [_at(_BASE_AT, 4, 16, 2, 64), _at(1 << 52, 4, 16, 2, 64), _at(_BASE_AT + 4 * 2 * _ROW - 2, 4, 16, 2, 64)],
    # One inside another.
    [_at(_BASE_AT + 2 * _ROW, 1, 16, 2, 64), _at(_BASE_AT, 9, 16, 2, 64)],
    # Rows in turn, one token too far.
    [_at(_BASE_AT, 4, 16, 2, 64, strides=[3 * _ROW, 128, 64, 1]),
     _at(_BASE_AT + 2 * (_ROW - 128), 4, 16, 2, 64, strides=[3 * _ROW, 128, 64, 1])],
])
def test_layers_that_overlap_are_refused(caches):
    for order in (caches, caches[::-1]):
        _refuses(_layers_check(order), "two of the layers' caches overlap")


@pytest.mark.parametrize("caches", [
    [],
    [_at(_BASE_AT, 4, 16, 2, 64)],
    # One behind the other.
    [_at(_BASE_AT + 2 * 4 * _ROW * i, 4, 16, 2, 64) for i in (3, 0, 1, 2)],
    # The layers' pages, K's and V's, in turn in one buffer; rows in turn; heads in turn.
    [_at(_BASE_AT + 2 * _ROW * i, 4, 16, 2, 64, strides=[10 * _ROW, 128, 64, 1]) for i in range(10)],
    [_at(_BASE_AT + 2 * 128 * i, 4, 16, 2, 64, strides=[6 * _ROW, 6 * 128, 64, 1]) for i in range(6)],
    [_at(_BASE_AT + 2 * 64 * i, 4, 16, 2, 64, strides=[6 * _ROW, 6 * 128, 6 * 64, 1]) for i in range(6)],
    # Heads before tokens.
    [_at(_BASE_AT + 2 * _ROW * i, 4, 16, 2, 64, strides=[10 * _ROW, 64, 1024, 1]) for i in range(10)],
    # Caches of no pages, and the same address on two GPUs.
    [_at(_BASE_AT, 0, 16, 2, 64), _at(_BASE_AT, 4, 16, 2, 64), _at(_BASE_AT, 4, 16, 2, 64, device=1)],
])
def test_layers_side_by_side_are_taken(caches):
    assert _layers_check(caches) == _lib.OK, L.lmc_last_error()


def test_many_layers_in_one_buffer_are_told_apart_at_once():
    n = 600
    caches = [_at(_BASE_AT + 2 * _ROW * i, 50, 16, 2, 64, strides=[n * _ROW, 128, 64, 1]) for i in range(n)]
    assert _layers_check(caches) == _lib.OK
    caches[400].data += 2 * 64
    _refuses(_layers_check(caches), "two of the layers' caches overlap")


def _outside(ranges, *tensors):
    flat = [x for r in ranges for x in r]
    ptrs = [None if t is None else ctypes.pointer(t) for t in tensors]
    return L.lmc_check_outside((ctypes.c_int64 * max(1, len(flat)))(*flat), len(ranges),
                               (ctypes.POINTER(_lib.LmcTensor) * max(1, len(ptrs)))(*ptrs), len(ptrs))


_RANGES = [(1 << 40, (1 << 40) + 4096), ((1 << 40) + 8192, (1 << 40) + 8208), (1 << 44, 1 << 45)]


@pytest.mark.parametrize("offset,shape,strides", [
    (0, (1,), None), (4092, (1,), None), (-4, (2,), None), (-64, (4000,), None), (4096, (1025,), None), (8204, (1,), None),
    (4096 - 8, (3, 2), [64, 1]), (4096, (2, 2), [1023, 1]), ((1 << 45) - (1 << 40) - 4, (7,), None), (-4, (1 << 43,), None),
])
def test_lists_over_the_caches_of_a_layer_are_refused(offset, shape, strides):
    t = _t(I32, *shape, data=(1 << 40) + offset, strides=strides)
    _refuses(_outside(_RANGES, None, _t(I32, 9, data=1 << 39), t), "overlap the paged caches of a layer")


@pytest.mark.parametrize("offset,shape,strides", [
    (-4, (1,), None), (4096, (1024,), None), (4096, (2, 2), [1022, 1]), (8208, (99,), None), ((1 << 45) - (1 << 40), (7,), None),
    (100, (0,), None), (100, (3, 0), None),
])
def test_lists_beside_the_caches_are_taken(offset, shape, strides):
    t = _t(I32, *shape, data=(1 << 40) + offset, strides=strides)
    assert _outside(_RANGES, t, None) == _lib.OK and _outside([], t) == _lib.OK and _outside(_RANGES) == _lib.OK


@pytest.mark.parametrize("direct", [False, True])
def test_address_ranges_are_put_in_order(monkeypatch, direct):
    if direct:
        monkeypatch.setattr(c_ops, "_ext", None)
    x = torch.zeros((6, 4, 8), dtype=torch.bfloat16)
    at = x.data_ptr()
    parts = [x[4:], x[0], x[1, :, :4], x[1, :, 4:], x[3, 0]]
    assert c_ops._address_ranges(parts).tolist() == [[at, at + 128], [at + 192, at + 208], [at + 256, at + 384]]
    assert c_ops._address_ranges([]).shape == (0, 2)


@pytest.mark.parametrize("T,R,Hq,Hk,dim,width,rows,pieces", [
    # Few rows (64 of a tile; the pieces that the keys allow), and a whole chip of them.
    (9, 3, 8, 2, 64, 5, 64, 6),
    (512, 32, 32, 8, 128, 512, 64, 64),
    (32, 32, 32, 8, 192, 512, 64, 32),
    (32, 32, 32, 8, 256, 512, 64, 32),
    # 65 to 128 rows; more; 192 dims have 128 rows at most, 256 dims 64.
    (1024, 32, 32, 8, 64, 512, 128, 96),
    (1024, 32, 32, 8, 128, 512, 128, 32),
    (2048, 32, 32, 8, 64, 512, 256, 32),
    (2048, 32, 32, 8, 96, 512, 256, 32),
    (2048, 32, 32, 8, 192, 512, 128, 32),
    (2048, 32, 32, 8, 256, 512, 64, 32),
    # More KV heads than places: one piece each.
    (1, 1, 600, 600, 128, 4096, 64, 1),
    # Seven heads a KV head; a table without pages.
    (13, 13, 28, 4, 64, 300, 64, 128),
    (4, 2, 4, 4, 128, 0, 64, 2),
])
def test_tree_attention_workspace_is_what_the_plan_needs(T, R, Hq, Hk, dim, width, rows, pieces):
    """Two places of `rows` rows (sums of `dim` and two more numbers) for each
    workgroup, and 16 bytes; a byte less is refused."""
    sizes = dict(q=_t(BF16, T, Hq, dim), out=_t(BF16, T, Hq, dim), lse=None, mask=_t(I64, T, 1),
                 caches=_caches(heads=Hk, dim=dim), table=_t(I32, R, width), seq=_t(I32, R), starts=_t(I32, R + 1))
    need = pieces * Hk * (2 * rows * (4 * dim + 8) + 16)
    assert _attend(True, **sizes) == (_lib.OK, need)
    _refuses(_attend(ws=_t(U8, need - 1), **sizes), f"at least {need} bytes")
