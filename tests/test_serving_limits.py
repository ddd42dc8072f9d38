"""Where the serving operators' sizes end, and calls next to those ends that
have to be taken (CPU: checks and sizes are the host's; descriptors carry
addresses that nothing reads)."""

import ctypes

import numpy as np
import pytest
import torch

from lmcache_amd import _lib

L = _lib.load()

I32, I64, BF16, F16, F32, U8 = _lib.I32, _lib.I64, _lib.BF16, _lib.F16, _lib.F32, _lib.U8


def _t(dtype, *shape, strides=None, data=None):
    d = _lib.LmcTensor()
    _t.next += 1 << 44
    d.data = data or _t.next
    d.dtype, d.device, d.ndim = dtype, 0, len(shape)
    step = 1
    for i in reversed(range(len(shape))):
        d.sizes[i], d.strides[i] = shape[i], step if strides is None else strides[i]
        step *= shape[i]
    return d


_t.next = 1 << 46


def _ref(t):
    return None if t is None else ctypes.byref(t)


def _array(*tensors):
    arr = (_lib.LmcTensor * len(tensors))()
    for i, t in enumerate(tensors):
        arr[i] = t
    return arr


def _refuses(status, text):
    assert status == _lib.ERR_VALUE, (status, L.lmc_last_error())
    assert text.encode() in L.lmc_last_error(), L.lmc_last_error()


def _rotary(T, dim, n_freq):
    q, pos = _t(BF16, T, dim), _t(I64, T)
    return L.lmc_rotary_embedding(_ref(pos), _ref(q), None, dim, 1 << 35, n_freq, 1.0, 1, 0, 0, None, None, None)


@pytest.mark.parametrize("T", [2**25 - 1, 2**25, 2**31 - 1, 2**31])
def test_rotary_refuses_more_tokens_than_a_launch_has_threads(T):
    """Two tokens a workgroup of 256 threads: 2^25 - 2 of them at most."""
    _refuses(_rotary(T, 64, 32), "too many tokens")


def _attention(T, R, Hq, Hk, dim, block=16, width=64, P=0, **over):
    """(status, workspace bytes): the call that only asks for the size."""
    a = dict(q=_t(BF16, T, Hq, dim), o=_t(BF16, T, Hq, dim), lse=None,
             caches=_array(*(_t(BF16, 6, block, Hk, dim) for _ in range(2))), fmt=2)
    a.update(over)
    table, seq, starts, shared = _t(I32, R, width), _t(I32, R), _t(I32, R + 1), _t(I32, -(-P // block))
    size = ctypes.c_int64(-1)
    status = L.lmc_shared_prefix_attention(_ref(a["q"]), a["caches"], len(a["caches"]), _ref(shared), P, _ref(table), _ref(seq),
                                           _ref(starts), 1.0, _ref(a["o"]), _ref(a["lse"]), None, ctypes.byref(size), a["fmt"],
                                           0, None)
    return status, size.value


@pytest.mark.parametrize("T,R,heads", [(1, 2**19 - 1, 256), (1, 2**17, 128), (2**14, 2**17, 128)])
def test_attention_refuses_more_parts_than_a_launch_has_threads(T, R, heads):
    """A wave for each request, KV head and part: 2^26 of them at most."""
    status, _ = _attention(T, R, heads, heads, 64, width=1024)     # eight parts of a request's own keys
    _refuses(status, "too many rows")


def test_attention_takes_as_many_as_a_launch_has_threads():
    status, size = _attention(1, 2**16, 64, 64, 64, width=1024)
    assert status == _lib.OK and size > 0


def _to_paged(caches, fmt=2, two_major=0):
    """A call of no tokens: the caches are looked at, nothing is launched."""
    pos, k, v, slots = _t(I64, 0), _t(BF16, 0, 128), _t(BF16, 0, 128), _t(I64, 0)
    return L.lmc_rotary_embedding_to_paged(_ref(pos), None, _ref(k), _ref(v), caches, len(caches), _ref(slots), 64, 1 << 35, 32,
                                           1.0, 1, 0, None, fmt, two_major, None)


# Two KV heads of 64 dims in blocks of 16: a row has 64 elements, a block 2048.
def _pair(by, strides, pages=6, v_strides=None):
    k = _t(BF16, pages, 16, 2, 64, strides=strides)
    return _array(k, _t(BF16, pages, 16, 2, 64, strides=v_strides or strides, data=k.data + 2 * by))


_PLAIN = [2048, 128, 64, 1]


@pytest.mark.parametrize("caches,fmt", [
    (_pair(0, _PLAIN), 2),                                          # one cache as K and as V
    (_pair(2048, _PLAIN), 2),                                       # a block further
    (_pair(-64, _PLAIN), 2),                                        # a head before
    (_pair(6 * 2048 - 64, _PLAIN), 2),                              # K's last row is V's first
    (_pair(2048 - 128, [4096, 128, 64, 1]), 2),                     # V begins inside K's part of a page
    (_pair(4096 - 128, [4096, 128, 64, 1]), 2),                     # V ends in the next page's K
    (_pair(64, [8192, 256, 128, 1], v_strides=[8192, 256, 64, 1]), 2),
    (_array(_t(BF16, 6, 2, 16, 2, 64, strides=[2048, 0, 128, 64, 1])), 1),
])
def test_rotary_to_paged_refuses_k_and_v_in_one_place(caches, fmt):
    """Both are written: a row of both would hold either."""
    _refuses(_to_paged(caches, fmt), "K and V caches overlap")


@pytest.mark.parametrize("caches,fmt,two_major", [
    (_pair(6 * 2048, _PLAIN), 2, 0),                                # one behind the other
    (_pair(-6 * 2048, _PLAIN), 2, 0),
    (_pair(2048, [4096, 128, 64, 1]), 2, 0),                        # beside each other in a page
    (_pair(-2048, [4096, 128, 64, 1]), 2, 0),
    (_pair(5 * 2048, [4096, 128, 64, 1]), 2, 0),                    # V from the third page on
    (_pair(2048, [4096, 128, 64, 1], v_strides=[4096, 64, 1024, 1]), 2, 0),  # V of a page head by head
    (_pair(128, [4096, 256, 64, 1]), 2, 0),                         # in turn, token by token
    (_pair(64, [4096, 256, 128, 1]), 2, 0),                         # in turn, row by row
    (_pair(64, [4096, 128, 2048, 1]), 2, 0),                        # in turn within a head
    (_pair(2048, [7, 128, 64, 1], pages=1, v_strides=[9, 128, 64, 1]), 2, 0),
    (_array(_t(BF16, 6, 2, 16, 2, 64)), 1, 0),
    (_array(_t(BF16, 2, 6, 16, 2, 64)), 1, 1),
    (_array(_t(BF16, 6, 2, 16, 2, 64, strides=[4096, 64, 256, 128, 1])), 1, 0),
])
def test_rotary_to_paged_takes_k_and_v_beside_each_other(caches, fmt, two_major):
    status = _to_paged(caches, fmt, two_major)
    assert status == _lib.OK, L.lmc_last_error()


@pytest.mark.parametrize("over,sizes", [
    ({"q": _t(BF16, 1, 8, 64, strides=[1203, 64, 1])}, (1, 8, 2)),              # a token of an odd projection
    ({"o": _t(BF16, 1, 8, 64, strides=[7, 64, 1])}, (1, 8, 2)),
    ({"q": _t(BF16, 5, 1, 64, strides=[64, 3, 1])}, (5, 1, 1)),                 # one head
    ({"o": _t(BF16, 5, 1, 64, strides=[64, 1, 1])}, (5, 1, 1)),
    ({"caches": _array(*(_t(BF16, 6, 16, 1, 64, strides=[1024, 64, 5, 1]) for _ in range(2)))}, (5, 4, 1)),
    ({"caches": _array(*(_t(BF16, 1, 16, 2, 64, strides=[9, 128, 64, 1]) for _ in range(2)))}, (5, 8, 2)),
])
def test_attention_takes_any_stride_of_a_dim_of_one(over, sizes):
    T, Hq, Hk = sizes
    status, size = _attention(T, 1, Hq, Hk, 64, **over)
    assert status == _lib.OK and size > 0, L.lmc_last_error()


@pytest.mark.parametrize("over", [
    {"q": _t(BF16, 2, 8, 64, strides=[1203, 64, 1])},
    {"o": _t(BF16, 2, 8, 64, strides=[1024, 100, 1])},
])
def test_attention_refuses_rows_off_a_16_byte_boundary(over):
    status, _ = _attention(2, 1, 8, 2, 64, **over)
    _refuses(status, "rows of query and output must start")


def _heads(base, by, H, row=3 * 64, T=5):
    """[T, H, 64] from element `by` on, rows `row` apart, tokens H rows."""
    return _t(BF16, T, H, 64, strides=[H * row, row, 1], data=base + 2 * by)


_BASE = 1 << 45


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls are taken, on addresses that are nobody's")
@pytest.mark.parametrize("q,k,qo", [
    (_heads(_BASE, 0, 8), _heads(_BASE, 64, 8), None),                  # q, k and v of a head beside each other
    (_heads(_BASE, 64, 8), _heads(_BASE, 0, 8), None),
    (_heads(_BASE, 0, 8), None, _heads(_BASE, 128, 8)),                 # q turned to v's place
    (_heads(_BASE, 0, 1), _heads(_BASE, 64, 1), None),
    (_heads(_BASE, 0, 8, T=1), _heads(_BASE, 64, 8, T=1), None),
    (_heads(_BASE, 0, 8, row=64), _heads(_BASE, 5 * 8 * 64, 8, row=64), None),
])
def test_rotary_takes_rows_in_turn_of_one_buffer(q, k, qo):
    status = L.lmc_rotary_embedding(_ref(_t(I64, q.sizes[0])), _ref(q), _ref(k), 64, 1 << 35, 32, 1.0, 1, 0, 0, _ref(qo), None,
                                    None)
    assert status != _lib.ERR_VALUE, L.lmc_last_error()


@pytest.mark.parametrize("q,k", [
    (_heads(_BASE, 0, 8), _heads(_BASE, 63, 8)),
    (_heads(_BASE, 0, 8), _heads(_BASE, 3 * 64, 8)),                     # a head further
    (_heads(_BASE, 0, 8), _heads(_BASE, -3 * 64 * 8 + 130, 8)),
    (_heads(_BASE, 0, 8), _t(BF16, 5, 512, strides=[3 * 512, 1], data=_BASE + 128)),
])
def test_rotary_refuses_rows_that_cross(q, k):
    status = L.lmc_rotary_embedding(_ref(_t(I64, 5)), _ref(q), _ref(k), 64, 1 << 35, 32, 1.0, 1, 0, 0, None, None, None)
    _refuses(status, "overlap")


def test_caches_that_are_taken_do_not_cross():
    """Layouts at random: none whose rows cross is taken, and of those whose
    rows do not, most are."""
    rng = np.random.default_rng(0)
    taken = apart = 0
    for _ in range(3000):
        pages, block, heads = (int(rng.integers(1, 4)) for _ in range(3))
        gaps = [int(rng.choice([1, 2, 3])) for _ in range(3)]
        sizes, names, strides, span = {"p": pages, "b": block, "h": heads}, list(rng.permutation(["p", "b", "h"])), {}, 64
        for name, gap in zip(names, gaps):
            strides[name] = span * gap
            span = strides[name] * sizes[name]
        by = 64 * int(rng.integers(-12, 13)) + int(rng.choice([0, 0, 0, 32]))
        st = [strides["p"], strides["b"], strides["h"], 1]
        at = (np.arange(pages)[:, None, None, None] * st[0] + np.arange(block)[:, None, None] * st[1]
              + np.arange(heads)[:, None] * st[2] + np.arange(64)).ravel()
        crosses = np.intersect1d(at, at + by).size > 0
        k = _t(BF16, pages, block, heads, 64, strides=st)
        caches = _array(k, _t(BF16, pages, block, heads, 64, strides=st, data=k.data + 2 * by))
        rows = _t(BF16, 0, heads * 64)
        status = L.lmc_rotary_embedding_to_paged(_ref(_t(I64, 0)), None, _ref(rows), _ref(rows), caches, 2, _ref(_t(I64, 0)), 64,
                                                 1 << 35, 32, 1.0, 1, 0, None, 2, 0, None)
        assert not (crosses and status == _lib.OK), (sizes, st, by)
        apart += not crosses
        taken += status == _lib.OK
    assert taken >= 0.95 * apart, (taken, apart)
