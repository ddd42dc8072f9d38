"""Where the serving operators' sizes end, and calls next to those ends that
have to be taken (CPU: checks and sizes are the host's; descriptors carry
addresses that nothing reads)."""

import ctypes

import pytest

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
