"""Refusals of the serving operators, and the rotary frequencies (CPU: the
checks run before any device call; descriptors carry addresses that nothing
reads)."""

import ctypes
import math

import pytest
import torch

from lmcache_amd import _lib, c_ops, formats

L = _lib.load()


def _t(dtype, *shape, device=0, data=None, strides=None):
    d = _lib.LmcTensor()
    _t.next += 1 << 32
    d.data = data or _t.next
    d.dtype, d.device, d.ndim = dtype, device, len(shape)
    step = 1
    for i in reversed(range(len(shape))):
        d.sizes[i], d.strides[i] = shape[i], step if strides is None else strides[i]
        step *= shape[i]
    return d


_t.next = 1 << 36

I32, I64, BF16, F16, F32 = _lib.I32, _lib.I64, _lib.BF16, _lib.F16, _lib.F32


def _refuses(status, text):
    assert status == _lib.ERR_VALUE, (status, L.lmc_last_error())
    assert text.encode() in L.lmc_last_error(), L.lmc_last_error()
    with pytest.raises(ValueError):
        _lib.raise_for(status)


def _ptr(t):
    return None if t is None else ctypes.byref(t)


def _slots(**over):
    a = dict(query=_t(I32, 4), context=_t(I32, 4), table=_t(I32, 4, 8), block=16, slots=_t(I64, 20), positions=_t(I64, 20),
             starts=_t(I32, 5), seq=_t(I32, 4), free=None, cursor=None, following=None)
    a.update(over)
    return L.lmc_build_slot_mapping(_ptr(a["query"]), _ptr(a["context"]), _ptr(a["table"]), a["block"], _ptr(a["slots"]),
                                    _ptr(a["positions"]), _ptr(a["starts"]), _ptr(a["seq"]), _ptr(a["free"]),
                                    _ptr(a["cursor"]), _ptr(a["following"]), None)


_LENS = _t(I32, 4)
_CURSOR = _t(I64, 1)


@pytest.mark.parametrize("over,text", [
    ({"query": None}, "query_lens is null"),
    ({"slots": _t(I64, 20, device=-1)}, "slot_mapping is not on a GPU"),
    ({"slots": _t(I32, 20)}, "slot_mapping has a dtype"),
    ({"slots": _t(I64, 20, strides=[2])}, "slot_mapping must be 1-D and contiguous"),
    ({"query": _t(I32, 4, device=1)}, "query_lens is not on the GPU"),
    ({"query": _t(F32, 4)}, "query_lens has a dtype"),
    ({"context": _t(I64, 4)}, "context_lens has a dtype"),
    ({"context": _t(I32, 5)}, "differ in length"),
    ({"table": _t(I64, 4, 8)}, "block_table has a dtype"),
    ({"table": _t(I32, 3, 8)}, "block_table must be"),
    ({"table": _t(I32, 4, 8, strides=[16, 2])}, "block_table rows must be contiguous"),
    ({"table": _t(I32, 4, 8, strides=[0, 1])}, "block_table rows overlap"),
    ({"block": 0}, "block_size must be positive"),
    ({"block": 2**31}, "block_size must be positive"),
    ({"block": 2**30}, "spans 2^31 positions"),
    ({"positions": _t(I64, 19)}, "positions and slot_mapping differ"),
    ({"positions": _t(I32, 20)}, "positions has a dtype"),
    ({"starts": _t(I32, 4)}, "query_start_loc must have"),
    ({"seq": _t(I32, 5)}, "seq_lens must have"),
    ({"context": _LENS, "seq": _LENS}, "overlaps the lengths"),
    ({"cursor": _CURSOR}, "go with free_blocks"),
    ({"free": _t(I64, 9)}, "free_blocks has a dtype"),
    ({"free": _t(I32, 9), "cursor": _t(I64, 2)}, "free_cursor must have one entry"),
    ({"free": _t(I32, 9), "cursor": _CURSOR, "following": _CURSOR}, "next_cursor is free_cursor"),
])
def test_slot_mapping_refusals(over, text):
    _refuses(_slots(**over), text)


def test_slot_mapping_refuses_too_many_requests():
    n = 16385
    _refuses(_slots(query=_t(I32, n), context=_t(I32, n), table=_t(I32, n, 8), starts=_t(I32, n + 1), seq=_t(I32, n)),
             "at most 16384 requests")


def _rotary(**over):
    a = dict(pos=_t(I64, 5), q=_t(BF16, 5, 256), k=_t(BF16, 5, 128), dim=64, inv=1 << 35, n=32, scale=1.0, neox=1, offset=0,
             qo=None, ko=None)
    a.update(over)
    return L.lmc_rotary_embedding(_ptr(a["pos"]), _ptr(a["q"]), _ptr(a["k"]), a["dim"], a["inv"], a["n"], a["scale"],
                                  a["neox"], a["offset"], 0, _ptr(a["qo"]), _ptr(a["ko"]), None)


_Q = _t(BF16, 5, 256)


@pytest.mark.parametrize("over,text", [
    ({"q": None, "k": None}, "neither query nor key"),
    ({"q": _t(BF16, 5, 256, device=-1)}, "must be on a GPU"),
    ({"q": _t(I32, 5, 256)}, "bfloat16, float16 or float32"),
    ({"k": _t(F16, 5, 128)}, "key has a dtype"),
    ({"k": _t(BF16, 5, 128, device=1)}, "key is not on the GPU"),
    ({"k": _t(BF16, 4, 128)}, "another number of tokens"),
    ({"k": _t(BF16, 5, 100)}, "not a multiple of head_size"),
    ({"k": _t(BF16, 5, 2, 32)}, "heads are not of head_size"),
    ({"k": _t(BF16, 640)}, "must be [tokens, heads"),
    ({"q": _t(BF16, 5, 256, strides=[512, 2])}, "dims must be adjacent"),
    ({"q": _t(BF16, 5, 256, strides=[0, 1])}, "overlapping rows"),
    ({"q": _t(BF16, 5, 256, strides=[200, 1])}, "overlapping rows"),
    ({"dim": 0}, "head_size must be between"),
    ({"dim": 8200}, "head_size must be between"),
    ({"inv": None}, "inv_freq is empty"),
    ({"n": 0}, "inv_freq is empty"),
    ({"n": 33}, "do not lie in a head"),
    ({"n": 16, "offset": 33}, "do not lie in a head"),
    ({"offset": -1}, "do not lie in a head"),
    ({"scale": math.inf}, "scale must be finite"),
    ({"pos": _t(I64, 4)}, "positions must have one entry"),
    ({"pos": _t(F32, 5)}, "positions has a dtype"),
    ({"pos": _t(I64, 5, strides=[2])}, "positions must be 1-D"),
    ({"qo": _t(BF16, 5, 128)}, "query_out differs in shape"),
    ({"qo": _t(F16, 5, 256)}, "query_out has a dtype"),
    ({"q": None, "qo": _t(BF16, 5, 256)}, "query_out without query"),
    ({"k": None, "ko": _t(BF16, 5, 128)}, "key_out without key"),
    ({"q": _Q, "k": _t(BF16, 5, 128, data=_Q.data + 64)}, "overlap"),
    ({"q": _Q, "qo": _t(BF16, 5, 256, data=_Q.data + 2)}, "overlap"),
    ({"q": _Q, "ko": _t(BF16, 5, 128, data=_Q.data)}, "overlap"),
])
def test_rotary_refusals(over, text):
    _refuses(_rotary(**over), text)


def _caches(n=2, pages=6, block=16, heads=2, dim=64, dtype=BF16, device=0):
    arr = (_lib.LmcTensor * n)()
    for i in range(n):
        arr[i] = _t(dtype, pages, block, heads, dim, device=device)
    return arr


def _paged(**over):
    a = dict(pos=_t(I64, 5), q=_t(BF16, 5, 256), k=_t(BF16, 5, 128), v=_t(BF16, 5, 128), caches=_caches(), slots=_t(I64, 5),
             dim=64, n=32, qo=None, fmt=2, two=0)
    a.update(over)
    return L.lmc_rotary_embedding_to_paged(_ptr(a["pos"]), _ptr(a["q"]), _ptr(a["k"]), _ptr(a["v"]), a["caches"],
                                           len(a["caches"]), _ptr(a["slots"]), a["dim"], 1 << 35, a["n"], 1.0, 1, 0,
                                           _ptr(a["qo"]), a["fmt"], a["two"], None)


def _one(t):
    arr = (_lib.LmcTensor * 1)()
    arr[0] = t
    return arr


_K = _t(BF16, 5, 128)


@pytest.mark.parametrize("over,text", [
    ({"k": None}, "key is null"),
    ({"v": None}, "value is null"),
    ({"fmt": 3}, "equal shape"),
    ({"fmt": 6}, "takes MERGED_KV or SEPARATE_KV"),
    ({"fmt": 9}, "is not a KV cache format"),
    ({"caches": _caches(device=-1)}, "not on a GPU"),
    ({"caches": _caches(device=1)}, "differ in device or dtype"),
    ({"caches": _caches(dtype=F16)}, "differ in device or dtype"),
    ({"caches": _caches(dim=32)}, "not of head_size"),
    ({"caches": _caches(heads=4)}, "another number of heads"),
    ({"caches": _one(_t(BF16, 6, 3, 16, 2, 64)), "fmt": 1}, "K and V along"),
    ({"caches": _one(_t(BF16, 1, 2, 16, 2, 64, strides=[0, 2048, 128, 64, 2])), "fmt": 1}, "must be adjacent"),
    ({"caches": _one(_t(BF16, 6, 2, 16, 2, 64, strides=[0, 2048, 128, 64, 1])), "fmt": 1}, "overlapping rows"),
    ({"caches": _one(_t(BF16, 6, 2, 16, 2, 64, data=_K.data)), "fmt": 1, "k": _K}, "overlap the call's rows"),
    ({"slots": _t(I64, 4)}, "slot_mapping must have one entry"),
    ({"slots": _t(F32, 5)}, "slot_mapping has a dtype"),
    ({"q": _K, "k": _K}, "overlap"),
])
def test_rotary_to_paged_refusals(over, text):
    _refuses(_paged(**over), text)


def _attention(**over):
    a = dict(q=_t(BF16, 5, 8, 64), caches=_caches(), shared=_t(I32, 3), P=40, table=_t(I32, 4, 9), seq=_t(I32, 4),
             starts=_t(I32, 5), scale=0.125, o=_t(BF16, 5, 8, 64), lse=_t(F32, 5, 8), ws=_t(_lib.U8, 1 << 20), fmt=2, two=0)
    a.update(over)
    return L.lmc_shared_prefix_attention(_ptr(a["q"]), a["caches"], len(a["caches"]), _ptr(a["shared"]), a["P"],
                                         _ptr(a["table"]), _ptr(a["seq"]), _ptr(a["starts"]), a["scale"], _ptr(a["o"]),
                                         _ptr(a["lse"]), _ptr(a["ws"]), None, a["fmt"], a["two"], None)


@pytest.mark.parametrize("over,text", [
    ({"q": None}, "query is null"),
    ({"caches": _caches(dtype=F32)}, "bfloat16 or float16 caches only"),
    ({"caches": _caches(dim=32)}, "heads of 64, 96, 128, 192 or 256"),
    ({"caches": _caches(heads=3)}, "not a multiple of the caches' heads"),
    ({"fmt": 6}, "takes MERGED_KV or SEPARATE_KV"),
    ({"q": _t(F16, 5, 8, 64)}, "query has a dtype"),
    ({"q": _t(BF16, 5, 512)}, "must be [tokens, heads, dim]"),
    ({"q": _t(BF16, 5, 8, 128), "o": _t(BF16, 5, 8, 128)}, "not of the caches' dim"),
    ({"o": _t(BF16, 5, 4, 64)}, "differ in shape"),
    ({"o": _t(BF16, 5, 8, 64, device=1)}, "output is not on the GPU"),
    ({"q": _t(BF16, 5, 8, 64, strides=[1024, 128, 2])}, "must be adjacent"),
    ({"shared": _t(I64, 3)}, "shared_blocks has a dtype"),
    ({"shared": _t(I32, 2)}, "too few blocks"),
    ({"P": -1}, "shared_len must be"),
    ({"P": 2**30 + 1}, "shared_len must be"),
    ({"table": _t(I32, 3, 9)}, "block_table must be"),
    ({"table": _t(I32, 4, 9, strides=[18, 2])}, "rows must be contiguous"),
    ({"table": _t(I32, 4, 2**26 + 1)}, "more than 2^30 keys"),
    ({"seq": _t(I64, 4)}, "seq_lens has a dtype"),
    ({"starts": _t(I32, 4)}, "query_start_loc must have"),
    ({"scale": 0.0}, "scale must be positive"),
    ({"scale": -1.0}, "scale must be positive"),
    ({"scale": math.nan}, "scale must be positive"),
    ({"lse": _t(F32, 5, 7)}, "lse must be"),
    ({"lse": _t(BF16, 5, 8)}, "lse has a dtype"),
    ({"ws": None}, "workspace is null"),
    ({"ws": _t(_lib.U8, 5000)}, "workspace must be"),
    ({"ws": _t(_lib.U8, 1 << 20, data=(1 << 35) + 8)}, "workspace must be"),
    ({"q": _t(BF16, 5, 8, 64, strides=[516, 64, 1])}, "rows of query and output must start"),
    ({"o": _t(BF16, 5, 8, 64, strides=[64, 64, 1])}, "output has overlapping rows"),
    ({"o": _t(BF16, 5, 8, 64, data=(1 << 35) + 2)}, "rows of query and output must start"),
    ({"caches": _one(_t(BF16, 6, 2, 16, 2, 64, data=(1 << 35) + 8)), "fmt": 1}, "the paged caches' rows must start"),
])
def test_prefix_attention_refusals(over, text):
    _refuses(_attention(**over), text)


_O = _t(BF16, 5, 8, 64)
_SEQ, _STARTS, _TABLE, _POOL = _t(I32, 4), _t(I32, 5), _t(I32, 4, 9), _t(I32, 9)
_PAGES = _caches()
_FLAT = _t(I64, 20)
_WIDE = 1 << 27


def _negative():
    arr = _caches()
    arr[1].strides[0] = -arr[1].strides[0]
    return arr


@pytest.mark.parametrize("call,over,text", [
    # what one workgroup reads while another writes it, and outputs over outputs
    (_slots, {"slots": _FLAT, "positions": _t(I64, 20, data=_FLAT.data + 8)}, "two outputs overlap"),
    (_slots, {"starts": _STARTS, "seq": _t(I32, 4, data=_STARTS.data)}, "two outputs overlap"),
    (_slots, {"table": _TABLE, "starts": _t(I32, 5, data=_TABLE.data + 16)}, "overlaps the table"),
    (_slots, {"free": _POOL, "seq": _t(I32, 4, data=_POOL.data)}, "overlaps the table or the free list"),
    (_slots, {"free": _POOL, "cursor": _CURSOR, "positions": _t(I64, 20, data=_CURSOR.data - 8)}, "free list"),
    (_slots, {"free": _POOL, "following": _t(I64, 1, data=_FLAT.data + 24), "slots": _FLAT}, "two outputs overlap"),
    (_rotary, {"pos": _FLAT, "q": _t(BF16, 20, 256, data=_FLAT.data), "k": None}, "overlap what the call writes"),
    (_rotary, {"q": _t(BF16, 5, 256, data=1 << 35), "k": None}, "overlap what the call writes"),
    (_rotary, {"q": _t(BF16, 5, 256), "k": None, "qo": _t(BF16, 5, 256, data=(1 << 35) + 16)}, "overlap what the call writes"),
    (_rotary, {"scale": 1e300}, "scale must be finite"),
    (_paged, {"slots": _t(I64, 5, data=_PAGES[0].data), "caches": _PAGES}, "overlap the paged caches"),
    (_paged, {"caches": _negative()}, "negative strides"),
    (_attention, {"caches": _negative()}, "negative strides"),
    (_attention, {"scale": 1e-60}, "scale must be positive"),
    (_attention, {"scale": 1e60}, "scale must be positive"),
    (_attention, {"lse": _t(F32, 5, 8, strides=[4, 1])}, "lse has overlapping rows"),
    (_attention, {"lse": _t(F32, 5, 8, strides=[0, 1])}, "lse has overlapping rows"),
    (_attention, {"o": _O, "lse": _t(F32, 5, 8, data=_O.data + 64)}, "output and lse overlap"),
    (_attention, {"o": _O, "ws": _t(_lib.U8, 1 << 20, data=_O.data)}, "workspace overlaps"),
    (_attention, {"q": _O, "ws": _t(_lib.U8, 1 << 20, data=_O.data)}, "workspace overlaps"),
    (_attention, {"lse": _t(F32, 5, 8, data=_SEQ.data), "seq": _SEQ}, "overlap the tables or the lengths"),
    (_attention, {"o": _t(BF16, 5, 8, 64, data=_STARTS.data), "starts": _STARTS}, "overlap the tables or the lengths"),
    (_attention, {"o": _t(BF16, 5, 8, 64, data=_PAGES[1].data), "caches": _PAGES}, "overlap the paged caches"),
    (_attention, {"ws": _t(_lib.U8, 1 << 20, data=_PAGES[0].data), "caches": _PAGES}, "overlap the paged caches"),
    # 15 rows of a group of 16 lie within 32 bits of its first
    (_attention, {"caches": _one(_t(BF16, 1, 2, 16, 2, 64, strides=[32 * _WIDE, 16 * _WIDE, _WIDE // 2, 64, 1])), "fmt": 1},
     "2^27 bytes or more apart"),
])
def test_overlaps_strides_and_scales_are_refused(call, over, text):
    _refuses(call(**over), text)


def test_python_refuses_cpu_tensors():
    x = torch.zeros((2, 64))
    f = torch.ones(32, dtype=torch.float64)
    with pytest.raises(ValueError):
        c_ops.rotary_embedding(torch.zeros(2, dtype=torch.int64), x, None, 64, f)
    with pytest.raises(ValueError):
        c_ops.rotary_embedding(torch.zeros(2, dtype=torch.int64), None, None, 64, f)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        c_ops.build_slot_mapping(i, i, i.view(1, 1), 16, torch.zeros(1, dtype=torch.int64))
    q = x.view(2, 1, 64).bfloat16()
    c = torch.zeros((1, 16, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        c_ops.shared_prefix_attention(q, (c, c), i, 0, i.view(1, 1), i, torch.zeros(2, dtype=torch.int32), 1.0, q.clone())


# ---------------------------------------------------------------------------
# Rotary frequencies
# ---------------------------------------------------------------------------


def test_inv_freq_default_and_linear():
    inv, scale = formats.rotary_inv_freq(8, 10000.0)
    assert scale == 1.0 and inv.dtype == torch.float64
    assert torch.allclose(inv, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    lin, _ = formats.rotary_inv_freq(8, 10000.0, {"type": "linear", "factor": 4})
    assert torch.equal(lin, inv / 4)


def test_inv_freq_dynamic():
    cfg = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 100}
    assert torch.equal(formats.rotary_inv_freq(8, 10000.0, cfg, 50)[0], formats.rotary_inv_freq(8, 10000.0)[0])
    inv, _ = formats.rotary_inv_freq(8, 10000.0, cfg, 300)
    base = 10000.0 * (2.0 * 300 / 100 - 1.0) ** (8 / 6)
    assert torch.allclose(inv, base ** -(torch.arange(4, dtype=torch.float64) / 4), rtol=1e-14)


def test_inv_freq_llama3():
    cfg = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
           "original_max_position_embeddings": 8192}
    inv, scale = formats.rotary_inv_freq(128, 500000.0, cfg)
    plain, _ = formats.rotary_inv_freq(128, 500000.0)
    assert scale == 1.0
    for f, g in zip(plain.tolist(), inv.tolist()):
        wave = 2 * math.pi / f
        if wave < 8192 / 4:
            want = f
        elif wave > 8192:
            want = f / 8
        else:
            keep = (8192 / wave - 1) / 3
            want = (1 - keep) * f / 8 + keep * f
        assert abs(g - want) <= 1e-14 * want


def test_inv_freq_yarn():
    cfg = {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096}
    inv, scale = formats.rotary_inv_freq(64, 10000.0, cfg)
    plain, _ = formats.rotary_inv_freq(64, 10000.0)
    assert abs(scale - (0.1 * math.log(32) + 1)) < 1e-14
    assert torch.allclose(inv[:8], plain[:8], rtol=1e-14)        # over 32 turns in 4096 positions
    assert torch.allclose(inv[-8:], plain[-8:] / 32, rtol=1e-14)  # under one
    assert ((inv[1:] - inv[:-1]) < 0).all()
    assert formats.rotary_inv_freq(64, 10000.0, dict(cfg, attention_factor=1.5))[1] == 1.5
    assert abs(formats.rotary_inv_freq(64, 10000.0, dict(cfg, mscale=0.707, mscale_all_dim=0.707))[1] - 1.0) < 1e-14


def test_inv_freq_longrope():
    cfg = {"rope_type": "longrope", "factor": 4.0, "original_max_position_embeddings": 4096,
           "short_factor": [1.0, 2.0], "long_factor": [3.0, 4.0]}
    plain, _ = formats.rotary_inv_freq(4)
    inv, scale = formats.rotary_inv_freq(4, scaling=cfg, seq_len=4096)
    assert torch.equal(inv, plain / torch.tensor([1.0, 2.0], dtype=torch.float64))
    assert abs(scale - math.sqrt(1 + math.log(4) / math.log(4096))) < 1e-14
    assert torch.equal(formats.rotary_inv_freq(4, scaling=cfg, seq_len=4097)[0], plain / torch.tensor([3.0, 4.0], dtype=torch.float64))


@pytest.mark.parametrize("args", [
    (7,), (0,), (8, 0.0), (8, 1e4, {"rope_type": "linear"}), (8, 1e4, {"rope_type": "linear", "factor": 0}),
    (8, 1e4, {"rope_type": "nothing", "factor": 2, "original_max_position_embeddings": 5}),
    (8, 1e4, {"rope_type": "yarn", "factor": 2}),
    (8, 1.0, {"rope_type": "yarn", "factor": 2, "original_max_position_embeddings": 5}),
    (8, 1e4, {"rope_type": "yarn", "factor": 2, "original_max_position_embeddings": 0}),
    (4, 1e4, {"rope_type": "longrope", "factor": 2, "original_max_position_embeddings": 1, "short_factor": [1.0, 1.0]}),
    (8, 1e4, {"rope_type": "longrope", "factor": 2, "original_max_position_embeddings": 5, "short_factor": [1.0]}),
])
def test_inv_freq_refusals(args):
    with pytest.raises(ValueError):
        formats.rotary_inv_freq(*args)
