"""Planted mistakes, on the CPU: outputs that are wrong in one place go through
the comparisons of the drafting operators' GPU tests and have to fail there."""

import numpy as np
import pytest
import torch

import test_gpu_kv_pages as pages_tests
import test_gpu_tree_attention as attention_tests
from oracle import drafting as od


def _outputs(c, **wrong):
    """What a kernel with these arguments would write: the oracle's outputs,
    rounded once."""
    a = dict(c, **wrong)
    out, low, _, _ = od.tree_attention(a["q"], a["k"], a["v"], a["table"].tolist(), a["seq"].tolist(), a["starts"].tolist(),
                                       a["mask"], a["scale"], a["out"], a["lse"], a["dtype"])
    return torch.from_numpy(out).to(a["dtype"]), torch.from_numpy(low).to(torch.float32)


def _plants(c):
    """(name, arguments that a mistake would work with)."""
    own = [m & ~(1 << i) for m, i in zip(c["mask"], [i for n in np.diff(c["starts"]) for i in range(n)])]
    yield "a token without its own bit", {"mask": own}
    yield "a mask one key late", {"mask": [m << 1 for m in c["mask"]]}
    yield "a causal mask", {"mask": [(2 << i) - 1 for n in np.diff(c["starts"]) for i in range(n)]}
    yield "the last key left out", {"seq": c["seq"] - 1, "mask": [m << 1 for m in c["mask"]]}
    yield "a key too many in the context", {"mask": [m | 1 for m in c["mask"]]}
    yield "a scale of powers of two", {"scale": c["scale"] * 1.4426950408889634}
    k, v, table = c["k"].clone(), c["v"].clone(), c["table"]
    k[int(c["table"][0, 0]), 3] = k[int(c["table"][0, 0]), 4]
    yield "one key read twice", {"k": k}
    v[int(c["table"][0, 0]), 3] = 0
    yield "one value not read", {"v": v}
    yield "the first block left out", {"table": torch.cat((torch.full_like(table[:, :1], -1), table[:, 1:]), dim=1)}
    yield "K in the place of V", {"v": c["k"]}
    yield "heads of the next group", {"k": c["k"].roll(1, 2), "v": c["v"].roll(1, 2)}


def _attention_case(dtype):
    c = attention_tests._case(3, [6, 9], [21, 17], 16, 4, 2, 64, dtype, density=0.3)
    c["k"].nan_to_num_(0.5)
    c["v"].nan_to_num_(0.25)
    # (each token sees itself, and the first and the last not every one of the others)
    c["mask"] = [(m | 1 << i) & ((2 << i) - 1) & ~(1 if i > 2 else 0)
                 for m, i in zip(c["mask"], [i for n in (6, 9) for i in range(n)])]
    return c


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_comparison_takes_what_is_right(dtype):
    c = _attention_case(dtype)
    attention_tests._hold(*_outputs(c), attention_tests._want(c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("plant", range(11))
def test_attention_comparison_finds_planted_mistakes(dtype, plant):
    c = _attention_case(dtype)
    name, wrong = list(_plants(c))[plant]
    out, lse = _outputs(c, **wrong)
    want = attention_tests._want(c)
    with pytest.raises(AssertionError):
        attention_tests._hold(out, None, want)
        pytest.fail(name)
    right = _outputs(c)
    # (a mistake in V alone leaves lse as it is)
    if not torch.equal(lse, right[1]):
        with pytest.raises(AssertionError):
            attention_tests._hold(right[0], lse, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_comparison_finds_single_values(dtype):
    """One value off by 3% of its row's largest, a NaN, an lse that is off as by
    a thousandth of a doubled sum, a row behind the last that was written."""
    c = _attention_case(dtype)
    want = attention_tests._want(c)
    for change in ("value", "nan", "lse", "padding"):
        d = attention_tests._case(3, [6, 9], [21, 17], 16, 4, 2, 64, dtype, pad=1) if change == "padding" else c
        expected = attention_tests._want(d) if change == "padding" else want
        out, lse = _outputs(d)
        if change == "value":
            out[4, 2, 63] += 0.03 * out[4, 2].abs().max()
        elif change == "nan":
            out[14, 3, 0] = float("nan")
        elif change == "lse":
            lse[7, 1] += 1e-3 * 0.6931
        else:
            out[15, 0, 0] += 1.0
        with pytest.raises(AssertionError):
            attention_tests._hold(out, lse, expected)


class _Holder(pages_tests.Caches):
    """The comparison of the page tests, over planes of the CPU."""

    def __init__(self, planes):
        self.gpu = planes


@pytest.fixture
def no_gpu(monkeypatch):
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)


def test_page_comparison_finds_planted_mistakes(no_gpu):
    gen = torch.Generator().manual_seed(1)
    planes = [torch.randn((2, 9, 4, 2, 8), generator=gen).to(torch.bfloat16) for _ in range(2)]
    pairs, moves = [(0, 8), (2, 1)], ([[4, 5, 6]], [3], [[0, 2, 5, 7]], [4])
    want = od.compact(od.copy_pages(planes, pairs), *moves)
    _Holder(want).hold(want)
    wrong = [
        od.compact(od.copy_pages(planes, pairs[:1]), *moves),                          # a pair left out
        od.compact(od.copy_pages(planes, [p[::-1] for p in pairs]), *moves),            # the wrong way
        od.compact(od.copy_pages(planes, pairs), *moves[:3], [3]),                      # the last row left out
        od.compact(od.copy_pages(planes, pairs), moves[0], [2], *moves[2:]),            # a base one off
        od.copy_pages(planes, pairs),                                                   # nothing moved
        [want[0], planes[1]],                                                           # V as it was
    ]
    one = [x.clone() for x in want]
    one[1].view(torch.int16)[1, 3, 2, 1, 7] ^= 1                                        # one bit of one row
    for planes_ in wrong + [one]:
        with pytest.raises(AssertionError):
            _Holder(planes_).hold(want)


def test_release_comparison_finds_planted_mistakes():
    """Equal arguments, one thing done wrong: the lists differ."""
    args = ([[3, 4, 5], [3, 4, 6], [7, -1, 2]], [48, 40, 48], [0, 16, 0], 16, [0, 0, 0, 1, 0, 0, 0, 0, 0], [99] * 9, 7)
    right = od.release(*args)
    assert right == ([0, 0, 0, 0, 0, 0, 0, 0, 0], [99] * 2 + [2, 4, 5, 6, 7] + [99] * 2, 2)

    def planted(last_page=True, holders=True, ascending=True, below=True, skip=True, reset=True):
        table, held, keep, block, refs, free, cursor = args
        refs, free = list(refs), list(free)
        for row, h, k in zip(table, held, keep):
            for j in range(-(-k // block), -(-h // block) - (not last_page)):
                if row[j] >= 0 or not skip:
                    refs[row[j]] = refs[row[j]] - 1 if holders else -1
        given = [p for p, n in enumerate(refs) if n < 0]
        for p in given:
            refs[p] = 0 if reset else refs[p]
        for i, p in enumerate(given if ascending else given[::-1]):
            free[cursor - (len(given) if below else 0) + i if below else min(cursor + i, 8)] = p
        return refs, free, cursor - len(given)

    assert planted() == right
    for name in ("last_page", "holders", "ascending", "below", "skip", "reset"):
        assert planted(**{name: False}) != right, name


def test_tree_comparison_finds_planted_mistakes():
    parents, starts, seq = [-1, 0, 1, 1, 3, 9, -1, 0], [0, 6, 8], [20, 9]
    mask, pos = od.draft_tree(parents, starts, seq, 8, 1)
    right = od.words_of(mask, 1)
    at = [0, 1, 2, 3, 4, 5, 0, 1]
    one_step = [1 << i | (1 << p if 0 <= p < i else 0) for i, p in zip(at, parents)]
    for wrong in ([m & ~(1 << i) for m, i in zip(mask, at)], one_step, [m << 1 for m in mask], mask[1:] + mask[:1]):
        assert not torch.equal(od.words_of(wrong, 1), right)
    by_index = [int(seq[r]) - (starts[r + 1] - starts[r]) + i for r in range(2) for i in range(starts[r + 1] - starts[r])]
    assert by_index != pos
