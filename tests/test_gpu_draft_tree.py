"""build_draft_tree against sets of ancestors, token by token."""

import pytest
import torch

from oracle import drafting as od

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    import lmcache_amd

    return lmcache_amd.c_ops


def _random(seed, lens, pad=0, deep=False):
    """(parents, starts, seq_lens): random trees; entries that say "the
    context" in every way; anything behind the last request."""
    gen = torch.Generator().manual_seed(seed)
    parents = []
    for n in lens:
        for i in range(n):
            x = torch.rand(2, generator=gen)
            p = i - 1 if deep else int(x[0] * (i + 1)) - 1
            if not deep and x[1] < 0.1:
                p = [-1, -7, i, i + 3, 2**31 - 1, -(2**31)][int(x[1] * 60)]
            parents.append(p)
    parents += [int(x) for x in torch.randint(-9, 99, (pad,), generator=gen)]
    starts = torch.zeros(len(lens) + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(lens).cumsum(0)
    seq = torch.tensor(lens) + torch.randint(0, 5000, (len(lens),), generator=gen)
    return torch.tensor(parents, dtype=torch.int32), starts, seq.to(torch.int32)


def _check(ops, parents, starts, seq, words, wide=0, with_positions=True):
    N = parents.numel()
    space = torch.full((N, words + wide), 77, dtype=torch.int64, device=DEV)
    mask = space[:, :words]
    pos = torch.full((N,), 77, dtype=torch.int64, device=DEV) if with_positions else None
    ops.build_draft_tree(parents.to(DEV), starts.to(DEV), seq.to(DEV), mask, pos)
    torch.cuda.synchronize()
    want, places = od.draft_tree(parents.tolist(), starts.tolist(), seq.tolist(), N, words)
    assert torch.equal(mask.cpu(), od.words_of(want, words))
    assert (space[:, words:] == 77).all()
    if with_positions:
        assert pos.tolist() == places


@pytest.mark.parametrize("lens", [[1], [2, 1, 3], [64], [63, 65, 1], [0, 5, 0, 0, 130], [200], [128, 127, 129]])
@pytest.mark.parametrize("words", [1, 2, 3, 5])
@pytest.mark.parametrize("deep", [False, True])
def test_lengths_and_words(ops, lens, words, deep):
    _check(ops, *_random(sum(lens) + words, lens, pad=3, deep=deep), words)


@pytest.mark.parametrize("deep", [False, True])
def test_the_longest_trees(ops, deep):
    _check(ops, *_random(3, [1024, 1030, 7], pad=1, deep=deep), 16)


def test_many_requests_strides_and_no_positions(ops):
    gen = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 20, (700,), generator=gen).tolist()
    _check(ops, *_random(4, lens, pad=500), 1, wide=2, with_positions=False)


def test_no_requests_and_no_tokens(ops):
    none = torch.zeros(1, dtype=torch.int32)
    _check(ops, torch.tensor([3, -1], dtype=torch.int32), none, torch.zeros(0, dtype=torch.int32), 1)
    _check(ops, torch.zeros(0, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.ones(2, dtype=torch.int32), 1)
    _check(ops, torch.zeros(0, dtype=torch.int32), none, torch.zeros(0, dtype=torch.int32), 2)


def test_a_context_shorter_than_the_drafts(ops):
    """seq_lens under the drafted tokens: positions below zero, as defined."""
    parents, starts, _ = _random(5, [4, 6])
    _check(ops, parents, starts, torch.tensor([0, 3], dtype=torch.int32), 1)


def test_a_chain_is_causal(ops):
    parents, starts, seq = _random(6, [100], deep=True)
    mask = torch.empty((100, 2), dtype=torch.int64, device=DEV)
    ops.build_draft_tree(parents.to(DEV), starts.to(DEV), seq.to(DEV), mask)
    assert od.mask_of(mask.cpu()) == [(1 << (i + 1)) - 1 for i in range(100)]


@pytest.mark.parametrize("words", [1, 12, 16])
def test_captured_and_replayed_on_other_trees(ops, words):
    """Rows in more LDS than a launch has by itself, captured too."""
    lens = [[64 * words, 3, 0], [1, 64 * words - 40, 30], [0, 0, 5], [200, 1, 64 * words - 300 if words > 9 else 9]]
    T = 64 * words + 300
    i32 = dict(dtype=torch.int32, device=DEV)
    parents, starts, seq = torch.zeros(T, **i32), torch.zeros(4, **i32), torch.zeros(3, **i32)
    mask, pos = (torch.empty(s, dtype=torch.int64, device=DEV) for s in ((T, words), (T,)))
    ops.build_draft_tree(parents, starts, seq, mask, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.build_draft_tree(parents, starts, seq, mask, pos)
    for n, some in enumerate(lens):
        x = _random(50 + n, some, pad=T - sum(some), deep=n % 2 == 0)
        for a, b in zip((parents, starts, seq), x):
            a.copy_(b)
        mask.fill_(77)
        pos.fill_(77)
        graph.replay()
        torch.cuda.synchronize()
        want, places = od.draft_tree(x[0].tolist(), x[1].tolist(), x[2].tolist(), T, words)
        assert torch.equal(mask.cpu(), od.words_of(want, words)) and pos.tolist() == places
