"""Drafts from a request's own tokens, and the layout of a tree, on the host."""
import numpy as np
import pytest

from photon_infer_b200.engine.drafting import lookup_tree
from photon_infer_b200.engine.runner import tree_layout
from photon_infer_b200.errors import ErrorCode, PhotonError


def _paths(tokens, parents):
    out = set()
    for i in range(len(tokens)):
        path, n = [], i
        while n > 0:
            path.append(tokens[n])
            n = parents[n]
        out.add(tuple(reversed(path)))
    return out


def test_lookup_follows_earlier_occurrences():
    #         0  1  2  3  4  5  6  7  8  9
    tokens = [7, 1, 2, 3, 9, 1, 2, 4, 1, 2]
    tree, parents = lookup_tree(tokens, 32, 3, ngram=2)
    assert tree[0] == 2 and parents[0] == -1
    assert _paths(tree, parents) >= {(4, 1, 2), (3, 9, 1)}
    assert tree[1] == 4                                 # the latest occurrence first
    assert all(0 <= p < i for i, p in enumerate(parents) if i)
    assert max(len(p) for p in _paths(tree, parents)) == 3


def test_lookup_bounds():
    tokens = [1, 2, 1, 3, 1, 4, 1]
    assert lookup_tree(tokens, 1, 4) == ([1], [-1])
    assert lookup_tree(tokens, 32, 0) == ([1], [-1])
    assert lookup_tree([5], 8, 4) == ([5], [-1])
    tree, parents = lookup_tree(tokens, 3, 2)
    assert len(tree) == 3
    tree, parents = lookup_tree(tokens, 32, 2)
    siblings = [(p, t) for p, t in zip(parents, tree)]
    assert len(siblings) == len(set(siblings))          # one child for a token


@pytest.mark.parametrize("n,words", [(1, 1), (5, 1), (32, 1), (33, 2), (70, 3)])
def test_layout(n, words):
    rng = np.random.default_rng(n)
    parents = [-1] + [int(rng.integers(0, i)) for i in range(1, n)]
    depth, mask = tree_layout(parents, words)
    assert mask.shape == (n, words) and mask.dtype == np.int32
    for i in range(n):
        sees, d, j = {i}, 0, i
        while parents[j] >= 0:
            j = parents[j]
            sees.add(j)
            d += 1
        bits = [(int(mask[i, k // 32]) >> (k % 32)) & 1 for k in range(words * 32)]
        assert {k for k, b in enumerate(bits) if b} == sees and depth[i] == d


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 2, 0], [-1, -1], [-1, -2]])
def test_layout_refuses_what_is_no_tree(parents):
    with pytest.raises(PhotonError) as e:
        tree_layout(parents, 1)
    assert e.value.code == ErrorCode.INVALID_ARGUMENT
