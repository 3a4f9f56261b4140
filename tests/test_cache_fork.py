"""Pages with several holders, forks, kept nodes and packed pools, on the host."""
import random

import pytest
import torch

from photon_infer_b200.cache import NO_PAGE, CacheManager, PagePool
from photon_infer_b200.errors import ErrorCode, PhotonError
from photon_infer_b200.parts.base import PagedCacheSpec, StateSpec

FULL = PagedCacheSpec(2, 16, None)
WIN = PagedCacheSpec(2, 16, 24)
SPLIT = PagedCacheSpec(2, 16, None, value_dim=24)


def _manager(num_pages=16, page_size=8, max_sequences=4, specs=(FULL,), device=None, state=False):
    needs = [(s, StateSpec((3,)) if state and i == 0 else None) for i, s in enumerate(specs)]
    return CacheManager(needs, [None] * len(specs), page_size, num_pages, max_sequences, torch.float32, device)


def test_a_shared_page_is_free_with_its_last_holder():
    pool = PagePool(3)
    a, b = pool.allocate(), pool.allocate()
    assert pool.share(a) == a and pool.holders(a) == 2 and pool.holders(b) == 1
    pool.free(a)
    assert pool.is_allocated(a) and pool.num_free == 1
    pool.free(a)
    assert not pool.is_allocated(a) and pool.num_free == 2 and pool.allocate() == a
    with pytest.raises(PhotonError) as e:
        pool.share(2)
    assert e.value.code == ErrorCode.INVALID_STATE
    pool.free(b)
    with pytest.raises(PhotonError) as e:
        pool.free(b)
    assert e.value.code == ErrorCode.DOUBLE_FREE


@pytest.mark.parametrize("length,shared,own", [(0, 0, 0), (1, 0, 1), (8, 1, 0), (20, 2, 1), (24, 3, 0)])
def test_forks_share_full_pages(length, shared, own):
    m = _manager()
    m.add_request("a")
    m.extend("a", length + 9)                           # pages taken ahead are not forked
    m.commit("a", length)
    m.fork("a", ["b", "c"])
    ta, tb, tc = (m.groups[0].tables[r] for r in "abc")
    assert len(tb) == len(tc) == shared + own and tb[:shared] == tc[:shared] == ta[:shared]
    if own:
        assert len({ta[shared], tb[-1], tc[-1]}) == 3
    assert m.length("b") == m.length("c") == length
    m.check_consistency()
    m.extend("b", 10)
    m.check_consistency()
    m.free_request("a")
    m.check_consistency()
    m.free_request("c")
    m.free_request("b")
    m.check_consistency()
    assert m.free_pages() == [16]


def test_forks_are_all_or_nothing():
    m = _manager(num_pages=3, max_sequences=3)
    m.add_request("a")
    m.extend("a", 12)
    m.commit("a", 12)                                   # two pages, the second partly filled: one page is left
    for new, code in ((["b", "c"], ErrorCode.OUT_OF_MEMORY), (["b", "b"], ErrorCode.INVALID_STATE), (["a"], ErrorCode.INVALID_STATE),
                      (["b", "c", "d"], ErrorCode.OUT_OF_MEMORY)):
        with pytest.raises(PhotonError) as e:
            m.fork("a", new)
        assert e.value.code == code
        assert m.live_requests() == ["a"] and m.free_pages() == [1] and m.states.num_free == 2
        m.check_consistency()
    with pytest.raises(PhotonError) as e:
        m.fork("x", ["b"])
    assert e.value.code == ErrorCode.INVALID_STATE
    m.fork("a", ["b"])
    assert m.free_pages() == [0]


def test_kept_nodes_give_the_other_pages_back():
    m = _manager()
    m.add_request("a")
    m.extend("a", 6)
    m.commit("a", 6)
    m.extend("a", 30)                                   # a tree of 30 nodes
    assert m.groups[0].pages_held("a") == 5
    m.commit_kept("a", 3)
    assert m.length("a") == 9 and m.groups[0].pages_held("a") == 2
    m.extend("a", 7)
    m.commit_kept("a", 7)                               # every node, up to a page's end
    assert m.length("a") == 16 and m.groups[0].pages_held("a") == 2
    m.extend("a", 4)
    m.commit_kept("a", 0)
    assert m.groups[0].pages_held("a") == 2
    m.check_consistency()


def test_windows_forks_and_trees_in_random_order():
    rng = random.Random(5)
    m = _manager(num_pages=60, max_sequences=9, specs=(WIN, FULL))
    live, n = [], 0
    for _ in range(600):
        what = rng.random()
        if what < 0.15 and len(live) < 9:
            live.append(n); m.add_request(n); n += 1
        elif what < 0.3 and live and len(live) < 8:
            new = [n, n + 1][:rng.randint(1, 2)]
            if m.groups[0].pool.num_free >= 2 and m.groups[1].pool.num_free >= 2:
                m.fork(rng.choice(live), new)
                live += new; n += 2
        elif what < 0.75 and live:
            r, k = rng.choice(live), rng.randint(1, 20)
            if m.try_extend(r, k):
                if rng.random() < 0.5:
                    m.commit(r, k)
                else:
                    m.commit_kept(r, rng.randint(1, k))
        elif what < 0.85 and live:
            m.free_request(live.pop(rng.randrange(len(live))))
        else:
            m.pack()
            for g in m.groups:
                held = [p for t in g.tables.values() for p in t if p != NO_PAGE]
                assert max(held, default=-1) < g.pool.num_allocated
        m.check_consistency()
        for r in live:
            for g in m.groups:                          # a page that may still be written belongs to one request alone
                t, length = g.tables[r], m.length(r)
                for i, page in enumerate(t):
                    if page != NO_PAGE and (i + 1) * g.page_size > length:
                        assert g.pool.holders(page) == 1
    for r in list(live):
        m.free_request(r)
    assert m.free_pages() == [60, 60]


def test_inconsistent_tables_are_seen():
    m = _manager()
    m.add_request("a")
    m.extend("a", 20)
    m.groups[0].tables["a"].append(m.groups[0].tables["a"][0])
    with pytest.raises(PhotonError):
        m.check_consistency()


@pytest.mark.gpu
def test_contents_follow_forks_kept_rows_and_packing():
    """What requests have cached, read back through their tables, while pools fork, keep and pack; values of another width, states."""
    dev = torch.device("cuda:0")
    m = _manager(num_pages=40, max_sequences=6, specs=(FULL, SPLIT, FULL), device=dev, state=True)
    rng = random.Random(3)
    torch.manual_seed(3)
    truth = {}

    def rows(g, t):                                     # [tokens, ...] of a table
        return [torch.cat([pools[:, :, p] for p in t], dim=3) for pools in g.pools()]

    def write(r, start, n):
        for gi, g in enumerate(m.groups):
            for pi, pools in enumerate(g.pools()):
                for j in range(start, start + n):
                    page, slot = g.tables[r][j // 8], j % 8
                    x = torch.randn(pools.shape[:2] + (pools.shape[3], pools.shape[5]), device=dev)
                    pools[:, :, page, :, slot] = x
                    truth[r].setdefault((gi, pi), {})[j] = x

    def check():
        for r in m.live_requests():
            for gi, g in enumerate(m.groups):
                for pi, pools in enumerate(g.pools()):
                    for j in range(m.length(r)):
                        assert torch.equal(pools[:, :, g.tables[r][j // 8], :, j % 8], truth[r][gi, pi][j])

    for r in ("a", "b"):
        truth[r] = {}
        m.add_request(r)
        m.extend(r, 21)
        write(r, 0, 21)
        m.commit(r, 21)
    m.states.tensors[0][m.states.slot_of("a")] = 5.0
    m.fork("a", ["c", "d"])
    assert all(float(m.states.tensors[0][m.states.slot_of(r)].sum()) == 15.0 for r in "acd")
    for r in "cd":
        truth[r] = {k: dict(v) for k, v in truth["a"].items()}
    check()
    for r in "acdb":                                    # trees of different sizes, of which some nodes stay
        n = rng.randint(5, 20)
        m.extend(r, n)
        write(r, 21, n)
        path = [0] + sorted(rng.sample(range(1, n), 3))
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
        from photon_infer_b200.kernels import ops
        for gi, g in enumerate(m.groups):
            for pi, pools in enumerate(g.pools()):
                ops.cache_keep(pools, ints([g.tables[r]]), ints([0, n]), ints([21 + n]), ints([path]), ints([4]), 1, None)
                old = truth[r][gi, pi]
                for j, node in enumerate(path):
                    old[21 + j] = old[21 + node]
        m.commit_kept(r, 4)
    check()
    m.free_request("b")
    assert m.pack() > 0
    check()
    m.check_consistency()
