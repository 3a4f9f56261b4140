"""Acceptance of drafted paths and rows and pages moved inside the cache, against plain implementations."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _draw(row, temperature, u):
    """The token of a row of logits, in 64 bits, and how far the number is from its nearest edge (as a part of the sum)."""
    x = row.double()
    if not temperature > 0:
        return int((x == x.max()).nonzero()[0]), 1.0
    p = torch.softmax(x / temperature, 0).cumsum(0)
    i = min(int(torch.searchsorted(p, torch.tensor(u, dtype=torch.float64) * p[-1])), len(p) - 1)
    return i, float((p - u * p[-1]).abs().min())


def _accept(logits, tokens, parents, nodes, D, temperature=None, uniforms=None):
    path, sampled, counts, at = [], [], [], 0
    for s, n in enumerate(nodes):
        node, p, y = 0, [], []
        while node is not None and len(p) < D and n > 0:
            got, margin = _draw(logits[at + node], temperature[s] if temperature is not None else 0.0, uniforms[at + node] if uniforms is not None else 0.0)
            assert margin > 1e-5, "the test's own numbers lie on an edge"
            p.append(node); y.append(got)
            children = [i for i in range(node + 1, n) if parents[at + i] == node and tokens[at + i] == got]
            node = children[0] if children else None
        path.append(p + [-1] * (D - len(p))); sampled.append(y + [-1] * (D - len(y))); counts.append(len(p))
        at += n
    return path, counts, sampled


def _run_accept(logits, tokens, parents, nodes, D, temperature=None, uniforms=None, S=None):
    from photon_infer_b200.kernels import ops
    S = len(nodes) if S is None else S
    path = torch.full((S, D), 99, dtype=torch.int32, device=DEV)
    sampled, counts = torch.full_like(path, 98), torch.full((S,), 97, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0] + list(nodes)).cumsum(0).int().to(DEV)
    ops.tree_accept(logits, _ints(tokens), _ints(parents), cu, S, max(nodes), path, counts, sampled,
                    None if temperature is None else torch.tensor(temperature, device=DEV), None if uniforms is None else torch.tensor(uniforms, device=DEV))
    return path.tolist(), counts.tolist(), sampled.tolist()


def _case(nodes, V, seed, temperature=0.0, follow=0.8):
    """Random trees whose nodes carry, with probability ``follow``, the token that their parent gives."""
    g = torch.Generator().manual_seed(seed)
    T = sum(nodes)
    logits = torch.randn(T, V, generator=g) * 3
    logits[torch.arange(T), torch.randint(0, V, (T,), generator=g)] += 9.0
    uniforms = [float(x) for x in torch.rand(T, generator=g)]
    if temperature > 0:
        for t in range(T):                                   # numbers a thousandth of the sum away from every edge do not depend on the order of sums
            while _draw(logits[t], temperature, uniforms[t])[1] < 1e-4:
                uniforms[t] = float(torch.rand((), generator=g))
    tokens, parents, at = [], [], 0
    for n in nodes:
        for i in range(n):
            p = -1 if i == 0 else int(torch.randint(0, i, (), generator=g))
            parents.append(p)
            y = _draw(logits[at + p], temperature, uniforms[at + p])[0] if i and float(torch.rand((), generator=g)) < follow else int(torch.randint(0, V, (), generator=g))
            tokens.append(y)
        at += n
    return logits, tokens, parents, uniforms


@pytest.mark.parametrize("V", [1, 3, 31, 1000, 1027, 8193, 32000, 128256])
@pytest.mark.parametrize("nodes", [[1], [5], [64, 1, 7], [3] * 20, [300, 2]])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_paths(V, nodes, temperature):
    if V > 10000 and sum(nodes) > 100:
        nodes = nodes[-1:] * 3
    logits, tokens, parents, uniforms = _case(nodes, V, seed=V + len(nodes), temperature=temperature if V > 3 else 0.0)
    temps = [temperature if s % 3 != 1 and V > 3 else 0.0 for s in range(len(nodes))]
    for D in (1, 3, 12):
        want = _accept(logits, tokens, parents, nodes, D, temps, uniforms)
        assert _run_accept(logits.to(DEV), tokens, parents, nodes, D, temps, uniforms) == want
    assert _run_accept(logits.to(DEV), tokens, parents, nodes, 9) == _accept(logits, tokens, parents, nodes, 9)


def test_ties_and_numbers_that_are_not_finite():
    """The first of equal largest logits; a NaN is never the largest; a row of -inf gives token 0; the first of two children with one token."""
    V = 5000
    logits = torch.full((6, V), -1.0)
    logits[0, [7, 4000, 4999]] = 2.0                          # node 0 -> 7
    logits[1] = float("nan"); logits[1, 3210] = -5.0          # node 1 (token 7) -> 3210
    logits[3] = -float("inf")                                 # node 3 -> 0
    logits[4, 4999] = float("inf")                            # node 4 -> 4999
    tokens, parents = [1, 7, 7, 3210, 0, 4999], [-1, 0, 0, 1, 3, 4]
    got = _run_accept(logits.to(DEV), tokens, parents, [6], 8)
    assert got == ([[0, 1, 3, 4, 5, -1, -1, -1]], [5], [[7, 3210, 0, 4999, 0, -1, -1, -1]])


def test_edges_of_the_sum():
    """u = 0 takes the first token that has any probability, u just below 1 the last."""
    V = 4096
    logits = torch.full((2, V), -float("inf"))
    logits[:, 100] = 1.0; logits[:, 3000] = 1.0
    for u, want in ((0.0, 100), (0.25, 100), (0.75, 3000), (1.0 - 2.0 ** -24, 3000)):
        got = _run_accept(logits.to(DEV), [5, 100], [-1, 0], [2], 4, [1.0], [u, 0.75])
        assert got[2][0][0] == want and got[1] == [2 if want == 100 else 1]


def test_parents_out_of_order_are_no_children():
    logits = torch.zeros(4, 64)
    logits[:, 9] = 1.0
    assert _run_accept(logits.to(DEV), [9, 9, 9, 9], [-1, 2, 1, 5], [4], 4) == ([[0, -1, -1, -1]], [1], [[9, -1, -1, -1]])


def test_rows_with_a_stride_and_a_request_without_nodes():
    logits, tokens, parents, _ = _case([4, 6], 777, seed=2)
    wide = torch.zeros(10, 900, device=DEV)
    wide[:, :777] = logits.to(DEV)
    want = _accept(logits, tokens, parents, [4, 0, 6], 5)
    assert _run_accept(wide[:, :777], tokens, parents, [4, 0, 6], 5) == want and want[1][1] == 0


@pytest.mark.parametrize("T,S", [(64, 8), (2048, 32)])
def test_a_batch_of_a_large_vocabulary(T, S):
    """Few logits and many (on the device): greedy walks that go as deep as the tree."""
    V, n = 128256, T // S
    g = torch.Generator(device=DEV).manual_seed(T)
    logits = torch.randn((T, V), generator=g, device=DEV)
    best = logits.argmax(-1).tolist()
    tokens, parents = [0] * T, [-1] * T
    for s in range(S):
        for i in range(1, n):
            parents[s * n + i] = i - 1 if i < 6 else i % 6          # a chain, and further children with the same tokens behind it
            tokens[s * n + i] = best[s * n + parents[s * n + i]]
    want_path, want_y = [], []
    for s in range(S):
        p = [0]
        while len(p) < 6:
            p.append(next(i for i in range(p[-1] + 1, n) if parents[s * n + i] == p[-1]))
        want_path.append(p); want_y.append([best[s * n + i] for i in p])
    assert _run_accept(logits, tokens, parents, [n] * S, 6) == (want_path, [6] * S, want_y)


def test_accept_refusals():
    from photon_infer_b200.errors import ErrorCode, PhotonError
    from photon_infer_b200.kernels import ops
    ok = dict(logits=torch.zeros(3, 8, device=DEV), tokens=_ints([0] * 3), parents=_ints([-1, 0, 0]), cu_tokens=_ints([0, 3]), num_seqs=1, max_tokens_per_seq=3,
              path=_ints([[0, 0]]), counts=_ints([0]), sampled=_ints([[0, 0]]))
    ops.tree_accept(**ok)
    for code, change in ((ErrorCode.INVALID_ARGUMENT, dict(logits=torch.zeros(3, 8, device=DEV).half())), (ErrorCode.INVALID_ARGUMENT, dict(logits=torch.zeros(3, 8))),
                         (ErrorCode.INVALID_ARGUMENT, dict(tokens=_ints([0] * 3).long())), (ErrorCode.SHAPE_MISMATCH, dict(parents=_ints([-1, 0]))),
                         (ErrorCode.SHAPE_MISMATCH, dict(num_seqs=2)), (ErrorCode.SHAPE_MISMATCH, dict(sampled=_ints([[0]]))),
                         (ErrorCode.SHAPE_MISMATCH, dict(temperature=torch.ones(1, device=DEV)))):
        with pytest.raises(PhotonError) as e:
            ops.tree_accept(**dict(ok, **change))
        assert e.value.code == code


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,n_kv,ps,layers", [(64, 8, 16, 3), (128, 2, 8, 2), (3, 1, 5, 1), (10, 3, 16, 2), (7, 2, 4, 1), (100, 1, 1, 2), (576, 1, 64, 2)])
def test_kept_rows(dtype, d, n_kv, ps, layers):
    """Accepted rows that lie where others go, rows that stay, paths of one node, of every node, across pages, beside requests that keep nothing."""
    from photon_infer_b200.kernels import ops
    torch.manual_seed(d)
    nodes, context = [9, 1, 40, 64, 6, 70], [0, 30, 17, 100, 3, 9]
    paths = [[0, 2, 5, 8], [0], [0, 1, 2, 3], list(range(0, 64, 2)), [0], [0] + list(range(2, 70))]
    counts = [4, 1, 4, 32, 0, 69]
    total = [n + c for n, c in zip(nodes, context)]
    per = [-(-t // ps) for t in total]
    pages = sum(per) + 2
    perm = torch.randperm(pages).tolist()
    table = torch.full((6, max(per) + 2), -1, dtype=torch.int32)
    for s in range(6):
        for i in range(per[s]):
            table[s, i] = perm.pop()
    kv = torch.randn(layers, 2, pages, n_kv, ps, d).to(dtype)
    want = kv.clone()
    D = 70
    path = torch.full((6, D), -1, dtype=torch.int32)
    for s in range(6):
        path[s, :len(paths[s])] = torch.tensor(paths[s], dtype=torch.int32)
        at = lambda key: (int(table[s, key // ps]), key % ps)
        for j in range(counts[s]):
            (fp, fs), (tp, ts) = at(context[s] + paths[s][j]), at(context[s] + j)
            want[:, :, tp, :, ts] = kv[:, :, fp, :, fs]
    err = torch.zeros(4, dtype=torch.int32, device=DEV)
    got = kv.to(DEV)
    cu = torch.tensor([0] + nodes).cumsum(0).int().to(DEV)
    ops.cache_keep(got, table.to(DEV), cu, _ints(total), path.to(DEV), _ints(counts), 6, err)
    assert torch.equal(got.cpu(), want) and int(err[0]) == 0
    # a path that points behind the tree or back is recorded, and nothing is read or written for it
    got = kv.to(DEV)
    bad = torch.full((6, 2), -1, dtype=torch.int32, device=DEV)
    bad[0, 1], bad[2, 1] = 9, 0
    ops.cache_keep(got, table.to(DEV), cu, _ints(total), bad, _ints([2, 1, 2, 0, 0, 0]), 6, err)
    assert torch.equal(got.cpu(), kv) and int(err[0]) == 1
    err.zero_()
    hole = table.clone()
    hole[3, (100 + 2) // ps] = -1
    ops.cache_keep(got, hole.to(DEV), cu, _ints(total), path.to(DEV), _ints([0, 0, 0, 2, 0, 0]), 6, err)
    assert int(err[0]) == 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 2, 40, 8, 16, 64), (1, 1, 9, 1, 1, 1), (2, 1, 12, 3, 5, 7), (2, 2, 300, 2, 8, 10), (1, 2, 70, 8, 64, 128)])
def test_copied_pages(dtype, shape):
    from photon_infer_b200.kernels import ops
    torch.manual_seed(shape[2])
    kv = torch.randn(shape).to(dtype)
    order = torch.randperm(shape[2]).tolist()
    for n in {0, 1, shape[2] // 2}:
        pairs = torch.tensor([order[:n], order[n:2 * n]], dtype=torch.int32).T.contiguous()
        want = kv.clone()
        want[:, :, pairs[:, 1].long()] = kv[:, :, pairs[:, 0].long()]
        got, err = kv.to(DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
        ops.cache_copy_pages(got, pairs.to(DEV), err)
        assert torch.equal(got.cpu(), want) and int(err[0]) == 0
    got = kv.to(DEV)
    ops.cache_copy_pages(got, _ints([[0, shape[2]], [-1, 0], [3 % shape[2], 3 % shape[2]]]), err)
    assert torch.equal(got.cpu(), kv) and int(err[0]) == 3


def test_copied_pages_beyond_32_bits():
    """A pool of more than 2^31 numbers in several planes, a first page onto the last."""
    from photon_infer_b200.kernels import ops
    pages = (1 << 16) + 8
    kv = torch.zeros((2, 2, pages, 8, 16, 64), dtype=torch.bfloat16, device=DEV)
    assert kv.numel() > 2 ** 31
    for p in range(4):
        kv.view(4, pages, -1)[p, 3] = p + 1.0
    ops.cache_copy_pages(kv, _ints([[3, pages - 1]]), None)
    flat = kv.view(4, pages, -1)
    assert all(bool((flat[p, -1] == p + 1.0).all()) for p in range(4)) and float(flat[:, 4:-1].abs().max()) == 0


def test_cache_refusals():
    from photon_infer_b200.errors import ErrorCode, PhotonError
    from photon_infer_b200.kernels import ops
    kv = torch.zeros((1, 2, 4, 2, 8, 16), device=DEV)
    for call in (lambda: ops.cache_copy_pages(kv[:, :, :, :, :, :8], _ints([[0, 1]]), None), lambda: ops.cache_copy_pages(kv, _ints([0, 1]), None),
                 lambda: ops.cache_copy_pages(kv[0], _ints([[0, 1]]), None),
                 lambda: ops.cache_keep(kv, _ints([[0, 1]]), _ints([0, 2]), _ints([9]), _ints([[0, 1]]), _ints([2]), 2, None)):
        with pytest.raises(PhotonError) as e:
            call()
        assert e.value.code == ErrorCode.SHAPE_MISMATCH
    with pytest.raises(PhotonError) as e:
        ops.cache_copy_pages(kv, _ints([[0, 1]]).long(), None)
    assert e.value.code == ErrorCode.INVALID_ARGUMENT
    with pytest.raises(PhotonError) as e:
        ops.cache_copy_pages(kv.half(), _ints([[0, 1]]), None)
    assert e.value.code == ErrorCode.INVALID_ARGUMENT
