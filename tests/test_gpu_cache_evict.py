"""Tokens that leave a paged cache: which ones stay, and where their rows go."""
import math

import pytest
import torch

from plain import kv4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _row_view(kv, packed, page, d):
    """The rows of pools [entries, planes, pages, n_kv, ..] as lists of views whose dimension 4 is the place in the page."""
    return list(plain.page_parts(kv, page, d)) if packed else [kv]


def _case(held, entries, n_kv, d, page, packed, dtype, seed, planes=2, values="normal"):
    g = torch.Generator().manual_seed(seed)
    need = [-(-h // page) for h in held]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(held), max(need + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    if packed:
        kv = torch.stack([torch.stack([plain.random_pool(pages, n_kv, page, d, g) for _ in range(planes)]) for _ in range(entries)])
    else:
        kv = torch.randn(entries, planes, pages, n_kv, page, d, generator=g).to(dtype)
    w = torch.rand(entries, pages, n_kv, page, generator=g)
    if values == "ties":
        w = torch.randint(0, 3, w.shape, generator=g).float()
        w = torch.where((w == 0) & (torch.rand(w.shape, generator=g) < 0.5), torch.tensor(-0.0), w)
    elif values == "odd":
        pick = torch.randint(0, 8, w.shape, generator=g)
        for i, v in enumerate((math.nan, math.inf, -math.inf, -1.0, 1e-42, -math.nan)):
            w = torch.where(pick == i, torch.tensor(v), w)
    elif values == "near":
        w = (w.view(torch.int32) % 5 + 0x3F800000).view(torch.float32)
    return kv, w, table, g


def _want(kv, w, table, held, keep, first, last, packed, page, d):
    kv, w, kept = kv.clone(), w.clone(), {}
    entries, _, _, n_kv, _ = w.unsqueeze(1).shape
    parts = _row_view(kv, packed, page, d)
    for e in range(entries):
        for s, n in enumerate(held):
            if n <= keep:
                continue
            at = [(int(table[s, j // page]), j % page) for j in range(n)]
            for h in range(n_kv):
                places = plain.kept_places([float(w[e, p, h, i]) for p, i in at], n, keep, first, last)
                kept[e, s, h] = places
                for x in parts + [w.unsqueeze(1)]:
                    rows = [x[e, :, at[j][0], h, at[j][1]].clone() for j in places]
                    for j, row in enumerate(rows):
                        x[e, :, at[j][0], h, at[j][1]] = row
    if packed:
        kv = torch.cat([p.flatten(4) for p in parts], 4)
    return kv, w, kept


def _bits(x):
    return x.contiguous().view(torch.uint8)


def _run(kv, w, table, held, keep, first, last, S=None, kept=True):
    from photon_infer_b200.kernels import ops
    S = len(held) if S is None else S
    kv, w, err = kv.to(DEV), w.to(DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    lens, places = torch.full((S + 1,), 77, dtype=torch.int32, device=DEV), torch.full((w.shape[0], S, w.shape[2], keep), -5, dtype=torch.int32, device=DEV) if kept else None
    ops.cache_evict(kv, w, table.to(DEV), torch.tensor(held, dtype=torch.int32, device=DEV), lens, S, max(held), keep, first, last, err, kept=places)
    return kv.cpu(), w.cpu(), lens.tolist(), None if places is None else places.cpu(), err.tolist()


SHAPES = [(True, torch.bfloat16, 2, 64, 16), (False, torch.bfloat16, 2, 64, 16), (False, torch.float32, 1, 40, 3), (True, torch.bfloat16, 1, 96, 16), (True, torch.bfloat16, 2, 128, 8),
          (True, torch.float32, 1, 32, 16), (False, torch.bfloat16, 3, 8, 4), (True, torch.bfloat16, 1, 256, 4), (False, torch.float32, 1, 512, 8)]


@pytest.mark.parametrize("held,keep,first,last", [([40], 20, 2, 4), ([1, 65, 300], 64, 4, 16), ([33, 20], 1, 0, 0), ([100], 99, 0, 0), ([9, 500], 8, 8, 8), ([60], 30, 30, 0), ([60], 30, 0, 30),
                                                 ([50, 70], 0, 0, 0), ([700], 650, 600, 3)])
@pytest.mark.parametrize("packed,dtype,n_kv,d,page", SHAPES)
def test_evict(packed, dtype, n_kv, d, page, held, keep, first, last):
    kv, w, table, _ = _case(held, 2, n_kv, d, page, packed, dtype, seed=sum(held) + d)
    want = _want(kv, w, table, held, keep, first, last, packed, page, d)
    got = _run(kv, w, table, held, keep, first, last)
    assert got[4][0] == 0 and got[2] == [min(h, keep) for h in held] + [77]
    for (e, s, h), places in want[2].items():
        assert got[3][e, s, h].tolist() == places
    for s, n in enumerate(held):
        if n <= keep:
            assert bool((got[3][:, s] == -5).all())
    assert torch.equal(got[1], want[1]) and torch.equal(_bits(got[0]), _bits(want[0]))


@pytest.mark.parametrize("values", ["ties", "odd", "near"])
@pytest.mark.parametrize("held,keep", [([900], 300), ([600, 2100], 599)])
def test_sums_that_are_alike_or_odd(values, held, keep):
    kv, w, table, _ = _case(held, 1, 2, 64, 16, True, torch.bfloat16, seed=3, values=values)
    want = _want(kv, w, table, held, keep, 3, 5, True, 16, 64)
    got = _run(kv, w, table, held, keep, 3, 5)
    for (e, s, h), places in want[2].items():
        assert got[3][e, s, h].tolist() == places
    assert torch.equal(_bits(got[1]), _bits(want[1])) and torch.equal(got[0], want[0])


def test_many_keys():
    held, keep = [40000], 33333
    kv, w, table, _ = _case(held, 1, 1, 32, 16, True, torch.bfloat16, seed=4)
    got = _run(kv, w, table, held, keep, 4, 100)
    order = table[0, :2500].long()
    flat = w[0, order, 0].reshape(-1)
    middle = flat[4:39900]
    places = torch.cat([torch.arange(4), 4 + torch.sort(torch.sort(middle, descending=True, stable=True).indices[:keep - 104]).values, torch.arange(39900, 40000)])
    assert torch.equal(got[3][0, 0, 0].long(), places)
    assert torch.equal(got[1][0, order, 0].reshape(-1)[:keep], flat[places])
    for part, mine in zip(_row_view(kv, True, 16, 32), _row_view(got[0], True, 16, 32)):
        old, new = (x[0, :, order, 0].flatten(1, 2) for x in (part, mine))
        assert torch.equal(new[:, :keep], old[:, places]) and torch.equal(new[:, keep:], old[:, keep:])


def test_one_plane_and_no_requests():
    kv, w, table, _ = _case([50], 3, 2, 64, 16, False, torch.bfloat16, seed=6, planes=1)
    want = _want(kv, w, table, [50], 20, 1, 1, False, 16, 64)
    got = _run(kv, w, table, [50], 20, 1, 1, kept=False)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = _run(kv, w, table, [50], 20, 1, 1, S=0, kept=False)
    assert torch.equal(got[0], kv) and got[2] == [77]


def test_a_missing_page():
    """It is recorded, its keys count for nothing and what would come from it stays away; the other request is as it should be."""
    held, keep = [100, 90], 80
    kv, w, table, _ = _case(held, 1, 2, 64, 16, True, torch.bfloat16, seed=8)
    want = _want(kv, w, table, held, keep, 2, 2, True, 16, 64)
    broken = table.clone()
    broken[0, 6] = -1                                       # the last four keys, two of which stay
    got = _run(kv, w, broken, held, keep, 2, 2)
    assert got[4][0] == 3 and got[4][1] == 0
    other = table[1, :6].long()
    assert torch.equal(got[0][:, :, other], want[0][:, :, other]) and torch.equal(got[1][:, other], want[1][:, other])


def test_captured_and_replayed():
    from photon_infer_b200.kernels import ops
    cases = [_case([300, 200], 2, 2, 64, 16, True, torch.bfloat16, seed=s) for s in (21, 22)]
    kv, w, table = (x.to(DEV) for x in cases[0][:3])
    held, lens = torch.tensor([300, 200], dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    call = lambda: ops.cache_evict(kv, w, table, held, lens, 2, 300, 150, 4, 10, None)     # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lengths, case in (([300, 140], cases[1]), ([151, 200], cases[0])):
        for to, of in zip((kv, w, table), case[:3]):
            to.copy_(of)
        held.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        want = _want(case[0], case[1], case[2], lengths, 150, 4, 10, True, 16, 64)
        assert torch.equal(kv.cpu(), want[0]) and torch.equal(w.cpu(), want[1]) and lens.tolist() == [min(x, 150) for x in lengths]


def test_more_keys_than_announced():
    """max_keys only decides where the sums are kept."""
    from photon_infer_b200.kernels import ops
    kv, w, table, _ = _case([2000, 90], 1, 2, 64, 16, True, torch.bfloat16, seed=31)
    want = _want(kv, w, table, [2000, 90], 700, 3, 5, True, 16, 64)
    for announced in (0, 100, 2000, 1 << 20):
        got, sums, lens = kv.to(DEV), w.to(DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
        ops.cache_evict(got, sums, table.to(DEV), torch.tensor([2000, 90], dtype=torch.int32, device=DEV), lens, 2, announced, 700, 3, 5, None)
        assert torch.equal(got.cpu(), want[0]) and torch.equal(sums.cpu(), want[1]) and lens.tolist() == [700, 90]
