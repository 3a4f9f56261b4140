"""Every way in which tree attention shares out its work, on the same steps: whole units, ranges, clusters of blocks, shares that a second kernel joins.  The
choice between them (``ops._tree_route``) goes by sizes, so that each test of the operator sees one of them; here each is asked for.  Tolerances are the operator's."""

import pytest
import torch

from test_gpu_tree_attention import TOL, Step

pytestmark = pytest.mark.gpu

# requests from one key, and less than a tile for every block of a cluster, to many tiles
NODES, CONTEXT = [9, 1, 14, 3, 16], [0, 0, 70, 700, 5100]


@pytest.fixture
def route(monkeypatch):
    from photon_infer_b200.kernels import ops

    def use(kernel, parts, cluster):
        def chosen(dtype, head_dim, group, page_size, cache_rows, aligned, num_seqs, n_kv, rows, keys, sms):
            units = num_seqs * n_kv * -(-rows // (128 // group * group))
            if kernel == "tree_attention_tc" and cluster > 1:
                return kernel, units * cluster, cluster
            return kernel, -min(units, 2 * sms) if parts == "whole" else parts, 1
        monkeypatch.setattr(ops, "_tree_route", chosen)
    return use


TC = [("tree_attention_tc", "whole", 1), ("tree_attention_tc", 7, 1), ("tree_attention_tc", 290, 1)] + [("tree_attention_tc", 0, n) for n in range(2, 9)]
FEW = [("tree_attention_few", n, 1) for n in range(1, 9)]
GENERAL = [("tree_attention", n, 1) for n in (1, 2, 3, 5, 8, 13)]
WAYS = [(torch.bfloat16, *w) for w in TC + FEW + GENERAL] + [(torch.float32, *w) for w in GENERAL]
ALL = pytest.mark.parametrize("dtype,kernel,parts,cluster", WAYS, ids=["-".join(str(x).split(".")[-1] for x in w) for w in WAYS])


@ALL
@pytest.mark.parametrize("d", [64, 128])
def test_every_way_gives_the_operator(route, dtype, kernel, parts, cluster, d):
    route(kernel, parts, cluster)
    step = Step(NODES, CONTEXT, 8, 2, d, 16, dtype, seed=21)
    first = step.check()
    for _ in range(5):
        assert torch.equal(step.run()[0], first)


@ALL
@pytest.mark.parametrize("d", [64, 128])
def test_windows_sinks_and_bounds_in_every_way(route, dtype, kernel, parts, cluster, d):
    route(kernel, parts, cluster)
    sink = torch.randn(6, generator=torch.Generator().manual_seed(4)) * 3
    Step(NODES, CONTEXT, 6, 3, d, 8, dtype, seed=22, fan=2).check(window=333, sink=sink, softcap=9.0)
    Step(NODES, CONTEXT, 6, 3, d, 64, dtype, seed=23, fan=2).check(window=3)


@ALL
def test_nothing_to_see_in_every_way(route, dtype, kernel, parts, cluster):
    """Requests without nodes, and rows whose masks have no bits."""
    route(kernel, parts, cluster)
    step = Step([6, 16], [0, 0], 8, 2, 64, 16, dtype, seed=24)
    step.seen[0][2] = False
    step.seen[1][9] = False
    for sink in (None, torch.full((8,), 2.0)):
        assert not bool(step.check(sink=sink)[[2, 15]].any())
    step = Step([4, 3, 6], [20, 700, 1], 8, 2, 64, 16, dtype, seed=25)
    want, largest = step.want()
    a = step.arguments()
    cu = torch.tensor([0, 0, 4, 7, 13, 13], dtype=torch.int32, device="cuda:0")
    lens = torch.tensor([50, 24, 703, 7, 0], dtype=torch.int32, device="cuda:0")
    table = torch.cat([a["block_table"][:1], a["block_table"], a["block_table"][:1]])
    got, err = step.run(cu_tokens=cu, context_lens=lens, block_table=table, num_seqs=5)
    assert float((got.double().cpu() - want).abs().max()) <= TOL[dtype] * largest and err[0] == 0


@ALL
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_hidden_values_in_every_way(route, dtype, kernel, parts, cluster, bad):
    """Values that are not finite reach the rows that see them and leave the others' bits, in whichever block's part they lie."""
    route(kernel, parts, cluster)
    step = Step([16, 9], [900, 20], 8, 2, 64, 16, dtype, seed=26, fan=3)
    window = 500
    clean, _ = step.run(window=window)
    poisoned = torch.zeros(step.T, dtype=torch.bool)
    for key in (900 + 4, 900 - window + 1, 5, 600):
        page, slot = step.slot(0, key)
        step.v[page, :, slot, 3 if key != 600 else 7] = bad
        if key != 600:
            where = int(key if key < 900 else 900 + step.depth[0][key - 900])
            poisoned[:16] |= torch.tensor([(key < 900 or bool(step.seen[0][i, key - 900])) and where > 900 + int(step.depth[0][i]) - window for i in range(16)])
    got, _ = step.run(window=window)
    view = lambda t: t.view(step.T, 8, 64).cpu()
    assert bool(poisoned.any()) and not bool(poisoned.all())
    assert torch.equal(view(got)[~poisoned][..., 3], view(clean)[~poisoned][..., 3])
    assert not bool(torch.isfinite(view(got)[poisoned][..., 3].float()).any())
    assert not bool(torch.isfinite(view(got)[:16][..., 7].float()).any()) and torch.equal(view(got)[16:][..., 7], view(clean)[16:][..., 7])
    others = [j for j in range(64) if j not in (3, 7)]
    assert torch.equal(view(got)[..., others], view(clean)[..., others])


@ALL
def test_missing_pages_in_every_way(route, dtype, kernel, parts, cluster):
    route(kernel, parts, cluster)
    step = Step([9, 12], [100, 900], 8, 2, 128, 16, dtype, seed=27)
    want, largest = step.want(missing=((1, 3), (1, 40)))
    step.table[1, 3] = -1
    step.table[1, 40] = step.pages + 5
    got, err = step.run()
    assert err[0] == 3 and bool(torch.isfinite(got).all())
    assert float((got.double().cpu() - want).abs().max()) <= TOL[dtype] * largest


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.float32, 128), (torch.float32, 200), (torch.bfloat16, 40), (torch.bfloat16, 96)])
@pytest.mark.parametrize("most", [3, 20])
def test_many_small_requests(dtype, d, most):
    """More row tiles than the chip has SMs, of up to 16 rows and of more."""
    nodes = [1 + i % most for i in range(60)]
    Step(nodes, [(29 * i) % 150 for i in range(60)], 4, 4, d, 16, dtype, seed=29).check()


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 40)])
@pytest.mark.parametrize("most,keys", [(0, 0), (16, 0), (40, 1000)])
def test_no_requests(dtype, d, most, keys):
    """A step of no requests, or of no nodes, leaves the output as it is."""
    step = Step([16, 9], [900, 20], 8, 2, d, 16, dtype, seed=30)
    a = step.arguments()
    bound = dict(max_tokens_per_seq=most, max_keys=keys, tree_mask=torch.zeros((step.T, 2), dtype=torch.int32, device="cuda:0"))
    got, err = step.run(num_seqs=0, **bound)
    assert bool((got == 7.0).all()) and err[0] == 0
    zero = torch.zeros(3, dtype=torch.int32, device="cuda:0")
    got, err = step.run(cu_tokens=zero, context_lens=zero[:2], **bound)
    assert bool((got == 7.0).all()) and err[0] == 0
    out = torch.empty((0, 8 * d), dtype=dtype, device="cuda:0")
    step.run(q=a["q"][:0], out=out, cu_tokens=zero, context_lens=zero[:2], **bound)


def test_ways_that_the_entry_points_refuse(route):
    from photon_infer_b200.errors import ErrorCode, PhotonError
    from photon_infer_b200.kernels import ops
    step = Step([9, 12], [100, 900], 8, 2, 64, 16, torch.bfloat16, seed=28)

    def refused(answer, code):
        ops._tree_route = lambda *a: answer
        with pytest.raises(PhotonError) as e:
            step.run()
        assert e.value.code == code
    route("tree_attention", 1, 1)                       # put back at the end
    refused(("tree_attention_tc", 13, 2), ErrorCode.INVALID_ARGUMENT)
    refused(("tree_attention_tc", 64, 16), ErrorCode.INVALID_ARGUMENT)
    refused(("tree_attention_tc", 400, 1), ErrorCode.INVALID_ARGUMENT)
    refused(("tree_attention_few", 9, 1), ErrorCode.INVALID_ARGUMENT)
    refused(("tree_attention", 0, 1), ErrorCode.INVALID_ARGUMENT)
