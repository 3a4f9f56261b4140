"""Tree attention and acceptance where a way of sharing out the work could lose something: values that are not finite in one segment behind the other, scores far
below 0; walks of many steps."""
import pytest
import torch

from test_gpu_tree_attention import TOL, Step
from test_gpu_tree_cache import _accept, _case, _run_accept
from test_gpu_tree_routes import ALL, CONTEXT, NODES, WAYS, route                      # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def _rows(step, out):
    return out.view(step.T, step.n_q, step.d).cpu()


@pytest.mark.parametrize("parts", [-5, 1, 5, 11])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("every", [1, 2, 3])
def test_segments_with_such_values_in_turn(route, d, parts, every):     # noqa: F811
    """Blocks that walk many short units, each with few rows, so that most warps have none and are a segment ahead: what a segment had to put back does not
    depend on the segments around it.  parts: blocks that take whole units (below zero) or ranges, which the one long request makes the kernel's choice."""
    route("tree_attention_tc", parts, 1)
    nodes = [1 + i % 3 for i in range(48)]
    step = Step(nodes, [(53 * i) % 200 if i != 20 else 2000 for i in range(48)], 8, 2, d, 16, torch.bfloat16, seed=31)
    clean, _ = step.run()
    hit = torch.zeros(step.T, dtype=torch.bool)
    at = 0
    for s, n in enumerate(nodes):
        if s % every == 0:
            page, slot = step.slot(s, step.context[s])                  # the first node, which all nodes of a request see
            step.v[page, :, slot, 3] = float("nan")
            hit[at:at + n] = True
        at += n
    others = [j for j in range(d) if j != 3]
    for _ in range(10):
        got, err = step.run()
        assert err[0] == 0
        assert bool(torch.isnan(_rows(step, got)[hit][..., 3]).all())
        assert torch.equal(_rows(step, got)[~hit], _rows(step, clean)[~hit]) and torch.equal(_rows(step, got)[..., others], _rows(step, clean)[..., others])


FEW_ROWS = [w for w in WAYS if w[1] != "tree_attention_tc" and w[2] != 13]


@pytest.mark.parametrize("dtype,kernel,parts,cluster", FEW_ROWS, ids=["-".join(str(x).split(".")[-1] for x in w) for w in FEW_ROWS])
@pytest.mark.parametrize("nodes", [[3], [7]])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), -float("inf")])
def test_a_seen_value_where_part_of_a_tile_is_hidden(route, dtype, kernel, parts, cluster, nodes, d, bad):      # noqa: F811
    """Up to 16 and up to 32 rows, whose warps have a part of every tile's keys each: the first keys of the first tile lie before the window, and a block may have that
    tile alone.  One value at a time, in each part of the first and the last tile: the rows that see it have it, and no other number changes."""
    route(kernel, parts, cluster)
    base, window = 855, 256                             # the first tile any row sees begins at 576, the first row's window at 600
    build = lambda: Step(nodes, [base], 4 * 2, 2, d, 16, dtype, seed=43, fan=2)
    clean, _ = build().run(window=window)
    for key in (577, 598, 610, 630, 639, 840, 852, base, base + 2):
        step = build()
        page, slot = step.slot(0, key)
        step.v[page, :, slot, 5] = bad
        got, err = step.run(window=window)
        where = key if key < base else base + int(step.depth[0][key - base])
        sees = torch.tensor([(key < base or bool(step.seen[0][i, key - base])) and where > base + int(step.depth[0][i]) - window for i in range(nodes[0])])
        assert err[0] == 0 and not bool(torch.isfinite(_rows(step, got)[sees][..., 5].float()).any()), key
        assert torch.equal(_rows(step, got)[~sees], _rows(step, clean)[~sees])
        others = [j for j in range(d) if j != 5]
        assert torch.equal(_rows(step, got)[..., others], _rows(step, clean)[..., others])


@ALL
@pytest.mark.parametrize("d", [64, 128])
def test_a_seen_value_beside_a_missing_page(route, dtype, kernel, parts, cluster, d):      # noqa: F811
    """A tile that no mask cuts, of a page that is missing and one with a value that is not finite: the missing keys are left out, the value is not."""
    route(kernel, parts, cluster)
    step = Step([7, 9], [500, 60], 8, 2, d, 16, dtype, seed=44)
    step.table[0, 9] = -1                               # keys 144 .. 159
    clean, err = step.run()
    assert err[0] == 3 and bool(torch.isfinite(clean).all())
    page, slot = step.slot(0, 170)
    step.v[page, :, slot, 5] = float("nan")
    got, err = step.run()
    assert err[0] == 3 and bool(torch.isnan(_rows(step, got)[:7][..., 5].float()).all())
    others = [j for j in range(d) if j != 5]
    assert torch.equal(_rows(step, got)[..., others], _rows(step, clean)[..., others]) and torch.equal(_rows(step, got)[7:], _rows(step, clean)[7:])


@ALL
@pytest.mark.parametrize("d", [64, 128])
def test_seen_values_of_no_weight(route, dtype, kernel, parts, cluster, d):      # noqa: F811
    """A value that is not finite shows in the rows that see it although its score lies 300 below the others', so that its weight, or that of the whole share that has
    this key alone, is 0 in 32 bits: 0 times it is not 0.  In tiles that masks cut and in tiles that they do not; rows that do not see it keep their bits."""
    route(kernel, parts, cluster)
    build = lambda: Step([9, 16], [700, 2300], 8, 2, d, 16, dtype, seed=45)
    step = build()
    step.q.view(step.T, 8, d)[..., 0] = 64.0
    there = ~step.k[..., 0].isnan()
    step.k[..., 0][there] = 0.0
    keys = [(0, 100), (0, 650), (1, 5), (1, 2299), (1, 2301)]
    for s, key in keys:
        page, slot = step.slot(s, key)
        step.k[page, :, slot, 0] = -float(round(300 * d ** 0.5 / 64))
    clean, _ = step.run()
    for s, key in keys:
        page, slot = step.slot(s, key)
        good = step.v[page, :, slot, 3].clone()
        step.v[page, :, slot, 3] = float("inf")
        got, err = step.run()
        step.v[page, :, slot, 3] = good
        sees = torch.zeros(step.T, dtype=torch.bool)
        first, base = (0, 700) if s == 0 else (9, 2300)
        sees[first:first + step.nodes[s]] = True if key < base else step.seen[s][:, key - base]
        assert err[0] == 0 and not bool(torch.isfinite(_rows(step, got)[sees][..., 3].float()).any()), (s, key)
        assert torch.equal(_rows(step, got)[~sees], _rows(step, clean)[~sees])
        others = [j for j in range(d) if j != 3]
        assert torch.equal(_rows(step, got)[..., others], _rows(step, clean)[..., others])


@ALL
@pytest.mark.parametrize("d", [64, 128])
def test_seen_values_in_shares_of_no_weight(route, dtype, kernel, parts, cluster, d):      # noqa: F811
    """The same where a run of keys has such scores, so that some blocks have no others."""
    route(kernel, parts, cluster)
    step = Step([9, 16], [700, 2300], 8, 2, d, 16, dtype, seed=46)
    step.q.view(step.T, 8, d)[..., 0] = 64.0
    there = ~step.k[..., 0].isnan()
    step.k[..., 0][there] = 0.0
    for key in range(64, 1100):
        page, slot = step.slot(1, key)
        step.k[page, :, slot, 0] = -float(round(300 * d ** 0.5 / 64))
    clean, _ = step.run()
    for key in (64, 500, 700, 900, 1099):
        page, slot = step.slot(1, key)
        good = step.v[page, :, slot, 3].clone()
        step.v[page, :, slot, 3] = float("inf")
        got, err = step.run()
        step.v[page, :, slot, 3] = good
        assert err[0] == 0 and not bool(torch.isfinite(_rows(step, got)[9:][..., 3].float()).any()), key
        assert torch.equal(_rows(step, got)[:9], _rows(step, clean)[:9])
        others = [j for j in range(d) if j != 3]
        assert torch.equal(_rows(step, got)[..., others], _rows(step, clean)[..., others])


def _below(step, level):
    """All scores of a step lie around ``-level``: one number of every query is 64, and the same one of every key what ``-level`` wants."""
    step.q.view(step.T, step.n_q, step.d)[..., 0] = 64.0
    there = ~step.k[..., 0].isnan()
    step.k[..., 0][there] = -float(round(level * step.d ** 0.5 / 64))


@ALL
@pytest.mark.parametrize("level", [95, 150, 300])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("with_sink", [False, True])
def test_scores_far_below_zero_in_every_way(route, dtype, kernel, parts, cluster, level, d, with_sink):     # noqa: F811
    """Requests from one key to 5,116: most shares of the short ones are empty, and an empty share has no maximum.  A score is a sum of d products of
    at most 1.2 level + 20 together, each addition off by 2^-23 of that at most (tensor cores cut off); weights and their sum by as much, beside the operator's tolerance."""
    route(kernel, parts, cluster)
    step = Step(NODES, CONTEXT, 8, 2, d, 16, dtype, seed=41)
    _below(step, level)
    sink = torch.randn(8, generator=torch.Generator().manual_seed(5)) * 2 - level if with_sink else None
    got, err = step.run(sink=sink)
    want, largest = step.want(sink=sink)
    off = 2 * (d + 4) * 2.0 ** -23 * (1.2 * level + 20)
    assert err[0] == 0 and float((got.double().cpu() - want).abs().max()) <= (TOL[dtype] + off) * largest


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 80)], ids=["f32", "bf16"])
@pytest.mark.parametrize("level", [95, 150])
def test_scores_far_below_zero_beside_a_long_request(dtype, d, level):
    """The rule's own choice: two requests of 8 nodes, one behind 16,000 keys and one behind 100."""
    step = Step([8, 8], [16000, 100], 32, 8, d, 16, dtype, seed=42)
    _below(step, level)
    got, err = step.run()
    want, largest = step.want()
    off = 2 * (d + 4) * 2.0 ** -23 * (1.2 * level + 20)
    assert err[0] == 0 and float((got.double().cpu() - want).abs().max()) <= (TOL[dtype] + off) * largest


@pytest.mark.parametrize("V", [5, 5000, 40000, 128256, 151936])
def test_long_greedy_walks(V):
    """Chains whose every step has another token, found by another warp of another block: a step's maxima are read by all before they are written again."""
    n = 150
    g = torch.Generator().manual_seed(V)
    logits = torch.rand((2 * n, V), generator=g)
    best = torch.randint(0, V, (2 * n,), generator=g)
    logits[torch.arange(2 * n), best] = 2.0
    best = best.tolist()
    tokens = [0] + best[:n - 1] + [0] + best[n:2 * n - 1]
    parents = (list(range(-1, n - 1))) * 2
    want = ([list(range(n))] * 2, [n] * 2, [best[:n], best[n:]])
    logits = logits.to("cuda:0")
    for _ in range(5):
        assert _run_accept(logits, tokens, parents, [n, n], n) == want


@pytest.mark.parametrize("V", [4096, 32768, 128256, 151936, 262144])
@pytest.mark.parametrize("walk", [False, True])
@pytest.mark.parametrize("below", [0.0, 60.0, 80.0, 86.0, 90.0, 95.0, 100.0])
def test_the_first_of_any_probability(monkeypatch, V, walk, below):
    """u = 0 takes the first token of any probability, in whichever block of a row's cluster it lies: here token 5 with several behind it, ``below`` temperatures under the largest logit,
    which lies at the row's end.  All nodes' logits at once, and as a walk."""
    from photon_infer_b200.kernels import ops
    if walk:
        monkeypatch.setattr(ops, "ACCEPT_AT_ONCE", 0)
    logits = torch.full((3, V), -float("inf"))
    logits[:, [5, 6, 700, 1500]] = 3.0 - below
    logits[:, V - 2] = 3.0
    got = _run_accept(logits.to("cuda:0"), [9, 5, V - 2], [-1, 0, 0], [3], 3, [1.0], [0.0, 0.5 if below > 0 else 0.9, 0.25])
    assert got == ([[0, 1, -1]], [2], [[5, V - 2, -1]])


@pytest.mark.parametrize("V", [131073, 151936, 262144, 500009])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
@pytest.mark.parametrize("walk", [False, True])
def test_vocabularies_that_threads_read_again(monkeypatch, V, temperature, walk):
    """More than 131,072 tokens: a thread has more numbers than it keeps.  Rows on and off 16-byte boundaries, all nodes at once and as a walk."""
    from photon_infer_b200.kernels import ops
    monkeypatch.setattr(ops, "ACCEPT_AT_ONCE", 0 if walk else 1 << 40)
    nodes = [7, 1, 5]
    logits, tokens, parents, uniforms = _case(nodes, V, seed=V, temperature=temperature)
    temps = [temperature, 0.0, temperature]
    want = _accept(logits, tokens, parents, nodes, 6, temps, uniforms)
    for width, at in ((V, 0), (V + 5, 0), (V + 8 - V % 4, 1)):
        rows = torch.zeros((13, width), device="cuda:0")[:, at:at + V].copy_(logits)
        assert _run_accept(rows, tokens, parents, nodes, 6, temps, uniforms) == want
    assert max(want[1]) > 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nodes,context", [([5, 3], [40, 300]), ([30, 17], [40, 900])])
def test_one_query_for_all_nodes(dtype, d, nodes, context):
    """A broadcast query, whose rows are no numbers apart, and a single row with any stride; outputs whose rows overlap are refused."""
    from photon_infer_b200.errors import ErrorCode, PhotonError
    step = Step(nodes, context, 8, 2, d, 16, dtype, seed=47)
    step.q[:] = step.q[:1].clone()
    want, _ = step.run()
    one = step.q[:1].to(dtype).to("cuda:0")
    got, err = step.run(q=one.expand(step.T, -1))
    assert err[0] == 0 and torch.equal(got, want)
    with pytest.raises(PhotonError) as e:
        step.run(out=torch.zeros((1, 8 * d), dtype=dtype, device="cuda:0").expand(step.T, -1))
    assert e.value.code == ErrorCode.SHAPE_MISMATCH
    single = Step([1], [context[1]], 8, 2, d, 16, dtype, seed=48)
    want, _ = single.run()
    row = single.q.to(dtype).to("cuda:0")
    for stride in (0, 1, 3 * 8 * d):
        assert torch.equal(single.run(q=row.as_strided((1, 8 * d), (stride, 1)))[0], want)
