"""Attention for trees of drafted tokens (``ops.tree_attention``) against a plain implementation in 64 bits.

Tolerances.  32 bits: a score is off by at most ``d`` roundings of its products, some 1e-5 of the scale of scores here, and so are the
weights; 4e-5 of the largest value seen.  bfloat16: weights rounded to 8 bits (2^-9 of each, so 2^-9 of the largest value at most) and the output rounded
once more (2^-9); 2^-8 of the largest value, and 2 % of that for sums and exponentials."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = {torch.float32: 4e-5, torch.bfloat16: 1.02 * 2.0 ** -8}


class Step:
    """A step of tree decoding with random trees over a paged cache in no order.  Places that no node may read hold NaN."""

    def __init__(self, nodes, context, n_q, n_kv, d, ps, dtype, seed=0, fan=None, spare=0):
        g = torch.Generator().manual_seed(seed)
        self.nodes, self.context, self.n_q, self.n_kv, self.d, self.ps, self.dtype = nodes, context, n_q, n_kv, d, ps, dtype
        self.S, self.T = len(nodes), sum(nodes)
        self.parents, self.seen, self.depth = [], [], []
        for n in nodes:
            parents = [-1] + [int(torch.randint(max(0, i - (fan or i)), i, (), generator=g)) for i in range(1, n)]
            seen, depth = torch.eye(n, dtype=torch.bool), [0] * n
            for i in range(1, n):
                seen[i] |= seen[parents[i]]
                depth[i] = depth[parents[i]] + 1
            self.parents.append(parents); self.seen.append(seen); self.depth.append(torch.tensor(depth))
        total = [n + c for n, c in zip(nodes, context)]
        counts = [-(-t // ps) for t in total]
        self.pages = sum(counts) + 3
        perm = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((self.S, max(counts) + 1), -1, dtype=torch.int32)
        self.k = torch.full((self.pages, n_kv, ps, d), float("nan"))
        self.v = torch.full((self.pages, n_kv, ps, d), float("nan"))
        for s, t in enumerate(total):
            for i in range(counts[s]):
                page = perm.pop()
                used = min(ps, t - i * ps)
                self.k[page, :, :used] = torch.randn(n_kv, used, d, generator=g)
                self.v[page, :, :used] = torch.randn(n_kv, used, d, generator=g)
                self.table[s, i] = page
        self.q = torch.randn(self.T, n_q * d + spare, generator=g).mul_(2.0)

    def slot(self, s, key):
        return int(self.table[s, key // self.ps]), key % self.ps

    def masks(self):
        words = -(-max(self.nodes) // 32)
        out = torch.zeros((self.T, words), dtype=torch.int64)
        at = 0
        for seen in self.seen:
            for i in range(seen.shape[0]):
                for j in seen[i].nonzero().flatten().tolist():
                    out[at + i, j // 32] |= 1 << (j % 32)
            at += seen.shape[0]
        return torch.where(out >= 1 << 31, out - (1 << 32), out).to(torch.int32)

    def positions(self):
        return torch.cat([c + d for c, d in zip(self.context, self.depth)]).int()

    def arguments(self, stride=0):
        cu = torch.tensor([0] + self.nodes).cumsum(0).int()
        lens = torch.tensor([n + c for n, c in zip(self.nodes, self.context)], dtype=torch.int32)
        q = self.q.to(self.dtype).to(DEV)[:, :self.n_q * self.d]
        put = lambda t: t.to(DEV)
        return dict(q=q, k_cache=put(self.k.to(self.dtype)), v_cache=put(self.v.to(self.dtype)), block_table=put(self.table), cu_tokens=put(cu),
                    context_lens=put(lens), positions=put(self.positions()), tree_mask=put(self.masks()), num_seqs=self.S,
                    max_tokens_per_seq=max(self.nodes), max_keys=max(n + c for n, c in zip(self.nodes, self.context)), n_q=self.n_q,
                    n_kv=self.n_kv, head_dim=self.d, scale=self.d ** -0.5)

    def run(self, window=None, sink=None, softcap=None, out=None, **changes):
        from photon_infer_b200.kernels import ops
        a = self.arguments()
        a.update(changes)
        err = torch.zeros(4, dtype=torch.int32, device=DEV)
        out = torch.full((self.T, self.n_q * self.d), 7.0, dtype=self.dtype, device=DEV) if out is None else out
        ops.tree_attention(a.pop("q"), out, a.pop("k_cache"), a.pop("v_cache"), a.pop("block_table"), a.pop("cu_tokens"), a.pop("context_lens"),
                           a.pop("positions"), a.pop("tree_mask"), window=window, err=err, sink=None if sink is None else sink.to(DEV),
                           softcap=softcap, **a)
        return out, err.tolist()

    def want(self, window=None, sink=None, softcap=None, missing=()):
        """In 64 bits from the rounded inputs; ``missing``: (request, page index) whose keys are left out."""
        r = lambda t: t.to(self.dtype).double()
        outs, largest, at = [], 0.0, 0
        for s, (n, c) in enumerate(zip(self.nodes, self.context)):
            L = n + c
            idx = [self.slot(s, j) for j in range(L)]
            pages, slots = torch.tensor([i for i, _ in idx]), torch.tensor([j for _, j in idx])
            k, v = r(self.k)[pages, :, slots], r(self.v)[pages, :, slots]           # [L, n_kv, d]
            where = torch.cat([torch.arange(c), c + self.depth[s]])
            vis = torch.ones((n, L), dtype=torch.bool)
            vis[:, c:] = self.seen[s]
            if window:
                vis &= where[None, :] > where[c:, None] - window
            for ms, mp in missing:
                if ms == s:
                    vis[:, mp * self.ps:(mp + 1) * self.ps] = False
            q = r(self.q[at:at + n, :self.n_q * self.d]).view(n, self.n_q, self.d)
            out = torch.zeros((n, self.n_q, self.d), dtype=torch.float64)
            for h in range(self.n_q):
                g = h // (self.n_q // self.n_kv)
                x = q[:, h] @ k[:, g].nan_to_num(0.0, 0.0, 0.0).T * self.d ** -0.5
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                x = torch.where(vis, x, torch.full_like(x, -math.inf))
                top = x.amax(1, keepdim=True)
                if sink is not None:
                    top = top.clamp(min=float(sink[h]))
                top = torch.where(top == -math.inf, torch.zeros_like(top), top)
                w = torch.exp(x - top)
                z = w.sum(1, keepdim=True) + (torch.exp(sink[h].double() - top) if sink is not None else 0.0)
                clean = v[:, g].nan_to_num(0.0, 0.0, 0.0)
                out[:, h] = (w @ clean) / torch.where(z == 0, torch.ones_like(z), z)
                if vis.any():
                    largest = max(largest, float(clean[vis.any(0)].abs().max()))
            outs.append(out.view(n, self.n_q * self.d))
            at += n
        return torch.cat(outs), largest

    def check(self, missing=(), **rules):
        got, err = self.run(**rules)
        want, largest = self.want(missing=missing, **rules)
        assert bool(torch.isfinite(got).all())
        worst = float((got.double().cpu() - want).abs().max())
        assert worst <= TOL[self.dtype] * max(largest, 1.0), (worst, largest)
        assert (err[0] == 3) == bool(missing), err
        return got


BOTH = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


@BOTH
@pytest.mark.parametrize("n_q,n_kv,d", [(8, 2, 64), (6, 2, 128), (4, 4, 64), (16, 1, 128), (5, 5, 128), (3, 1, 64), (32, 1, 64)])
@pytest.mark.parametrize("nodes,context", [([1], [0]), ([5], [640]), ([1, 33, 7], [0, 63, 64]), ([64, 2], [1, 1200]), ([31, 32, 33, 1], [127, 128, 129, 300]),
                                           ([129], [255])])
def test_trees_against_64_bits(dtype, n_q, n_kv, d, nodes, context):
    """One node to several tiles of rows, contexts that end at, before and behind a tile's end, none at all, heads in groups of odd sizes."""
    Step(nodes, context, n_q, n_kv, d, 16, dtype, seed=sum(nodes) + d).check()


@BOTH
@pytest.mark.parametrize("ps", [1, 5, 8, 16, 32, 48, 64, 128, 256])
@pytest.mark.parametrize("d", [64, 128])
def test_page_sizes(dtype, ps, d):
    """Pages that end inside a tile, at its end and far behind it."""
    Step([9, 20, 1], [0, 333, 77], 8, 2, d, ps, dtype, seed=ps).check()


@BOTH
@pytest.mark.parametrize("d", [8, 16, 40, 65, 80, 96, 192, 256])
def test_head_sizes(dtype, d):
    Step([9, 20], [50, 133], 4, 2, d, 16, dtype, seed=d).check()


@BOTH
@pytest.mark.parametrize("window", [1, 2, 5, 64, 100, 128, 1000])
@pytest.mark.parametrize("d", [64, 128])
def test_windows_follow_each_nodes_path(dtype, window, d):
    """A node's window is counted along its path, so its first key differs from a sibling subtree's; windows inside the tree leave out ancestors."""
    Step([40, 3, 17], [300, 0, 95], 8, 2, d, 16, dtype, seed=window, fan=2).check(window=window)


@BOTH
@pytest.mark.parametrize("rules", [dict(softcap=5.0), dict(sink=True), dict(sink=True, softcap=20.0, window=70)], ids=["cap", "sink", "all"])
@pytest.mark.parametrize("d", [64, 128])
def test_sinks_and_bounded_scores(dtype, rules, d):
    step = Step([12, 40], [200, 31], 8, 2, d, 16, dtype, seed=3)
    rules = dict(rules)
    if rules.get("sink"):
        rules["sink"] = torch.randn(8, generator=torch.Generator().manual_seed(4)) * 3
    step.check(**rules)


@BOTH
@pytest.mark.parametrize("nodes,context,n_q,n_kv,d", [([64, 20, 33], [5000, 30, 2111], 8, 2, 64), ([16], [9000], 8, 1, 128), ([100] * 3, [700] * 3, 32, 2, 128)])
def test_many_keys_shared_out(dtype, nodes, context, n_q, n_kv, d):
    """Keys of a request that several blocks share, requests of very different lengths side by side."""
    Step(nodes, context, n_q, n_kv, d, 16, dtype, seed=len(nodes)).check()


@BOTH
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nodes,context,n_q,n_kv", [([40] * 40, [1600] * 40, 8, 2), ([12, 90, 33], [3000, 20000, 900], 8, 4), ([100] * 3, [700] * 3, 32, 2)])
def test_maxima_that_keep_growing(dtype, d, nodes, context, n_q, n_kv):
    """Scores that get larger along the keys: the running maximum moves in every tile and what was added up is scaled again, in requests whose keys one block
    walks alone and in requests that several share; the same bits every time. """
    step = Step(nodes, context, n_q, n_kv, d, 16, dtype, seed=13)
    for s in range(step.S):
        length = context[s] + nodes[s]
        for i in range(-(-length // 16)):
            step.k[int(step.table[s, i])] *= 1 + 9.0 * i * 16 / length
    first, err = step.run()
    assert err[0] == 0 and bool(torch.isfinite(first).all())
    for _ in range(20):
        assert torch.equal(step.run()[0], first)
    if step.T <= 400:
        want, largest = step.want()
        # scores of up to some 200, summed up in 32 bits in either type, are off by 2e-5 of themselves at most: weights by 4e-3, and their sum as well
        assert float((first.double().cpu() - want).abs().max()) <= (8e-3 + TOL[dtype]) * largest


@BOTH
def test_many_requests(dtype):
    """More requests than a block has threads in a warp, some without context, one without nodes."""
    nodes = [1 + (7 * i) % 19 for i in range(75)]
    context = [(37 * i) % 211 for i in range(75)]
    Step(nodes, context, 8, 2, 64, 16, dtype, seed=9).check()
    step = Step([4, 3, 6], [20, 50, 1], 8, 2, 64, 16, dtype, seed=10)
    want, largest = step.want()
    a = step.arguments()
    # a request of no nodes between the first and the second
    cu = torch.tensor([0, 4, 4, 7, 13], dtype=torch.int32, device=DEV)
    lens = torch.tensor([24, 9, 53, 7], dtype=torch.int32, device=DEV)
    table = torch.cat([a["block_table"][:1], a["block_table"][:1], a["block_table"][1:]])
    got, err = step.run(cu_tokens=cu, context_lens=lens, block_table=table, num_seqs=4)
    assert float((got.double().cpu() - want).abs().max()) <= TOL[dtype] * largest and err[0] == 0


@BOTH
@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_see_nothing_are_zero(dtype, d):
    """A mask of no bits without cached tokens, beside rows that see one key; a sink does not change a row of zeros."""
    step = Step([6, 40], [0, 0], 8, 2, d, 16, dtype, seed=5)
    step.seen[0][2] = False
    step.seen[1][33] = False
    step.seen[1][0] = False
    for sink in (None, torch.full((8,), 2.0), torch.full((8,), -math.inf)):
        got = step.check(sink=sink)
        assert not bool(got[[2, 6, 39]].any())


@BOTH
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, d, bad):
    """Keys and values that are not finite, at a node that only its descendants see, at cached keys before the window of all rows and of some:
    every row that does not see them keeps its bits; a row that sees such a value has it."""
    step = Step([48, 9], [150, 20], 8, 2, d, 16, dtype, seed=6, fan=3)
    window = 60
    clean, _ = step.run(window=window)
    poisoned = torch.zeros(step.T, dtype=torch.bool)
    at, c = 0, step.context[0]
    deepest = int(step.depth[0].max())
    node = 4
    keys = [c + node, c - window + 1, c - window + deepest - 1, 5]
    for key in keys:
        page, slot = step.slot(0, key)
        step.v[page, :, slot, 3] = bad
        step.k[page, :, slot] = step.k[page, :, slot]
        where = int(key if key < c else c + step.depth[0][key - c])
        sees = torch.tensor([(key < c or bool(step.seen[0][i, key - c])) and where > c + int(step.depth[0][i]) - window for i in range(48)])
        poisoned[:48] |= sees
    assert bool(poisoned.any()) and not bool(poisoned[:48].all())
    got, _ = step.run(window=window)
    view = lambda t: t.view(step.T, step.n_q, d).cpu()
    assert torch.equal(view(got)[~poisoned], view(clean)[~poisoned])
    others = [j for j in range(d) if j != 3]
    assert torch.equal(view(got)[..., others], view(clean)[..., others])
    assert not bool(torch.isfinite(view(got)[poisoned][..., 3].float()).any())
    # a key that is not finite, at the node
    page, slot = step.slot(0, c + node)
    step2 = Step([48, 9], [150, 20], 8, 2, d, 16, dtype, seed=6, fan=3)
    step2.k[page, :, slot, 1] = bad
    got, _ = step2.run(window=window)
    sees = torch.cat([step2.seen[0][:, node], torch.zeros(9, dtype=torch.bool)])
    assert torch.equal(view(got)[~sees], view(clean)[~sees])


@BOTH
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nodes,context", [([9, 4], [30, 200]), ([48, 9], [150, 700])])
def test_a_query_that_is_not_finite_stays_in_its_row(dtype, d, nodes, context):
    step = Step(nodes, context, 8, 2, d, 16, dtype, seed=12)
    clean, _ = step.run()
    step.q[3, 2 * d:3 * d] = float("nan")
    got, _ = step.run()
    view = lambda t: t.view(step.T, 8, d)
    assert bool(torch.isnan(view(got)[3, 2].float()).all())
    rest = torch.ones((step.T, 8), dtype=torch.bool, device=DEV)
    rest[3, 2] = False
    assert torch.equal(view(got)[rest], view(clean)[rest])


@BOTH
def test_strides_streams_and_order(dtype):
    """Queries as a view with a row stride, outputs with another; a stream of the caller's; a chain is ordinary causal attention."""
    from photon_infer_b200.kernels import ops
    step = Step([7, 30], [65, 300], 8, 2, 64, 16, dtype, seed=7, fan=1, spare=64)
    want, largest = step.want()
    wide = torch.full((step.T, 8 * 64 + 24), 3.0, dtype=dtype, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = step.run(out=wide[:, :512])
    torch.cuda.current_stream().wait_stream(side)
    assert float((got.double().cpu() - want).abs().max()) <= TOL[dtype] * largest
    assert bool((wide[:, 512:] == 3.0).all())
    a = step.arguments()
    causal = torch.empty((step.T, 512), dtype=dtype, device=DEV)
    seq = torch.tensor([0] * 7 + [1] * 30, dtype=torch.int32, device=DEV)
    ops.paged_attention(a["q"], causal, a["k_cache"], a["v_cache"], a["block_table"], seq, a["positions"], 8, 2, 64, None, a["scale"], None)
    assert float((got.double() - causal.double()).abs().max()) <= 2 * TOL[dtype] * largest


@BOTH
@pytest.mark.parametrize("d", [64, 128])
def test_the_same_bits_again_and_under_a_graph(dtype, d):
    step = Step([33, 9], [1500, 100], 8, 2, d, 16, dtype, seed=8)
    first, _ = step.run()
    again, _ = step.run()
    assert torch.equal(first, again)
    from photon_infer_b200.kernels import ops
    a = step.arguments()
    q, kc, vc = a.pop("q"), a.pop("k_cache"), a.pop("v_cache")
    tables = [a.pop(x) for x in ("block_table", "cu_tokens", "context_lens", "positions", "tree_mask")]
    out = torch.zeros_like(first)
    call = lambda: ops.tree_attention(q, out, kc, vc, *tables, window=None, err=None, **a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    out.zero_()
    graph.replay()
    assert torch.equal(out, first)
    # another length in the same buffers: the grid was chosen from the bounds, the lengths come from the device
    tables[2].copy_(torch.tensor([33 + 900, 109], dtype=torch.int32))
    graph.replay()
    shorter, _ = step.run(context_lens=tables[2])
    assert torch.equal(out, shorter)


@BOTH
@pytest.mark.parametrize("d", [64, 128])
def test_missing_pages_are_left_out_and_reported(dtype, d):
    step = Step([9, 12], [100, 300], 8, 2, d, 16, dtype, seed=11)
    want, largest = step.want(missing=((1, 3),))
    step.table[1, 3] = -1
    got, err = step.run()
    assert err[0] == 3 and bool(torch.isfinite(got).all())
    assert float((got.double().cpu() - want).abs().max()) <= TOL[dtype] * largest


def test_offsets_beyond_32_bits():
    """A pool of more than 2^31 numbers whose last pages are used."""
    from photon_infer_b200.kernels import ops
    for dtype, pages in ((torch.bfloat16, 140000), (torch.float32, 140000)):
        n_kv, ps, d, n = 8, 16, 128, 5
        k = torch.zeros((pages, n_kv, ps, d), dtype=dtype, device=DEV)
        v = torch.zeros_like(k)
        k[-3:].normal_(); v[-3:].normal_()
        assert k.numel() > 2 ** 31
        q = torch.randn((n, n_kv * d), device=DEV).to(dtype)
        table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device=DEV)
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        out = torch.empty_like(q)
        ops.tree_attention(q, out, k, v, table, ints([0, n]), ints([40]), ints([35, 36, 36, 37, 38]), ints([[1], [3], [5], [11], [27]]), num_seqs=1,
                           max_tokens_per_seq=n, max_keys=40, n_q=n_kv, n_kv=n_kv, head_dim=d, window=None, scale=d ** -0.5, err=None)
        keys = torch.cat([k[p].double() for p in (-1, -3, -2)], dim=1)[:, :40]
        vals = torch.cat([v[p].double() for p in (-1, -3, -2)], dim=1)[:, :40]
        seen = torch.ones((n, 40), dtype=torch.bool, device=DEV)
        for i, bits in enumerate((1, 3, 5, 11, 27)):
            seen[i, 35:] = torch.tensor([bool(bits >> j & 1) for j in range(5)], device=DEV)
        x = torch.einsum("thd,hkd->htk", q.double().view(n, n_kv, d), keys) * d ** -0.5
        want = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ vals
        assert float((out.double().view(n, n_kv, d).transpose(0, 1) - want).abs().max()) <= TOL[dtype] * float(vals.abs().max())
        del k, v


def test_refusals():
    from photon_infer_b200.errors import ErrorCode, PhotonError

    def refused(code, **changes):
        step = Step([3, 4], [20, 5], 8, 2, 64, 16, torch.bfloat16, seed=1)
        with pytest.raises(PhotonError) as e:
            step.run(**changes)
        assert e.value.code == code, e.value

    step = Step([3, 4], [20, 5], 8, 2, 64, 16, torch.bfloat16, seed=1)
    a = step.arguments()
    refused(ErrorCode.INVALID_ARGUMENT, q=a["q"].cpu())
    refused(ErrorCode.INVALID_ARGUMENT, q=a["q"].float())
    refused(ErrorCode.SHAPE_MISMATCH, q=a["q"][:, :-1])
    refused(ErrorCode.SHAPE_MISMATCH, k_cache=a["k_cache"][:, :, :, :32])
    refused(ErrorCode.SHAPE_MISMATCH, k_cache=a["k_cache"].transpose(1, 2))
    refused(ErrorCode.INVALID_ARGUMENT, tree_mask=a["tree_mask"].long())
    refused(ErrorCode.SHAPE_MISMATCH, tree_mask=a["tree_mask"], max_tokens_per_seq=33)
    refused(ErrorCode.SHAPE_MISMATCH, positions=a["positions"][:-1])
    refused(ErrorCode.SHAPE_MISMATCH, num_seqs=3)
    refused(ErrorCode.INVALID_ARGUMENT, cu_tokens=a["cu_tokens"].long())
    refused(ErrorCode.UNSUPPORTED_SIZE, n_q=8, n_kv=3)
    refused(ErrorCode.INVALID_ARGUMENT, scale=0.0)
    refused(ErrorCode.INVALID_ARGUMENT, softcap=-1.0)
    refused(ErrorCode.SHAPE_MISMATCH, sink=torch.zeros(7))
