"""What cached keys got of a softmax, added beside them, against the definition in 64 bits."""
import math

import pytest
import torch

from plain import kv4_plain as plain
from test_gpu_kv4_attention import Step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Weigh(Step):
    """A step over a cache in 4 bits, or over a plain one with the same numbers."""

    def __init__(self, *args, packed=True, **kw):
        super().__init__(*args, **kw)
        self.packed = packed
        self.before = torch.rand(self.pages, self.n_kv, self.page, generator=self.g)

    def cache(self):
        return self.k if self.packed else plain.numbers(self.k, self.page, self.d, False).to(self.dtype)

    def weigh(self, held=None, lse=None, q=None, **more):
        from photon_infer_b200.kernels import ops
        weights, err = self.before.to(DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
        more = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in more.items()}
        ops.key_weights(self.q.to(DEV) if q is None else q, weights, self.cache().to(DEV), self.table.to(DEV), self.cu.to(DEV), self.lens.to(DEV), err=err,
                        held=None if held is None else torch.tensor(held, dtype=torch.int32, device=DEV), lse=lse, **self.args(**more))
        return weights.cpu(), err.tolist()

    def wanted(self, held=None, **more):
        """The weights, and what each may be off by: every term by its score's and its row's sum's roundings."""
        _, _, _, weights = self.want(**more)
        want, off = self.before.double().clone(), torch.zeros(self.before.shape, dtype=torch.float64)
        for s, p in enumerate(weights):
            if self.count[s] == 0:
                continue
            known = held[s] if held is not None else self.held[s] - self.count[s]
            sums = p.view(self.count[s], self.n_kv, -1, self.held[s]).sum((0, 2))
            terms = self.count[s] * self.n_q // self.n_kv
            at = int(self.cu[s])
            q, k = self.q[at:at + self.count[s]].double().abs().max(), self.rows(s, self.k, False).abs().sum(-1).max()
            part = 2 * (q * k * self.d ** -0.5 * (self.d + 8) * 2.0 ** -24 + (self.held[s] + 32) * 2.0 ** -24)
            for key in range(self.held[s]):
                page, slot = int(self.table[s, key // self.page]), key % self.page
                old = want[page, :, slot] if key < known else 0.0
                want[page, :, slot] = old + sums[:, key]
                off[page, :, slot] = sums[:, key] * part + (want[page, :, slot] * (terms + 2)) * 2.0 ** -24
        return want, off


def _near(got, want, off):
    assert bool(((got.double() - want).abs() <= off).all()), float(((got.double() - want).abs() - off).max())


@pytest.mark.parametrize("count,held", [([1], [1]), ([1, 1, 1], [5, 300, 64]), ([1, 0, 3, 2], [700, 9, 3, 131]), ([33], [400]), ([17, 64], [120, 64])])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (6, 2, 128, 16), (3, 1, 96, 16), (2, 2, 64, 32), (16, 1, 128, 8)])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights(dtype, packed, n_q, n_kv, d, page, count, held):
    step = Weigh(count, held, n_q, n_kv, d, page, dtype, seed=d + sum(held), packed=packed)
    got, err = step.weigh()
    assert err[0] == 0
    _near(got, *step.wanted())
    again, _ = step.weigh()
    assert torch.equal(got, again)
    known = [max(0, h - n - 2) if i % 2 else h for i, (n, h) in enumerate(zip(count, held))]
    got, _ = step.weigh(held=known)
    _near(got, *step.wanted(held=known))


@pytest.mark.parametrize("more", [dict(window=64), dict(window=1), dict(softcap=5.0), dict(sink=True), dict(window=100, softcap=20.0, sink=True)])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks(dtype, packed, more):
    more = dict(more)
    if more.get("sink"):
        more["sink"] = torch.linspace(-4, 6, 8)
    step = Weigh([1, 3, 40], [1, 300, 215], 8, 2, 64, 16, dtype, seed=7, packed=packed)
    got, err = step.weigh(**more)
    assert err[0] == 0
    _near(got, *step.wanted(**more))


@pytest.mark.parametrize("more", [dict(), dict(window=90, softcap=20.0, sink=True)])
@pytest.mark.parametrize("tokens", [1, 3, 9])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (4, 1, 128, 8), (3, 1, 96, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_behind_the_attention_of_the_same_queries(dtype, n_q, n_kv, d, page, tokens, more):
    more = dict(more)
    if more.get("sink"):
        more["sink"] = torch.linspace(-4, 6, n_q)
    step = Weigh([tokens, 1], [400, 150], n_q, n_kv, d, page, dtype, seed=9)
    _, _, lse = step.run(lse=True, **more)
    got, _ = step.weigh(lse=lse, **more)
    _near(got, *step.wanted(**more))


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_plain_caches_of_other_sizes(dtype, packed):
    """Heads of 40 (a plain cache takes multiples of 8) and pages of 3; 40 rows a head."""
    from photon_infer_b200.kernels import ops
    if packed:
        pytest.skip("4 bits take multiples of 32")
    g = torch.Generator().manual_seed(5)
    n_q, n_kv, d, page, held, n = 4, 2, 40, 3, 50, 20
    k = torch.randn(18, n_kv, page, d, generator=g).to(dtype)
    q = torch.randn(n, n_q * d, generator=g).to(dtype)
    table = torch.randperm(18, generator=g)[:17].int()[None]
    weights = torch.zeros(18, n_kv, page, device=DEV)
    ops.key_weights(q.to(DEV), weights, k.to(DEV), table.to(DEV), torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.tensor([held], dtype=torch.int32, device=DEV),
                    1, n, held, n_q, n_kv, d, None, d ** -0.5, None)
    rows = k[table[0].long()].transpose(0, 1).reshape(n_kv, -1, d)[:, :held]
    _, _, p, _ = plain.attention(q.view(n, n_q, d), rows, None, n, held, 2, d ** -0.5)
    got = weights.cpu()[table[0].long()].transpose(0, 1).reshape(n_kv, -1)
    want = p.view(n, n_kv, 2, held).sum((0, 2))
    part = 2 * (q.double().abs().max() * rows.double().abs().sum(-1).max() * d ** -0.5 * (d + 8) + held + 32) * 2.0 ** -24
    assert bool(((got[:, :held].double() - want).abs() <= want * (part + 42 * 2.0 ** -24)).all()) and bool((got[:, held:] == 0).all())


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_missing_pages_and_what_is_not_finite(dtype, packed, tokens):
    step = Weigh([tokens, 1], [250, 60], 8, 2, 64, 16, dtype, seed=11, packed=packed)
    clean, _ = step.weigh()
    T, W = step.T, 8 * 64
    wide = torch.zeros(T + 3, W + 3, dtype=dtype, device=DEV)
    wide[:T, 3:] = step.q.to(DEV)
    got, _ = step.weigh(q=wide[:, 3:])
    assert torch.equal(got, clean)
    # what lies behind the last key is not read
    page, slot = int(step.table[0, 250 // 16]), 250 % 16 + 1
    step.k[page, :, 16 * 32 + slot * 2] = 255
    assert torch.equal(step.weigh()[0], clean)
    # a NaN among request 0's keys: its rows' weights are, the other request's are not
    page, slot = int(step.table[0, 2]), 5
    step.k[page, :, 16 * 32 + slot * 2] = 255
    got, _ = step.weigh()
    mine = torch.zeros(step.pages, dtype=torch.bool)
    mine[step.table[0, :16].long()] = True
    assert torch.equal(got[~mine], clean[~mine])
    assert bool(torch.isnan(got[page, :, slot]).all())
    step.table[0, 2] = -1
    got, err = step.weigh()
    assert err[0] == 3 and torch.equal(got[page], step.before[page]) and bool(torch.isfinite(got).all()) and torch.equal(got[~mine], clean[~mine])


def test_captured_and_replayed():
    from photon_infer_b200.kernels import ops
    step = Weigh([1, 1], [250, 60], 8, 2, 64, 16, torch.bfloat16, seed=13)
    t = [x.to(DEV) for x in (step.q, step.before, step.k, step.table, step.cu, step.lens)]
    call = lambda: ops.key_weights(*t, err=None, **step.args())       # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    t[1].copy_(step.before)
    graph.replay()
    first = t[1].cpu()
    _near(first, *step.wanted())
    step.before = first.clone()
    graph.replay()
    _near(t[1].cpu(), *step.wanted())
