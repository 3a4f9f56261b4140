"""Calls on caches that hold less that few make: many rows beside few, limits far above what is there, two streams at once, a budget that is met already."""
import pytest
import torch

from test_gpu_cache_evict import _case
from test_gpu_key_weights import Weigh, _near
from test_gpu_kv4_attention import Step, near

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("more", [dict(), dict(window=150), dict(softcap=12.0, sink=True)])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (6, 2, 128, 16), (3, 3, 128, 8), (32, 1, 64, 24)])
@pytest.mark.parametrize("packed", [True, False])
def test_weights_of_many_rows_beside_few(packed, n_q, n_kv, d, page, more):
    more = dict(more)
    if more.get("sink"):
        more["sink"] = torch.linspace(-4, 6, n_q)
    step = Weigh([97, 33, 0, 1], [900, 33, 20, 300], n_q, n_kv, d, page, torch.bfloat16, seed=d + n_q, packed=packed)
    got, err = step.weigh(**more)
    assert err[0] == 0
    _near(got, *step.wanted(**more))
    again, _ = step.weigh(**more)
    assert torch.equal(got, again)
    known = [500, 33, 0, 300]
    got, _ = step.weigh(held=known, **more)
    _near(got, *step.wanted(held=known, **more))


@pytest.mark.parametrize("tokens", [1, 12, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_limits_far_above_what_is_there(dtype, tokens):
    step = Weigh([tokens, 1], [260, 60], 8, 2, 64, 16, dtype, seed=3)
    far = dict(max_tokens_per_seq=2 ** 31 - 1, max_keys=2 ** 31 - 1)
    want, _, off, _ = step.want()
    got, err = step.run(**far)
    assert err[0] == 0
    near(got, want, off)
    got, err = step.weigh(**far)
    assert err[0] == 0
    _near(got, *step.wanted())


@pytest.mark.parametrize("tokens", [1, 40])
def test_two_streams_at_once(tokens):
    steps = [Weigh([tokens, 1], [700 + 100 * i, 90], 8, 2, 64, 16, torch.bfloat16, seed=i) for i in range(2)]
    from photon_infer_b200.kernels import ops
    runs = []
    for step in steps:
        runs.append([t.to(DEV) for t in (step.q, step.k, step.v, step.table, step.cu, step.lens, step.before)])

    def work(step, t):
        q, k, v, table, cu, lens, before = t
        out, lse, weights = torch.zeros_like(q), torch.zeros(step.T, 8, device=DEV), before.clone()
        ops.kv4_attention(q, out, k, v, table, cu, lens, err=None, lse=lse, **step.args())
        ops.key_weights(q, weights, k, table, cu, lens, err=None, lse=lse, **step.args())
        ops.key_weights(q, weights, k, table, cu, lens, err=None, **step.args())
        return out, lse, weights

    alone = [work(step, t) for step, t in zip(steps, runs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    both = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                both[i].append(work(steps[i], runs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for results in both[i]:
            assert all(torch.equal(a, b) for a, b in zip(results, alone[i]))


@pytest.mark.parametrize("packed", [True, False])
def test_a_budget_that_is_met_already(packed):
    """The second of two calls finds nothing to do; a third with the same budget after new tokens works on what is left."""
    from photon_infer_b200.kernels import ops
    held, keep = [90, 20, 41], 40
    kv, w, table, _ = _case(held, 2, 2, 64, 16, packed, torch.bfloat16, 5)
    kv, w, table, lens = kv.to(DEV), w.to(DEV), table.to(DEV), torch.tensor(held, dtype=torch.int32, device=DEV)
    new, newer = torch.full_like(lens, -1), torch.full_like(lens, -1)
    call = (3, max(held), keep, 4, 8)
    ops.cache_evict(kv, w, table, lens, new, *call, None)
    assert new.tolist() == [40, 20, 40]
    once, sums = kv.clone(), w.clone()
    kept = torch.full((2, 3, 2, keep), -7, dtype=torch.int32, device=DEV)
    ops.cache_evict(kv, w, table, new, newer, *call, None, kept=kept)
    assert newer.tolist() == [40, 20, 40] and torch.equal(kv, once) and torch.equal(w, sums) and bool((kept == -7).all())


def test_a_budget_of_nothing_and_one_above_all():
    from photon_infer_b200.kernels import ops
    kv, w, table, _ = _case([30, 0], 1, 2, 64, 16, False, torch.float32, 6)
    kv, w, table, lens = kv.to(DEV), w.to(DEV), table.to(DEV), torch.tensor([30, 0], dtype=torch.int32, device=DEV)
    before, sums, new = kv.clone(), w.clone(), torch.full_like(lens, -1)
    for keep, left in ((0, [0, 0]), (31, [30, 0]), (30, [30, 0])):
        ops.cache_evict(kv, w, table, lens, new, 2, 30, keep, 4, 4, None)
        assert new.tolist() == left and torch.equal(kv, before) and torch.equal(w, sums)


def test_one_step_of_each_length_from_one_on():
    """Every length around a tile's and a page's end."""
    for held in (1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257):
        step = Step([1], [held], 8, 2, 128, 8, torch.bfloat16, seed=held)
        want, wanted, off, _ = step.want()
        got, err, lse = step.run(lse=True)
        assert err[0] == 0
        near(got, want, off)
        near(lse, wanted, torch.cat(step.lse_off))
