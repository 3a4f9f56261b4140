"""Attention of many rows in 32 bits over a cache in 4 bits: the kernel for much work, at sizes that would go to the other one as well, and by itself."""
import pytest
import torch

import test_gpu_kv4_attention as few
from test_gpu_kv4_attention import DEV, Step, near

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[1, 3])
def routed(request, monkeypatch):
    """All that is not the tensor cores' goes to the kernel for many rows, with the keys in one share or in three."""
    from photon_infer_b200.kernels import ops
    rule = ops._kv4_route

    def route(dtype, d, page, page_heads, seqs, n_kv, rows, keys, all_rows, sms):
        found = rule(dtype, d, page, page_heads, seqs, n_kv, rows, keys, all_rows, sms)
        if found[0] == "kv4_attention_mma":
            return found
        return "kv4_attention_rows", request.param, all_rows * request.param * (d + 2) if request.param > 1 else 0

    monkeypatch.setattr(ops, "_kv4_route", route)


@pytest.mark.parametrize("count,held", [([1], [1]), ([40], [40]), ([17, 1, 33], [200, 90, 33]), ([1, 70, 0, 5], [600, 450, 3, 5])])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (4, 1, 128, 8), (3, 1, 96, 16), (40, 1, 64, 16), (1, 1, 256, 4), (6, 3, 32, 16), (5, 1, 160, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompts(routed, dtype, n_q, n_kv, d, page, count, held):
    step = Step(count, held, n_q, n_kv, d, page, dtype, seed=13)
    got, err = step.run()
    want, wanted, off, _ = step.want()
    assert err[0] == 0
    near(got, want, off)
    got, err, lse = step.run(lse=True)
    near(got, want, off)
    near(lse, wanted, torch.cat(step.lse_off))
    again, _, _ = step.run(lse=True)
    assert torch.equal(got, again)


@pytest.mark.parametrize("more", [dict(window=64), dict(window=1), dict(softcap=5.0), dict(sink=True), dict(window=100, softcap=20.0, sink=True)])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (3, 1, 96, 16)])
def test_masks(routed, n_q, n_kv, d, page, more):
    few.test_masks(torch.float32, n_q, n_kv, d, page, more)


@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (4, 1, 128, 8), (3, 1, 96, 16)])
@pytest.mark.parametrize("tokens", [2, 40])
def test_what_is_not_finite(routed, n_q, n_kv, d, page, tokens):
    few.test_values_that_are_not_finite(torch.float32, n_q, n_kv, d, page, tokens)
    few.test_keys_that_are_not_finite(torch.float32, n_q, n_kv, d, page, tokens)


@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_a_missing_page_and_strides(routed, tokens):
    few.test_a_missing_page(torch.float32, tokens)
    few.test_strides_and_rows_behind_the_last(torch.float32, tokens)


@pytest.mark.parametrize("n_q,n_kv,d", [(32, 8, 64), (6, 2, 128), (3, 1, 256)])
def test_much_work(n_q, n_kv, d):
    from photon_infer_b200.kernels import ops
    step = Step([150, 31, 7], [1500, 900, 300], n_q, n_kv, d, 16, torch.float32, seed=d)
    name, _, _ = ops._kv4_route(torch.float32, d, 16, 10 ** 6, 3, n_kv, 150 * n_q // n_kv, 1500, step.T * n_q, torch.cuda.get_device_properties(0).multi_processor_count)
    assert name == "kv4_attention_rows"
    got, err = step.run()
    want, _, off, _ = step.want()
    assert err[0] == 0
    near(got, want, off)


def test_a_prompt_of_16400_tokens():
    step = Step([16400], [16400], 32, 8, 32, 16, torch.float32, seed=1)
    got, err = step.run()
    assert err[0] == 0 and bool(torch.isfinite(got).all())
    step.count, step.T, step.q, step.cu = [3], 3, step.q[-3:], torch.tensor([0, 3], dtype=torch.int32)
    want, _, off, _ = step.want()
    near(got[-3:], want, off)


def test_captured_and_replayed():
    from photon_infer_b200.kernels import ops
    step = Step([150, 31], [1500, 900], 32, 8, 64, 16, torch.float32, seed=4)
    t = [x.to(DEV) for x in (step.q, step.k, step.v, step.table, step.cu, step.lens)]
    out = torch.zeros_like(t[0])
    call = lambda: ops.kv4_attention(t[0], out, *t[1:], err=None, **step.args())      # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    t[0].mul_(0.5)
    step.q = step.q * 0.5
    out.zero_()
    graph.replay()
    want, _, off, _ = step.want()
    near(out, want, off)
