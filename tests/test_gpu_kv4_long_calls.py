"""Lengths on the device that are more work than the tensor-core kernel counts: recorded, and nothing is done."""
import pytest
import torch

from test_gpu_kv4_attention import Step, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
def test_lengths_beyond_the_limits(d):
    step = Step([1, 40], [70, 90], 8, 2, d, 16, torch.bfloat16, seed=d)
    held = step.lens.clone()
    step.lens[1] = 2147483647
    got, err, lse = step.run(lse=True)
    assert err[0] == 5 and bool((got == 7).all()) and bool((lse == 9).all())
    step.lens = held
    got, err, lse = step.run(lse=True)
    want, wanted, off, _ = step.want()
    assert err[0] == 0
    near(got, want, off)
    near(lse, wanted, torch.cat(step.lse_off))


def test_the_general_kernels_take_such_calls(monkeypatch):
    """Their results where the tensor-core kernel's count is taken as full."""
    from photon_infer_b200.kernels import ops
    route = ops._kv4_route
    monkeypatch.setattr(ops, "_kv4_route", lambda dtype, *sizes: route(torch.float32, *sizes))
    for count, held in (([1, 2], [300, 70]), ([40, 130], [600, 1200])):
        step = Step(count, held, 8, 2, 64, 16, torch.bfloat16, seed=9)
        got, err, lse = step.run(lse=True, sink=torch.linspace(-4, 6, 8), window=100, softcap=20.0)
        want, wanted, off, _ = step.want(sink=torch.linspace(-4, 6, 8), window=100, softcap=20.0)
        assert err[0] == 0
        near(got, want, off)
        near(lse, wanted, torch.cat(step.lse_off))
