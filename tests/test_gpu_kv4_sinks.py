"""Sinks that weigh nothing: a row that sees nothing is zero all the same."""
import math

import pytest
import torch

from test_gpu_kv4_attention import Step, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,held", [(1, 10), (2, 10), (1, 3000), (40, 40), (40, 3000)])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (4, 1, 128, 8), (3, 1, 96, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_see_nothing(dtype, n_q, n_kv, d, page, tokens, held):
    """The first request has no page, the others have all; a sink of minus infinity, one of a number, none."""
    step = Step([tokens, 1], [held, 70], n_q, n_kv, d, page, dtype, seed=3)
    step.table[0] = -1
    for value in (-math.inf, 2.0):
        sink = torch.full((n_q,), value)
        sink[n_q - 1] = 1.0
        got, err = step.run(sink=sink)
        also, _, lse = step.run(sink=sink, lse=True)
        assert err[0] == 3
        for x in (got, also):
            assert bool((x[:tokens] == 0).all())
        wanted = sink.expand(tokens, n_q)
        seen = lse.cpu()[:tokens]
        # the maximum is held 15 below a row's largest score: numbers of up to 16, rounded three times
        assert bool(((seen == wanted) | ((seen - wanted).abs() <= 2.0 ** -20 + wanted.abs() * 2.0 ** -22)).all())


@pytest.mark.parametrize("tokens", [1, 3, 40])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (3, 1, 96, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_see_something(dtype, n_q, n_kv, d, page, tokens):
    """A sink of minus infinity is none."""
    step = Step([tokens, 1], [400, 70], n_q, n_kv, d, page, dtype, seed=5)
    got, err = step.run(sink=torch.full((n_q,), -math.inf))
    want, _, off, _ = step.want()
    assert err[0] == 0
    near(got, want, off)
