"""Queries that are not finite, over keys of one sign: every score is minus infinity, and yet the row sees something."""
import math

import pytest
import torch

from test_gpu_kv4_attention import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[None, False, True], ids=["rule", "laid-out", "codes"])
def way(request, monkeypatch):
    from photon_infer_b200.kernels import ops
    if request.param is not None:
        monkeypatch.setattr(ops, "_kv4_few", lambda *sizes: request.param)
    return request.param


@pytest.mark.parametrize("more", [dict(), dict(softcap=5.0), dict(window=9), dict(sink=True)])
@pytest.mark.parametrize("tokens,held", [(1, 1), (1, 70), (1, 5000), (3, 3), (40, 40), (40, 2000)])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (4, 1, 128, 8), (3, 1, 96, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_number_is_infinite(way, dtype, n_q, n_kv, d, page, tokens, held, more):
    """The row becomes NaN, and its logarithm; the other rows and heads stay."""
    if way is not None and (dtype == torch.float32 or tokens < 40 or d == 96):
        pytest.skip("one way only")
    more = dict(more)
    if more.get("sink"):
        more["sink"] = torch.linspace(-4, 6, n_q)
    step = Step([tokens, 1], [held, 60], n_q, n_kv, d, page, dtype, seed=tokens + held)
    g = torch.Generator().manual_seed(1)
    codes = page * d // 2
    step.k[:, :, :codes] = (torch.randint(1, 8, (step.pages, n_kv, codes), generator=g) | torch.randint(1, 8, (step.pages, n_kv, codes), generator=g) << 4).to(torch.uint8)
    clean, _ = step.run(**more)
    _, _, clean_lse = step.run(lse=True, **more)
    for row, number in ((0, 5), (tokens - 1, d + 7)):
        keep = step.q.clone()
        for value in (math.inf, -math.inf, math.nan):
            step.q[row, number] = value
            head = number // d
            got, err = step.run(**more)
            also, _, lse = step.run(lse=True, **more)
            assert err[0] == 0
            for x, c, w in ((got, clean, d), (lse, clean_lse, 1)):
                bad = torch.zeros(x.shape, dtype=torch.bool, device=x.device)
                bad[row, head * w:(head + 1) * w] = True
                assert bool(torch.isnan(x[bad].float()).all()), (value, row)
                assert torch.equal(x[~bad], c[~bad])
            assert bool(torch.isnan(also[row, head * d:(head + 1) * d].float()).all())
        step.q = keep


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_row_that_sees_nothing_stays_zero(way, dtype, tokens):
    """With a query that is not finite, too."""
    step = Step([tokens, 1], [90, 60], 8, 2, 64, 16, dtype, seed=11)
    step.table[0] = -1
    step.q[0, 3] = math.inf
    got, err = step.run()
    assert err[0] == 3 and bool((got[:tokens] == 0).all()) and bool(torch.isfinite(got.float()).all())


