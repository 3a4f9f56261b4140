"""Scores bounded far above their size: the bound must not cost their last bits."""
import pytest
import torch

from test_gpu_key_weights import Weigh, _near
from test_gpu_kv4_attention import near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("softcap", [100.0, 250.0, 260.0, 1e4, 1e6, 1e9])
@pytest.mark.parametrize("count,held", [([1], [700]), ([3, 2], [300, 90]), ([40, 1], [200, 70])])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (4, 1, 128, 8)])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_and_weights(dtype, packed, n_q, n_kv, d, page, count, held, softcap, monkeypatch):
    from photon_infer_b200.kernels import ops
    step = Weigh(count, held, n_q, n_kv, d, page, dtype, seed=d + sum(held), packed=packed)
    want, wanted, off, _ = step.want(softcap=softcap)
    sums, within = step.wanted(softcap=softcap)
    # up to 256 a bounded score may be off by 2^-22 of the bound, and a logarithm with it; a weight by the score's and the logarithm's
    slack = softcap * 2.0 ** -22 if softcap <= 256 else 0.0
    for few in (ops._kv4_few, lambda *sizes: False):
        monkeypatch.setattr(ops, "_kv4_few", few)
        got, err = step.run(softcap=softcap)
        assert err[0] == 0
        near(got, want, off)
    got, err, lse = step.run(softcap=softcap, lse=True)
    near(got, want, off)
    near(lse, wanted, torch.cat(step.lse_off) + slack)
    for known in (None, lse) if packed else (None,):
        weights, err = step.weigh(softcap=softcap, lse=known)
        assert err[0] == 0
        _near(weights, sums, within + sums.abs() * (2 * slack + 2.0 ** -20))
