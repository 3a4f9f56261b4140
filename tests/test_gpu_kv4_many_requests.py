"""As many requests as the tensor-core kernels take, and one more, which go to the general ones."""
import pytest
import torch

from test_gpu_key_weights import Weigh, _near
from test_gpu_kv4_attention import near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests", [1024, 1025, 1500])
@pytest.mark.parametrize("more", [dict(), dict(window=20)])
def test_attention_and_weights(requests, more):
    count, held = [1 + (s % 5 == 0) for s in range(requests)], [2 + s % 37 for s in range(requests)]
    step = Weigh(count, held, 2, 1, 64, 8, torch.bfloat16, seed=requests)
    want, wanted, off, _ = step.want(**more)
    got, err, lse = step.run(lse=True, **more)
    assert err[0] == 0
    near(got, want, off)
    near(lse, wanted, torch.cat(step.lse_off))
    sums, within = step.wanted(**more)
    for known in (None, lse):
        weights, err = step.weigh(lse=known, **more)
        assert err[0] == 0
        # a logarithm in 32 bits, times log2 e, gives its own rounding to the weight
        _near(weights, sums, within + (0 if known is None else sums.abs() * 2.0 ** -20))
