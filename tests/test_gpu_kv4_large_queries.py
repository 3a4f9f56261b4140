"""Queries near the largest numbers that there are, over keys that keep the scores finite."""
import pytest
import torch

from plain import kv4_plain as plain
from test_gpu_kv4_attention import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exponent", [30, 36, 44, 60, 100, 118, 121, 124, 127])
@pytest.mark.parametrize("softcap", [None, 30.0])
@pytest.mark.parametrize("tokens", [1, 2])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_key_takes_all(dtype, d, tokens, softcap, exponent):
    """Queries are positive and so is one key, the first; the others are negative: scores of up to 2^124, so far apart that the first key has all the weight, bounded or not."""
    step = Step([tokens], [300], 4, 2, d, 16, dtype, seed=d + exponent)
    step.q = ((step.q.float().abs() % 0.5 + 0.5) * 2.0 ** exponent).to(dtype)
    n = 16 * d // 2
    g = torch.Generator().manual_seed(2)
    step.k[:, :, :n] = (torch.randint(1, 7, (step.pages, 2, n), generator=g) | torch.randint(1, 7, (step.pages, 2, n), generator=g) << 4).to(torch.uint8)
    step.k[:, :, n:] = 8                                              # 2^-14
    page, slot = int(step.table[0, 0]), 0
    step.k[page, :, slot * d // 2:(slot + 1) * d // 2] = 0x99         # 1
    got, err = step.run(softcap=softcap)
    want = step.rows(0, step.v, True)[:, 0].repeat_interleave(2, 0).flatten().expand(tokens, -1)
    assert err[0] == 0
    if softcap is None:
        assert bool((got.double().cpu() == want).all())
    else:
        # the others have e^-60 of its weight each
        half = torch.finfo(dtype).eps / 2
        assert bool(((got.double().cpu() - want).abs() <= want.abs() * (half + 2.0 ** -21) + 300 * 8.8e-27 * plain.scale_of(104) * 14).all())
