"""Queries of the weights of keys that begin or follow one another off 16-byte boundaries."""
import pytest
import torch

from test_gpu_key_weights import Weigh, _near
from test_gpu_kv4_unaligned import VIEWS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("view", list(VIEWS))
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("n_q,n_kv,d", [(8, 2, 64), (4, 1, 128), (80, 2, 64)])
@pytest.mark.parametrize("count,held", [([1], [90]), ([3, 1], [90, 200]), ([40], [90])])
def test_weights(view, packed, n_q, n_kv, d, count, held):
    step = Weigh(count, held, n_q, n_kv, d, 16, torch.bfloat16, seed=4, packed=packed)
    got, err = step.weigh(q=VIEWS[view](step.q))
    assert err[0] == 0
    _near(got, *step.wanted())
