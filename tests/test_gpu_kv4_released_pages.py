"""Pages in front of a window, which the cache gives back: no row sees their keys, and nothing looks for them."""
import pytest
import torch

from test_gpu_kv4_attention import Step, near
from test_gpu_key_weights import Weigh, _near

pytestmark = pytest.mark.gpu


def _release(step, window):
    for s, (n, held) in enumerate(zip(step.count, step.held)):
        front = max(0, held - n - window + 1) // step.page
        step.table[s, :front] = -1
        if front > 1:
            step.table[s, front // 2] = step.pages + 7
    return (step.table[:, 0] < 0).any()


BATCHES = [([1, 1], [700, 90]), ([3, 2], [300, 515]), ([40, 1, 130], [600, 700, 1000]), ([64], [2050])]
SHAPES = [(8, 2, 64, 16), (4, 1, 128, 8), (3, 1, 96, 16), (2, 2, 64, 64)]


@pytest.mark.parametrize("window", [1, 20, 64, 130])
@pytest.mark.parametrize("count,held", BATCHES)
@pytest.mark.parametrize("n_q,n_kv,d,page", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("laid_out", [True, False])
def test_attention(laid_out, dtype, n_q, n_kv, d, page, count, held, window, monkeypatch):
    from photon_infer_b200.kernels import ops
    if not laid_out and dtype == torch.float32:
        pytest.skip("one way only")
    monkeypatch.setattr(ops, "_kv4_few", lambda *sizes: not laid_out)
    step = Step(count, held, n_q, n_kv, d, page, dtype, seed=window + d)
    clean, err = step.run(window=window)
    assert err[0] == 0
    assert _release(step, window)
    got, err = step.run(window=window)
    assert err[0] == 0 and torch.equal(got, clean)
    if not laid_out:
        also, err, _ = step.run(window=window, lse=True)
        assert err[0] == 0 and torch.equal(also, step.run(window=window)[0])


@pytest.mark.parametrize("window", [1, 20, 130])
@pytest.mark.parametrize("count,held", BATCHES)
@pytest.mark.parametrize("n_q,n_kv,d,page", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("packed", [True, False])
def test_weights(packed, dtype, n_q, n_kv, d, page, count, held, window):
    """Without the rows' logarithms and, over 4 bits, with them."""
    step = Weigh(count, held, n_q, n_kv, d, page, dtype, seed=window + d, packed=packed)
    want, off = step.wanted(window=window)
    lse = step.run(lse=True, window=window)[2] if packed else None
    clean = [step.weigh(window=window, lse=x)[0] for x in ([None, lse] if packed else [None])]
    assert _release(step, window)
    for x, before in zip([None, lse], clean):
        got, err = step.weigh(window=window, lse=x)
        assert err[0] == 0 and torch.equal(got, before)
        _near(got, want, off)


def test_keys_without_a_sum_are_looked_for():
    """Whoever says that keys in front of the window have no sum yet has their pages."""
    step = Weigh([2], [300], 8, 2, 64, 16, torch.bfloat16, seed=1, packed=False)
    want, off = step.wanted(held=[40], window=64)
    got, err = step.weigh(held=[40], window=64)
    assert err[0] == 0
    _near(got, want, off)
    step.table[0, 4] = -1
    assert step.weigh(held=[40], window=64)[1][0] == 3
