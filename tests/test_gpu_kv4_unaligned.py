"""Queries that begin or follow one another off 16-byte boundaries, as sections of other tensors do."""
import pytest
import torch

from test_gpu_kv4_attention import Step, near

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _shifted(q):
    """The same rows one behind the other, from an odd number on."""
    flat = torch.zeros(q.numel() + 1, dtype=q.dtype, device=DEV)
    flat[1:] = q.to(DEV).flatten()
    x = flat[1:].view(q.shape)
    assert x.is_contiguous() and x.data_ptr() % 16
    return x


def _section(q, start, pad):
    """Rows of a wider tensor."""
    wide = torch.zeros(q.shape[0], q.shape[1] + pad, dtype=q.dtype, device=DEV)
    x = wide[:, start:start + q.shape[1]]
    x.copy_(q)
    return x


VIEWS = {"shifted": _shifted, "odd rows": lambda q: _section(q, 0, 3), "odd start": lambda q: _section(q, 1, 8), "both": lambda q: _section(q, 1, 3)}


@pytest.fixture(params=[False, True], ids=["laid-out", "codes"])
def way(request, monkeypatch):
    from photon_infer_b200.kernels import ops
    monkeypatch.setattr(ops, "_kv4_few", lambda *sizes: request.param)


@pytest.mark.parametrize("view", list(VIEWS))
@pytest.mark.parametrize("count,held", [([40], [90]), ([1], [90]), ([33, 1], [33, 200])])
def test_attention(way, view, count, held):
    step = Step(count, held, 8, 2, 64, 16, torch.bfloat16, seed=2)
    got, err = step.run(q=VIEWS[view](step.q))
    want, _, off, _ = step.want()
    assert err[0] == 0
    near(got, want, off)


def test_one_row_of_many_heads(way):
    """A single token whose heads of a key/value head are a prompt's worth of rows."""
    step = Step([1], [90], 64, 2, 64, 16, torch.bfloat16, seed=3)
    want, _, off, _ = step.want()
    for view in VIEWS.values():
        got, err = step.run(q=view(step.q))
        assert err[0] == 0
        near(got, want, off)


@pytest.mark.parametrize("view", list(VIEWS))
@pytest.mark.parametrize("tokens,group", [(1, 32), (40, 4)])
def test_results(way, view, tokens, group):
    """Results into such a view; what lies beside them, and rows behind the last request, stay as they were."""
    step = Step([tokens], [90], 2 * group, 2, 64, 16, torch.bfloat16, seed=5)
    rows, W = tokens + (tokens > 1), 128 * group
    q = torch.zeros(rows, W, dtype=torch.bfloat16)
    q[:tokens] = step.q
    into = VIEWS[view](torch.full((rows, W), 5.0, dtype=torch.bfloat16))
    _, err = step.run(q=q.to(DEV), out=into)
    want, _, off, _ = step.want()
    assert err[0] == 0
    near(into[:tokens], want, off)
    assert bool((into[tokens:] == 5).all())
    if into._base is not None and into._base.dim() == 2:
        beside = into._base.clone()
        beside[:, into.storage_offset():into.storage_offset() + W] = 0
        assert not bool(beside.any())
