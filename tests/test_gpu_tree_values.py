"""Tree attention over scores and values where a way of sharing out the work could lose something: values that are not finite in one segment behind the other."""
import pytest
import torch

from test_gpu_tree_attention import Step
from test_gpu_tree_routes import route                      # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def _rows(step, out):
    return out.view(step.T, step.n_q, step.d).cpu()


@pytest.mark.parametrize("parts", [-5, 1, 5, 11])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("every", [1, 2, 3])
def test_segments_with_such_values_in_turn(route, d, parts, every):     # noqa: F811
    """Blocks that walk many short units, each with few rows, so that most warps have none and are a segment ahead: what a segment had to put back does not
    depend on the segments around it.  parts: blocks that take whole units (below zero) or ranges, which the one long request makes the kernel's choice."""
    route("tree_attention_tc", parts, 1)
    nodes = [1 + i % 3 for i in range(48)]
    step = Step(nodes, [(53 * i) % 200 if i != 20 else 2000 for i in range(48)], 8, 2, d, 16, torch.bfloat16, seed=31)
    clean, _ = step.run()
    hit = torch.zeros(step.T, dtype=torch.bool)
    at = 0
    for s, n in enumerate(nodes):
        if s % every == 0:
            page, slot = step.slot(s, step.context[s])                  # the first node, which all nodes of a request see
            step.v[page, :, slot, 3] = float("nan")
            hit[at:at + n] = True
        at += n
    others = [j for j in range(d) if j != 3]
    for _ in range(10):
        got, err = step.run()
        assert err[0] == 0
        assert bool(torch.isnan(_rows(step, got)[hit][..., 3]).all())
        assert torch.equal(_rows(step, got)[~hit], _rows(step, clean)[~hit]) and torch.equal(_rows(step, got)[..., others], _rows(step, clean)[..., others])
