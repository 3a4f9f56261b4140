"""Prompt portions over values of which many are not finite: the rows that see one, in its group's numbers, and no others, in a time of the attention's size."""
import pytest
import torch

from test_gpu_kv4_attention import Step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def laid_out(monkeypatch):
    from photon_infer_b200.kernels import ops
    monkeypatch.setattr(ops, "_kv4_few", lambda *sizes: False)


def _break(step, s, key, group):
    page, slot = int(step.table[s, key // step.page]), key % step.page
    step.v[page, :, step.page * step.d // 2 + slot * (step.d // 32) + group] = 255


@pytest.mark.parametrize("window", [None, 1, 7, 64, 1000])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (4, 1, 128, 8), (2, 2, 64, 32)])
def test_which_rows(n_q, n_kv, d, page, window):
    """A few of all keys, in one group or another, of requests of any length, beside a decoded token."""
    count, held = [70, 1, 130, 33], [200, 50, 131, 33]
    step = Step(count, held, n_q, n_kv, d, page, torch.bfloat16, seed=d)
    clean, _ = step.run(window=window)
    for share in (0.004, 0.05, 1.0):
        keep = step.v.clone()
        bad = torch.zeros(step.T, d // 32, dtype=torch.bool)
        at = 0
        for s, n in enumerate(count):
            for key in range(held[s]):
                for group in range(d // 32):
                    if float(torch.rand((), generator=step.g)) >= share:
                        continue
                    _break(step, s, key, group)
                    for i in range(n):
                        place = held[s] - n + i
                        if key <= place and (window is None or key > place - window):
                            bad[at + i, group] = True
            at += n
        got, err = step.run(window=window)
        assert err[0] == 0
        got = got.cpu().view(step.T, n_q, d // 32, 32)
        mask = bad[:, None, :, None].expand_as(got)
        assert bool(torch.isnan(got[mask].float()).all())
        assert torch.equal(got[~mask], clean.cpu().view(got.shape)[~mask])
        step.v = keep


@pytest.mark.parametrize("window", [None, 512])
def test_all_of_them(window):
    """2,048 tokens behind 2,048: one pass over the rows beside the attention, and not one for every key that is broken."""
    from photon_infer_b200.kernels import ops
    step = Step([2048], [4096], 8, 2, 128, 16, torch.bfloat16, seed=7)
    device = {n: getattr(step, n).to(DEV) for n in ("q", "k", "v", "table", "cu", "lens")}
    out = torch.empty(2048, 1024, dtype=torch.bfloat16, device=DEV)

    def run(v):
        ops.kv4_attention(device["q"], out, device["k"], v, device["table"], device["cu"], device["lens"], err=None, **step.args(window=window))

    broken = device["v"].clone()
    broken[:, :, 16 * 64:] = 255
    times = []
    for v in (device["v"], broken):
        run(v)
        torch.cuda.synchronize()
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(3):
            run(v)
        end.record()
        torch.cuda.synchronize()
        times.append(begin.elapsed_time(end) / 3)
    assert bool(torch.isnan(out.float()).all())
    # the host's share of a call is the same; without one store a number the second takes hundreds of times the first
    assert times[1] <= 10 * times[0], times
