"""Weights of keys under queries that are not finite, over keys of one sign: every score is minus infinity, and yet the row sees the keys."""
import math

import pytest
import torch

from test_gpu_key_weights import Weigh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("more", [dict(), dict(softcap=5.0), dict(window=9), dict(sink=True)])
@pytest.mark.parametrize("tokens,held", [(1, 1), (1, 400), (3, 300), (6, 700), (40, 400)])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (4, 1, 128, 8), (3, 1, 96, 16)])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_number_is_infinite(dtype, packed, n_q, n_kv, d, page, tokens, held, more):
    """The keys that the row sees have NaN, for its key/value head; the others keep their sums."""
    more = dict(more)
    if more.get("sink"):
        more["sink"] = torch.linspace(-4, 6, n_q)
    step = Weigh([tokens, 1], [held, 60], n_q, n_kv, d, page, dtype, seed=tokens + held, packed=packed)
    g = torch.Generator().manual_seed(1)
    codes = page * d // 2
    step.k[:, :, :codes] = (torch.randint(1, 8, (step.pages, n_kv, codes), generator=g) | torch.randint(1, 8, (step.pages, n_kv, codes), generator=g) << 4).to(torch.uint8)
    lse = step.run(lse=True, **more)[2] if packed else None
    clean = step.weigh(**more)[0]
    clean_known = step.weigh(lse=lse, **more)[0] if packed else None
    for row, head in ((0, 0), (tokens - 1, n_q - 1)):
        place = held - tokens + row
        bad = torch.zeros(step.before.shape, dtype=torch.bool)
        for key in range(held):
            if key <= place and ("window" not in more or key > place - more["window"]):
                bad[int(step.table[0, key // page]), head * n_kv // n_q, key % page] = True
        keep = step.q.clone()
        for value in (math.inf, -math.inf, math.nan):
            step.q[row, head * d + 5] = value
            results = [(step.weigh(**more)[0], clean)]
            if packed:
                results.append((step.weigh(lse=step.run(lse=True, **more)[2], **more)[0], clean_known))
            for got, before in results:
                assert bool(torch.isnan(got[bad]).all()), value
                assert torch.equal(got[~bad], before[~bad])
        step.q = keep
