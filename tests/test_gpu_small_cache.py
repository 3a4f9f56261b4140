"""The operators of smaller caches as a program uses them: a prompt, decoded tokens that keep account of their keys, and a request that falls back to its budget."""
import pytest
import torch

from plain import kv4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
N_Q, N_KV, D, PAGE, SCALE = 8, 2, 64, 16, 64 ** -0.5
BUDGET, FIRST, LAST = 72, 4, 16


class Model:
    """What the cache should hold: per head, the rows and sums that are left, in 64 bits."""

    def __init__(self):
        self.k = [[] for _ in range(N_KV)]
        self.v = [[] for _ in range(N_KV)]
        self.w = [[] for _ in range(N_KV)]

    def write(self, k, v):
        for t in range(k.shape[0]):
            for h in range(N_KV):
                for to, x, values in ((self.k, k, False), (self.v, v, True)):
                    bits, scales = plain.row_bits(x[t, h * D:(h + 1) * D].float().tolist(), values)
                    row = torch.tensor([bits + scales], dtype=torch.uint8)
                    to[h].append(plain.numbers(row, 1, D, values)[0, 0])
                self.w[h].append(0.0)

    def attend(self, q, window_rows=None):
        n = q.shape[0]
        k, v = (torch.stack([torch.stack(x) for x in y]) for y in (self.k, self.v))
        return plain.attention(q.view(n, N_Q, D), k, v, n, k.shape[1], N_Q // N_KV, SCALE)

    def weigh(self, p):
        sums = p.view(p.shape[0], N_KV, N_Q // N_KV, -1).sum((0, 2))
        for h in range(N_KV):
            self.w[h] = [a + float(b) for a, b in zip(self.w[h], sums[h])]

    def evict(self):
        held = len(self.w[0])
        for h in range(N_KV):
            stay = plain.kept_places(self.w[h], held, BUDGET, FIRST, LAST)
            for x in (self.k, self.v, self.w):
                x[h] = [x[h][j] for j in stay]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_decode_and_budget(dtype):
    from photon_infer_b200.kernels import ops
    g = torch.Generator().manual_seed(71)
    model, err = Model(), torch.zeros(4, dtype=torch.int32, device=DEV)
    pools = torch.randint(0, 256, (1, 2, 12, N_KV, ops.kv4_page_bytes(PAGE, D)), generator=g, dtype=torch.uint8).to(DEV)      # whatever was there before
    weights = torch.full((1, 12, N_KV, PAGE), float("nan"), device=DEV)
    table = torch.randperm(12, generator=g)[:10].int()[None].to(DEV)
    held = 0
    rounding = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -12         # scores of up to 25, 72 roundings of 2^-24 each, twice

    def step(n, weigh_last):
        nonlocal held
        q, k, v = (torch.randn(n, h * D, generator=g).to(dtype) for h in (N_Q, N_KV, N_KV))
        places = torch.arange(held, held + n, device=DEV)
        slots = table[0].long()[places // PAGE] * PAGE + places % PAGE
        ops.kv4_write(k.to(DEV), v.to(DEV), slots.int(), pools[0, 0], pools[0, 1], N_KV, D, err)
        before, held = held, held + n
        model.write(k, v)
        lens = torch.tensor([held], dtype=torch.int32, device=DEV)
        args = dict(num_seqs=1, max_keys=held, n_q=N_Q, n_kv=N_KV, head_dim=D, window=None, scale=SCALE, err=err)
        cu = lambda m: torch.tensor([0, m], dtype=torch.int32, device=DEV)       # noqa: E731
        out, single = torch.empty(n, N_Q * D, dtype=dtype, device=DEV), n == 1
        lse = torch.empty(n, N_Q, device=DEV) if single else None
        ops.kv4_attention(q.to(DEV), out, pools[0, 0], pools[0, 1], table, cu(n), lens, max_tokens_per_seq=n, lse=lse, **args)
        last = q[-weigh_last:]
        ops.key_weights(last.to(DEV), weights[0], pools[0, 0], table, cu(weigh_last), lens, max_tokens_per_seq=weigh_last, lse=lse,
                        held=torch.tensor([before], dtype=torch.int32, device=DEV), **args)
        want, _, p, mass = model.attend(q)
        assert bool(((out.double().cpu().view(n, N_Q, D) - want).abs() <= (mass + want.abs()) * rounding).all())
        model.weigh(p[-weigh_last:])

    step(80, 9)
    for _ in range(30):
        step(1, 1)
        if held > BUDGET + 20:
            old = torch.tensor([held], dtype=torch.int32, device=DEV)
            new = torch.empty_like(old)
            ops.cache_evict(pools, weights[None, 0], table, old, new, 1, held, BUDGET, FIRST, LAST, err)
            held = int(new)
            model.evict()
            assert held == BUDGET == len(model.w[0])
        places = torch.arange(held)
        sums = weights[0].cpu()[table[0].cpu().long()[places // PAGE], :, places % PAGE].double()          # [held, n_kv]
        assert bool(((sums.t() - torch.tensor(model.w)).abs() <= 3e-3).all())     # sums of up to 12, off by 2.2e-4 of that at most
    assert err[0].item() == 0
