"""Attention over caches in 4 bits: calls of more steps than the tensor-core kernel counts go to another one."""
import torch

from photon_infer_b200.kernels import ops


def _route(tokens, seqs, n_q, n_kv, keys, head_dim=128):
    most = min(tokens, -(-tokens // seqs)) * (n_q // n_kv)
    return ops._kv4_route(torch.bfloat16, head_dim, 16, 1 << 20, seqs, n_kv, most, keys, tokens * n_q, 148)[0]


def test_steps_fit_31_bits():
    # 8 rows and 32 keys a step: 64 requests of 2,048 tokens behind 129,024, 32/8 heads, are 64 * 1,024 * 8 * 4,096 = 2^31 steps
    assert _route(64 * 2048, 64, 32, 8, 131072) == "kv4_attention_rows"
    assert _route(8192, 1, 128, 128, 532480) == "kv4_attention_rows"
    assert _route(8192, 1, 128, 128, 520000) == "kv4_attention_mma"
    # single tokens of very many heads over shared pages
    assert _route(1024, 1024, 512, 512, 262144, 64) != "kv4_attention_mma"
    # what is far below stays
    assert _route(32 * 2048, 32, 32, 8, 131072) == "kv4_attention_mma" and _route(1024, 1024, 32, 8, 1 << 20) == "kv4_attention_mma"


def test_no_route_passes_the_count():
    import random
    rng = random.Random(5)
    seen = 0
    for _ in range(4000):
        seqs, group, n_kv, keys = rng.randint(1, 1024), rng.choice([1, 2, 3, 4, 8, 16, 64]), rng.randint(1, 128), 1 << rng.randint(5, 22)
        counts = [rng.randint(0, 1 << rng.randint(0, 12)) for _ in range(seqs)]
        rows = max(counts) * group
        if rows == 0:
            continue
        name, _, _ = ops._kv4_route(torch.bfloat16, 64, 16, 1000, seqs, n_kv, rows, keys, sum(counts) * group * n_kv, 148)
        tile = 4 if rows <= 4 else 8
        steps = sum(-(-n * group // tile) for n in counts) * n_kv * (keys // 32)
        seen += steps >= (1 << 31) - 1
        assert name != "kv4_attention_mma" or steps < (1 << 31) - 1
    assert seen > 100
