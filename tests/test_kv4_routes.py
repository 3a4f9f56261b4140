"""Which kernel a call on caches that hold less goes to, and its scratch: rules on sizes and types, checked on the host."""
import random

import torch

from photon_infer_b200.kernels import ops


def test_attention():
    rng = random.Random(1)
    for _ in range(3000):
        dtype, d, page = rng.choice([torch.bfloat16, torch.float32]), rng.choice([32, 64, 96, 128, 256]), rng.choice([2, 8, 16, 24, 64])
        seqs, n_kv, rows, keys, tokens = rng.randint(1, 2000), rng.randint(1, 64), rng.randint(1, 300), rng.randint(1, 200000), rng.randint(1, 500)
        name, parts, floats = ops._kv4_route(dtype, d, page, rng.choice([4, 10 ** 9]), seqs, n_kv, rows, keys, tokens, 148)
        assert parts >= 1
        if name == "kv4_attention_mma":
            assert dtype == torch.bfloat16 and d in (64, 128) and page % 8 == 0 and seqs <= 1024
            # eight warps of a block, each with a tile of rows and a place for what it leaves, and the requests' sums in front
            assert parts <= 4 * 148 and floats == 8 * parts * (4 if rows <= 4 else 8) * (d + 2) + seqs + 1
        else:
            assert (name == "kv4_attention_rows") == (rows > 24 and seqs * n_kv * -(-rows // 8) * -(-keys // 128) > 4 * 148) and name in ("kv4_attention", "kv4_attention_rows")
            assert parts <= 64 and floats == (tokens * parts * (d + 2) if parts > 1 else 0)


def test_few_rows_stay_with_the_codes():
    few = lambda **k: ops._kv4_few(**dict(dict(head_dim=128, page_size=16, num_seqs=1, n_kv=8, rows=32, keys=6000), **k))
    assert few() and few(head_dim=64) and few(rows=17, keys=100000)
    assert not few(rows=2048) and not few(num_seqs=16, rows=256) and not few(head_dim=256) and not few(page_size=4) and not few(num_seqs=1025)


def test_weights():
    rng = random.Random(2)
    seen = set()
    for _ in range(4000):
        dtype, d, page, packed, known = rng.choice([torch.bfloat16, torch.float32]), rng.choice([32, 64, 96, 128]), rng.choice([4, 8, 16]), rng.random() < 0.5, rng.random() < 0.5
        seqs, n_kv, rows, keys, all_rows = rng.randint(1, 2000), rng.randint(1, 64), rng.randint(1, 300), rng.randint(1, 200000), rng.randint(1, 5000)
        name, parts, floats, keep = ops._key_weights_route(dtype, d, page, 1000, packed, known, seqs, n_kv, rows, keys, all_rows, 148)
        seen.add(name)
        assert parts >= 1
        if name == "kv4_key_weights":
            assert packed and known and rows <= 8 and page % 8 == 0 and seqs <= 1024 and floats == 0
        elif name in ("key_weights", "key_weights_rows"):
            assert (dtype, d) not in ((torch.bfloat16, 64), (torch.bfloat16, 128)) and not keep
            assert (name == "key_weights") == (rows <= 8) and floats == all_rows * (2 * parts + (0 if rows <= 8 else 1))
        else:
            assert dtype == torch.bfloat16 and d in (64, 128) and (name == "key_weights_tc") == (rows > 32)
            assert floats == all_rows * (2 * parts + 1 + (keys if keep else 0)) and (not keep or (rows <= 16 and not known and floats <= (1 << 26) + all_rows * (2 * parts + 1)))
    assert seen == {"key_weights", "key_weights_rows", "key_weights_mma", "key_weights_tc", "kv4_key_weights"}
